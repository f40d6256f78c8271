"""MLX-semantics quantized ops on torch CUDA tensors, executed by libmoe_b200.so.

Mirrors the reference's Array methods (crates/mlx-core/src/ops.rs):
  quantized_matmul(x, w, scales, biases, transpose, group_size, bits)   ops.rs:592-637
  gather_qmm(x, w, scales, biases, lhs_indices, rhs_indices, transpose,
             group_size, bits, sorted_indices)                           ops.rs:830-891
  fast_rms_norm(x, weight, eps)                                          ops.rs:691-701
  fast_rope(x, dims, traditional, base, scale, offset, freqs)            mlx_fast_rope
Failures raise MlxError("<mlx fn> failed (rc=N): reason"), the Error::Mlx message
of crates/mlx-core/src/array.rs:43-49.

Tensor conventions: activations and scales/biases are torch.bfloat16 (quantized_matmul,
gated_ffn: or float16; fast_rope: or float32 too); packed weights
are 32-bit words (torch.int32 holding the uint32 bit patterns, or torch.uint32);
indices are 32-bit integers (uint32 semantics). All tensors live on one CUDA device
and calls are ordered on torch's current stream.
"""
from __future__ import annotations

import ctypes as C
import functools
import importlib
import os
import warnings

import torch

from ._lib import (ACT_GELU, ACT_SILU, DTYPE_BF16, DTYPE_F16, DTYPE_F32, FfnConfig, FfnWeights, MlxError, QWeight,
                   RopeConfig, context_for, library)

_calls = None


def load_calls():
    """The dense operators' calls without ctypes (build.py), where they were built for this torch;
    what they decline is made here."""
    global _calls
    _calls = None
    if not os.path.exists(os.path.join(os.path.dirname(os.path.abspath(__file__)), "_calls.so")):
        return None
    try:
        importlib.invalidate_caches()
        module = importlib.import_module(__package__ + "._calls")
        if not torch.__version__.startswith(module.torch_version):
            raise ImportError(f"built for torch {module.torch_version}")
    except ImportError as e:
        warnings.warn(f"_calls.so is not used, the calls go through ctypes: {e}")
        return None
    module.set_error(MlxError)
    _calls = module
    return module


load_calls()

_WORD_DTYPES = {torch.int32} | ({torch.uint32} if hasattr(torch, "uint32") else set())


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _ctx(t: torch.Tensor):
    if not t.is_cuda:
        raise MlxError("moe_b200", 1, "tensors must be on a CUDA device")
    ctx = context_for(t.device.index)
    ctx.bind_stream(torch.cuda.current_stream(t.device).cuda_stream)
    return ctx


def _need(t, dtypes, name):
    if t is None:
        return
    if t.dtype not in dtypes:
        raise MlxError("moe_b200", 1, f"{name}: dtype {t.dtype} not in {sorted(map(str, dtypes))}")
    if not t.is_contiguous():
        raise MlxError("moe_b200", 1, f"{name}: must be contiguous")


_DTYPES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16, torch.float32: DTYPE_F32}
_I64x3 = C.c_int64 * 3
ACTIVATIONS = {"silu": ACT_SILU, "gelu": ACT_GELU}


# The raw handle of torch's current stream on a device; through the stream object where this
# torch has no direct way (that costs a few microseconds of each call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _context(fn, t):
    """This thread's context of the tensor's device, on torch's current stream."""
    index = t.get_device()
    if index < 0:
        raise MlxError(fn, 1, "tensors must be on a CUDA device")
    ctx = context_for(index)
    ctx.bind_stream(_raw_stream(index))
    return ctx


def _no_graph(fn, *tensors):
    """Refuses inputs whose gradient torch would look for: the calls record no graph."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise MlxError(fn, 1, "an input requires a gradient, and this call records no graph: make it under "
                              "torch.no_grad(); its gradient has a call of its own")


def _workspace(nbytes, device):
    # from torch's allocator on the current stream: each call and each captured graph has its own
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=4096)
def _qmm_workspace(dtype, M, K, N, transpose, group_size, bits):
    need = C.c_size_t()
    rc = library().moe_quantized_matmul_workspace(dtype, M, K, N, transpose, group_size, bits, C.byref(need))
    if rc:
        raise MlxError("mlx_quantized_matmul", rc, f"unsupported call: M={M}, K={K}, N={N}")
    return need.value


@functools.lru_cache(maxsize=4096)
def _ffn_workspace(hidden, inter, group_size, dtype, T, backward):
    need = C.c_size_t()
    cfg = FfnConfig(hidden, inter, ACT_SILU, group_size, 4, dtype)
    rc = library().moe_gated_ffn_workspace(C.byref(cfg), T, backward, C.byref(need))
    if rc:
        raise MlxError("moe_gated_ffn", rc, f"unsupported call: T={T}, hidden={hidden}, inter={inter}")
    return need.value


def _check_packed(fn, name, w, scales, biases, rows, cols, dtype, index, group_size):
    """A packed matrix [rows, cols] with scales and biases of `dtype`, all on device `index`."""
    if w.shape != (rows, cols // 8) or w.dtype not in _WORD_DTYPES or not w.is_contiguous() or w.get_device() != index:
        raise MlxError(fn, 1, f"{name}.w: contiguous 32-bit words {(rows, cols // 8)} on the input's device expected, "
                              f"got {w.dtype} {tuple(w.shape)} on {w.device}")
    shape = (rows, cols // group_size)
    for part, t in (("scales", scales), ("biases", biases)):
        if t is None and part == "biases":
            continue
        if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != index:
            raise MlxError(fn, 1, f"{name}.{part}: contiguous {dtype} {shape} on the input's device expected, "
                                  f"got {t.dtype} {tuple(t.shape)} on {t.device}")


def check_qweight(fn, name, q, rows, cols, dtype, index, group_size):
    _check_packed(fn, name, q.w, q.scales, q.biases, rows, cols, dtype, index, group_size)


def _quantized_matmul_ex(x, w, scales, biases, transpose, group_size, bits):
    fn = "mlx_quantized_matmul"
    dt = _DTYPES.get(x.dtype)
    if dt is None or dt == DTYPE_F32 or x.dim() < 1 or not x.is_contiguous():
        raise MlxError(fn, 1, "x must be contiguous bf16 or f16 [..., K]")
    if bits not in (2, 3, 4, 5, 6, 8) or group_size not in (32, 64, 128):
        raise MlxError(fn, 1, f"bits={bits}, group_size={group_size} is not a valid MLX affine format")
    if bits != 4:
        raise MlxError(fn, 2, f"bits={bits} is not implemented")
    if w.dim() != 2:
        raise MlxError(fn, 1, "w must be [rows, cols*bits/32]")
    K = x.shape[-1]
    rows, words = w.shape
    cols = words * 8
    N = rows if transpose else cols
    if (cols if transpose else rows) != K or cols % group_size or K == 0:
        raise MlxError(fn, 1, f"x [..., {K}] does not fit w {tuple(w.shape)} (transpose={bool(transpose)}, "
                              f"group_size={group_size})")
    _check_packed(fn, "w", w, scales, biases, rows, cols, x.dtype, x.get_device(), group_size)
    _no_graph(fn, x)
    M = x.numel() // K
    tr = 1 if transpose else 0
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    need = _qmm_workspace(dt, M, K, N, tr, group_size, bits)
    ws = _workspace(need, x.device) if need else None
    ctx = _context(fn, x)
    rc = library().moe_quantized_matmul_ex(ctx.handle, dt, x.data_ptr(), M, K, w.data_ptr(), scales.data_ptr(),
                                           biases.data_ptr() if biases is not None else None, N, tr, group_size, bits,
                                           out.data_ptr(), ws.data_ptr() if need else None, need)
    ctx.check(fn, rc)
    return out


def quantized_matmul(x, w, scales, biases=None, transpose=True, group_size=64, bits=4):
    """out[..., N] = x[..., K] @ dequant(w)^T (transpose=True), or x[..., K] @ dequant(w)
    for w [K, N*bits/32] (transpose=False: the gradient of the first with respect to x).
    bf16 or f16, group_size 32, 64 or 128, bits 4. Records no graph: an x that requires a gradient
    is refused outside torch.no_grad(), except at bf16, group_size 64 and transpose, where the
    result has none, as with the package's other operators."""
    if group_size != 64 or x.dtype != torch.bfloat16 or not transpose:
        if _calls is not None and bits == 4:
            out = _calls.quantized_matmul(x, w, scales, biases, transpose, group_size)
            if out is not None:
                return out
        if group_size in (32, 64, 128) or x.dtype != torch.bfloat16 or not transpose:
            return _quantized_matmul_ex(x, w, scales, biases, transpose, group_size, bits)
    _need(x, {torch.bfloat16}, "x")
    _need(w, _WORD_DTYPES, "w")
    _need(scales, {torch.bfloat16}, "scales")
    _need(biases, {torch.bfloat16}, "biases")
    K = x.shape[-1]
    N = w.shape[-2] if transpose else w.shape[-1] * 32 // bits
    lead = x.shape[:-1]
    M = 1
    for d in lead:
        M *= d
    out = torch.empty(*lead, N, dtype=torch.bfloat16, device=x.device)
    ctx = _ctx(x)
    rc = library().moe_quantized_matmul(ctx.handle, _ptr(x), M, K, _ptr(w), _ptr(scales),
                                        _ptr(biases), N, int(bool(transpose)), group_size, bits,
                                        _ptr(out))
    ctx.check("mlx_quantized_matmul", rc)
    return out


def gather_qmm(x, w, scales, biases=None, lhs_indices=None, rhs_indices=None, transpose=True,
               group_size=64, bits=4, sorted_indices=False):
    """MLX gather_qmm: out[b..., M, N] = x[lhs[b]] @ dequant(w[rhs[b]])^T.

    x is [..., M, K]; w is [E, N, K*bits/32]; lhs/rhs index the flattened batch
    dimensions of x and w and broadcast with each other (and with x's batch shape
    when lhs is omitted). The SwitchGLU form (x [T,1,1,K] with rhs [T,k], or
    x [T,k,1,I] with rhs [T,k]) maps onto the kernel without building indices.
    """
    _need(x, {torch.bfloat16}, "x")
    _need(w, _WORD_DTYPES, "w")
    _need(scales, {torch.bfloat16}, "scales")
    _need(biases, {torch.bfloat16}, "biases")
    if not transpose:
        raise MlxError("mlx_gather_qmm", 2, "transpose=false is not implemented")
    if w.dim() != 3:
        raise MlxError("mlx_gather_qmm", 1, "w must be [E, N, K*bits/32]")
    E, N = w.shape[0], w.shape[1]
    K = x.shape[-1]
    M = x.shape[-2] if x.dim() >= 2 else 1
    xb = tuple(x.shape[:-2])
    dev = x.device
    if rhs_indices is None:
        rhs_indices = torch.zeros((), dtype=torch.int32, device=dev)
    if lhs_indices is None:
        bshape = torch.broadcast_shapes(xb, tuple(rhs_indices.shape))
    else:
        bshape = torch.broadcast_shapes(tuple(lhs_indices.shape), tuple(rhs_indices.shape))
    nb = 1
    for d in bshape:
        nb *= d
    lhs_flat = None
    x_repeat = 1
    fast = (lhs_indices is None and M == 1 and len(bshape) >= 1 and
            (xb == bshape or (len(xb) == len(bshape) and xb[:-1] == bshape[:-1] and xb[-1] == 1)))
    rhs_flat = rhs_indices.expand(bshape).reshape(-1).to(torch.int32).contiguous()
    if fast:
        x_repeat = 1 if xb == bshape else bshape[-1]
        batch = nb
    else:
        if lhs_indices is None:
            nxb = 1
            for d in xb:
                nxb *= d
            lhs_b = torch.arange(nxb, device=dev, dtype=torch.int32).reshape(xb if xb else ())
            lhs_b = lhs_b.expand(bshape).reshape(-1)
        else:
            lhs_b = lhs_indices.expand(bshape).reshape(-1).to(torch.int32)
        # one kernel row per (batch element, m): x row = lhs*M + m, weight = rhs
        m = torch.arange(M, device=dev, dtype=torch.int32)
        lhs_flat = (lhs_b[:, None] * M + m[None, :]).reshape(-1).contiguous()
        rhs_flat = rhs_flat[:, None].expand(nb, M).reshape(-1).contiguous()
        batch = nb * M
    out = torch.empty(*bshape, M, N, dtype=torch.bfloat16, device=dev)
    xc = x.contiguous()
    x_rows = xc.numel() // K
    ctx = _ctx(x)
    rc = library().moe_gather_qmm(ctx.handle, _ptr(xc), x_rows, K, x_repeat, _ptr(lhs_flat), _ptr(w),
                                  _ptr(scales), _ptr(biases), E, N, _ptr(rhs_flat), batch, 1,
                                  group_size, bits, int(bool(sorted_indices)), _ptr(out))
    ctx.check("mlx_gather_qmm", rc)
    return out


def fast_rms_norm(x, weight, eps):
    """bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight) over the last axis."""
    _need(x, {torch.bfloat16}, "x")
    _need(weight, {torch.bfloat16}, "weight")
    dim = x.shape[-1]
    rows = x.numel() // dim if dim else 0
    out = torch.empty_like(x)
    ctx = _ctx(x)
    rc = library().moe_fast_rms_norm(ctx.handle, _ptr(x), _ptr(weight), float(eps), rows, dim,
                                     _ptr(out))
    ctx.check("mlx_fast_rms_norm", rc)
    return out


def _ffn_call(fn, x, gate, up, down, activation, group_size, bits):
    """Config and weights of a feed-forward call whose arguments have been checked."""
    if activation not in ACTIVATIONS:
        raise MlxError(fn, 1, f"activation {activation!r} is not one of {sorted(ACTIVATIONS)}")
    if x.dtype not in (torch.bfloat16, torch.float16) or x.dim() < 1 or not x.is_contiguous():
        raise MlxError(fn, 1, "x must be contiguous bf16 or f16 [..., hidden]")
    if bits != 4 or group_size not in (32, 64, 128):
        raise MlxError(fn, 2, f"bits={bits}, group_size={group_size} is not implemented")
    H, I = x.shape[-1], gate.w.shape[0]
    if H == 0 or H % group_size or I == 0 or I % group_size:
        raise MlxError(fn, 1, f"hidden={H} and inter={I} must be positive multiples of group_size={group_size}")
    for name, q, rows, cols in (("gate", gate, I, H), ("up", up, I, H), ("down", down, H, I)):
        check_qweight(fn, name, q, rows, cols, x.dtype, x.get_device(), group_size)
    return ffn_config(H, I, x.dtype, activation, group_size, bits), ffn_tensors(gate, up, down)


def ffn_config(H, I, dtype, activation, group_size, bits):
    return FfnConfig(H, I, ACTIVATIONS[activation], group_size, bits, _DTYPES[dtype])


def ffn_tensors(gate, up, down):
    return (gate.w, gate.scales, gate.biases, up.w, up.scales, up.biases, down.w, down.scales, down.biases)


def ffn_weights(fn, cfg, weights, x):
    """The weight structs of a call on x, checked against its config."""
    H, I = cfg.hidden, cfg.inter
    parts = []
    for i, (name, rows, cols) in enumerate((("gate", I, H), ("up", I, H), ("down", H, I))):
        w, s, b = weights[3 * i:3 * i + 3]
        _check_packed(fn, name, w, s, b, rows, cols, x.dtype, x.get_device(), cfg.group_size)
        parts.append(QWeight(w.data_ptr(), s.data_ptr(), None if b is None else b.data_ptr()))
    return FfnWeights(*parts)


def _like(fn, name, t, shape, x):
    if tuple(t.shape) != tuple(shape) or t.dtype != x.dtype or t.device != x.device or not t.is_contiguous():
        raise MlxError(fn, 1, f"{name}: contiguous {x.dtype} {tuple(shape)} on {x.device} expected")


def _ffn_forward(cfg, weights, x, residual, save):
    fn = "moe_gated_ffn_forward"
    if _calls is not None:
        r = _calls.ffn_forward(C.addressof(cfg), weights, x, residual, save)
        if r is not None:
            return r
    _no_graph(fn, x, residual)
    wts = ffn_weights(fn, cfg, weights, x)
    T = x.numel() // cfg.hidden
    out = torch.empty_like(x)
    g = u = None
    if save:
        g = torch.empty((*x.shape[:-1], cfg.inter), dtype=x.dtype, device=x.device)
        u = torch.empty_like(g)
    need = _ffn_workspace(cfg.hidden, cfg.inter, cfg.group_size, cfg.dtype, T, 0)
    ws = _workspace(need, x.device) if need else None
    ctx = _context(fn, x)
    rc = library().moe_gated_ffn_forward(ctx.handle, cfg, wts, x.data_ptr(), T,
                                         None if residual is None else residual.data_ptr(),
                                         g.data_ptr() if save else None, u.data_ptr() if save else None,
                                         out.data_ptr(), ws.data_ptr() if need else None, need)
    ctx.check(fn, rc)
    return (out, g, u) if save else out


def _ffn_backward(cfg, weights, g, u, dy):
    fn = "moe_gated_ffn_backward"
    if _calls is not None:
        r = _calls.ffn_backward(C.addressof(cfg), weights, g, u, dy)
        if r is not None:
            return r
    _no_graph(fn, g, u, dy)
    wts = ffn_weights(fn, cfg, weights, dy)
    T = dy.numel() // cfg.hidden
    _like(fn, "gate", g, (*dy.shape[:-1], cfg.inter), dy)
    _like(fn, "up", u, (*dy.shape[:-1], cfg.inter), dy)
    dx, dgate, dup = torch.empty_like(dy), torch.empty_like(g), torch.empty_like(u)
    need = _ffn_workspace(cfg.hidden, cfg.inter, cfg.group_size, cfg.dtype, T, 1)
    ws = _workspace(need, dy.device) if need else None
    ctx = _context(fn, dy)
    rc = library().moe_gated_ffn_backward(ctx.handle, cfg, wts, g.data_ptr(), u.data_ptr(), dy.data_ptr(), T,
                                          dgate.data_ptr(), dup.data_ptr(), dx.data_ptr(),
                                          ws.data_ptr() if need else None, need)
    ctx.check(fn, rc)
    return dx, dgate, dup


def gated_ffn(x, gate, up, down, activation="silu", group_size=64, bits=4, residual=None, save=False):
    """(act(x gate^T) * (x up^T)) down^T (+ residual): the dense feed-forward block on 4-bit
    weights (QWeight triples; gate, up [I, H], down [H, I]), activation "silu" or "gelu"
    (tanh form). With save, (out, g, u): the two projections' outputs, what gated_ffn_vjp
    takes. bf16 or f16, group_size 32, 64 or 128. Records no graph: inputs that require a gradient
    are refused outside torch.no_grad(); gated_ffn_vjp gives it."""
    cfg, weights = _ffn_call("moe_gated_ffn_forward", x, gate, up, down, activation, group_size, bits)
    if residual is not None:
        _like("moe_gated_ffn_forward", "residual", residual, x.shape, x)
    return _ffn_forward(cfg, weights, x, residual, save)


def gated_ffn_vjp(g, u, dy, gate, up, down, activation="silu", group_size=64, bits=4):
    """(dx, dg, du): the gradients of gated_ffn with respect to x and to the projections'
    outputs g, u (as saved by it), for the gradient dy of its output. The quantised weights
    are frozen."""
    cfg, weights = _ffn_call("moe_gated_ffn_backward", dy, gate, up, down, activation, group_size, bits)
    return _ffn_backward(cfg, weights, g, u, dy)


def fast_rope(x, dims, traditional=False, base=10000.0, scale=1.0, offset=0, freqs=None, mscale=1.0, inverse=False,
              out=None):
    """Rotary positions of x [..., L, D] (the axes before L: any batch and heads; two of them,
    [B, H, L, D], may have any strides). Pair i of the first `dims` channels at position
    offset + l is turned by (offset + l) * scale / wavelength_i, wavelength_i =
    base**(2 i / dims) or freqs[i] (float32 [dims/2]), and scaled by mscale; traditional:
    pairs (2i, 2i+1), else (i, i + dims/2); channels from dims on are copied. offset: an
    int, or an int32 / int64 tensor [B] with one offset per batch element. inverse: the
    transposed rotation, the gradient with respect to x. out: where to write, x itself
    included, else memory apart from x's (default: a new contiguous tensor). An int offset is
    at most 2**53 in magnitude. bf16, f16 or f32. Records no graph: an x that requires a gradient
    is refused outside torch.no_grad()."""
    if out is None and _calls is not None:
        r = _calls.fast_rope(x, dims, traditional, base, scale, offset, freqs, mscale, inverse)
        if r is not None:
            return r
    fn = "mlx_fast_rope"
    dt = _DTYPES.get(x.dtype)
    nd = x.dim()
    if dt is None or nd < 2:
        raise MlxError(fn, 1, "x must be bf16, f16 or f32 [..., L, D]")
    _no_graph(fn, x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise MlxError(fn, 1, f"out: {x.dtype} {tuple(x.shape)} on {x.device} expected")
    elif out.data_ptr() == x.data_ptr() and out.stride() != x.stride():
        raise MlxError(fn, 1, "out shares x's memory with other strides")
    xs, os_ = x.stride(), out.stride()
    if nd == 4:
        B, H, L, D = x.shape
    elif nd == 3:
        (B, L, D), H = x.shape, 1
        xs, os_ = (xs[0], 0, xs[1], xs[2]), (os_[0], 0, os_[1], os_[2])
    else:
        if not (x.is_contiguous() and out.is_contiguous()):
            raise MlxError(fn, 1, "x and out: must be contiguous unless [B, H, L, D] or [B, L, D]")
        L, D = x.shape[-2:]
        B, H = 1, x.numel() // (L * D) if L * D else 0
        xs = os_ = (0, L * D, D, 1)
    if D > 1 and (xs[3] != 1 or os_[3] != 1):
        raise MlxError(fn, 1, "the channels of x and out must be contiguous")
    if not 0 < dims <= D or dims % 2:
        raise MlxError(fn, 1, f"dims={dims} must be even and in 2..{D}")
    reach = D - 1  # by rising stride, each step of out is longer than all that the smaller ones reach
    for s, n in sorted(zip(os_[:3], (B, H, L))):
        if n > 1:
            if s <= reach:
                raise MlxError(fn, 1, "rows of out overlap one another")
            reach += (n - 1) * s
    offs, offs_bits, off = None, 0, 0
    if isinstance(offset, torch.Tensor):
        if nd not in (3, 4) and offset.dim():
            raise MlxError(fn, 1, "offsets per batch element need x [B, H, L, D] or [B, L, D]")
        if offset.dtype not in (torch.int32, torch.int64) or offset.device != x.device or offset.dim() > 1 \
                or offset.numel() != B or not offset.is_contiguous():
            raise MlxError(fn, 1, f"offset: contiguous int32 or int64 [{B}] on {x.device} expected")
        offs, offs_bits = offset.data_ptr(), 32 if offset.dtype == torch.int32 else 64
    else:
        off = int(offset)
        if abs(off) > 2 ** 53:
            raise MlxError(fn, 1, f"offset={off} is beyond 2**53")
    if freqs is not None and (freqs.dtype != torch.float32 or freqs.device != x.device or
                              freqs.shape != (dims // 2,) or not freqs.is_contiguous()):
        raise MlxError(fn, 1, f"freqs: contiguous float32 [{dims // 2}] on {x.device} expected")
    cfg = RopeConfig(dt, dims, 1 if traditional else 0, 1 if inverse else 0, 0.0 if base is None else base, scale, mscale)
    ctx = _context(fn, x)
    rc = library().moe_fast_rope(ctx.handle, cfg, x.data_ptr(), _I64x3(*xs[:3]), B, H, L, D, off, offs, offs_bits,
                                 None if freqs is None else freqs.data_ptr(), out.data_ptr(), _I64x3(*os_[:3]))
    ctx.check(fn, rc)
    return out
