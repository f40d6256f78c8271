"""CPU checks of the dense operators: the 64-bit forms the GPU tests compare with, their
gradients against differences, and what the entry points refuse."""
import ctypes as C

import pytest
import torch

import dense_ref as R
import mlx_rs_b200
from mlx_rs_b200 import _lib, ops
from mlx_rs_b200.block import DenseMlp
from mlx_rs_b200.synth import QWeight


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_gradient_formulas_match_differences(kind):
    gen = _gen(1)
    H, I, T, g = 64, 96, 5, 32
    gate, up = (R.QW(gen, I, H, g, torch.bfloat16) for _ in range(2))
    down = R.QW(gen, H, I, g, torch.bfloat16)
    x, dy, v = (torch.randn(T, H, generator=gen, dtype=torch.float64) for _ in range(3))
    _, pg, pu = R.ffn(x, gate, up, down, kind)
    dx, dg, du = R.ffn_vjp(pg, pu, dy, gate, up, down, kind)
    eps = 1e-5
    diff = ((R.ffn(x + eps * v, gate, up, down, kind)[0] - R.ffn(x - eps * v, gate, up, down, kind)[0]) * dy).sum() / (2 * eps)
    # central differences: error O(eps^2) of order 1e-10, rounding 2^-53 |y| / eps of order 1e-9
    assert abs(float(diff - (dx * v).sum())) <= 1e-6 * float((dx * v).abs().sum())
    wd = down.dense()
    for which, grad in ((0, dg), (1, du)):
        w = torch.randn(T, I, generator=gen, dtype=torch.float64)
        y = [((R.act(pg + (e * w if which == 0 else 0), kind)[0] * (pu + (e * w if which == 1 else 0))) @ wd.t() * dy).sum()
             for e in (eps, -eps)]
        assert abs(float((y[0] - y[1]) / (2 * eps) - (grad * w).sum())) <= 1e-6 * float((grad * w).abs().sum())


def test_rope_reference_is_a_rotation_and_its_inverse_the_transpose():
    gen = _gen(2)
    x, y = (torch.randn(2, 3, 5, 24, generator=gen) for _ in range(2))
    for trad in (False, True):
        kw = dict(dims=16, traditional=trad, offset=torch.tensor([7, 900000]), scale=0.25, mscale=1.25)
        a, b = R.rope(x, **kw)[0], R.rope(y, inverse=True, **kw)[0]
        # <R x, y> = <x, R^T y> over the rotated channels; |R x| = mscale |x|
        assert torch.allclose((a * y.double())[..., :16].sum(), (b * x.double())[..., :16].sum(), rtol=1e-10, atol=1e-10)
        assert torch.allclose(a[..., :16].norm(), 1.25 * x.double()[..., :16].norm(), rtol=1e-12)
        assert torch.equal(a[..., 16:], x.double()[..., 16:])


def test_workspace_queries_refuse_what_the_calls_refuse():
    lib, n = mlx_rs_b200.library(), C.c_size_t(1)
    q = lib.moe_quantized_matmul_workspace
    assert q(0, 4, 64, 8, 1, 32, 4, C.byref(n)) == 0
    assert q(0, 0, 64, 8, 1, 32, 4, C.byref(n)) == 0 and n.value == 0
    assert q(0, 4, 64, 8, 1, 32, 3, C.byref(n)) == _lib.MOE_ERR_UNSUPPORTED
    assert q(2, 4, 64, 8, 1, 32, 4, C.byref(n)) == _lib.MOE_ERR_UNSUPPORTED
    for bad in ((0, 4, 64, 8, 1, 48, 4), (0, 4, 64, 8, 1, 32, 7), (0, 4, 80, 8, 1, 32, 4), (0, 4, 64, 40, 0, 32, 4),
                (0, -1, 64, 8, 1, 32, 4), (0, 4, 64, 0, 1, 32, 4), (0, 4, 0, 8, 1, 32, 4), (5, 4, 64, 8, 1, 32, 4),
                (0, 2 ** 40, 64, 8, 1, 32, 4)):
        assert q(*bad, C.byref(n)) == _lib.MOE_ERR_INVALID, bad
    assert q(0, 4, 64, 8, 1, 32, 4, None) == _lib.MOE_ERR_INVALID
    f = lib.moe_gated_ffn_workspace
    ok = dict(hidden=64, inter=96, activation=0, group_size=32, bits=4, dtype=0)
    cfg = lambda **kw: C.byref(_lib.FfnConfig(**{**ok, **kw}))  # noqa: E731
    assert f(cfg(), 3, 0, C.byref(n)) == 0
    assert f(cfg(bits=8), 3, 0, C.byref(n)) == _lib.MOE_ERR_UNSUPPORTED
    for bad in (dict(hidden=48), dict(inter=0), dict(inter=-32), dict(activation=2), dict(group_size=16), dict(dtype=9)):
        assert f(cfg(**bad), 3, 0, C.byref(n)) == _lib.MOE_ERR_INVALID, bad
    assert f(cfg(), -1, 0, C.byref(n)) == _lib.MOE_ERR_INVALID
    assert f(None, 1, 0, C.byref(n)) == _lib.MOE_ERR_INVALID


def test_null_context_is_refused():
    lib = mlx_rs_b200.library()
    assert lib.moe_quantized_matmul_ex(None, 0, None, 1, 32, None, None, None, 1, 1, 32, 4, None, None, 0) == 1
    assert lib.moe_gated_ffn_forward(None, None, None, None, 1, None, None, None, None, None, 0) == 1
    assert lib.moe_gated_ffn_backward(None, None, None, None, None, None, 1, None, None, None, None, 0) == 1
    assert lib.moe_fast_rope(None, None, None, None, 1, 1, 1, 2, 0, None, 0, None, None, None) == 1


def _refused(f, *a, **kw):
    with pytest.raises(_lib.MlxError) as e:
        f(*a, **kw)
    return str(e.value)


def test_quantized_matmul_refusals():
    gen = _gen(3)
    q = R.QW(gen, 40, 64, 32, torch.bfloat16)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    mm = lambda x, w=q.w, s=q.scales, b=q.biases, **kw: ops.quantized_matmul(x, w, s, b, **{"group_size": 32, **kw})  # noqa: E731
    assert "CUDA" in _refused(mm, x)
    assert "does not fit" in _refused(mm, x[:, :32].contiguous())
    assert "does not fit" in _refused(mm, x, transpose=False)  # x must then have 40 columns
    assert "contiguous" in _refused(mm, x.t())
    assert "f16" in _refused(mm, x.float())
    assert "scales" in _refused(mm, x, s=q.scales.half())
    assert "scales" in _refused(mm, x, s=q.scales[:, :1].contiguous())
    assert "biases" in _refused(mm, x, b=q.biases[:5])
    assert "w.w" in _refused(mm, x, w=q.w.to(torch.int64))
    assert "rc=2" in _refused(mm, x, bits=8)


def test_ffn_refusals():
    gen = _gen(4)
    mk = lambda r, c, d=torch.bfloat16: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 32, d))  # noqa: E731
    gate, up, down = mk(96, 64), mk(96, 64), mk(64, 96)
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    call = lambda g=gate, u=up, d=down, x=x, **kw: ops.gated_ffn(x, g, u, d, **{"group_size": 32, **kw})  # noqa: E731
    assert "CUDA" in _refused(call)
    assert "up.w" in _refused(call, u=mk(64, 64))
    assert "down.w" in _refused(call, d=mk(96, 64))
    assert "gate.scales" in _refused(call, g=mk(96, 64, torch.float16))
    assert "activation" in _refused(call, activation="relu")
    assert "rc=2" in _refused(call, bits=3)
    assert "rc=2" in _refused(call, group_size=16)
    assert "residual" in _refused(call, residual=x[:1])
    mlp = DenseMlp(gate, up, down, group_size=32)
    assert "CUDA" in _refused(mlp, x)
    assert "expected" in _refused(mlp, x[:, :32].contiguous())
    assert "expected" in _refused(mlp, x.half())
    assert "expected" in _refused(mlp.vjp, (x, x), x)
    assert "up" in _refused(DenseMlp, gate, mk(32, 64), down, group_size=32)
    assert "multiples" in _refused(DenseMlp, gate, up, down, group_size=64)


def test_rope_refusals():
    x = torch.zeros(2, 3, 5, 24)
    r = lambda x=x, dims=16, **kw: ops.fast_rope(x, dims, **kw)  # noqa: E731
    assert "CUDA" in _refused(r)
    assert "f32" in _refused(r, x.double())
    assert "channels" in _refused(r, x.transpose(2, 3), dims=4)
    assert "offset" in _refused(r, offset=torch.zeros(3, dtype=torch.int32))
    assert "offset" in _refused(r, offset=torch.zeros(2))
    assert "freqs" in _refused(r, freqs=torch.ones(7))
    assert "out" in _refused(r, out=torch.zeros(2, 3, 5, 23))
    assert "other strides" in _refused(r, out=torch.as_strided(x, x.shape, (24, 240, 48, 1)))


@pytest.mark.parametrize("offset", [2 ** 53 + 1, -2 ** 60, 2 ** 63, 2 ** 64])
def test_rope_refuses_offsets_beyond_64_bit_angles(offset):
    assert "offset" in _refused(ops.fast_rope, torch.zeros(1, 1, 2, 8), 8, offset=offset)


@pytest.mark.parametrize("dims", [0, -2, 7, 10, 2 ** 32 + 8])
def test_rope_refuses_dims(dims):
    assert "dims" in _refused(ops.fast_rope, torch.zeros(1, 1, 2, 8), dims)


def test_rope_refuses_an_output_that_overlaps_itself():
    row = torch.zeros(1, 1, 5, 8)
    x = row.expand(2, 3, 5, 8)
    assert "overlap" in _refused(ops.fast_rope, x, 8, out=x)
    assert "overlap" in _refused(ops.fast_rope, x[0], 8, out=x[0])
    rows = torch.zeros(64).as_strided((1, 1, 5, 8), (40, 40, 6, 1))
    assert "overlap" in _refused(ops.fast_rope, rows, 8, out=rows)
    # heads of a fused projection do not: this gets as far as the device
    fused = torch.zeros(2, 5, 6, 8)[:, :, 1:4].transpose(1, 2)
    assert "CUDA" in _refused(ops.fast_rope, fused, 8, out=fused)


def test_dense_mlp_refuses_a_scalar():
    gen = _gen(9)
    mk = lambda r, c: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 32, torch.bfloat16))  # noqa: E731
    mlp = DenseMlp(mk(96, 64), mk(96, 64), mk(64, 96), group_size=32)
    assert "expected" in _refused(mlp, torch.zeros((), dtype=torch.bfloat16))


@pytest.mark.parametrize("bits,group,rc", [(7, 32, 1), (0, 128, 1), (3, 32, 2), (8, 128, 2), (4, 16, 1)])
def test_quantized_matmul_tells_invalid_from_unsupported(bits, group, rc):
    """rc 1: no format of MLX; rc 2: one that is not implemented. As the C entries do."""
    q, x = R.QW(_gen(12), 40, 64, 32, torch.float16), torch.zeros(3, 64, dtype=torch.float16)
    assert f"rc={rc}" in _refused(ops.quantized_matmul, x, q.w, q.scales, q.biases, group_size=group, bits=bits)


def test_inputs_that_require_gradients_are_refused():
    """No call records a graph, so that a backward pass would pass by it in silence."""
    gen = _gen(11)
    mk = lambda r, c, d=torch.bfloat16: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 32, d))  # noqa: E731
    x = torch.zeros(2, 64, dtype=torch.bfloat16, requires_grad=True)
    p, mlp = mk(96, 64), DenseMlp(mk(96, 64), mk(96, 64), mk(64, 96), group_size=32)
    w = (mlp.gate, mlp.up, mlp.down)
    h, z = torch.zeros(2, 96, dtype=torch.bfloat16), x.detach()
    calls = [lambda: ops.quantized_matmul(x, p.w, p.scales, p.biases, group_size=32), lambda: mlp(x), lambda: mlp.forward_saved(x),
             lambda: ops.gated_ffn(x, *w, group_size=32), lambda: ops.gated_ffn(z, *w, group_size=32, residual=x),
             lambda: mlp.vjp((h, h), x), lambda: ops.gated_ffn_vjp(h.requires_grad_(), h, z, *w, group_size=32),
             lambda: ops.fast_rope(x[None, None], 64)]
    for f in calls:
        assert "requires a gradient" in _refused(f)
    with torch.no_grad():  # this gets as far as the device
        for f in calls:
            assert "CUDA" in _refused(f)


def test_dense_mlp_checks_the_weights_it_has_now():
    """Weights put in place of others are looked at by the next call (it refuses what does not fit)."""
    gen = _gen(10)
    mk = lambda r, c, d=torch.bfloat16: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 32, d))  # noqa: E731
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    mlp = DenseMlp(mk(96, 64), mk(96, 64), mk(64, 96), group_size=32)
    mlp.up = mk(64, 64)
    assert "up.w" in _refused(mlp, x)
    mlp.up = mk(96, 64)
    mlp.down.scales = mlp.down.scales.half()
    assert "down.scales" in _refused(mlp, x)
    mlp.down = mk(64, 96)
    assert "CUDA" in _refused(mlp, x)
