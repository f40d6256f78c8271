"""GPU parity of the dense operators against their 64-bit forms (tests/dense_ref.py, which
derives the bounds), at the sizes, types, strides and streams where they can go wrong."""
import ctypes as C

import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(*seed):
    return torch.Generator().manual_seed(hash(seed) & 0x7FFFFFFF)


def _close(got, want, bound, what):
    assert got.shape == want.shape
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), f"{what}: worst {float((d / bound).max()):.3f} of the bound"


def _status_is_clean():
    import mlx_rs_b200
    from mlx_rs_b200._lib import context_for
    s = C.c_int32(-1)
    ctx = context_for(0)
    assert mlx_rs_b200.library().moe_ctx_status(ctx.handle, C.byref(s)) == 0 and s.value == 0


QMM = [  # M, N, K, group, dtype, biases
    (1, 2048, 2048, 32, BF16, True), (1, 1, 32, 32, F16, True), (2, 40, 128, 128, BF16, False),
    (3, 1001, 1408, 64, F16, False), (7, 130, 96, 32, BF16, True), (8, 256, 2048, 128, BF16, True),
    (9, 129, 640, 128, F16, True), (16, 33, 4096, 64, F16, True), (17, 96, 5632, 32, BF16, True),
    (31, 511, 512, 32, F16, False), (33, 300, 352, 32, BF16, True), (64, 257, 1024, 128, BF16, True),
    (127, 1000, 256, 64, F16, True), (128, 512, 704, 64, F16, True), (129, 513, 736, 32, BF16, True),
    (300, 1408, 2048, 128, BF16, False), (1000, 2048, 768, 32, BF16, True),
    (1100, 700, 416, 32, BF16, True), (2049, 513, 256, 128, F16, False), (1024, 66001, 512, 64, F16, True),
    (200, 2048, 8192, 32, BF16, True), (2050, 66001, 512, 64, F16, True), (1024, 300, 256, 32, BF16, True)]


@pytest.mark.parametrize("M,N,K,g,dt,biases", QMM)
def test_quantized_matmul(M, N, K, g, dt, biases):
    from mlx_rs_b200 import ops
    gen = _gen(M, N, K)
    q = R.QW(gen, N, K, g, dt, biases, "cuda")
    x = R.rand(gen, M, K, dtype=dt, device="cuda")
    got = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=g)
    assert got.dtype == dt
    _close(got, *R.qmm(x, q), "product")
    assert R.rel(got, R.qmm(x, q)[0]) <= 2 * R.U[dt]  # two independent roundings of at most u each
    assert torch.equal(got, ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=g))
    _status_is_clean()


@pytest.mark.parametrize("M,K,N,g,dt,biases", [
    (1, 2048, 2048, 64, BF16, True), (5, 33, 64, 64, BF16, True), (32, 1001, 128, 128, F16, False),
    (130, 100, 352, 32, F16, True), (512, 5632, 2048, 32, BF16, True), (257, 768, 1408, 64, BF16, False),
    (1030, 520, 320, 64, F16, True), (1025, 99, 256, 128, BF16, True), (130, 8192, 544, 32, F16, True)])
def test_quantized_matmul_not_transposed(M, K, N, g, dt, biases):
    from mlx_rs_b200 import ops
    gen = _gen(M, K, N)
    q = R.QW(gen, K, N, g, dt, biases, "cuda")
    x = R.rand(gen, M, K, dtype=dt, device="cuda")
    got = ops.quantized_matmul(x, q.w, q.scales, q.biases, transpose=False, group_size=g)
    want, bound = R.qmm(x, q, transpose=False)
    _close(got, want, bound, "product")
    assert R.rel(got, want) <= 2 * R.U[dt]


def test_quantized_matmul_leading_axes_and_empty_batch():
    from mlx_rs_b200 import ops
    gen = _gen(11)
    q = R.QW(gen, 72, 128, 32, BF16, True, "cuda")
    x = R.rand(gen, 2, 3, 128, dtype=BF16, device="cuda")
    got = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=32)
    assert got.shape == (2, 3, 72)
    assert torch.equal(got.reshape(6, 72), ops.quantized_matmul(x.reshape(6, 128), q.w, q.scales, q.biases, group_size=32))
    assert ops.quantized_matmul(x[:0], q.w, q.scales, q.biases, group_size=32).shape == (0, 3, 72)


def test_quantized_matmul_c_entry_with_the_contexts_scratch():
    """moe_quantized_matmul itself at group size 32: no workspace argument."""
    import mlx_rs_b200
    from mlx_rs_b200 import ops
    from mlx_rs_b200._lib import context_for
    gen = _gen(12)
    q = R.QW(gen, 200, 512, 32, BF16, True, "cuda")
    for M in (3, 150):
        x = R.rand(gen, M, 512, dtype=BF16, device="cuda")
        out = torch.empty(M, 200, dtype=BF16, device="cuda")
        ctx = context_for(0)
        ctx.bind_stream(torch.cuda.current_stream().cuda_stream)
        rc = mlx_rs_b200.library().moe_quantized_matmul(ctx.handle, x.data_ptr(), M, 512, q.w.data_ptr(),
                                                        q.scales.data_ptr(), q.biases.data_ptr(), 200, 1, 32, 4,
                                                        out.data_ptr())
        ctx.check("moe_quantized_matmul", rc)
        assert torch.equal(out, ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=32))


FFN = [  # T, H, I, group, dtype, act
    (1, 2048, 5632, 64, BF16, "silu"), (1, 32, 32, 32, F16, "gelu"), (2, 256, 128, 128, BF16, "gelu"),
    (8, 2048, 1792, 32, F16, "gelu"), (9, 96, 1120, 32, BF16, "silu"), (32, 704, 320, 64, BF16, "silu"),
    (33, 384, 256, 128, F16, "silu"), (128, 192, 448, 64, F16, "gelu"), (129, 2048, 768, 128, BF16, "silu"),
    (333, 1024, 736, 32, BF16, "gelu"), (700, 640, 1408, 64, BF16, "silu"),
    (1025, 256, 352, 32, F16, "silu"), (2500, 384, 640, 128, BF16, "gelu"),
    (20, 1024, 8192, 64, BF16, "silu"), (13, 512, 64, 32, F16, "gelu"), (2047, 128, 192, 64, BF16, "silu")]


def _ffn_case(T, H, I, g, dt):
    from mlx_rs_b200.synth import QWeight
    gen = _gen(T, H, I)
    qs = [R.QW(gen, I, H, g, dt, True, "cuda"), R.QW(gen, I, H, g, dt, True, "cuda"), R.QW(gen, H, I, g, dt, True, "cuda")]
    x, dy = (R.rand(gen, T, H, dtype=dt, device="cuda") for _ in range(2))
    return qs, [QWeight(q.w, q.scales, q.biases) for q in qs], x, dy


# Normwise, with independent roundings of at most u each: g and u (their weights), h (its own
# rounding), the down weights, the output: sqrt(2 + 1 + 1 + 1) u < 3 u. The gradients start from
# g and u rounded to the type (the activation's derivative passes that on with a factor of at
# most about 2 where it is large) and add dh's weights, their own rounding, and for dx the
# weights' and the output's: sqrt(4 + 4 + 1 + 1 + 1 + 1) u < 4 u.
@pytest.mark.parametrize("T,H,I,g,dt,kind", FFN)
def test_ffn_and_its_gradients(T, H, I, g, dt, kind):
    from mlx_rs_b200.block import DenseMlp
    qs, ws, x, dy = _ffn_case(T, H, I, g, dt)
    mlp = DenseMlp(*ws, activation=kind, group_size=g)
    want, pg, pu = R.ffn(x, *qs, kind)
    u = R.U[dt]
    out = mlp(x)
    assert R.rel(out, want) <= 3 * u
    out2, saved = mlp.forward_saved(x)
    assert torch.equal(out, out2)
    assert R.rel(saved[0], pg) <= 2 * u and R.rel(saved[1], pu) <= 2 * u
    for got, w, name in zip(mlp.vjp(saved, dy), R.ffn_vjp(pg, pu, dy, *qs, kind), ("dx", "dg", "du")):
        assert got.shape == w.shape and R.rel(got, w) <= 4 * u, (name, R.rel(got, w) / u)
    _status_is_clean()


@pytest.mark.parametrize("T", [1, 40, 150])
def test_ffn_elementwise_bound(T):
    """Element by element, worst cases added up: dh <= 1.13 |u| dg + |act| du + 1.13 dg du + u |h|
    (1.13 bounds both activations' slope), then the down product of h as computed."""
    from mlx_rs_b200.block import DenseMlp
    H, I, g, dt = 256, 160, 32, BF16
    qs, ws, x, _ = _ffn_case(T, H, I, g, dt)
    (pg, bg), (pu, bu) = R.qmm(x, qs[0]), R.qmm(x, qs[1])
    a = R.act(pg, "silu")[0]
    h = a * pu
    u = R.U[dt]
    bh = (1.13 * bg * pu.abs() + a.abs() * bu + 1.13 * bg * bu) * (1 + u) + u * h.abs() + 2.0 ** -20 * h.abs()
    wd = qs[2].dense().abs().t()
    y = h @ qs[2].dense().t()
    bound = (bh @ wd) * (1 + u) + u * (h.abs() @ wd) + (I + 16) * 2.0 ** -23 * ((h.abs() + bh) @ qs[2].spread(144.0).t())
    bound = bound * (1 + u) + u * y.abs()
    _close(DenseMlp(*ws, group_size=g)(x), y, bound, "ffn")


def test_ffn_gradient_against_differences_of_the_kernel():
    """(f(x + e v) - f(x - e v)) / 2 e along v, contracted with dy, against dx . v. f16 rounds each
    of the two outputs with relative error <= 3 u normwise, so the quotient is off by at most
    3 u |dy| (|f+| + |f-|) / 2 e, and by the curvature, taken from the 64-bit form at the same
    points; dx . v is off by 4 u |dx| |v|."""
    from mlx_rs_b200.block import DenseMlp
    T, H, I, g, dt = 40, 128, 256, 64, F16
    qs, ws, x, dy = _ffn_case(T, H, I, g, dt)
    mlp = DenseMlp(*ws, group_size=g)
    gen = _gen(5)
    v = torch.randn(T, H, generator=gen).sign().double().cuda()
    e = 0.125
    xp, xm = (x.double() + e * v).to(dt), (x.double() - e * v).to(dt)
    step = xp.double() - xm.double()
    fp, fm = mlp(xp).double(), mlp(xm).double()
    diff = ((fp - fm) * dy.double()).sum()
    exact = ((R.ffn(xp, *qs, "silu")[0] - R.ffn(xm, *qs, "silu")[0]) * dy.double()).sum()
    noise = 3 * R.U[dt] * dy.double().norm() * (fp.norm() + fm.norm())
    assert abs(float(diff - exact)) <= float(noise)
    _, saved = mlp.forward_saved(x)
    dx = mlp.vjp(saved, dy)[0].double()
    _, pg, pu = R.ffn(x, *qs, "silu")
    curve = abs(float(exact - (R.ffn_vjp(pg, pu, dy, *qs, "silu")[0] * step).sum()))
    assert abs(float(diff - (dx * step).sum())) <= float(noise) + curve + float(4 * R.U[dt] * dx.norm() * step.norm())


@pytest.mark.parametrize("T", [1, 20, 200])
def test_ffn_residual_and_layer(T):
    from mlx_rs_b200 import ops
    from mlx_rs_b200.block import DenseMlp
    qs, ws, x, _ = _ffn_case(T, 256, 384, 64, BF16)
    norm = (1 + 0.1 * torch.randn(256, generator=_gen(6))).to(BF16).cuda()
    mlp = DenseMlp(*ws)
    h = ops.fast_rms_norm(x, norm, 1e-6)
    want = R.ffn(h, *qs, "silu", residual=x)[0]
    got = mlp.forward_layer(x, norm, 1e-6)
    assert R.rel(got, want) <= 3 * R.U[BF16]
    assert torch.equal(got, ops.gated_ffn(h, *ws, residual=x))


def test_ffn_empty_batch():
    from mlx_rs_b200.block import DenseMlp
    qs, ws, x, dy = _ffn_case(4, 64, 96, 32, F16)
    mlp = DenseMlp(*ws, group_size=32)
    out, saved = mlp.forward_saved(x[:0])
    assert out.shape == (0, 64) and [t.shape for t in mlp.vjp(saved, dy[:0])] == [(0, 64), (0, 96), (0, 96)]


def test_rows_do_not_depend_on_their_batch_neighbours():
    """NaN and infinities in one token stay in its row; the rows beside it keep their values."""
    from mlx_rs_b200.block import DenseMlp
    for T in (4, 20, 150):
        qs, ws, x, _ = _ffn_case(T, 256, 384, 64, BF16)
        mlp = DenseMlp(*ws)
        a = mlp(x)
        x[1, 3], x[2, 5] = float("nan"), float("inf")
        b = mlp(x)
        keep = [i for i in range(T) if i not in (1, 2)]
        assert torch.equal(a[keep], b[keep])
        assert not bool(torch.isfinite(b[1]).any()) and not bool(torch.isfinite(b[2]).any())


ROPE = [  # B, H, L, D, dims, dtype, traditional
    (1, 4, 7, 128, 128, BF16, False), (64, 36, 1, 128, 128, BF16, False), (2, 3, 33, 80, 64, F32, True),
    (1, 1, 1, 2, 2, F32, False), (3, 2, 5, 94, 94, F16, False), (3, 2, 5, 94, 30, F16, True), (2, 5, 9, 66, 34, BF16, True),
    (1, 2, 1100, 64, 32, F16, False), (2, 1, 700, 256, 256, F32, False), (1, 3, 4, 4096, 4096, BF16, False)]


@pytest.mark.parametrize("B,H,L,D,dims,dt,trad", ROPE)
def test_rope(B, H, L, D, dims, dt, trad):
    from mlx_rs_b200 import ops
    gen = _gen(B, H, L, D, dims)
    x = R.rand(gen, B, H, L, D, dtype=dt, device="cuda")
    off = torch.randint(0, 1000000, (B,), generator=gen)
    wave = (10000.0 ** (torch.arange(0, dims, 2) / dims) * 1.5).float()
    for kw in (dict(), dict(offset=12345, scale=0.125, base=500000.0), dict(offset=off, mscale=1.25),
               dict(offset=off.int(), freqs=wave), dict(offset=off, inverse=True, scale=0.3), dict(offset=-3)):
        dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        got = ops.fast_rope(x, dims, traditional=trad, **dev)
        want, bound = R.rope(x, dims, traditional=trad, **dev)
        _close(got, want, bound, kw)


def test_rope_strides_in_place_and_axes():
    from mlx_rs_b200 import ops
    gen = _gen(21)
    B, L, h, D = 2, 19, 5, 64
    fused = R.rand(gen, B, L, (h + 2) * D, dtype=BF16, device="cuda")
    heads = fused.view(B, L, h + 2, D)[:, :, :h].transpose(1, 2)
    want = ops.fast_rope(heads.contiguous(), D, offset=3)
    assert torch.equal(ops.fast_rope(heads, D, offset=3), want)
    before = fused.clone()
    ops.fast_rope(heads, D, offset=3, out=heads)
    assert torch.equal(heads, want)
    assert torch.equal(fused.view(B, L, h + 2, D)[:, :, h:], before.view(B, L, h + 2, D)[:, :, h:])
    # odd strides and addresses: one element in front, rows of D + 1
    odd = torch.zeros(1 + B * h * L * (D + 1), dtype=BF16, device="cuda")
    view = odd[1:].view(B, h, L, D + 1)[..., :D]
    view.copy_(before.view(B, L, h + 2, D)[:, :, :h].transpose(1, 2))
    assert torch.equal(ops.fast_rope(view, D, offset=3), want)
    x3 = R.rand(gen, 4, 6, D, dtype=F32, device="cuda")
    off = torch.tensor([5, 0, 9, 100], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.fast_rope(x3, D, offset=off), ops.fast_rope(x3[:, None], D, offset=off)[:, 0])
    assert torch.equal(ops.fast_rope(x3[0], D, offset=7), ops.fast_rope(x3[:1, None], D, offset=7)[0, 0])
    x5 = x3.view(1, 2, 2, 6, D)
    assert torch.equal(ops.fast_rope(x5, D, offset=7).view(4, 6, D), ops.fast_rope(x3, D, offset=7))
    assert ops.fast_rope(x3[:0], D).shape == (0, 6, D)
    # every head and batch reading one row (stride 0)
    wide = x3[:1, None].expand(3, 2, 6, D)
    assert torch.equal(ops.fast_rope(wide, D)[2, 1], ops.fast_rope(x3[:1, None], D)[0, 0])


def test_rope_rotates_back():
    from mlx_rs_b200 import ops
    x = R.rand(_gen(22), 2, 3, 50, 96, dtype=F32, device="cuda")
    off = torch.tensor([0, 10 ** 6], device="cuda")
    y = ops.fast_rope(ops.fast_rope(x, 96, offset=off), 96, offset=off, inverse=True)
    # two rotations of 8 steps of 2^-24 (|a| + |b|) each
    assert float((y - x).abs().max()) <= 2 * 8 * 2.0 ** -24 * 2 * 1.5 * float(x.abs().max())


def test_c_entry_refusals_launch_nothing():
    import mlx_rs_b200
    from mlx_rs_b200 import _lib
    ctx = _lib.context_for(0)
    lib = mlx_rs_b200.library()
    t = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = t.data_ptr()
    q = lib.moe_quantized_matmul_ex
    need = C.c_size_t()  # rows of 33 elements are copied to rows of 40
    assert lib.moe_quantized_matmul_workspace(0, 200, 33, 64, 0, 32, 4, C.byref(need)) == 0 and need.value >= 200 * 80
    assert q(ctx.handle, 0, p, 200, 33, p, p, p, 64, 0, 32, 4, p, p, need.value - 1) == 1
    assert b"workspace" in lib.moe_last_error(ctx.handle)
    assert q(ctx.handle, 0, p, 200, 33, p, p, p, 64, 0, 32, 4, p, None, 0) == 1
    assert q(ctx.handle, 0, p, 200, 33, p, p, p, 64, 0, 32, 4, p, p + 16, need.value) == 1
    assert q(ctx.handle, 0, p + 2, 1, 64, p, p, p, 64, 1, 32, 4, p, p, 1 << 16) == 1
    assert q(ctx.handle, 0, p, 1, 64, p, p + 2, p, 64, 1, 32, 4, p, p, 1 << 16) == 1
    assert q(ctx.handle, 0, p, 1, 64, None, p, p, 64, 1, 32, 4, p, p, 1 << 16) == 1
    cfg = _lib.FfnConfig(64, 64, 0, 32, 4, 0)
    w = _lib.FfnWeights(*[_lib.QWeight(p, p, p)] * 3)
    f = lib.moe_gated_ffn_forward
    assert f(ctx.handle, C.byref(cfg), C.byref(w), p, 200, None, None, None, p, None, 0) == 1
    assert f(ctx.handle, C.byref(cfg), C.byref(w), p, 1, None, p, None, p, p, 1 << 16) == 1
    assert b"together" in lib.moe_last_error(ctx.handle)
    assert f(ctx.handle, C.byref(cfg), None, p, 1, None, None, None, p, p, 1 << 16) == 1
    rc = _lib.RopeConfig(0, 64, 0, 0, 10000.0, 1.0, 1.0)
    s3 = (C.c_int64 * 3)(64, 64, 64)
    r = lambda cfg=rc, D=64, base=p: lib.moe_fast_rope(ctx.handle, C.byref(cfg), base, s3, 1, 1, 1, D, 0, None, 0, None, p, s3)  # noqa: E731
    assert r(D=32) == 1 and r(D=8192) == 2 and r(base=p + 1) == 1
    assert r(_lib.RopeConfig(0, 63, 0, 0, 10000.0, 1.0, 1.0)) == 1
    assert r(_lib.RopeConfig(0, 64, 0, 0, -1.0, 1.0, 1.0)) == 1
    assert r(_lib.RopeConfig(0, 64, 0, 0, 10000.0, float("nan"), 1.0)) == 1
    assert r(_lib.RopeConfig(7, 64, 0, 0, 10000.0, 1.0, 1.0)) == 1
    torch.cuda.synchronize()
    assert int(t.sum()) == 0


# ---- a decoder layer's pieces together: projections -> rotation -> feed-forward, beside MoE blocks

class _Layer:
    def __init__(self, seed, H=256, heads=4, D=64, I=384):
        from mlx_rs_b200.block import DenseMlp
        from mlx_rs_b200.synth import QWeight
        gen = _gen(seed)
        self.heads, self.D = heads, D
        self.qkv = R.QW(gen, 3 * heads * D, H, 32, BF16, True, "cuda", scale=0.005)
        self.qs = [R.QW(gen, I, H, 64, BF16, True, "cuda", 0.01), R.QW(gen, I, H, 64, BF16, True, "cuda", 0.01),
                   R.QW(gen, H, I, 64, BF16, True, "cuda", 0.01)]
        self.mlp = DenseMlp(*[QWeight(q.w, q.scales, q.biases) for q in self.qs])

    def __call__(self, x):
        from mlx_rs_b200 import ops
        T = x.shape[0]
        qkv = ops.quantized_matmul(x, self.qkv.w, self.qkv.scales, self.qkv.biases, group_size=32)
        v = qkv.view(1, T, 3 * self.heads, self.D).transpose(1, 2)
        ops.fast_rope(v[:, :2 * self.heads], self.D, offset=100, out=v[:, :2 * self.heads])
        return self.mlp(v[0, self.heads:2 * self.heads].transpose(0, 1).reshape(T, -1).contiguous())


@pytest.mark.parametrize("T", [1, 6, 50, 200])
def test_projection_rotation_and_block_together(T):
    layer = _Layer(31)
    x = R.rand(_gen(T), T, 256, dtype=BF16, device="cuda")
    want, _ = R.qmm(x, layer.qkv)
    u = R.U[BF16]
    r, _ = R.rope(want.to(BF16).view(1, T, 12, 64).transpose(1, 2)[:, :8], 64, offset=100)
    k = r[0, 4:8].transpose(0, 1).reshape(T, -1)
    y = R.ffn(k.to(BF16), *layer.qs, "silu")[0]
    # the block's input is off by sqrt(2 + 1 + 1) u normwise (the product's two roundings against
    # one here, the rotation's, and the rounding of k); the block passes that on about twice
    # (both projections) and adds its own 3 u
    assert R.rel(layer(x), y) <= (2 * 2 * 2 ** 0.5 + 3) * u


def test_two_captured_graphs_and_eager_calls_share_nothing():
    """Graphs of two layers replayed in turn on two streams, an eager call of a larger batch in
    between: every output has the bits of the eager one."""
    from mlx_rs_b200.graph import GraphedForward
    a, b = _Layer(41), _Layer(42)
    for T in (3, 150):
        xs = [R.rand(_gen(T, i), T, 256, dtype=BF16, device="cuda") for i in range(4)]
        want = [(a(x).clone(), b(x).clone()) for x in xs]
        ga, gb = GraphedForward(a, xs[0]), GraphedForward(b, xs[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        big = R.rand(_gen(9), 700, 256, dtype=BF16, device="cuda")
        for i, x in enumerate(xs):
            ya = ga(x).clone()
            with torch.cuda.stream(side):
                yb = gb(x).clone()
            a(big)
            torch.cuda.synchronize()
            assert torch.equal(ya, want[i][0]) and torch.equal(yb, want[i][1])


def test_calls_on_two_streams_and_threads():
    import threading
    layers = [_Layer(51), _Layer(52)]
    xs = [R.rand(_gen(60 + i), 40 + 100 * i, 256, dtype=BF16, device="cuda") for i in range(2)]
    want = [l(x) for l, x in zip(layers, xs)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                y = layers[i](xs[i])
                s.synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


@pytest.mark.parametrize("T", [2, 140])
def test_dense_layer_in_a_moe_stack(T):
    """A residual stack whose first layer is dense, eager and as one graph."""
    import mlx_rs_b200.synth as S
    from gpu_util import make_block
    from mlx_rs_b200.block import MoeStack, RmsNorm
    from mlx_rs_b200.graph import GraphedForward
    moe = make_block(S.host_block(S.MoeConfig(256, 8, 2, 128, 0, S.SCORING_SOFTMAX, True, False), 3))
    dense = _Layer(71).mlp
    norms = [RmsNorm((1 + 0.1 * torch.randn(256, generator=_gen(i))).to(BF16).cuda()) for i in range(2)]
    stack = MoeStack([dense, moe], norms, residual=True)
    x = R.rand(_gen(T), T, 256, dtype=BF16, device="cuda")
    y = stack(x)
    assert torch.equal(y, moe.forward_layer(dense.forward_layer(x, norms[0].weight, 1e-6), norms[1].weight, 1e-6))
    assert torch.equal(GraphedForward(stack, x)(x), y)


def test_backward_captured_in_a_graph():
    layer = _Layer(81)
    x, dy = (R.rand(_gen(82 + i), 130, 256, dtype=BF16, device="cuda") for i in range(2))
    step = lambda: layer.mlp.vjp(layer.mlp.forward_saved(x)[1], dy)  # noqa: E731
    want = [t.clone() for t in step()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_of_huge_activations_are_finite():
    """Where the derivative is 0 or 1 to the last bit, its factors must not overflow: dg and du
    of large g, u, against the formulas' limits."""
    from mlx_rs_b200 import ops
    H, I, T = 64, 64, 140
    gen = _gen(91)
    from mlx_rs_b200.synth import QWeight
    q = [R.QW(gen, r, c, 32, BF16, True, "cuda") for r, c in ((I, H), (I, H), (H, I))]
    w = [QWeight(a.w, a.scales, a.biases) for a in q]
    g = torch.tensor([1e4, -1e4, 1e15, -1e15, 1e25, -1e25, 3e38, -3e38], device="cuda").to(BF16).repeat(T, I // 8)
    u, dy = torch.ones_like(g), R.rand(gen, T, H, dtype=BF16, device="cuda")
    dh = R.qmm(dy, q[2], transpose=False)[0]
    for act in ("silu", "gelu"):
        _, dg, du = ops.gated_ffn_vjp(g, u, dy, *w, activation=act, group_size=32)
        assert bool(torch.isfinite(dg).all())
        # u = 1, act' = 1 or 0: dg is dh (weights and result rounded once each) or 0
        assert R.rel(dg[g > 0], dh[g > 0]) <= 2 * R.U[BF16] and float(dg[g < 0].abs().max()) == 0
        assert float(du[g < 0].abs().max()) == 0


def test_calls_with_and_without_ctypes_agree(monkeypatch):
    from mlx_rs_b200 import ops
    assert ops._calls is not None
    qs, ws, x, dy = _ffn_case(37, 256, 384, 64, BF16)
    xr = R.rand(_gen(92), 2, 3, 5, 64, dtype=F32, device="cuda")
    off = torch.tensor([4, 9], device="cuda")
    freqs = torch.linspace(1, 50, 16, device="cuda")

    def run():
        out, g, u = ops.gated_ffn(x, *ws, residual=x, save=True)
        return [out, g, u, *ops.gated_ffn_vjp(g, u, dy, *ws),
                ops.quantized_matmul(x, qs[0].w, qs[0].scales, qs[0].biases, transpose=True, group_size=64),
                ops.quantized_matmul(dy, qs[2].w, qs[2].scales, qs[2].biases, transpose=False, group_size=64),
                ops.quantized_matmul(x.view(1, 37, 256), qs[1].w.view(torch.uint32), qs[1].scales, None, group_size=64),
                ops.fast_rope(xr, 32, True, 1000.0, 0.5, off, None, 1.5, True), ops.fast_rope(xr, 32, freqs=freqs, offset=-3)]

    with_c = run()
    monkeypatch.setattr(ops, "_calls", None)
    for a, b in zip(with_c, run()):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


def test_first_calls_inside_a_capture():
    """A process whose first calls of every operator are captured, with sizes of each form."""
    import subprocess
    import sys
    code = """
import torch
from mlx_rs_b200 import ops
import dense_ref as R
from mlx_rs_b200.synth import QWeight
gen = torch.Generator().manual_seed(5)
bf = torch.bfloat16
q = [R.QW(gen, r, c, 32, bf, True, "cuda") for r, c in ((192, 128), (192, 128), (128, 192))]
w = [QWeight(a.w, a.scales, a.biases) for a in q]
xs = [R.rand(gen, T, 128, dtype=bf, device="cuda") for T in (1, 40, 300, 2100)]
def step(x):
    out, g, u = ops.gated_ffn(x, *w, group_size=32, save=True)
    y = ops.quantized_matmul(out, q[0].w, q[0].scales, q[0].biases, group_size=32)
    return [*ops.gated_ffn_vjp(g, u, out, *w, group_size=32), ops.fast_rope(y.view(1, -1, 3, 64).transpose(1, 2), 64)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = [step(x) for x in xs]
graph.replay()
torch.cuda.synchronize()
for x, g in zip(xs, got):
    assert all(torch.equal(a, b) for a, b in zip(step(x), g))
print("same")
"""
    import os
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.dirname(here)]))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240, env=env)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_rope_entry_refuses_overlapping_rows_and_far_offsets():
    import mlx_rs_b200
    from mlx_rs_b200 import _lib, ops
    from mlx_rs_b200._lib import MlxError
    ctx = _lib.context_for(0)
    lib = mlx_rs_b200.library()
    t = torch.ones(1 << 12, dtype=torch.float32, device="cuda")
    cfg = _lib.RopeConfig(2, 8, 0, 0, 10000.0, 1.0, 1.0)

    def call(strides, offset=0, sizes=(2, 2, 2)):
        s = (C.c_int64 * 3)(*strides)
        return lib.moe_fast_rope(ctx.handle, C.byref(cfg), t.data_ptr(), s, *sizes, 8, offset, None, 0, None, t.data_ptr(), s)
    assert call((0, 16, 8)) == 1 and b"overlap" in lib.moe_last_error(ctx.handle)
    assert call((32, 16, 4)) == 1 and call((8, 8, 16)) == 1 and call((-32, 16, 8)) == 1 and call((2 ** 61, 16, 8)) == 1
    assert call((32, 16, 8), 2 ** 53 + 1) == 1 and call((32, 16, 8), -2 ** 60) == 1
    torch.cuda.synchronize()
    assert float(t.sum()) == t.numel()
    with pytest.raises(MlxError, match="offset"):
        ops.fast_rope(t.view(1, 1, -1, 8), 8, offset=2 ** 53 + 1)
    with pytest.raises(MlxError, match="dims"):
        ops.fast_rope(t.view(1, 1, -1, 8), 2 ** 32 + 8)
