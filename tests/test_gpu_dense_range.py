"""Few-token products at the ends of the type's range: infinities, NaN, and finite tokens whose
products with the offset weight fields (16 + q) leave the range of fp32 although the result does
not. Expected values in 64 bits."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def _acc(x, q, terms):
    """What fp32 sums of `terms` products that are not zero may be off by: the kernel sums x (16 + q)
    and x, so that its factors are up to 31 s and b; 16 more steps for the scales and the warps."""
    return (terms + 16) * 2.0 ** -23 * (x.double().abs() @ q.spread(31.0).t())


def _same(got, want, acc=0.0):
    """Rounded once, plus acc: infinities, NaN and overflow where the 64-bit result has them.
    Results within a part in 2^-7 of the largest finite value may round either way."""
    big = torch.finfo(got.dtype).max
    g, edge = got.double(), (want.abs() > big * (1 - 2 ** -7)) & (want.abs() < big * (1 + 2 ** -7))
    assert torch.equal(g.isnan(), want.isnan())
    over = (want.abs() >= big) & ~edge
    assert torch.equal(g[over], torch.sign(want[over]) * INF)
    fin = (want.abs() < big) & ~edge
    bound = R.U[got.dtype] * want.abs() + acc * (1 + R.U[got.dtype])
    assert bool((g[fin] - want[fin]).abs().le(bound[fin]).all())


@pytest.mark.parametrize("M", [1, 3, 8, 13, 32])
@pytest.mark.parametrize("N,K,g", [(40, 64, 32), (300, 1408, 64), (129, 2048, 128), (64, 96, 32)])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_products_of_infinities(M, N, K, g, dt):
    from mlx_rs_b200 import ops
    gen = torch.Generator().manual_seed(M * N + K)
    q = R.QW(gen, N, K, g, dt, True, "cuda")
    x = R.rand(gen, M, K, dtype=dt, device="cuda")
    clean = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=g, transpose=True) if g != 64 or dt == F16 else None
    bad = x.clone()
    bad[0, K - 1] = INF
    if M > 2:
        bad[1, 5], bad[1, K // 2], bad[2, 7] = INF, -INF, NAN
    want = bad.double() @ q.dense().t()
    got = ops.quantized_matmul(bad, q.w, q.scales, q.biases, group_size=g)
    rows = [i for i in range(M) if i > 2 or (M <= 2 and i > 0)]
    if clean is None:
        return  # bf16 at group 64 is the package's other product
    assert torch.equal(got[rows], clean[rows])
    _same(got[:3 if M > 2 else 1], want[:3 if M > 2 else 1])


@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("N,K,g", [(40, 64, 32), (257, 1024, 128)])
def test_products_of_huge_tokens(M, N, K, g):
    from mlx_rs_b200 import ops
    gen = torch.Generator().manual_seed(M + N)
    q = R.QW(gen, N, K, g, BF16, True, "cuda")
    for big in (2e37, 3e38):
        x = torch.zeros(M, K, dtype=BF16, device="cuda")
        x[:, 3::g] = big * torch.sign(torch.randn(M, x[:, 3::g].shape[1], generator=gen)).to(BF16).cuda()
        got = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=g)
        want = x.double() @ q.dense().t()
        # where the sum is finite in 64 bits and its terms do not cancel below a tenth
        keep = want.abs() > 0.1 * (x.double().abs() @ q.dense().abs().t())
        assert bool(keep.any())
        _same(torch.where(keep, got, 0), torch.where(keep, want, 0), _acc(x, q, K // g))


@pytest.mark.parametrize("T", [1, 6])
@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_block_of_huge_and_infinite_tokens(T, kind):
    """g, u as saved, by the same rule; a token of one element makes both exact products."""
    from mlx_rs_b200 import ops
    from mlx_rs_b200.synth import QWeight
    gen = torch.Generator().manual_seed(T)
    q = [R.QW(gen, r, c, 32, BF16, True, "cuda") for r, c in ((96, 64), (96, 64), (64, 96))]
    w = [QWeight(a.w, a.scales, a.biases) for a in q]
    x = torch.zeros(T, 64, dtype=BF16, device="cuda")
    x[0, 9] = INF
    x[1:, 5] = 2e37
    _, g, u = ops.gated_ffn(x, *w, activation=kind, group_size=32, save=True)
    x[0, 9] = 0  # the row is infinite or NaN whatever its sums
    acc = [_acc(x, a, 1) for a in q[:2]]
    x[0, 9] = INF
    _same(g, x.double() @ q[0].dense().t(), acc[0])
    _same(u, x.double() @ q[1].dense().t(), acc[1])


@pytest.mark.parametrize("T", [1, 6, 20])
@pytest.mark.parametrize("in_place", [False, True])
def test_block_of_infinite_tokens_with_a_residual(T, in_place):
    """h is infinite in one element of one token: that token's outputs are infinities, in place too."""
    import ctypes as C

    import mlx_rs_b200
    from mlx_rs_b200 import _lib, ops
    from mlx_rs_b200.synth import QWeight
    gen = torch.Generator().manual_seed(T)
    q = [R.QW(gen, r, c, 32, BF16, True, "cuda") for r, c in ((96, 64), (96, 64), (64, 96))]
    keep = torch.zeros(96, 1, dtype=BF16, device="cuda")
    keep[7] = 1  # u is zero but in one row, so h is but there
    q[1].scales, q[1].biases = q[1].scales * keep, q[1].biases * keep
    w = [QWeight(a.w, a.scales, a.biases) for a in q]
    x, r = (R.rand(gen, T, 64, dtype=BF16, device="cuda") for _ in range(2))
    clean = ops.gated_ffn(x, *w, group_size=32, residual=r)
    x[0] = 0
    x[0, 9] = 1e23 * torch.sign(q[0].dense()[7, 9])  # g u is beyond the range there
    h = torch.zeros(T, 96, dtype=torch.float64, device="cuda")
    h[0, 7] = INF * torch.sign(x[0, 9] * q[1].dense()[7, 9])
    want = r.double() + h @ q[2].dense().t()
    assert bool(want[0].isinf().all())
    out = r.clone() if in_place else torch.empty_like(r)
    lib, ctx = mlx_rs_b200.library(), _lib.context_for(0)
    ctx.bind_stream(torch.cuda.current_stream().cuda_stream)
    cfg = ops.ffn_config(64, 96, BF16, "silu", 32, 4)
    wts = ops.ffn_weights("ffn", cfg, ops.ffn_tensors(*w), x)
    need = C.c_size_t()
    assert lib.moe_gated_ffn_workspace(C.byref(cfg), T, 0, C.byref(need)) == 0
    ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    ctx.check("ffn", lib.moe_gated_ffn_forward(ctx.handle, cfg, wts, x.data_ptr(), T, (out if in_place else r).data_ptr(),
                                               None, None, out.data_ptr(), ws.data_ptr(), need.value))
    assert torch.equal(out[1:], clean[1:])
    assert torch.equal(out[0].double(), want[0])
