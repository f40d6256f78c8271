"""GPU parity of the dense operators element by element, within dense_bounds.py, over every form of
the products and the block; and the uses of the residual."""
import pytest
import torch

import dense_bounds as B
import dense_ref as R
from test_gpu_dense import FFN, QMM, _close, _ffn_case, _gen

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("M,N,K,g,dt,biases", QMM + [
    (2048, 2048, 2048, 64, F16, True), (40, 4100, 1024, 32, BF16, True), (12, 11264, 512, 32, BF16, True)])
def test_products(M, N, K, g, dt, biases):
    from mlx_rs_b200 import ops
    gen = _gen(M, N, K, 1)
    q = R.QW(gen, N, K, g, dt, biases, "cuda")
    x = R.rand(gen, M, K, dtype=dt, device="cuda")
    got = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=g)
    for m in range(0, M, 512):  # a piece of the tokens at a time
        y, bound = B.product(x[m:m + 512], q, few=M <= 32)
        _close(got[m:m + 512], y, bound, "product")


@pytest.mark.parametrize("M,K,N,g,dt,biases", [
    (1, 2048, 2048, 64, BF16, True), (5, 33, 64, 64, BF16, True), (32, 1001, 128, 128, F16, False),
    (130, 100, 352, 32, F16, True), (512, 5632, 2048, 32, BF16, True), (257, 768, 1408, 64, BF16, False),
    (1030, 520, 320, 64, F16, True), (1025, 99, 256, 128, BF16, True), (130, 8192, 544, 32, F16, True),
    (2300, 1024, 1088, 64, BF16, True)])
def test_products_not_transposed(M, K, N, g, dt, biases):
    from mlx_rs_b200 import ops
    gen = _gen(M, K, N, 1)
    q = R.QW(gen, K, N, g, dt, biases, "cuda")
    x = R.rand(gen, M, K, dtype=dt, device="cuda")
    got = ops.quantized_matmul(x, q.w, q.scales, q.biases, transpose=False, group_size=g)
    _close(got, *B.product(x, q, transpose=False), "product")


@pytest.mark.parametrize("T,H,I,g,dt,kind", FFN + [(200, 2048, 1408, 64, BF16, "silu"), (3, 4096, 1024, 128, F16, "silu")])
def test_block_and_gradients(T, H, I, g, dt, kind):
    """Step by step, each from what the kernel handed on: g and u from x, the output from g and u, dg
    and du from g, u and dy, dx from dg and du."""
    from mlx_rs_b200.block import DenseMlp
    qs, ws, x, dy = _ffn_case(T, H, I, g, dt)
    mlp = DenseMlp(*ws, activation=kind, group_size=g)
    out, (pg, pu) = mlp.forward_saved(x)
    few = T <= 32
    _close(pg, *B.product(x, qs[0], few=few), "g")
    _close(pu, *B.product(x, qs[1], few=few), "u")
    _close(out, *B.block(pg, pu, qs[2], kind, few=few), "out")
    dx, dg, du = mlp.vjp((pg, pu), dy)
    for got, (v, e), name in zip((dg, du), B.gradients(pg, pu, dy, *qs, kind), ("dg", "du")):
        _close(got, v, e, name)
    _close(dx, *B.sums([(dg, qs[0]), (du, qs[1])], False), "dx")


@pytest.mark.parametrize("T,H,I,dt", [(1, 256, 384, BF16), (6, 64, 96, F16), (20, 256, 160, BF16), (90, 128, 96, F16),
                                      (200, 256, 384, BF16), (700, 640, 1408, BF16), (1500, 96, 352, F16), (2100, 384, 640, BF16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_block_with_a_residual(T, H, I, dt, in_place):
    """Every form of the product, several token tiles and the weights dequantised once among them;
    and out in the residual's own memory, as the C entry allows."""
    import ctypes as C

    import mlx_rs_b200
    from mlx_rs_b200 import _lib, ops
    g = 32
    qs, ws, x, r = _ffn_case(T, H, I, g, dt)
    plain, pg, pu = ops.gated_ffn(x, *ws, group_size=g, save=True)
    want = ops.gated_ffn(x, *ws, group_size=g, residual=r)
    _close(want, *B.block(pg, pu, qs[2], "silu", residual=r, few=T <= 32), "out")
    lib, ctx = mlx_rs_b200.library(), _lib.context_for(0)
    ctx.bind_stream(torch.cuda.current_stream().cuda_stream)
    cfg = ops.ffn_config(H, I, dt, "silu", g, 4)
    wts = ops.ffn_weights("ffn", cfg, ops.ffn_tensors(*ws), x)
    need = C.c_size_t()
    assert lib.moe_gated_ffn_workspace(C.byref(cfg), T, 0, C.byref(need)) == 0
    ws_ = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    buf = torch.full((T + 2, H), 7.0, dtype=dt, device="cuda")  # a row on either side stays as it is
    out = buf[1:-1]
    if in_place:
        out.copy_(r)
    ctx.check("ffn", lib.moe_gated_ffn_forward(ctx.handle, cfg, wts, x.data_ptr(), T, (out if in_place else r).data_ptr(),
                                               None, None, out.data_ptr(), ws_.data_ptr(), need.value))
    assert torch.equal(out, want)
    assert bool((buf[0] == 7).all() and (buf[-1] == 7).all())
