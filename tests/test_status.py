"""Expired waits are reported once, in bits of their own, and not to later contexts."""
import ctypes as C

import pytest

import mlx_rs_b200
from mlx_rs_b200 import _lib


def test_refusals_without_a_context():
    lib, s = mlx_rs_b200.library(), C.c_int32(7)
    assert lib.moe_ctx_expire_wait(None, 1000) == _lib.MOE_ERR_INVALID
    assert lib.moe_ctx_status(None, C.byref(s)) == _lib.MOE_ERR_INVALID


@pytest.mark.gpu
def test_an_expired_wait_is_reported_once():
    import torch

    import dense_ref as R
    from mlx_rs_b200 import ops
    lib = mlx_rs_b200.library()

    def status(ctx):
        s = C.c_int32(-1)
        ctx.check("status", lib.moe_ctx_status(ctx.handle, C.byref(s)))
        return s.value
    a, b = _lib.Context(0), _lib.Context(0)
    assert lib.moe_ctx_expire_wait(a.handle, 0) == _lib.MOE_ERR_INVALID
    assert lib.moe_ctx_expire_wait(a.handle, 10 ** 6 + 1) == _lib.MOE_ERR_INVALID
    assert status(a) == 0 and status(b) == 0
    a.check("wait", lib.moe_ctx_expire_wait(a.handle, 1000))
    assert status(a) == 256 << 16
    assert status(a) == 0 and status(b) == 0 and status(_lib.Context(0)) == 0
    # a product between an expired wait and its report runs as ever and takes nothing away
    q = R.QW(torch.Generator().manual_seed(1), 200, 512, 32, torch.bfloat16, True, "cuda")
    x = torch.ones(40, 512, dtype=torch.bfloat16, device="cuda")
    want = ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=32)
    a.check("wait", lib.moe_ctx_expire_wait(a.handle, 1))
    assert torch.equal(ops.quantized_matmul(x, q.w, q.scales, q.biases, group_size=32), want)
    torch.cuda.synchronize()
    assert status(b) == 256 << 16 and status(a) == 0
