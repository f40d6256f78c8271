"""Uses of the dense operators that their documentation allows, beyond the parity cases."""
import pytest
import torch

import dense_ref as R

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _mk(gen, r, c, g=64, dt=BF16):
    from mlx_rs_b200.synth import QWeight
    q = R.QW(gen, r, c, g, dt, True, "cuda")
    return QWeight(q.w, q.scales, q.biases)


@pytest.mark.parametrize("through", ["calls", "ctypes"])
def test_replaced_weights_are_used(through, monkeypatch):
    """A block whose weights, or one of their tensors, were replaced computes with the new ones."""
    from mlx_rs_b200 import ops
    from mlx_rs_b200.block import DenseMlp
    if through == "ctypes":
        monkeypatch.setattr(ops, "_calls", None)
    gen = torch.Generator().manual_seed(1)
    x = R.rand(gen, 5, 256, dtype=BF16, device="cuda")
    mlp = DenseMlp(_mk(gen, 384, 256), _mk(gen, 384, 256), _mk(gen, 256, 384))
    mlp(x)
    mlp.up = _mk(gen, 384, 256)
    assert torch.equal(mlp(x), ops.gated_ffn(x, mlp.gate, mlp.up, mlp.down))
    mlp.down.scales = mlp.down.scales * 2
    mlp.down.biases = None
    out, saved = mlp.forward_saved(x)
    assert torch.equal(out, ops.gated_ffn(x, mlp.gate, mlp.up, mlp.down))
    want = ops.gated_ffn_vjp(*saved, x, mlp.gate, mlp.up, mlp.down)
    assert all(torch.equal(a, b) for a, b in zip(mlp.vjp(saved, x), want))
    mlp.gate.w = torch.nn.Parameter(mlp.gate.w.flip(0), requires_grad=False)
    assert torch.equal(mlp(x), ops.gated_ffn(x, mlp.gate, mlp.up, mlp.down))
