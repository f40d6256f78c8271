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


@pytest.mark.parametrize("through", ["calls", "ctypes"])
def test_inputs_that_require_gradients(through, monkeypatch):
    """Refused while torch would record a graph; the same values under no_grad()."""
    from mlx_rs_b200 import ops
    from mlx_rs_b200._lib import MlxError
    from mlx_rs_b200.block import DenseMlp
    if through == "ctypes":
        monkeypatch.setattr(ops, "_calls", None)
    gen = torch.Generator().manual_seed(2)
    w = [_mk(gen, r, c, 32) for r, c in ((96, 64), (96, 64), (64, 96))]
    x = R.rand(gen, 3, 64, dtype=BF16, device="cuda")
    xg, h = x.clone().requires_grad_(), R.rand(gen, 3, 96, dtype=BF16, device="cuda")
    mlp = DenseMlp(*w, group_size=32)
    calls = [lambda x: ops.quantized_matmul(x, w[0].w, w[0].scales, w[0].biases, group_size=32), lambda x: mlp(x),
             lambda x: mlp.forward_layer(x, torch.ones(64, dtype=BF16, device="cuda")),
             lambda x: mlp.vjp((h, h), x)[0], lambda x: ops.fast_rope(x[None, None], 64)]
    for f in calls:
        with pytest.raises(MlxError, match="requires a gradient"):
            f(xg)
        with torch.no_grad():
            assert torch.equal(f(xg), f(x))
