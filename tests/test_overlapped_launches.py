"""Kernels start while the launch before them may still run (programmatic launches): what that
launch writes is not read-only for their lifetime, and is read by plain loads after the wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-rs_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,tokens", [("qmv.cu", r"xr|a\.x|residual"), ("rope.cu", r"a\.x|xb|offsets"),
                                         ("dense_gemm.cu", r"residual|e\.gate|e\.up"),
                                         ("route.cuh", r"a\.x|a\.xf|p"), ("router.cu", r"a\.x")])
def test_tokens_are_not_read_through_the_read_only_path(name, tokens):
    for call in re.findall(r"(?:__ldg|ldg_\w+)(?:<\w+>)?\(([^;]*);", _code(name)):
        assert not re.search(rf"\b(?:{tokens})\b", call), call


def test_padded_rows_are_not_read_through_the_read_only_path():
    assert "__restrict__" not in _code("dense_pad.cu") and "__ldg" not in _code("dense_pad.cu")


@pytest.mark.parametrize("kernel", ["rms_norm_kernel", "gemma_router_input_kernel"])
def test_norms_do_not_take_their_input_as_read_only(kernel):
    first = re.search(rf"{kernel}\(([^,]*),", _code("combine.cu")).group(1)
    assert first.split() == ["const", "uint16_t*", "x"]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 20, 150])
def test_two_inputs_in_turn_keep_their_bits(T):
    """One block, two inputs in turn through the same workspace and outputs, so that a value left
    from the call before shows; also behind a normalisation and a product that writes x."""
    import torch

    import dense_ref as R
    from mlx_rs_b200 import ops
    from mlx_rs_b200.block import DenseMlp
    from mlx_rs_b200.synth import QWeight
    bf, gen = torch.bfloat16, torch.Generator().manual_seed(17)
    mk = lambda r, c: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 64, bf, True, "cuda"))  # noqa: E731
    mlp, p = DenseMlp(mk(1408, 512), mk(1408, 512), mk(512, 1408)), mk(512, 512)
    back = mk(T + 32 - T % 32 + 33, 512)  # an odd number of rows: x is copied to padded rows first
    odd = back.w.shape[0]
    norm = torch.ones(512, dtype=bf, device="cuda")
    xs = [R.rand(gen, T, 512, dtype=bf, device="cuda") for _ in range(2)]
    zs = [R.rand(gen, T, odd, dtype=bf, device="cuda") for _ in range(2)]

    def call(i):
        y = mlp.forward_layer(xs[i], norm)
        y = mlp(ops.quantized_matmul(y, p.w, p.scales, p.biases, transpose=False))
        z = ops.quantized_matmul(zs[i] * 1, back.w, back.scales, back.biases, transpose=False)
        return y, z
    want = [[t.clone() for t in call(i)] for i in range(2)]
    torch.cuda.synchronize()
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for n in range(600):
        for a, e in zip(call(n & 1), want[n & 1]):
            differ += (a.view(torch.int16) != e.view(torch.int16)).any()
    assert int(differ) == 0
