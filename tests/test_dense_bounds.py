"""The bounds of dense_bounds.py: they hold for roundings as the kernels make them, and one element
that is wrong exceeds them."""
import pytest
import torch

import dense_bounds as B
import dense_ref as R

BF16, F16 = torch.bfloat16, torch.float16

# the forms of the GPU tests, with up to 16 of their tokens and 512 of their outputs
FORMS = [  # M, N, K, group, dtype, transpose
    (1, 512, 2048, 32, BF16, True), (16, 33, 4096, 64, F16, True), (17, 96, 5632, 32, BF16, True), (3, 512, 1408, 64, F16, True),
    (200, 512, 2048, 32, BF16, True), (200, 512, 8192, 32, BF16, True), (1024, 512, 512, 64, F16, True), (130, 544, 8192, 32, F16, False),
    (512, 512, 5632, 32, BF16, False), (257, 512, 768, 64, BF16, False), (1, 512, 2048, 64, BF16, False)]


@pytest.mark.parametrize("M,N,K,g,dt,tr", FORMS)
def test_a_zeroed_element_exceeds_the_bound(M, N, K, g, dt, tr):
    """The bound is under 0.12 of the results' rms in bf16 and 0.06 in f16, so at least 9 (19) of 10
    (20) elements exceed it when they are zero; those it covers are themselves that small."""
    gen = torch.Generator().manual_seed(M + K)
    rows, cols = (N, K) if tr else (K, N)
    q = R.QW(gen, rows, cols, g, dt)
    x = R.rand(gen, min(M, 16), K, dtype=dt)
    y, bound = B.product(x, q, tr, tr and M <= 32)
    rms = float(y.square().mean().sqrt())
    assert float((bound - R.U[dt] * y.abs()).mean()) < (0.12 if dt == BF16 else 0.06) * rms
    assert float((y.abs() > bound).double().mean()) >= (0.9 if dt == BF16 else 0.95)
    # with the operator's roundings, its weights to the type and the result, it holds
    w = q.dense().to(dt).double()
    got = (x.double() @ (w.t() if tr else w)).to(dt).double()
    assert bool(((got - y).abs() <= bound).all())
    # and where an output's largest g weights are left out, some token shows it
    col = (w.t() if tr else w)[:, 3]
    largest = torch.topk(col.abs(), g).indices
    lost = x.double()[:, largest] @ col[largest]
    assert M == 1 or bool((lost.abs() > bound[:, 3]).any())


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_the_blocks_bound_holds_and_shows_a_zeroed_element(kind, dt):
    gen = torch.Generator().manual_seed(4)
    T, H, I = 24, 256, 640
    gate, up, down = (R.QW(gen, r, c, 32, dt) for r, c in ((I, H), (I, H), (H, I)))
    x = R.rand(gen, T, H, dtype=dt)
    g, u = (x.double() @ q.dense().to(dt).double().t() for q in (gate, up))
    h = (R.act(g, kind)[0] * u).to(dt)
    got = (h.double() @ down.dense().to(dt).double().t()).to(dt).double()
    y, bound = B.block(g.to(dt), u.to(dt), down, kind)
    assert bool(((got - y).abs() <= bound).all())
    assert float((y.abs() > bound).double().mean()) >= (0.8 if dt == BF16 else 0.95)
    dy = R.rand(gen, T, H, dtype=dt)
    gs, us = g.to(dt), u.to(dt)
    dh = dy.double() @ down.dense().to(dt).double()
    a, da = R.act(gs.double(), kind)
    for got, (v, e) in zip((dh * us.double() * da, dh * a), B.gradients(gs, us, dy, gate, up, down, kind)):
        got = got.to(dt).double()
        assert bool(((got - v).abs() <= e).all())
        big = v.abs() > 0.1 * v.square().mean().sqrt()
        assert float((v.abs() > e)[big].double().mean()) >= 0.9
