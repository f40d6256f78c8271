"""Calls from several threads: each has contexts of its own, with one stream and one scratch."""
import gc
import threading

import pytest
import torch

from mlx_rs_b200 import _lib


def _run(*fs):
    """The results of the functions, each on a thread of its own."""
    out = [None] * len(fs)

    def work(i):
        out[i] = fs[i]()
    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(fs))]
    [t.start() for t in ts]
    [t.join() for t in ts]
    return out


class _Fake:
    closed = []

    def __init__(self, device):
        self.device, self.captured = device, False

    def __del__(self):
        _Fake.closed.append(self.device)


def test_threads_have_contexts_of_their_own(monkeypatch):
    monkeypatch.setattr(_lib, "Context", _Fake)
    gate = threading.Barrier(3)

    def mine():
        a, b = _lib.context_for(3), _lib.context_for(4)
        gate.wait(20)  # all of them live at once
        return id(a), id(b), _lib.context_for(3) is a
    got = _run(mine, mine, mine)
    assert len({i for a, b, _ in got for i in (a, b)}) == 6 and all(same for _, _, same in got)


def test_contexts_end_with_their_thread_unless_captured(monkeypatch):
    monkeypatch.setattr(_lib, "Context", _Fake)
    monkeypatch.setattr(_lib, "_kept", [])
    _Fake.closed = []

    def use():
        _lib.context_for(5)
        _lib.context_for(6).captured = True
    _run(use)
    gc.collect()
    assert _Fake.closed == [5] and [c.device for c in _lib._kept] == [6]


def _layers():
    import dense_ref as R
    import mlx_rs_b200.synth as S
    from gpu_util import make_block
    from mlx_rs_b200 import ops
    from mlx_rs_b200.block import DenseMlp
    from mlx_rs_b200.synth import QWeight
    bf, gen = torch.bfloat16, torch.Generator().manual_seed(23)
    mk = lambda r, c: (lambda q: QWeight(q.w, q.scales, q.biases))(R.QW(gen, r, c, 64, bf, True, "cuda", 0.01))  # noqa: E731
    moe = make_block(S.host_block(S.MoeConfig(256, 8, 2, 128, 0, S.SCORING_SOFTMAX, True, False), 3))
    mlp, p = DenseMlp(mk(384, 256), mk(384, 256), mk(256, 384)), mk(256, 256)
    norm = (1 + 0.1 * torch.randn(256, generator=gen)).to(bf).cuda()

    def step(x):
        y = mlp.forward_layer(x, norm)
        y = ops.quantized_matmul(y, p.w, p.scales, p.biases)  # the context's own entry, group size 64
        return ops.fast_rope(moe.forward_layer(y, norm)[None], 64)[0]
    xs = [R.rand(gen, T, 256, dtype=bf, device="cuda") for T in (40, 140, 3)]
    return step, xs


@pytest.mark.gpu
@pytest.mark.parametrize("through", ["calls", "ctypes"])
def test_layers_on_threads_with_streams_of_their_own(through, monkeypatch):
    """Norm, dense block, product and MoE block in one step, three threads, a stream each: every
    launch of a step has to go to its thread's stream and its thread's scratch."""
    from mlx_rs_b200 import ops
    if through == "ctypes":
        monkeypatch.setattr(ops, "_calls", None)
    step, xs = _layers()
    want = [step(x) for x in xs]
    torch.cuda.synchronize()

    def work(i):
        def f():
            s, bad = torch.cuda.Stream(), 0
            with torch.cuda.stream(s):
                for _ in range(150):
                    y = step(xs[i])
                    s.synchronize()
                    bad += not torch.equal(y, want[i])
            return bad
        return f
    assert _run(*[work(i) for i in range(3)]) == [0, 0, 0]


@pytest.mark.gpu
def test_a_thread_captures_what_another_warmed_up():
    """Its first call of a MoE block is captured, so its scratch comes in the capture; the graph
    outlives the thread."""
    step, xs = _layers()
    want = [step(x) for x in xs]
    torch.cuda.synchronize()

    def capture():
        g, x = torch.cuda.CUDAGraph(), xs[1].clone()
        with torch.cuda.graph(g):
            y = step(x)
        return g, x, y
    ((g, x, y),) = _run(capture)
    gc.collect()
    _run(lambda: step(xs[0]).sum().item())
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[1])


@pytest.mark.gpu
def test_a_thread_may_end_while_another_captures():
    """Its context's scratch is freed meanwhile; the capture goes on."""
    step, xs = _layers()
    want = [step(x) for x in xs]
    torch.cuda.synchronize()
    used, end = threading.Event(), threading.Event()

    def worker():
        step(xs[0])
        torch.cuda.synchronize()
        used.set()
        end.wait(60)
    t = threading.Thread(target=worker)
    t.start()
    assert used.wait(60)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(xs[1])
        end.set()
        t.join()
        gc.collect()
        z = step(xs[2])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[1]) and torch.equal(z, want[2])


@pytest.mark.gpu
def test_a_graph_outlives_the_growth_of_its_scratch():
    """After the capture a larger eager call makes the context's scratch grow, and a larger capture
    again; each graph goes on with the scratch it was captured with."""
    import mlx_rs_b200.synth as S
    from gpu_util import make_block

    def thread():  # a context of its own, whose scratch starts small
        blk = make_block(S.host_block(S.MoeConfig(256, 8, 2, 128, 0, S.SCORING_SOFTMAX, True, False), 3))
        gen = torch.Generator().manual_seed(29)
        xs = [torch.randn(T, 256, generator=gen).to(torch.bfloat16).cuda() for T in (20, 6000, 12000, 24000)]
        graphs = []
        for x in (xs[0], xs[2]):
            blk.forward(xs[0])
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = blk.forward(x)
            graphs.append((g, x, y))
            blk.forward(xs[1])
        blk.forward(xs[3])
        junk = [torch.full((1 << 22,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(8)]  # noqa: F841
        for g, x, y in graphs * 2:
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, blk.forward(x))
        return True
    assert _run(thread) == [True]
