"""Backward passes that fill the device, in flight together: each has a launch whose CTAs wait for
one another, from two contexts' streams and from two graphs."""
import numpy as np
import pytest

from helpers import d, dev, empty, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu


class Backward:
    def __init__(self, seed, m, k, n, scale):
        def normal(i, *s):
            return datagen.normal(seed + i, s, 0, 1).astype(np.float16)

        self.t = [dev(v) for v in (normal(0, m, k), (normal(1, k, n) * np.float16(1 / 32)).astype(np.float16),
                                   normal(2, m, n), (normal(3, m, n) * np.float16(scale)).astype(np.float16))]
        self.out = [empty((m, k), np.float16), empty((k, n), np.float16), empty((n,), np.float32)]

    def run(self, ctx):
        x, w, pre, dy = (d(v) for v in self.t)
        ctx.linear_backward(x, w, abi.ACT_GELU, pre, dy, *(d(v) for v in self.out))

    def values(self):
        return [host(v) for v in self.out]


# dy of ordinary size, and one for which dz is computed twice
@pytest.mark.parametrize("scale", [1, 2.0 ** -9])
@pytest.mark.parametrize("graphs", [False, True])
def test_two_at_once(scale, graphs):
    import torch
    torch.cuda.set_device(0)
    ctxs, streams = [abi.Context(0), abi.Context(0)], [torch.cuda.Stream(), torch.cuda.Stream()]
    work = [Backward(1, 4096, 256, 2048, scale), Backward(11, 3000, 328, 1544, scale)]
    want, replay = [], []
    for c, s, w in zip(ctxs, streams, work):
        torch.cuda.synchronize()
        c.set_stream(s.cuda_stream)
        w.run(c)
        c.synchronize()
        want.append(w.values())
        g = torch.cuda.CUDAGraph()
        if graphs:
            with torch.cuda.graph(g, stream=s):
                for _ in range(5):
                    w.run(c)
        replay.append(g)
        for v in w.out:
            v.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, w, g in zip(ctxs, streams, work, replay):
            if graphs:
                with torch.cuda.stream(s):
                    g.replay()
            else:
                w.run(c)
    for c, w, v in zip(ctxs, work, want):
        c.synchronize()  # no wait ran out
        assert all(np.array_equal(a, b) for a, b in zip(w.values(), v))
    del replay
    torch.cuda.synchronize()
    for c in ctxs:
        c.close()


def test_a_graph_beside_its_own_context(ctx):
    """Eager calls of the context that a graph was captured from, on another stream, between and under
    the graph's replays."""
    import torch
    stream, before = torch.cuda.Stream(), ctx.stream()
    a, b = Backward(21, 4096, 256, 2048, 1), Backward(31, 2000, 264, 1032, 2.0 ** 10)
    want = []
    for w in (a, b):
        w.run(ctx)
        want.append(w.values())
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.graph(g, stream=stream):
            a.run(ctx)
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(before)
    for w in (a, b):
        for v in w.out:
            v.fill_(float("nan"))
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(stream):
            g.replay()
        b.run(ctx)
    torch.cuda.synchronize()
    ctx.synchronize()
    for w, v in zip((a, b), want):
        assert all(np.array_equal(p, q) for p, q in zip(w.values(), v))
