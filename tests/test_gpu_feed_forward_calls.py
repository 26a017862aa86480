"""How the feed-forward operators are called: bounded device-side waits that run out, other
streams, and two contexts at work at once.

A wait limit of one cycle makes the first wait for a copy still in flight run out;
qsml_synchronize then reports QSML_E_TIMEOUT once, and with the default limit the next call of the
same context gives the right result.  Every wait stays bounded, and the waits that drain a kernel's
own copies and MMAs keep the full limit."""
import os
import subprocess
import sys

import numpy as np
import pytest

from helpers import d, dev, empty, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture
def fresh():
    """A context of its own, so a recorded timeout cannot reach another test."""
    import torch
    torch.cuda.set_device(0)
    c = abi.Context(0)
    yield c
    c.set_wait_limit(0)
    torch.cuda.synchronize()
    c.close()


def expect_timeout(c):
    with pytest.raises(abi.QsmlError) as e:
        c.synchronize()
    assert e.value.status == abi.E_TIMEOUT, e.value
    c.synchronize()  # reported once, then cleared


def normal(seed, *shape, s=1.0, dt=np.float16):
    return datagen.normal(seed, shape, 0.0, s).astype(dt)


# a lone CTA a tile, a cluster that shares the sum, binary32's three parts
@pytest.mark.parametrize("m,k,n,dt", [(300, 640, 4096, np.float16), (1, 4096, 512, np.float16),
                                      (200, 512, 384, np.float32)])
def test_linear_wait_expires_then_recovers(fresh, m, k, n, dt):
    x, w = normal(1, m, k, dt=dt), normal(2, k, n, s=k ** -0.5, dt=dt)
    tx, tw, y = dev(x), dev(w), empty((m, n), dt)
    fresh.set_wait_limit(1)
    fresh.linear(d(tx), d(tw), None, abi.ACT_NONE, None, None, d(y))
    assert fresh.last_kernel().startswith("k_linear_tc"), fresh.last_kernel()
    expect_timeout(fresh)
    fresh.set_wait_limit(0)
    fresh.linear(d(tx), d(tw), None, abi.ACT_NONE, None, None, d(y))
    fresh.synchronize()
    ref = x.astype(np.float64) @ w.astype(np.float64)
    # sums of k terms in binary32 and one rounding, over the largest result
    bar = 2.0 ** -11 + (k + 100) * 2.0 ** -24 if dt == np.float16 else (k + 100) * 2.0 ** -24
    assert np.max(np.abs(host(y) - ref)) <= bar * np.max(np.abs(ref))


@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_backward_wait_expires_then_recovers(fresh, dt):
    """Both gradients in one launch."""
    m, k, n = 512, 1024, 1024
    x, w, dy = normal(1, m, k, dt=dt), normal(2, k, n, s=k ** -0.5, dt=dt), normal(3, m, n, dt=dt)
    tx, tw, tdy, dx, dw = dev(x), dev(w), dev(dy), empty((m, k), dt), empty((k, n), dt)

    def call():
        fresh.linear_backward(d(tx), d(tw), abi.ACT_NONE, None, d(tdy), d(dx), d(dw))
    fresh.set_wait_limit(1)
    call()
    expect_timeout(fresh)
    fresh.set_wait_limit(0)
    call()
    fresh.synchronize()
    x, w, dy = (v.astype(np.float64) for v in (x, w, dy))
    step = 2.0 ** -11 if dt == np.float16 else 2.0 ** -24
    for out, a, b, terms in ((dx, dy, w.T, n), (dw, x.T, dy, m)):
        # as many roundings of a binary32 sum as terms, 100 for the operands' parts, one of the result
        ref, bar = a @ b, (terms + 100) * 2.0 ** -24 * (np.abs(a) @ np.abs(b))
        assert np.all(np.abs(host(out) - ref) <= bar + step * (np.abs(ref) + bar))


def test_no_memory_for_a_workspace():
    """The first driver allocation reports out-of-memory (on the host): the call returns it, the
    next one works."""
    code = """
import sys
sys.path.insert(0, %r)
sys.path.insert(0, %r)
import torch
from helpers import d
from quasarml_b200 import abi
c = abi.Context(0)
x, w, dy = (torch.ones(s, device="cuda") for s in ((40, 64), (64, 72), (40, 72)))
dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(72, device="cuda")
for _ in range(2):
    try:
        c.linear_backward(d(x), d(w), abi.ACT_NONE, None, d(dy), d(dx), d(dw), d(db))
        c.synchronize()
        print("SUMS", dx.unique().tolist(), dw.unique().tolist(), db.unique().tolist())
    except abi.QsmlError as e:
        print("STATUS", e.status)
""" % (os.path.dirname(HERE), HERE)
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, QSML_FAULT_ALLOC_N="1"),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert r.stdout.splitlines() == [f"STATUS {abi.E_OOM}", "SUMS [72.0] [40.0] [40.0]"], r.stdout


# larger than L2 and bound by HBM, so that among the rows of ten calls some are waited for
@pytest.mark.parametrize("shape", [(16384, 4096), (8192, 8192)])
def test_layer_norm_backward_wait_expires_then_recovers(fresh, shape):
    import torch
    tx, tdy = (torch.randn(shape, device="cuda") for _ in range(2))
    tg, dx = dev(normal(5, shape[1], dt=np.float32)), empty(shape, np.float32)
    dg, db = empty(shape[1:], np.float32), empty(shape[1:], np.float32)
    want = [t.clone() for t in (dx, dg, db)]
    fresh.layer_norm_backward(d(tx), d(tg), d(tdy), 1e-5, *(d(t) for t in want))
    fresh.synchronize()
    fresh.set_wait_limit(1)
    for _ in range(10):
        fresh.layer_norm_backward(d(tx), d(tg), d(tdy), 1e-5, d(dx), d(dg), d(db))
    expect_timeout(fresh)
    fresh.set_wait_limit(0)
    fresh.layer_norm_backward(d(tx), d(tg), d(tdy), 1e-5, d(dx), d(dg), d(db))
    fresh.synchronize()
    for t, w in zip((dx, dg, db), want):
        assert np.array_equal(host(t), host(w))


class Step:
    """One context's inputs and outputs of every operator, and the calls."""

    def __init__(self, seed, dt, m, c, f):
        self.x, self.g, self.dy = dev(normal(seed, m, c, dt=dt)), dev(normal(seed + 1, c, dt=np.float32)), \
            dev(normal(seed + 2, m, c, dt=dt))
        self.wg, self.wu = (dev(normal(seed + 3 + i, c, f, s=c ** -0.5, dt=dt)) for i in (0, 1))
        self.wd = dev(normal(seed + 5, f, c, s=f ** -0.5, dt=dt))
        mf, mc = (m, f), (m, c)
        names = dict(gate=mf, up=mf, h=mf, y=mc, dh=mf, dwd=(f, c), dx=mc, dwg=(c, f), dwu=(c, f), dn=mc)
        self.out = {k: empty(s, dt) for k, s in names.items()}
        self.out.update(dg=empty((c,), np.float32), db=empty((c,), np.float32), dbg=empty((f,), np.float32))

    def run(self, ctx):
        o = {k: d(v) for k, v in self.out.items()}
        x, wg, wu, wd, dy = d(self.x), d(self.wg), d(self.wu), d(self.wd), d(self.dy)
        ctx.gated_linear(x, wg, wu, None, None, abi.ACT_GELU, o["gate"], o["up"], o["h"])
        ctx.linear(o["h"], wd, None, abi.ACT_NONE, x, None, o["y"])
        ctx.linear_backward(o["h"], wd, abi.ACT_NONE, None, dy, o["dh"], o["dwd"])
        ctx.gated_linear_backward(x, wg, wu, abi.ACT_GELU, o["gate"], o["up"], o["dh"], o["dx"], o["dwg"], o["dwu"],
                                  o["dbg"])
        ctx.layer_norm_backward(x, d(self.g), o["dx"], 1e-5, o["dn"], o["dg"], o["db"])

    def values(self):
        return {k: host(v) for k, v in self.out.items()}

    def clear(self):
        for v in self.out.values():
            v.fill_(float("nan"))


@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_two_contexts_at_once(dt):
    """Two contexts on streams of their own, their calls in flight together: the bits of each alone."""
    import torch
    ctxs = [abi.Context(0), abi.Context(0)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    steps = [Step(11, dt, 333, 256, 704), Step(31, dt, 150, 520, 1000)]
    want = []
    for c, s, st in zip(ctxs, streams, steps):
        torch.cuda.synchronize()
        c.set_stream(s.cuda_stream)
        st.run(c)
        c.synchronize()
        want.append(st.values())
        st.clear()
    torch.cuda.synchronize()
    for _ in range(5):
        for c, st in zip(ctxs, steps):
            st.run(c)
    for c, st, w in zip(ctxs, steps, want):
        c.synchronize()
        got = st.values()
        assert all(np.array_equal(got[k], w[k]) for k in w)
        c.close()


def test_a_stream_of_the_contexts_own():
    """A context that nobody gave a stream, and one whose stream changes between calls."""
    import torch
    c = abi.Context(0, use_torch_stream=False)
    st = Step(51, np.float16, 90, 128, 264)
    torch.cuda.synchronize()
    st.run(c)
    c.synchronize()
    want = st.values()
    other = torch.cuda.Stream()
    for s in (other.cuda_stream, 0):
        st.clear()
        torch.cuda.synchronize()
        c.set_stream(s)
        st.run(c)
        c.synchronize()
        got = st.values()
        assert all(np.array_equal(got[k], want[k]) for k in want)
    c.close()


def test_calls_between_overlapping_ones(fresh):
    """With overlap on, the operators end the window of calls that may run together: a reduction of
    their result, and their read of a reduction's, see each other's writes."""
    import torch
    fresh.set_overlap(True)
    x = dev(normal(61, 512, 1024, dt=np.float32))
    w = dev(normal(62, 1024, 512, s=1 / 32, dt=np.float32))
    y, s, z = empty((512, 512), np.float32), empty((512,), np.float32), empty((512, 512), np.float32)
    r = [empty((1024,), np.float32) for _ in range(3)]
    for _ in range(20):
        for v in (y, s, z):
            v.fill_(float("nan"))
        for t in r:
            fresh.reduce(abi.RED_SUM, d(x), 0, False, d(t))
        fresh.linear(d(x), d(w), None, abi.ACT_RELU, None, None, d(y))
        fresh.reduce(abi.RED_MAX, d(y), 0, False, d(s))
        fresh.linear(d(x), d(w), d(s), abi.ACT_NONE, None, None, d(z))
    fresh.synchronize()
    ref = x.double() @ w.double()
    assert torch.allclose(s.double(), torch.relu(ref).max(0).values, rtol=0, atol=1124 * 2.0 ** -24 * 40)
    assert torch.allclose(z.double(), ref + s.double(), rtol=0, atol=1124 * 2.0 ** -24 * 40)
