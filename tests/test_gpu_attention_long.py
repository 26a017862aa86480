"""GPU attention over tens of thousands of keys in binary16: sums that leave the tensor cores' accumulators on the
way.  Against binary64 (torch, on the device, in rows of 2000)."""
import numpy as np
import pytest

from helpers import d
from quasarml_b200 import abi

pytestmark = pytest.mark.gpu
NAN = float("nan")

# An accumulator's sum of 8192 numbers of one sign loses 5e-5 of itself (the header); twice that is allowed.
LOSS = 1e-4
# Roundings of weights and of dS are 2^-11 at most each and independent, so a sum's norm of errors is below the
# root of their squares' sum times 2^-11; the output's own adds 2^-11.
NORM = 2 * 2.0 ** -11


def tensors(B, sq, sk, hq, hk, D, seed=1, positive=True):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")
    q, k = (0.5 * normal(B, sq, hq, D)).half(), normal(B, sk, hk, D).half()
    if positive:
        v, do = (1 + torch.rand(s, generator=g, device="cuda") for s in ((B, sk, hk, D), (B, sq, hq, D)))
    else:
        v, do = normal(B, sk, hk, D), normal(B, sq, hq, D)
    return q, k, v.half(), do.half()


def exact(q, k, v, do, scale, window=0, sinks=0, nq=None, nk=None, given=None):
    """o, dq, dk, dv in binary64; do None: o alone.  Gradients go by sum(dout o) of the o given, as the operator's do;
    queries of the first 128 positions, which see the first tile of keys alone, by sum(P dP)."""
    import torch
    B, sq, hq, D = q.shape
    hk = k.shape[2]
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(o), *(torch.zeros(k.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(B):
        n, m = (nq[b] if nq else sq), (nk[b] if nk else k.shape[1])
        j = torch.arange(m, device="cuda")[None]
        for h in range(hq):
            c = h // (hq // hk)
            kk, vv = k[b, :m, c].double(), v[b, :m, c].double()
            for r in range(0, n, 2000):
                at = slice(r, min(r + 2000, n))
                p = torch.arange(at.start, at.stop, device="cuda")[:, None] + m - n
                seen = j <= p
                if window:
                    seen &= (p - j < window) | (j < sinks)
                w = torch.softmax((q[b, at, h].double() @ kk.T * scale).masked_fill(~seen, -np.inf), 1).nan_to_num(0.0)
                o[b, at, h] = w @ vv
                if do is None:
                    continue
                g = do[b, at, h].double()
                dv[b, :m, c] += w.T @ g
                dp = g @ vv.T
                delta = (w * dp).sum(1, keepdim=True)
                if given is not None:
                    delta = torch.where(p < 128, delta, (g * given[b, at, h].double()).sum(1, keepdim=True))
                w *= dp - delta
                dq[b, at, h] = w @ kk * scale
                dk[b, :m, c] += w.T @ q[b, at, h].double() * scale
    return o, dq, dk, dv


def run(ctx, q, k, v, do, scale, window=0, sinks=0, nq=None, nk=None):
    import torch
    lengths = [None if n is None else torch.tensor(n, dtype=torch.int32, device="cuda") for n in (nq, nk)]
    how = {"window": window, "sinks": sinks, "q_lengths": None if nq is None else d(lengths[0]),
           "k_lengths": None if nk is None else d(lengths[1])}
    o, lse = torch.full_like(q, NAN), torch.full((q.shape[0], q.shape[2], q.shape[1]), NAN, device="cuda")
    ctx.attention(d(q), d(k), d(v), d(o), scale, lse=d(lse), **how)
    assert ctx.last_kernel() == "k_attention_tc"
    out = [torch.full_like(x, NAN) for x in (q, k, v)]
    if do is not None:
        ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in out], scale, **how)
    ctx.synchronize()
    return o, *out


def norm_error(x, ref):
    return float((x.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("D", [64, 128])
def test_sums_over_many_keys(ctx, D):
    q, k, v, _ = tensors(1, 128, 100000, 1, 1, D)
    o = run(ctx, q, k, v, None, D ** -0.5)[0]
    ref = exact(q, k, v, None, D ** -0.5)[0]
    error = (o.double() - ref) / ref
    assert abs(float(error.mean())) <= LOSS
    assert float(error.abs().max()) <= 2.0 ** -11 + LOSS


@pytest.mark.parametrize("D", [64, 128])
def test_sums_over_many_queries_of_a_group(ctx, D):
    """dv of a key adds up 8 heads' queries."""
    q, k, v, do = tensors(1, 20000, 20000, 8, 1, D)
    got = run(ctx, q, k, v, do, D ** -0.5)
    ref = exact(q, k, v, do, D ** -0.5, given=got[0])
    early = (got[3][:, :128].double() - ref[3][:, :128]) / ref[3][:, :128]
    assert abs(float(early.mean())) <= LOSS
    assert float(early.abs().max()) <= 2.0 ** -11 + LOSS + 2.0 ** -11  # the weights' roundings, at most
    for x, r in zip(got, ref):
        assert norm_error(x, r) <= NORM


@pytest.mark.parametrize("D", [64, 128])
def test_next_tokens_over_many_keys(ctx, D):
    """As many sequences' heads as the device holds CTAs, so that nothing else asks for parts."""
    import torch
    q, k, v, _ = tensors(37, 1, 100000, 8, 8, D)
    o = torch.full_like(q, NAN)
    ctx.attention(d(q), d(k), d(v), d(o), D ** -0.5)
    ctx.synchronize()
    q, k, v, o = (x[[0, 36]] for x in (q, k, v, o))
    ref = exact(q, k, v, None, D ** -0.5)[0]
    error = (o.double() - ref) / ref
    assert abs(float(error.mean())) <= LOSS
    assert float(error.abs().max()) <= 2.0 ** -11 + LOSS


@pytest.mark.parametrize("size", [(2, 300, 20000, 4, 2, 128, 9000, 130), (1, 700, 30000, 2, 1, 72, 20000, 0), (1, 200, 17000, 3, 3, 64, 0, 0),
                                  (1, 17000, 17000, 1, 1, 24, 10000, 1000)], ids=str)
def test_long_windows(ctx, size):
    B, sq, sk, hq, hk, D, window, sinks = size
    q, k, v, do = tensors(B, sq, sk, hq, hk, D, 2, positive=False)
    got = run(ctx, q, k, v, do, D ** -0.5, window, sinks)
    for x, r in zip(got, exact(q, k, v, do, D ** -0.5, window, sinks)):
        assert norm_error(x, r) <= NORM


def test_long_sequences_of_ragged_lengths(ctx):
    nq, nk = [300, 129, 0, 70], [20000, 8193, 5000, 8320]
    q, k, v, do = tensors(4, 300, 20000, 2, 1, 64, 3, positive=False)
    got = run(ctx, q, k, v, do, 0.125, 0, 0, nq, nk)
    for x, r in zip(got, exact(q, k, v, do, 0.125, 0, 0, nq, nk)):
        assert norm_error(x, r) <= NORM
        assert not x.double()[r == 0].any()


@pytest.mark.parametrize("back", [False, True])
def test_maxima_that_move_across_long_sums(ctx, back):
    """Keys whose scores rise along 20000 of them, and fall."""
    import torch
    q, k, v, do = tensors(1, 140, 20000, 1, 1, 64, 4, positive=False)
    ramp = torch.arange(20000, device="cuda") / 2000.0
    k = (k.abs() * (ramp.flip(0) if back else ramp)[None, :, None, None]).half()
    q = q.abs()
    # scores to 100: the weights are off by their roundings, 100 u of binary32, besides
    got = run(ctx, q, k, v, do, 0.125)
    for x, r in zip(got, exact(q, k, v, do, 0.125)):
        assert norm_error(x, r) <= 2 * NORM


def test_long_gradients_left_out(ctx):
    import torch
    q, k, v, do = tensors(1, 9000, 9000, 2, 1, 64, 5, positive=False)
    o, dq, dk, dv = run(ctx, q, k, v, do, 0.125)
    lse = torch.empty(1, 2, 9000, device="cuda")
    ctx.attention(d(q), d(k), d(v), d(torch.empty_like(o)), 0.125, lse=d(lse))
    for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1)):
        out = [torch.full_like(x, NAN) if w else None for x, w in zip((q, k, v), want)]
        ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[None if x is None else d(x) for x in out], 0.125)
        ctx.synchronize()
        for x, y in zip(out, (dq, dk, dv)):
            assert x is None or torch.equal(x, y)


def test_two_long_calls_in_flight(ctx):
    """One after the other without a wait, the same bits as alone: their rows in memory are not each other's."""
    import torch
    q, k, v, do = tensors(1, 260, 20000, 2, 1, 64, 6, positive=False)
    want = run(ctx, q, k, v, do, 0.125)
    lse, outs = torch.empty(1, 2, 260, device="cuda"), [[torch.empty_like(x) for x in (q, q, k, v)] for _ in range(4)]
    for o, *g in outs:
        ctx.attention(d(q), d(k), d(v), d(o), 0.125, lse=d(lse))
        ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in g], 0.125)
    ctx.synchronize()
    for out in outs:
        for x, y in zip(out, want):
            assert torch.equal(x, y)


def test_waits_that_run_out_in_long_sums():
    """The call reports it and the context stays usable."""
    import torch
    torch.cuda.set_device(0)
    c = abi.Context(0)
    q, k, v, do = tensors(1, 260, 20000, 2, 1, 64, 7, positive=False)
    want = run(c, q, k, v, do, 0.125)
    o, lse = torch.empty_like(q), torch.empty(1, 2, 260, device="cuda")
    grads, expired = [torch.empty_like(x) for x in (q, k, v)], 0
    for limit in [1] + [int(1000 * 1.5 ** i) for i in range(16)]:
        c.set_wait_limit(limit)
        c.attention(d(q), d(k), d(v), d(o), 0.125, lse=d(lse))
        c.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in grads], 0.125)
        try:
            c.synchronize()
        except abi.QsmlError as e:
            assert e.status == abi.E_TIMEOUT
            expired += 1
    assert expired
    c.set_wait_limit(0)
    for x, y in zip(run(c, q, k, v, do, 0.125), want):
        assert torch.equal(x, y)
    c.close()


def test_long_sums_in_two_graphs(ctx):
    """Two captured graphs, replayed together with eager calls between, keep the bits: each has rows of its own."""
    import torch
    q, k, v, do = tensors(1, 260, 20000, 2, 1, 64, 8, positive=False)
    want = run(ctx, q, k, v, do, 0.125)
    lse, sets = [torch.empty(1, 2, 260, device="cuda") for _ in range(3)], [[torch.empty_like(x) for x in (q, q, k, v)] for _ in range(3)]

    def call(n):
        o, *g = sets[n]
        ctx.attention(d(q), d(k), d(v), d(o), 0.125, lse=d(lse[n]))
        ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse[n]), d(do), *[d(x) for x in g], 0.125)
    own, graphs, streams = ctx.stream(), [], [torch.cuda.Stream() for _ in range(2)]
    try:
        for n, s in enumerate(streams):
            ctx.set_stream(s.cuda_stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call(n)
            graphs.append(graph)
        ctx.set_stream(own)
        for _ in range(3):
            for t in sum(sets, []):
                t.fill_(NAN)
            torch.cuda.synchronize()
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            call(2)
            torch.cuda.synchronize()
            for out in sets:
                for x, y in zip(out, want):
                    assert torch.equal(x, y)
    finally:
        ctx.set_stream(own)
