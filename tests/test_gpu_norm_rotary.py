"""GPU norm and rotation of heads, and the backward pass (through the C ABI), against binary64 with
the bounds of attention_reference."""
import numpy as np
import pytest

from attention_reference import angles, near, rotary, rotary_backward
from helpers import dev, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
PAIRING = {False: abi.ROTARY_HALVES, True: abi.ROTARY_PAIRS}


def d(t):
    return None if t is None else abi.desc_of(t)


def frequencies(n):
    return (10000.0 ** (-np.arange(n) / n)).astype(np.float32)


class Case:
    def __init__(self, tokens, hq, hk, D, rot, dt, sections=None, pairs=False, wdt=np.float32, norm=(True, True), far=0,
                 seed=5):
        self.q = datagen.normal(seed, (tokens, hq, D), 0.2, 1.3).astype(dt)
        self.k = datagen.normal(seed + 1, (tokens, hk, D), -0.1, 0.8).astype(dt)
        self.gq = datagen.normal(seed + 2, (tokens, hq, D), 0, 1).astype(dt)
        self.gk = datagen.normal(seed + 3, (tokens, hk, D), 0, 1).astype(dt)
        self.wq = datagen.normal(seed + 4, (D,), 1, 0.2).astype(wdt) if norm[0] else None
        self.wk = datagen.normal(seed + 5, (D,), 1, 0.2).astype(wdt) if norm[1] else None
        rng = np.random.RandomState(seed)
        shape = (tokens,) if sections is None else (tokens, len(sections))
        self.pos = (rng.randint(0, 5000, shape) + far).astype(np.int32)
        self.freq, self.sections, self.pairs, self.eps = frequencies(rot // 2), sections, pairs, 1e-6
        self.t = angles(self.pos, self.freq, sections)

    def how(self):
        return {"eps": self.eps, "sections": self.sections, "pairing": PAIRING[self.pairs]}

    def device(self):
        return [None if x is None else dev(x) for x in (self.q, self.k, self.wq, self.wk, self.pos, self.freq)]


def check(ctx, c):
    import torch
    inputs = c.device()
    out = [torch.full_like(inputs[0], float("nan")), torch.full_like(inputs[1], float("nan"))]
    ctx.norm_rotary(*[d(x) for x in inputs], *[d(x) for x in out], **c.how())
    ctx.synchronize()
    for x, w, y, what in ((c.q, c.wq, out[0], "q"), (c.k, c.wk, out[1], "k")):
        near(host(y), *rotary(x, w, c.eps, c.t, c.pairs), what)
    gq, gk = dev(c.gq), dev(c.gk)
    grads = [torch.full_like(inputs[0], float("nan")), torch.full_like(inputs[1], float("nan"))]
    dw = [None if w is None else torch.full(w.shape, float("nan"), device="cuda") for w in inputs[2:4]]
    ctx.norm_rotary_backward(*[d(x) for x in inputs], d(gq), d(gk), d(grads[0]), d(grads[1]), d(dw[0]), d(dw[1]), **c.how())
    ctx.synchronize()
    for x, w, g, dx, dww, what in ((c.q, c.wq, c.gq, grads[0], dw[0], "dq"), (c.k, c.wk, c.gk, grads[1], dw[1], "dk")):
        ref, err, refw, errw = rotary_backward(x, w, c.eps, c.t, c.pairs, g)
        near(host(dx), ref, err, what)
        if w is not None:
            near(host(dww), refw, errw, what + "'s weight")


@pytest.mark.parametrize("dt", [np.float16, np.float32])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,D,rot", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (7, 3, 1, 64, 64), (33, 4, 4, 80, 80),
                                                (5, 6, 2, 100, 50), (19, 2, 1, 72, 72), (3, 5, 5, 256, 128), (2, 2, 1, 512, 512),
                                                (9, 3, 2, 38, 38), (4, 1, 2, 510, 254), (3, 2, 2, 384, 384), (211, 8, 2, 128, 64)])
def test_forward_and_backward(ctx, dt, pairs, tokens, hq, hk, D, rot):
    check(ctx, Case(tokens, hq, hk, D, rot, dt, pairs=pairs))


@pytest.mark.parametrize("dt", [np.float16, np.float32])
@pytest.mark.parametrize("sections", [(32,), (8, 12, 12), (0, 16, 0, 16), (1, 30, 1)])
def test_axes(ctx, dt, sections):
    check(ctx, Case(23, 3, 1, 64, 64, dt, sections=list(sections), pairs=len(sections) == 3))


@pytest.mark.parametrize("norm", [(True, False), (False, True), (False, False)])
def test_without_norms(ctx, norm):
    check(ctx, Case(17, 5, 3, 64, 64, np.float16, norm=norm))


def test_half_precision_weights(ctx):
    check(ctx, Case(17, 5, 3, 64, 32, np.float16, wdt=np.float16))


@pytest.mark.parametrize("far", [-3000, 1000000, 2 ** 31 - 6000])
def test_far_positions(ctx, far):
    check(ctx, Case(40, 2, 1, 64, 64, np.float32, far=far))


def test_many_tokens_share_the_device(ctx):
    check(ctx, Case(5003, 4, 2, 32, 32, np.float16))


def test_rows_of_zeros_and_of_huge_numbers(ctx):
    c = Case(6, 2, 1, 32, 32, np.float32)
    c.q[2] = 0.0
    c.q[3] *= np.float32(1e15)
    c.k[1] *= np.float32(1e-12)
    check(ctx, c)


@pytest.mark.parametrize("off", [0, 1])
def test_slices_of_one_projection_in_and_out(ctx, off):
    """q and k out of a packed projection (starting off 16 bytes with off = 1), into a packed buffer, and in place."""
    import torch
    c = Case(2 * 21, 4, 2, 64, 64, np.float16)
    wide = 8 * 64 + 8

    def packed():
        buf = torch.zeros(2, 21, wide, dtype=torch.float16, device="cuda")
        body = buf[:, :, off:off + 8 * 64].unflatten(2, (8, 64))
        return buf, body[:, :, :4], body[:, :, 4:6]
    buf, q, k = packed()
    q.copy_(dev(c.q).view(2, 21, 4, 64)), k.copy_(dev(c.k).view(2, 21, 2, 64))
    pos, freq, wq, wk = dev(c.pos.reshape(2, 21)), dev(c.freq), dev(c.wq), dev(c.wk)
    ref = [rotary(c.q, c.wq, c.eps, c.t, False), rotary(c.k, c.wk, c.eps, c.t, False)]
    to, tq, tk = packed()
    ctx.norm_rotary(d(q), d(k), d(wq), d(wk), d(pos), d(freq), d(tq), d(tk), **c.how())
    ctx.norm_rotary(d(q), d(k), d(wq), d(wk), d(pos), d(freq), d(q), d(k), **c.how())
    ctx.synchronize()
    for out in ((tq, tk), (q, k)):
        for y, (r, e) in zip(out, ref):
            near(host(y.contiguous()).reshape(r.shape), r, e, "packed")
    # nothing beside the heads is written
    assert not host(to[:, :, off + 6 * 64:]).any() and not host(to[:, :, :off]).any()
    gq, gk = dev(c.gq).view(2, 21, 4, 64).clone(), dev(c.gk).view(2, 21, 2, 64).clone()
    q.copy_(dev(c.q).view(2, 21, 4, 64)), k.copy_(dev(c.k).view(2, 21, 2, 64))
    grad, dq, dk = packed()
    dwq, dwk = torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
    ctx.norm_rotary_backward(d(q), d(k), d(wq), d(wk), d(pos), d(freq), d(gq), d(gk), d(dq), d(dk), d(dwq), d(dwk), **c.how())
    ctx.norm_rotary_backward(d(q), d(k), d(wq), d(wk), d(pos), d(freq), d(gq), d(gk), d(gq), d(gk), **c.how())
    ctx.synchronize()
    for out in ((dq, dk), (gq, gk)):
        for y, x, w, g in zip(out, (c.q, c.k), (c.wq, c.wk), (c.gq, c.gk)):
            r, e, _, _ = rotary_backward(x, w, c.eps, c.t, False, g)
            near(host(y.contiguous()).reshape(r.shape), r, e, "packed gradient")


def test_broadcast_heads_and_reversed_tokens(ctx):
    import torch
    c = Case(12, 3, 1, 32, 32, np.float32)
    c.q[:] = c.q[:, :1]
    q = dev(c.q)[:, :1].expand(12, 3, 32)
    rev = dev(c.k[::-1].copy())
    view = abi.desc_of(rev)
    view.data += 11 * 32 * 4
    view.stride[0] = -32
    out = [torch.empty(12, 3, 32, device="cuda"), torch.empty(12, 1, 32, device="cuda")]
    x = c.device()
    ctx.norm_rotary(d(q), view, d(x[2]), d(x[3]), d(x[4]), d(x[5]), d(out[0]), d(out[1]), **c.how())
    ctx.synchronize()
    near(host(out[0]), *rotary(c.q, c.wq, c.eps, c.t, False), "q")
    near(host(out[1]), *rotary(c.k, c.wk, c.eps, c.t, False), "k")


def test_keys_alone_absent_and_gradients_left_out(ctx):
    import torch
    c = Case(9, 3, 2, 64, 64, np.float16)
    x = c.device()
    out = torch.empty_like(x[0])
    ctx.norm_rotary(d(x[0]), None, d(x[2]), None, d(x[4]), d(x[5]), d(out), None, **c.how())
    gq, gk, dk, dwk = dev(c.gq), dev(c.gk), torch.empty_like(x[1]), torch.empty(64, device="cuda")
    ctx.norm_rotary_backward(*[d(t) for t in x], d(gq), d(gk), None, d(dk), None, d(dwk), **c.how())
    only = torch.empty(64, device="cuda", dtype=torch.float16)
    ctx.norm_rotary_backward(*[d(t) for t in x], d(gq), d(gk), None, None, d(only), None, **c.how())
    ctx.norm_rotary_backward(*[d(t) for t in x], d(gq), d(gk), None, None, None, None, **c.how())
    ctx.synchronize()
    near(host(out), *rotary(c.q, c.wq, c.eps, c.t, False), "q alone")
    ref, err, refw, errw = rotary_backward(c.k, c.wk, c.eps, c.t, False, c.gk)
    near(host(dk), ref, err, "dk alone")
    near(host(dwk), refw, errw, "dwk alone")
    _, _, refw, errw = rotary_backward(c.q, c.wq, c.eps, c.t, False, c.gq)
    near(host(only), refw, errw, "dwq alone, in F16")


def test_no_tokens(ctx):
    import torch
    q, pos = torch.empty(0, 2, 8, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    w, f, dw = torch.ones(8, device="cuda"), torch.ones(4, device="cuda"), torch.full((8,), 3.0, device="cuda")
    ctx.norm_rotary(d(q), None, d(w), None, d(pos), d(f), d(q.clone()), None)
    ctx.norm_rotary_backward(d(q), None, d(w), None, d(pos), d(f), d(q.clone()), None, d(q.clone()), None, d(dw))
    ctx.synchronize()
    assert not host(dw).any()


def test_gradients_against_differences(ctx):
    """The sum of the outputs times fixed weights, along a direction: its binary64 central difference
    (error h^2 of the third derivative: 1e-7) against the gradients' product with that direction."""
    import torch
    c = Case(11, 3, 2, 32, 32, np.float32, sections=[8, 4, 4])
    x = c.device()
    gq, gk = dev(c.gq), dev(c.gk)
    out = [torch.empty_like(x[0]), torch.empty_like(x[1]), torch.empty(32, device="cuda"), torch.empty(32, device="cuda")]
    ctx.norm_rotary_backward(*[d(t) for t in x], d(gq), d(gk), *[d(t) for t in out], **c.how())
    ctx.synchronize()
    rng = np.random.RandomState(2)
    way = [rng.randn(*np.shape(host(t))) for t in out]
    size = sum((np.abs(host(t).astype(np.float64)) * np.abs(w)).sum() for t, w in zip(out, way))

    def total(h):
        q, k = c.q.astype(np.float64) + h * way[0], c.k.astype(np.float64) + h * way[1]
        a = rotary(q, c.wq + h * way[2], c.eps, c.t, False)[0]
        b = rotary(k, c.wk + h * way[3], c.eps, c.t, False)[0]
        return (a * c.gq).sum() + (b * c.gk).sum()
    h = 1e-4
    diff = (total(h) - total(-h)) / (2 * h)
    got = sum((host(t).astype(np.float64) * w).sum() for t, w in zip(out, way))
    # binary32 gradients: rounded, and off by what rotary_backward bounds (below 2^-16 of their size)
    assert abs(diff - got) <= size * 2.0 ** -16 + 1e-6 * abs(diff)


def test_the_same_bits_at_every_call_and_in_a_graph(ctx):
    import torch
    c = Case(700, 6, 2, 64, 64, np.float16)
    x = c.device()
    gq, gk = dev(c.gq), dev(c.gk)

    def outputs():
        return [torch.zeros_like(x[0]), torch.zeros_like(x[1]), torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")]
    first, second = outputs(), outputs()

    def call(o):
        ctx.norm_rotary_backward(*[d(t) for t in x], d(gq), d(gk), *[d(t) for t in o], **c.how())
    call(first)
    ctx.synchronize()
    own, s = ctx.stream(), torch.cuda.Stream()
    ctx.set_stream(s.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call(second)
        for _ in range(3):
            for t in second:
                t.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(first, second):
                assert torch.equal(a, b)
    finally:
        ctx.set_stream(own)


def refused(ctx, status, call, *args, **how):
    before = ctx.launch_count()
    with pytest.raises(abi.QsmlError) as e:
        call(*args, **how)
    assert e.value.status == status, e.value
    assert ctx.launch_count() == before


def test_refusals(ctx):
    import torch
    z = dict(device="cuda")
    q, k = torch.zeros(4, 3, 8, **z), torch.zeros(4, 1, 8, **z)
    w, pos, f = torch.ones(8, **z), torch.zeros(4, dtype=torch.int32, **z), torch.ones(4, **z)
    oq, ok = torch.zeros(4, 3, 8, **z), torch.zeros(4, 1, 8, **z)

    def no(status, **change):
        a = {"q": q, "k": k, "wq": w, "wk": w, "pos": pos, "f": f, "oq": oq, "ok": ok}
        how = {x: change.pop(x) for x in ("eps", "sections", "pairing") if x in change}
        a.update(change)
        refused(ctx, status, ctx.norm_rotary, *[None if t is None else d(t) for t in a.values()], **how)
    E = abi
    no(E.E_DTYPE, q=q.to(torch.int32))
    no(E.E_DTYPE, k=k.half())
    no(E.E_DTYPE, wq=w.half())
    no(E.E_DTYPE, pos=pos.float())
    no(E.E_DTYPE, f=f.half())
    no(E.E_DTYPE, oq=oq.half())
    no(E.E_SHAPE, q=q[0])
    no(E.E_SHAPE, k=k[:3])
    no(E.E_SHAPE, wq=w[:7])
    no(E.E_SHAPE, pos=pos[:3])
    no(E.E_SHAPE, pos=pos[:, None].expand(4, 2))
    no(E.E_SHAPE, f=torch.ones(5, **z))
    no(E.E_SHAPE, f=torch.ones(0, **z))
    no(E.E_SHAPE, oq=oq[:, :2])
    no(E.E_SHAPE, pos=torch.zeros(4, 2, dtype=torch.int32, **z), sections=[1, 1])
    no(E.E_SHAPE, sections=[2, 2])
    no(E.E_SHAPE, q=torch.zeros(4, 3, 7, **z), k=None, wk=None, wq=None, oq=torch.zeros(4, 3, 7, **z), ok=None, f=f[:3])
    no(E.E_INVALID, pos=torch.zeros(4, 5, dtype=torch.int32, **z), sections=[1, 1, 1, 1, 0])
    no(E.E_INVALID, pos=torch.zeros(4, 2, dtype=torch.int32, **z), sections=[5, -1])
    no(E.E_INVALID, pairing=2)
    no(E.E_INVALID, eps=-1.0)
    no(E.E_INVALID, eps=float("nan"))
    no(E.E_INVALID, ok=None)
    no(E.E_INVALID, k=None)
    no(E.E_INVALID, k=None, ok=None)  # wk without k
    no(E.E_UNSUPPORTED, q=torch.zeros(4, 3, 16, **z)[..., ::2])
    no(E.E_UNSUPPORTED, oq=torch.zeros(4, 1, 8, **z).expand(4, 3, 8))
    no(E.E_UNSUPPORTED, q=torch.zeros(1, 1, 514, **z), k=None, wq=None, wk=None, pos=pos[:1], oq=torch.zeros(1, 1, 514, **z), ok=None)
    buf = torch.zeros(4, 6, 8, **z)
    no(E.E_INVALID, q=buf[:, :3], oq=buf[:, 1:4])
    no(E.E_INVALID, oq=buf[:, :3], ok=buf[:, 2:3])
    no(E.E_INVALID, k=buf[:, 2:3], oq=buf[:, :3])
    g, dw = torch.zeros(4, 3, 8, **z), torch.zeros(8, **z)

    def nob(status, **change):
        a = {"q": q, "k": None, "wq": w, "wk": None, "pos": pos, "f": f, "gq": g, "gk": None, "dq": oq, "dk": None, "dwq": dw, "dwk": None}
        a.update(change)
        refused(ctx, status, ctx.norm_rotary_backward, *[None if t is None else d(t) for t in a.values()])
    nob(E.E_INVALID, wq=None)
    nob(E.E_INVALID, k=k)
    nob(E.E_INVALID, dk=ok)
    nob(E.E_INVALID, dq=q)
    nob(E.E_SHAPE, gq=g[:, :2])
    nob(E.E_SHAPE, dwq=dw[:4])
    nob(E.E_DTYPE, dwq=dw.to(torch.int32))
