"""GPU attention with a window and first tokens, and its backward pass (through the C ABI), against
binary64 with the bounds of attention_reference."""
import numpy as np
import pytest

from attention_reference import Attention, F64, near, visible
from helpers import dev, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
NAN = float("nan")


def d(t):
    return None if t is None else abi.desc_of(t)


class Case:
    """B sequences; nq, nk: their lengths (None: all).  Behind the lengths q, k, v and dout are NaN."""

    def __init__(self, dt, sq, sk, hq, hk, D, window=0, sinks=0, nq=None, nk=None, B=None, scale=None, seed=7, std=1.0):
        self.B = B or (len(nk) if nk is not None else len(nq) if nq is not None else 1)
        self.dt, self.sq, self.sk, self.hq, self.hk, self.D = dt, sq, sk, hq, hk, D
        self.window, self.sinks, self.scale = window, sinks, float(np.float32(scale or D ** -0.5))
        self.q = datagen.normal(seed, (self.B, sq, hq, D), 0, 1.5 * std).astype(dt)
        self.k = datagen.normal(seed + 1, (self.B, sk, hk, D), 0.1, std).astype(dt)
        self.v = datagen.normal(seed + 2, (self.B, sk, hk, D), 0.3, 1).astype(dt)
        self.do = datagen.normal(seed + 3, (self.B, sq, hq, D), 0, 1).astype(dt)
        self.nq, self.nk = nq, nk
        self.lq = [min(max(n, 0), sq) for n in nq] if nq is not None else [sq] * self.B
        self.lk = [min(max(n, 0), sk) for n in nk] if nk is not None else [sk] * self.B
        for b in range(self.B):
            for x, n in ((self.q, self.lq), (self.do, self.lq), (self.k, self.lk), (self.v, self.lk)):
                x[b, n[b]:] = NAN

    def how(self):
        def lengths(n):
            return None if n is None else dev(np.array(n, np.int32))
        self.kept = lengths(self.nq), lengths(self.nk)
        return {"scale": self.scale, "window": self.window, "sinks": self.sinks, "q_lengths": d(self.kept[0]),
                "k_lengths": d(self.kept[1])}

    def heads(self):
        for b in range(self.B):
            seen = visible(self.sq, self.sk, self.lq[b], self.lk[b], self.window, self.sinks)
            for h in range(self.hq):
                g = h // (self.hq // self.hk)
                yield b, h, g, Attention(self.q[b, :, h], self.k[b, :, g], self.v[b, :, g], seen, self.scale, self.dt)

    def forward(self):
        shape = (self.B, self.sq, self.hq, self.D)
        o, eo = np.zeros(shape), np.zeros(shape)
        lse, el = np.zeros((self.B, self.hq, self.sq)), np.zeros((self.B, self.hq, self.sq))
        for b, h, _, a in self.heads():
            o[b, :, h], eo[b, :, h], lse[b, h], el[b, h] = a.forward()
        return o, eo, lse, el

    def backward(self, o, lse):
        out = [np.zeros(self.q.shape), np.zeros(self.k.shape), np.zeros(self.k.shape)]
        err = [np.zeros(x.shape) for x in out]
        for b, h, g, a in self.heads():
            x, e = a.backward(o[b, :, h], lse[b, h], self.do[b, :, h])
            for i, at in enumerate((h, g, g)):
                out[i][b, :, at] += x[i]
                err[i][b, :, at] += e[i]
        return out, err


def run_forward(ctx, c, lse=True):
    import torch
    q, k, v = dev(c.q), dev(c.k), dev(c.v)
    o = torch.full_like(q, NAN)
    s = torch.full((c.B, c.hq, c.sq), NAN, device="cuda") if lse else None
    ctx.attention(d(q), d(k), d(v), d(o), lse=d(s), **c.how())
    ctx.synchronize()
    return host(o), host(s) if lse else None


def check_forward(ctx, c, lse=True):
    o, s = run_forward(ctx, c, lse)
    ro, eo, rl, el = c.forward()
    near(o, ro, eo, "o")
    if lse:
        near(s, rl, el, "lse")


def check_backward(ctx, c):
    import torch
    ro, _, rl, _ = c.forward()
    o, lse = ro.astype(c.dt), rl.astype(np.float32)
    for b in range(c.B):  # not used there
        o[b, c.lq[b]:] = NAN
        lse[b, :, c.lq[b]:] = NAN
    t = [dev(x) for x in (c.q, c.k, c.v, o, lse, c.do)]
    out = [torch.full_like(t[i], NAN) for i in range(3)]
    ctx.attention_backward(*[d(x) for x in t], *[d(x) for x in out], **c.how())
    ctx.synchronize()
    ref, err = c.backward(o, lse)
    for x, r, e, what in zip(out, ref, err, ("dq", "dk", "dv")):
        near(host(x), r, e, what)


DT = pytest.mark.parametrize("dt", [np.float16, np.float32])
SIZES = [  # sq, sk, hq, hk, D, window, sinks
    (1, 1, 1, 1, 64, 0, 0), (70, 70, 2, 1, 64, 0, 0), (128, 128, 1, 1, 128, 0, 0), (129, 129, 2, 2, 128, 0, 0),
    (200, 200, 3, 1, 72, 50, 0), (300, 300, 2, 1, 128, 100, 4), (257, 257, 4, 2, 64, 1, 0), (257, 257, 1, 1, 64, 1, 3),
    (513, 513, 2, 1, 96, 130, 130), (100, 400, 2, 2, 80, 0, 0), (90, 700, 4, 1, 128, 64, 7), (150, 90, 2, 1, 64, 0, 0),
    (200, 130, 1, 1, 128, 33, 2), (640, 640, 1, 1, 128, 0, 0), (333, 333, 2, 1, 40, 77, 1), (65, 65, 3, 3, 8, 0, 0),
    (130, 130, 2, 1, 200, 60, 5), (140, 140, 1, 1, 256, 0, 0), (75, 75, 2, 1, 33, 20, 2), (385, 1000, 1, 1, 128, 500, 0),
    (1000, 1000, 1, 1, 64, 0, 0), (700, 1500, 2, 1, 64, 600, 300), (900, 900, 1, 1, 128, 0, 0), (777, 777, 2, 1, 104, 300, 140),
]


@DT
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(ctx, dt, size):
    check_forward(ctx, Case(dt, *size))


@DT
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_backward(ctx, dt, size):
    check_backward(ctx, Case(dt, *size))


FEW = [(1, 1, 1, 1, 64, 0, 0), (1, 77, 4, 1, 128, 0, 0), (1, 1000, 8, 2, 64, 0, 0), (1, 3001, 6, 2, 128, 500, 4),
       (1, 640, 16, 1, 96, 0, 0), (3, 900, 4, 1, 128, 0, 0), (5, 700, 8, 2, 128, 100, 130), (2, 515, 24, 1, 72, 60, 1),
       (8, 260, 2, 1, 256, 0, 0), (1, 333, 5, 1, 33, 90, 3), (16, 16, 1, 1, 64, 0, 0), (1, 4096, 32, 8, 128, 1024, 4),
       (4, 2, 1, 1, 64, 0, 0), (1, 5000, 1, 1, 200, 0, 0), (13, 1300, 5, 1, 40, 700, 0)]


@DT
@pytest.mark.parametrize("size", FEW, ids=str)
def test_few_queries(ctx, dt, size):
    check_forward(ctx, Case(dt, *size, B=2))


@DT
@pytest.mark.parametrize("size", FEW[:9], ids=str)
def test_few_queries_backward(ctx, dt, size):
    check_backward(ctx, Case(dt, *size))


RAGGED = [  # sq, sk, hq, hk, D, window, sinks, nq, nk
    (200, 200, 2, 1, 64, 0, 0, [200, 0, 1, 127, 130], [200, 0, 1, 127, 130]),
    (300, 300, 2, 2, 128, 90, 3, [300, 290, 129, 128], [300, 290, 129, 128]),
    (150, 500, 3, 1, 72, 0, 0, [150, 100, 3, 150], [500, 333, 260, 150]),
    (150, 260, 2, 1, 128, 40, 2, [150, 100, 150, 7], [260, 60, 0, 6]),     # queries that stand before the first key
    (200, 200, 1, 1, 64, 0, 0, [400, -5, 200], [1 << 30, 100, -(1 << 31)]),  # taken into range
    (130, 130, 1, 1, 64, 10, 0, None, [130, 64, 5]),
    (130, 200, 1, 1, 64, 0, 0, [130, 64, 0], None),
    (1, 700, 8, 2, 128, 0, 0, None, [700, 1, 0, 333, 512]),
    (1, 700, 8, 2, 64, 100, 4, None, [700, 1, 0, 333, 512]),
    (4, 300, 4, 1, 128, 0, 0, [4, 2, 0, 3], [300, 1, 20, 257]),
]


@DT
@pytest.mark.parametrize("size", RAGGED, ids=str)
def test_ragged_forward(ctx, dt, size):
    check_forward(ctx, Case(dt, *size))


@DT
@pytest.mark.parametrize("size", RAGGED, ids=str)
def test_ragged_backward(ctx, dt, size):
    check_backward(ctx, Case(dt, *size))


@DT
def test_scores_of_all_sizes(ctx, dt):
    """Scores up to some hundreds: one key takes all of a row, the others underflow; and nearly equal ones."""
    check_forward(ctx, Case(dt, 200, 200, 1, 1, 64, scale=3.0))
    check_forward(ctx, Case(dt, 1, 900, 4, 1, 64, scale=3.0))
    check_backward(ctx, Case(dt, 200, 200, 1, 1, 64, scale=1.0))
    check_forward(ctx, Case(dt, 300, 300, 1, 1, 128, scale=1e-6))


@DT
def test_maxima_that_grow_with_every_tile(ctx, dt):
    """Keys whose scores rise along the sequence, by more than any reference kept from before covers."""
    c = Case(dt, 300, 700, 1, 1, 64)
    ramp = (np.arange(700) / 100.0)[None, :, None, None]
    c.q[...] = np.abs(c.q)
    c.k[...] = (np.abs(c.k) * ramp).astype(dt)
    check_forward(ctx, c)
    check_backward(ctx, c)
    c.k[...] = c.k[:, ::-1]
    check_forward(ctx, c)


@DT
@pytest.mark.parametrize("gain", [1e-4, 300.0])
def test_small_and_large_gradients(ctx, dt, gain):
    c = Case(dt, 260, 260, 2, 1, 64, 100, 2)
    c.do[...] = (c.do.astype(F64) * gain).astype(dt)
    check_backward(ctx, c)
    c.do[:, ::2] = (c.do[:, ::2].astype(F64) * 1e-3).astype(dt)
    check_backward(ctx, c)


def views(ctx, c, permuted, off):
    """q, k, v as views of larger buffers: [B, heads, tokens, D] permuted, or one packed projection."""
    import torch
    dt = torch.float16 if c.dt == np.float16 else torch.float32
    t = [dev(x) for x in (c.q, c.k, c.v)]
    if permuted:
        return [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in t]
    n = c.hq + 2 * c.hk
    buf = torch.full((c.B, c.sq, n * c.D + 16), NAN, dtype=dt, device="cuda")
    body = buf[:, :, off:off + n * c.D].unflatten(2, (n, c.D))
    out = [body[:, :, :c.hq], body[:, :, c.hq:c.hq + c.hk], body[:, :, c.hq + c.hk:]]
    for x, y in zip(out, t):
        x.copy_(y)
    return out


@DT
@pytest.mark.parametrize("D", [64, 128, 36])
@pytest.mark.parametrize("permuted,off", [(True, 0), (False, 0), (False, 1), (False, 8)])
def test_layouts(ctx, dt, D, permuted, off):
    import torch
    for sq in (1, 150):
        c = Case(dt, sq, sq, 4, 2, D, 60, 2, B=2)
        q, k, v = views(ctx, c, permuted, off)
        o = torch.full((2, 4, sq, D), NAN, dtype=q.dtype, device="cuda").permute(0, 2, 1, 3)
        lse = torch.full((2, 4, sq), NAN, device="cuda")
        ctx.attention(d(q), d(k), d(v), d(o), lse=d(lse), **c.how())
        ctx.synchronize()
        ro, eo, rl, el = c.forward()
        near(host(o.contiguous()), ro, eo, "o")
        near(host(lse), rl, el, "lse")
        # gradients into one packed buffer, dout in [B, heads, tokens, D]
        do = dev(c.do).permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        grad = torch.full((2, sq, 8 * D + 16), 5.0, dtype=q.dtype, device="cuda")
        body = grad[:, :, off:off + 8 * D].unflatten(2, (8, D))
        dq, dk, dv = body[:, :, :4], body[:, :, 4:6], body[:, :, 6:]
        ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), d(dq), d(dk), d(dv), **c.how())
        ctx.synchronize()
        ref, err = c.backward(host(o.contiguous()), host(lse))
        for x, r, e, what in zip((dq, dk, dv), ref, err, ("dq", "dk", "dv")):
            near(host(x.contiguous()), r, e, what)
        beside = torch.cat([grad[:, :, :off], grad[:, :, off + 8 * D:]], 2)
        assert bool((beside == 5.0).all())


@DT
@pytest.mark.parametrize("sq", [1, 3, 140])
def test_keys_shared_by_heads_and_read_backwards(ctx, dt, sq):
    """kv heads of stride 0, and a cache whose tokens lie in descending order."""
    import torch
    c = Case(dt, sq, 140, 4, 2, 64, 50, 2, B=2)
    c.k[:, :, 1], c.v[:, :, 1] = c.k[:, :, 0], c.v[:, :, 0]
    q, do = dev(c.q), dev(c.do)
    ro, eo, rl, el = c.forward()
    k, v = (dev(x[:, :, :1]).expand(2, 140, 2, 64) for x in (c.k, c.v))
    flipped = [dev(np.ascontiguousarray(x[:, ::-1])) for x in (c.k, c.v)]

    def backwards(t):
        view = d(t)
        view.data += 139 * t.stride(1) * t.element_size()
        view.stride[1] = -t.stride(1)
        return view
    for keys, values in ((d(k), d(v)), (backwards(flipped[0]), backwards(flipped[1]))):
        o, lse = torch.full_like(q, NAN), torch.full((2, 4, sq), NAN, device="cuda")
        ctx.attention(d(q), keys, values, d(o), lse=d(lse), **c.how())
        grads = [torch.full_like(q, NAN)] + [torch.full((2, 140, 2, 64), NAN, dtype=q.dtype, device="cuda") for _ in range(2)]
        ctx.attention_backward(d(q), keys, values, d(o), d(lse), d(do), *[d(x) for x in grads], **c.how())
        ctx.synchronize()
        near(host(o), ro, eo, "o")
        near(host(lse), rl, el, "lse")
        ref, err = c.backward(host(o), host(lse))
        for x, r, e, what in zip(grads, ref, err, ("dq", "dk", "dv")):
            near(host(x), r, e, what)


@DT
def test_shared_keys_of_broadcast_sequences(ctx, dt):
    """Sequences that share their keys and values (stride 0): gradients are each sequence's own."""
    import torch
    c = Case(dt, 140, 140, 2, 1, 64, B=3)
    c.k[1:], c.v[1:] = c.k[:1], c.v[:1]
    q = dev(c.q)
    k, v = (dev(x[:1]).expand(3, 140, 1, 64) for x in (c.k, c.v))
    o, lse = torch.empty_like(q), torch.empty(3, 2, 140, device="cuda")
    ctx.attention(d(q), d(k), d(v), d(o), lse=d(lse), **c.how())
    out = [torch.empty_like(q), torch.empty(3, 140, 1, 64, dtype=q.dtype, device="cuda"), torch.empty(3, 140, 1, 64, dtype=q.dtype, device="cuda")]
    do = dev(c.do)
    ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in out], **c.how())
    ctx.synchronize()
    ro, eo, _, _ = c.forward()
    near(host(o), ro, eo, "o")
    ref, err = c.backward(host(o), host(lse))
    for x, r, e in zip(out, ref, err):
        near(host(x), r, e, "gradient")


@DT
def test_no_keys_and_no_queries(ctx, dt):
    import torch
    tdt = torch.float16 if dt == np.float16 else torch.float32
    z = dict(device="cuda", dtype=tdt)
    q, k = torch.ones(2, 3, 2, 64, **z), torch.ones(2, 0, 1, 64, **z)
    o, lse = torch.full((2, 3, 2, 64), NAN, **z), torch.full((2, 2, 3), NAN, device="cuda")
    ctx.attention(d(q), d(k), d(k.clone()), d(o), 0.125, lse=d(lse))
    dq = torch.full_like(q, NAN)
    ctx.attention_backward(d(q), d(k), d(k.clone()), d(o), d(lse), d(q.clone()), d(dq), d(k.clone()), d(k.clone()), 0.125)
    ctx.synchronize()
    assert not host(o).any() and np.isneginf(host(lse)).all() and not host(dq).any()
    q, k = torch.ones(2, 0, 2, 64, **z), torch.ones(2, 5, 1, 64, **z)
    e = torch.empty(2, 2, 0, device="cuda")
    ctx.attention(d(q), d(k), d(k.clone()), d(q.clone()), 0.125, lse=d(e))
    dk, dv = torch.full_like(k, NAN), torch.full_like(k, NAN)
    ctx.attention_backward(d(q), d(k), d(k.clone()), d(q.clone()), d(e), d(q.clone()), d(q.clone()), d(dk), d(dv), 0.125)
    ctx.synchronize()
    assert not host(dk).any() and not host(dv).any()


@DT
def test_gradients_left_out(ctx, dt):
    import torch
    c = Case(dt, 150, 150, 2, 1, 64)
    ro, _, rl, _ = c.forward()
    o, lse = ro.astype(dt), rl.astype(np.float32)
    t = [dev(x) for x in (c.q, c.k, c.v, o, lse, c.do)]
    ref, err = c.backward(o, lse)
    for want in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (0, 0, 0)):
        out = [torch.full_like(t[i], NAN) if w else None for i, w in enumerate(want)]
        ctx.attention_backward(*[d(x) for x in t], *[d(x) for x in out], **c.how())
        ctx.synchronize()
        for x, r, e in zip(out, ref, err):
            if x is not None:
                near(host(x), r, e, str(want))


@DT
@pytest.mark.parametrize("size", [(1, 1, 4, 2, 64, 0, 0), (1, 1, 2, 1, 128, 0, 0), (200, 200, 2, 1, 64, 1, 0), (140, 260, 2, 2, 128, 1, 0),
                                  (3, 3, 1, 1, 33, 1, 0)], ids=str)
def test_a_row_of_one_key_has_no_gradient_but_its_value(ctx, dt, size):
    """With one key its weight is 1 whatever the score: dq and dk are 0, dv is the sum of the group's dout."""
    import torch
    c = Case(dt, *size, B=2)
    ro, _, rl, _ = c.forward()
    t = [dev(x) for x in (c.q, c.k, c.v, ro.astype(dt), rl.astype(np.float32), c.do)]
    out = [torch.full_like(t[i], NAN) for i in range(3)]
    ctx.attention_backward(*[d(x) for x in t], *[d(x) for x in out], **c.how())
    ctx.synchronize()
    assert not host(out[0]).any() and not host(out[1]).any()
    want = np.zeros(c.v.shape)
    want[:, c.sk - c.sq:] = c.do.astype(F64).reshape(2, c.sq, c.hk, c.hq // c.hk, c.D).sum(3)
    size = np.abs(c.do.astype(F64)).max() * (c.hq // c.hk)
    # the weight is off by 2^-11 in F16, and by the scores' rounding against lse's
    near(host(out[2]), want, size * ((2.0 ** -11 if dt == np.float16 else 0) + 400 * 2.0 ** -24), "dv")


@DT
def test_gradients_against_differences(ctx, dt):
    """sum(o * dout) along a direction: the binary64 forward pass's central difference against the
    gradients' product with that direction, whose rounding is that of F16's P and dS (2^-11 each of
    gradients of this size) or of binary32."""
    import torch
    c = Case(dt, 90, 90, 2, 1, 32, 30, 2)
    ro, _, rl, _ = c.forward()
    t = [dev(x) for x in (c.q, c.k, c.v, ro.astype(dt), rl.astype(np.float32), c.do)]
    out = [torch.empty_like(t[i]) for i in range(3)]
    ctx.attention_backward(*[d(x) for x in t], *[d(x) for x in out], **c.how())
    ctx.synchronize()
    rng = np.random.RandomState(1)
    way = [rng.randn(*x.shape) for x in (c.q, c.k, c.v)]
    base = [x.astype(F64) for x in (c.q, c.k, c.v)]

    def total(h):
        c.q, c.k, c.v = (x + h * w for x, w in zip(base, way))
        return (c.forward()[0] * c.do.astype(F64)).sum()
    h = 1e-4
    diff = (total(h) - total(-h)) / (2 * h)
    got = sum((host(x).astype(F64) * w).sum() for x, w in zip(out, way))
    size = sum((np.abs(host(x).astype(F64)) * np.abs(w)).sum() for x, w in zip(out, way))
    assert abs(got - diff) <= (2.0 ** -9 if dt == np.float16 else 2.0 ** -16) * size + 1e-5 * abs(diff)


@DT
@pytest.mark.parametrize("sq,sk", [(1, 1500), (260, 260)])
def test_the_same_bits_at_every_call_and_in_graphs(ctx, dt, sq, sk):
    """Two captured graphs of one context, replayed together on two streams, and eager calls in between."""
    import torch
    c = Case(dt, sq, sk, 4, 2, 64, 200, 3, nk=[sk, sk - 20])
    q, k, v, do = dev(c.q), dev(c.k), dev(c.v), dev(c.do)
    how = c.how()

    def outputs():
        return [torch.zeros_like(q), torch.zeros(2, 4, sq, device="cuda"), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]

    def call(o):
        ctx.attention(d(q), d(k), d(v), d(o[0]), lse=d(o[1]), **how)
        ctx.attention_backward(d(q), d(k), d(v), d(o[0]), d(o[1]), d(do), d(o[2]), d(o[3]), d(o[4]), **how)
    first, again, sets = outputs(), outputs(), [outputs(), outputs()]
    call(first)
    call(again)
    ctx.synchronize()
    own, graphs, streams = ctx.stream(), [], [torch.cuda.Stream() for _ in range(2)]
    try:
        for o, s in zip(sets, streams):
            ctx.set_stream(s.cuda_stream)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                call(o)
            graphs.append(graph)
        ctx.set_stream(own)
        for _ in range(3):
            for o in sets:
                for t in o:
                    t.zero_()
            torch.cuda.synchronize()
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            call(again)
            torch.cuda.synchronize()
            for o in sets + [again]:
                for a, b in zip(first, o):
                    assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    finally:
        ctx.set_stream(own)


@DT
@pytest.mark.parametrize("sq,sk,D", [(200, 200, 64), (200, 200, 128), (5, 300, 64), (90, 90, 36)])
def test_what_is_no_number_stays_with_the_rows_that_see_it(ctx, dt, sq, sk, D):
    """A query of NaN is NaN in its row alone, a key of NaN in the rows that see it; the others keep their bits."""
    c = Case(dt, sq, sk, 2, 1, D, 50, 2)
    clean, lse = run_forward(ctx, c)
    row, key = sq // 2, sk - sq // 2
    c.q[0, row, 0] = NAN
    o, s = run_forward(ctx, c)
    hit = np.zeros((1, sq, 2), bool)
    hit[0, row, 0] = True
    assert np.isnan(o[hit]).all() and np.array_equal(o[~hit], clean[~hit])
    assert np.array_equal(np.isnan(s), hit.transpose(0, 2, 1))
    c = Case(dt, sq, sk, 2, 1, D, 50, 2)
    c.k[0, key] = NAN
    o, s = run_forward(ctx, c)
    sees = visible(sq, sk, sq, sk, 50, 2)[:, key]
    assert sees.any() and not sees.all()
    assert np.isnan(o[0, sees]).all() and np.array_equal(o[0, ~sees], clean[0, ~sees])
    assert np.array_equal(s[0][:, ~sees], lse[0][:, ~sees])


def test_two_contexts_at_once():
    """Two contexts on streams of their own, in flight together, give what each gives alone."""
    import torch
    torch.cuda.set_device(0)
    ctxs, streams = [abi.Context(0), abi.Context(0)], [torch.cuda.Stream(), torch.cuda.Stream()]
    work, want = [], []
    for n, (c, s) in enumerate(zip(ctxs, streams)):
        case = Case(np.float16, 700 + 60 * n, 700 + 60 * n, 4, 2, 128 if n else 64, 300, 5, B=2, seed=30 + n)
        t = [dev(x) for x in (case.q, case.k, case.v, case.do)]
        out = [torch.zeros_like(t[0]), torch.zeros(2, 4, case.sq, device="cuda")] + [torch.zeros_like(t[i]) for i in range(3)]
        token = torch.zeros_like(t[0][:, :1])
        how = case.how()

        def call(ctx=c, t=t, out=out, token=token, how=how):
            ctx.attention(d(t[0]), d(t[1]), d(t[2]), d(out[0]), lse=d(out[1]), **how)
            ctx.attention_backward(*[d(x) for x in (t[0], t[1], t[2], out[0], out[1], t[3], out[2], out[3], out[4])], **how)
            ctx.attention(d(t[0][:, -1:]), d(t[1]), d(t[2]), d(token), **how)
        torch.cuda.synchronize()
        c.set_stream(s.cuda_stream)
        call()
        c.synchronize()
        want.append([host(x) for x in out + [token]])
        for x in out + [token]:
            x.zero_()
        work.append((call, out + [token], case))
    torch.cuda.synchronize()
    for _ in range(10):
        for call, _, _ in work:
            call()
    for c, (_, out, _), w in zip(ctxs, work, want):
        c.synchronize()
        for x, y in zip(out, w):
            assert np.array_equal(host(x), y)
    for c in ctxs:
        c.close()


def test_offsets_beyond_2_to_the_31(ctx):
    """A cache whose second sequence starts past 2^31 elements, read in place."""
    import torch
    c = Case(np.float16, 1, 300, 2, 1, 64, B=2)
    step = (1 << 31) + 64 * 8
    buf = torch.zeros(step + 300 * 64, dtype=torch.float16, device="cuda")
    k = buf.as_strided((2, 300, 1, 64), (step, 64, 64, 1))
    k.copy_(dev(c.k))
    v, q = dev(c.v), dev(c.q)
    o = torch.empty_like(q)
    ctx.attention(d(q), d(k), d(v), d(o), **c.how())
    ctx.synchronize()
    ro, eo, _, _ = c.forward()
    near(host(o), ro, eo, "o")
    c = Case(np.float16, 160, 160, 1, 1, 64, B=2)
    k = buf.as_strided((2, 160, 1, 64), (step, 64, 64, 1))
    k.copy_(dev(c.k))
    v, q = dev(c.v), dev(c.q)
    o = torch.empty_like(q)
    ctx.attention(d(q), d(k), d(v), d(o), **c.how())
    ctx.synchronize()
    ro, eo, _, _ = c.forward()
    near(host(o), ro, eo, "o")


def refused(ctx, status, call, *args, **how):
    before = ctx.launch_count()
    with pytest.raises(abi.QsmlError) as e:
        call(*args, **how)
    assert e.value.status == status, e.value
    assert ctx.launch_count() == before


def test_refusals(ctx):
    import torch
    z = dict(device="cuda", dtype=torch.float16)
    good = {"q": torch.zeros(2, 5, 4, 64, **z), "k": torch.zeros(2, 7, 2, 64, **z), "v": torch.zeros(2, 7, 2, 64, **z),
            "o": torch.zeros(2, 5, 4, 64, **z)}
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    lse = torch.zeros(2, 4, 5, device="cuda")

    def no(status, scale=0.125, **change):
        how = {x: change.pop(x) for x in ("window", "sinks", "q_lengths", "k_lengths", "lse") if x in change}
        how = {x: d(y) if isinstance(y, torch.Tensor) else y for x, y in how.items()}
        refused(ctx, status, ctx.attention, *[d(t) for t in {**good, **change}.values()], scale, **how)
    E = abi
    no(E.E_DTYPE, q=good["q"].to(torch.int32))
    no(E.E_DTYPE, k=good["k"].float())
    no(E.E_DTYPE, o=good["o"].float())
    no(E.E_DTYPE, q_lengths=n.long().to(torch.int16))
    no(E.E_DTYPE, lse=lse.half())
    no(E.E_SHAPE, q=good["q"][0])
    no(E.E_SHAPE, q=good["q"][:, :, :3], o=good["o"][:, :, :3])
    no(E.E_SHAPE, q=good["q"][..., :32], o=good["o"][..., :32])
    no(E.E_SHAPE, k=good["k"][:1])
    no(E.E_SHAPE, v=good["v"][:, :6])
    no(E.E_SHAPE, o=good["o"][:, :4])
    no(E.E_SHAPE, k_lengths=n[:1])
    no(E.E_SHAPE, lse=lse[:, :, :4])
    no(E.E_SHAPE, lse=lse.permute(0, 2, 1))
    no(E.E_INVALID, scale=0.0)
    no(E.E_INVALID, scale=-1.0)
    no(E.E_INVALID, scale=float("inf"))
    no(E.E_INVALID, scale=NAN)
    no(E.E_INVALID, window=-1)
    no(E.E_INVALID, sinks=-1)
    no(E.E_INVALID, o=good["q"])
    no(E.E_UNSUPPORTED, q=torch.zeros(2, 5, 4, 128, **z)[..., ::2])
    no(E.E_UNSUPPORTED, o=torch.zeros(2, 1, 4, 64, **z).expand(2, 5, 4, 64))
    big = torch.zeros(1, 1, 1, 257, **z)
    no(E.E_UNSUPPORTED, q=big, k=big.clone(), v=big.clone(), o=big.clone())
    g = {**good, "lse": lse, "do": torch.zeros(2, 5, 4, 64, **z), "dq": torch.zeros(2, 5, 4, 64, **z),
         "dk": torch.zeros(2, 7, 2, 64, **z), "dv": torch.zeros(2, 7, 2, 64, **z)}

    def nob(status, scale=0.125, **change):
        refused(ctx, status, ctx.attention_backward, *[d(t) for t in {**g, **change}.values()], scale)
    nob(E.E_DTYPE, do=g["do"].float())
    nob(E.E_DTYPE, lse=lse.half())
    nob(E.E_DTYPE, dk=g["dk"].float())
    nob(E.E_SHAPE, dv=g["dv"][:, :6])
    nob(E.E_SHAPE, do=g["do"][:, :4])
    nob(E.E_INVALID, dq=g["do"])
    nob(E.E_INVALID, dk=g["dv"])
    nob(E.E_INVALID, scale=0.0)
