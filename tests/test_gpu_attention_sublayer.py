"""The attention sublayer as a program runs it: one projection, norms and rotation of its heads in place,
attention over slices of it, the output projection with its residual; its gradients back to the input, all
heads' gradients in one buffer that linear_backward reads; and the same tokens one by one over a cache."""
import numpy as np
import pytest

from attention_reference import F64, U, Attention, angles, rotary, visible
from helpers import dev, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
B, T, C, HQ, HK, D = 2, 150, 96, 4, 2, 32
WINDOW, SINKS, EPS = 40, 3, 1e-6
HEADS = HQ + 2 * HK


def d(t):
    return None if t is None else abi.desc_of(t)


class Layer:
    def __init__(self, dt):
        s = C ** -0.5
        self.dt = dt
        self.x = datagen.normal(21, (B, T, C), 0, 1).astype(dt)
        self.w = datagen.normal(22, (C, HEADS * D), 0, s).astype(dt)
        self.wo = datagen.normal(23, (HQ * D, C), 0, (HQ * D) ** -0.5).astype(dt)
        self.wq, self.wk = (datagen.normal(24 + i, (D,), 1, 0.2).astype(np.float32) for i in range(2))
        self.dy = datagen.normal(26, (B, T, C), 0, 1).astype(dt)
        self.freq = (10000.0 ** (-np.arange(D // 2) / (D // 2))).astype(np.float32)
        self.pos = np.tile(np.arange(T, dtype=np.int32), (B, 1))
        self.scale = float(np.float32(D ** -0.5))

    def exact(self, x, w=None):
        """y in binary64."""
        qkv = (x @ (self.w.astype(F64) if w is None else w)).reshape(B * T, HEADS, D)
        t = angles(self.pos.reshape(-1), self.freq, None)
        q = rotary(qkv[:, :HQ], self.wq, EPS, t, False)[0].reshape(B, T, HQ, D)
        k = rotary(qkv[:, HQ:HQ + HK], self.wk, EPS, t, False)[0].reshape(B, T, HK, D)
        v = qkv[:, HQ + HK:].reshape(B, T, HK, D)
        seen = visible(T, T, T, T, WINDOW, SINKS)
        o = np.stack([np.stack([Attention(q[b, :, h], k[b, :, h // 2], v[b, :, h // 2], seen, self.scale, F64).forward()[0]
                                for h in range(HQ)], 1) for b in range(B)])
        return x + o.reshape(B, T, HQ * D) @ self.wo.astype(F64)


def forward(ctx, c, keep):
    import torch
    x, w, wo = dev(c.x), dev(c.w), dev(c.wo)
    qkv = torch.empty(B, T, HEADS * D, dtype=x.dtype, device="cuda")
    ctx.linear(d(x), d(w), None, abi.ACT_NONE, None, None, d(qkv))
    keep["qkv"] = qkv.clone()
    heads = qkv.view(B, T, HEADS, D)
    q, k, v = heads[:, :, :HQ], heads[:, :, HQ:HQ + HK], heads[:, :, HQ + HK:]
    side = {n: dev(getattr(c, n)) for n in ("wq", "wk", "pos", "freq")}
    ctx.norm_rotary(d(q), d(k), d(side["wq"]), d(side["wk"]), d(side["pos"]), d(side["freq"]), d(q), d(k), eps=EPS)
    o, lse = torch.empty(B, T, HQ, D, dtype=x.dtype, device="cuda"), torch.empty(B, HQ, T, device="cuda")
    ctx.attention(d(q), d(k), d(v), d(o), c.scale, window=WINDOW, sinks=SINKS, lse=d(lse))
    y = torch.empty_like(x)
    ctx.linear(d(o.view(B, T, HQ * D)), d(wo), None, abi.ACT_NONE, d(x), None, d(y))
    keep.update(x=x, w=w, wo=wo, q=q, k=k, v=v, o=o, lse=lse, y=y, **side)
    return y


def backward(ctx, c, s):
    import torch
    dy, do = dev(c.dy), torch.empty(B, T, HQ * D, dtype=s["x"].dtype, device="cuda")
    dwo, dw, dx = torch.empty_like(s["wo"]), torch.empty_like(s["w"]), torch.empty_like(s["x"])
    ctx.linear_backward(d(s["o"].view(B, T, HQ * D)), d(s["wo"]), abi.ACT_NONE, None, d(dy), d(do), d(dwo))
    dqkv = torch.empty(B, T, HEADS, D, dtype=s["x"].dtype, device="cuda")
    dq, dk, dv = dqkv[:, :, :HQ], dqkv[:, :, HQ:HQ + HK], dqkv[:, :, HQ + HK:]
    ctx.attention_backward(d(s["q"]), d(s["k"]), d(s["v"]), d(s["o"]), d(s["lse"]), d(do.view(B, T, HQ, D)), d(dq), d(dk),
                           d(dv), c.scale, window=WINDOW, sinks=SINKS)
    raw = s["qkv"].view(B, T, HEADS, D)
    ctx.norm_rotary_backward(d(raw[:, :, :HQ]), d(raw[:, :, HQ:HQ + HK]), d(s["wq"]), d(s["wk"]), d(s["pos"]), d(s["freq"]),
                             d(dq), d(dk), d(dq), d(dk), eps=EPS)
    ctx.linear_backward(d(s["x"]), d(s["w"]), abi.ACT_NONE, None, d(dqkv.view(B, T, HEADS * D)), d(dx), d(dw))
    ctx.binary(abi.OP_ADD, d(dx), d(dy), d(dx))  # the residual's part
    ctx.synchronize()
    return host(dx).astype(F64), host(dw).astype(F64)


# Roundings on the way from x to y, each of half a step of the type, in numbers of the size of 1: qkv, q
# and k, the weights P, o, y.  q and k move a score by scale * |q| |k| of them (2 sqrt(D) at most here), which
# moves o by that times |v|.  Forty steps of the type cover them; binary32's products add their
# 100 u of sums of at most 150 terms.
STEPS = 40


@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_sublayer_and_gradients(ctx, dt):
    c, s = Layer(dt), {}
    y = host(forward(ctx, c, s)).astype(F64)
    half = 2.0 ** -11 if dt == np.float16 else 2.0 ** -24
    tol = STEPS * half + 400 * U
    x = c.x.astype(F64)
    ref = c.exact(x)
    assert np.abs(y - ref).max() <= tol * np.abs(ref).max()
    dx, dw = backward(ctx, c, s)
    rng = np.random.RandomState(0)
    h = 1e-5
    dy = c.dy.astype(F64)
    for g, value in ((dx, "x"), (dw, "w")):
        way = rng.randn(*g.shape)
        if value == "x":
            diff = ((c.exact(x + h * way) - c.exact(x - h * way)) * dy).sum() / (2 * h)
        else:
            w = c.w.astype(F64)
            diff = ((c.exact(x, w + h * way) - c.exact(x, w - h * way)) * dy).sum() / (2 * h)
        # independent roundings of a gradient's elements add up as their root of squares along a random way
        size = np.sqrt(((g * way) ** 2).sum()) * STEPS
        assert abs((g * way).sum() - diff) <= size * tol + 1e-6 * abs(diff), value


@pytest.mark.parametrize("dt", [np.float16, np.float32])
def test_tokens_one_by_one_over_a_cache(ctx, dt):
    """Each token's query over the keys so far, normed and rotated straight into the cache, gives what the
    prompt's pass gave for it: their P are rounded apart, 2^-11 each (binary32: sums of 150 terms)."""
    import torch
    c, s = Layer(dt), {}
    forward(ctx, c, s)
    want = host(s["o"]).astype(F64)
    raw = s["qkv"].view(B, T, HEADS, D)
    cache = torch.full((2, B, T, HK, D), float("nan"), dtype=s["x"].dtype, device="cuda")
    got = torch.empty_like(s["o"])
    q = torch.empty(B, 1, HQ, D, dtype=s["x"].dtype, device="cuda")
    lengths = [torch.full((B,), t + 1, dtype=torch.int32, device="cuda") for t in range(T)]
    o = torch.empty_like(q)
    for t in range(T):
        row = raw[:, t:t + 1]
        ctx.norm_rotary(d(row[:, :, :HQ]), d(row[:, :, HQ:HQ + HK]), d(s["wq"]), d(s["wk"]), d(s["pos"][:, t:t + 1]), d(s["freq"]),
                        d(q), d(cache[0][:, t:t + 1]), eps=EPS)
        ctx.gather(d(row[:, :, HQ + HK:]), d(cache[1][:, t:t + 1]))
        ctx.attention(d(q), d(cache[0]), d(cache[1]), d(o), c.scale, window=WINDOW, sinks=SINKS, k_lengths=d(lengths[t]))
        ctx.gather(d(o), d(got[:, t:t + 1]))
    ctx.synchronize()
    assert np.array_equal(host(cache[0].contiguous()), host(s["k"].contiguous()))
    tol = 4 * 2.0 ** -11 if dt == np.float16 else 600 * U
    assert np.abs(host(got).astype(F64) - want).max() <= tol * np.abs(want).max()
