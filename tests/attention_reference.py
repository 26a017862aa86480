"""Binary64 forms of the attention operators with the bounds that their binary32 arithmetic keeps.

u = 2^-24 is half a step of binary32; each bound counts roundings (see the functions), and an
output's own rounding to its type is added where it is compared (helpers' ``near``)."""
import numpy as np

F64 = np.float64
U = 2.0 ** -24
STEP = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float16): 2.0 ** -11}
TINY = {np.dtype(np.float32): 2.0 ** -149, np.dtype(np.float16): 2.0 ** -25}


def near(out, ref, err, what):
    """|out - ref| <= err and the output's own rounding; infinities and zeros where ref has them."""
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    inf = np.isinf(ref)
    assert np.array_equal(np.isinf(out), inf) and np.array_equal(out[inf], ref[inf]), what
    with np.errstate(invalid="ignore"):
        bound = err + STEP[out.dtype] * (np.abs(ref) + err) + TINY[out.dtype] + 1e-300
        bad = np.where(inf, 0.0, np.abs(out.astype(F64) - ref) / bound)
    assert not np.isnan(bad).any(), (what, "NaN")
    assert bad.max(initial=0) <= 1.0, (what, float(bad.max()), np.unravel_index(np.argmax(bad), bad.shape))


# ---- norm and rotation ------------------------------------------------------------------------
def angles(pos, freq, sections):
    """[tokens, pairs] from positions [tokens] or [tokens, axes]."""
    pos = pos.astype(F64)
    if sections is None:
        return pos[:, None] * freq.astype(F64)
    axis = np.repeat(np.arange(len(sections)), sections)
    return pos[:, axis] * freq.astype(F64)


def halves(x, n, pairs):
    return (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if pairs else (x[..., :n], x[..., n:2 * n])


def turned(x, t, pairs, magnitude=False):
    """x [tokens, heads, D] with its pairs turned by t; magnitude: the sums of both terms' sizes."""
    n = t.shape[1]
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    a, b = halves(x, n, pairs)
    y = x.copy()
    ya, yb = halves(y, n, pairs)
    if magnitude:
        ya[...], yb[...] = abs(a) + abs(b), abs(a) + abs(b)
    else:
        p, q = a * c - b * s, b * c + a * s
        ya[...], yb[...] = p, q
    return np.abs(y) if magnitude else y


def slope(t, n_cols, pairs):
    """What an angle's error in binary64 (three roundings of its size) adds, per column."""
    e = np.zeros((t.shape[0], 1, n_cols))
    a, b = halves(e, t.shape[1], pairs)
    a[...] = b[...] = (np.abs(t) * 2.0 ** -51)[:, None]
    return e


def rotary(x, w, eps, t, pairs):
    """Outputs and bound: the norm's factor is off by (D / 2 + 6) u (the sum of squares by D u, of which
    the root takes half), sine and cosine by 4 u (a turn rounded to binary32: 1.6 u, and 2 ulp), the
    products by 4 u."""
    x = x.astype(F64)
    D = x.shape[-1]
    r = 1.0 if w is None else 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = x * r * (1.0 if w is None else w.astype(F64))
    size = turned(y, t, pairs, magnitude=True)
    return turned(y, t, pairs), size * ((D / 2 + 16) * U + slope(t, D, pairs))


def rotary_backward(x, w, eps, t, pairs, dy):
    """dx, its bound, dw, its bound.  g is off by 8 u of its two terms (and the angle); the means along
    the row by a further (D + 16) u of their terms; rstd as in rotary; dw by a rounding a row."""
    x, dy = x.astype(F64), dy.astype(F64)
    D = x.shape[-1]
    g = turned(dy, -t, pairs)
    eg = turned(dy, -t, pairs, magnitude=True) * (8 * U + slope(t, D, pairs))
    if w is None:
        return g, eg, None, None
    w = w.astype(F64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh, h = x * r, g * w
    rel = (D / 2 + 16) * U
    c = (h * xh).mean(-1, keepdims=True)
    eh = eg * np.abs(w) + 2 * U * np.abs(h)
    ec = (eh * np.abs(xh)).mean(-1, keepdims=True) + (2 * D + 32) * U * np.abs(h * xh).mean(-1, keepdims=True)
    err = r * (eh + np.abs(xh) * ec + rel * (np.abs(h) + 2 * np.abs(xh * c)))
    n = x.shape[0] * x.shape[1]
    edw = (eg * np.abs(xh) + rel * np.abs(g * xh)).sum((0, 1)) + (n + 32) * U * np.abs(g * xh).sum((0, 1))
    return r * (h - xh * c), err, (g * xh).sum((0, 1)), edw


# ---- attention --------------------------------------------------------------------------------
def visible(sq, sk, nq, nk, window, sinks):
    i, j = np.arange(sq)[:, None], np.arange(sk)[None]
    p = i + nk - nq
    seen = (j <= p) & (i < nq) & (j < nk)
    if window:
        seen &= (p - j < window) | (j < sinks)
    return seen


class Attention:
    """One sequence and head: q [sq, D], k and v [sk, D], and its mask."""

    def __init__(self, q, k, v, seen, scale, dtype):
        self.q, self.k = q.astype(F64), np.where(seen.any(0)[:, None], k.astype(F64), 0.0)
        self.v = np.where(seen.any(0)[:, None], v.astype(F64), 0.0)
        self.q = np.where(seen.any(1)[:, None], self.q, 0.0)
        self.seen, self.scale, self.half = seen, scale, np.dtype(dtype) == np.float16
        D = q.shape[1]
        z = self.q @ self.k.T * scale
        self.z = np.where(seen, z, -np.inf)
        self.m = np.where(seen.any(1), self.z.max(1, initial=-np.inf), 0.0)[:, None]
        # a score is off by its sum's (D + 100) u sum|q||k| and its scaling
        self.es = np.where(seen, (D + 100) * U * (np.abs(self.q) @ np.abs(self.k).T) * scale + 4 * U * np.abs(z), 0.0)

    def forward(self):
        """o, bound, lse, bound.  A weight's relative error ep is its score's and the maximum's, and 8 u of
        exp; F16 rounds it by 2^-11, or 2^-25 (of a largest weight of at least 1) where it is small.  Sums
        over n weights add (n + 100) u of their terms, twice (values and norm)."""
        e = np.exp(self.z - self.m)
        total = e.sum(1, keepdims=True)
        any_ = total[:, 0] > 0
        p = e / np.where(total == 0, 1, total)
        n = self.seen.sum(1, keepdims=True)
        ep = (self.es + 4 * U * np.abs(self.m)).max(1, keepdims=True, initial=0) + 8 * U
        lse = np.where(any_, self.m[:, 0] + np.log(np.where(total == 0, 1, total))[:, 0], -np.inf)
        rel = 2 * ep + 2 * (n + 100) * U + (2.0 ** -11 if self.half else 0)
        err = rel * (p @ np.abs(self.v))
        if self.half:
            err = err + 2.0 ** -25 * (self.seen @ np.abs(self.v))
        el = np.where(any_, ep[:, 0] + (n[:, 0] + 100) * U + 4 * U * np.abs(np.where(any_, lse, 0)), 0)
        return p @ self.v, err, lse, el

    def backward(self, o, lse, do):
        """(dq, dk, dv) and their bounds, from the o and lse given.  P as in forward (lse is an input);
        dP and delta are off by (D + 100) u of their terms.  delta is sum(P dP) = sum(dout o), which the
        operator may take either way: o is rounded by half a step of its type, so the second differs from the
        first by at most that of sum|dout||o| (2^-11; binary32's 2^-24 is within the 100 u).  F16 rounds P
        (2^-11, 2^-25 at least) and dS (2^-11; below 2^-39 of a bound on the largest, 2 |dout| |v|, bits go:
        the power of two brings that bound to 2^14 at least and a step of the smallest numbers is 2^-25)."""
        live = self.seen.any(1)[:, None]
        do, o = np.where(live, do.astype(F64), 0.0), np.where(live, o.astype(F64), 0.0)
        lse = np.where(live, lse.astype(F64)[:, None], 0.0)
        D = self.q.shape[1]
        p = np.where(self.seen, np.exp(np.where(self.seen, self.z, 0.0) - lse), 0.0)
        dp = do @ self.v.T
        delta = (p * dp).sum(1, keepdims=True)
        ds = p * (dp - delta)
        ep = self.es + 6 * U * np.abs(lse) + 8 * U
        ed = (D + 100) * U * (np.abs(do) @ np.abs(self.v).T + (np.abs(do) * np.abs(o)).sum(1, keepdims=True))
        if self.half:
            ed = ed + 2.0 ** -11 * (np.abs(do) * np.abs(o)).sum(1, keepdims=True)
        eds = p * ((ep + 4 * U) * np.abs(dp - delta) + ed)
        epp = p * ep
        if self.half:
            size = np.sqrt((do ** 2).sum(1).max(initial=0) * (self.v ** 2).sum(1).max(initial=0))
            eds = np.where(self.seen, eds + 2.0 ** -11 * np.abs(ds) + 2.0 ** -39 * 2 * size, 0)
            epp = np.where(self.seen, epp + 2.0 ** -11 * p + 2.0 ** -25, 0)
        rows, cols = self.seen.sum(1, keepdims=True), self.seen.sum(0)[:, None]
        s = self.scale

        def product(x, ex, y, n):
            return x @ y, ex @ np.abs(y) + (n + 104) * U * (np.abs(x) @ np.abs(y))
        dq, edq = product(ds * s, eds * s, self.k, rows)
        dk, edk = product(ds.T * s, eds.T * s, self.q, cols)
        dv, edv = product(p.T, epp.T, do, cols)
        return (dq, dk, dv), (edq, edk, edv)
