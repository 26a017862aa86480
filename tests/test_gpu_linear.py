"""GPU linear and gated linear layers and their backward passes (through the C ABI) against binary64.

Tolerances count roundings, element by element.  With u = 2^-24 and h = half a step of the type:
* a product summed over k terms in binary32, in any order and with truncating accumulators or
  operands split into parts, is off by at most E = (k + 100) u sum|x||w|: a rounding (or two
  truncations) for each of the k additions of a chain no longer than k / 4 + 8, and 100 for the
  operands' split (three dropped products below 2^-22) and the joining of partial sums;
* an activation has a slope of at most 1.13, and is itself off by at most 16 u (1 + |z|)
  (binary32) or 2^-18 (1 + |z|) (binary16, fast exponential: 2^-21 and 2^-24 |z| of exp, through
  the slope of the sigmoid and a product), its derivative by at most four times that;
* outputs are rounded once: h |y|, and half the smallest subnormal.
The backward passes round dz once to the dtype (a binary16 dz of up to 2^16 elements to two parts:
2^-22 and the two roundings' ends), which the products' bound carries on."""
import numpy as np
import pytest

from helpers import dev, empty, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
STEP = {np.float32: 2.0 ** -24, np.float16: 2.0 ** -11}
TINY = {np.float32: 2.0 ** -149, np.float16: 2.0 ** -25}
ACT = {"none": abi.ACT_NONE, "relu": abi.ACT_RELU, "gelu": abi.ACT_GELU, "silu": abi.ACT_SILU,
       "sigmoid": abi.ACT_SIGMOID}
F64 = np.float64


def d(t):
    return None if t is None else abi.desc_of(t)


def act64(z, act):
    if act == "none":
        return z, np.ones_like(z)
    if act == "relu":
        return np.maximum(z, 0), (z > 0).astype(F64)
    if act == "gelu":
        t = np.tanh(0.7978845608 * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608 * (1 + 3 * 0.044715 * z * z)
    with np.errstate(over="ignore"):
        p = 1 / (1 + np.exp(-z))
    return (z * p, p + z * p * (1 - p)) if act == "silu" else (p, p * (1 - p))


def act_error(z, act, dt):
    if act in ("none", "relu"):
        return np.zeros_like(z)
    return (16 * U if dt == np.float32 else 2.0 ** -18) * (1 + np.abs(z))


def near(out, ref, err, what):
    """|out - ref| <= err and the output's own rounding."""
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    s = out.dtype.type
    bound = err + STEP[s] * (np.abs(ref) + err) + TINY[s] + 1e-300
    bad = np.abs(out.astype(F64) - ref) / bound
    assert not np.isnan(bad).any() and bad.max(initial=0) <= 1.0, (what, float(np.nanmax(bad)))


def product(x, w, b=None):
    z = x @ w
    err = (x.shape[1] + 100) * U * (np.abs(x) @ np.abs(w))
    if b is None:
        return z, err
    return z + b, err + 2 * U * (np.abs(z) + np.abs(b))


class Case:
    """Inputs of one layer: x [m, k], weights [k, n] (one or two), biases, residual, dy."""

    def __init__(self, m, k, n, dt, gated=False, bias=True, bdt=np.float32, seed=3):
        s = max(k, 1) ** -0.5
        self.m, self.k, self.n, self.dt, self.nw = m, k, n, dt, 2 if gated else 1
        self.x = datagen.normal(seed, (m, k), 0, 1).astype(dt)
        self.w = [datagen.normal(seed + 1 + i, (k, n), 0, s).astype(dt) for i in range(self.nw)]
        self.b = [datagen.normal(seed + 3 + i, (n,), 0, 0.5).astype(bdt) if bias else None for i in range(self.nw)]
        self.r = datagen.normal(seed + 5, (m, n), 0, 1).astype(dt)
        self.dy = datagen.normal(seed + 6, (m, n), 0, 1).astype(dt)
        self.bdt = bdt

    def products(self):
        x = self.x.astype(F64)
        return [product(x, w.astype(F64), None if b is None else b.astype(F64)) for w, b in zip(self.w, self.b)]

    def kept(self):
        return [z.astype(self.dt) for z, _ in self.products()]


def check_forward(c, act, y, pre, residual=False):
    zs = c.products()
    for (z, e), p in zip(zs, pre):
        if p is not None:
            near(p, z, e, "pre")
    z, e = zs[0]
    a, _ = act64(z, act)
    ea = 1.13 * e + act_error(z, act, c.dt)
    if c.nw == 2:
        u, eu = zs[1]
        ref, err = a * u, ea * (np.abs(u) + eu) + np.abs(a) * eu
    else:
        r = c.r.astype(F64) if residual else 0.0
        ref, err = a + r, ea
    near(y, ref, err + 4 * U * np.abs(ref) + 2 * U * np.abs(a), "y")


def check_backward(c, act, kept, dx, dw, db):
    x, dy = c.x.astype(F64), c.dy.astype(F64)
    z = kept[0].astype(F64) if act != "none" or c.nw == 2 else np.zeros_like(dy)
    a, g = act64(z, act)
    ea = act_error(z, act, c.dt)
    if c.nw == 2:
        u = kept[1].astype(F64)
        dz = [dy * u * g, dy * a]
        ez = [np.abs(dy * u) * 4 * ea, np.abs(dy) * ea]
    else:
        dz, ez = [dy * g], [np.abs(dy) * 4 * ea]
    ez = [e + 4 * U * np.abs(v) for e, v in zip(ez, dz)]
    for v, e, o in zip(dz, ez, db):
        if o is not None:
            near(o, v.sum(0), e.sum(0) + (c.m + 40) * U * np.abs(v).sum(0), "db")
    if not (c.nw == 1 and act == "none"):
        step = 2.0 ** -21 if c.dt == np.float16 and c.m * c.n <= 65536 else STEP[c.dt]
        ez = [e + step * (np.abs(v) + e) + TINY[c.dt] for e, v in zip(ez, dz)]
    w = [v.astype(F64) for v in c.w]
    if dx is not None:
        ref = sum(v @ m.T for v, m in zip(dz, w))
        mag = sum((np.abs(v) + e) @ np.abs(m).T for v, e, m in zip(dz, ez, w))
        err = sum(e @ np.abs(m).T for e, m in zip(ez, w)) + (c.nw * c.n + 100) * U * mag
        near(dx, ref, err, "dx")
    for v, e, o in zip(dz, ez, dw):
        if o is not None:
            ax = np.abs(x).T
            near(o, x.T @ v, ax @ e + (c.m + 100) * U * (ax @ (np.abs(v) + e)), "dw")


def nan(shape, dt):
    t = empty(shape, dt)
    t.fill_(float("nan"))
    return t


def forward(ctx, c, act, residual=False, keep=True, precision=abi.MM_AUTO, tx=None, tw=None):
    import torch  # noqa: F401
    tx = dev(c.x) if tx is None else tx
    tw = [dev(w) for w in c.w] if tw is None else tw
    tb = [None if b is None else dev(b) for b in c.b]
    y = nan((c.m, c.n), c.dt)
    pre = [nan((c.m, c.n), c.dt) if keep else None for _ in c.w]
    if c.nw == 2:
        ctx.gated_linear(d(tx), d(tw[0]), d(tw[1]), d(tb[0]), d(tb[1]), ACT[act], d(pre[0]), d(pre[1]), d(y), precision)
    else:
        tr = dev(c.r) if residual else None
        ctx.linear(d(tx), d(tw[0]), d(tb[0]), ACT[act], d(tr), d(pre[0]), d(y), precision)
    return host(y), [None if p is None else host(p) for p in pre]


def backward(ctx, c, act, kept, want="xwb", precision=abi.MM_AUTO, tx=None, tw=None, tdy=None):
    tx = dev(c.x) if tx is None else tx
    tw = [dev(w) for w in c.w] if tw is None else tw
    tdy = dev(c.dy) if tdy is None else tdy
    tk = [dev(v) for v in kept]
    dx = nan((c.m, c.k), c.dt) if "x" in want else None
    dw = [nan((c.k, c.n), c.dt) if "w" in want else None for _ in c.w]
    db = [nan((c.n,), c.bdt) if "b" in want else None for _ in c.w]
    if c.nw == 2:
        ctx.gated_linear_backward(d(tx), d(tw[0]), d(tw[1]), ACT[act], d(tk[0]), d(tk[1]), d(tdy), d(dx), d(dw[0]),
                                  d(dw[1]), d(db[0]), d(db[1]), precision)
    else:
        ctx.linear_backward(d(tx), d(tw[0]), ACT[act], d(tk[0]) if tk else None, d(tdy), d(dx), d(dw[0]), d(db[0]),
                            precision)
    return [None if t is None else host(t) for t in (dx,)] + [[None if t is None else host(t) for t in v]
                                                             for v in (dw, db)]


# one element; one token; sizes that fill no load, no tile and no group of 8 columns; whole tiles
# and one past them; many rows, many columns, a long sum
SIZES = [(1, 1, 1), (1, 64, 64), (1, 512, 1000), (3, 5, 7), (2, 33, 129), (128, 64, 128), (129, 65, 127),
         (100, 72, 200), (257, 136, 264), (64, 1000, 8), (300, 520, 1366), (1, 4096, 1024), (5, 2048, 520),
         (33, 16, 2050), (17, 4100, 72), (700, 24, 40), (1000, 8, 1)]
DTYPES = [np.float32, np.float16]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act,residual", [("none", False), ("gelu", True)])
def test_linear(ctx, size, dt, act, residual):
    c = Case(*size, dt, bias=residual)
    y, pre = forward(ctx, c, act, residual)
    check_forward(c, act, y, pre, residual)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("keep", [False, True])
def test_gated_linear(ctx, size, dt, keep):
    c = Case(*size, dt, gated=True, bias=keep)
    y, pre = forward(ctx, c, "silu", keep=keep)
    check_forward(c, "silu", y, pre)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_backward(ctx, size, dt, act):
    c = Case(*size, dt)
    kept = c.kept()
    check_backward(c, act, kept, *backward(ctx, c, act, kept if act != "none" else []))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
def test_gated_linear_backward(ctx, size, dt):
    c = Case(*size, dt, gated=True)
    kept = c.kept()
    check_backward(c, "silu", kept, *backward(ctx, c, "silu", kept))


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_activations(ctx, act, dt, gated):
    c = Case(70, 48, 104, dt, gated=gated, bdt=dt)
    for w in c.w:
        w *= dt(6)  # products far into both tails
    y, pre = forward(ctx, c, act, True)
    check_forward(c, act, y, pre, True)
    kept = c.kept()
    check_backward(c, act, kept, *backward(ctx, c, act, kept))


# the forward product, dx and dw in turn large enough for pairs of SMs, ragged in every size
@pytest.mark.parametrize("size", [(2200, 136, 2500), (2200, 2500, 136), (136, 2200, 2500)])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_pairs_of_sms(ctx, size, dt, gated):
    c = Case(*size, dt, gated=gated)
    y, pre = forward(ctx, c, "silu", True)
    assert ctx.last_kernel().startswith("k_linear_pair") == (size[1] == 136), ctx.last_kernel()
    check_forward(c, "silu", y, pre, True)
    kept = c.kept()
    check_backward(c, "silu", kept, *backward(ctx, c, "silu", kept))


# x's and the weights' gradients by one launch: tiles and sums of all ragged, shared out over
# clusters or not, dz in two parts or one, operands that are copied and ones read in place; the
# last size takes two launches
@pytest.mark.parametrize("size", [(17, 48, 64), (40, 264, 1000), (128, 1024, 256), (129, 130, 1), (200, 300, 64), (131, 257, 450), (777, 136, 256), (520, 512, 1030),
                                  (1100, 260, 130), (8192, 256, 512)])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_both_gradients(ctx, size, dt, gated):
    c = Case(*size, dt, gated=gated)
    kept = c.kept()
    dx, dw, db = backward(ctx, c, "gelu", kept)
    check_backward(c, "gelu", kept, dx, dw, db)
    before = [ctx.launch_count()]
    for want in ("xwb", "xb", "w"):  # dz, its column sums, products; no sums for the last
        backward(ctx, c, "gelu", kept, want)
        before.append(ctx.launch_count())
    if dt == np.float16 and size[1] % 8 == 0 and size[2] % 8 == 0:  # nothing is copied
        assert list(np.diff(before)) == [4 if size[0] == 8192 else 3, 3, 2], before


# fewer of the pairs' tiles than 60 % of them, but more of the others than SMs
@pytest.mark.parametrize("size,gated", [((130, 72, 10100), False), ((200, 40, 5000), True), ((9600, 24, 250), False)])
def test_few_tiles_for_pairs(ctx, size, gated):
    c = Case(*size, np.float16, gated=gated)
    y, pre = forward(ctx, c, "silu", True)
    assert ctx.last_kernel().startswith("k_linear_pair")
    check_forward(c, "silu", y, pre, True)
    kept = c.kept()
    check_backward(c, "silu", kept, *backward(ctx, c, "silu", kept))


def strided(a, how):
    """A device view with the values of `a`: transposed storage, an odd row pitch, columns of a
    wider matrix, every other column, a start off the 16-byte boundary."""
    import torch
    t = dev(a)
    r, c = a.shape
    if how == "transposed":
        return t.t().contiguous().t()
    big = torch.full((2 * r + 3, 2 * c + 11), float("nan"), dtype=t.dtype, device="cuda")
    v = {"pitch": lambda: big[:r, :c], "columns": lambda: big[1:1 + r, 8:8 + c], "odd": lambda: big[:r, 3:3 + c],
         "step": lambda: big[:r, :2 * c:2], "rows": lambda: big[:2 * r:2, :c],
         "flat": lambda: big.view(-1)[1:1 + r * c].view(r, c)}[how]()
    v.copy_(t)
    return v


@pytest.mark.parametrize("how", ["transposed", "pitch", "columns", "odd", "step", "rows", "flat"])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(37, 40, 56), (200, 136, 264)])
def test_strides(ctx, how, dt, size):
    c = Case(*size, dt)
    tx, tw = strided(c.x, how), [strided(w, how) for w in c.w]
    y, pre = forward(ctx, c, "silu", True, tx=tx, tw=tw)
    check_forward(c, "silu", y, pre, True)
    kept = c.kept()
    tdy = strided(c.dy, how) if how in ("pitch", "columns", "odd", "rows", "flat") else None
    check_backward(c, "silu", kept, *backward(ctx, c, "silu", kept, tx=tx, tw=tw, tdy=tdy))
    c = Case(*size, dt, gated=True)
    tw = [strided(w, h) for w, h in zip(c.w, (how, "pitch"))]
    y, pre = forward(ctx, c, "relu", tx=tx, tw=tw)
    check_forward(c, "relu", y, pre)
    kept = c.kept()
    check_backward(c, "relu", kept, *backward(ctx, c, "relu", kept, tx=tx, tw=tw, tdy=tdy))


@pytest.mark.parametrize("m", [1, 3, 8, 9, 16])
@pytest.mark.parametrize("how", ["plain", "transposed", "odd", "step"])
@pytest.mark.parametrize("dt", DTYPES)
def test_few_rows(ctx, m, how, dt):
    """A handful of rows, both orders of the weight, loads that fit and loads that do not; a long sum
    that several CTAs share, and columns past the last whole tile."""
    for k, n in ((1100, 332), (515, 37)):
        for gated in (False, True):
            c = Case(m, k, n, dt, gated=gated)
            tw = [dev(w) if how == "plain" else strided(w, how) for w in c.w]
            y, pre = forward(ctx, c, "silu", True, tw=tw)
            check_forward(c, "silu", y, pre, True)
            kept = c.kept()
            check_backward(c, "silu", kept, *backward(ctx, c, "silu", kept, tw=tw))


def test_one_row_for_all_and_reversed_rows(ctx):
    """Stride 0 (a broadcast input) and a negative stride."""
    for dt in DTYPES:
        c = Case(19, 48, 40, dt)
        c.x[:] = c.x[:1]
        tx, tw, y = dev(c.x[:1]), dev(c.w[0]), nan((19, 40), dt)
        tb, code = dev(c.b[0]), abi.torch_dtype_code(tx.dtype)
        ctx.linear(abi.make_desc(tx.data_ptr(), code, (19, 48), (0, 1)), d(tw), d(tb), abi.ACT_RELU, None, None, d(y))
        check_forward(c, "relu", host(y), [None])
        c = Case(19, 48, 40, dt)
        tx = dev(c.x[::-1])
        at = tx.data_ptr() + 18 * 48 * tx.element_size()
        ctx.linear(abi.make_desc(at, code, (19, 48), (-48, 1)), d(tw), d(tb), abi.ACT_RELU, None, None, d(y))
        c.w = [host(tw)]
        check_forward(c, "relu", host(y), [None])


def test_leading_dims_and_vectors(ctx):
    c = Case(24, 40, 32, np.float16)
    tx, tw, tb, tr = dev(c.x), dev(c.w[0]), dev(c.b[0]), dev(c.r)
    y, pre = nan((2, 3, 4, 32), np.float16), nan((2, 3, 4, 32), np.float16)
    ctx.linear(d(tx.view(2, 3, 4, 40)), d(tw), d(tb), abi.ACT_GELU, d(tr.view(2, 3, 4, 32)), d(pre), d(y))
    check_forward(c, "gelu", host(y).reshape(24, 32), [host(pre).reshape(24, 32)], True)
    v = nan((32,), np.float16)
    ctx.linear(d(tx[5]), d(tw), d(tb), abi.ACT_NONE, None, None, d(v))
    z, e = c.products()[0]
    near(host(v), z[5], e[5], "vector")


def test_residual_added_in_place(ctx):
    for size in ((1, 2048, 1024), (33, 40, 57), (300, 256, 512)):
        c = Case(*size, np.float16)
        tx, tw, tb, y = dev(c.x), dev(c.w[0]), dev(c.b[0]), dev(c.r)
        ctx.linear(d(tx), d(tw), d(tb), abi.ACT_SILU, d(y), None, d(y))
        check_forward(c, "silu", host(y), [None], True)


@pytest.mark.parametrize("dt", DTYPES)
def test_nothing_to_sum_and_no_rows(ctx, dt):
    c = Case(5, 0, 24, dt)
    y, pre = forward(ctx, c, "gelu", True)
    check_forward(c, "gelu", y, pre, True)
    c = Case(0, 16, 24, dt)
    forward(ctx, c, "gelu", True)
    for gated in (False, True):
        c = Case(0, 16, 24, dt, gated=gated)
        _, dw, db = backward(ctx, c, "silu", c.kept())
        assert all(np.all(v == 0) for v in dw + db)
        c = Case(6, 16, 0, dt, gated=gated)
        dx, _, _ = backward(ctx, c, "silu", c.kept())
        assert np.all(dx == 0)


@pytest.mark.parametrize("want", ["x", "w", "b", "xb", "wb"])
@pytest.mark.parametrize("gated", [False, True])
def test_only_what_is_asked_for(ctx, want, gated):
    for act in ("none", "sigmoid"):
        c = Case(150, 64, 72, np.float16, gated=gated)
        kept = c.kept()
        check_backward(c, act, kept, *backward(ctx, c, act, kept, want=want))


def test_one_weight_of_two(ctx):
    c = Case(90, 40, 48, np.float16, gated=True)
    kept = c.kept()
    t = [dev(v) for v in (c.x, c.w[0], c.w[1], kept[0], kept[1], c.dy)]
    for which in (0, 1):
        out = nan((40, 48), np.float16)
        a = [d(out), None] if which == 0 else [None, d(out)]
        ctx.gated_linear_backward(*(d(v) for v in t[:3]), abi.ACT_SILU, *(d(v) for v in t[3:]), None, *a)
        check_backward(c, "silu", kept, None, [host(out), None] if which == 0 else [None, host(out)], [None, None])


@pytest.mark.parametrize("size", [(70, 72, 136), (300, 100, 200)])
def test_ffma(ctx, size):
    for gated in (False, True):
        c = Case(*size, np.float32, gated=gated)
        y, pre = forward(ctx, c, "gelu", True, precision=abi.MM_FP32_FFMA)
        check_forward(c, "gelu", y, pre, True)
        kept = c.kept()
        check_backward(c, "gelu", kept, *backward(ctx, c, "gelu", kept, precision=abi.MM_FP32_FFMA))


def rel(out, ref):
    return float((out.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(4096, 2048, 4096), (1000, 1027, 2050), (1, 8192, 4096), (2048, 4100, 520)])
def test_large_products(ctx, dt, size):
    """Norm of the error over the norm.  binary16: a fraction of half a step.  binary32: a chain of k
    additions of independent terms has partial sums of size sqrt(j / k) of the last one, each
    rounded with an error of variance at most (u sqrt(j / k))^2 / 3, together u^2 k / 6: a relative
    error of u sqrt(k / 6), times sqrt(2) for a product of two such sums.  The bar is twice that
    (one binary32 constant for all k, as 2^-20 would be, is below it from k = 1536 on)."""
    import torch
    m, k, n = size
    g = torch.Generator(device="cuda").manual_seed(1)
    tdt = torch.float32 if dt == np.float32 else torch.float16

    def bar(terms):
        return 2 * U * (terms / 3) ** 0.5 if dt == np.float32 else 2.0 ** -11

    def normal(r, c, s):
        return (torch.randn(r, c, generator=g, device="cuda") * s).to(tdt)

    x, w, w2, dy = normal(m, k, 1), normal(k, n, k ** -0.5), normal(k, n, k ** -0.5), normal(m, n, 1)
    y, gate, up = (torch.empty(m, n, dtype=tdt, device="cuda") for _ in range(3))
    ctx.linear(d(x), d(w), None, abi.ACT_NONE, None, None, d(y))
    assert rel(y, x.double() @ w.double()) <= bar(k)
    ctx.gated_linear(d(x), d(w), d(w2), None, None, abi.ACT_SILU, d(gate), d(up), d(y))
    g64, u64 = x.double() @ w.double(), x.double() @ w2.double()
    assert rel(gate, g64) <= bar(k) and rel(up, u64) <= bar(k)
    assert rel(y, g64 * torch.sigmoid(g64) * u64) <= bar(k)
    dx, dw, dw2 = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    ctx.gated_linear_backward(d(x), d(w), d(w2), abi.ACT_SILU, d(gate), d(up), d(dy), d(dx), d(dw), d(dw2))
    g64, u64, dy64 = gate.double(), up.double(), dy.double()
    p = torch.sigmoid(g64)
    dg, du = dy64 * u64 * (p + g64 * p * (1 - p)), dy64 * g64 * p
    # one more rounding, of dz (a single row has no other: m = 1 counts as a chain of 64)
    m = max(m, 64)
    assert rel(dx, dg @ w.double().t() + du @ w2.double().t()) <= 2 * bar(2 * n)
    assert rel(dw, x.double().t() @ dg) <= 2 * bar(m) and rel(dw2, x.double().t() @ du) <= 2 * bar(m)


def whole(tdt, seed, *shape):
    """Whole numbers from -2 to 2."""
    import torch
    return torch.randint(-2, 3, shape, generator=torch.Generator(device="cuda").manual_seed(seed),
                         device="cuda", dtype=torch.int8).to(tdt)


@pytest.mark.parametrize("precision", [abi.MM_AUTO, abi.MM_FP32_FFMA])
@pytest.mark.parametrize("dt", DTYPES)
def test_more_than_2_to_the_31_outputs(ctx, dt, precision):
    """Whole numbers, whose products (at most 8 x 4 + 4) are exact in every type."""
    import torch
    if dt == np.float16 and precision == abi.MM_FP32_FFMA:
        precision = abi.MM_FP16_F32ACC
    tdt = torch.float32 if dt == np.float32 else torch.float16
    m, k, n = 2**21 + 77, 8, 1032
    x, w, b, res = whole(tdt, 1, m, k), whole(tdt, 2, k, n), whole(tdt, 3, n), whole(tdt, 4, m, n)
    y, pre = torch.empty_like(res), torch.empty_like(res)
    ctx.linear(d(x), d(w), d(b), abi.ACT_RELU, d(res), d(pre), d(y), precision)
    for i in range(0, m, 2**18):
        want = x[i:i + 2**18] @ w + b
        assert torch.equal(pre[i:i + 2**18], want)
        assert torch.equal(y[i:i + 2**18], want.relu() + res[i:i + 2**18])
    # and back: few rows of dy are not 0, so that every sum stays exact
    del y
    dy, dx = res.zero_(), torch.full_like(x, float("nan"))
    rows = torch.tensor([0, 1000, 2**20 + 3, m - 200, m - 1], device="cuda")
    dy[rows] = whole(tdt, 5, 5, n)
    dw, db = torch.empty_like(w), torch.empty(n, device="cuda")
    few = torch.randint(0, 50, (2, 16), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    w.zero_()[:, few[0] * 20 + few[1] % 20] = 1  # at most 16 columns of 1: dx is at most 32
    ctx.linear_backward(d(x), d(w), abi.ACT_RELU, d(pre), d(dy), d(dx), d(dw), d(db), precision)
    dz = dy[rows] * (pre[rows] > 0)
    want = torch.zeros_like(x)
    want[rows] = (dz.double() @ w.double().t()).to(tdt)
    assert torch.equal(dx, want)
    assert torch.equal(dw, (x[rows].double().t() @ dz.double()).to(tdt))
    assert torch.equal(db, dz.float().sum(0))


@pytest.mark.parametrize("m", [1, 3, 40])
@pytest.mark.parametrize("dt", DTYPES)
def test_weight_of_more_than_2_to_the_31_elements(ctx, dt, m):
    """As above; x is 0 but for its ends."""
    import torch
    tdt = torch.float32 if dt == np.float32 else torch.float16
    k, n = 2**16 + 8, 2**15 + 24
    w, x = whole(tdt, 1, k, n), torch.zeros(m, k, dtype=tdt, device="cuda")
    x[:, :4], x[:, -4:] = whole(tdt, 2, m, 4), whole(tdt, 3, m, 4)
    y, dx = torch.empty(m, n, dtype=tdt, device="cuda"), torch.empty_like(x)
    ctx.linear(d(x), d(w), None, abi.ACT_NONE, None, None, d(y))
    ends = torch.tensor([0, 1, 2, 3, k - 4, k - 3, k - 2, k - 1], device="cuda")
    assert torch.equal(y, (x[:, ends].double() @ w[ends].double()).to(tdt))
    dy = torch.zeros_like(y)
    dy[:, :4], dy[:, -4:] = whole(tdt, 4, m, 4), whole(tdt, 5, m, 4)
    ctx.linear_backward(d(x), d(w), abi.ACT_NONE, None, d(dy), d(dx), None, None)
    ends = torch.tensor([0, 1, 2, 3, n - 4, n - 3, n - 2, n - 1], device="cuda")
    assert torch.equal(dx, (dy[:, ends].double() @ w[:, ends].double().t()).to(tdt))


@pytest.mark.parametrize("size", [(1, 4096, 1000), (200, 1024, 256), (600, 512, 1024)])
@pytest.mark.parametrize("dt", DTYPES)
def test_same_bits_again(ctx, size, dt):
    c = Case(*size, dt, gated=True)
    kept = c.kept()
    for _ in range(2):
        a, b = backward(ctx, c, "silu", kept), backward(ctx, c, "silu", kept)
        assert np.array_equal(a[0], b[0])
        assert all(np.array_equal(p, q) for i in (1, 2) for p, q in zip(a[i], b[i]))
        assert np.array_equal(forward(ctx, c, "silu")[0], forward(ctx, c, "silu")[0])


def test_against_differences(ctx):
    """Gradients against central differences of the formulas in binary64 (a step of 1e-4 truncates
    below 1e-7 of the loss's scale; the kernels' own error is a few 1e-7)."""
    for gated in (False, True):
        c = Case(4, 6, 9, np.float32, gated=gated)
        kept = c.kept()
        dx, dw, db = backward(ctx, c, "gelu", kept)

        def loss(v):
            z = [v[0] @ v[1 + 2 * i] + v[2 + 2 * i] for i in range(c.nw)]
            y = act64(z[0], "gelu")[0]
            return float(((y * z[1] if gated else y) * c.dy).sum())

        base = [c.x.astype(F64)]
        grads = [dx]
        for i in range(c.nw):
            base += [c.w[i].astype(F64), c.b[i].astype(F64)]
            grads += [dw[i], db[i]]
        for i, gr in enumerate(grads):
            for at in list(np.ndindex(*gr.shape))[::4]:
                t, v = 1e-4, [q.copy() for q in base]
                v[i][at] += t
                hi = loss(v)
                v[i][at] -= 2 * t
                assert abs((hi - loss(v)) / (2 * t) - gr[at]) <= 1e-5 * (1 + np.abs(gr).max())


def test_rows_behind_the_last_stay(ctx):
    """Outputs that are the first rows of larger buffers: what lies behind them is not written."""
    import torch
    for dt in DTYPES:
        for size in ((1, 512, 264), (5, 64, 33), (130, 72, 200)):
            c = Case(*size, dt)
            tx, tw, tb = dev(c.x), dev(c.w[0]), dev(c.b[0])
            big = [torch.full((c.m + 200, c.n), 5.0, dtype=tx.dtype, device="cuda") for _ in range(2)]
            ctx.linear(d(tx), d(tw), d(tb), abi.ACT_GELU, None, d(big[0][:c.m]), d(big[1][:c.m]))
            pre, y = host(big[0]), host(big[1])
            check_forward(c, "gelu", y[:c.m], [pre[:c.m]])
            assert np.all(pre[c.m:] == 5) and np.all(y[c.m:] == 5)


def feed_forward(ctx, t, out):
    """y = x + (act(ln(x) wg) * (ln(x) wu)) wd and its gradients, in place of one model's sublayer."""
    eps = 1e-5
    ctx.layer_norm(d(t["x"]), d(t["g"]), d(t["b"]), eps, d(out["n"]))
    ctx.gated_linear(d(out["n"]), d(t["wg"]), d(t["wu"]), None, None, abi.ACT_SILU, d(out["gate"]), d(out["up"]),
                     d(out["h"]))
    ctx.linear(d(out["h"]), d(t["wd"]), None, abi.ACT_NONE, d(t["x"]), None, d(out["y"]))
    ctx.linear_backward(d(out["h"]), d(t["wd"]), abi.ACT_NONE, None, d(t["dy"]), d(out["dh"]), d(out["dwd"]))
    ctx.gated_linear_backward(d(out["n"]), d(t["wg"]), d(t["wu"]), abi.ACT_SILU, d(out["gate"]), d(out["up"]),
                              d(out["dh"]), d(out["dn"]), d(out["dwg"]), d(out["dwu"]))
    ctx.layer_norm_backward(d(t["x"]), d(t["g"]), d(out["dn"]), eps, d(out["dx"]), d(out["dg"]), d(out["db"]))
    ctx.binary(abi.OP_ADD, d(out["dx"]), d(t["dy"]), d(out["dxr"]))


def sublayer(m, c, f, tdt):
    import torch
    g = torch.Generator(device="cuda").manual_seed(7)

    def r(*s, scale=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * scale).to(tdt)

    t = {"x": r(m, c), "g": 1 + 0.1 * r(c), "b": 0.1 * r(c), "wg": r(c, f, scale=c ** -0.5),
         "wu": r(c, f, scale=c ** -0.5), "wd": r(f, c, scale=f ** -0.5), "dy": r(m, c)}
    shape = {"n": (m, c), "gate": (m, f), "up": (m, f), "h": (m, f), "y": (m, c), "dh": (m, f), "dwd": (f, c),
             "dn": (m, c), "dwg": (c, f), "dwu": (c, f), "dx": (m, c), "dg": (c,), "db": (c,), "dxr": (m, c)}
    return t, {k: torch.full(v, float("nan"), dtype=tdt, device="cuda") for k, v in shape.items()}


def sublayer64(t):
    import torch
    v = {k: x.double().requires_grad_(k != "dy") for k, x in t.items()}
    n = torch.nn.functional.layer_norm(v["x"], (v["x"].shape[1],), v["g"], v["b"], 1e-5)
    h = torch.nn.functional.silu(n @ v["wg"]) * (n @ v["wu"])
    y = v["x"] + h @ v["wd"]
    y.backward(v["dy"])
    return y.detach(), {k: x.grad for k, x in v.items() if k != "dy"}


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [(1, 256, 704), (77, 200, 333), (512, 512, 1408)])
def test_feed_forward_sublayer(ctx, dt, size):
    """The operators in a row against binary64 with gradients by differentiation.  About ten
    roundings of intermediate tensors of independent sign lie between the inputs and a gradient."""
    import torch
    tdt = torch.float32 if dt == np.float32 else torch.float16
    bar = 10 * (2.0 ** -20 if dt == np.float32 else 2.0 ** -11)
    t, out = sublayer(*size, tdt)
    feed_forward(ctx, t, out)
    y, g = sublayer64(t)
    assert rel(out["y"], y) <= bar
    for name, ref in (("dwd", g["wd"]), ("dwg", g["wg"]), ("dwu", g["wu"]), ("dg", g["g"]), ("db", g["b"]),
                      ("dxr", g["x"])):
        assert rel(out[name], ref) <= bar, name


@pytest.mark.parametrize("dt", DTYPES)
def test_captured_step_replays(ctx, dt):
    """A captured step, replayed twice on new inputs between eager calls of the same context; a
    second captured graph replays in between.  Neither shares workspace with the other."""
    import torch
    tdt = torch.float32 if dt == np.float32 else torch.float16
    sets = [sublayer(130, 264, 520, tdt), sublayer(61, 136, 248, tdt)]
    stream, before = torch.cuda.Stream(), ctx.stream()
    for t, o in sets:
        feed_forward(ctx, t, o)
    want = [{k: v.clone() for k, v in o.items()} for _, o in sets]
    torch.cuda.synchronize()
    graphs = []
    try:
        ctx.set_stream(stream.cuda_stream)
        for t, o in sets:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                feed_forward(ctx, t, o)
            graphs.append(g)
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(before)
    for _ in range(2):
        for _, o in sets:
            for v in o.values():
                v.fill_(float("nan"))
        for i in (0, 1, 0):
            graphs[i].replay()
        c = Case(90, 64, 128, dt)
        y, pre = forward(ctx, c, "relu")
        check_forward(c, "relu", y, pre)
        torch.cuda.synchronize()
        for (_, o), w in zip(sets, want):
            assert all(torch.equal(o[k], w[k]) for k in w)


def refused(status, fn, *a):
    with pytest.raises(abi.QsmlError) as e:
        fn(*a)
    assert e.value.status == status, e.value


def test_refusals(ctx):
    f32, f16 = np.float32, np.float16

    def t(*shape, dt=f32):
        return d(hold(empty(shape, dt)))

    kept = []

    def hold(v):
        kept.append(v)
        return v

    x, w, y, b, n = t(4, 8), t(8, 16), t(4, 16), t(16), abi.ACT_NONE
    L, G = ctx.linear, ctx.gated_linear
    refused(abi.E_DTYPE, L, x, t(8, 16, dt=f16), None, n, None, None, y)
    refused(abi.E_DTYPE, L, t(4, 8, dt=np.int32), t(8, 16, dt=np.int32), None, n, None, None, t(4, 16, dt=np.int32))
    refused(abi.E_DTYPE, L, x, w, t(16, dt=f16), n, None, None, y)
    refused(abi.E_DTYPE, L, x, w, None, n, None, None, t(4, 16, dt=f16))
    refused(abi.E_SHAPE, L, x, t(9, 16), None, n, None, None, y)
    refused(abi.E_SHAPE, L, x, w, t(15), n, None, None, y)
    refused(abi.E_SHAPE, L, x, w, None, n, None, None, t(5, 16))
    refused(abi.E_SHAPE, L, x, w, None, n, t(1, 16), None, y)
    refused(abi.E_SHAPE, L, x, w, None, n, None, t(16, 4), y)
    refused(abi.E_SHAPE, L, x, t(2, 8, 16), None, n, None, None, y)
    refused(abi.E_SHAPE, L, abi.make_desc(kept[0].data_ptr(), abi.F32, ()), w, None, n, None, None, y)
    refused(abi.E_INVALID, L, x, w, None, 5, None, None, y)
    refused(abi.E_INVALID, L, x, w, None, -1, None, None, y)
    refused(abi.E_INVALID, L, x, w, None, n, None, None, y, abi.MM_FP16_F32ACC)
    refused(abi.E_INVALID, L, x, w, None, n, None, None, y, abi.MM_FP32_3XTF32)
    big = hold(empty((8, 32), f32))
    refused(abi.E_UNSUPPORTED, L, x, w, None, n, None, None, d(big[:4, :16]))
    three = hold(empty((2, 3, 8), f32)).transpose(0, 1)
    refused(abi.E_UNSUPPORTED, L, d(three[:2]), w, None, n, None, None, t(2, 2, 16))
    # overlaps: y over x, over the residual with a shift, over pre
    flat = hold(empty((400,), f32))
    at = lambda off, *s: abi.make_desc(flat.data_ptr() + 4 * off, abi.F32, s)  # noqa: E731
    refused(abi.E_INVALID, L, at(0, 4, 8), w, None, n, None, None, at(16, 4, 16))
    refused(abi.E_INVALID, L, x, w, None, n, at(0, 4, 16), None, at(16, 4, 16))
    refused(abi.E_INVALID, L, x, w, None, n, None, at(0, 4, 16), at(0, 4, 16))
    refused(abi.E_INVALID, L, x, at(0, 8, 16), None, n, None, None, at(100, 4, 16))
    refused(abi.E_SHAPE, G, x, w, t(8, 15), None, None, n, None, None, y)
    refused(abi.E_DTYPE, G, x, w, t(8, 16, dt=f16), None, None, n, None, None, y)
    h = [t(4, 8, dt=f16), t(8, 16, dt=f16), t(8, 16, dt=f16)]
    refused(abi.E_DTYPE, G, *h, t(16), t(16, dt=f16), n, None, None, t(4, 16, dt=f16))
    refused(abi.E_INVALID, G, x, w, t(8, 16), None, None, n, y, None, y)
    B, GB = ctx.linear_backward, ctx.gated_linear_backward
    refused(abi.E_INVALID, B, x, w, abi.ACT_GELU, None, y, t(4, 8), None, None)
    refused(abi.E_SHAPE, B, x, w, n, None, t(4, 15), t(4, 8), None, None)
    refused(abi.E_SHAPE, B, x, w, n, None, y, t(4, 9), None, None)
    refused(abi.E_SHAPE, B, x, w, n, None, y, None, t(16, 8), None)
    refused(abi.E_DTYPE, B, x, w, n, None, y, None, t(8, 16, dt=f16), None)
    refused(abi.E_INVALID, B, x, w, n, None, y, x, None, None)
    refused(abi.E_UNSUPPORTED, B, x, w, n, None, d(hold(empty((16, 4), f32)).t()), t(4, 8), None, None)
    dw = t(8, 16)
    refused(abi.E_INVALID, GB, x, w, t(8, 16), n, t(4, 16), t(4, 16), y, None, dw, dw)
    refused(abi.E_SHAPE, GB, x, w, t(8, 16), n, t(4, 16), t(4, 17), y, None, dw, None)


def test_refused_calls_leave_the_context_usable(ctx):
    c = Case(20, 16, 24, np.float32)
    y, pre = forward(ctx, c, "relu")
    check_forward(c, "relu", y, pre)
    ctx.synchronize()
