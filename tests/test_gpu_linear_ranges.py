"""Linear layers at the ends of their types' ranges, against binary64: gradients far above and far
below 1, activations far out, sums of a million terms of one sign, binary32 operands far from 1.

The bounds are those of test_gpu_linear.py's docstring, with U = 2^-24, unless a test says more."""
import numpy as np
import pytest

from helpers import dev, empty, host
from quasarml_b200 import abi, datagen
from test_gpu_linear import ACT, DTYPES, F64, STEP, TINY, U, Case, act64, act_error, backward, d, near

pytestmark = pytest.mark.gpu


def check_scaled(c, act, kept, dx, dw, db):
    """test_gpu_linear.py's check of a binary16 backward pass, but for dz's rounding between its
    computation and the products: 2^-11 of each element (in two parts 2^-21), or 2^-33 of the
    largest element of all (dg and du together), whichever is more."""
    x, dy = c.x.astype(F64), c.dy.astype(F64)
    z = kept[0].astype(F64)
    a, g = act64(z, act)
    ea = act_error(z, act, c.dt)
    if c.nw == 2:
        u = kept[1].astype(F64)
        dz, ez = [dy * u * g, dy * a], [np.abs(dy * u) * 4 * ea, np.abs(dy) * ea]
    else:
        dz, ez = [dy * g], [np.abs(dy) * 4 * ea]
    ez = [e + 4 * U * np.abs(v) for e, v in zip(ez, dz)]
    for v, e, o in zip(dz, ez, db):
        near(o, v.sum(0), e.sum(0) + (c.m + 40) * U * np.abs(v).sum(0), "db")
    floor = 2.0 ** -33 * max(np.abs(v).max() for v in dz)
    step = 2.0 ** -21 if c.m * c.n <= 65536 else STEP[c.dt]
    ez = [e + step * (np.abs(v) + e) + floor for e, v in zip(ez, dz)]
    w = [v.astype(F64) for v in c.w]
    ref = sum(v @ m.T for v, m in zip(dz, w))
    mag = sum((np.abs(v) + e) @ np.abs(m).T for v, e, m in zip(dz, ez, w))
    near(dx, ref, sum(e @ np.abs(m).T for e, m in zip(ez, w)) + (c.nw * c.n + 100) * U * mag, "dx")
    ax = np.abs(x).T
    for v, e, o in zip(dz, ez, dw):
        near(o, x.T @ v, ax @ e + (c.m + 100) * U * (ax @ (np.abs(v) + e)), "dw")


def times(a, p):
    return (a.astype(np.float32) * 2.0 ** p).astype(a.dtype)


# dy far above 1 (with x and w small, so that dx and dw are numbers of binary16), far below 1 (with
# x and w large); dz in two parts, in one, products by pairs of SMs
@pytest.mark.parametrize("size", [(100, 72, 200), (700, 264, 520), (2200, 136, 2500)])
@pytest.mark.parametrize("act", ["gelu", "silu", "relu"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("up", [12, 0, -14, -20])
def test_gradients_far_from_1(ctx, size, act, gated, up):
    c = Case(*size, np.float16, gated=gated)
    kept = c.kept()
    c.dy = times(c.dy, up)
    if gated and up > 0:
        kept[1] = times(kept[1], 5)
    shift = {12: -12, 0: 0, -14: 5, -20: 8}[up]
    c.x, c.w = times(c.x, shift), [times(w, shift + (3 if up < 0 else 0)) for w in c.w]
    check_scaled(c, act, kept, *backward(ctx, c, act, kept))


@pytest.mark.parametrize("size", [(60, 64, 96), (700, 264, 520)])
@pytest.mark.parametrize("gated", [False, True])
def test_gradients_of_zeros_and_of_one_large_row(ctx, size, gated):
    """dy 0 but for one row: of ordinary size, or far above the others."""
    for rest, row in ((0.0, 1.0), (2.0 ** -10, 2.0 ** 11), (0.0, 0.0)):
        c = Case(*size, np.float16, gated=gated)
        kept = c.kept()
        c.dy = (c.dy * np.float16(rest)).astype(np.float16)
        c.dy[size[0] // 2] = datagen.normal(9, (size[2],), 0, row).astype(np.float16) if row else 0
        c.x, c.w = times(c.x, -6), [times(w, -6) for w in c.w]
        check_scaled(c, "silu", kept, *backward(ctx, c, "silu", kept))


@pytest.mark.parametrize("size", [(60, 64, 96), (700, 264, 520)])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_a_gradient_that_is_no_number_stays_in_its_row(ctx, size, bad):
    """dx's other rows and dw's other columns are those of the rest, which lies far above 1 or below."""
    for up in (0, 12, -14):
        c = Case(*size, np.float16, gated=True)
        kept = c.kept()
        c.dy = times(c.dy, up)
        if up > 0:
            kept[1] = times(kept[1], 5)
        c.x, c.w = times(c.x, -up // 2 - 4), [times(w, -up // 2 - 4) for w in c.w]
        dx, dw, db = backward(ctx, c, "silu", kept)
        c.dy[7, 11] = bad
        bx, bw, bb = backward(ctx, c, "silu", kept)
        rows, cols = np.arange(size[0]) != 7, np.arange(size[2]) != 11
        assert not np.isfinite(bx[7]).any()
        assert np.array_equal(bx[rows], dx[rows])
        for p, q in zip(bw, dw):
            assert not np.isfinite(p[:, 11]).any()
            assert np.array_equal(p[:, cols], q[:, cols])
        for p, q in zip(bb, db):
            assert not np.isfinite(p[11]) and np.array_equal(p[cols], q[cols])


def test_scale_of_a_captured_gradient(ctx):
    """A captured backward pass finds the scale of each replay's dz, not the capture's."""
    import torch
    c = Case(700, 264, 520, np.float16, gated=True)
    kept = c.kept()
    c.x, c.w = times(c.x, -12), [times(w, -12) for w in c.w]  # 2^-4 left dw of dz near 2^17 beyond 65504
    t = [dev(v) for v in (c.x, c.w[0], c.w[1], kept[0], kept[1], c.dy)]
    out = [empty(s, np.float16) for s in ((c.m, c.k), (c.k, c.n), (c.k, c.n))]
    db = [empty((c.n,), np.float32) for _ in range(2)]
    stream, before, graph = torch.cuda.Stream(), ctx.stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            ctx.gated_linear_backward(*(d(v) for v in t[:3]), abi.ACT_SILU, *(d(v) for v in t[3:]),
                                      *(d(v) for v in out), *(d(v) for v in db))
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(before)
    dy, u = c.dy, kept[1]
    for up, more in ((0, 0), (12, 5), (-10, 0), (0, 0)):
        c.dy, kept[1] = times(dy, up), times(u, more)
        t[5].copy_(torch.from_numpy(c.dy))
        t[4].copy_(torch.from_numpy(kept[1]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_scaled(c, "silu", kept, host(out[0]), [host(v) for v in out[1:]], [host(v) for v in db])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
def test_sigmoid_gradient_far_out(ctx, dt, gated):
    """sigmoid'(z) = p (1 - p) to a relative error, on both sides: exp carries a few u, binary16's fast
    one 2^-21 and 2^-24 |z| of its argument, and the sum and products 4 u more.  One row, so that the
    binary32 bias gradient is dz itself."""
    z = np.concatenate([np.linspace(-16, 16, 201), [-30.0, 30.0, -80.0, 80.0]])[None, :].astype(dt)
    n = z.shape[1]
    up = np.full((1, n), 3.0, dt)
    dy = np.full((1, n), 0.5, dt)
    x, w = np.ones((1, 8), dt), np.ones((8, n), dt)
    t = [dev(v) for v in (x, w, w, z, up, dy)]
    db = [empty((n,), np.float32) for _ in range(2)]
    if gated:
        ctx.gated_linear_backward(*(d(v) for v in t[:3]), abi.ACT_SIGMOID, *(d(v) for v in t[3:]), None, None, None,
                                  d(db[0]), d(db[1]))
    else:
        ctx.linear_backward(d(t[0]), d(t[1]), abi.ACT_SIGMOID, d(t[3]), d(t[5]), None, None, d(db[0]))
    z = z[0].astype(F64)
    p, q = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
    rel = 12 * U if dt == np.float32 else 2.0 ** -20 + 2.0 ** -23 * np.abs(z)
    want = p * q * (1.5 if gated else 0.5)
    assert np.all(np.abs(host(db[0]) - want) <= rel * want + 2.0 ** -126)
    if gated:
        assert np.all(np.abs(host(db[1]) - 0.5 * p) <= rel * p + 2.0 ** -126)


def test_gelu_gradient_far_out(ctx):
    """gelu' of a binary32 number whose square is beyond binary32 is 1 or 0."""
    z = np.array([[1e18, 2e19, 1e30, 3e38, -1e18, -2e19, -1e30, -3e38, 1e10, -1e10]], np.float32)
    n = z.shape[1]
    t = [dev(v) for v in (np.ones((1, 4), np.float32), np.ones((4, n), np.float32), z, np.full((1, n), 2, np.float32))]
    db = empty((n,), np.float32)
    ctx.linear_backward(d(t[0]), d(t[1]), abi.ACT_GELU, d(t[2]), d(t[3]), None, None, d(db))
    assert np.array_equal(host(db), np.where(z[0] > 0, 2, 0))


def uniform(seed, *shape, dt, scale=1.0):
    """Numbers in [1/2, 1] times scale."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.rand(shape, generator=g, device="cuda") * 0.5 + 0.5) * scale).to(dt)


def one_sign(out, ref, dt):
    """The mean relative error of sums of one sign, where roundings to nearest cancel.  A tensor-core
    accumulator is cut at each step of 8 terms, by less than 2^-23 of it, and stands for at most
    8192 terms of binary16: 1024 steps, the accumulator half its last value in the mean, 2^-14.
    binary32's main accumulator stands for 256 terms: 32 steps, 2^-19 at the most, 2^-20 in the mean;
    that of the lesser products (2^-7 of each operand, so 2^-6 of the sum) for 2048 terms of five products,
    1280 steps: 2^-6 2^-23 640 = 2^-19.7.  2^-18.8 in all.  A thousandth of 2^-11 for binary16's own roundings,
    of which there are thousands."""
    import torch
    e = float((out.double() / ref - 1).mean())
    assert abs(e) <= (2.0 ** -14 + 2.0 ** -11 / 64 if dt == torch.float16 else 2.0 ** -18.8), e


# few tiles, whose sums are shared out over clusters, and pairs of SMs
@pytest.mark.parametrize("m,k,n", [(2**20, 64, 72), (2**17, 2048, 2048)])
@pytest.mark.parametrize("half", [False, True])
def test_long_sums_of_one_sign(ctx, m, k, n, half):
    import torch
    dt = torch.float16 if half else torch.float32
    x, dy = uniform(1, m, k, dt=dt), uniform(2, m, n, dt=dt, scale=2.0 ** -5)
    x *= 2.0 ** -5
    dw = torch.empty(k, n, dtype=dt, device="cuda")
    w = torch.zeros(k, n, dtype=dt, device="cuda")
    ctx.linear_backward(d(x), d(w), abi.ACT_NONE, None, d(dy), None, d(dw))
    ref = torch.zeros(k, n, dtype=torch.float64, device="cuda")
    for i in range(0, m, 2**16):
        ref += x[i:i + 2**16].double().t() @ dy[i:i + 2**16].double()
    one_sign(dw, ref, dt)
    # the forward product, of the transposes
    y = torch.empty(k, n, dtype=dt, device="cuda")
    ctx.linear(d(x.t()), d(dy), None, abi.ACT_NONE, None, None, d(y))
    assert torch.equal(y, dw)
    # two weights
    gate, up = torch.empty_like(y), torch.empty_like(y)
    ctx.gated_linear(d(x.t()), d(dy), d(dy), None, None, abi.ACT_RELU, d(gate), d(up), d(y))
    one_sign(gate, ref, dt)
    assert torch.equal(gate, up)
    # more terms than one accumulator takes by one block, and by a part of one
    for terms in (16384 + 64, 16384 + 3, 3 * 16384 + 100, 2048 + 1, 8192 + 8):
        ref = x[:terms].double().t() @ dy[:terms].double()
        ctx.linear_backward(d(x[:terms]), d(w), abi.ACT_NONE, None, d(dy[:terms]), None, d(dw))
        one_sign(dw, ref, dt)


def test_long_sums_of_a_gradient_in_two_parts(ctx):
    """dz of 40000 rows of one column, kept in two parts: both are in the sum."""
    import torch
    m, k, n = 40000, 16, 1
    x, dy = uniform(1, m, k, dt=torch.float16), uniform(2, m, n, dt=torch.float16)
    pre = uniform(3, m, n, dt=torch.float16)
    w, dw, db = torch.ones(k, n, dtype=torch.float16, device="cuda"), empty((k, n), np.float16), empty((n,), np.float32)
    ctx.linear_backward(d(x), d(w), abi.ACT_SIGMOID, d(pre), d(dy), None, d(dw), d(db))
    p = torch.sigmoid(pre.double())
    dz = dy.double() * p * (1 - p)
    ref = x.double().t() @ dz
    assert torch.all((dw.double() / ref - 1).abs() <= 2.0 ** -11 + 2.0 ** -13)
    assert torch.all((db.double() / dz.sum(0) - 1).abs() <= 2.0 ** -18)


# binary32 products of 17 rows and more run as three bf16 parts of each operand, cut: the parts are below
# |x|, 2^-7 |x| and 2^-15 |x|.  The dropped x1 w2, x2 w1 and x2 w2 are below 2^-21 |x w| together.
@pytest.mark.parametrize("rows", [17, 300])
def test_the_largest_dropped_products(ctx, rows):
    x = np.full((rows, 1), 1 + 2.0 ** -7 - 2.0 ** -23, np.float32)
    w = np.full((1, 40), 1 + 2.0 ** -7 - 2.0 ** -23, np.float32)
    y = empty((rows, 40), np.float32)
    tx, tw = dev(x), dev(w)
    ctx.linear(d(tx), d(tw), None, abi.ACT_NONE, None, None, d(y))
    want = float(x[0, 0]) * float(w[0, 0])
    assert np.all(np.abs(host(y) - want) <= (2.0 ** -21 + 2 * U) * want)


@pytest.mark.parametrize("size", [(1, 300, 40), (100, 300, 200), (300, 520, 136), (2200, 136, 2500)])
@pytest.mark.parametrize("px,pw", [(-60, 0), (-60, -40), (100, -90), (60, 60), (-100, 90), (-100, 10)])
def test_binary32_far_from_1(ctx, size, px, pw):
    """Operands of 2^px and 2^pw, none below 2^-110, so that all three parts are whole."""
    m, k, n = size
    x = datagen.normal(1, (m, k), 0, 1).astype(np.float32)
    w = datagen.normal(2, (k, n), 0, 1).astype(np.float32)
    x, w = (np.where(np.abs(v) < 2.0 ** -9, 0, v).astype(np.float32) for v in (x, w))
    x, w = np.ldexp(x, px), np.ldexp(w, pw)
    tx, tw, y = dev(x), dev(w), empty((m, n), np.float32)
    ctx.linear(d(tx), d(tw), None, abi.ACT_NONE, None, None, d(y))
    x, w = x.astype(F64), w.astype(F64)
    near(host(y), x @ w, (k + 100) * U * (np.abs(x) @ np.abs(w)) + 2.0 ** -126, "y")


@pytest.mark.parametrize("rows", [3, 17, 300])
def test_infinite_binary32_operands(ctx, rows):
    """An infinite x is an infinity or, beside a w that fewer than three parts hold, no number; it
    stays in its row.  The CUDA cores give the infinity."""
    k, n = 24, 40
    x = datagen.normal(1, (rows, k), 0, 1).astype(np.float32)
    w = datagen.normal(2, (k, n), 0, 1).astype(np.float32)
    w[5, ::2] = 1.5
    want = x.astype(F64) @ w.astype(F64)
    x[1, 5] = np.inf
    tx, tw = dev(x), dev(w)
    for precision in (abi.MM_AUTO, abi.MM_FP32_FFMA):
        y = empty((rows, n), np.float32)
        ctx.linear(d(tx), d(tw), None, abi.ACT_NONE, None, None, d(y), precision)
        y = host(y)
        rest = np.arange(rows) != 1
        near(y[rest], want[rest], (k + 100) * U * (np.abs(np.where(np.isinf(x), 0, x)) @ np.abs(w))[rest], "y")
        inf = np.sign(w[5]) * np.inf
        if rows == 3 or precision == abi.MM_FP32_FFMA:
            assert np.array_equal(y[1], inf)
        else:
            assert np.all(np.isnan(y[1]) | (y[1] == inf)) and not np.isfinite(y[1]).any()
