"""GPU layer norm backward pass (through the C ABI) against binary64.

Tolerances count roundings.  With u = 2^-24 (binary32) and n columns, every dx
element is rstd * (h - c1 - xh * c2): its terms are rounded a few times each,
the sums along the row are at most 32 + 10 additions deep at these widths (a thread's
elements one after another, then two trees of 32; cols / 512 + 10 in the
kernel for the widest rows, whose bound is wider by that, and mean, variance and rstd carry at most
as many.  So |dx - ref| <= 60 u * rstd * (|h| + |c1| + |xh| |c2| + mean(|h|) + |xh| mean(|h xh|)
+ |xh| |c2|) plus half a step of the output type, 60 being 42 for the sums and 18 for the single roundings.
x itself is exact, and x - mean is off by u |x| + the mean's error, which
moves xh by at most 60 u * rstd * max|x|: that factor is added to the relative bound.
dgamma and dbeta sum over rows in at most rows / CTAs + 40 steps:
|err| <= (60 + rows / 148) u * sum |terms|, plus xh's error, plus half a step."""
import numpy as np
import pytest
import torch

from helpers import d, dev, empty, host
from quasarml_b200 import abi, datagen

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
STEP = {np.float32: 2.0 ** -24, np.float16: 2.0 ** -11}
TINY = {np.float32: 2.0 ** -149, np.float16: 2.0 ** -25}


def reference(x, g, dy, eps):
    x, g, dy = (v.astype(np.float64) for v in (x, g, dy))
    n = x.shape[-1]
    mean = x.sum(-1, keepdims=True) / n
    var = ((x - mean) ** 2).sum(-1, keepdims=True) / n
    rstd = 1.0 / np.sqrt(var + np.float64(np.float32(eps)))
    xh, h = (x - mean) * rstd, dy * g
    c1, c2 = h.sum(-1, keepdims=True) / n, (h * xh).sum(-1, keepdims=True) / n
    dx = rstd * (h - c1 - xh * c2)
    shift = 1.0 + rstd * np.abs(x).max(-1, keepdims=True)  # xh's own relative error, in units of 60 u
    mag = rstd * (np.abs(h) + np.abs(h).sum(-1, keepdims=True) / n
                  + 2 * (np.abs(xh) + 1) * np.abs(h * (np.abs(xh) + 1)).sum(-1, keepdims=True) / n) * shift
    return dx, (dy * xh), dy, mag, np.abs(dy) * (np.abs(xh) + 1) * shift


def check(x, g, dy, eps, dx, dg, db):
    rdx, tg, tb, mag, gmag = reference(x, g, dy, eps)
    rows, n = int(np.prod(x.shape[:-1])), x.shape[-1]
    flat = lambda v: v.reshape(rows, -1)  # noqa: E731
    if dx is not None:
        s = STEP[dx.dtype.type]
        bound = (60 + n / 512) * U * mag + s * np.abs(rdx) + TINY[dx.dtype.type]
        assert np.all(np.abs(dx.astype(np.float64) - rdx) <= bound)
    for out, terms, m in ((dg, tg, gmag), (db, tb, np.abs(tb))):
        if out is None:
            continue
        ref, s = flat(terms).sum(0), STEP[out.dtype.type]
        bound = (60 + rows / 148) * U * flat(m).sum(0) + s * np.abs(ref) + TINY[out.dtype.type]
        assert np.all(np.abs(out.astype(np.float64) - ref) <= bound)


def run(ctx, x, g, dy, eps=1e-5, want=(True, True, True), pdt=np.float32):
    n = x.shape[-1]
    out = [empty(x.shape, x.dtype), empty((n,), pdt), empty((n,), pdt)]
    for t in out:
        t.fill_(float("nan"))
    args = [d(t) if w else None for t, w in zip(out, want)]
    tx, tg, tdy = dev(x), dev(g), dev(dy)
    ctx.layer_norm_backward(d(tx), d(tg), d(tdy), eps, *args)
    return [host(t) if w else None for t, w in zip(out, want)]


def make(shape, dtype, seed=71, gdt=np.float32):
    x = datagen.normal(seed, shape, 0.5, 2.0).astype(dtype)
    g = datagen.normal(seed + 1, shape[-1:], 1.0, 0.1).astype(gdt)
    dy = datagen.normal(seed + 2, shape, 0.0, 1.0).astype(dtype)
    return x, g, dy


# one element, one row, one warp a row, widths that fill no load, the last width of each kernel
# and the first of the next, rows too wide for the registers
SHAPES = [(1, 1), (3, 2), (1, 8), (7, 33), (300, 64), (2, 5, 96), (19, 256), (1000, 512), (64, 520), (33, 1001),
          (5, 1537), (600, 1024), (9, 4096), (150, 4099), (4, 8192), (3, 8200), (2, 16384), (11, 9001),
          (700, 8200), (600, 12296), (450, 16384), (7, 40000), (300, 20000), (2, 70000)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_shapes(ctx, shape, dtype):
    x, g, dy = make(shape, dtype)
    check(x, g, dy, 1e-5, *run(ctx, x, g, dy))


@pytest.mark.parametrize("cols", [4095, 4097, 6143, 6145, 8191])
@pytest.mark.parametrize("rows", [2, 310])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_wide_rows_of_single_elements(ctx, rows, cols, dtype):
    x, g, dy = make((rows, cols), dtype)
    check(x, g, dy, 1e-5, *run(ctx, x, g, dy))


@pytest.mark.parametrize("gdt", [np.float32, np.float16])
@pytest.mark.parametrize("cols", [64, 4096, 8200, 16384])
def test_gamma_off_16_bytes(ctx, cols, gdt):
    x, g, dy = make((5, cols), np.float16, gdt=gdt)
    wide = dev(np.concatenate([g[:1], g]))
    out = [empty(x.shape, x.dtype), empty((cols,), np.float32), empty((cols,), np.float32)]
    tx, tdy = dev(x), dev(dy)
    ctx.layer_norm_backward(d(tx), d(wide[1:]), d(tdy), 1e-5, *[d(t) for t in out])
    check(x, g, dy, 1e-5, *[host(t) for t in out])


def test_workload_16384x4096_f16(ctx):
    x, g, dy = make((16384, 4096), np.float16)
    check(x, g, dy, 1e-5, *run(ctx, x, g, dy))


@pytest.mark.parametrize("cols", [64, 1001, 9000])
@pytest.mark.parametrize("want", [(True, False, False), (False, True, True), (False, True, False),
                                  (True, False, True)])
def test_only_what_is_asked_for(ctx, cols, want):
    x, g, dy = make((37, cols), np.float16, gdt=np.float16)
    check(x, g, dy, 1e-5, *run(ctx, x, g, dy, want=want, pdt=np.float16))


def test_large_mean_and_constant_rows(ctx):
    # the deviations are small against the mean; a constant row has rstd = eps^-1/2 and xh = 0
    x, g, dy = make((40, 1024), np.float32)
    x += 1000.0
    x[5] = 3.0
    check(x, g, dy, 1e-3, *run(ctx, x, g, dy, eps=1e-3))


@pytest.mark.parametrize("rows", [1, 3, 9, 200])
@pytest.mark.parametrize("cols", [24, 200, 1024])
def test_eps_zero(ctx, rows, cols):
    """Lanes and warps without a row have nothing to add, not 0 times an infinite rstd."""
    x, g, dy = make((rows, cols), np.float32)
    check(x, g, dy, 0.0, *run(ctx, x, g, dy, eps=0.0))


def test_widest_row(ctx):
    """2^31 - 1 columns.  x alternates 1, -1 and dy 1, 1, -1, -1: a thread's sums are
    whole numbers below 2^24, the means 0 to 2^-30, and with eps = 3, rstd = 1/2 and
    dx = dy / 2 to within 2^-28, which rounds to 1/2."""
    n = 2**31 - 1
    fill = lambda *v: torch.tensor(v, dtype=torch.float16, device="cuda").repeat(2**29)[:n]  # noqa: E731
    x, dy, g = fill(1, -1, 1, -1), fill(1, 1, -1, -1), fill(1, 1, 1, 1)
    dx = torch.zeros(n, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.layer_norm_backward(d(x), d(g), d(dy), 3.0, d(dx), None, None)
    ctx.synchronize()
    assert torch.equal(dx, dy.mul_(0.5))


def test_non_finite_rows_stay_in_their_rows(ctx):
    x, g, dy = make((6, 256), np.float32)
    x[2, 7] = np.inf
    dy[4, 9] = np.nan
    dx, dg, _ = run(ctx, x, g, dy)
    assert np.isnan(dx[2]).all() and np.isnan(dx[4]).all() and np.isfinite(dx[[0, 1, 3, 5]]).all()
    assert np.isnan(dg).all() or np.isnan(dg[9])


@pytest.mark.parametrize("cols", [128, 2048, 9000])
def test_unaligned_views_and_neighbours(ctx, cols):
    """Tensors that begin off a 16-byte boundary, inside a larger buffer whose other bytes stay."""
    import torch
    rows = 21
    x, g, dy = make((rows, cols), np.float16)
    buf = [torch.full((rows * cols + 16,), 7.0, dtype=torch.float16, device="cuda") for _ in range(3)]
    buf[0][3:3 + rows * cols] = dev(x).reshape(-1)
    buf[1][5:5 + rows * cols] = dev(dy).reshape(-1)

    def at(i, off):
        return abi.make_desc(buf[i].data_ptr() + 2 * off, abi.F16, (rows, cols))

    dg, db, tg = empty((cols,), np.float32), empty((cols,), np.float32), dev(g)
    ctx.layer_norm_backward(at(0, 3), d(tg), at(1, 5), 1e-5, at(2, 1), d(dg), d(db))
    out = host(buf[2])
    check(x, g, dy, 1e-5, out[1:1 + rows * cols].reshape(rows, cols), host(dg), host(db))
    assert np.all(out[:1] == 7.0) and np.all(out[1 + rows * cols:] == 7.0)


def test_no_rows_and_no_columns(ctx):
    dg, db = dev(np.ones(8, np.float32)), dev(np.ones(8, np.float16))
    e, tg = empty((0, 8), np.float16), dev(np.ones(8, np.float32))
    ctx.layer_norm_backward(d(e), d(tg), d(e), 1e-5, d(e), d(dg), d(db))
    assert np.all(host(dg) == 0) and np.all(host(db) == 0)
    e, z = empty((4, 0), np.float32), empty((0,), np.float32)
    ctx.layer_norm_backward(d(e), d(z), d(e), 1e-5, d(e), d(z), d(z))


@pytest.mark.parametrize("shape", [(500, 300), (257, 4096), (20, 9000)])
def test_same_bits_again(ctx, shape):
    x, g, dy = make(shape, np.float16)
    a, b = run(ctx, x, g, dy), run(ctx, x, g, dy)
    for p, q in zip(a, b):
        assert np.array_equal(p, q)


def test_against_differences(ctx):
    """The gradients against central differences of the forward formula in binary64: the truncation
    error of a step t is t^2 / 6 times the third derivative, here below 1e-6 of the loss's scale."""
    rng = np.random.default_rng(5)
    x, g, b, dy = rng.normal(size=(3, 24)), rng.normal(size=24), rng.normal(size=24), rng.normal(size=(3, 24))
    x, g, dy = (v.astype(np.float32) for v in (x, g, dy))
    dx, dg, db = run(ctx, x, g, dy, eps=1e-2)

    def loss(x, g, b):
        dv = x - x.mean(-1, keepdims=True)
        y = dv / np.sqrt((dv * dv).mean(-1, keepdims=True) + np.float64(np.float32(1e-2))) * g + b
        return float((y * dy.astype(np.float64)).sum())

    base = [x.astype(np.float64), g.astype(np.float64), b]
    for i, grad in enumerate((dx, dg, db)):
        for at in list(np.ndindex(*grad.shape))[::5]:
            t, v = 1e-4, [w.copy() for w in base]
            v[i][at] += t
            hi = loss(*v)
            v[i][at] -= 2 * t
            assert abs((hi - loss(*v)) / (2 * t) - grad[at]) <= 1e-5 * (1 + np.abs(grad).max())


def test_graph_replays_while_other_calls_run(ctx):
    """A captured call and eager calls of the same context do not share workspace."""
    import torch
    x, g, dy = make((333, 768), np.float16)
    x2, g2, dy2 = make((333, 768), np.float16, seed=90)
    tx, tg, tdy = dev(x), dev(g), dev(dy)
    outs = [empty(x.shape, np.float16), empty((768,), np.float32), empty((768,), np.float32)]
    want = run(ctx, x, g, dy)
    args = [d(tx), d(tg), d(tdy), 1e-5] + [d(t) for t in outs]
    stream = torch.cuda.Stream()
    before = ctx.stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        ctx.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            ctx.layer_norm_backward(*args)
    finally:
        torch.cuda.synchronize()
        ctx.set_stream(before)
    run(ctx, x2, g2, dy2)
    for _ in range(3):
        for t in outs:
            t.fill_(float("nan"))
        graph.replay()
        other = run(ctx, x2, g2, dy2)
        torch.cuda.synchronize()
        for t, w in zip(outs, want):
            assert np.array_equal(host(t), w)
        check(x2, g2, dy2, 1e-5, *other)


def refused(ctx, status, *a):
    with pytest.raises(abi.QsmlError) as e:
        ctx.layer_norm_backward(*a)
    assert e.value.status == status, e.value


def test_refusals(ctx):
    def t(*shape, dt=np.float32):
        return empty(shape, dt)

    x, dy, dx, g, dg = t(4, 32), t(4, 32), t(4, 32), t(32), t(32)
    half = t(4, 32, dt=np.float16)
    refused(ctx, abi.E_DTYPE, d(x), d(g), d(half), 1e-5, d(dx))
    refused(ctx, abi.E_DTYPE, d(x), d(g), d(dy), 1e-5, d(half))
    refused(ctx, abi.E_DTYPE, d(x), d(t(32, dt=np.float16)), d(dy), 1e-5, d(dx))
    refused(ctx, abi.E_DTYPE, d(x), d(g), d(dy), 1e-5, d(dx), d(t(32, dt=np.int32)))
    refused(ctx, abi.E_SHAPE, d(x), d(t(31)), d(dy), 1e-5, d(dx))
    refused(ctx, abi.E_SHAPE, d(x), d(g), d(t(4, 31)), 1e-5, d(dx))
    refused(ctx, abi.E_SHAPE, d(x), d(g), d(dy), 1e-5, d(t(32, 4)))
    refused(ctx, abi.E_SHAPE, d(x), d(g), d(dy), 1e-5, d(dx), d(t(33)))
    refused(ctx, abi.E_UNSUPPORTED, d(x.t()), d(t(4)), d(dy.t()), 1e-5, d(t(32, 4)))
    refused(ctx, abi.E_INVALID, d(x), d(g), d(dy), 1e-5, d(dy))
    refused(ctx, abi.E_INVALID, d(x), d(g), d(dy), 1e-5, d(dx), d(dg), d(dg))
    refused(ctx, abi.E_SHAPE, abi.make_desc(g.data_ptr(), abi.F32, ()), d(g), d(dy), 1e-5, None)


@pytest.mark.parametrize("shape", [(6, 256), (6, 1001), (6, 4096), (6, 9000)])
def test_column_sums_of_non_finite_rows(ctx, shape):
    """A row with an infinite x has no xh, so dgamma is no number anywhere; dbeta is dy's sum and has
    none only where dy has none."""
    x, g, dy = make(shape, np.float32)
    want = run(ctx, x, g, dy)
    dy[4, 9] = np.nan
    _, dg, db = run(ctx, x, g, dy)
    others = np.arange(shape[1]) != 9
    assert np.isnan(db[9]) and np.array_equal(db[others], want[2][others])
    x[2, 7] = np.inf
    _, dg, db = run(ctx, x, g, dy)
    assert np.isnan(dg).all()
    assert np.isnan(db[9]) and np.array_equal(db[others], want[2][others])
