"""GPU attention's gradients: what a sequence, a kv head or a query head holds is kept out of the others' gradients,
and sizes that differ between them cost no bits."""
import numpy as np
import pytest

from helpers import d, dev, host
from attention_reference import F64
from test_gpu_attention import Case, DT, NAN, check_backward

pytestmark = pytest.mark.gpu


def gradients(ctx, c):
    """dq, dk, dv with the forward pass's own o and lse."""
    import torch
    q, k, v, do = (dev(x) for x in (c.q, c.k, c.v, c.do))
    o, lse = torch.zeros_like(q), torch.zeros(c.B, c.hq, c.sq, device="cuda")
    ctx.attention(d(q), d(k), d(v), d(o), lse=d(lse), **c.how())
    out = [torch.full_like(x, NAN) for x in (q, k, v)]
    ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in out], **c.how())
    ctx.synchronize()
    return [host(x) for x in out]


def scaled(x, at, factor):
    x[at] = (x[at].astype(F64) * factor).astype(x.dtype)


@DT
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("small,large", [(1e-3, 1e3), (1e-4, 1.0)])
def test_sequences_of_different_sizes(ctx, dt, D, small, large):
    c = Case(dt, 300, 300, 2, 1, D, B=2)
    scaled(c.do, np.s_[0], small)
    scaled(c.do, np.s_[1], large)
    check_backward(ctx, c)
    c = Case(dt, 300, 300, 2, 1, D, B=2)
    scaled(c.do, np.s_[:], small)
    scaled(c.v, np.s_[1], 3e3)
    check_backward(ctx, c)


@DT
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("apart", [2, 1])
def test_heads_of_different_sizes(ctx, dt, D, apart):
    """apart 2: the query heads of two kv heads; 1: those of one."""
    c = Case(dt, 300, 300, 4, 2, D, 200, 1)
    scaled(c.do, np.s_[:, :, ::2] if apart == 1 else np.s_[:, :, :2], 1e-3)
    scaled(c.do, np.s_[:, :, 1::2] if apart == 1 else np.s_[:, :, 2:], 1e3)
    check_backward(ctx, c)


@DT
@pytest.mark.parametrize("D", [64, 128, 36])
@pytest.mark.parametrize("bad", [1e3, np.inf, -np.inf, NAN])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
def test_sequences_keep_their_bits(ctx, dt, D, which, bad):
    """Whatever one sequence holds, numbers or not, the other's gradients are the same bits."""
    def case():
        c = Case(dt, 200, 200, 2, 1, D, B=2)
        scaled(c.do, np.s_[:], 1e-3)
        return c
    want = [x[0] for x in gradients(ctx, case())]
    assert all(np.isfinite(x).all() and x.any() for x in want)
    c = case()
    getattr(c, which)[1, 100, 0] = bad
    for x, w in zip(gradients(ctx, c), want):
        assert np.array_equal(x[0], w)


@DT
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [1e3, np.inf, NAN])
def test_heads_keep_their_bits(ctx, dt, D, bad):
    """As above for kv heads, and for dq of the query heads of one kv head."""
    def case():
        c = Case(dt, 200, 200, 4, 2, D)
        scaled(c.do, np.s_[:], 1e-3)
        return c
    want = gradients(ctx, case())
    for which in ("k", "v"):
        c = case()
        getattr(c, which)[0, 100, 1] = bad
        got = gradients(ctx, c)
        assert np.array_equal(got[0][:, :, :2], want[0][:, :, :2])
        assert np.array_equal(got[1][:, :, 0], want[1][:, :, 0]) and np.array_equal(got[2][:, :, 0], want[2][:, :, 0])
    c = case()
    c.do[0, 100, 3] = bad
    got = gradients(ctx, c)
    assert np.array_equal(got[0][:, :, :3], want[0][:, :, :3])
    assert np.array_equal(got[1][:, :, 0], want[1][:, :, 0]) and np.array_equal(got[2][:, :, 0], want[2][:, :, 0])


@DT
def test_what_no_query_sees_costs_no_bits(ctx, dt):
    """Values before the window and gradients of queries before the first key, infinite and in tiles of their own."""
    c = Case(dt, 100, 700, 2, 1, 64, 64)
    scaled(c.do, np.s_[:], 1e-4)
    want = gradients(ctx, c)
    c.v[:, :400] = np.inf
    for x, w in zip(gradients(ctx, c), want):
        assert np.array_equal(x, w)
    c = Case(dt, 300, 100, 2, 1, 64)
    scaled(c.do, np.s_[:], 1e-4)
    want = gradients(ctx, c)
    c.do[:, :128] = 6e4
    for x, w in zip(gradients(ctx, c), want):
        assert np.array_equal(x, w)
