"""GPU attention whose keys (backward: steps) are split into parts: odd numbers of rows, columns and parts, so that
nothing kept of a part lies on more than its own alignment; and which kernel takes which call."""
import numpy as np
import pytest

from helpers import d, dev
from test_gpu_attention import Case, DT, NAN, check_backward, check_forward, views

pytestmark = pytest.mark.gpu

ODD_FEW = [  # sq, sk, hq, hk, D, window, sinks; one query row or few, 3 or 5 parts
    (1, 300, 1, 1, 33, 0, 0), (1, 300, 1, 1, 1, 0, 0), (1, 600, 3, 1, 33, 0, 0), (3, 333, 1, 1, 7, 0, 0),
    (5, 300, 3, 3, 129, 0, 0), (1, 300, 5, 1, 255, 0, 0), (1, 2000, 1, 1, 33, 300, 3), (7, 600, 7, 1, 65, 0, 0),
]
ODD_TILES = [  # more rows: tiles, 3 or 5 parts of their steps
    (65, 65, 1, 1, 33, 0, 0), (65, 65, 1, 1, 1, 0, 0), (65, 160, 3, 1, 33, 0, 0), (97, 150, 1, 1, 95, 90, 2),
    (67, 150, 1, 1, 129, 0, 0), (71, 71, 3, 3, 255, 0, 0), (129, 129, 1, 1, 33, 20, 1),
]


@DT
@pytest.mark.parametrize("size", ODD_FEW, ids=str)
def test_few_queries_of_odd_sizes(ctx, dt, size):
    check_forward(ctx, Case(dt, *size))
    assert ctx.last_kernel() == "k_attention_join"  # there were parts


@DT
@pytest.mark.parametrize("size", ODD_TILES, ids=str)
def test_tiles_of_odd_sizes(ctx, dt, size):
    check_forward(ctx, Case(dt, *size))
    assert ctx.last_kernel() == "k_attention_join"


@DT
@pytest.mark.parametrize("size", ODD_FEW[:4] + ODD_TILES, ids=str)
def test_gradients_of_odd_sizes(ctx, dt, size):
    check_backward(ctx, Case(dt, *size))


@DT
@pytest.mark.parametrize("B", [3, 5])
def test_odd_sequences_of_ragged_lengths(ctx, dt, B):
    check_forward(ctx, Case(dt, 1, 600, 1, 1, 33, nk=[600, 1, 333, 0, 127][:B]))
    check_forward(ctx, Case(dt, 65, 97, 1, 1, 33, nq=[65, 1, 33, 0, 64][:B], nk=[97, 1, 33, 0, 70][:B]))


KEY_TILES = [  # several tiles of queries of several heads, in parts: of 4; of 8 (with sinks) and 3; of 2 (with sinks) and 1
    (1000, 1000, 4, 1, 64, 0, 0), (1000, 1000, 8, 1, 128, 200, 3), (700, 1100, 6, 2, 72, 130, 140),
    (900, 900, 4, 1, 64, 0, 0, [900, 300, 513], [900, 300, 513]),
    (600, 900, 8, 1, 128, 300, 1, [600, 500, 10], [900, 333, 600]),
]


@pytest.mark.parametrize("size", KEY_TILES, ids=str)
def test_steps_of_key_tiles_in_parts(ctx, size):
    """A part's steps begin and end within a head's tiles of queries."""
    check_backward(ctx, Case(np.float16, *size))
    assert ctx.last_kernel() == "k_attention_dkv_join"


def kernels(ctx, c, permuted=False, off=0):
    """The last kernels of a forward and a backward call."""
    import torch
    q, k, v = views(ctx, c, permuted, off) if c.sq == c.sk else (dev(x) for x in (c.q, c.k, c.v))
    o, lse, do = dev(np.zeros_like(c.q)), torch.zeros(c.B, c.hq, c.sq, device="cuda"), dev(c.do)
    ctx.attention(d(q), d(k), d(v), d(o), lse=d(lse), **c.how())
    forward = ctx.last_kernel()
    out = [torch.full(x.shape, NAN, dtype=x.dtype, device="cuda") for x in (q, k, v)]
    ctx.attention_backward(d(q), d(k), d(v), d(o), d(lse), d(do), *[d(x) for x in out], **c.how())
    backward = ctx.last_kernel()
    ctx.synchronize()
    return forward, backward


@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("permuted,off", [(True, 0), (False, 0), (False, 8)])
def test_tensor_cores_take_views_on_16_bytes(ctx, D, permuted, off):
    assert kernels(ctx, Case(np.float16, 150, 150, 4, 2, D, 60, 2, B=2), permuted, off) == ("k_attention_tc", "k_attention_dkv")
    assert kernels(ctx, Case(np.float16, 4, 60, 4, 2, D)) == ("k_attention_few_tc", "k_attention_dkv")
    assert kernels(ctx, Case(np.float16, 1, 1000, 4, 2, D))[0] == "k_attention_join"


@pytest.mark.parametrize("dt,D,off", [(np.float32, 64, 0), (np.float16, 36, 0), (np.float16, 64, 1), (np.float16, 136, 0)])
def test_cuda_cores_take_the_others(ctx, dt, D, off):
    """One step a tile: nothing to join."""
    assert kernels(ctx, Case(dt, 30, 30, 4, 4, D), off=off) == ("k_attention_simt", "k_attention_bwd_simt")
    if off == 0:
        assert kernels(ctx, Case(dt, 4, 60, 4, 2, D))[0] == "k_attention_few"
    assert kernels(ctx, Case(dt, 150, 150, 4, 2, D), off=off) == ("k_attention_join", "k_attention_sum")
