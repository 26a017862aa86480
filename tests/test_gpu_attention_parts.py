"""GPU attention whose keys (backward: steps) are split into parts: odd numbers of rows, columns and parts, so that
nothing kept of a part lies on more than its own alignment."""
import numpy as np
import pytest

from test_gpu_attention import Case, DT, check_backward, check_forward

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
