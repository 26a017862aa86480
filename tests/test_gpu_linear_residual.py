"""The linear layer's residual as it may lie: rows with a pitch, one row for all of them, y itself; each with
the kernels that read it (CUDA cores, few rows, tiles with vectors, pairs and single columns, pairs
of SMs)."""
import numpy as np
import pytest

from helpers import dev, host
from quasarml_b200 import abi
from test_gpu_linear import ACT, DTYPES, Case, check_forward, d, nan

pytestmark = pytest.mark.gpu

# 8 columns together, pairs, single columns; one row, few, many, pairs of SMs
SIZES = [(1, 300, 264), (5, 64, 34), (9, 40, 33), (130, 72, 200), (200, 136, 70), (77, 64, 129), (300, 1000, 256),
         (2200, 136, 2504), (2200, 40, 2502), (2200, 40, 2501)]


def call(ctx, c, act, residual, y, pre, precision):
    tx, tw, tb = dev(c.x), dev(c.w[0]), dev(c.b[0])
    ctx.linear(d(tx), d(tw), d(tb), ACT[act], residual, None if pre is None else d(pre), d(y), precision)


def precisions(dt):
    return (abi.MM_AUTO, abi.MM_FP32_FFMA) if dt == np.float32 else (abi.MM_AUTO,)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("pitch", [1, 2, 8, 72])
def test_rows_with_a_pitch(ctx, size, dt, pitch):
    import torch
    for precision in precisions(dt):
        c = Case(*size, dt)
        big = torch.full((c.m, c.n + pitch), float("nan"), dtype=dev(c.r).dtype, device="cuda")
        big[:, :c.n] = dev(c.r)
        y, pre = nan((c.m, c.n), dt), nan((c.m, c.n), dt)
        call(ctx, c, "silu", d(big[:, :c.n]), y, pre, precision)
        check_forward(c, "silu", host(y), [host(pre)], True)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
def test_one_row_for_all(ctx, size, dt):
    for precision in precisions(dt):
        c = Case(*size, dt)
        row = dev(c.r[:1])
        c.r[:] = c.r[:1]
        y = nan((c.m, c.n), dt)
        call(ctx, c, "none", d(row.expand(c.m, c.n)), y, None, precision)
        check_forward(c, "none", host(y), [None], True)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("dt", DTYPES)
def test_in_place(ctx, size, dt):
    for precision in precisions(dt):
        c = Case(*size, dt)
        y, pre = dev(c.r), nan((c.m, c.n), dt)
        call(ctx, c, "gelu", d(y), y, pre, precision)
        check_forward(c, "gelu", host(y), [host(pre)], True)


@pytest.mark.parametrize("dt", DTYPES)
def test_off_16_bytes(ctx, dt):
    """Residual and y that begin one element past a boundary."""
    import torch
    for size in ((5, 64, 40), (130, 72, 200), (2200, 40, 2504)):
        c = Case(*size, dt)
        flat = [torch.full((c.m * c.n + 9,), 5.0, dtype=dev(c.r).dtype, device="cuda") for _ in range(2)]
        r, y = (f[1:1 + c.m * c.n].view(c.m, c.n) for f in flat)
        r.copy_(dev(c.r))
        call(ctx, c, "relu", d(r), y, None, abi.MM_AUTO)
        check_forward(c, "relu", host(y), [None], True)
        assert torch.all(flat[1][:1] == 5) and torch.all(flat[1][1 + c.m * c.n:] == 5)
