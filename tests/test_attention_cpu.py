"""The attention operators' part of the C ABI, without a GPU: constants, calls without a context, and the
binary64 gradients that the GPU's are compared with against differences."""
import ctypes
import re

import numpy as np
import pytest

from attention_reference import Attention, angles, rotary, rotary_backward, visible
from quasarml_b200 import abi


def test_pairings_match_the_header():
    defs = dict(re.findall(r"#define\s+QSML_ROTARY_(\w+)\s+(\d+)", open(abi.HEADER_PATH).read()))
    assert sorted(defs) == ["HALVES", "PAIRS"]
    for name, value in defs.items():
        assert getattr(abi, "ROTARY_" + name) == int(value)


@pytest.mark.parametrize("name", ["qsml_norm_rotary", "qsml_norm_rotary_backward", "qsml_attention",
                                  "qsml_attention_backward"])
def test_a_call_without_a_context_is_refused(name):
    lib = abi.load()
    t = abi.TDesc()
    args = []
    for kind in abi._SIGS[name][1][1:]:
        args.append(ctypes.byref(t) if kind is ctypes.POINTER(abi.TDesc) else None if hasattr(kind, "contents") else 0)
    assert getattr(lib, name)(None, *args) == abi.E_INVALID


def test_which_keys_are_seen():
    assert visible(3, 5, 3, 5, 2, 1).tolist() == [[True, True, True, False, False], [True, False, True, True, False],
                                                  [True, False, False, True, True]]
    assert visible(2, 2, 2, 1, 0, 0).tolist() == [[False, False], [True, False]]


@pytest.mark.parametrize("window,sinks", [(0, 0), (4, 0), (3, 2)])
def test_reference_gradients_of_attention(window, sinks):
    rng = np.random.RandomState(3)
    q, k, v, do = (rng.randn(n, 6) for n in (9, 12, 12, 9))
    seen = visible(9, 12, 9, 12, window, sinks)

    def forward(a, b, c):
        return Attention(a, b, c, seen, 0.4, np.float64).forward()
    o, _, lse, _ = forward(q, k, v)
    grads, _ = Attention(q, k, v, seen, 0.4, np.float64).backward(o, lse, do)
    for i, g in enumerate(grads):
        way = rng.randn(*g.shape)
        h = 1e-5
        x = [[a + s * h * way if n == i else a for n, a in enumerate((q, k, v))] for s in (1, -1)]
        diff = ((forward(*x[0])[0] - forward(*x[1])[0]) * do).sum() / (2 * h)
        assert abs(diff - (g * way).sum()) <= 1e-7 * np.abs(g * way).sum()


@pytest.mark.parametrize("pairs", [False, True])
def test_reference_gradients_of_norm_and_rotation(pairs):
    rng = np.random.RandomState(4)
    x, w, dy = rng.randn(5, 2, 8), 1 + 0.2 * rng.randn(8), rng.randn(5, 2, 8)
    t = angles(np.arange(10).reshape(5, 2), np.array([1.0, 0.3, 0.1]), [2, 1])
    dx, _, dw, _ = rotary_backward(x, w, 1e-6, t, pairs, dy)
    h = 1e-5
    for g, way, step in ((dx, rng.randn(5, 2, 8), 0), (dw, rng.randn(8), 1)):
        y = [rotary(x + (s * h * way if step == 0 else 0), w + (s * h * way if step == 1 else 0), 1e-6, t, pairs)[0] for s in (1, -1)]
        diff = ((y[0] - y[1]) * dy).sum() / (2 * h)
        assert abs(diff - (g * way).sum()) <= 1e-7 * np.abs(g * way).sum()
