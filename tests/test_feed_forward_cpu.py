"""The feed-forward operators' part of the C ABI, without a GPU: constants, and calls without a
context."""
import ctypes
import re

import pytest

from quasarml_b200 import abi


def test_activations_match_the_header():
    defs = dict(re.findall(r"#define\s+QSML_ACT_(\w+)\s+(\d+)", open(abi.HEADER_PATH).read()))
    assert sorted(defs) == ["GELU", "NONE", "RELU", "SIGMOID", "SILU"]
    for name, value in defs.items():
        assert getattr(abi, "ACT_" + name) == int(value)


@pytest.mark.parametrize("name", ["qsml_layer_norm_backward", "qsml_linear", "qsml_linear_backward",
                                  "qsml_gated_linear", "qsml_gated_linear_backward"])
def test_a_call_without_a_context_is_refused(name):
    lib = abi.load()
    t = abi.TDesc()
    args = []
    for kind in abi._SIGS[name][1][1:]:
        args.append(ctypes.byref(t) if hasattr(kind, "contents") else 0)
    assert getattr(lib, name)(None, *args) == abi.E_INVALID
