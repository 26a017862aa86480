"""The caching allocator gives out the block of a size that was freed last, whatever was freed between."""
import pytest

from quasarml_b200 import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [512, 100_000, 5 << 20])
def test_the_last_freed_of_a_size_is_given_out_first(size):
    c = abi.Context(0)
    a, b, other = c.alloc(size), c.alloc(size), c.alloc(8 * size)
    for first, last in ((a, b), (b, a)):
        c.free(first)
        c.free(other)
        c.free(last)
        assert c.alloc(size) == last and c.alloc(size) == first
        assert c.alloc(8 * size) == other
    for p in (a, b, other):
        c.free(p)
    s = c.allocator_stats()
    assert s["live_bytes"] == 0 and s["misses"] == 3
    c.close()
