"""Key ranges of sequences near the longest that a table can have (csrc/kq4_kv.h, compiled for the host)."""
import pytest

from test_kv_layout import ints, lib  # noqa: F401


@pytest.mark.parametrize("length", [(1 << 30) + 5, (1 << 31) - 65536])
@pytest.mark.parametrize("chunk", [64, 1 << 20, 1 << 29, 1 << 30])
@pytest.mark.parametrize("ns", [1, 2, 3, 1024])
def test_ranges_near_2_to_the_31(lib, length, chunk, ns):  # noqa: F811
    o = ints(2)
    used = lib.t_ranges(1, length - 1, length, 0, 0, 0, chunk, ns, o)
    assert list(o) == [0, length] and used == min(ns, -(-length // chunk))
