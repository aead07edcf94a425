"""Arguments of the 4-bit cache's calls that leave Python by ctypes, which takes numbers as they wrap."""

from __future__ import annotations

import pytest

from test_paged import heads, stub


def test_rotate_refuses_a_first_position_of_more_than_32_bits():
    vm = stub()
    for pos in (2 ** 31, -2 ** 31 - 1, 2 ** 64, 2 ** 64 + 5, -2 ** 70):
        with pytest.raises(ValueError):
            vm.rotate_heads(heads(6, 4), None, pos)
    assert vm.lib.seen == []
    for pos in (2 ** 31 - 6, -2 ** 31, 0):
        vm.rotate_heads(heads(6, 4), None, pos)
    assert vm.lib.seen == ["fdllm_rotate_heads"] * 3
