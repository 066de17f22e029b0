"""Sizes and windows that a C int does not hold."""
import pytest
import torch

from my_nn_engine_b200 import ops


def test_windows_become_the_nearest_int():
    for x, want in ((0, 0), (-1, -1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31, 2 ** 31 - 1), (5 - 2 ** 32, 1 - 2 ** 31), (2 ** 40, 2 ** 31 - 1)):
        assert ops._nearest_int(x) == want


def test_more_pages_than_an_int_holds_are_refused():
    k, table, n = torch.zeros(1, 2, 16, 64).expand(2 ** 32 + 3, 2, 16, 64), torch.zeros(1, 5, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="pages"):
        ops.paged_attention(torch.zeros(1, 4, 1, 64), k, k, table, n, 1.0)
    with pytest.raises(ValueError, match="pages"):
        ops.paged_rotary_append(torch.zeros(1, 1, 8 * 64), n, table, k, k, 4)
