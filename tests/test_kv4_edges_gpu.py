"""The 4-bit paged KV cache at inputs on the edge of what it takes."""
import math

import pytest
import torch

import kv4_ref as R
import kv4_tight as T
from test_kv4_gpu import BF, FP, _dev, _run, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [-1, -4, -(1 << 31)])
def test_page_release_with_a_negative_count(dip, count):
    """It counts as an empty list: nothing is written before the list."""
    room = _dev([77] * 8 + [-1] * 6 + [77] * 4)
    free, fc = room[8:14], _dev([count])
    lens, table = _dev([33, 5]), _dev([[4, 9, 2, -1], [7, -1, -1, -1]])
    dip.page_release(_dev([True, False], torch.bool), lens, table, free, fc, 16)
    assert room.tolist() == [77] * 8 + [4, 9, 2, -1, -1, -1] + [77] * 4
    assert fc.tolist() == [3] and lens.tolist() == [0, 5]
    assert table.tolist() == [[-1] * 4, [7, -1, -1, -1]]


def test_page_release_past_the_capacity(dip):
    room = _dev([77] * 2 + [3, -1] + [77] * 4)
    free, fc = room[2:4], _dev([1])
    lens, table = _dev([33]), _dev([[4, 9, 2]])
    dip.page_release(_dev([True], torch.bool), lens, table, free, fc, 16)
    assert room.tolist() == [77, 77, 3, 4] + [77] * 4 and fc.tolist() == [2]
