"""What a step of several new tokens does with requests that it cannot take: pages that run out, bounds that are passed, rows without
tokens -- through the slot maps, the attention and the layer."""
import pytest
import torch

from lsvd_b200 import _lib
from test_gpu_chunk import _check_maps, _maps_case, _run_maps

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("in_place", [False, True])
def test_a_free_list_without_entries_has_run_out(in_place):
    """It is not a missing one: entries that need a page are refused, the others get their slots, nothing is overwritten."""
    c = _maps_case(4, 16, [2, 3, 20, 5], [0, 10, 20, 32])
    c["free"], c["head"] = [], 0
    _check_maps(c, refused=[0, 2, 3], in_place=in_place)
    _check_maps(c, refused=[0, 2, 3], rebuild=True, in_place=in_place)
    c["head"] = 3                                          # and a head behind its end is no place in it
    _check_maps(c, refused=[0, 2, 3], in_place=in_place)
    got, table, _, status = _run_maps(c)
    assert status == _lib.ERR_BOUNDS and table == c["table"] and got[4] == [3]
