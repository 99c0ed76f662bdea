"""kvattn_paged_decode_tree at the ends of its ranges, without a GPU."""
import pytest

from test_tree_cpu import TREE, _status


@pytest.mark.parametrize("kw", [
    dict(B=65535, NH=16, num_tokens=65535 * 16, max_new=16, max_pages=1 << 17), dict(B=8192, NH=25, num_tokens=600000, max_new=256, mask_words=4,
                                                                                      max_pages=1 << 10),
    dict(B=5000, NH=200, num_tokens=60000, max_new=64, max_pages=1 << 14), dict(B=60000, NH=16, num_tokens=60000, max_new=16, max_pages=1 << 17)])
def test_many_heads_with_long_tables_are_taken(kw):
    """The segments that the library picks fit a grid (refused here for the missing workspace alone)."""
    assert _status("kvattn_paged_decode_tree", TREE, S=0, **kw) == 7


def test_more_heads_than_a_grid_holds():
    kw = dict(B=65535, NH=20, num_tokens=800000, max_new=256, mask_words=4, max_pages=64)
    assert _status("kvattn_paged_decode_tree", TREE, S=0, **kw) == 4
