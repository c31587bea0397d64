"""What the copies of cache blocks take for a pair."""
import pytest
import torch

from ml_framework_b200.ops import native


@pytest.mark.parametrize("pairs", [[(0, 1, 2), (3,)], [(3,), (0, 1, 2)], [(0, 1), (2, 3, 0), (1,)], [(), (0, 1, 2, 3)], [(0, 1, 2)], [(0,)]])
def test_entries_that_are_no_pairs_are_refused(pairs):
    """Also where their numbers add up to two for each entry."""
    with pytest.raises(ValueError, match="block numbers"):
        native.kv_copy_blocks_([torch.zeros(4, 2)], pairs)


def test_no_pairs_is_nothing_to_do():
    t = torch.arange(8.0).view(4, 2)
    native.kv_copy_blocks_([t], [])
    native.kv_copy_blocks_([], [(0, 1)])
    assert torch.equal(t, torch.arange(8.0).view(4, 2))
