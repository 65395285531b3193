"""Host side of the drafted-token step at its edges (no GPU needed)."""

import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT


def test_tree_work_list_refuses_batches_whose_last_tile_passes_32_bits():
    """A key's number in an item, its drafted tokens and the tile's end included, is an int32."""
    from akv_b200.context_tree import tree_work_list

    for keys, new in ((2**31 - 1, 1), (2**31 - 64, 64), (2**31 - 150, 64)):
        with pytest.raises(ValueError, match="2\\^31"):
            tree_work_list([0, keys], [0, new], 8, 1, True, 1)
    items, *_ = tree_work_list([0, 2**31 - 400], [0, 64], 8, 1, True, 1)
    assert items.dtype == np.int32 and (items[:, 4] >= 0).all() and (items[:, 5] > items[:, 4]).all()
    assert items[:, 5].max() == 2**31 - 336
