"""Views of caches in 8 bits in Python, without a GPU."""
import pytest
import torch

import ellm_amd
from ellm_amd.attention import E4m3LayerView


@pytest.mark.parametrize("first", [0, 2])
def test_a_view_without_a_table_is_refused_as_one(first):
    """A cache with one capacity has no sequence table; its view in the place of one is refused with a reason, ahead of all else."""
    view = E4m3LayerView(None, (16, 16, 16, 16), [64 * 128, 64 * 128, 128, 1], None, first)
    x = torch.zeros((1, 2, 1, 128), dtype=torch.float16)
    with pytest.raises(ValueError, match="one capacity"):
        ellm_amd.Attention(x, x, x, x, 2, 1, 1, 128, view.strides, 1.0, seq_table=view, kv_scales=(x, x))
