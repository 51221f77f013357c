"""What the attention layer and its cache refuse, before anything is written."""
import pytest
import torch


@pytest.mark.parametrize("channels, heads", [(32, 8), (36, 3), (272, 2), (1, 1)])
def test_heads_that_the_kernels_do_not_take(channels, heads):
    from FGMS import nn
    with pytest.raises(ValueError, match="multiple of 8"):
        nn.VoxelAttention(channels, heads)


@pytest.mark.parametrize("sections", [(3, 3, 3), (9,), (-1, 4), (), (1, 1, 1, 1, 1)], ids=str)
def test_sections_that_do_not_fit(sections):
    from FGMS import nn
    with pytest.raises(ValueError, match="sections"):
        nn.VoxelAttention(64, 4, sections=sections)
    assert nn.VoxelAttention(64, 4, sections=(3, 0, 2)).sections == (3, 0, 2)
