"""A position offset past 32 bits is refused, not cut to its lowest 32 (no GPU needed)."""
import pytest
import torch

import bnhip as B


@pytest.mark.parametrize("offset", [2 ** 31, -2 ** 31 - 1, 2 ** 32, 2 ** 32 + 7])
def test_offsets_past_32_bits_are_refused(offset):
    q, w = torch.zeros((3, 8, 64)), torch.zeros(64)
    with pytest.raises(ValueError, match="position_offset"):
        B.qk_norm_rope(q, None, w, None, position_offset=offset)
    with pytest.raises(ValueError, match="position_offset"):
        B.qk_norm_rope_backward(q, None, w, None, q, None, position_offset=offset)


@pytest.mark.parametrize("offset", [2 ** 31 - 1, -2 ** 31, 0])
def test_others_are_not(offset):
    q, w = torch.zeros((3, 8, 64)), torch.zeros(64)
    with pytest.raises(ValueError, match="not on a GPU"):
        B.qk_norm_rope(q, None, w, None, position_offset=offset)
