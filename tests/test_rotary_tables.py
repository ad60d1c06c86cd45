"""rotary_tables on the CPU."""
import pytest
import torch

from sandmuon_amd.attention import rotary_tables


def test_angles_and_refusals():
    cos, sin = rotary_tables(5, 6, base=100.0, device="cpu")
    angle = torch.arange(5, dtype=torch.float64)[:, None] * 100.0 ** (-torch.tensor([0, 2, 4], dtype=torch.float64) / 6)
    assert torch.equal(cos, angle.cos().float()) and torch.equal(sin, angle.sin().float())
    assert rotary_tables(3, 0, device="cpu")[0].shape == (3, 0)
    for positions, rot in ((5, 7), (5, -2), (-1, 4)):  # (7 elements make no pairs)
        with pytest.raises(ValueError):
            rotary_tables(positions, rot, device="cpu")
