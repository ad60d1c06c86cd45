"""qk_norm_rotary's arguments: results in place, the first position."""
import pytest
import torch

from sandmuon_amd.attention import qk_norm_rotary, rotary_tables

pytestmark = pytest.mark.gpu


def test_out_over_other_operands_is_refused(device):
    cos, sin = rotary_tables(8, 16, device=device)
    q, k = torch.randn(1, 4, 2, 16, device=device), torch.randn(1, 4, 2, 16, device=device)
    both = torch.randn(1, 8, 2, 16, device=device)
    for a, b, out in ((q, k, (k, q)), (q, k, (q, q)), (both[:, :4], k, (both[:, 1:5], k))):
        with pytest.raises((RuntimeError, ValueError)):
            qk_norm_rotary(a, b, None, None, cos, sin, out=out)
    # halves of one buffer, in place, are fine
    fused = torch.randn(1, 4, 2, 2, 16, device=device)
    want = qk_norm_rotary(fused[:, :, 0], fused[:, :, 1], None, None, cos, sin)
    a, b = fused[:, :, 0], fused[:, :, 1]
    got = qk_norm_rotary(a, b, None, None, cos, sin, out=(a, b))
    assert torch.equal(got[0], want[0]) and torch.equal(fused[:, :, 1], want[1])
