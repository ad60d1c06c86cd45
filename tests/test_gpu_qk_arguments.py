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


def test_out_raises_its_version(device):
    cos, sin = rotary_tables(8, 16, device=device)
    q, k = torch.randn(1, 4, 2, 16, device=device), torch.randn(1, 4, 2, 16, device=device)
    scale = torch.ones(16, device=device, requires_grad=True)
    y = q * scale  # saves q
    versions = q._version, k._version
    with torch.no_grad():
        qk_norm_rotary(q, k, None, None, cos, sin, out=(q, k))
    assert q._version > versions[0] and k._version > versions[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_out_that_requires_a_gradient(device):
    cos, sin = rotary_tables(8, 16, device=device)
    q, k = torch.randn(1, 4, 2, 16, device=device), torch.randn(1, 4, 2, 16, device=device)
    out = torch.empty_like(q).requires_grad_(), torch.empty_like(k)
    with pytest.raises(ValueError, match="out="):
        qk_norm_rotary(q, k, None, None, cos, sin, out=out)
    want = qk_norm_rotary(q, k, None, None, cos, sin)
    with torch.no_grad():
        assert torch.equal(qk_norm_rotary(q, k, None, None, cos, sin, out=out)[0], want[0])
    with torch.inference_mode():
        a, b = q.clone(), k.clone()
        qk_norm_rotary(a, b, None, None, cos, sin, out=(a, b))
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_first_position_is_a_whole_number(device):
    cos, sin = rotary_tables(8, 16, device=device)
    q = torch.randn(1, 2, 1, 16, device=device)
    with pytest.raises(TypeError):
        qk_norm_rotary(q, q, None, None, cos, sin, 2.5)
    want = qk_norm_rotary(q, q, None, None, cos, sin, torch.tensor([3, 4], device=device))
    assert torch.equal(qk_norm_rotary(q, q, None, None, cos, sin, 3)[0], want[0])
