"""Forward-mode derivatives are refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from sandmuon_amd import losses
from sandmuon_amd.attention import qk_norm_rotary, rotary_tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(device, grad):
    cos, sin = rotary_tables(8, 16, device=device)
    z, y = torch.randn(2, 3, 40, device=device), torch.zeros(2, 3, dtype=torch.long, device=device)
    q, k, w = torch.randn(1, 4, 2, 16, device=device), torch.randn(1, 4, 1, 16, device=device), torch.ones(16, device=device)
    adv, ref = torch.ones(2, device=device), torch.zeros(2, 3, device=device)
    with torch.set_grad_enabled(grad), fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        calls = [lambda: losses.token_logprobs(dual(z), y), lambda: losses.policy_loss(dual(z), y, adv),
                 lambda: losses.preference_loss(dual(z), y, ref),
                 lambda: qk_norm_rotary(dual(q), k, w, w, cos, sin), lambda: qk_norm_rotary(q, dual(k), None, None, cos, sin),
                 lambda: qk_norm_rotary(q, k, dual(w), w, cos, sin), lambda: qk_norm_rotary(q, k, w, dual(w), cos, sin),
                 lambda: qk_norm_rotary(q, k, w, w, dual(cos), sin)]
        for call in calls:
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        # without a tangent, as ever
        assert losses.token_logprobs(z, y).shape == (2, 3)
        assert qk_norm_rotary(q, k, w, w, cos, sin)[0].shape == q.shape
