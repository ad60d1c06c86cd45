"""What is no number among a live token's inputs reaches the policy loss and its
gradient, as the other losses'."""
import math

import pytest
import torch

from sandmuon_amd import losses

pytestmark = pytest.mark.gpu


def inputs(device, b, t, v, dtype, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    logits = (torch.randn(b, t, v, device=device, generator=g) * 2).to(dtype)
    targets = torch.randint(0, v, (b, t), device=device, generator=g)
    lp = torch.stack([torch.log_softmax(z.double(), 1).gather(1, y[:, None]).squeeze(1) for z, y in zip(logits, targets)])
    noise = lambda: torch.randn(b, t, device=device, generator=g)
    mask = torch.rand(b, t, device=device, generator=g) < 0.8
    return logits, targets, lp, (lp + 0.1 * noise()).float(), (lp + 0.3 * noise()).float(), noise(), mask


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [97, 4099])
def test_what_is_no_number_reaches_the_gradient(device, v, dtype):
    logits, targets, _, old, ref, _, _ = inputs(device, 3, 5, v, dtype, 3)
    adv = torch.tensor([0.7, -0.4, 0.2], device=device)
    outside = targets.clone()
    outside[0, 1], outside[1, 2] = -100, v
    spoilt = [(0, 1), (1, 2)]
    bad = torch.full_like(old, 0.0)
    bad[0, 1] = bad[1, 2] = math.nan
    spots = torch.zeros(3, 5, dtype=torch.bool, device=device)
    for at in spoilt:
        spots[at] = True
    whole = adv[:, None].expand(3, 5)
    for kw in (dict(targets=outside), dict(targets=outside, old_logprobs=old), dict(targets=outside, ref_logprobs=ref),
               dict(targets=outside, old_logprobs=old, ref_logprobs=ref), dict(old_logprobs=old + bad),
               dict(ref_logprobs=ref + bad), dict(advantages=whole + bad),
               dict(advantages=whole + bad, old_logprobs=old + 5)):
        kw = dict(dict(targets=targets, advantages=adv), **kw)
        leaf = logits.clone().requires_grad_()
        loss, lp = losses.policy_loss(leaf, kl_coef=0.1 if "ref_logprobs" in kw else 0.0, **kw)
        grad, = torch.autograd.grad(loss, leaf)
        assert torch.isnan(loss), kw.keys()
        assert torch.equal(torch.isnan(lp), spots) or kw["targets"] is targets
        assert torch.isnan(grad[spots]).all() and torch.isfinite(grad[~spots]).all(), kw.keys()
        # the same tokens masked: no trace of them
        loss, _ = losses.policy_loss(logits, kl_coef=0.1 if "ref_logprobs" in kw else 0.0, mask=~spots, **kw)
        assert torch.isfinite(loss)
    leaf = logits[:2].clone().requires_grad_()
    loss, margins = losses.preference_loss(leaf, outside[:2], ref[:2])
    grad, = torch.autograd.grad(loss, leaf)
    assert torch.isnan(loss) and torch.isnan(margins).all() and torch.isnan(grad[spots[:2]]).all()
