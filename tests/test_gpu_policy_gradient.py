"""The policy loss's gradient to FP16 logits under a loss scaler's factor."""
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


@pytest.mark.parametrize("factor", [1.0, 65536.0])
@pytest.mark.parametrize("b,t,v", [(1, 1, 1), (2, 6, 130), (1, 3, 4099), (4, 512, 50257), (1, 2, 131073)])
def test_scaled_loss_of_f16_logits(device, b, t, v, factor):
    # An element is rounded once, to f16: 2^-11 of it or half the smallest step, and carries
    # 2^-18 of |c| (onehot + p) as the other types' do.
    logits, targets, lp, old, ref, adv, mask = inputs(device, b, t, v, torch.float16, t)
    leaf = logits.clone().requires_grad_()
    loss, _ = losses.policy_loss(leaf, targets, adv, old_logprobs=old, ref_logprobs=ref, mask=mask, clip_low=0.9,
                                 clip_high=9.0, kl_coef=0.1, scale=0.5)
    grad, = torch.autograd.grad(loss * factor, leaf)
    n = max(1, int(mask.sum()))
    coef = 0.5 * factor / n * (-adv.double() * (lp - old.double()).exp() - 0.1 * torch.expm1(ref.double() - lp))
    coef = torch.where(mask, coef, 0.0)
    for i in range(b):
        p = torch.softmax(logits[i].double(), 1)
        hot = torch.zeros_like(p).scatter_(1, targets[i, :, None], 1.0)
        want = coef[i, :, None] * (hot - p)
        # (the ratio and the KL term carry the log probability's 2^-20 each)
        slack = 2.0 ** -18 * (coef[i].abs() + factor / n * (adv[i].abs().double() + 0.1))[:, None] * (hot + p)
        bar = 2.0 ** -11 * want.abs() + 2.0 ** -25 + slack
        assert grad.dtype == torch.float16 and ((grad[i].double() - want).abs() <= bar).all()
        assert not grad[i][~mask[i]].any()
