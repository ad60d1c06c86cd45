"""Errors of one sign in log probabilities, which sums over tokens do not
average out, against 64 bits.

Bars, derived beforehand.  A token's log probability is (z - max) - hi - lo, three
FP32 roundings to nearest of what is left (and of the sum, below them): errors of
either sign, each uniform within half a place, a standard deviation of 2^-23 /
sqrt(12) of the value at the most.  What has one sign comes from the
exponentials, whose argument is carried to 2^-47: the instruction's own mean
error, 2^-28 as measured over its fractions; 2^-26 is granted.  A mean or a sum
over N tokens is then within 2^-26 (or N times it) and a few standard deviations of
the roundings' sum."""
import pytest
import torch

from sandmuon_amd import _native, losses

pytestmark = pytest.mark.gpu


def batch(device, b, t, v, dtype, seed):
    """Logits that favour their targets, the targets, and per token the exact log
    probability and the standard deviation of the roundings of an FP32 one."""
    g = torch.Generator(device=device).manual_seed(seed)
    logits = torch.empty(b, t, v, dtype=dtype, device=device)
    targets = torch.randint(0, v, (b, t), device=device, generator=g)
    exact = torch.empty(b, t, dtype=torch.float64, device=device)
    spread = torch.empty_like(exact)
    for i in range(b):
        z = torch.randn(t, v, device=device, generator=g) * 2
        z.scatter_add_(1, targets[i, :, None], torch.full((t, 1), 10.0, device=device))
        logits[i] = z.to(dtype)
        z = logits[i].double()
        first = z.gather(1, targets[i, :, None]).squeeze(1) - z.amax(1)
        exact[i] = torch.log_softmax(z, 1).gather(1, targets[i, :, None]).squeeze(1)
        # (what is left after hi lies between the two)
        each = torch.maximum(first.abs(), exact[i].abs())
        spread[i] = 2.0 ** -23 / 12 ** 0.5 * (first.square() + each.square() + exact[i].square()).sqrt()
    return logits, targets, exact, spread


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("b,t,v", [(8, 1024, 50257), (8, 2048, 1031)])
def test_log_probabilities_err_to_neither_side(device, b, t, v, dtype):
    logits, targets, exact, spread = batch(device, b, t, v, dtype, 1)
    off = losses.token_logprobs(logits, targets).double() - exact
    assert abs(off.mean().item()) <= 2.0 ** -26 + 6 * spread.square().sum().sqrt().item() / (b * t)


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_margins_of_long_sequences(device, seed):
    pairs, t, v, beta = 4, 1024, 50257, 0.1
    logits, targets, exact, spread = batch(device, 2 * pairs, t, v, torch.bfloat16, seed)
    # chosen ones of full length beside rejected ones of a few tokens, and between
    live = torch.tensor([1024, 1024, 900, 512, 1, 5, 40, 500], device=device)
    mask = torch.arange(t, device=device)[None, :] < live[:, None]
    noise = torch.randn(exact.shape, device=device, generator=torch.Generator(device=device).manual_seed(seed))
    ref = (exact + 0.3 * noise).float()
    _, margins = losses.preference_loss(logits, targets, ref, mask=mask, beta=beta)
    gap = torch.where(mask, exact - ref.double(), 0.0)
    want = beta * (gap[:pairs].sum(1) - gap[pairs:].sum(1))
    # (lp - ref is rounded too)
    each = torch.where(mask, spread.square() + (2.0 ** -24 * gap).square(), 0.0).sum(1)
    one_sided = 2.0 ** -26 * (live[:pairs] - live[pairs:]).abs()
    bar = beta * (one_sided + 4 * (each[:pairs] + each[pairs:]).sqrt()) + 2.0 ** -23 * want.abs()
    assert ((margins.double() - want).abs() <= bar).all()


@pytest.mark.parametrize("smoothing", [0.0, 1.0, 0.25])
def test_slopes_of_large_margins(device, smoothing):
    # d loss / d lp is beta (s sigmoid(m) - (1 - s) sigmoid(-m)) / pairs, whatever is left of it:
    # FP32 roundings of m (2^-24 of it), of exp(-|m|) and of the result
    margins = torch.tensor([0.0, 0.3, -0.3, 9.0, -9.0, 20.0, -20.0, 33.0, 45.0, -45.0, 80.0, -80.0])
    pairs, beta = len(margins), 0.5
    lp = torch.cat([margins / beta, torch.zeros(pairs)])[:, None].contiguous().to(device)
    loss, got = torch.empty((), device=device), torch.empty(pairs, device=device)
    coef = torch.empty(2 * pairs, device=device)
    rc = _native.lib().smx_preference_loss(lp.data_ptr(), torch.zeros_like(lp).data_ptr(), None, pairs, 1, beta, smoothing,
                                           loss.data_ptr(), got.data_ptr(), coef.data_ptr(), _native.stream_of(lp.device))
    assert rc == 0 and torch.equal(got.cpu(), margins)
    m = margins.double()
    want = beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m)) / pairs
    bar = (2.0 ** -22 + 2.0 ** -24 * m.abs()) * (smoothing * torch.sigmoid(m) + (1 - smoothing) * torch.sigmoid(-m)) * beta / pairs
    for side, sign in ((coef[:pairs], 1), (coef[pairs:], -1)):
        assert ((side.cpu().double() - sign * want).abs() <= bar + 1e-45).all()
