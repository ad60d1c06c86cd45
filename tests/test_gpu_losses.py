"""Log probabilities, the policy loss and the preference loss against their
formulas in 64 bits.

Bars, derived beforehand.  A log probability is the FP32 rounding of a
difference whose only error is the FP32 sum of exponentials: 2^-23 of its
magnitude and 2^-20 (a chain of `vocab / 1024 + 10` roundings of a sum of
positive terms, below 2^-20 for every vocabulary here).  A gradient element is
c (onehot - p): one place of its type (2^-23, 2^-8, 2^-11), and 2^-18 of |c| p
(p's error: that of the log sum and 2^-22 per unit of z - lse, 40 at the
most where p matters) and of c's own.  A loss is a weighted sum of terms
whose ratios carry the log probabilities' 2^-20 each."""
import math

import pytest
import torch

from sandmuon_amd import _native, losses

pytestmark = pytest.mark.gpu

PLACE = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def make(device, b, t, v, dtype, seed=0, live=0.7):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(b, t, v, generator=g) * 3).to(dtype)
    targets = torch.randint(0, v, (b, t), generator=g)
    mask = torch.rand(b, t, generator=g) < live
    lp = torch.log_softmax(logits.double(), -1).gather(2, targets[..., None]).squeeze(2)
    old = (lp + torch.randn(b, t, generator=g) * 0.2).float()
    ref = (lp + torch.randn(b, t, generator=g) * 0.3).float()
    adv = torch.randn(b, t, generator=g)
    return [x.to(device) for x in (logits, targets, mask, old, ref, adv)]


def lp64(logits, targets):
    z = logits.detach().cpu().double()
    return torch.log_softmax(z, -1).gather(2, targets.cpu()[..., None]).squeeze(2), torch.softmax(z, -1)


def check_grad(got, p, targets, coef, dtype, slack=None):
    got, coef = got.detach().cpu().double(), coef.double()
    hot = torch.zeros_like(p).scatter_(2, targets.cpu()[..., None], 1.0)
    want = coef[..., None] * (hot - p)
    # c's own error, where a ratio makes it (2^-20 of the log probability)
    bar = PLACE[dtype] * want.abs() + 2.0 ** -18 * coef.abs()[..., None] * (hot + p)
    bar = bar + (2.0 ** -25 if dtype == torch.float16 else 0)
    if slack is not None:
        bar = bar + slack[..., None] * (hot + p)
    assert ((got - want).abs() <= bar).all(), ((got - want).abs() - bar).max()


SIZES = [(1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 7, 64), (3, 5, 97), (2, 9, 1000), (1, 4, 4099), (2, 2, 8192), (1, 3, 50257),
         (1, 2, 131073), (33, 3, 40), (1, 2, 300001)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,t,v", SIZES)
def test_token_logprobs(device, b, t, v, dtype):
    logits, targets, mask, *_ = make(device, b, t, v, dtype, b + t + v)
    want, p = lp64(logits, targets)
    for m in (None, mask):
        live = torch.ones(b, t, dtype=torch.bool) if m is None else m.cpu()
        leaf = logits.clone().requires_grad_()
        got = losses.token_logprobs(leaf, targets, m)
        assert got.dtype == torch.float32 and torch.equal(got.detach(), losses.token_logprobs(logits, targets, m))
        off = (got.detach().cpu().double() - want)[live].abs()
        assert (off <= 2.0 ** -23 * want[live].abs() + 2.0 ** -20).all()
        assert not got.detach().cpu()[~live].any()
        coef = torch.randn(b, t)
        grad, = torch.autograd.grad(got, leaf, coef.to(device))
        assert grad.dtype == dtype and grad.is_contiguous()
        check_grad(grad, p, targets, coef * live, dtype)
        assert not grad.cpu()[~live].any()


def policy64(lp, old, ref, adv, mask, low, high, kl, reduction):
    """(loss, d loss / d lp) in float64."""
    lp = lp.clone().requires_grad_()
    old = lp.detach() if old is None else old.cpu().double()
    a = adv.cpu().double()
    a = a[:, None] if a.dim() == 1 else a
    r = torch.exp(lp - old)
    term = -torch.minimum(r * a, r.clamp(1 - low, 1 + high) * a)
    if ref is not None:
        gap = ref.cpu().double() - lp
        term = term + kl * (torch.expm1(gap) - gap)
    live = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask.cpu()
    term = torch.where(live, term, 0.0)
    n = live.sum(1)
    if reduction == "token":
        loss = term.sum() / max(1, int(n.sum()))
    else:
        loss = (term.sum(1) / n.clamp(min=1)).sum() / max(1, int((n > 0).sum()))
    grad, = torch.autograd.grad(loss, lp, allow_unused=True)
    return loss.item(), grad


@pytest.mark.parametrize("reduction", ["token", "sequence"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,t,v", SIZES)
def test_policy_loss(device, b, t, v, dtype, reduction):
    logits, targets, mask, old, ref, adv = make(device, b, t, v, dtype, b + t + v)
    if b > 1:
        mask[1] = False  # a sequence with no live token
    want_lp, p = lp64(logits, targets)
    for m, o, f, a in ((mask, old, ref, adv), (None, old, ref, adv[:, 0].clone()), (mask, None, None, adv)):
        leaf = logits.clone().requires_grad_()
        loss, lp = losses.policy_loss(leaf, targets, a, old_logprobs=o, ref_logprobs=f, mask=m, clip_low=0.2,
                                      clip_high=0.3, kl_coef=0.1 if f is not None else 0.0, reduction=reduction)
        grad, = torch.autograd.grad(loss, leaf)
        want, back = policy64(want_lp, o, f, a, m, 0.2, 0.3, 0.1, reduction)
        live = torch.ones(b, t, dtype=torch.bool) if m is None else m.cpu()
        size = (a.abs().max().item() * 2 + 1) if live.any() else 0
        assert abs(loss.item() - want) <= 2.0 ** -18 * size + 2.0 ** -22 * abs(want)
        assert not lp.requires_grad and not lp.cpu()[~live].any()
        w = back.abs().max().item() if live.any() else 0.0
        check_grad(grad, p, targets, back, dtype, torch.full((b, t), 2.0 ** -18 * (w + 1) * (1 if live.any() else 0)) /
                   max(1, int(live.sum())))
        assert not grad.cpu()[~live].any()
        # without a gradient asked for: the same loss
        again, _ = losses.policy_loss(logits, targets, a, old_logprobs=o, ref_logprobs=f, mask=m, clip_low=0.2,
                                      clip_high=0.3, kl_coef=0.1 if f is not None else 0.0, reduction=reduction)
        assert torch.equal(again, loss.detach())


def test_policy_loss_without_live_tokens(device):
    logits, targets, mask, old, ref, adv = make(device, 2, 5, 70, torch.bfloat16, 1)
    leaf = logits.clone().requires_grad_()
    loss, lp = losses.policy_loss(leaf, targets, adv, old_logprobs=old, mask=torch.zeros_like(mask))
    grad, = torch.autograd.grad(loss, leaf)
    assert loss.item() == 0 and not grad.any() and not lp.any()
    empty = logits[:, :0].clone().requires_grad_()
    loss, lp = losses.policy_loss(empty, targets[:, :0], adv[:, 0])
    assert loss.item() == 0 and lp.shape == (2, 0) and torch.autograd.grad(loss, empty)[0].shape == (2, 0, 70)


@pytest.mark.parametrize("v", [97, 50257])
def test_masked_places_may_hold_anything(device, v):
    logits, targets, mask, old, ref, adv = make(device, 3, 6, v, torch.bfloat16, 2)
    dirty = [x.clone() for x in (logits, targets, old, ref, adv)]
    dead = ~mask
    dirty[0][dead] = math.nan
    dirty[1][dead] = -100
    for x in dirty[2:]:
        x[dead] = math.inf
    results = []
    for z, y, o, f, a in ((logits, targets, old, ref, adv), dirty):
        z = z.clone().requires_grad_()
        loss, lp = losses.policy_loss(z, y, a, old_logprobs=o, ref_logprobs=f, mask=mask, kl_coef=0.1)
        pl, margins = losses.preference_loss(z[:2], y[:2], f[:2], mask=mask[:2])
        results.append((loss, lp, torch.autograd.grad(loss, z)[0], pl, margins, torch.autograd.grad(pl, z)[0][:2]))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("v", [97, 50257])
def test_special_logits(device, v, dtype):
    logits, targets, *_ = make(device, 1, 8, v, dtype, 3)
    targets[0] = torch.arange(8, device=device)
    low = torch.finfo(dtype).min
    logits[0, 0, 20:60] = -math.inf          # tokens ruled out
    logits[0, 1, 1] = -math.inf              # the target ruled out
    logits[0, 2] = -math.inf                 # every token ruled out
    logits[0, 3, 30] = math.nan
    logits[0, 4, 30] = math.inf
    logits[0, 5, 20:60] = low                # masked by the type's lowest value
    logits[0, 6] = low
    logits[0, 7, 7] = 30000.0
    leaf = logits.clone().requires_grad_()
    lp = losses.token_logprobs(leaf, targets)
    grad, = torch.autograd.grad(lp.sum(), leaf)
    want, p = lp64(logits, targets)
    lp, grad = lp.detach().cpu().double()[0], grad.cpu().double()[0]
    for t in (0, 5, 6, 7):
        assert abs(lp[t] - want[0, t]) <= 2.0 ** -20 + 2.0 ** -23 * want[0, t].abs()
        hot = torch.zeros(v, dtype=torch.float64)
        hot[targets[0, t]] = 1
        assert ((grad[t] - (hot - p[0, t])).abs() <= PLACE[dtype] + 2.0 ** -18).all()
    assert lp[1] == -math.inf
    assert not grad[0, 20:60].any()
    for t in (2, 3, 4):
        assert torch.isnan(lp[t]) and torch.isnan(grad[t]).any()


def test_targets_outside_the_vocabulary(device):
    for v in (97, 4099):
        logits, targets, *_ = make(device, 1, 3, v, torch.float32, 4)
        targets[0, 0], targets[0, 1] = -1, v
        leaf = logits.clone().requires_grad_()
        lp = losses.token_logprobs(leaf, targets)
        grad, = torch.autograd.grad(lp.sum(), leaf)
        assert torch.isnan(lp[0, :2]).all() and torch.isfinite(lp[0, 2])
        assert torch.isnan(grad[0, :2]).all() and torch.isfinite(grad[0, 2]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strided_logits(device, dtype):
    big = make(device, 3, 9, 1031, dtype, 5)[0]
    for view in (big[:, :-1], big[:, 1:], big[:, ::2], big[..., 3:700], big[..., 8:1000], big.transpose(0, 1),
                 big[..., ::2], big[1:2].expand(2, 9, 1031)):
        b, t, v = view.shape
        _, targets, mask, old, ref, adv = make(device, b, t, v, dtype, 6)
        want = losses.token_logprobs(view.contiguous(), targets, mask)
        assert torch.equal(losses.token_logprobs(view, targets, mask), want)
        grads = []
        for z in (view, view.contiguous()):
            z = z.detach().requires_grad_()
            loss, _ = losses.policy_loss(z, targets, adv, old_logprobs=old, ref_logprobs=ref, mask=mask, kl_coef=0.1)
            grads.append(torch.autograd.grad(loss, z)[0])
        assert torch.equal(*grads)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("pairs,t,v,smoothing", [(1, 1, 3, 0.0), (2, 7, 97, 0.1), (5, 30, 200, 0.0), (1, 70, 5003, 0.0),
                                                 (40, 3, 64, 0.2)])
def test_preference_loss(device, pairs, t, v, smoothing, dtype):
    logits, targets, mask, _, ref, _ = make(device, 2 * pairs, t, v, dtype, t + v)
    mask[0] = False
    beta = 0.3
    want_lp, p = lp64(logits, targets)
    for m in (mask, None):
        live = torch.ones_like(want_lp) if m is None else m.cpu().double()
        leaf = logits.clone().requires_grad_()
        loss, margins = losses.preference_loss(leaf, targets, ref, mask=m, beta=beta, label_smoothing=smoothing)
        lp = want_lp.clone().requires_grad_()
        gain = ((lp - ref.cpu().double()) * live).sum(1)
        margin = beta * (gain[:pairs] - gain[pairs:])
        ls = torch.nn.functional.logsigmoid
        want = -((1 - smoothing) * ls(margin) + smoothing * ls(-margin)).mean()
        back, = torch.autograd.grad(want, lp)
        tol = beta * 2 * t * (2.0 ** -20 + 2.0 ** -23 * want_lp.abs().max())
        assert ((margins.cpu().double() - margin.detach()).abs() <= tol + 2.0 ** -23 * margin.detach().abs()).all()
        assert abs(loss.item() - want.item()) <= tol + 2.0 ** -23 * want.item()
        grad, = torch.autograd.grad(loss * 3, leaf)
        check_grad(grad, p, targets, 3 * back, dtype, torch.full((2 * pairs, t), 3 * beta * float(tol) / pairs) * live)


def test_scaled_backward(device):
    logits, targets, mask, old, ref, adv = make(device, 2, 6, 130, torch.float32, 7)
    grads = []
    for factor, scale in ((1.0, 1.0), (1.0, 0.25), (0.25, 1.0), (3.0, 1.0)):
        z = logits.clone().requires_grad_()
        loss, _ = losses.policy_loss(z, targets, adv, old_logprobs=old, mask=mask, scale=scale)
        grads.append(torch.autograd.grad(loss * factor, z)[0])
    assert torch.equal(grads[1], grads[0] / 4) and torch.equal(grads[2], grads[0] / 4)
    assert torch.equal(grads[3], grads[0] * 3)


def test_policy_gradient_is_handed_out_once(device):
    logits, targets, mask, old, ref, adv = make(device, 1, 4, 50, torch.float32, 8)
    z = logits.requires_grad_()
    loss, _ = losses.policy_loss(z, targets, adv)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="handed out once"):
        loss.backward()


def test_gradients_against_differences(device):
    logits, targets, mask, old, ref, adv = make(device, 2, 4, 33, torch.float32, 9)
    step = torch.randn(logits.shape, dtype=torch.float64)
    h = 2.0 ** -8

    def policy(z):
        lp = torch.log_softmax(z, -1).gather(2, targets.cpu()[..., None]).squeeze(2)
        return policy64(lp, old, ref, adv, mask, 0.9, 5.0, 0.1, "token")[0]

    def preference(z):
        lp = torch.log_softmax(z, -1).gather(2, targets.cpu()[..., None]).squeeze(2)
        gain = ((lp - ref.cpu().double()) * mask.cpu()).sum(1)
        return -torch.nn.functional.logsigmoid(0.2 * (gain[:1] - gain[1:])).mean().item()

    for f, call in ((policy, lambda z: losses.policy_loss(z, targets, adv, old_logprobs=old, ref_logprobs=ref, mask=mask,
                                                          clip_low=0.9, clip_high=5.0, kl_coef=0.1)),
                    (preference, lambda z: losses.preference_loss(z, targets, ref, mask=mask, beta=0.2))):
        leaf = logits.clone().requires_grad_()
        grad, = torch.autograd.grad(call(leaf)[0], leaf)
        z = logits.detach().cpu().double()
        want = (f(z + h * step) - f(z - h * step)) / (2 * h)
        terms = (grad.cpu().double() * step)
        # h^2 = 2^-16 of a third derivative of the order of the terms
        assert abs(terms.sum().item() - want) <= 2.0 ** -12 * terms.abs().sum().item()


def test_more_than_2_31_logits(device):
    rows, v = (1 << 31) // 50257 + 5, 50257
    logits = torch.zeros(1, rows, v, dtype=torch.bfloat16, device=device)
    logits[0, -1] = make(device, 1, 1, v, torch.bfloat16, 10)[0][0, 0]
    targets = torch.full((1, rows), 17, device=device)
    mask = torch.zeros(1, rows, dtype=torch.bool, device=device)
    mask[0, -1] = True
    leaf = logits.requires_grad_()
    loss, lp = losses.policy_loss(leaf, targets, torch.ones(1, device=device), mask=mask)
    grad, = torch.autograd.grad(loss, leaf)
    want, p = lp64(logits[:, -1:], targets[:, -1:])
    assert abs(lp[0, -1].item() - want.item()) <= 2.0 ** -20 + 2.0 ** -23 * abs(want.item())
    check_grad(grad[:, -1:], p, targets[:, -1:], torch.full((1, 1), -1.0), torch.bfloat16)
    assert not grad[0, :-1].any()


def test_side_stream_and_graph(device):
    logits, targets, mask, old, ref, adv = make(device, 2, 6, 1000, torch.bfloat16, 11)

    def step(z):
        z = z.detach().requires_grad_()
        loss, lp = losses.policy_loss(z, targets, adv, old_logprobs=old, ref_logprobs=ref, mask=mask, kl_coef=0.1)
        pref, _ = losses.preference_loss(z, targets, ref, mask=mask)
        return (loss.detach(), lp, *torch.autograd.grad(loss, z), pref.detach(), *torch.autograd.grad(pref, z))

    want = step(logits)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(logits)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    held = logits.clone()
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held)
    for k in range(4):
        held.copy_(logits * (1 + 0.1 * k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step(held)))


def test_refusals(device):
    logits, targets, mask, old, ref, adv = make(device, 2, 3, 50, torch.bfloat16, 12)
    with pytest.raises(ValueError, match="reduction"):
        losses.policy_loss(logits, targets, adv, reduction="sum")
    with pytest.raises(ValueError, match="without ref_logprobs"):
        losses.policy_loss(logits, targets, adv, kl_coef=0.1)
    with pytest.raises(ValueError, match="clip_low"):
        losses.policy_loss(logits, targets, adv, clip_low=1.5)
    with pytest.raises(ValueError, match="advantages"):
        losses.policy_loss(logits, targets, adv[:, :2])
    with pytest.raises(ValueError, match="old_logprobs"):
        losses.policy_loss(logits, targets, adv, old_logprobs=old[0])
    with pytest.raises(ValueError, match="mask"):
        losses.token_logprobs(logits, targets, mask.float())
    with pytest.raises(ValueError, match="targets"):
        losses.token_logprobs(logits, targets[:, :2])
    with pytest.raises(ValueError, match="logits"):
        losses.token_logprobs(logits[0], targets[0])
    with pytest.raises(ValueError, match="unsupported dtype"):
        losses.token_logprobs(logits.double(), targets)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        losses.token_logprobs(logits.cpu(), targets.cpu())
    with pytest.raises(ValueError, match="no pairs"):
        losses.preference_loss(logits[:1], targets[:1], ref[:1])
    with pytest.raises(ValueError, match="label_smoothing"):
        losses.preference_loss(logits, targets, ref, label_smoothing=1.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_that_overlap(device, dtype):
    one, targets, mask, old, ref, adv = make(device, 4, 6, 97, dtype, 30)
    strip = make(device, 1, 1, 400, dtype, 31)[0][0, 0]
    for view in (one[:, :1].expand(4, 6, 97), one[:1, :1].expand(4, 6, 97), strip.unfold(0, 97, 10)[:24].view(4, 6, 97),
                 one[..., :1].expand(4, 6, 97)):
        results = []
        for z in (view, view.contiguous()):
            z = z.detach().requires_grad_()
            lp = losses.token_logprobs(z, targets, mask)
            lp_grad, = torch.autograd.grad(lp.sum(), z)
            loss, _ = losses.policy_loss(z, targets, adv, old_logprobs=old, ref_logprobs=ref, mask=mask, kl_coef=0.1)
            policy, = torch.autograd.grad(loss, z)
            loss2, margins = losses.preference_loss(z, targets, ref, mask=mask)
            pref, = torch.autograd.grad(loss2, z)
            results.append((lp.detach(), lp_grad, loss.detach(), policy, loss2.detach(), margins, pref))
        for a, b in zip(*results):
            assert torch.equal(a, b)


def test_more_rows_than_threads_along_one_axis(device):
    # 2^26 waves of 64 are 2^32 threads
    rows = (1 << 26) + 5
    logits = torch.zeros(1, rows, 2, dtype=torch.float16, device=device)
    logits[0, -1, 0] = 3
    targets = torch.zeros(1, rows, dtype=torch.int64, device=device)
    lp = losses.token_logprobs(logits, targets)[0]
    assert lp[-1].item() == pytest.approx(-math.log1p(math.exp(-3)), rel=1e-6)
    assert torch.equal(lp[:-1].min(), lp[:-1].max()) and lp[0].item() == pytest.approx(-math.log(2), rel=1e-6)


@pytest.mark.parametrize("v", [97, 5003])
def test_preference_of_impossible_tokens(device, v):
    # a target ruled out: an infinite margin for (loss 0) or against (loss inf) the chosen one
    logits, targets, mask, _, ref, _ = make(device, 2, 5, v, torch.float32, 32)
    for row, want in ((1, 0.0), (0, math.inf)):
        leaf = logits.clone()
        leaf[row, 2, targets[row, 2]] = -math.inf
        leaf.requires_grad_()
        loss, margins = losses.preference_loss(leaf, targets, ref, beta=0.3)
        grad, = torch.autograd.grad(loss, leaf)
        assert loss.item() == want and margins.item() == (math.inf if row else -math.inf)
        assert torch.isfinite(grad).all() and grad.any().item() == (row == 0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [1, 7, 8, 1031, 1 << 20])
def test_scale(device, dtype, n):
    x = (torch.randn(n + 3, generator=torch.Generator().manual_seed(n)) * 10).to(dtype).to(device)
    for at in (0, 3):  # (at 16-byte boundaries and off them)
        for factor in (1.0, 0.37, -2.0 ** 20, 0.0, math.inf):
            got = x.clone()
            scale = torch.tensor([factor], device=device)
            rc = _native.lib().smx_scale(got.data_ptr() + at * x.element_size(), _native.dtype_code(dtype), n,
                                         scale.data_ptr(), _native.stream_of(x.device))
            assert rc == 0
            want = x.clone()
            want[at:at + n] = (x[at:at + n].float() * factor).to(dtype)
            if factor != 0.37:  # (exact products, rounded once)
                assert torch.equal(torch.nan_to_num(got, nan=5.0), torch.nan_to_num(want, nan=5.0))
                continue
            # half a place of the type, and an FP32 rounding of the product where the kernel makes one
            assert torch.equal(got[:at], x[:at]) and torch.equal(got[at + n:], x[at + n:])
            exact = x[at:at + n].double() * scale.double()
            assert ((got[at:at + n].double() - exact).abs() <= (PLACE[dtype] + 2.0 ** -24) * exact.abs() + 2.0 ** -25).all()
