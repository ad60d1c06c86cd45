"""Query and key norms with rotation against the formula in 64 bits.

Bars, derived beforehand: an output element is a sum of two products of FP32
values with a handful of roundings each, within 2^-20 of its vector's largest
element (in dx, of the larger of the two terms that it is the difference of),
plus one place of the output type (2^-23, 2^-8, 2^-11).  A weight
gradient sums `tokens * heads` FP32 terms: (terms + 8) 2^-24 and 2^-20 of the sum of
their magnitudes."""
import math

import pytest
import torch

from sandmuon_amd.attention import qk_norm_rotary, rotary_tables

pytestmark = pytest.mark.gpu

PLACE = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def oracle(x, w, cos, sin, pos, eps, style, dy=None):
    """(y, dx, sum of dw, sum of dw's magnitudes, dx's terms) in float64 on the CPU."""
    x = x.detach().cpu().double()
    b, t, h, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().cpu().double()
    half = cos.shape[1]
    rot = 2 * half
    c, s = (m.cpu().double()[pos.cpu()][:, :, None] for m in (cos, sin))
    first = torch.arange(half) if style == "half" else 2 * torch.arange(half)
    second = first + half if style == "half" else first + 1
    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r * w
    y = n.clone()
    y[..., first] = n[..., first] * c - n[..., second] * s
    y[..., second] = n[..., first] * s + n[..., second] * c
    assert rot <= d
    if dy is None:
        return y
    g = dy.detach().cpu().double()
    back = g.clone()
    back[..., first] = g[..., first] * c + g[..., second] * s
    back[..., second] = g[..., second] * c - g[..., first] * s
    u = x * r
    gw = back * w
    dx = r * (gw - u * (gw * u).mean(-1, keepdim=True))
    terms = (back * u).flatten(0, 2)
    return y, dx, terms.sum(0), terms.abs().sum(0), torch.maximum((r * gw).abs(), (r * gw - dx).abs())


def close(got, want, dtype, size=None):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    if not want.numel():
        return
    bar = PLACE[dtype] * want.abs() + 2.0 ** -20 * (want if size is None else size).abs().amax(-1, keepdim=True)
    bar = bar + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((got - want).abs() <= bar).all(), ((got - want).abs() - bar).max()


def make(device, b, t, hq, hk, d, rot, dtype, seed=0, table=64):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(b, t, hq, d, generator=g) * 3).to(dtype).to(device)
    k = (torch.randn(b, t, hk, d, generator=g) * 0.2 + 0.1).to(dtype).to(device)
    qw = (1 + 0.3 * torch.randn(d, generator=g)).to(device)
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(device)
    cos, sin = rotary_tables(table, rot, device=device)
    return q, k, qw, kw, cos, sin


@pytest.mark.parametrize("style", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("b,t,hq,hk,d,rot", [
    (1, 1, 1, 1, 64, 64), (2, 7, 3, 1, 64, 64), (3, 5, 4, 2, 32, 16), (1, 33, 2, 2, 80, 80), (2, 9, 8, 8, 128, 128),
    (1, 6, 3, 3, 96, 32), (2, 3, 2, 1, 256, 256), (1, 4, 1, 2, 512, 512), (1, 3, 2, 2, 520, 8), (2, 4, 3, 2, 20, 12),
    (1, 5, 2, 1, 7, 6), (1, 2, 1, 1, 1, 0), (2, 3, 2, 2, 64, 0), (1, 1, 1, 1, 2, 2), (1, 300, 12, 12, 16, 16)])
def test_forward_and_backward(device, b, t, hq, hk, d, rot, dtype, style):
    q, k, qw, kw, cos, sin = make(device, b, t, hq, hk, d, rot, dtype, d + t, 320)
    leaves = [v.clone().requires_grad_() for v in (q, k, qw, kw)]
    yq, yk = qk_norm_rotary(*leaves, cos, sin, eps=1e-5, style=style)
    dq, dk = torch.randn_like(yq), torch.randn_like(yk)
    grads = torch.autograd.grad((yq, yk), leaves, (dq, dk))
    pos = torch.arange(t).expand(b, t)
    for x, w, y, dy, gx, gw in ((q, qw, yq, dq, grads[0], grads[2]), (k, kw, yk, dk, grads[1], grads[3])):
        want_y, want_dx, want_dw, size, dx_size = oracle(x, w, cos, sin, pos, 1e-5, style, dy)
        close(y, want_y, dtype)
        close(gx, want_dx, dtype, dx_size)
        terms = b * t * x.shape[2]
        assert ((gw.cpu().double() - want_dw).abs() <= ((terms + 8) * 2.0 ** -24 + 2.0 ** -20) * size).all()
    # no gradient asked for: the same forward
    yq2, yk2 = qk_norm_rotary(q, k, qw, kw, cos, sin, eps=1e-5, style=style)
    assert torch.equal(yq2, yq.detach()) and torch.equal(yk2, yk.detach())


def test_gradient_against_differences(device):
    q, k, qw, kw, cos, sin = make(device, 2, 3, 2, 1, 32, 32, torch.float32, 4)
    g = torch.randn(q.shape, dtype=torch.float64)
    pos = torch.arange(3).expand(2, 3)
    leaf, weight = q.clone().requires_grad_(), qw.clone().requires_grad_()
    y, _ = qk_norm_rotary(leaf, k, weight, kw, cos, sin)
    dx, dw = torch.autograd.grad(y, (leaf, weight), g.float().to(device))
    h = 1e-4
    for grad, at in ((dx, 0), (dw, 1)):
        base = (q.cpu().double(), qw.cpu().double())[at]
        step = torch.randn(base.shape, dtype=torch.float64)
        values = []
        for sign in (1, -1):
            moved = [q.cpu().double(), qw.cpu().double()]
            moved[at] = base + sign * h * step
            values.append((oracle(moved[0], moved[1], cos, sin, pos, 1e-6, "half") * g).sum())
        want = (values[0] - values[1]) / (2 * h)
        got = (grad.cpu().double() * step).sum()
        # (g and its float32 rounding: 2^-24 of each term; h^2 of a third derivative of order one)
        assert abs(got - want) <= 1e-5 * (grad.cpu().double() * step).abs().sum()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_positions(device, dtype):
    q, k, qw, kw, cos, sin = make(device, 3, 4, 2, 1, 64, 32, dtype, 5)
    per_token = torch.randint(0, 64, (3, 4))
    for given, pos in ((None, torch.arange(4).expand(3, 4)), (9, (9 + torch.arange(4)).expand(3, 4)),
                       (per_token.to(device), per_token), (per_token.int().to(device), per_token),
                       (per_token[0].to(device), per_token[:1].expand(3, 4)),
                       (per_token[:, :1].to(device).expand(3, 4), per_token[:, :1].expand(3, 4))):
        yq, yk = qk_norm_rotary(q, k, qw, kw, cos, sin, given)
        close(yq, oracle(q, qw, cos, sin, pos, 1e-6, "half"), dtype)
        close(yk, oracle(k, kw, cos, sin, pos, 1e-6, "half"), dtype)


def test_positions_outside_the_tables_give_nan(device):
    for d, rot in ((64, 32), (20, 12)):
        q, k, qw, kw, cos, sin = make(device, 1, 3, 2, 1, d, rot, torch.float32, 6)
        pos = torch.tensor([[5, 64, -1]], device=device)
        y, _ = qk_norm_rotary(q, k, qw, kw, cos, sin, pos)
        assert torch.isfinite(y[:, 0]).all()
        assert torch.isnan(y[:, 1:, :, :rot]).all() and torch.isfinite(y[..., rot:]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_of_any_stride_and_out(device, dtype):
    b, t, d = 2, 5, 64
    qkv = torch.randn(b, t, 3 * 4 * d, device=device).to(dtype)
    odd = torch.randn(b, t, 4, d + 3, device=device).to(dtype)
    heads_first = torch.randn(b, 4, t, d, device=device).to(dtype)
    cos, sin = rotary_tables(16, d, device=device)
    pos = torch.arange(t).expand(b, t)
    pairs = [(qkv[..., :4 * d].view(b, t, 4, d), qkv[..., 4 * d:8 * d].view(b, t, 4, d)),
             (odd[..., 1:d + 1], odd[..., 3:]), (heads_first.transpose(1, 2), qkv[..., :2 * d].unflatten(-1, (2, d))),
             (qkv.view(b, t, 12, d)[:, :, ::3], odd.transpose(2, 3)[:, :, :4, :].reshape(b, t, 4, 4).repeat(1, 1, 1, 16))]
    for q, k in pairs:
        want_q, want_k = (oracle(x, None, cos, sin, pos, 1e-6, "half") for x in (q, k))
        yq, yk = qk_norm_rotary(q, k, None, None, cos, sin)
        close(yq, want_q, dtype)
        close(yk, want_k, dtype)
        # into slots of a cache, heads first
        cache = torch.zeros(b, k.shape[2], 12, d, device=device, dtype=dtype)
        slot = cache[:, :, 3:3 + t].transpose(1, 2)
        yq2, yk2 = qk_norm_rotary(q, k, None, None, cos, sin, out=(torch.empty_like(yq), slot))
        assert yk2 is slot and torch.equal(slot, yk) and torch.equal(yq2, yq)
        assert not cache[:, :, :3].any() and not cache[:, :, 3 + t:].any()
        # in place
        own = q.clone()
        qk_norm_rotary(own, k, None, None, cos, sin, out=(own, torch.empty_like(yk)))
        assert torch.equal(own, yq)
        # strided cotangents
        leaf = q.detach().clone().requires_grad_()
        y, _ = qk_norm_rotary(leaf, k, None, None, cos, sin)
        dy = torch.randn(b, q.shape[2], t, d + 1, device=device).to(dtype)[..., 1:].transpose(1, 2)
        dx, = torch.autograd.grad(y, leaf, dy)
        want = oracle(q, None, cos, sin, pos, 1e-6, "half", dy)
        close(dx, want[1], dtype, want[4])


def test_one_sided_gradients_and_weight_types(device):
    q, k, qw, kw, cos, sin = make(device, 2, 6, 4, 2, 64, 64, torch.bfloat16, 8)
    qw, kw = qw.to(torch.bfloat16).requires_grad_(), kw.half()
    leaf = q.clone().requires_grad_()
    yq, yk = qk_norm_rotary(leaf, k, qw, kw, cos, sin)
    dy = torch.randn_like(yq)
    dx, dw = torch.autograd.grad(yq, (leaf, qw), dy)
    want = oracle(q, qw, cos, sin, torch.arange(6).expand(2, 6), 1e-6, "half", dy)
    close(dx, want[1], torch.bfloat16, want[4])
    assert dw.dtype == torch.bfloat16
    assert ((dw.cpu().double() - want[2]).abs() <= 2.0 ** -8 * want[2].abs() + 2.0 ** -18 * want[3]).all()
    close(yk, oracle(k, kw, cos, sin, torch.arange(6).expand(2, 6), 1e-6, "half"), torch.bfloat16)


def test_zero_vectors_and_infinities(device):
    q, k, qw, kw, cos, sin = make(device, 1, 4, 2, 1, 64, 64, torch.float32, 9)
    q[0, 0, 0] = 0
    q[0, 1, 1, 5] = math.inf
    q[0, 2, 0, 7] = math.nan
    y, _ = qk_norm_rotary(q, k, qw, kw, cos, sin)
    assert not y[0, 0, 0].any()
    assert torch.isnan(y[0, 2, 0]).all()
    clean = torch.ones(4, 2, dtype=torch.bool)
    clean[1, 1] = clean[2, 0] = False
    assert torch.isfinite(y[0][clean.to(device)]).all()


def test_empty_batches(device):
    q, k, qw, kw, cos, sin = make(device, 2, 3, 2, 1, 64, 64, torch.bfloat16, 10)
    leaves = [v.requires_grad_() for v in (q[:0].clone(), k[:0].clone(), qw, kw)]
    yq, yk = qk_norm_rotary(*leaves, cos, sin)
    grads = torch.autograd.grad((yq, yk), leaves, (torch.empty_like(yq), torch.empty_like(yk)))
    assert yq.shape == (0, 3, 2, 64) and grads[0].shape == (0, 3, 2, 64)
    assert not grads[2].any() and not grads[3].any()


def test_backward_is_deterministic(device):
    q, k, qw, kw, cos, sin = make(device, 4, 300, 8, 4, 64, 64, torch.bfloat16, 11, 512)
    leaves = [v.requires_grad_() for v in (q, k, qw, kw)]
    out = qk_norm_rotary(*leaves, cos, sin)
    dy = [torch.randn_like(o) for o in out]
    first = torch.autograd.grad(out, leaves, dy, retain_graph=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, dy, retain_graph=True)))


def test_refusals(device):
    q, k, qw, kw, cos, sin = make(device, 2, 3, 2, 1, 64, 64, torch.bfloat16, 12)
    for bad, match in ((dict(style="both"), "style"), (dict(positions=torch.zeros(2, 3, device=device)), "positions"),
                       (dict(positions=torch.zeros(5, dtype=torch.long, device=device)), "expand")):
        with pytest.raises((ValueError, RuntimeError), match=bad and match):
            qk_norm_rotary(q, k, qw, kw, cos, sin, **bad)
    with pytest.raises(ValueError, match="expected"):
        qk_norm_rotary(q, k[..., :32], qw, kw, cos, sin)
    with pytest.raises(ValueError, match="expected"):
        qk_norm_rotary(q, k.float(), qw, kw, cos, sin)
    with pytest.raises(ValueError, match="cos"):
        qk_norm_rotary(q, k, qw, kw, cos.double(), sin.double())
    with pytest.raises(ValueError, match="q_weight"):
        qk_norm_rotary(q, k, qw[:32], kw, cos, sin)
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        qk_norm_rotary(q.cpu(), k.cpu(), qw.cpu(), kw.cpu(), cos.cpu(), sin.cpu())
    with pytest.raises(ValueError, match="autograd"):
        qk_norm_rotary(q.clone().requires_grad_(), k, qw, kw, cos, sin, out=(q, k))
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rotary(q, k, qw, kw, cos, sin, eps=-1.0)


def test_out_that_names_places_twice_is_refused(device):
    q, k, qw, kw, cos, sin = make(device, 2, 3, 4, 1, 64, 64, torch.bfloat16, 13)
    same = torch.empty(2, 3, 1, 64, dtype=q.dtype, device=device).expand(2, 3, 4, 64)
    with pytest.raises(ValueError, match="twice"):
        qk_norm_rotary(q, k, qw, kw, cos, sin, out=(same, torch.empty_like(k)))
    y, z = qk_norm_rotary(q, k, qw, kw, cos, sin, out=(torch.empty_like(q), torch.empty_like(k)))
    assert y.shape == q.shape and z.shape == k.shape
