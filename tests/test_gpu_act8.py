"""8-bit activations against their definition in 64 bits.

Bars, derived beforehand:
* codes read back: equal to the definition, every bit;
* weight gradient: products are exact and sums FP32, so each element is within
  (rows + 8) 2^-24 of the sum of its terms' magnitudes (any order of summation
  keeps rows 2^-24), plus the output type's rounding (one place: 2^-23, 2^-8,
  2^-11);
* GELU and its gradient: the output type's rounding (one place) plus 2^-21 of
  |h| (|dy| in the gradient) for the FP32 evaluation of 1 + erf near its zero."""
import math

import pytest
import torch
import torch.nn.functional as F

from sandmuon_amd import act8

pytestmark = pytest.mark.gpu

PLACE = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def oracle(x, fmt):
    """The kept values of x [rows, cols] by the definition, float64 on the CPU."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    out = torch.empty_like(x)
    for at in range(0, cols, 32):
        v = x[:, at:at + 32]
        bad = ~torch.isfinite(v).all(1)
        peak = torch.where(torch.isfinite(v), v, 0.0).abs().amax(1)
        e = torch.frexp(peak)[1] - 1  # 0 for a block of zeros, whose codes are zero at any scale
        if fmt == "int8":
            scale = 2.0 ** torch.clamp(e - 6, min=-126).double()
            held = torch.clamp(torch.round(v / scale[:, None]), -127, 127)
        else:
            scale = 2.0 ** torch.where(e == 127, e - 6, torch.clamp(e - 7, min=-117)).double()
            u = v / scale[:, None]
            step = 2.0 ** torch.clamp(torch.frexp(u)[1] - 4, min=-9).double()
            held = torch.round(u / step) * step
            held = torch.where((e == 127)[:, None], held.clamp(-120, 120), held)
        held = held * scale[:, None]
        held[bad] = math.nan
        out[:, at:at + 32] = held
    return out


def activation(rows, cols, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(1, cols, generator=g) * 1.5)
    return x.to(dtype).to(device)


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (7, 33), (1, 8), (130, 777), (9, 2056), (1030, 96)])
def test_kept_values_are_the_definitions(device, rows, cols, dtype, fmt):
    x = activation(rows, cols, dtype, device, rows + cols)
    saved = act8.encode(x, fmt)
    assert saved.nbytes == rows * saved.pitch * 33 // 32
    assert same(act8.decode(saved, torch.float32).cpu().double(), oracle(x, fmt))
    assert same(act8.decode(saved).cpu().double(), oracle(x, fmt))  # (exact in bf16)
    assert (saved.codes[:, cols:] == 0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_extreme_blocks(device, fmt):
    x = torch.zeros(13, 64)
    x[1] = 1e-45
    x[2] = torch.linspace(-3.4e38, 3.4e38, 64)
    x[3, 5] = math.inf
    x[4, 40] = math.nan
    x[5, 0], x[5, 1:32] = 1e30, 1e-30
    x[6] = 127.5
    x[7] = -0.99999994
    x[8] = 2.0 ** -120
    x[9] = torch.arange(64) * 2.0 ** -126
    x[10] = -0.0
    x[11, 33] = -math.inf
    x[12] = torch.linspace(-1, 1, 64) * 3.4e38
    x = x.to(device)
    got = act8.decode(act8.encode(x, fmt), torch.float32).cpu().double()
    want = oracle(x, fmt)
    assert same(got, want)
    assert torch.isnan(got[3, :32]).all() and torch.isfinite(got[3, 32:]).all()
    assert torch.isfinite(act8.decode(act8.encode(x[12:], fmt)).float()).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_of_any_stride(device, dtype, fmt):
    base = activation(40, 200, dtype, device, 3)
    for x in (base[:, 3:100], base[::3, 8:72], base[:, ::2], base.t(), base.view(4, 10, 200)[:, 1:, :64],
              base.view(2, 20, 200).transpose(0, 1)):
        want = oracle(x.reshape(-1, x.shape[-1]), fmt)
        saved = act8.encode(x, fmt)
        assert saved.shape == x.shape
        assert same(act8.decode(saved, torch.float32).reshape(want.shape).cpu().double(), want)


def test_empty(device):
    for shape in ((0, 5), (4, 0), (0, 0), (2, 0, 7)):
        x = torch.empty(shape, device=device)
        assert act8.decode(act8.encode(x)).shape == x.shape
    dw, db = act8.linear_backward(torch.empty(0, 3, device=device), act8.encode(torch.empty(0, 5, device=device)))
    assert dw.shape == (3, 5) and not dw.any() and not db.any()
    dw, db = act8.linear_backward(torch.ones(4, 3, device=device), act8.encode(torch.empty(4, 0, device=device)))
    assert dw.shape == (3, 0) and torch.equal(db.cpu(), torch.full((3,), 4.0))


def test_more_than_2_31_elements(device):
    x = torch.zeros((1 << 31) // 8192 + 3, 8192, dtype=torch.bfloat16, device=device)
    x[-1] = activation(1, 8192, torch.bfloat16, device, 5)
    saved = act8.encode(x)
    assert same(act8.decode(saved)[-1:].cpu().double(), oracle(x[-1:], "int8"))
    # only the last row has a cotangent
    delta = torch.zeros(x.shape[0], 8, dtype=torch.bfloat16, device=device)
    delta[-1] = 1
    dw, _ = act8.linear_backward(delta, saved, torch.float32)
    assert same(dw[:1].cpu().double(), oracle(x[-1:], "int8"))


# ------------------------------------------------------------ linear backward ---
def check_linear(delta, saved, kept, dtype):
    dw, db = act8.linear_backward(delta, saved, dtype)
    d = delta.reshape(-1, delta.shape[-1]).cpu().double()
    k = kept.reshape(-1, kept.shape[-1])
    rows = d.shape[0]
    for got, want, size in ((dw, d.t() @ k, d.abs().t() @ k.abs()), (db, d.sum(0), d.abs().sum(0))):
        got = got.cpu().double()
        assert got.shape == want.shape
        off = (got - want).abs()
        bar = (rows + 8) * 2.0 ** -24 * size + PLACE[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        assert (off <= bar).all(), (off - bar).max()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (1, 32, 8), (2, 33, 65), (17, 40, 24), (63, 96, 128), (64, 64, 64),
                                      (65, 130, 300), (300, 257, 96), (1000, 128, 256), (4099, 72, 56),
                                      (520, 800, 520)])
def test_weight_gradient(device, rows, k, n, dtype, fmt):
    x = activation(rows, k, dtype, device, rows)
    delta = activation(rows, n, dtype, device, rows + 1) * 0.1
    check_linear(delta, act8.encode(x, fmt), oracle(x, fmt), torch.float32)


@pytest.mark.parametrize("out", DTYPES, ids=IDS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_weight_gradient_types(device, dtype, out):
    x = activation(700, 200, torch.float32, device, 1)
    delta = activation(700, 136, dtype, device, 2) * 0.01
    check_linear(delta, act8.encode(x), oracle(x, "int8"), out)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_weight_gradient_of_views(device, dtype):
    x = activation(6 * 50, 160, dtype, device, 4)
    base = activation(6 * 50, 400, dtype, device, 5)
    saved, kept = act8.encode(x.view(6, 50, 160)), oracle(x, "int8")
    for delta in (base[:, 1:78], base[:, 8:136], base[:, ::3], base[:, 64:64 + 128]):
        check_linear(delta.reshape(6, 50, -1) if delta.stride(1) == 1 else delta.unflatten(0, (6, 50)), saved, kept,
                     torch.float32)


def test_weight_gradient_keeps_infinities_and_nans(device):
    x = activation(96, 64, torch.bfloat16, device, 6)
    delta = activation(96, 48, torch.bfloat16, device, 7)
    x[5, 3] = math.nan
    delta[7, 9] = math.inf
    dw, db = act8.linear_backward(delta, act8.encode(x), torch.float32)
    assert torch.isnan(dw[:, :32]).all()
    assert not torch.isfinite(dw[9]).any()
    rest = torch.ones(48, dtype=torch.bool, device=device)
    rest[9] = False
    assert torch.isfinite(dw[rest][:, 32:]).all()
    assert db[9] == math.inf and torch.isfinite(db[rest]).all()


def test_small_and_large_float32_cotangents(device):
    # three BF16 parts hold the 24 bits of a float32 across its range
    x = activation(256, 64, torch.float32, device, 8)
    delta = activation(256, 32, torch.float32, device, 9) * torch.exp(torch.linspace(-40, 40, 32, device=device))
    check_linear(delta, act8.encode(x), oracle(x, "int8"), torch.float32)


def test_weight_gradient_is_deterministic(device):
    x, delta = activation(3000, 256, torch.bfloat16, device, 1), activation(3000, 192, torch.bfloat16, device, 2)
    saved = act8.encode(x)
    first = act8.linear_backward(delta, saved, torch.float32)
    for _ in range(3):
        again = act8.linear_backward(delta, saved, torch.float32)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ----------------------------------------------------------------------- gelu ---
def gelu64(h):
    return h * 0.5 * torch.special.erfc(-h / math.sqrt(2))


def slope64(h):
    return 0.5 * torch.special.erfc(-h / math.sqrt(2)) + h * torch.exp(-h * h / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 37), (65, 96), (260, 200), (33, 2080)])
def test_gelu(device, rows, cols, dtype, fmt):
    h = (activation(rows, cols, torch.float32, device, cols) * 1.5).to(dtype)
    dy = activation(rows, cols, dtype, device, cols + 1)
    y, saved_h, saved_y = act8.gelu_forward(h, fmt)
    h64 = h.cpu().double()
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0
    assert ((y.cpu().double() - gelu64(h64)).abs() <= PLACE[dtype] * gelu64(h64).abs() + 2.0 ** -21 * h64.abs() + tiny).all()
    assert same(act8.decode(saved_h, torch.float32).cpu().double(), oracle(h, fmt))
    assert same(act8.decode(saved_y, torch.float32).cpu().double(), oracle(y, fmt))
    without, again, none = act8.gelu_forward(h, fmt, keep_output=False)
    assert none is None and torch.equal(without, y) and torch.equal(again.data, saved_h.data)
    kept = oracle(h, fmt)
    dh = act8.gelu_backward(dy, saved_h).cpu().double()
    dy64 = dy.cpu().double()
    want = dy64 * slope64(kept)
    assert ((dh - want).abs() <= PLACE[dtype] * want.abs() + 2.0 ** -21 * dy64.abs() + tiny).all()
    # the slope itself against central differences in 64 bits (error: h^2 / 6 of a third derivative below 2)
    step = 2.0 ** -12
    diff = (gelu64(kept + step) - gelu64(kept - step)) / (2 * step)
    assert ((dh - dy64 * diff).abs() <= PLACE[dtype] * want.abs() + (2.0 ** -21 + step * step) * dy64.abs() + tiny).all()


def test_gelu_of_every_bf16(device):
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    h = bits.view(torch.bfloat16).to(device).view(2048, 32)
    y, _, _ = act8.gelu_forward(h)
    want = F.gelu(h.float())
    fine = torch.isfinite(want) & torch.isfinite(h.float())
    off = (y.float() - want).abs()
    # (one place of a subnormal is 2^-133 whatever its size)
    place = torch.clamp(PLACE[torch.bfloat16] * want.abs(), min=2.0 ** -133)
    assert (off[fine] <= (place + 2.0 ** -21 * h.float().abs())[fine]).all()
    assert torch.equal(torch.isnan(y.float()), torch.isnan(want.to(torch.bfloat16).float()))
    assert torch.equal(torch.isinf(y.float()), torch.isinf(want.to(torch.bfloat16).float()))


def test_gelu_of_views(device):
    base = activation(30, 300, torch.bfloat16, device, 3)
    for h in (base[:, 5:101], base[:, 8:104], base[::2], base.t()):
        y, saved, _ = act8.gelu_forward(h)
        y2, saved2, _ = act8.gelu_forward(h.contiguous())
        assert torch.equal(y, y2) and torch.equal(saved.data, saved2.data)
        dy = activation(300, 310, torch.bfloat16, device, 4)[:h.shape[0], 2:2 + h.shape[1]]
        assert torch.equal(act8.gelu_backward(dy, saved), act8.gelu_backward(dy.contiguous(), saved))


# ------------------------------------------------------------------- autograd ---
def relative(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("autocast", [False, True])
def test_linear_and_mlp_against_torch(device, autocast):
    torch.manual_seed(0)
    fc, proj = torch.nn.Linear(72, 200).to(device), torch.nn.Linear(200, 56).to(device)
    x = activation(6 * 33, 72, torch.float32, device, 2).view(6, 33, 72)
    grad = torch.randn(6, 33, 56, device=device)

    def run(forward):
        leaf = x.clone().requires_grad_()
        for p in (*fc.parameters(), *proj.parameters()):
            p.grad = None
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            out = forward(leaf)
        out.backward(grad.to(out.dtype))
        return out.detach(), [leaf.grad] + [p.grad.clone() for p in (*fc.parameters(), *proj.parameters())]

    want, want_grads = run(lambda t: proj(F.gelu(fc(t))))
    for forward in (lambda t: act8.mlp(t, fc.weight, fc.bias, proj.weight, proj.bias),
                    lambda t: act8.linear(act8.gelu(act8.linear(t, fc.weight, fc.bias)), proj.weight, proj.bias)):
        out, grads = run(forward)
        assert out.dtype == want.dtype
        assert relative(out, want) < (1e-2 if autocast else 1e-6)
        for g, w in zip(grads, want_grads):
            assert g.dtype == w.dtype and g.shape == w.shape
            # int8: half a step is 2^-7 of a block's largest, and the slope's curvature keeps it below 2 %
            assert relative(g, w) < 2e-2


def test_checkpointed_linears_keep_outputs_and_hooks(device):
    torch.manual_seed(1)
    model = torch.nn.Sequential(torch.nn.Linear(40, 64), torch.nn.Tanh(), torch.nn.Linear(64, 24)).to(device)
    x = torch.randn(50, 40, device=device)
    want = model(x).detach()
    seen = []
    model[0].register_forward_hook(lambda m, i, o: seen.append(i[0].shape))
    handle = act8.checkpoint_linears(model)
    assert len(handle.modules) == 2
    out = model(x)
    assert torch.equal(out.detach(), want) and len(seen) == 1
    out.sum().backward()
    assert model[0].weight.grad is not None and model[2].bias.grad is not None
    handle.close()
    assert "forward" not in model[0].__dict__
    assert torch.equal(model(x), want)


def test_refusals(device):
    x = torch.randn(4, 32, device=device)
    saved = act8.encode(x)
    with pytest.raises(ValueError, match="unknown 8-bit format"):
        act8.encode(x, "int4")
    with pytest.raises(ValueError, match="unsupported dtype"):
        act8.encode(x.double())
    with pytest.raises(RuntimeError, match="GPU tensors only"):
        act8.encode(x.cpu())
    with pytest.raises(ValueError, match="unsupported dtype"):
        act8.decode(saved, torch.float64)
    with pytest.raises(ValueError, match="cotangent"):
        act8.linear_backward(torch.randn(5, 8, device=device), saved)
    with pytest.raises(ValueError, match="cotangent"):
        act8.gelu_backward(torch.randn(4, 31, device=device), saved)
    with pytest.raises(TypeError, match="Act8"):
        act8.gelu_backward(x, x)
    with pytest.raises(ValueError, match="dimension"):
        act8.encode(torch.tensor(1.0, device=device))


def test_side_stream_and_graph(device):
    """On a stream of their own, and replayed from a graph, the same bits."""
    from sandmuon_amd.attention import qk_norm_rotary, rotary_tables
    x = activation(3000, 256, torch.bfloat16, device, 1)
    delta = activation(3000, 192, torch.bfloat16, device, 2)
    cos, sin = rotary_tables(64, 64, device=device)
    w = torch.ones(64, device=device)

    def step(x, delta):
        saved = act8.encode(x)
        y, kept, kept_y = act8.gelu_forward(x, "e4m3")
        q = x[:2944].view(46, 64, 4, 64).detach().requires_grad_()
        k = delta[:2944].view(46, 64, 3, 64).detach().requires_grad_()
        out = qk_norm_rotary(q, k, w.requires_grad_(), None, cos, sin)
        grads = torch.autograd.grad(out, (q, k, w), (out[1].detach().repeat(1, 1, 2, 1)[:, :, :4], out[0].detach()[:, :, :3]))
        return (*act8.linear_backward(delta, saved, torch.float32), act8.decode(saved), y, act8.gelu_backward(y, kept),
                act8.decode(kept_y), *(o.detach() for o in out), *grads)

    want = step(x, delta)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, delta)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    held = x.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held, delta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held, delta)
    for k in range(3):
        held.copy_(x * (1 + 0.5 * k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step(held, delta)))


def test_no_double_backward(device):
    from sandmuon_amd import losses
    from sandmuon_amd.attention import qk_norm_rotary, rotary_tables
    z = torch.randn(2, 3, 40, device=device, requires_grad=True)
    y = torch.zeros(2, 3, dtype=torch.long, device=device)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(losses.token_logprobs(z, y).sum(), z, create_graph=True)
    q = torch.randn(1, 2, 1, 64, device=device, requires_grad=True)
    out, _ = qk_norm_rotary(q, q.detach(), None, None, *rotary_tables(4, 64, device=device))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out.sum(), q, create_graph=True)


def test_bytes_that_do_not_fit_their_shape_are_refused(device):
    saved = act8.encode(torch.randn(8, 64, device=device))
    for shape, data in ((torch.Size([9, 64]), saved.data), (torch.Size([8, 64]), saved.data[:-1]),
                        (torch.Size([8, 64]), saved.data.float()), (torch.Size([8, 64]), saved.data.cpu())):
        with pytest.raises(ValueError, match="bytes of a kept"):
            act8.decode(act8.Act8(data, shape, "int8"))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_that_overlap(device, dtype):
    row = activation(1, 70, dtype, device, 21)
    strip = activation(1, 300, dtype, device, 22)[0]
    for x in (row.expand(9, 70), row.expand(3, 3, 70), strip.unfold(0, 70, 3), row[:, :1].expand(9, 70)):
        plain = x.contiguous()
        saved = act8.encode(x)
        assert torch.equal(saved.data, act8.encode(plain).data)
        y, kept, _ = act8.gelu_forward(x)
        assert torch.equal(y, act8.gelu_forward(plain)[0]) and torch.equal(kept.data, saved.data)
        assert torch.equal(act8.gelu_backward(x, saved), act8.gelu_backward(plain, saved))
        for got, want in zip(act8.linear_backward(x, saved), act8.linear_backward(plain, saved)):
            assert torch.equal(got, want)


def test_gradients_of_sums_over_rows(device):
    # the cotangent is one row, repeated
    h = activation(33, 40, torch.float32, device, 23)
    w = activation(24, 40, torch.float32, device, 24) / 8
    for fn in (lambda x, v: act8.gelu(x), lambda x, v: act8.linear(x, v), lambda x, v: act8.mlp(x, v, None, v.t(), None)):
        grads = []
        for repeat in (False, True):
            leaf, weight = h.clone().requires_grad_(), w.clone().requires_grad_()
            y = fn(leaf, weight)
            cot = torch.linspace(-1, 1, y.shape[-1], device=device)
            if repeat:
                y.sum(0).backward(cot)
            else:
                y.backward(cot.expand(33, -1).contiguous())
            grads.append((leaf.grad, weight.grad))
        for a, b in zip(*grads):
            assert (a is None and b is None) or torch.equal(a, b)


def test_frozen_parts(device):
    torch.manual_seed(2)
    x = activation(70, 40, torch.float32, device, 25)
    fc, proj = torch.nn.Linear(40, 64).to(device), torch.nn.Linear(64, 24).to(device)
    params = [fc.weight, fc.bias, proj.weight, proj.bias]

    def run(forward, wanted):
        leaves = [t.detach().clone().requires_grad_(want) for t, want in zip([x] + params, wanted)]
        y = forward(*leaves)
        if any(wanted):
            y.sum().backward()
        return [y.detach()] + [t.grad for t in leaves]

    mlp = lambda t, w1, b1, w2, b2: act8.mlp(t, w1, b1, w2, b2)
    linear = lambda t, w1, b1, w2, b2: act8.linear(t, w1, b1)
    for forward, used in ((mlp, 5), (linear, 3)):
        whole = run(forward, [True] * 5)
        for bits in range(2 ** used):
            wanted = [bool(bits >> i & 1) for i in range(5)]
            got = run(forward, wanted)
            assert torch.equal(got[0], whole[0])
            for want, a, b in zip(wanted, got[1:], whole[1:]):
                assert torch.equal(a, b) if want else a is None
        with torch.no_grad():
            assert torch.equal(forward(x, *params), whole[0])
