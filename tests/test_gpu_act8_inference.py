"""8-bit activations around the training step: nothing kept where no gradient is
wanted, types under autocast and of biases, copies of a model."""
import pytest
import torch

from sandmuon_amd import act8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_nothing_is_kept_without_gradients(device, dtype):
    rows, cols = 2048, 1024
    codes = rows * cols * 33 // 32
    h = torch.randn(rows, cols, device=device).to(dtype)
    w = (torch.randn(cols, cols, device=device) / 32).to(dtype)
    leaf = h.clone().requires_grad_()
    want = act8.gelu(leaf).detach(), act8.mlp(leaf, w, None, w, None).detach()
    del leaf
    out = h.numel() * h.element_size()
    torch.cuda.synchronize()

    def peak(f):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        start = torch.cuda.memory_allocated()
        y = f()
        return y, torch.cuda.max_memory_allocated() - start

    for ctx in (torch.no_grad(), torch.enable_grad()):  # (nothing here requires a gradient either)
        with ctx:
            y, more = peak(lambda: act8.gelu(h))
            assert torch.equal(y, want[0]) and more < out + codes // 2
            y, more = peak(lambda: act8.mlp(h, w, None, w, None))
            assert torch.equal(y, want[1]) and more < 3 * out + codes // 2
    with torch.no_grad():
        leaf = h.requires_grad_()
        y, more = peak(lambda: act8.gelu(leaf))
        assert torch.equal(y, want[0]) and more < out + codes // 2


def test_float64_is_not_cast_by_autocast(device):
    # as F.linear: autocast leaves float64 alone, and the types do not fit
    w = torch.randn(8, 32, device=device, requires_grad=True)
    x = torch.randn(4, 32, device=device, dtype=torch.float64)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for f in (lambda: torch.nn.functional.linear(x, w), lambda: act8.linear(x, w),
                  lambda: act8.mlp(x, w, None, w.t().contiguous(), None)):
            with pytest.raises((RuntimeError, ValueError)):
                f()




def test_bias_gradient_is_rounded_once(device):
    # a bias of more bits than its weight: db in its own type, not through the weight's
    x = torch.randn(300, 64, device=device)
    w = (torch.randn(40, 64, device=device) / 8).to(torch.bfloat16).requires_grad_()
    b = torch.zeros(40, device=device, requires_grad=True)
    proj = (torch.randn(24, 40, device=device) / 8).to(torch.bfloat16).requires_grad_()
    c = torch.zeros(24, device=device, requires_grad=True)
    cot = torch.randn(300, 24, device=device).to(torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = act8.mlp(x, w, b, proj, c)
        z = act8.linear(x, w, b)
    y.backward(cot)
    want = cot.double().sum(0)
    # an FP32 sum of 300 terms: 308 * 2^-24 of their magnitudes
    assert ((c.grad.double() - want).abs() <= 308 * 2.0 ** -24 * cot.double().abs().sum(0)).all()
    b.grad = None
    cot = torch.randn(300, 40, device=device).to(torch.bfloat16)
    z.backward(cot)
    assert ((b.grad.double() - cot.double().sum(0)).abs() <= 308 * 2.0 ** -24 * cot.double().abs().sum(0)).all()
    assert w.grad.dtype == torch.bfloat16 and b.grad.dtype == torch.float32


def test_checkpointed_models_pickle_and_copy(device):
    import copy
    import pickle
    model = torch.nn.Sequential(torch.nn.Linear(64, 48), torch.nn.Linear(48, 8)).to(device)
    act8.checkpoint_linears(model, fmt="e4m3")
    x = torch.randn(32, 64, device=device)
    want = model(x)
    want.sum().backward()
    for other in (pickle.loads(pickle.dumps(model)), copy.deepcopy(model)):
        other.zero_grad(set_to_none=True)
        assert "forward" in other[0].__dict__ and "forward" in other[1].__dict__
        with torch.no_grad():  # (its own weights, not the first model's)
            other[0].weight.add_(0)
            other[1].bias.add_(1)
        sizes = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.dtype) or t, lambda t: t):
            y = other(x)
        assert sizes.count(torch.uint8) == 2
        assert torch.allclose(y, want + 1)
        y.sum().backward()
        assert torch.equal(other[0].weight.grad, model[0].weight.grad)
