"""What the differentiable functions on 8-bit activations keep, and for how long."""
import pytest
import torch
import torch.utils.checkpoint

from sandmuon_amd import act8

pytestmark = pytest.mark.gpu

ROWS, COLS = 4096, 512
KEPT = ROWS * COLS * 33 // 32  # bytes of one kept activation


def functions(device):
    torch.manual_seed(0)
    w1, w2 = (torch.nn.Parameter(torch.randn(COLS, COLS, device=device) / 23) for _ in range(2))
    bias = torch.nn.Parameter(torch.zeros(COLS, device=device))
    return {"linear": (lambda x: act8.linear(x, w1, bias), (w1, bias), 1),
            "shared": (lambda x: act8.linear(x, w1, bias, kept=act8.encode(x)), (w1, bias), 1),
            "gelu": (lambda x: act8.gelu(x), (), 1),
            "mlp": (lambda x: act8.mlp(x, w1, bias, w2, bias), (w1, bias, w2), 3)}


@pytest.mark.parametrize("name", ["linear", "shared", "gelu", "mlp"])
def test_kept_bytes_end_with_the_backward(device, name):
    f, params, kept = functions(device)[name]
    x = torch.randn(ROWS, COLS, device=device, requires_grad=True)
    f(x).sum().backward()  # (gradients exist, the library's workspaces too)
    torch.cuda.synchronize()
    start = torch.cuda.memory_allocated()
    loss = f(x).sum()
    held = torch.cuda.memory_allocated() - start
    assert held >= kept * KEPT
    loss.backward()
    # loss still refers to its graph
    assert torch.cuda.memory_allocated() - start < KEPT // 8
    del loss


@pytest.mark.parametrize("name", ["linear", "shared", "gelu", "mlp"])
def test_saved_tensor_hooks_see_the_bytes(device, name):
    f, params, kept = functions(device)[name]
    x = torch.randn(ROWS, COLS, device=device, requires_grad=True)

    def run():
        leaf = x.detach().clone().requires_grad_()
        for p in params:
            p.grad = None
        y = f(leaf)
        y.backward(torch.ones_like(y))
        return [leaf.grad] + [p.grad.clone() for p in params]

    want = run()
    seen = []

    def pack(t):
        seen.append(t.numel() * t.element_size())
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(device)):
        got = run()
    assert seen.count(KEPT) == kept
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    checkpointed = torch.utils.checkpoint.checkpoint(f, x, use_reentrant=False)
    assert torch.equal(checkpointed, f(x))


def test_weights_are_kept_only_for_input_gradients(device):
    w1, w2 = (torch.nn.Parameter(torch.randn(COLS, COLS, device=device)) for _ in range(2))
    x = torch.randn(8, COLS, device=device)
    for f in (lambda x: act8.linear(x, w1), lambda x: act8.mlp(x, w1.detach(), None, w2, None)):
        sizes = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel()) or t, lambda t: t):
            f(x)
        assert COLS * COLS not in sizes and sizes


def test_no_growth_from_step_to_step(device):
    # the loop of a training script: `loss` of the last step lives through the next forward
    f, params, kept = functions(device)["mlp"]
    x = torch.randn(ROWS, COLS, device=device, requires_grad=True)

    def forward():
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        loss = f(x).sum()
        return loss, torch.cuda.max_memory_allocated()

    loss, _ = forward()
    loss.backward()
    del loss
    loss, alone = forward()
    loss.backward()
    for _ in range(3):
        after, peak = forward()
        assert peak <= alone + KEPT // 8
        loss = after
        loss.backward()
