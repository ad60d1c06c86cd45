"""Linears without outputs, inputs or rows."""
import pytest
import torch
import torch.nn.functional as F

from sandmuon_amd import act8

pytestmark = pytest.mark.gpu


def test_weight_gradient_of_no_outputs(device):
    for shape in ((4,), (2, 3), ()):
        dw, db = act8.linear_backward(torch.empty(*shape, 0, device=device), act8.encode(torch.ones(*shape, 40, device=device)))
        assert dw.shape == (0, 40) and db.shape == (0,)


@pytest.mark.parametrize("rows,cin,cout", [(4, 40, 0), (0, 40, 8), (4, 0, 8), (0, 0, 0)])
def test_linear_of_nothing(device, rows, cin, cout):
    grads = []
    for f in (act8.linear, F.linear):
        x = torch.ones(2, rows, cin, device=device, requires_grad=True)
        w, b = torch.ones(cout, cin, device=device, requires_grad=True), torch.ones(cout, device=device, requires_grad=True)
        y = f(x, w, b)
        y.backward(torch.ones_like(y))
        grads.append((y.detach(), x.grad, w.grad, b.grad))
    for a, c in zip(*grads):
        assert a.shape == c.shape and torch.equal(a, c)


def test_mlp_of_no_hidden_units(device):
    x = torch.ones(3, 8, device=device, requires_grad=True)
    w1, w2 = torch.ones(0, 8, device=device, requires_grad=True), torch.ones(5, 0, device=device, requires_grad=True)
    c = torch.ones(5, device=device, requires_grad=True)
    act8.mlp(x, w1, None, w2, c).sum().backward()
    assert not x.grad.any() and w1.grad.shape == (0, 8) and w2.grad.shape == (5, 0) and torch.equal(c.grad, torch.full_like(c, 3))
