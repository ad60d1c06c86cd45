"""The fine-tuning example: the operators together under the optimizer.

* A step's gradients equal those of the same model in plain torch (float32,
  nothing kept in 8 bits) within the 8-bit rounding: an int8 code is off by at
  most 2^-7 of its block's largest value, some 1 % of an element in the 2-norm
  for the roughly normal activations here, and errors of different elements
  average out; 3 % is asked for.
* Some steps on one batch raise what the loss rewards."""
import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

from sandmuon_amd import act8
from sandmuon_amd.losses import policy_loss
from sandmuon_amd.workloads import GPTConfig

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "sandmuon_amd" / "examples" / "finetune.py"
CFG = GPTConfig(vocab=97, ctx=48, layers=2, width=96, heads=3, mlp=264)


def example():
    spec = importlib.util.spec_from_file_location("finetune_example", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def plain_logits(policy, tokens, heads):
    """The example's model in elementary torch operations."""
    x = policy.transformer["wte"](tokens)
    cos, sin = (t[:tokens.shape[1]] for t in policy.tables)
    half = cos.shape[1]

    def norm_turn(v, w):  # [b, t, h, d]
        n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = n[..., :half], n[..., half:]
        c, s = cos[:, None], sin[:, None]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    lin = lambda m, v: F.linear(v, m.weight, m.bias)
    for block in policy.transformer["h"]:
        b, t, c = x.shape
        v0 = block.ln_1(x)
        at = block.attn
        q, k, v = (lin(m, v0).view(b, t, heads, -1) for m in (at.q_proj, at.k_proj, at.v_proj))
        q, k = norm_turn(q, at.q_norm), norm_turn(k, at.k_norm)
        q, k, v = (m.transpose(1, 2).contiguous() for m in (q, k, v))
        w = (q @ k.transpose(2, 3).contiguous()) / q.shape[-1] ** 0.5
        w = w.masked_fill(torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1), -torch.inf).softmax(-1)
        x = x + lin(at.c_proj, (w @ v).transpose(1, 2).reshape(b, t, c))
        x = x + lin(block.mlp["c_proj"], F.gelu(lin(block.mlp["c_fc"], block.ln_2(x))))
    return policy.transformer["ln_f"](x) @ policy.transformer["wte"].weight.t()


def test_gradients_match_plain_torch(device):
    module = example()
    torch.manual_seed(3)
    policy = module.Policy(CFG, device)
    tokens = torch.randint(0, CFG.vocab, (4, CFG.ctx), device=device)
    targets = torch.randint(0, CFG.vocab, (4, CFG.ctx), device=device)
    adv = torch.randn(4, CFG.ctx, device=device)
    loss, lp = policy_loss(policy(tokens), targets, adv)
    loss.backward()
    got = {n: p.grad.clone() for n, p in policy.named_parameters()}
    for p in policy.parameters():
        p.grad = None
    z = plain_logits(policy, tokens, CFG.heads)
    want_lp = torch.log_softmax(z, -1).gather(2, targets[..., None]).squeeze(2)
    want = -(torch.exp(want_lp - want_lp.detach()) * adv).mean()
    want.backward()
    assert abs(loss.item() - want.item()) < 1e-5
    assert torch.allclose(lp, want_lp.detach(), atol=1e-4)
    for n, p in policy.named_parameters():
        if n.endswith("k_proj.bias"):
            continue  # all but no gradient: a shift of every key alike, up to the norm
        rel = ((got[n] - p.grad).norm() / p.grad.norm()).item()
        assert rel < 3e-2, (n, rel)


@pytest.mark.parametrize("loss", ["policy", "preference"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_steps_raise_what_is_rewarded(device, loss, dtype):
    lines = []
    _, losses, gain = example().finetune(CFG, loss, batch=6, steps=5, dtype=dtype, report=lines.append)
    assert len(losses) == 5 and all(abs(v) < 10 for v in losses)
    assert losses[-1] < losses[0]
    assert (gain[:3] - gain[3:]).mean() > 0
    assert len(lines) == 6


def test_shared_kept_input(device):
    torch.manual_seed(0)
    a, b = torch.nn.Linear(64, 32).to(device), torch.nn.Linear(64, 48).to(device)
    x = torch.randn(20, 64, device=device)
    grads = []
    for shared in (False, True):
        for m in (a, b):
            m.weight.grad = m.bias.grad = None
        leaf = x.clone().requires_grad_()
        kept = act8.encode(leaf) if shared else None
        (act8.linear(leaf, a.weight, a.bias, kept=kept).sum() + act8.linear(leaf, b.weight, b.bias, kept=kept).sin().sum()).backward()
        grads.append([leaf.grad, a.weight.grad, a.bias.grad, b.weight.grad, b.bias.grad])
    assert all(torch.equal(p, q) for p, q in zip(*grads))
    with pytest.raises(ValueError, match="kept"):
        act8.linear(x[:10], a.weight, a.bias, kept=act8.encode(x))
