"""Fine-tuning a small GPT with the SandMuon optimizer by a policy or a
preference loss, on the training operators of this package:

* every Linear under ``transformer.h`` and the GELU between the MLP's keep their
  inputs in 8 bits (``act8.checkpoint_linears``, ``act8.gelu``); q, k and v share
  one kept input;
* queries and keys are normalised per head and turned by their positions in one
  pass (``attention.qk_norm_rotary``);
* the loss and its gradient to the logits come from ``losses``.

Synthetic tokens; a sequence's reward is the share of even tokens it holds (the
policy loss), or the sequence with more of them is the chosen one.

Usage: python sandmuon_amd/examples/finetune.py [--loss policy|preference]
           [--width 768 --layers 9 --heads 12 --mlp 3072 --vocab 50257 --seq 1024] [--batch 8] [--steps 4]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch
from torch import nn
from torch.nn import functional as F

if __package__ in (None, ""):
    sys.path.insert(0, str(Path(__file__).resolve().parents[2]))

from sandmuon_amd import RankOneAWeightedPE, act8  # noqa: E402
from sandmuon_amd.attention import qk_norm_rotary, rotary_tables  # noqa: E402
from sandmuon_amd.losses import policy_loss, preference_loss, token_logprobs  # noqa: E402
from sandmuon_amd.workloads import GPTConfig, transformer_filter  # noqa: E402


class Attention(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.heads = cfg.heads
        self.q_proj, self.k_proj, self.v_proj, self.c_proj = (nn.Linear(cfg.width, cfg.width) for _ in range(4))
        self.q_norm, self.k_norm = (nn.Parameter(torch.ones(cfg.width // cfg.heads)) for _ in range(2))

    def forward(self, x, tables):
        b, t, c = x.shape
        shared = {}
        if torch.is_grad_enabled():
            shared["kept"] = act8.encode(x)
        q, k, v = (proj(x, **shared).view(b, t, self.heads, -1) for proj in (self.q_proj, self.k_proj, self.v_proj))
        q, k = qk_norm_rotary(q, k, self.q_norm, self.k_norm, *tables)
        y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        return self.c_proj(y.transpose(1, 2).reshape(b, t, c))


class Block(nn.Module):
    def __init__(self, cfg: GPTConfig):
        super().__init__()
        self.ln_1, self.ln_2 = nn.LayerNorm(cfg.width), nn.LayerNorm(cfg.width)
        self.attn = Attention(cfg)
        self.mlp = nn.ModuleDict(dict(c_fc=nn.Linear(cfg.width, cfg.mlp), c_proj=nn.Linear(cfg.mlp, cfg.width)))

    def forward(self, x, tables):
        x = x + self.attn(self.ln_1(x), tables)
        h = self.mlp["c_fc"](self.ln_2(x))
        return x + self.mlp["c_proj"](act8.gelu(h))


class Policy(nn.Module):
    """A GPT with normalised, rotated queries and keys; tied embeddings."""

    def __init__(self, cfg: GPTConfig, device):
        super().__init__()
        self.transformer = nn.ModuleDict(dict(wte=nn.Embedding(cfg.vocab, cfg.width),
                                              h=nn.ModuleList([Block(cfg) for _ in range(cfg.layers)]),
                                              ln_f=nn.LayerNorm(cfg.width)))
        nn.init.normal_(self.transformer.wte.weight, std=0.02)
        self.to(device)
        self.tables = rotary_tables(cfg.ctx, cfg.width // cfg.heads, device=device)
        self.kept = act8.checkpoint_linears(self, transformer_filter)

    def forward(self, tokens):
        x = self.transformer.wte(tokens)
        for block in self.transformer.h:
            x = block(x, self.tables)
        return self.transformer.ln_f(x) @ self.transformer.wte.weight.t()


def finetune(cfg: GPTConfig, loss_name: str = "policy", batch: int = 8, steps: int = 4, lr: float = 3e-3, seed: int = 0,
             dtype: torch.dtype = torch.bfloat16, report=print):
    """`steps` steps on one batch; returns the policy, its loss of each step and
    the mean log probability of the good tokens' continuations before and after."""
    device = torch.device("cuda", 0)
    torch.manual_seed(seed)
    policy = Policy(cfg, device)
    optimizer = RankOneAWeightedPE(policy, lr, module_filter=transformer_filter)
    tokens = torch.randint(0, cfg.vocab, (batch, cfg.ctx + 1), device=device)
    # later sequences hold more even tokens, the chosen half of the batch most
    share = torch.linspace(0.9, 0.1, batch, device=device)[:, None]
    even = torch.rand(tokens.shape, device=device) < share
    tokens = torch.where(even, tokens // 2 * 2, tokens // 2 * 2 + 1).clamp(max=cfg.vocab - 1)
    inputs, targets = tokens[:, :-1].contiguous(), tokens[:, 1:].contiguous()
    mask = torch.arange(cfg.ctx, device=device).expand(batch, -1) >= cfg.ctx // 4  # the first quarter is the prompt
    reward = (targets % 2 == 0).float().mean(1)
    advantages = (reward - reward.mean()) / reward.std()

    def logits():
        with torch.autocast("cuda", dtype=dtype, enabled=dtype != torch.float32):
            return policy(inputs)

    with torch.no_grad():
        old = token_logprobs(logits(), targets, mask)
    losses = []
    for step in range(steps):
        torch.cuda.reset_peak_memory_stats()
        if loss_name == "policy":
            loss, lp = policy_loss(logits(), targets, advantages, old_logprobs=old, ref_logprobs=old, mask=mask,
                                   kl_coef=0.02)
        else:
            loss, margins = preference_loss(logits(), targets, old, mask=mask, beta=0.1)
        loss.backward()
        optimizer.step()
        optimizer.zero_grad(set_to_none=True)
        losses.append(loss.item())
        report(f"step {step}: {loss_name} loss {losses[-1]:+.5f}, peak memory "
               f"{torch.cuda.max_memory_allocated() / 2 ** 20:.0f} MiB")
    with torch.no_grad():
        gain = (token_logprobs(logits(), targets, mask) - old).sum(1)
    report(f"gain of the better half over the worse: {(gain[:batch // 2] - gain[batch // 2:]).mean().item():+.3f}")
    optimizer.close()
    return policy, losses, gain


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--loss", choices=("policy", "preference"), default="policy")
    for name, value in (("width", 128), ("layers", 2), ("heads", 4), ("mlp", 512), ("vocab", 97), ("seq", 64),
                        ("batch", 8), ("steps", 4)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args()
    cfg = GPTConfig(vocab=a.vocab, ctx=a.seq, layers=a.layers, width=a.width, heads=a.heads, mlp=a.mlp)
    finetune(cfg, a.loss, a.batch, a.steps)


if __name__ == "__main__":
    main()
