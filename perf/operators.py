"""The operators of a fine-tuning step around the optimizer, at the sizes they are used at.

Kinds of case:

* ``store``: an activation kept in 8 bits for the backward pass and read back.
* ``linear``: the input of a Linear kept in 8 bits, and the Linear's weight and
  bias gradients computed from it.
* ``gelu``: the exact GELU of an MLP's hidden layer, its input and output kept
  in 8 bits, and its gradient from the kept input.
* ``qk``: RMS norms of queries and keys per head with the rotary position
  rotation, forward and backward.
* ``qk_token``: the same for one new token of each sequence, forward only.
* ``policy``: the clipped policy loss with a KL term over a batch's logits, and
  its gradient to the logits.
* ``preference``: the preference loss of chosen and rejected sequences (paired
  log ratios) over their logits, and its gradient to the logits.

8-bit values: the elements of a row in blocks of 32 neighbours share a power of
two.  With E the exponent of the block's largest magnitude, ``int8`` holds
round(x / 2^(E-6)) in [-127, 127] and ``e4m3`` holds x / 2^(E-7) rounded to a
float of 4 exponent and 3 fraction bits.

Every quantity is drawn on the GPU from the seed.
"""
from __future__ import annotations

import math

import torch

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 32
EPS = 1e-6
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.05
BETA, SMOOTHING = 0.1, 0.05

own = False


# ------------------------------------------------------------------ cases ---
def _case(kind, name=None, **sizes):
    case = dict(kind=kind, **sizes)
    return dict(case, name=name) if name else case


def listed():
    return [
        # an evaluation-sized activation of odd sizes, checkpointed whole
        _case("store", "store-odd", rows=1023, cols=777, dtype="f16", fmt="e4m3"),
        # a full-precision Linear of odd sizes on a short ragged batch
        _case("linear", "linear-odd-f32", rows=1000, cin=300, cout=514, dtype="f32", grad="f32", fmt="int8"),
        # the q projection of the 103M GPT on 16 sequences of 1024
        _case("linear", "linear-103m-q", rows=16384, cin=768, cout=768, dtype="bf16", grad="f32", fmt="int8"),
        # c_fc of the 2048-wide GPT on 8 sequences of 1024
        _case("linear", "linear-2048-fc", rows=8192, cin=2048, cout=8192, dtype="bf16", grad="bf16", fmt="e4m3"),
        # the hidden layer of a small MLP of odd width, without autocast
        _case("gelu", "gelu-odd-f32", rows=999, cols=1100, dtype="f32", fmt="e4m3"),
        # the hidden layer of the 103M GPT on 16 sequences of 1024
        _case("gelu", "gelu-103m", rows=16384, cols=3072, dtype="bf16", fmt="int8"),
        # queries and keys of the 103M GPT on 16 sequences of 1024
        _case("qk", "qk-103m", batch=16, seq=1024, hq=12, hk=12, dim=64, rot=64, style="half", dtype="bf16"),
        # a sampling step of the 2048-wide GPT, 64 sequences, with shared key heads
        _case("qk_token", "qk-token", batch=64, hq=16, hk=4, dim=128, rot=128, style="half", dtype="bf16"),
        # a character-level policy: the vocabulary of the tiny GPT
        _case("policy", "policy-tiny", batch=4, seq=16, vocab=97, dtype="f32", reduction="sequence"),
        # 8 completions of the 103M GPT
        _case("policy", "policy-103m", batch=8, seq=1024, vocab=50257, dtype="bf16", reduction="token"),
        # pairs of short sequences over a small odd vocabulary
        _case("preference", "preference-small", pairs=3, seq=200, vocab=1031, dtype="f16"),
        # 4 pairs of sequences of the 103M GPT
        _case("preference", "preference-103m", pairs=4, seq=1024, vocab=50257, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly over [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choice(["store", "linear", "gelu", "qk", "qk_token", "policy", "preference"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    fmt = rng.choice(["int8", "e4m3"])
    if kind in ("store", "gelu"):
        rows = _spread(rng, 1, 16384)
        return _case(kind, rows=rows, cols=_spread(rng, 8, 8192), dtype=dtype, fmt=fmt)
    if kind == "linear":
        cin, cout = _spread(rng, 16, 8192), _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(16384, 8192 * 8192 * 2048 // (cin * cout)))
        return _case(kind, rows=rows, cin=cin, cout=cout, dtype=dtype, grad=rng.choice(["f32", dtype]), fmt=fmt)
    if kind in ("qk", "qk_token"):
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        hk = rng.choice([1, 2, 3, 4, 8])
        sizes = dict(hq=hk * rng.choice([1, 2, 4]), hk=hk, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                     style=rng.choice(["half", "half", "interleaved"]), dtype=dtype)
        if kind == "qk_token":
            return _case(kind, batch=_spread(rng, 1, 512), **sizes)
        return _case(kind, batch=_spread(rng, 1, 16), seq=_spread(rng, 1, 2048), **sizes)
    vocab = _spread(rng, 64, 131072)
    most = 8 * 1024 * 50257 // vocab
    if kind == "policy":
        batch = _spread(rng, 1, 8)
        return _case(kind, batch=batch, seq=_spread(rng, 1, min(2048, most // batch)), vocab=vocab, dtype=dtype,
                     reduction=rng.choice(["token", "sequence"]))
    pairs = _spread(rng, 1, 4)
    return _case(kind, pairs=pairs, seq=_spread(rng, 1, min(2048, most // (2 * pairs))), vocab=vocab, dtype=dtype)


# ---------------------------------------------------------------- prepare ---
def _activation(g, rows, cols, dtype):
    """Channels of means and scales of their own, as hidden states have them."""
    sigma = torch.exp(torch.empty(cols, device=DEVICE).uniform_(math.log(0.1), math.log(10.0), generator=g))
    mu = torch.randn(cols, device=DEVICE, generator=g) * 0.3
    return (torch.randn(rows, cols, device=DEVICE, generator=g) * sigma + mu).to(dtype)


def _cotangent(g, rows, cols, dtype):
    """Gradients whose scale differs from token to token."""
    scale = torch.exp(torch.randn(rows, 1, device=DEVICE, generator=g)) * 1e-2
    return (torch.randn(rows, cols, device=DEVICE, generator=g) * scale).to(dtype)


def _tables(positions, rot):
    """cos and sin [positions, rot / 2] of the rotary angles."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
    angle = torch.arange(positions, device=DEVICE, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _live(batch, seq):
    """Prompt lengths: from none to 3/5 of the sequence, evenly spread."""
    return [min(seq - 1, int(seq * 0.6 * b / max(1, batch - 1))) for b in range(batch)]


def _batch(g, batch, seq, vocab, dtype):
    """Logits [batch, seq, vocab] that favour their targets, the targets, the
    mask of the completions and the log probabilities of the targets."""
    logits = torch.randn(batch, seq, vocab, device=DEVICE, generator=g).mul_(2.0).to(dtype)
    targets = torch.randint(0, vocab, (batch, seq), device=DEVICE, generator=g)
    at = targets[..., None]
    logits.scatter_(2, at, logits.gather(2, at) + math.log(vocab))
    order = torch.randperm(batch, device=DEVICE, generator=g)
    prompt = torch.tensor(_live(batch, seq), device=DEVICE)[order]
    mask = torch.arange(seq, device=DEVICE)[None, :] >= prompt[:, None]
    logp = torch.stack([row.gather(1, y[:, None]).squeeze(1).float() - torch.logsumexp(row.float(), 1)
                        for row, y in zip(logits, targets)])
    return logits, targets, mask, logp


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    state = dict(case=case)
    if kind == "store":
        state["x"] = _activation(g, case["rows"], case["cols"], dtype)
    elif kind == "linear":
        state["x"] = _activation(g, case["rows"], case["cin"], dtype)
        state["delta"] = _cotangent(g, case["rows"], case["cout"], dtype)
    elif kind == "gelu":
        h = torch.randn(case["rows"], case["cols"], device=DEVICE, generator=g) * 1.5 - 0.3
        state["h"] = h.to(dtype)
        state["dy"] = _cotangent(g, case["rows"], case["cols"], dtype)
    elif kind in ("qk", "qk_token"):
        b, t, d = case["batch"], case.get("seq", 1), case["dim"]
        for name, heads in (("q", case["hq"]), ("k", case["hk"])):
            state[name] = _activation(g, b * t, heads * d, dtype).view(b, t, heads, d)
            state["w" + name] = 1 + 0.2 * torch.randn(d, device=DEVICE, generator=g)
            state["d" + name] = _cotangent(g, b * t, heads * d, dtype).view(b, t, heads, d)
        longest = 4096
        state["cos"], state["sin"] = _tables(longest, case["rot"])
        state["positions"] = None
        if kind == "qk_token":
            state["positions"] = torch.randint(0, longest, (b, 1), device=DEVICE, generator=g)
    elif kind == "policy":
        logits, targets, mask, logp = _batch(g, case["batch"], case["seq"], case["vocab"], dtype)
        # the policy that sampled is a few steps old; no ratio within 1e-3 of a clip
        step = torch.randn(logp.shape, device=DEVICE, generator=g) * 0.15
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            step = torch.where((step - edge).abs() < 1e-3, step + 4e-3, step)
        state.update(logits=logits, targets=targets, mask=mask, old=logp - step,
                     ref=logp + torch.randn(logp.shape, device=DEVICE, generator=g) * 0.3,
                     advantages=torch.randn(case["batch"], device=DEVICE, generator=g))
    else:
        logits, targets, mask, logp = _batch(g, 2 * case["pairs"], case["seq"], case["vocab"], dtype)
        state.update(logits=logits, targets=targets, mask=mask,
                     ref=logp + torch.randn(logp.shape, device=DEVICE, generator=g) * 0.3)
    return state


# ------------------------------------------------------------- plain form ---
def _power(field):
    """2^(field - 127) of whole numbers in [1, 254]."""
    return (field << 23).view(torch.float32)


def _held(x, fmt):
    """The values that 8 bits an element and one byte a block of 32 stand for."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, BLOCK)
    top = (v.abs().amax(2, keepdim=True).view(torch.int32) >> 23) & 255
    if fmt == "int8":
        scale = _power((top - 6).clamp(min=1))
        held = torch.round(v / scale).clamp(-127, 127) * scale
    else:
        scale = _power((top - 7).clamp(min=10))
        v = v / scale
        # a step is 2^-3 of the element's power of two, 2^-9 at the least
        step = _power((((v.abs().view(torch.int32) >> 23) & 255) - 3).clamp(min=127 - 9))
        held = torch.round(v / step) * step * scale
    return held.view(rows, cols + pad)[:, :cols]


def _phi(h):
    return 0.5 * (1 + torch.erf(h * math.sqrt(0.5)))


def _pairs(x, rot, style):
    if style == "half":
        return x[..., :rot // 2], x[..., rot // 2:rot]
    return x[..., 0:rot:2], x[..., 1:rot:2]


def _unpaired(a, b, rest, style):
    if style == "half":
        return torch.cat([a, b, rest], -1)
    return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)


def _angles(state):
    b, t = state["q"].shape[:2]
    pos = state["positions"]
    if pos is None:
        pos = torch.arange(t, device=DEVICE).expand(b, t)
    return state["cos"][pos][:, :, None], state["sin"][pos][:, :, None]


def _norm_rotate(x, w, cos, sin, rot, style):
    f = x.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * w
    a, b = _pairs(n, rot, style)
    return _unpaired(a * cos - b * sin, a * sin + b * cos, n[..., rot:], style).to(x.dtype)


def _norm_rotate_back(x, w, cos, sin, rot, style, dy):
    f, g = x.float(), dy.float()
    a, b = _pairs(g, rot, style)
    g = _unpaired(a * cos + b * sin, b * cos - a * sin, g[..., rot:], style)
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    unit = f * r
    gw = g * w
    dx = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
    return dx.to(x.dtype), (g * unit).sum((0, 1, 2)).to(w.dtype)


def _log_probs(z, targets):
    """Log probability of the targets and softmax of the logits, in FP32."""
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    lp = (z.gather(-1, targets[..., None]) - top - torch.log(total)).squeeze(-1)
    return lp, e / total


def _to_logits(p, targets, weight, dtype):
    """weight * (onehot - p), rounded to the logits' type."""
    d = p * -weight[..., None]
    d.scatter_add_(-1, targets[..., None], weight[..., None])
    return d.to(dtype)


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "store":
        return {"x": _held(state["x"], case["fmt"]).to(state["x"].dtype)}
    if kind == "linear":
        delta = state["delta"].float()
        grad = DTYPES[case["grad"]]
        return {"dw": (delta.t() @ _held(state["x"], case["fmt"])).to(grad), "db": delta.sum(0).to(grad)}
    if kind == "gelu":
        h, dtype = state["h"].float(), state["h"].dtype
        y = (h * _phi(h)).to(dtype)
        kept = _held(state["h"], case["fmt"])
        slope = _phi(kept) + kept * torch.exp(-0.5 * kept * kept) * (1 / math.sqrt(2 * math.pi))
        return {"y": y, "held": _held(y, case["fmt"]).to(torch.bfloat16), "dh": (state["dy"].float() * slope).to(dtype)}
    if kind in ("qk", "qk_token"):
        cos, sin = _angles(state)
        rot, style = case["rot"], case["style"]
        out = {n: _norm_rotate(state[n], state["w" + n], cos, sin, rot, style) for n in ("q", "k")}
        if kind == "qk":
            for n in ("q", "k"):
                out["d" + n], out["dw" + n] = _norm_rotate_back(state[n], state["w" + n], cos, sin, rot, style,
                                                                state["d" + n])
        return out
    logits, targets, mask = state["logits"], state["targets"], state["mask"]
    lp, p = _log_probs(logits.float(), targets)
    live = mask.float()
    if kind == "policy":
        if case["reduction"] == "token":
            weight = live / live.sum()
        else:
            each = live.sum(1, keepdim=True)
            weight = live / each / (each > 0).sum()
        adv = state["advantages"][:, None]
        ratio = torch.exp(lp - state["old"])
        clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
        gap = state["ref"] - lp
        loss = (weight * (KL * (torch.exp(gap) - gap - 1) - torch.minimum(ratio * adv, clipped * adv))).sum()
        moves = torch.where(adv > 0, ratio <= 1 + CLIP_HIGH, ratio >= 1 - CLIP_LOW)
        back = weight * (KL * (1 - torch.exp(gap)) - torch.where(moves, ratio * adv, 0.0))
        return {"loss": loss, "logprobs": lp * live, "dlogits": _to_logits(p, targets, back, logits.dtype)}
    pairs = case["pairs"]
    gain = ((lp - state["ref"]) * live).sum(1)
    margin = BETA * (gain[:pairs] - gain[pairs:])
    soft = torch.log1p(torch.exp(-margin.abs()))
    loss = ((1 - SMOOTHING) * (soft - margin.clamp(max=0)) + SMOOTHING * (soft + margin.clamp(min=0))).mean()
    up = 1 / (1 + torch.exp(-margin))
    slope = BETA * (up - (1 - SMOOTHING)) / pairs
    back = torch.cat([slope, -slope])[:, None] * live
    return {"loss": loss, "margins": margin, "dlogits": _to_logits(p, targets, back, logits.dtype)}


# --------------------------------------------------------- the framework's ---
def _own(state):
    case = state["case"]
    kind = case["kind"]
    if kind in ("store", "linear", "gelu"):
        from sandmuon_amd import act8
        if kind == "store":
            return {"x": act8.decode(act8.encode(state["x"], case["fmt"]), state["x"].dtype)}
        if kind == "linear":
            saved = act8.encode(state["x"], case["fmt"])
            dw, db = act8.linear_backward(state["delta"], saved, dtype=DTYPES[case["grad"]])
            return {"dw": dw, "db": db}
        y, saved_h, saved_y = act8.gelu_forward(state["h"], case["fmt"])
        return {"y": y, "held": act8.decode(saved_y), "dh": act8.gelu_backward(state["dy"], saved_h)}
    if kind in ("qk", "qk_token"):
        from sandmuon_amd.attention import qk_norm_rotary
        rest = dict(positions=state["positions"], eps=EPS, style=case["style"])
        if kind == "qk_token":
            q, k = qk_norm_rotary(state["q"], state["k"], state["wq"], state["wk"], state["cos"], state["sin"], **rest)
            return {"q": q, "k": k}
        leaves = [state[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
        q, k = qk_norm_rotary(*leaves, state["cos"], state["sin"], **rest)
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), leaves, (state["dq"], state["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    from sandmuon_amd import losses
    logits = state["logits"].detach().requires_grad_()
    if kind == "policy":
        loss, logprobs = losses.policy_loss(logits, state["targets"], state["advantages"],
                                            old_logprobs=state["old"], ref_logprobs=state["ref"], mask=state["mask"],
                                            clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL,
                                            reduction=case["reduction"])
        dlogits, = torch.autograd.grad(loss, logits)
        return {"loss": loss.detach(), "logprobs": logprobs, "dlogits": dlogits}
    loss, margins = losses.preference_loss(logits, state["targets"], state["ref"], mask=state["mask"], beta=BETA,
                                           label_smoothing=SMOOTHING)
    dlogits, = torch.autograd.grad(loss, logits)
    return {"loss": loss.detach(), "margins": margins, "dlogits": dlogits}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------- work ---
def work(case):
    kind, e = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "store":
        n = case["rows"] * case["cols"]
        return dict(bytes=2 * n * e, flops=4.0 * n)
    if kind == "linear":
        m, k, n = case["rows"], case["cin"], case["cout"]
        return dict(bytes=m * (k + n) * e + (n * k + n) * DTYPES[case["grad"]].itemsize, flops=2.0 * m * n * k)
    if kind == "gelu":
        n = case["rows"] * case["cols"]
        return dict(bytes=n * (4 * e + 2), flops=30.0 * n)  # h, dy; y, dh; what is held of y
    if kind in ("qk", "qk_token"):
        heads = case["batch"] * case.get("seq", 1) * (case["hq"] + case["hk"])
        n = heads * case["dim"]
        tables = min(4096, case["batch"] if kind == "qk_token" else case["seq"]) * case["rot"] * 4
        passes = 2 if kind == "qk_token" else 4  # q, k and their results; their gradients and the results'
        return dict(bytes=passes * n * e + tables + 8 * case["dim"], flops=(8.0 if passes == 2 else 24.0) * n)
    batch = case["batch"] if kind == "policy" else 2 * case["pairs"]
    rows, vocab = batch * case["seq"], case["vocab"]
    live = rows - sum(_live(batch, case["seq"]))
    per_row = 8 + 1 + 4 * (3 if kind == "policy" else 1)
    # a masked row's logits need not be read, its gradient is zero
    return dict(bytes=(live + rows) * vocab * e + rows * per_row, flops=6.0 * live * vocab)


# ------------------------------------------------------------------ exact ---
def _two(e):
    """2^e of whole numbers in 64 bits."""
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _held64(x, fmt):
    """_held's definition in 64 bits, from the mantissas and exponents of frexp."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    v = torch.cat([x.double(), x.new_zeros(rows, pad, dtype=torch.float64)], 1).reshape(-1, BLOCK)
    low, under = (-126, 6) if fmt == "int8" else (-117, 7)
    peak = v.abs().max(1, keepdim=True).values
    e = torch.where(peak > 0, torch.frexp(peak)[1] - 1 - under, low).clamp(min=low)
    v = v * _two(-e)
    if fmt == "int8":
        v = v.round().clamp(-127, 127)
    else:
        unit = torch.where(v == 0, -9, torch.frexp(v)[1] - 4).clamp(min=-9)
        v = (v * _two(-unit)).round() * _two(unit)
    return (v * _two(e)).reshape(rows, cols + pad)[:, :cols].contiguous()


def exact(case, seed):
    state = prepare(case, seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "store":
        return {"x": _held64(state["x"], case["fmt"])}
    if kind == "linear":
        delta = state["delta"].double()
        return {"dw": delta.t().contiguous() @ _held64(state["x"], case["fmt"]), "db": delta.sum(0)}
    if kind == "gelu":
        h = state["h"].double()
        y = h * torch.special.ndtr(h)
        kept = _held64(state["h"], case["fmt"])
        slope = torch.special.ndtr(kept) + kept * torch.exp(-kept.square() / 2) / math.sqrt(2 * math.pi)
        return {"y": y, "held": _held64(y.to(dtype), case["fmt"]), "dh": state["dy"].double() * slope}
    if kind in ("qk", "qk_token"):
        return _exact_qk(state, case)
    batch = case["batch"] if kind == "policy" else 2 * case["pairs"]
    logits, targets, mask = state["logits"], state["targets"], state["mask"]
    lp = torch.stack([torch.log_softmax(logits[b].double(), -1).gather(1, targets[b, :, None]).squeeze(1)
                      for b in range(batch)])
    lp.requires_grad_()
    live = mask.double()
    kept = torch.where(mask, lp, 0.0)
    if kind == "policy":
        old, ref, adv = state["old"].double(), state["ref"].double(), state["advantages"].double()[:, None]
        ratio = (lp - old).exp()
        term = -torch.min(ratio * adv, ratio.clip(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv)
        term = term + KL * ((ref - lp).expm1() - (ref - lp))
        if case["reduction"] == "token":
            loss = (term * live).sum() / live.sum()
        else:
            has = live.sum(1) > 0
            loss = ((term * live).sum(1)[has] / live.sum(1)[has]).mean()
        first = {"loss": loss, "logprobs": kept.detach()}
    else:
        gain = (torch.where(mask, lp - state["ref"].double(), 0.0)).sum(1)
        margin = BETA * (gain[:case["pairs"]] - gain[case["pairs"]:])
        sig = torch.nn.functional.logsigmoid
        loss = -((1 - SMOOTHING) * sig(margin) + SMOOTHING * sig(-margin)).mean()
        first = {"loss": loss, "margins": margin.detach()}
    back, = torch.autograd.grad(loss, lp)
    first["loss"] = loss.detach()
    dlogits = torch.empty(logits.shape, dtype=torch.float64, device=DEVICE)
    for b in range(batch):
        torch.mul(torch.softmax(logits[b].double(), -1), -back[b, :, None], out=dlogits[b])
        dlogits[b].scatter_add_(1, targets[b, :, None], back[b, :, None])
    return dict(first, dlogits=dlogits)


def _exact_qk(state, case):
    """The pairs as complex numbers in 64 bits, the gradients by autograd."""
    b, t = state["q"].shape[:2]
    rot = case["rot"]
    pos = state["positions"] if state["positions"] is not None else torch.arange(t, device=DEVICE).repeat(b, 1)
    turn = torch.complex(state["cos"].double(), state["sin"].double())[pos].unsqueeze(2)
    out = {}
    for n in ("q", "k"):
        x = state[n].double().requires_grad_()
        w = state["w" + n].double().requires_grad_()
        unit = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS) * w
        head, tail = unit.split([rot, case["dim"] - rot], -1)
        if case["style"] == "half":
            z = torch.complex(head[..., :rot // 2], head[..., rot // 2:]) * turn
            y = torch.cat([z.real, z.imag, tail], -1)
        else:
            z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
            y = torch.cat([torch.view_as_real(z).flatten(-2), tail], -1)
        out[n] = y.detach()
        if case["kind"] == "qk":
            out["d" + n], out["dw" + n] = torch.autograd.grad(y, (x, w), state["d" + n].double())
    return out
