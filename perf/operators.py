"""What the speed of this framework's training operators is measured on: the loss over the vocabulary, the gated feed-forward block's
gradients and attention's gradients, over the sizes that its users meet.

  score        log-probabilities of given tokens: softmax cross entropy of x W^T, logits kept nowhere
  loss_grad    the same with the gradients of the rows and of the output weight
  ff_grad      gradients of down(act(gate(x)) * up(x)) by x and by the three weights
  attn_grad    gradients of rotated grouped-query attention by q, k and v

`run` computes them in their plain form, products, sums and exponentials in 32 bits over whole matrices, or, with `own`, by the
framework's entry points.  Widths are those of the benchmark's configuration where a case does not say otherwise; values are drawn on
the GPU from the seed, at the scale of a model in training: normed rows, weights of small spread, gradients of a mean over tokens."""
import math

import torch

own = False

WIDTH, VOCAB, FF, THETA = 2048, 32000, 5632, 10000.0
HEADS, KV_HEADS, DIM = 32, 4, 64
IGNORED = -100


def listed():
    return [
        # the answer to one question is scored, and the documents of an evaluation
        {"name": "score_64", "path": "score", "tokens": 64, "hidden": WIDTH, "vocab": VOCAB},
        {"name": "score_8192", "path": "score", "tokens": 8192, "hidden": WIDTH, "vocab": VOCAB},
        # a training step's loss: one short sequence, a narrow model with a vocabulary of no particular size, a whole batch
        {"name": "loss_grad_200", "path": "loss_grad", "tokens": 200, "hidden": WIDTH, "vocab": VOCAB},
        {"name": "loss_grad_1531_odd", "path": "loss_grad", "tokens": 1531, "hidden": 1000, "vocab": 10007},
        {"name": "loss_grad_8192", "path": "loss_grad", "tokens": 8192, "hidden": WIDTH, "vocab": VOCAB},
        # the feed-forward block of a short sequence, of a narrow model with GELU and odd sizes, of a whole batch
        {"name": "ff_grad_64", "path": "ff_grad", "tokens": 64, "hidden": WIDTH, "inter": FF, "act": "silu"},
        {"name": "ff_grad_1371_odd", "path": "ff_grad", "tokens": 1371, "hidden": 1000, "inter": 2712, "act": "gelu_tanh"},
        {"name": "ff_grad_16384", "path": "ff_grad", "tokens": 16384, "hidden": WIDTH, "inter": FF, "act": "silu"},
        # attention over one short sequence, heads of their own keys without a mask, a batch of documents of no particular length, a
        # batch of long ones
        {"name": "attn_grad_1x333", "path": "attn_grad", "batch": 1, "seq": 333, "heads": HEADS, "kv_heads": KV_HEADS, "offset": 0, "causal": True},
        {"name": "attn_grad_2x1000_full", "path": "attn_grad", "batch": 2, "seq": 1000, "heads": 8, "kv_heads": 8, "offset": 0, "causal": False},
        {"name": "attn_grad_3x1371", "path": "attn_grad", "batch": 3, "seq": 1371, "heads": HEADS, "kv_heads": KV_HEADS, "offset": 5, "causal": True},
        {"name": "attn_grad_8x2048", "path": "attn_grad", "batch": 8, "seq": 2048, "heads": HEADS, "kv_heads": KV_HEADS, "offset": 0, "causal": True},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    path = rng.choice(["score", "loss_grad", "ff_grad", "attn_grad", "loss_grad", "attn_grad"])
    if path in ("score", "loss_grad"):
        return {"path": path, "tokens": log_int(16, 8192), "hidden": 8 * rng.randint(32, 256), "vocab": log_int(1000, VOCAB)}
    if path == "ff_grad":
        return {"path": path, "tokens": log_int(16, 16384), "hidden": 8 * rng.randint(32, 256), "inter": 8 * rng.randint(64, 704),
                "act": rng.choice(["silu", "gelu_tanh"])}
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (32, 8), (16, 2), (8, 8), (12, 4), (4, 1)])
    causal = rng.random() < 0.8
    seq = log_int(16, 4096 if causal else 2048)
    most = 8 * HEADS * 2048 * 2048 // (1 if causal else 2)
    batch = log_int(1, min(8, max(1, most // (heads * seq * seq))))
    return {"path": path, "batch": batch, "seq": seq, "heads": heads, "kv_heads": kv_heads, "offset": rng.choice([0, 0, rng.randint(1, 1000)]),
            "causal": causal}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _normal(gen, *shape, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["path"] in ("score", "loss_grad"):
        tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        state["x"] = _normal(gen, tokens, hidden)
        state["weight"] = _normal(gen, vocab, hidden, std=2.0 / math.sqrt(hidden))
        targets = torch.randint(0, vocab, (tokens,), generator=gen, device="cuda")
        # padding and the tokens of the question have no loss
        ignored = torch.rand((tokens,), generator=gen, device="cuda") < 0.1
        state["targets"] = torch.where(ignored, torch.full_like(targets, IGNORED), targets).to(torch.int32)
        state["grad_loss"] = torch.full((tokens,), 1.0 / tokens, dtype=torch.float32, device="cuda")
    elif case["path"] == "ff_grad":
        tokens, hidden, inter = case["tokens"], case["hidden"], case["inter"]
        state["x"] = _normal(gen, tokens, hidden)
        state["gate"], state["up"] = (_normal(gen, inter, hidden, std=1.0 / math.sqrt(hidden)) for _ in range(2))
        state["down"] = _normal(gen, hidden, inter, std=1.0 / math.sqrt(inter))
        state["dy"] = _normal(gen, tokens, hidden, std=1.0 / tokens)
    else:
        batch, seq, heads, kv_heads = case["batch"], case["seq"], case["heads"], case["kv_heads"]
        state["q"] = _normal(gen, batch, seq, heads, DIM)
        state["k"], state["v"] = (_normal(gen, batch, seq, kv_heads, DIM) for _ in range(2))
        state["dout"] = _normal(gen, batch, seq, heads, DIM, std=1.0 / (batch * seq))
        # what the forward pass has left: its output, and the log of each row's sum of exponentials
        out, lse = zip(*(_attention(state["q"][b:b + 1], state["k"][b:b + 1], state["v"][b:b + 1], case) for b in range(batch)))
        state["out"], state["lse"] = torch.cat(out).to(torch.bfloat16), torch.cat(lse)
    return state


# --------------------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, offset, sign):
    """Pairs (2i, 2i + 1) of (batch, seq, heads, DIM) turned by sign * position * THETA ** (-2i / DIM)"""
    i = torch.arange(0, DIM, 2, dtype=torch.float64, device="cuda")
    angle = (torch.arange(x.shape[1], dtype=torch.float64, device="cuda") + offset)[:, None] * THETA ** (-i / DIM)
    c, s = torch.cos(angle)[:, None].to(x.dtype), (sign * torch.sin(angle))[:, None].to(x.dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)


def _grouped(q, k, v, case, dtype=torch.float32):
    """Rotated q (batch, kv heads, heads of a group, seq, DIM), rotated k and v (batch, kv heads, 1, seq, DIM)"""
    batch, seq, heads, _ = q.shape
    q, k = _rotate(q.to(dtype), case["offset"], 1), _rotate(k.to(dtype), case["offset"], 1)
    q = q.view(batch, seq, case["kv_heads"], heads // case["kv_heads"], DIM).permute(0, 2, 3, 1, 4)
    return q, k.permute(0, 2, 1, 3)[:, :, None], v.to(dtype).permute(0, 2, 1, 3)[:, :, None]


def _scores(q, k, case):
    s = q @ k.transpose(-1, -2) / math.sqrt(DIM)
    if case["causal"]:
        at = torch.arange(s.shape[-1], device="cuda")
        s = torch.where(at[None, :] <= at[:, None] + case["offset"], s, -math.inf)
    return s


def _attention(q, k, v, case):
    """(batch, seq, heads, DIM) and the log-sum-exp (batch, heads, seq)"""
    batch, seq, heads, _ = q.shape
    q, k, v = _grouped(q, k, v, case)
    s = _scores(q, k, case)
    lse = torch.logsumexp(s, dim=-1)
    out = torch.exp(s - lse[..., None]) @ v
    return out.permute(0, 3, 1, 2, 4).reshape(batch, seq, heads, DIM), lse.reshape(batch, heads, seq)


def _plain_attn_grad(state):
    case = state["case"]
    batch, seq, heads, kv_heads = case["batch"], case["seq"], case["heads"], case["kv_heads"]
    q, k, v = _grouped(state["q"], state["k"], state["v"], case)
    do = state["dout"].float().view(batch, seq, kv_heads, heads // kv_heads, DIM).permute(0, 2, 3, 1, 4)
    s = _scores(q, k, case)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(DIM)
    dq = (ds @ k).permute(0, 3, 1, 2, 4).reshape(batch, seq, heads, DIM)
    dk = (ds.transpose(-1, -2) @ q).sum(2).transpose(1, 2)
    return tuple(t.to(torch.bfloat16) for t in (_rotate(dq, case["offset"], -1), _rotate(dk, case["offset"], -1), dv.transpose(1, 2)))


def _plain_loss(x, weight, targets):
    """Loss of every row, the log-sum-exp, the logits and which rows count"""
    z = x @ weight.T
    top = z.amax(-1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(-1, keepdim=True)))[:, 0]
    counts = targets >= 0
    picked = z.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]
    return torch.where(counts, lse - picked, torch.zeros_like(lse)), lse, z, counts


def _plain_loss_grad(state):
    x, weight, targets = state["x"].float(), state["weight"].float(), state["targets"]
    loss, lse, z, counts = _plain_loss(x, weight, targets)
    dz = torch.exp(z - lse[:, None])
    dz.scatter_add_(1, targets.clamp(min=0).long()[:, None], -torch.ones_like(lse)[:, None])
    dz = dz * torch.where(counts, state["grad_loss"], torch.zeros_like(lse))[:, None]
    return loss, (dz @ weight).to(torch.bfloat16), (dz.T @ x).to(torch.bfloat16)


def _activation(z, act):
    """The activation and its derivative"""
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_ff_grad(state):
    x, dy, gate, up, down = (state[n].float() for n in ("x", "dy", "gate", "up", "down"))
    g, u, dh = x @ gate.T, x @ up.T, dy @ down
    a, slope = _activation(g, state["case"]["act"])
    dg, du = dh * u * slope, dh * a
    grads = dg @ gate + du @ up, dg.T @ x, du.T @ x, dy.T @ (a * u)
    return tuple(t.to(torch.bfloat16) for t in grads)


def run(state):
    case = state["case"]
    if own:
        from baranet_bdml_b200 import ops
        if case["path"] == "score":
            return ops.linear_cross_entropy(state["x"], state["weight"], state["targets"])
        if case["path"] == "loss_grad":
            loss, lse = ops.linear_cross_entropy(state["x"], state["weight"], state["targets"])
            return (loss,) + ops.linear_cross_entropy_backward(state["x"], state["weight"], state["targets"], lse, state["grad_loss"])
        if case["path"] == "ff_grad":
            return ops.gated_ff_backward(state["dy"], state["x"], state["gate"], state["up"], state["down"], act=case["act"])
        return ops.attn_prefill_bf16_backward(state["dout"], state["q"], state["k"], state["v"], state["out"], state["lse"], theta=THETA,
                                              position_offset=case["offset"], causal=case["causal"])
    if case["path"] == "score":
        return _plain_loss(state["x"].float(), state["weight"].float(), state["targets"])[:2]
    if case["path"] == "loss_grad":
        return _plain_loss_grad(state)
    return _plain_ff_grad(state) if case["path"] == "ff_grad" else _plain_attn_grad(state)


def work(case):
    if case["path"] in ("score", "loss_grad"):
        tokens, hidden, vocab = case["tokens"], case["hidden"], case["vocab"]
        rows, product = (tokens + vocab) * hidden * 2, 2 * tokens * vocab * hidden
        if case["path"] == "score":
            return {"bytes": rows + tokens * 12, "flops": product}
        return {"bytes": 2 * rows + tokens * 12, "flops": 3 * product}
    if case["path"] == "ff_grad":
        tokens, hidden, inter = case["tokens"], case["hidden"], case["inter"]
        return {"bytes": 2 * (3 * tokens * hidden + 6 * inter * hidden), "flops": 16 * tokens * inter * hidden}
    batch, seq, heads, kv_heads = case["batch"], case["seq"], case["heads"], case["kv_heads"]
    last = range(seq)
    pairs = sum(min(seq, i + case["offset"] + 1) for i in last) if case["causal"] else seq * seq
    return {"bytes": batch * seq * (heads * (4 * DIM * 2 + 4) + kv_heads * 4 * DIM * 2), "flops": 10 * batch * heads * pairs * DIM}


# ------------------------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    wide = {n: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for n, t in state.items()}
    if case["path"] in ("score", "loss_grad"):
        x, w, targets = wide["x"], wide["weight"], state["targets"].long()
        z = torch.einsum("th,vh->tv", x, w)
        lse = torch.logsumexp(z, 1)
        rows = torch.arange(case["tokens"], device="cuda")
        counted = (targets != IGNORED).double()
        label = torch.where(targets == IGNORED, 0, targets)
        loss = counted * (lse - z[rows, label])
        if case["path"] == "score":
            return loss, lse
        dz = torch.exp(z.sub_(lse[:, None]))
        dz[rows, label] -= 1
        dz *= (counted * wide["grad_loss"])[:, None]
        return loss, torch.einsum("tv,vh->th", dz, w), torch.einsum("tv,th->vh", dz, x)
    if case["path"] == "ff_grad":
        x, dy, gate, up, down = (wide[n] for n in ("x", "dy", "gate", "up", "down"))
        g = torch.einsum("th,ih->ti", x, gate).requires_grad_(True)
        u = torch.einsum("th,ih->ti", x, up).requires_grad_(True)
        act = torch.nn.functional.silu(g) if case["act"] == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
        h = act * u
        dg, du = torch.autograd.grad(h, (g, u), torch.einsum("th,hi->ti", dy, down))
        return (torch.einsum("ti,ih->th", dg, gate) + torch.einsum("ti,ih->th", du, up), torch.einsum("ti,th->ih", dg, x),
                torch.einsum("ti,th->ih", du, x), torch.einsum("th,ti->hi", dy, h.detach()))
    # attention of one sequence at a time, as complex rotations, differentiated by its own graph
    seq, group = case["seq"], case["heads"] // case["kv_heads"]
    position = torch.arange(seq, dtype=torch.float64, device="cuda") + case["offset"]
    freq = torch.tensor([THETA ** (-2.0 * i / DIM) for i in range(DIM // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones((seq, DIM // 2), dtype=torch.float64, device="cuda"), position[:, None] * freq[None])
    hidden = torch.ones((seq, seq), dtype=torch.bool, device="cuda").triu(1 + case["offset"]) if case["causal"] else None

    def turned(t):
        return torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (DIM // 2, 2)).contiguous()) * turn[:, None]).flatten(-2)

    grads = []
    for b in range(case["batch"]):
        leaves = [wide[n][b].clone().requires_grad_(True) for n in ("q", "k", "v")]
        qr, kr = turned(leaves[0]), turned(leaves[1])
        total = 0.0
        for h in range(case["kv_heads"]):
            for j in range(group):
                s = qr[:, h * group + j] @ kr[:, h].T * DIM ** -0.5
                if hidden is not None:
                    s = s.masked_fill(hidden, -math.inf)
                o = torch.softmax(s, -1) @ leaves[2][:, h]
                total = total + (o * wide["dout"][b, :, h * group + j]).sum()
        grads.append(torch.autograd.grad(total, leaves))
    return tuple(torch.stack(g) for g in zip(*grads))
