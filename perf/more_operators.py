"""What the speed of this framework's serving operators over a cache in 8 bits is measured on, and of its sampling:

  write    new tokens of every sequence into a paged cache of 8 bits (keys rotated, a scale for each token and key head), read back
  read     whole sequences out of such a cache
  decode   one new token of every sequence against its cached keys and values
  sample   token ids from logits and random numbers: temperature, top-k, top-p, min-p

`run` computes them in their plain form, or, with `own`, by the framework's entry points.  Head counts are those of the benchmark's
configuration where a case does not say otherwise; values are drawn on the GPU from the seed.

A block of the cache, (page, key head), is 2112 bytes: the keys of 16 tokens, 64 bytes each; their values, of which the 16-byte piece
c of token t lies in place c ^ (t // 2 % 4); 16 pairs (key scale, value scale) of bf16."""
import math

import torch

own = False

HEADS, KV_HEADS, DIM, THETA, VOCAB = 32, 4, 64, 10000.0, 32000
PAGE, BLOCK = 16, 2112
LEAST, MOST = 2.0 ** -100, 2.0 ** 122                  # of a scale


def listed():
    return [
        # a decode step of a serving batch; prompts as they come in: a batch of short ones, three of no particular length that continue
        # cached ones, a batch of long ones
        {"name": "write_64x1", "path": "write", "values": "e4m3", "batch": 64, "seq": 1, "kv_heads": KV_HEADS, "longest": 4096},
        {"name": "write_3x1371_odd", "path": "write", "values": "int8", "batch": 3, "seq": 1371, "kv_heads": 8, "longest": 2000},
        {"name": "write_8x2048", "path": "write", "values": "e4m3", "batch": 8, "seq": 2048, "kv_heads": KV_HEADS, "longest": 2048},
        # one cached prompt, and all of a serving batch (to move it, or to go on with it elsewhere)
        {"name": "read_1x333", "path": "read", "values": "int8", "batch": 1, "kv_heads": KV_HEADS, "shortest": 333, "longest": 333},
        {"name": "read_64", "path": "read", "values": "e4m3", "batch": 64, "kv_heads": KV_HEADS, "shortest": 1024, "longest": 4096},
        # attention of one user's short conversation, of a batch behind its prompts, of a serving batch of unequal sequences, of few long ones
        {"name": "decode_1x100", "path": "decode", "values": "e4m3", "batch": 1, "heads": HEADS, "kv_heads": KV_HEADS, "shortest": 100, "longest": 100},
        {"name": "decode_16x576", "path": "decode", "values": "int8", "batch": 16, "heads": HEADS, "kv_heads": KV_HEADS, "shortest": 513,
         "longest": 576},
        {"name": "decode_64", "path": "decode", "values": "e4m3", "batch": 64, "heads": HEADS, "kv_heads": KV_HEADS, "shortest": 1024, "longest": 4096},
        {"name": "decode_4_long", "path": "decode", "values": "int8", "batch": 4, "heads": HEADS, "kv_heads": KV_HEADS, "shortest": 262144,
         "longest": 262144},
        # one user with the usual settings, a batch with each its own and some ids forbidden, a large batch that keeps all but the unlikely
        {"name": "sample_1_k50", "path": "sample", "rows": 1, "vocab": VOCAB, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0,
         "each": False, "forbidden": 0.0},
        {"name": "sample_37_each", "path": "sample", "rows": 37, "vocab": 10007, "temperature": 1.0, "top_k": 200, "top_p": 0.9, "min_p": 0.02,
         "each": True, "forbidden": 0.3},
        {"name": "sample_256_p90", "path": "sample", "rows": 256, "vocab": VOCAB, "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "each": False, "forbidden": 0.0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    path = rng.choice(["write", "read", "decode", "sample", "decode", "sample"])
    if path == "sample":
        vocab = log_int(100, 131072)
        return {"path": path, "rows": log_int(1, min(256, 256 * VOCAB // vocab)), "vocab": vocab, "temperature": round(rng.uniform(0.2, 1.5), 2),
                "top_k": rng.choice([0, 0, log_int(1, 1000)]), "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 2)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 3)]), "each": rng.random() < 0.3,
                "forbidden": rng.choice([0.0, 0.0, 0.5])}
    values = rng.choice(["e4m3", "int8"])
    if path == "write":
        seq = rng.choice([1, log_int(2, 4096)])
        batch = log_int(1, min(256, 16384 // seq))
        return {"path": path, "values": values, "batch": batch, "seq": seq, "kv_heads": rng.choice([4, 4, 1, 2, 8]) if batch * seq <= 8192 else 4,
                "longest": seq + log_int(1, 4096)}
    if path == "read":
        longest = log_int(16, 8192)
        return {"path": path, "values": values, "batch": log_int(1, min(64, 131072 // longest)), "kv_heads": rng.choice([4, 4, 1, 2]),
                "shortest": max(1, longest // rng.randint(1, 8)), "longest": longest}
    longest = log_int(16, 262144)
    heads, kv_heads = rng.choice([(32, 4), (32, 4), (16, 2), (12, 4), (4, 4), (8, 1), (6, 2)])
    return {"path": path, "values": values, "batch": log_int(1, min(256, 1048576 // longest)), "heads": heads, "kv_heads": kv_heads,
            "shortest": max(1, longest // rng.randint(1, 8)), "longest": longest}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _quantise(x, values):
    """The 8-bit values of x (..., DIM) fp32 and their scales (...)"""
    most = x.abs().amax(-1)
    if values == "e4m3":
        # the smallest power of two that leaves no more than 448 = 1.75 * 2 ** 8
        m, e = torch.frexp(most)
        scale = torch.ldexp(torch.ones_like(most), e - 9 + (m > 0.875).int()).clamp(LEAST, MOST)
        return (x / scale[..., None]).to(torch.float8_e4m3fn), scale
    scale = most / 127
    near = scale.to(torch.bfloat16)                    # rounded up to bf16
    up = (near.view(torch.int16) + (near.float() < scale).to(torch.int16)).view(torch.bfloat16)
    scale = up.float().clamp(LEAST, MOST)
    return torch.round(x / scale[..., None]).to(torch.int8), scale


def _places():
    """(PAGE, DIM): which byte of a token's values in a block holds element d"""
    t, d = torch.arange(PAGE, device="cuda")[:, None], torch.arange(DIM, device="cuda")[None]
    return (d // 16 ^ t // 2 % 4) * 16 + d % 16


def _pages(case, gen):
    """A cache that holds case["longest"] tokens a sequence, its pages in no particular order: (pages, table)"""
    per_seq = -(-case["longest"] // PAGE)
    pages = case["batch"] * per_seq
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(case["batch"], per_seq)
    return pages, table


def _filled(case, pages, gen):
    """A pool of random keys and values: norm 1 an element, some tokens larger, keys and values of other sizes"""
    pool = torch.empty((pages, case["kv_heads"], BLOCK), dtype=torch.uint8, device="cuda")
    places = _places()
    for at in range(0, pages, 16384):
        part = pool[at:at + 16384]
        scales = torch.empty((*part.shape[:2], PAGE, 2), dtype=torch.bfloat16, device="cuda")
        for i, size in enumerate((1.0, 0.5)):
            x = torch.randn((*part.shape[:2], PAGE, DIM), generator=gen, device="cuda") * size
            x *= torch.exp(0.3 * torch.randn((*part.shape[:2], PAGE, 1), generator=gen, device="cuda"))
            q, s = _quantise(x, case["values"])
            q = q.view(torch.uint8)
            if i == 1:
                q = torch.empty_like(q).scatter_(-1, places.expand_as(q), q)
            part[..., 1024 * i:1024 * (i + 1)] = q.flatten(-2)
            scales[..., i] = s.to(torch.bfloat16)
        part[..., 2048:] = scales.view(torch.uint8).flatten(-2)
    return pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    if case["path"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a few likely ids over a broad rest, as a model's logits have them
        logits = 2.5 * torch.randn((rows, vocab), generator=gen, device="cuda")
        logits += 6 * (torch.rand((rows, vocab), generator=gen, device="cuda") < 20 / vocab)
        if case["forbidden"]:
            out = torch.rand((rows, vocab), generator=gen, device="cuda") < case["forbidden"]
            logits = torch.where(out, torch.full_like(logits, -math.inf), logits)
        state["logits"] = logits
        state["uniform"] = torch.rand((rows,), generator=gen, device="cuda")
        for name in ("temperature", "top_k", "top_p", "min_p"):
            if not case["each"]:
                state[name] = case[name]
                continue
            spread = torch.rand((rows,), generator=gen, device="cuda")
            if name == "top_k":
                state[name] = (case[name] * (0.5 + spread)).to(torch.int32)
            else:
                state[name] = case[name] * (0.5 + 0.5 * spread)
        return state
    batch, kv_heads = case["batch"], case["kv_heads"]
    pages, state["table"] = _pages(case, gen)
    if case["path"] == "write":
        seq, before = case["seq"], case["longest"] - case["seq"]
        state["pool"] = torch.zeros((pages, kv_heads, BLOCK), dtype=torch.uint8, device="cuda")
        state["starts"] = torch.randint(before // 2, before + 1, (batch,), generator=gen, device="cuda").to(torch.int32)
        state["positions"] = (state["starts"][:, None] + torch.arange(seq, dtype=torch.int32, device="cuda")).flatten()
        state["rows"] = torch.arange(batch, dtype=torch.int32, device="cuda")
        state["seq_ids"] = state["rows"].repeat_interleave(seq)
        state["k"], state["v"] = (torch.randn((batch * seq, kv_heads * DIM), generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
        return state
    state["pool"] = _filled(case, pages, gen)
    state["lens"] = torch.randint(case["shortest"], case["longest"] + 1, (batch,), generator=gen, device="cuda").to(torch.int32)
    state["rows"], state["starts"] = torch.arange(batch, dtype=torch.int32, device="cuda"), torch.zeros((batch,), dtype=torch.int32, device="cuda")
    if case["path"] == "decode":
        state["q"] = torch.randn((batch, case["heads"], DIM), generator=gen, device="cuda").to(torch.bfloat16)
    return state


# --------------------------------------------------------------------------------------------------------------- plain forms
def _rotate(x, positions):
    """Pairs (2i, 2i + 1) of (tokens, heads, DIM) turned by position * THETA ** (-2i / DIM), the angle in 64 bits"""
    i = torch.arange(0, DIM, 2, dtype=torch.float64, device="cuda")
    angle = positions.double()[:, None] * THETA ** (-i / DIM)
    c, s = torch.cos(angle)[:, None].to(x.dtype), torch.sin(angle)[:, None].to(x.dtype)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)


def _plain_write(state):
    case = state["case"]
    batch, seq, kv_heads = case["batch"], case["seq"], case["kv_heads"]
    k, v = (state[n].float().view(batch * seq, kv_heads, DIM) for n in ("k", "v"))
    read = []
    for x in (_rotate(k, state["positions"]), v):
        q, scale = _quantise(x, case["values"])
        read.append((q.float() * scale[..., None]).to(torch.bfloat16).view(batch, seq, kv_heads, DIM))
    return tuple(read)


def _tokens(blocks, values):
    """The keys and values in blocks (..., BLOCK), fp32 (..., PAGE, DIM), and their scales (..., PAGE)"""
    dtype = torch.float8_e4m3fn if values == "e4m3" else torch.int8
    k, v = (blocks[..., a:a + 1024].contiguous().view(dtype).float().unflatten(-1, (PAGE, DIM)) for a in (0, 1024))
    v = v.gather(-1, _places().expand_as(v))
    scales = blocks[..., 2048:].contiguous().view(torch.bfloat16).float().unflatten(-1, (PAGE, 2))
    return k, v, scales[..., 0], scales[..., 1]


def _cached(state):
    """Keys and values of every sequence, (batch, kv heads, tokens, DIM) fp32, and (batch, tokens): which of them there are"""
    case = state["case"]
    blocks = state["pool"][state["table"].long()].transpose(1, 2)
    k, v, ks, vs = _tokens(blocks, case["values"])
    k, v = ((x * s[..., None]).flatten(2, 3)[:, :, :case["longest"]] for x, s in ((k, ks), (v, vs)))
    return k, v, torch.arange(case["longest"], device="cuda")[None] < state["lens"][:, None]


def _plain_read(state):
    k, v, there = _cached(state)
    return tuple(torch.where(there[:, :, None, None], x.transpose(1, 2), 0.0).to(torch.bfloat16) for x in (k, v))


def _plain_decode(state):
    case = state["case"]
    k, v, there = _cached(state)
    q = _rotate(state["q"].float(), state["lens"] - 1).view(case["batch"], case["kv_heads"], -1, DIM)
    s = (q @ k.transpose(-1, -2)) / math.sqrt(DIM)
    s = torch.where(there[:, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    out = (p / p.sum(-1, keepdim=True)) @ v
    return out.view(case["batch"], case["heads"], DIM).to(torch.bfloat16)


def _plain_sample(state):
    """Weights, their sums and what stands at a border in 64 bits"""
    x = state["logits"].double()
    rows, vocab = x.shape
    temperature, top_p, min_p = (torch.as_tensor(state[n], dtype=torch.float32, device="cuda").double().expand(rows)[:, None]
                                 for n in ("temperature", "top_p", "min_p"))
    top_k = torch.as_tensor(state["top_k"], device="cuda").expand(rows)[:, None]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((ordered - ordered[:, :1]) / temperature)
    w = torch.where((top_k > 0) & (torch.arange(vocab, device="cuda") >= top_k), 0.0, w)
    before = torch.cumsum(w, 1) - w
    keep = (before < top_p * w.sum(1, keepdim=True)) | (top_p >= 1)
    keep &= w >= min_p
    keep[:, 0] = True
    w = torch.zeros_like(x).scatter_(1, index, torch.where(keep, w, 0.0))
    running = torch.cumsum(w, 1)
    reach = state["uniform"].double()[:, None] * running[:, -1:]
    return (running > reach).int().argmax(1).to(torch.int32)


def _own(state):
    from baranet_bdml_b200 import ops
    case = state["case"]
    if case["path"] == "sample":
        return ops.sample_rows(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                               min_p=state["min_p"])
    cache = state.get("cache")
    if cache is None:                                  # a serving program makes it once
        from baranet_bdml_b200.kv_cache import QuantizedKVCache
        pages, per_seq = state["pool"].shape[0], state["table"].shape[1]
        lens = state["lens"] if "lens" in state else state["starts"] + case["seq"]
        cache = state["cache"] = QuantizedKVCache(pages, case["batch"], per_seq, case["kv_heads"], DIM, THETA, values=case["values"],
                                                  storage=(state["pool"], state["table"], lens))
    if case["path"] == "write":
        cache.append(state["seq_ids"], state["positions"], state["k"], state["v"])
        return cache.gather(state["rows"], state["starts"], case["seq"])
    if case["path"] == "read":
        return cache.gather(state["rows"], state["starts"], case["longest"])
    return cache.decode(state["q"], num_heads=case["heads"], max_seq_len=case["longest"])


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "sample": _plain_sample}[state["case"]["path"]](state)


def work(case):
    if case["path"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 8), "flops": 0}
    tokens = case["batch"] * (case["seq"] if case["path"] == "write" else (case["shortest"] + case["longest"]) / 2)
    held, wide = case["kv_heads"] * (2 * DIM + 4), case["kv_heads"] * 2 * DIM * 2
    if case["path"] == "write":
        return {"bytes": tokens * (2 * wide + 2 * held), "flops": 0}
    if case["path"] == "read":
        return {"bytes": tokens * held + case["batch"] * case["longest"] * wide, "flops": 0}
    return {"bytes": tokens * held + case["batch"] * case["heads"] * DIM * 4, "flops": 4 * tokens * case["heads"] * DIM}


# ------------------------------------------------------------------------------------------------------ definition in 64 bits
def _nearest(x, values):
    """x (..., DIM) in 64 bits -> the value that its nearest 8-bit number stands for"""
    most = x.abs().amax(-1, keepdim=True)
    if values == "int8":
        e = torch.floor(torch.log2(most / 127)) - 7    # the exponent of the last of a bf16 number's 8 places
        scale = (torch.ceil(most / 127 / 2 ** e) * 2 ** e).clamp(LEAST, MOST)
        return torch.round(x / scale) * scale
    scale = (2.0 ** torch.ceil(torch.log2(most / 448))).clamp(LEAST, MOST)
    y = x / scale
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["path"] == "write":
        positions = (state["starts"].double()[:, None] + torch.arange(case["seq"], dtype=torch.float64, device="cuda")).flatten()
        freq = torch.tensor([THETA ** (-2.0 * i / DIM) for i in range(DIM // 2)], dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((positions.numel(), DIM // 2), dtype=torch.float64, device="cuda"), positions[:, None] * freq)
        k, v = (state[n].double().unflatten(-1, (case["kv_heads"], DIM)) for n in ("k", "v"))
        k = torch.view_as_real(torch.view_as_complex(k.unflatten(-1, (DIM // 2, 2)).contiguous()) * turn[:, None]).flatten(-2)
        return tuple(_nearest(x, case["values"]).unflatten(0, (case["batch"], case["seq"])) for x in (k, v))
    if case["path"] == "sample":
        # ids one row at a time, by an order of Python's own kind: value first, then place
        found = []
        for r in range(case["rows"]):
            x = state["logits"][r].double().cpu()
            knob = {n: float(torch.as_tensor(state[n], dtype=torch.float32).reshape(-1)[r if case["each"] else 0]) for n in
                    ("temperature", "top_p", "min_p")}
            top_k = int(torch.as_tensor(state["top_k"]).reshape(-1)[r if case["each"] else 0])
            w = torch.exp((x - x.max()) / knob["temperature"])
            order = torch.argsort(-x, stable=True)
            order = order[:top_k] if top_k > 0 else order
            sums = torch.cumsum(w[order], 0)
            if knob["top_p"] < 1:
                order = order[:1 + int((sums[:-1] < knob["top_p"] * sums[-1]).sum())]
            order = order[(w[order] >= knob["min_p"]) | (torch.arange(len(order)) == 0)]
            order = torch.sort(order).values
            sums = torch.cumsum(w[order], 0)
            found.append(int(order[int((sums <= float(state["uniform"][r]) * sums[-1]).sum().clamp(max=len(order) - 1))]))
        return torch.tensor(found, dtype=torch.int32)
    dtype, kept = torch.float8_e4m3fn if case["values"] == "e4m3" else torch.int8, []
    place = torch.tensor([[((d >> 4) ^ ((t >> 1) & 3)) << 4 | (d & 15) for d in range(DIM)] for t in range(PAGE)], device="cuda")
    for b in range(case["batch"]):
        n = int(state["lens"][b])
        blocks = state["pool"].index_select(0, state["table"][b, :-(-n // PAGE)].long())
        scale = blocks[:, :, 2048:].contiguous().view(torch.bfloat16).double().view(*blocks.shape[:2], PAGE, 2)
        bytes_ = [blocks[:, :, :1024].reshape(*blocks.shape[:2], PAGE, DIM),
                  torch.gather(blocks[:, :, 1024:2048].reshape(*blocks.shape[:2], PAGE, DIM), 3, place.expand(*blocks.shape[:2], PAGE, DIM))]
        k, v = ((x.contiguous().view(dtype).float().double() * scale[..., i:i + 1]).transpose(1, 2).reshape(-1, case["kv_heads"], DIM)[:n]
                for i, x in enumerate(bytes_))
        if case["path"] == "read":
            kept.append([torch.cat((x, x.new_zeros((case["longest"] - n, case["kv_heads"], DIM)))) for x in (k, v)])
            continue
        q = state["q"][b].double()
        angle = (n - 1) * torch.tensor([THETA ** (-2.0 * i / DIM) for i in range(DIM // 2)], dtype=torch.float64, device="cuda")
        q = torch.view_as_real(torch.view_as_complex(q.view(-1, DIM // 2, 2).contiguous()) * torch.polar(torch.ones_like(angle), angle)).flatten(1)
        group = case["heads"] // case["kv_heads"]
        s = torch.einsum("hgd,lhd->hgl", q.view(case["kv_heads"], group, DIM), k) * DIM ** -0.5
        kept.append(torch.einsum("hgl,lhd->hgd", torch.softmax(s, -1), v).reshape(case["heads"], DIM))
    if case["path"] == "read":
        return tuple(torch.stack([x[i] for x in kept]) for i in range(2))
    return torch.stack(kept)
