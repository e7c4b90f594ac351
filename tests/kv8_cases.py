"""The 8-bit cache and sampling in 64 bits or more, written from their definitions: what the tests compare the kernels with."""
import numpy as np
import torch

PAGE, D, BLOCK = 16, 64, 2112
LEAST, MOST = 2.0 ** -100, 2.0 ** 122


def rotated(x, positions, theta=10000.0):
    """x (T, heads, 64) fp64 CPU, positions (T,)"""
    freq = float(theta) ** (-np.arange(0, D, 2) / D)
    angle = np.asarray(positions, dtype=np.float64)[:, None] * freq
    c, s = torch.from_numpy(np.cos(angle))[:, None], torch.from_numpy(np.sin(angle))[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def v_places():
    """byte of a token's V that holds element d"""
    return torch.tensor([[(((d // 16) ^ (t // 2 % 4)) * 16) + d % 16 for d in range(D)] for t in range(PAGE)])


def unpacked(pool, values):
    """pool (pages, heads, 2112) uint8 -> K, V numbers (pages, heads, 16, 64) fp64 and their scales (pages, heads, 16), on the CPU"""
    pool = pool.cpu()
    dtype = torch.float8_e4m3fn if values == "e4m3" else torch.int8
    k, v = (pool[..., a:a + 1024].contiguous().view(dtype).float().double().unflatten(-1, (PAGE, D)) for a in (0, 1024))
    v = v.gather(-1, v_places().expand_as(v))
    scales = pool[..., 2048:].contiguous().view(torch.bfloat16).double().unflatten(-1, (PAGE, 2))
    return k, v, scales[..., 0], scales[..., 1]


def packed(k, v, ks, vs, values):
    """The inverse: numbers that are representable, scales that are bf16"""
    dtype = torch.float8_e4m3fn if values == "e4m3" else torch.int8
    kb, vb = (x.float().to(dtype).view(torch.uint8) for x in (k, v))
    vb = torch.empty_like(vb).scatter_(-1, v_places().expand_as(vb), vb)
    scales = torch.stack((ks, vs), -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)
    return torch.cat((kb.flatten(-2), vb.flatten(-2), scales), -1)


def scale_rule(most, values):
    """Scales that the largest magnitudes ask for, fp64"""
    most = np.maximum(np.asarray(most, dtype=np.float64), 1e-300)
    if values == "e4m3":
        s = 2.0 ** np.ceil(np.log2(most / 448))
    else:
        e = 2.0 ** (np.floor(np.log2(most / 127)) - 7)
        s = np.ceil(most / 127 / e) * e
    return np.clip(s, LEAST, MOST)


def attention(q, k, v, scale):
    """q (heads, 64), k, v (tokens, kv heads, 64), fp64 -> out, lse, and what bounds on rounding need: sum p |v| and the largest
    scale * sum |q| |k| of a head"""
    heads, kv = q.shape[0], k.shape[1]
    k, v = (x.repeat_interleave(heads // kv, 1) for x in (k, v))
    s = torch.einsum("hd,lhd->hl", q, k) * scale
    p = torch.softmax(s, -1)
    return (torch.einsum("hl,lhd->hd", p, v), torch.logsumexp(s, -1), torch.einsum("hl,lhd->hd", p, v.abs()),
            (torch.einsum("hd,lhd->hl", q.abs(), k.abs()) * abs(scale)).amax(-1))


def choose(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The id of one row, in the widest floats that numpy has"""
    wide = np.longdouble
    f = lambda v: wide(np.float32(v))      # noqa: E731
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if not np.any(x > -np.inf):
        return 0
    if not f(temperature) > 0:
        return int(np.argmax(x))
    top = x.max()
    z = np.zeros(len(x), dtype=wide)
    with np.errstate(invalid="ignore"):
        z = np.where(x == top, wide(0), (x.astype(wide) - wide(top)) / f(temperature)) if np.isfinite(top) else np.where(x == top, wide(0), wide(-np.inf))
    w = np.where(x > -np.inf, np.exp(z), wide(0))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if 0 < top_k < len(order):
        order = order[:top_k]
    if f(top_p) < 1:
        before = np.cumsum(w[order]) - w[order]
        before[0] = 0
        order = order[(before < f(top_p) * w[order].sum()) | (np.arange(len(order)) == 0)]
    order = order[(w[order] >= f(min_p)) | (np.arange(len(order)) == 0)]
    order = np.sort(order)
    run = np.cumsum(w[order])
    return int(order[min(int((run <= wide(u) * run[-1]).sum()), len(order) - 1)])
