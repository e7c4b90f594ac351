"""Attention's gradients row by row (a position of a head), where the norm of a whole result would not see a last key or a lost block.

What a row may be off by, in the 2-norm.  Rounded to bf16, each by at most HALF of its size: the rotated q and k, of which a score is a sum
of D products; P, for dV; dS, for dQ and dK; the other operand of those products (dO and v are exact); the output, which d = sum dO O comes
from; the result.  The fp32 angle is off by a few units of its own size, (S + offset) 2^-22, which moves q and k alike.
A score's error is a sum of 2 D independent ones: `step` below, HALF scale sqrt(2 sum (q k)^2), and P is off by that factor and by the one of
lse, a mean of the row's steps.  So of an element of P dO, dS q or dS k
    HALF for its own rounding, HALF for its operand's, 2 step for P, and P HALF sqrt(sum (dO O)^2) for d,
independent from element to element, are added up as squares; what a query's lse and d have in common for all keys moves dQ as a whole and
is added as it is.  A half step is the largest that a rounding can do, 1.7 times its root mean square: TWICE the sum is far outside, and half
of that for all rows together, whose errors are no longer those of a few unlucky roundings."""
import numpy as np
import pytest
import torch

from test_gpu_training import HALF, attention_oracle, bf16, turned

pytestmark = pytest.mark.gpu
TWICE = 2.0


def row_bounds(q, k, v, dout, offset, causal, scale):
    """(want, bound of every row) of dq, dk, dv for one sequence (S, heads, D) in 64 bits"""
    S, Hq, D = q.shape
    rep = Hq // k.shape[1]
    angle = (S + offset) * 2.0 ** -22
    qr, kr = turned(q[None], offset)[0], turned(k[None], offset)[0]
    at = torch.arange(S, device=q.device)
    hidden = at[None, :] > at[:, None] + offset if causal else None
    dq, dq2, dqc = torch.zeros_like(q), torch.zeros(S, Hq, dtype=torch.float64, device=q.device), torch.zeros(S, Hq, dtype=torch.float64, device=q.device)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dk2, dv2 = (torch.zeros(S, k.shape[1], dtype=torch.float64, device=q.device) for _ in range(2))
    for h in range(Hq):
        g = h // rep
        Q, K, V, O = qr[:, h], kr[:, g], v[:, g], dout[:, h]
        s = Q @ K.T * scale
        if causal:
            s = s.masked_fill(hidden, -float("inf"))
        P = torch.softmax(s, -1)
        out, dP = P @ V, O @ V.T
        d = (P * dP).sum(-1, keepdim=True)
        dS = P * (dP - d) * scale
        step = (HALF + angle) * scale * torch.sqrt(2 * (Q ** 2 @ (K ** 2).T))
        step = step if not causal else step.masked_fill(hidden, 0.0)
        mean_step = (P * step).sum(-1, keepdim=True)
        d_off = HALF * torch.sqrt((O ** 2 * out ** 2).sum(-1, keepdim=True))
        p_off = P * (HALF + step + mean_step)
        s_off = dS.abs() * (2 * HALF + angle + step + mean_step) + scale * P * (d_off + dP.abs() * 2.0 ** -20)
        rows = lambda off, x: (off ** 2) @ (x ** 2).sum(-1)      # noqa: E731
        dq[:, h] = dS @ K
        dq2[:, h] = rows(s_off, K)
        # the row's lse and d: the same for all of its keys
        dqc[:, h] = (mean_step * (dS @ K)).norm(dim=-1) + scale * (d_off * (P @ K)).norm(dim=-1)
        dk[:, g] += dS.T @ Q
        dk2[:, g] += rows(s_off.T, Q)
        dv[:, g] += P.T @ O
        dv2[:, g] += rows(p_off.T, O)
    back = lambda t: turned_back(t, offset)      # noqa: E731
    tiny = 1e-30
    return [(back(dq), TWICE * (torch.sqrt(dq2) + dqc) + (HALF * 1.01 + angle) * dq.norm(dim=-1) + tiny),
            (back(dk), TWICE * torch.sqrt(dk2) + (HALF * 1.01 + angle) * dk.norm(dim=-1) + tiny),
            (dv, TWICE * torch.sqrt(dv2) + HALF * 1.01 * dv.norm(dim=-1) + tiny)]


def turned_back(x, offset, theta=10000.0):
    D = x.shape[-1]
    freq = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    angle = (torch.arange(x.shape[0], dtype=torch.float64, device=x.device) + offset)[:, None] * freq
    z = torch.view_as_complex(x.unflatten(-1, (D // 2, 2)).contiguous()) * torch.polar(torch.ones_like(angle), -angle)[:, None]
    return torch.view_as_real(z).flatten(-2)


def check_rows(got, wanted):
    """The worst row of each gradient as a share of what it may be off by; `wanted` from row_bounds"""
    worst = []
    for name, a, (want, bound) in zip(("dq", "dk", "dv"), got, wanted):
        assert torch.isfinite(a).all(), name
        error = (a.double() - want).norm(dim=-1)
        assert error.norm() <= 0.5 * bound.norm(), (name, error.norm().item(), bound.norm().item())
        ratio = error / bound
        at = int(ratio.argmax())
        worst.append(ratio.max().item())
        assert worst[-1] <= 1.0, (name, divmod(at, ratio.shape[1]), worst[-1])
    return worst


def inputs(B, S, Hq, Hkv, seed, std=1.0):
    rng = np.random.default_rng(seed)
    return tuple(bf16(rng, B, S, h, 64, std=std) for h in (Hq, Hkv, Hkv, Hq))


def gradients(q, k, v, dout, offset, causal, scale=0.125):
    from baranet_bdml_b200 import ops
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device="cuda")
    out = ops.attn_prefill_bf16(q, k, v, scale=scale, position_offset=offset, causal=causal, lse=lse)
    got = ops.attn_prefill_bf16_backward(dout, q, k, v, out, lse, scale=scale, position_offset=offset, causal=causal)
    ops.gemm_status()
    return got, (out, lse)


@pytest.mark.parametrize("S", [2, 63, 64, 65, 127, 128, 129, 191, 193, 333, 513])
@pytest.mark.parametrize("offset,causal", [(0, True), (5, True), (1000, True), (0, False), (3, False)])
def test_every_row(lib, S, offset, causal):
    q, k, v, dout = inputs(2, S, 8, 2, S + offset)
    got, _ = gradients(q, k, v, dout, offset, causal)
    for b in range(2):
        wanted = row_bounds(q[b].double(), k[b].double(), v[b].double(), dout[b].double(), offset, causal, 0.125)
        check_rows([g[b] for g in got], wanted)
        for want, bound in wanted if S > 2 else []:       # (a row that is 0 would be seen wherever it does not cancel)
            assert (want.norm(dim=-1) > bound)[-13:].double().mean() >= 0.5


@pytest.mark.parametrize("B,S,Hq,Hkv,offset,causal", [(1, 300, 1, 1, 0, True), (3, 130, 6, 2, 7, True), (1, 257, 7, 1, 0, True), (5, 70, 12, 12, 0, False),
                                                      (1, 1500, 32, 4, 0, True)])
def test_every_row_of_heads(lib, B, S, Hq, Hkv, offset, causal):
    q, k, v, dout = inputs(B, S, Hq, Hkv, B + S)
    got, _ = gradients(q, k, v, dout, offset, causal)
    for b in range(B):
        check_rows([g[b] for g in got], row_bounds(q[b].double(), k[b].double(), v[b].double(), dout[b].double(), offset, causal, 0.125))


def test_every_row_of_a_batch_of_long_sequences(lib):
    """31 blocks a CTA: the ring of blocks (8 places) and those of tiles wrap many times; the same bits again"""
    from baranet_bdml_b200 import ops
    q, k, v, dout = inputs(8, 2048, 32, 4, 42)
    got, (out, lse) = gradients(q, k, v, dout, 0, True)
    for b in (0, 3, 7):
        check_rows([g[b] for g in got], row_bounds(q[b].double(), k[b].double(), v[b].double(), dout[b].double(), 0, True, 0.125))
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, ops.attn_prefill_bf16_backward(dout, q, k, v, out, lse, scale=0.125)))
    ops.gemm_status()


def test_many_short_sequences(lib):
    """Blocks of one tile, and so of one softmax group, each: 64 sequences of 50 tokens, and of 1"""
    for S in (50, 1):
        q, k, v, dout = inputs(64, S, 16, 4, 7 + S)
        got, _ = gradients(q, k, v, dout, 0, True)
        for b in range(0, 64, 9):
            check_rows([g[b] for g in got], row_bounds(q[b].double(), k[b].double(), v[b].double(), dout[b].double(), 0, True, 0.125))
