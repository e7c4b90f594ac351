"""Loss over the vocabulary and gradients of a training step against plain restatements in 64 bits on the same bf16 inputs.

Tolerances, relative to the 2-norm of the result.  A bf16 rounding moves a value by at most 2^-8 relative, half a step is 2^-9 where the
mantissa is full and 2^-8 where it is empty; a result that is rounded at n places on its way (itself, and each bf16 operand that was
computed) is off by at most n 2^-8 of the sizes that are summed.  In the 2-norm the sums of independent roundings are far below that, so
n 2^-8 holds with room wherever the summands do not cancel by more than their number's root."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = torch.finfo(torch.bfloat16).eps / 2


def bf16(rng, *shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).cuda().to(torch.bfloat16)


def off(got, want):
    want = want.double()
    norm = want.norm().item()
    return (got.double() - want).norm().item() / norm if norm else got.double().abs().max().item()


@pytest.mark.parametrize("M,N,K", [(1, 8, 8), (3, 264, 72), (128, 256, 64), (129, 520, 200), (64, 2048, 5632), (700, 1000, 1000), (2500, 2048, 1032),
                                   (5000, 4096, 264)])
def test_product_across_the_weights_rows(lib, M, N, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + N + K)
    a, b = bf16(rng, M, K), bf16(rng, K, N, std=K ** -0.5)
    assert off(ops.gemm_bf16_nn(a, b), a.double() @ b.double()) <= HALF
    ops.gemm_status()


@pytest.mark.parametrize("M,N,K", [(8, 8, 1), (264, 72, 3), (128, 256, 64), (136, 520, 129), (2048, 2048, 64), (1000, 1000, 700), (10000, 2048, 333),
                                   (4096, 1032, 1000)])
def test_product_of_two_transposed_operands(lib, M, N, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + N + K)
    a, b = bf16(rng, K, M), bf16(rng, K, N, std=K ** -0.5)
    assert off(ops.gemm_bf16_tn(a, b), a.double().T @ b.double()) <= HALF
    ops.gemm_status()


def loss_inputs(rows, hidden, vocab, seed):
    rng = np.random.default_rng(seed)
    x, w = bf16(rng, rows, hidden), bf16(rng, vocab, hidden, std=2 * hidden ** -0.5)
    targets = rng.integers(0, vocab, rows).astype(np.int32)
    targets[rng.random(rows) < 0.2] = -100
    return x, w, torch.from_numpy(targets).cuda(), torch.from_numpy(rng.uniform(0.5, 1.5, rows).astype(np.float32) / rows).cuda()


def loss_oracle(x, w, targets, grad):
    x, w, t = x.double(), w.double(), targets.long()
    z = x @ w.T
    lse = torch.logsumexp(z, 1)
    counts = t >= 0
    hot = torch.nn.functional.one_hot(t.clamp(min=0), w.shape[0]).double()
    loss = torch.where(counts, lse - (z * hot).sum(1), 0.0)
    dz = (torch.exp(z - lse[:, None]) - hot) * torch.where(counts, grad.double(), 0.0)[:, None]
    return loss, lse, dz @ w, dz.T @ x


LOSS_SIZES = [(1, 8, 1), (1, 64, 1000), (3, 72, 255), (33, 264, 257), (128, 256, 512), (130, 1000, 10007), (700, 520, 2001), (1500, 2048, 4096),
              (16500, 64, 4500)]


@pytest.mark.parametrize("rows,hidden,vocab", LOSS_SIZES)
def test_loss_and_its_gradients(lib, rows, hidden, vocab):
    from baranet_bdml_b200 import ops
    x, w, targets, grad = loss_inputs(rows, hidden, vocab, rows + hidden)
    loss, lse = ops.linear_cross_entropy(x, w, targets)
    dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    ops.gemm_status()
    want = loss_oracle(x, w, targets, grad)
    # a logit is an fp32 sum to which the tensor core adds 16 products at a time, each time losing up to a unit in the last place (2^-23 of
    # a sum of at most |z|, cut rather than rounded); exponentials, their sum and the logarithm add a few more; a loss has two logits
    largest = (x.double() @ w.double().T).abs().max().item()
    within = (hidden / 16 + 8) * 2.0 ** -23 * max(1.0, largest)
    assert (loss.double() - want[0]).abs().max().item() <= 2 * within and (lse.double() - want[1]).abs().max().item() <= within
    assert not loss[targets < 0].any()
    assert off(dx, want[2]) <= 2 * HALF and off(dw, want[3]) <= 2 * HALF


@pytest.mark.parametrize("rows,hidden,inter,act", [(1, 8, 8, "silu"), (3, 72, 136, "gelu_tanh"), (64, 256, 512, "silu"), (129, 264, 520, "silu"),
                                                   (333, 1000, 712, "gelu_tanh"), (64, 2048, 5632, "silu"), (2500, 512, 1416, "silu")])
def test_gated_block_gradients(lib, rows, hidden, inter, act):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(rows + hidden)
    x, dy = bf16(rng, rows, hidden), bf16(rng, rows, hidden, std=1.0 / rows)
    gate, up, down = bf16(rng, inter, hidden, std=hidden ** -0.5), bf16(rng, inter, hidden, std=hidden ** -0.5), bf16(rng, hidden, inter, std=inter ** -0.5)
    got = ops.gated_ff_backward(dy, x, gate, up, down, act=act)
    ops.gemm_status()
    leaves = [t.double().requires_grad_(True) for t in (x, gate, up, down)]
    g = leaves[0] @ leaves[1].T
    a = torch.nn.functional.silu(g) if act == "silu" else torch.nn.functional.gelu(g, approximate="tanh")
    want = torch.autograd.grad((a * (leaves[0] @ leaves[2].T)) @ leaves[3].T, leaves, dy.double())
    for name, a, b in zip(("dx", "dgate", "dup", "ddown"), got, want):
        assert off(a, b) <= 3 * HALF, name


# ------------------------------------------------------------------------------------------------------------- attention
def turned(x, offset, theta=10000.0):
    """(B, S, heads, D) in 64 bits, pairs turned by their position's angle"""
    D = x.shape[-1]
    freq = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=x.device) / D)
    angle = (torch.arange(x.shape[1], dtype=torch.float64, device=x.device) + offset)[:, None] * freq
    z = torch.view_as_complex(x.unflatten(-1, (D // 2, 2)).contiguous()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.view_as_real(z).flatten(-2)


def attention_oracle(q, k, v, offset, causal, scale):
    """out, lse of (B, S, heads, D) operands in 64 bits, differentiable"""
    S, rep = q.shape[1], q.shape[2] // k.shape[2]
    s = torch.einsum("bqhd,bkhd->bhqk", turned(q, offset), turned(k, offset).repeat_interleave(rep, 2)) * scale
    if causal:
        at = torch.arange(S, device=q.device)
        s = s.masked_fill(at[None, :] > at[:, None] + offset, -float("inf"))
    return torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), v.repeat_interleave(rep, 2)), torch.logsumexp(s, -1)


def attention_grads(B, S, Hq, Hkv, offset, causal, seed, scale=0.125, std=1.0):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(seed)
    q, k, v, dout = (bf16(rng, B, S, h, 64, std=std) for h in (Hq, Hkv, Hkv, Hq))
    lse = torch.empty((B, Hq, S), dtype=torch.float32, device="cuda")
    out = ops.attn_prefill_bf16(q, k, v, scale=scale, position_offset=offset, causal=causal, lse=lse)
    got = ops.attn_prefill_bf16_backward(dout, q, k, v, out, lse, scale=scale, position_offset=offset, causal=causal)
    ops.gemm_status()
    leaves = [t.double().requires_grad_(True) for t in (q, k, v)]
    return got, torch.autograd.grad(attention_oracle(*leaves, offset, causal, scale)[0], leaves, dout.double()), (q, k, v, dout)


# Rounded on the way: the rotated q and k (their product moves a score s by at most 2 * 2^-8 |q||k| scale, and P by that factor), P or dS,
# the other operand, the output that d comes from, and the result.
WITHIN = 6 * HALF


@pytest.mark.parametrize("S", [2, 63, 64, 65, 127, 128, 129, 200, 333, 513])
@pytest.mark.parametrize("offset,causal", [(0, True), (5, True), (1000, True), (0, False), (3, False)])
def test_attention_gradients_of_lengths(lib, S, offset, causal):
    got, want, _ = attention_grads(2, S, 8, 2, offset, causal, S + offset)
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        assert off(a, b) <= WITHIN, name


@pytest.mark.parametrize("B,S,Hq,Hkv", [(1, 300, 1, 1), (3, 130, 6, 2), (1, 257, 7, 1), (5, 70, 12, 12), (1, 1500, 32, 4), (8, 700, 16, 2)])
def test_attention_gradients_of_heads(lib, B, S, Hq, Hkv):
    got, want, _ = attention_grads(B, S, Hq, Hkv, 0, True, B + S)
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        assert off(a, b) <= WITHIN, name


def test_attention_gradients_of_a_single_key(lib):
    """One key has all the weight: the gradients of its score are 0.  What is left is P (dP - d): the output that d = sum dO O comes from is
    v with two roundings to bf16 (P, and the output), so |dP - d| <= 2 * 2^-8 sum |dO v|; times scale |k| for dq, scale |q| and the group's
    heads for dk (a sixteenth more: the last roundings, fp32)."""
    got, want, (q, k, v, dout) = attention_grads(3, 1, 8, 2, 0, True, 11)
    left = 2 * HALF * (dout.double() * v.double().repeat_interleave(4, 2)).abs().sum(-1, keepdim=True) * 0.125 * 17 / 16
    assert ((got[0].double().abs() <= left * k.double().abs().max()).all())
    assert (got[1].double().abs() <= left.unflatten(2, (2, 4)).sum(3) * q.double().abs().max()).all()
    assert off(got[2], want[2]) <= WITHIN
