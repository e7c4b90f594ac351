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


# ----------------------------------------------------------------------------------- where these operators go wrong, if they do
def test_rows_without_a_target(lib):
    """No loss and no gradient for negative targets; targets behind the vocabulary likewise, and they raise the error word."""
    from baranet_bdml_b200 import ops
    x, w, targets, grad = loss_inputs(300, 264, 700, 5)
    targets[:] = -100
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, targets, id_error=error)
    dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    assert not loss.any() and not dx.any() and not dw.any() and int(error) == 0
    targets[7], targets[8] = 700, 699
    loss, lse = ops.linear_cross_entropy(x, w, targets, id_error=error)
    dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    assert int(error) == 1 and torch.nonzero(loss).view(-1).tolist() == [8] and torch.nonzero(dx.any(1)).view(-1).tolist() == [8]
    want = loss_oracle(x, w, torch.where(targets == 700, -1, targets), grad)
    assert off(dx, want[2]) <= 2 * HALF and off(dw, want[3]) <= 2 * HALF


def test_gradients_that_differ_by_row(lib):
    """Row gradients of many sizes and signs, the first 0, tiny or negative: what the rows are divided by before they are rounded."""
    from baranet_bdml_b200 import ops
    x, w, targets, _ = loss_inputs(257, 264, 1000, 6)
    targets = targets.abs() % 1000
    for first in (0.0, 1e-30, -3.0, 1e-7):
        grad = torch.from_numpy((np.random.default_rng(1).standard_normal(257) * 1e-3).astype(np.float32)).cuda()
        grad[0] = first
        _, lse = ops.linear_cross_entropy(x, w, targets)
        dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
        want = loss_oracle(x, w, targets, grad)
        assert off(dx, want[2]) <= 2 * HALF and off(dw, want[3]) <= 2 * HALF, first
        if first == 0.0:
            assert not dx[0].any()


def test_large_logits(lib):
    """Logits of some hundreds, one of them far ahead: exp(z - lse) neither overflows nor loses the target"""
    from baranet_bdml_b200 import ops
    x, w, targets, grad = loss_inputs(130, 256, 1500, 7)
    x *= 40
    targets = targets.abs() % 1500
    loss, lse = ops.linear_cross_entropy(x, w, targets)
    dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    want = loss_oracle(x, w, targets, grad)
    largest = (x.double() @ w.double().T).abs().max().item()
    assert largest > 200 and (loss.double() - want[0]).abs().max().item() <= 2 * (256 / 16 + 8) * 2.0 ** -23 * largest
    # p is exp of a difference of two numbers of that size: off by their roundings, 24 2^-23 of `largest` each
    assert off(dx, want[2]) <= 2 * HALF + 2 * 24 * 2.0 ** -23 * largest and off(dw, want[3]) <= 2 * HALF + 2 * 24 * 2.0 ** -23 * largest


def test_one_of_the_gradients_alone(lib):
    from baranet_bdml_b200 import ops
    x, w, targets, grad = loss_inputs(200, 264, 5000, 8)
    _, lse = ops.linear_cross_entropy(x, w, targets)
    both = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    dx, none = ops.linear_cross_entropy_backward(x, w, targets, lse, grad, want_dweight=False)
    assert none is None and torch.equal(dx, both[0])
    none, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad, want_dx=False)
    assert none is None and torch.equal(dw, both[1])


def test_no_rows(lib):
    from baranet_bdml_b200 import ops
    x, w = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda"), bf16(np.random.default_rng(1), 104, 64)
    targets, grad = torch.empty((0,), dtype=torch.int32, device="cuda"), torch.empty((0,), dtype=torch.float32, device="cuda")
    loss, lse = ops.linear_cross_entropy(x, w, targets)
    dx, dw = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    assert loss.shape == (0,) and dx.shape == (0, 64) and not dw.any()
    grads = ops.gated_ff_backward(x, x, w, w, w.T.contiguous())
    assert grads[0].shape == (0, 64) and not any(g.any() for g in grads[1:])
    q = torch.empty((2, 0, 8, 64), dtype=torch.bfloat16, device="cuda")
    assert ops.attn_prefill_bf16_backward(q, q, q, q, q, torch.empty((2, 8, 0), device="cuda"))[0].shape == q.shape
    assert not ops.gemm_bf16_tn(x, x).any() and ops.gemm_bf16_nn(x, w.T.contiguous()).shape == (0, 104)


def test_attention_gradients_against_differences(lib):
    """The derivative along a direction against two forward passes: in 64 bits the oracle's, so that its own formula is not taken on trust."""
    rng = np.random.default_rng(3)
    q, k, v, dout = (torch.from_numpy(rng.standard_normal((1, 70, h, 64))) for h in (4, 2, 2, 4))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad((attention_oracle(*leaves, 3, True, 0.125)[0] * dout).sum(), leaves)
    for i, g in enumerate(grads):
        step = torch.from_numpy(rng.standard_normal(g.shape))
        value = [(attention_oracle(*[t + (s * step if j == i else 0) for j, t in enumerate((q, k, v))], 3, True, 0.125)[0] * dout).sum() for s in (1e-5, -1e-5)]
        assert abs((value[0] - value[1]).item() / 2e-5 - (g * step).sum().item()) <= 1e-6 * g.norm().item() * step.norm().item()


@pytest.mark.parametrize("std,scale", [(4.0, 0.125), (1.0, 1.0), (0.01, 0.125)])
def test_attention_gradients_of_sharp_and_flat_rows(lib, std, scale):
    """Scores of about std^2 scale 8: rows that one key has almost alone, and rows that all keys have alike.  A score is off by the roundings
    of the rotated q and k, 2^-8 of |q||k| scale each at most, sqrt(64) below that for independent ones; P is off by that factor."""
    got, want, (q, k, _, dout) = attention_grads(1, 200, 8, 2, 0, True, 17, scale=scale, std=std)
    scores = std * std * 8 * scale
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        assert off(a, b) <= WITHIN + 2 * HALF * scores, name


def test_bits_streams_and_graphs(lib):
    """The same bits in every run, on another stream, beside a second call under way, and from a captured graph on new inputs."""
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(23)

    def inputs():
        q, k, v, dout = (bf16(rng, 2, 300, h, 64) for h in (8, 2, 2, 8))
        x, w, targets, grad = loss_inputs(333, 512, 3001, int(rng.integers(1 << 30)))
        return [q, k, v, dout, x, w, targets, grad, bf16(rng, 640, 512, std=0.05), bf16(rng, 640, 512, std=0.05), bf16(rng, 512, 640, std=0.05)]

    def step(q, k, v, dout, x, w, targets, grad, gate, up, down):
        lse = torch.empty((2, 8, 300), dtype=torch.float32, device="cuda")
        out = ops.attn_prefill_bf16(q, k, v, lse=lse)
        loss, total = ops.linear_cross_entropy(x, w, targets)
        dx, dw = ops.linear_cross_entropy_backward(x, w, targets, total, grad)
        return [loss, dx, dw, *ops.gated_ff_backward(dx, x, gate, up, down), *ops.attn_prefill_bf16_backward(dout, q, k, v, out, lse)]

    a, b = inputs(), inputs()
    first, other = step(*a), step(*b)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, step(*a)))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side[0]):
            got_a = step(*a)
        with torch.cuda.stream(side[1]):
            got_b = step(*b)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(first, got_a)) and all(torch.equal(p, q) for p, q in zip(other, got_b))
    static = [t.clone() for t in a]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    for source, want in ((b, other), (a, first)):
        for t, s in zip(static, source):
            t.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, captured))
    ops.gemm_status()


def test_a_block_and_its_loss_together(lib):
    """x + attention(x), + the gated block of that, loss over the vocabulary; then all gradients, by the layers' own backward calls."""
    from baranet_bdml_b200 import ops
    from baranet_bdml_b200.layers import GroupedQueryAttentionBF16, LLaMAConfig, MLPBF16
    np.random.seed(4)
    cfg = LLaMAConfig(vocab_size=777, hidden_size=512, intermediate_size=1416, num_attention_heads=8, num_key_value_heads=2)
    attn, mlp = GroupedQueryAttentionBF16(cfg), MLPBF16(cfg)
    rng = np.random.default_rng(4)
    B, S, H = 2, 150, 512
    x, head = bf16(rng, B, S, H), bf16(rng, 777, H, std=2 * H ** -0.5)
    targets = torch.from_numpy(rng.integers(-50, 777, B * S).astype(np.int32)).cuda()
    grad = torch.full((B * S,), 1.0 / (B * S), device="cuda")
    h1 = x + attn(x)
    h2 = h1 + mlp(h1.view(-1, H)).view(B, S, H)
    loss, lse = ops.linear_cross_entropy(h2.view(-1, H), head, targets)
    d2, dhead = ops.linear_cross_entropy_backward(h2.view(-1, H), head, targets, lse, grad)
    dmlp, gmlp = mlp.backward(d2, h1.view(-1, H))
    d1 = (d2 + dmlp).view(B, S, H)
    dattn, gattn = attn.backward(d1, x)
    dx = d1 + dattn
    ops.gemm_status()

    leaves = [t.double().requires_grad_(True) for t in (x, *attn.parameters(), *mlp.parameters(), head)]
    X, wq, wk, wv, wo, wg, wu, wd, whead = leaves
    o, _ = attention_oracle((X @ wq.T).view(B, S, 8, 64), (X @ wk.T).view(B, S, 2, 64), (X @ wv.T).view(B, S, 2, 64), 0, True, 0.125)
    H1 = X + o.reshape(B, S, H) @ wo.T
    H2 = H1 + (torch.nn.functional.silu(H1 @ wg.T) * (H1 @ wu.T)) @ wd.T
    z = H2.view(B * S, H) @ whead.T
    picked = z.gather(1, targets.clamp(min=0).long()[:, None])[:, 0]
    losses = torch.where(targets >= 0, torch.logsumexp(z, 1) - picked, 0.0)
    want = torch.autograd.grad((losses * grad.double()).sum(), leaves)
    # roundings on the way, each of at most half a step of what is summed: forward q, k, v, P, rows, o, h1, gate and up, h, y, h2 (11), back dz, d2,
    # dh .. dmlp, d1 (5), the attention's own (6), and the result's
    for name, a, b in zip(("x", "q", "k", "v", "o", "gate", "up", "down", "head"), (dx, *gattn, *gmlp, dhead), want):
        assert off(a, b.view(a.shape)) <= 23 * HALF, name
    # logits move by the roundings of h2 and what it comes from: 11 half steps of values of size |z|
    assert (loss.double() - losses).abs().max().item() <= 11 * HALF * z.abs().max().item()


def test_attention_layers_gradients_follow_weights_written_in_place(lib):
    from baranet_bdml_b200.layers import GroupedQueryAttentionBF16, LLaMAConfig
    np.random.seed(9)
    attn = GroupedQueryAttentionBF16(LLaMAConfig(vocab_size=100, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2))
    rng = np.random.default_rng(9)
    x, dy = bf16(rng, 60, 256), bf16(rng, 60, 256)
    attn(x)                                               # packs its weights
    for w in attn.parameters():
        w.mul_(-0.5)
    got, grads = attn.backward(dy, x)
    leaves = [t.double().requires_grad_(True) for t in (x, *attn.parameters())]
    X, wq, wk, wv, wo = leaves
    o, _ = attention_oracle((X @ wq.T).view(1, 60, 4, 64), (X @ wk.T).view(1, 60, 2, 64), (X @ wv.T).view(1, 60, 2, 64), 0, True, 0.125)
    want = torch.autograd.grad(o.reshape(60, 256) @ wo.T, leaves, dy.double())
    # the attention's own roundings, q, k, v, dattn, the gradients of q, k and v, and the result's
    for name, a, b in zip(("x", "q", "k", "v", "o"), (got, *grads), want):
        assert off(a, b) <= 12 * HALF, name


def test_scores_of_a_model(lib):
    """LLaMAModelBF16.score against the log-softmax of the logits that __call__ gives on the same weights"""
    from baranet_bdml_b200.layers import LLaMAConfig
    from baranet_bdml_b200.model import LLaMAModelBF16
    np.random.seed(5)
    cfg = LLaMAConfig(vocab_size=1008, hidden_size=256, intermediate_size=704, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)
    model = LLaMAModelBF16(cfg)
    ids = torch.from_numpy(np.random.default_rng(6).integers(0, 1008, (3, 37)).astype(np.int32)).cuda()
    got = model.score(ids)
    logits = model(ids).double()
    want = torch.log_softmax(logits[:, :-1], -1).gather(2, ids[:, 1:, None].long())[..., 0]
    # `__call__` rounds its logits to bf16: half a step of |z| for the picked one, and no more for the mean that lse takes of them
    assert got.shape == (3, 36) and (got.double() - want).abs().max().item() <= 2 * HALF * logits.abs().max().item()
    with pytest.raises(IndexError):
        model.score(torch.full((1, 4), 1008, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="at least two"):
        model.score(ids[:, :1])
    model.status()


def test_refusals(lib):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(1)
    x, w, t = bf16(rng, 10, 64), bf16(rng, 100, 64), torch.zeros(10, dtype=torch.int32, device="cuda")
    one = torch.ones(10, device="cuda")
    for bad in (lambda: ops.linear_cross_entropy(x.float(), w, t), lambda: ops.linear_cross_entropy(x, w.T, t), lambda: ops.linear_cross_entropy(x, w, t.long()),
                lambda: ops.linear_cross_entropy(x, w, t[:9]), lambda: ops.linear_cross_entropy(x[:, :60].contiguous(), w[:, :60].contiguous(), t),
                lambda: ops.linear_cross_entropy(x.cpu(), w, t), lambda: ops.linear_cross_entropy_backward(x, w, t, one, one.double()),
                lambda: ops.linear_cross_entropy_backward(x, w, t, one, one, want_dx=False, want_dweight=False),
                lambda: ops.gated_ff_backward(x, x, w, w, w), lambda: ops.gated_ff_backward(x, x, w, w, w.T.contiguous(), act="relu2"),
                lambda: ops.gated_ff_backward(x[:5], x, w, w, w.T.contiguous()), lambda: ops.gemm_bf16_nn(x, w), lambda: ops.gemm_bf16_tn(x, w),
                lambda: ops.gemm_bf16_tn(bf16(rng, 10, 60), x)):
        with pytest.raises(RuntimeError):
            bad()
    q, k, lse = bf16(rng, 1, 20, 8, 64), bf16(rng, 1, 20, 2, 64), torch.zeros((1, 8, 20), device="cuda")
    back = ops.attn_prefill_bf16_backward
    for bad in (lambda: back(q, q, k, k, q, lse[:, :4]), lambda: back(q, q, k, k[:, :10], q, lse), lambda: back(q[:, ::2], q, k, k, q, lse),
                lambda: back(q, q, bf16(rng, 1, 20, 3, 64), bf16(rng, 1, 20, 3, 64), q, lse), lambda: back(q, q, k, k, q, lse, position_offset=-1),
                lambda: back(*(t.reshape(1, 40, -1, 32) for t in (q, q, k, k, q)), lse)):
        with pytest.raises(RuntimeError):
            bad()
