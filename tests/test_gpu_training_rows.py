"""The training operators element by element and row by row, where a norm over a whole result would not see a tile that is missing.

Bounds.  A result is off by its own rounding, HALF of its size; by what its bf16 operands were off, HALF of their sizes, carried through
the product of absolute values; and by the tensor core's sums, which add 16 products at a time and cut each time up to a unit in the last
place, 2^-23 of a sum that is at most the product of absolute values (sums of ranges of K add a few more)."""
import numpy as np
import pytest
import torch

from test_gpu_training import HALF, bf16, loss_inputs

pytestmark = pytest.mark.gpu
UNIT = 2.0 ** -23


def sums(K):
    return (K / 16 + 40) * UNIT


def within(got, want, bound):
    """Every element within `bound` and its own rounding; and the bound is one that a lost tile of 32 x 64 does not keep."""
    assert torch.isfinite(got).all()
    bound = bound + HALF * 1.01 * want.abs() + 1e-300
    ratio = (got.double() - want).abs() / bound
    worst = int(ratio.argmax())
    assert ratio.max().item() <= 1.0, (divmod(worst, want.shape[1]), ratio.max().item())
    for rows in (slice(0, 32), slice(-32, None)):
        assert (want[rows, -64:].abs() > bound[rows, -64:]).any()


def again(call, first, times=4):
    for _ in range(times):
        for a, b in zip(call(), first):
            assert torch.equal(a, b)


# (rows of the result that leave warps of a CTA's last tile without one, behind a tile that was full, and a K of few steps)
@pytest.mark.parametrize("M,N,K", [(10056, 2048, 64), (10008, 2048, 8), (32008, 2048, 40), (10056, 1032, 200)])
def test_product_of_two_transposed_operands_by_elements(lib, M, N, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + K)
    a, b = bf16(rng, K, M), bf16(rng, K, N, std=K ** -0.5)
    got = ops.gemm_bf16_tn(a, b)
    within(got, a.double().T @ b.double(), sums(K) * (a.double().abs().T @ b.double().abs()))
    again(lambda: [ops.gemm_bf16_tn(a, b)], [got])
    ops.gemm_status()


@pytest.mark.parametrize("M,N,K", [(2200, 8192, 64), (16400, 1032, 200), (2049, 8200, 8), (40, 2048, 8192)])
def test_product_across_the_weights_rows_by_elements(lib, M, N, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + K)
    a, b = bf16(rng, M, K), bf16(rng, K, N, std=K ** -0.5)
    got = ops.gemm_bf16_nn(a, b)
    within(got, a.double() @ b.double(), sums(K) * (a.double().abs() @ b.double().abs()))
    again(lambda: [ops.gemm_bf16_nn(a, b)], [got])
    ops.gemm_status()


def check_loss_gradients(x, w, targets, grad):
    from baranet_bdml_b200 import ops
    rows, hidden, vocab = *x.shape, w.shape[0]
    _, lse = ops.linear_cross_entropy(x, w, targets)
    got = ops.linear_cross_entropy_backward(x, w, targets, lse, grad)
    X, W, t = x.double(), w.double(), targets.long()
    z = X @ W.T
    total = torch.logsumexp(z, 1)
    # exp(z - lse): z by its sum, twice (it is in lse as well); the product with log2 e and lse by their roundings; the exponential by 2 units
    off = sums(hidden) * 2 * (X.abs() @ W.abs().T).amax().item() + 4 * UNIT * (z.abs().max().item() + total.abs().max().item()) + 2 * UNIT
    size = torch.where(t >= 0, grad.double(), 0.0).abs()[:, None]
    p = torch.exp(z - total[:, None])
    p_off = size * (p * 1.01 * off + UNIT) + 2.0 ** -126  # (the difference to 1 at the target rounds too; what is below normal numbers may be lost)
    p[torch.arange(rows, device="cuda"), t.clamp(min=0)] -= 1.0
    dz = p * torch.where(t >= 0, grad.double(), 0.0)[:, None]
    dz_off = p_off + (HALF * 1.01 + sums(max(rows, vocab))) * dz.abs()
    within(got[0], dz @ W, dz_off @ W.abs())
    within(got[1], dz.T @ X, dz_off.T @ X.abs())
    again(lambda: ops.linear_cross_entropy_backward(x, w, targets, lse, grad), got)
    ops.gemm_status()


@pytest.mark.parametrize("rows,hidden,vocab", [(64, 2048, 10007), (16, 2048, 10007), (1531, 1000, 10007), (600, 2048, 32000), (2100, 1032, 30522)])
def test_loss_gradients_by_elements(lib, rows, hidden, vocab):
    check_loss_gradients(*loss_inputs(rows, hidden, vocab, rows + vocab))


@pytest.mark.parametrize("first,others", [(1.5 * 2.0 ** -40, 1e30), (1.3 * 2.0 ** 40, 1e-30), (-1e-30, 1e-3), (1e-45, 1.0), (0.0, 1e-3), (-3e38, 1e-6)])
def test_gradients_of_any_size_beside_the_first_rows(lib, first, others):
    """Rows' gradients far above or below the first one's, which they are written as multiples of."""
    x, w, targets, grad = loss_inputs(100, 264, 1000, 12)
    grad = grad * 100 * others * torch.where(torch.arange(100, device="cuda") % 3 == 0, -1.0, 1.0)
    grad[0], targets[0] = first, -100 if abs(first) > 1e38 else 5
    check_loss_gradients(x, w, targets, grad)


def check_gated(x, dy, gate, up, down, act):
    from baranet_bdml_b200 import ops
    rows, inter, hidden = x.shape[0], *gate.shape
    got = ops.gated_ff_backward(dy, x, gate, up, down, act=act)
    X, DY, G, U, D = (t.double() for t in (x, dy, gate, up, down))
    g, u, dh = X @ G.T, X @ U.T, DY @ D
    z = g.clone().requires_grad_(True)
    a = torch.nn.functional.silu(z) if act == "silu" else torch.nn.functional.gelu(z, approximate="tanh")
    slope, = torch.autograd.grad(a.sum(), z)
    a = a.detach()
    # gate, up and dh by their sums; the activation and its slope (both at most |z| + 1.2 in size, with slopes of at most 1.2) by that and by 2^-18
    g_off, u_off, dh_off = (sums(hidden) * (p.abs() @ q.abs()) for p, q in ((X, G.T), (X, U.T), (DY, D)))
    a_off = 1.2 * g_off + 2.0 ** -18 * (g.abs() + 1.2)
    h, dg, du = a * u, dh * u * slope, dh * a
    half = HALF * 1.01 + sums(max(rows, 2 * inter))       # an operand's rounding, and the sums that it goes into
    h_off = half * h.abs() + a_off * u.abs() + a.abs() * u_off
    dg_off = half * dg.abs() + dh_off * (u * slope).abs() + (dh * slope).abs() * u_off + (dh * u).abs() * a_off
    du_off = half * du.abs() + dh_off * a.abs() + dh.abs() * a_off
    within(got[0], dg @ G + du @ U, dg_off @ G.abs() + du_off @ U.abs())
    within(got[1], dg.T @ X, dg_off.T @ X.abs())
    within(got[2], du.T @ X, du_off.T @ X.abs())
    within(got[3], DY.T @ h, DY.abs().T @ h_off)
    again(lambda: ops.gated_ff_backward(dy, x, gate, up, down, act=act), got)
    ops.gemm_status()


@pytest.mark.parametrize("rows,hidden,inter,act", [(64, 1000, 2712, "silu"), (1371, 1000, 2712, "gelu_tanh"), (5000, 2048, 5632, "silu")])
def test_gated_block_gradients_by_elements(lib, rows, hidden, inter, act):
    rng = np.random.default_rng(rows + inter)
    x, dy = bf16(rng, rows, hidden), bf16(rng, rows, hidden, std=1.0 / rows)
    check_gated(x, dy, bf16(rng, inter, hidden, std=hidden ** -0.5), bf16(rng, inter, hidden, std=hidden ** -0.5),
                bf16(rng, hidden, inter, std=inter ** -0.5), act)


# few tiles and a long K: a weight's gradient of a narrow layer over many tokens
@pytest.mark.parametrize("M,N,K", [(256, 256, 16384), (256, 2048, 16384), (8, 8, 16383), (264, 520, 5001)])
def test_product_of_two_transposed_operands_with_a_long_sum(lib, M, N, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + K)
    a, b = bf16(rng, K, M), bf16(rng, K, N, std=K ** -0.5)
    got = ops.gemm_bf16_tn(a, b)
    within(got, a.double().T @ b.double(), sums(K) * (a.double().abs().T @ b.double().abs()))
    again(lambda: [ops.gemm_bf16_tn(a, b)], [got])
    ops.gemm_status()


def test_gated_block_gradients_of_a_narrow_layer(lib):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(9)
    rows, hidden, inter = 16384, 256, 512
    x, dy = bf16(rng, rows, hidden), bf16(rng, rows, hidden, std=1.0 / rows)
    weights = bf16(rng, inter, hidden, std=hidden ** -0.5), bf16(rng, inter, hidden, std=hidden ** -0.5), bf16(rng, hidden, inter, std=inter ** -0.5)
    check_gated(x, dy, *weights, "silu")
