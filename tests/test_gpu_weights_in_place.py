"""The bf16 layers read their weights as they are at the time of a call, forward and backward alike: written in place, through `.data`,
assigned anew (twice, so that an address comes back), and by a captured graph."""
import numpy as np
import pytest
import torch

from test_gpu_training import bf16, off

pytestmark = pytest.mark.gpu
HALF = torch.finfo(torch.bfloat16).eps / 2


def changes(owner, names):
    """Ways to write a layer's weights, each a function that does it"""
    def in_place():
        for n in names:
            getattr(owner, n).mul_(-0.75)

    def through_data():
        for n in names:
            getattr(owner, n).data.add_(0.01)

    def another_storage():
        for n in names:
            getattr(owner, n).data = getattr(owner, n).data * 1.25

    def anew_twice():
        for n in names:
            for factor in (0.9, -0.8):
                setattr(owner, n, getattr(owner, n) * factor)

    def one_alone():
        setattr(owner, names[0], getattr(owner, names[0]) * -0.7)
        getattr(owner, names[-1]).mul_(1.5)

    return [in_place, through_data, another_storage, anew_twice, one_alone, in_place, through_data]


def mlp_of(seed, hidden=256, inter=712):
    from baranet_bdml_b200.layers import LLaMAConfig, MLPBF16
    np.random.seed(seed)
    return MLPBF16(LLaMAConfig(vocab_size=100, hidden_size=hidden, intermediate_size=inter, num_attention_heads=4, num_key_value_heads=2))


def mlp_oracle(mlp, x, leaves=None):
    X, G, U, D = leaves or [t.double() for t in (x, *mlp.parameters())]
    return (torch.nn.functional.silu(X @ G.T) * (X @ U.T)) @ D.T


def test_gated_block(lib):
    mlp, rng = mlp_of(1), np.random.default_rng(1)
    x, dy = bf16(rng, 333, 256), bf16(rng, 333, 256)
    for change in [lambda: None] + changes(mlp, ("gate_proj", "up_proj", "down_proj")):
        change()
        # rounded on the way: the product of gate and up, and the result
        assert off(mlp(x), mlp_oracle(mlp, x)) <= 2 * HALF, change
        assert off(mlp(x[:40], few_rows=True), mlp_oracle(mlp, x[:40])) <= 2 * HALF, change
        got, grads = mlp.backward(dy, x)
        leaves = [t.double().requires_grad_(True) for t in (x, *mlp.parameters())]
        for a, b in zip((got, *grads), torch.autograd.grad(mlp_oracle(mlp, x, leaves), leaves, dy.double())):
            assert off(a, b) <= 3 * HALF, change


def test_gated_block_in_a_graph(lib):
    mlp, rng = mlp_of(2), np.random.default_rng(2)
    x = bf16(rng, 200, 256)
    mlp(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x)
    for factor in (1.0, -0.5, 3.0):
        for w in mlp.parameters():
            w.mul_(factor)
        graph.replay()
        torch.cuda.synchronize()
        assert off(out, mlp_oracle(mlp, x)) <= 2 * HALF, factor


# both routes of few rows, single tiles and pairs, and sizes that no tile divides
@pytest.mark.parametrize("M,inter,K", [(1, 8, 8), (17, 712, 256), (20, 2816, 2048), (64, 5632, 2048), (100, 2816, 2048), (128, 136, 1288), (333, 712, 256),
                                       (2500, 5632, 2048), (4097, 2712, 1000), (3000, 1416, 1024)])
def test_weights_apart_are_the_packed_ones_bits(lib, M, inter, K):
    from baranet_bdml_b200 import ops
    rng = np.random.default_rng(M + inter)
    x, gate, up = bf16(rng, M, K), bf16(rng, inter, K, std=K ** -0.5), bf16(rng, inter, K, std=K ** -0.5)
    got = ops.gemm_swiglu_bf16_nt_separate(x, gate, up)
    assert torch.equal(got, ops.gemm_swiglu_bf16_nt(x, ops.pack_gate_up(gate, up), inter))
    g = x.double() @ gate.double().T
    # the product's own rounding, half a step of every element; sums and the fast exponential are far below the other half
    assert off(got, torch.nn.functional.silu(g) * (x.double() @ up.double().T)) <= HALF
    ops.gemm_status()
