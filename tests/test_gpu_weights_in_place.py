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


# ------------------------------------------------------------------------------------------------------------- attention
from test_gpu_training import attention_oracle      # noqa: E402


def attention_of(seed, hidden=256):
    from baranet_bdml_b200.layers import GroupedQueryAttentionBF16, LLaMAConfig
    np.random.seed(seed)
    return GroupedQueryAttentionBF16(LLaMAConfig(vocab_size=100, hidden_size=hidden, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2))


def layer_oracle(attn, x, leaves=None):
    X, wq, wk, wv, wo = leaves or [t.double() for t in (x, *attn.parameters())]
    S = x.shape[0]
    o, _ = attention_oracle((X @ wq.T).view(1, S, 4, 64), (X @ wk.T).view(1, S, 2, 64), (X @ wv.T).view(1, S, 2, 64), 0, True, 0.125)
    return o.reshape(S, 256) @ wo.T


def check_attention(attn, x, dy, what):
    # q, k, v (as projected, and rotated), P, the attention rows, the result
    assert off(attn(x), layer_oracle(attn, x)) <= 6 * HALF, what
    got, grads = attn.backward(dy, x)
    leaves = [t.double().requires_grad_(True) for t in (x, *attn.parameters())]
    # the attention's own roundings, q, k, v, dattn, the gradients of q, k and v, and the result's
    for a, b in zip((got, *grads), torch.autograd.grad(layer_oracle(attn, x, leaves), leaves, dy.double())):
        assert off(a, b) <= 12 * HALF, what


def test_attention(lib):
    attn, rng = attention_of(3), np.random.default_rng(3)
    x, dy = bf16(rng, 60, 256), bf16(rng, 60, 256)
    for change in [lambda: None] + changes(attn, ("q_proj", "k_proj", "v_proj", "o_proj")) + [attn.stack_qkv] + changes(attn, ("v_proj", "k_proj", "q_proj")):
        change()
        check_attention(attn, x, dy, change)


def test_attention_weights_kept_and_put_back(lib):
    """A weight that is taken out and put back later is the one that it was."""
    attn, rng = attention_of(4), np.random.default_rng(4)
    x = bf16(rng, 60, 256)
    first, kept = attn(x), attn.k_proj
    attn.k_proj = bf16(rng, 128, 256, std=0.1)
    assert not torch.equal(attn(x), first) and off(attn(x), layer_oracle(attn, x)) <= 6 * HALF
    attn.stack_qkv()
    assert off(attn(x), layer_oracle(attn, x)) <= 6 * HALF
    attn.k_proj = kept
    assert torch.equal(attn(x), first)


def test_attention_of_neighbouring_rows_of_another_tensor(lib):
    """Weights that lie one behind the other in a tensor of the caller's own, in another order, or as copies of one."""
    attn, rng = attention_of(5), np.random.default_rng(5)
    x, dy = bf16(rng, 60, 256), bf16(rng, 60, 256)
    own = bf16(rng, 512, 256, std=0.1)
    for q, k, v in (((0, 256), (256, 384), (384, 512)), ((256, 512), (0, 128), (128, 256)), ((0, 256), (256, 384), (256, 384))):
        attn.q_proj, attn.k_proj, attn.v_proj = own[q[0]:q[1]], own[k[0]:k[1]], own[v[0]:v[1]]
        own.mul_(-0.9)
        check_attention(attn, x, dy, (q, k, v))


@pytest.mark.parametrize("assigned", [False, True])
def test_a_captured_layer_follows_its_weights(lib, assigned):
    from baranet_bdml_b200.layers import GraphedDecoderLayerBF16, LLaMAConfig, LLaMADecoderLayerBF16
    np.random.seed(6)
    layer = LLaMADecoderLayerBF16(LLaMAConfig(vocab_size=100, hidden_size=256, intermediate_size=712, num_attention_heads=4, num_key_value_heads=2))
    rng = np.random.default_rng(6)
    if assigned:
        for n in ("q_proj", "k_proj", "v_proj"):
            setattr(layer.self_attn, n, getattr(layer.self_attn, n) * 0.5)
    x = bf16(rng, 1, 70, 256)
    graphed = GraphedDecoderLayerBF16(layer, x)
    for factor in (1.0, -0.8, 1.3):
        for w in layer.self_attn.parameters() + layer.mlp.parameters():
            w.mul_(factor)
        residual, out = (t.clone() for t in graphed(x))
        eager = layer.forward_parts(x)
        assert torch.equal(residual, eager[0]) and torch.equal(out, eager[1]), factor


def test_steps_and_prompts_of_a_model_follow_its_weights(lib):
    """`__call__`, prefill and the following step before and after a write, against the same model built from the new weights."""
    from baranet_bdml_b200.layers import LLaMAConfig
    from baranet_bdml_b200.model import LLaMAModelBF16
    cfg = LLaMAConfig(vocab_size=504, hidden_size=256, intermediate_size=712, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)
    np.random.seed(7)
    model = LLaMAModelBF16(cfg)
    ids = torch.from_numpy(np.random.default_rng(7).integers(0, 504, (2, 21)).astype(np.int32)).cuda()
    run = lambda m: (m(ids), m.prefill(ids, 30), m.decode_step(ids[:, 0].contiguous()), m.score(ids))      # noqa: E731
    before = run(model)
    for w in model.parameters():
        w.mul_(1.5)
    after = run(model)
    np.random.seed(7)
    other = LLaMAModelBF16(cfg)
    for w, o in zip(model.parameters(), other.parameters()):
        o.copy_(w)
    for a, b, c in zip(before, after, run(other)):
        assert torch.equal(b, c) and not torch.equal(a, b)
