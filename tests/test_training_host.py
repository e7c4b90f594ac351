"""The training operators' argument checks and workspace sizes: status codes, no GPU needed (every call here is refused before a launch)."""
import pytest
import torch

P = 1 << 20            # an aligned address that no refused call touches


def refused(lib, status, text, name, *args):
    from baranet_bdml_b200 import _lib
    assert getattr(lib, name)(*args) == status, (name, args)
    assert text in _lib.last_error(), _lib.last_error()


def test_products(lib):
    from baranet_bdml_b200 import _lib
    bad, unsupported = _lib.BN_ERR_INVALID_ARG, _lib.BN_ERR_UNSUPPORTED
    refused(lib, bad, "null pointer", "bn_gemm_bf16_nn", None, P, P, 8, 8, 8, None, 0, None, None)
    refused(lib, bad, "bad shape", "bn_gemm_bf16_nn", P, P, P, -1, 8, 8, None, 0, None, None)
    refused(lib, unsupported, "multiples of 8", "bn_gemm_bf16_nn", P, P, P, 8, 12, 8, None, 0, None, None)
    refused(lib, unsupported, "multiples of 8", "bn_gemm_bf16_nn", P, P, P, 8, 8, 12, None, 0, None, None)
    refused(lib, unsupported, "multiples of 8", "bn_gemm_bf16_tn", P, P, P, 12, 8, 8, None, None)
    refused(lib, bad, "16-byte aligned", "bn_gemm_bf16_tn", P + 2, P, P, 8, 8, 8, None, None)
    assert lib.bn_gemm_bf16_nn_workspace_bytes(0, 8, 8) == 0
    # few tiles and a long K: ranges of K, whose fp32 sums need room; many tiles: none
    assert lib.bn_gemm_bf16_nn_workspace_bytes(64, 2048, 32000) >= 2 * 64 * 2048 * 4
    assert lib.bn_gemm_bf16_nn_workspace_bytes(16384, 2048, 2048) == 0


def test_loss(lib):
    from baranet_bdml_b200 import _lib
    bad, unsupported = _lib.BN_ERR_INVALID_ARG, _lib.BN_ERR_UNSUPPORTED
    call = "bn_linear_cross_entropy_bf16"
    refused(lib, bad, "null pointer", call, P, None, P, P, P, 4, 100, 64, P, 1 << 20, None, None, None)
    refused(lib, bad, "null pointer", call, P, P, P, None, P, 4, 100, 64, P, 1 << 20, None, None, None)
    refused(lib, bad, "bad shape", call, P, P, P, P, P, 4, 0, 64, P, 1 << 20, None, None, None)
    refused(lib, unsupported, "multiple of 8", call, P, P, P, P, P, 4, 100, 60, P, 1 << 20, None, None, None)
    refused(lib, bad, "16-byte aligned", call, P + 8, P, P, P, P, 4, 100, 64, P, 1 << 20, None, None, None)
    back = "bn_linear_cross_entropy_backward_bf16"
    refused(lib, bad, "null pointer", back, P, P, P, P, P, None, None, 4, 100, 64, P, 1 << 20, None, None)
    refused(lib, bad, "null pointer", back, P, P, P, None, P, P, P, 4, 100, 64, P, 1 << 20, None, None)
    refused(lib, bad, "16-byte aligned", back, P, P, P, P, P, P + 4, P, 4, 100, 64, P, 1 << 20, None, None)


@pytest.mark.parametrize("rows,vocab,hidden", [(1, 1, 8), (64, 32000, 2048), (8192, 32000, 2048), (100000, 50000, 64), (3, 1 << 24, 8)])
def test_the_logits_take_no_room(lib, rows, vocab, hidden):
    """A maximum, a sum and a logit for 128 columns at least; a backward pass: a piece of 128 MB or 4096 columns, and the rows' fp32 gradients"""
    forward = lib.bn_linear_cross_entropy_bf16_workspace_bytes(rows, vocab, hidden)
    assert 0 < forward <= rows * 8 * (vocab // 128 + 1) + rows * 4 + 512
    back = lib.bn_linear_cross_entropy_backward_bf16_workspace_bytes(rows, vocab, hidden)
    assert 0 < back <= max(128 << 20, rows * 4096 * 2) + rows * 512 + 32 * rows * hidden * 4 + 512


def test_gated_block(lib):
    from baranet_bdml_b200 import _lib
    bad, unsupported = _lib.BN_ERR_INVALID_ARG, _lib.BN_ERR_UNSUPPORTED
    call, tail = "bn_gated_ff_backward_bf16", (P, 1 << 30, None, None)
    refused(lib, bad, "null pointer", call, *[P] * 8, None, 4, 64, 64, _lib.BN_ACT_SILU, *tail)
    refused(lib, bad, "bad shape", call, *[P] * 9, -4, 64, 64, _lib.BN_ACT_SILU, *tail)
    refused(lib, unsupported, "multiples of 8", call, *[P] * 9, 4, 64, 60, _lib.BN_ACT_SILU, *tail)
    refused(lib, unsupported, "activation", call, *[P] * 9, 4, 64, 64, _lib.BN_ACT_RELU2, *tail)
    refused(lib, bad, "16-byte aligned", call, P + 2, *[P] * 8, 4, 64, 64, _lib.BN_ACT_SILU, *tail)
    assert lib.bn_gated_ff_backward_bf16_workspace_bytes(0, 64, 64) == 0
    assert lib.bn_gated_ff_backward_bf16_workspace_bytes(16384, 2048, 5632) >= 16384 * 5632 * (3 * 2 + 4)


def test_attention(lib):
    from baranet_bdml_b200 import _lib
    bad, unsupported = _lib.BN_ERR_INVALID_ARG, _lib.BN_ERR_UNSUPPORTED
    call, tail = "bn_attn_prefill_bf16_backward", (P, 1 << 30, None, None)
    refused(lib, bad, "null pointer", call, *[P] * 8, None, 1, 10, 8, 2, 64, 0.125, 1e4, 0, 1, *tail)
    refused(lib, bad, "bad shape", call, *[P] * 9, 1, -1, 8, 2, 64, 0.125, 1e4, 0, 1, *tail)
    refused(lib, bad, "not a multiple", call, *[P] * 9, 1, 10, 8, 3, 64, 0.125, 1e4, 0, 1, *tail)
    refused(lib, unsupported, "head_dim", call, *[P] * 9, 1, 10, 8, 2, 128, 0.125, 1e4, 0, 1, *tail)
    refused(lib, bad, "position_offset", call, *[P] * 9, 1, 10, 8, 2, 64, 0.125, 1e4, -1, 1, *tail)
    refused(lib, bad, "16-byte aligned", call, P + 2, *[P] * 8, 1, 10, 8, 2, 64, 0.125, 1e4, 0, 1, *tail)
    size = lib.bn_attn_prefill_bf16_backward_workspace_bytes
    assert size(1, 10, 8, 2, 128, 1) == 0 and size(1, 10, 8, 3, 64, 1) == 0 and size(0, 10, 8, 2, 64, 1) == 0
    # rotated copies of q and k, two numbers a query, nothing of size S x S
    assert 8 * 2048 * 36 * 128 <= size(8, 2048, 32, 4, 64, 1) <= 8 * 2048 * 36 * 128 + 8 * 32 * 2048 * 8 + 2048 * 256 + 2048


def test_operators_refuse_host_tensors():
    from baranet_bdml_b200 import ops
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((100, 64), dtype=torch.bfloat16)
    q = torch.zeros((1, 4, 8, 64), dtype=torch.bfloat16)
    for call in (lambda: ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int32)), lambda: ops.gemm_bf16_nn(x, w.T.contiguous()),
                 lambda: ops.gemm_bf16_tn(x, x), lambda: ops.gated_ff_backward(x, x, w, w, w.T.contiguous()),
                 lambda: ops.linear_cross_entropy_backward(x, w, torch.zeros(4, dtype=torch.int32), torch.zeros(4), torch.zeros(4)),
                 lambda: ops.attn_prefill_bf16_backward(q, q, q, q, q, torch.zeros((1, 8, 4)))):
        with pytest.raises(RuntimeError, match="only GPU implementation available"):
            call()


LONGEST = 2**31 - 1


def test_sizes_that_tiles_do_not_number(lib):
    """Lengths that leave 32 bits when they are rounded up to a tile"""
    from baranet_bdml_b200 import _lib
    unsupported = _lib.BN_ERR_UNSUPPORTED
    refused(lib, unsupported, "too large", "bn_gemm_bf16_nn", P, P, P, LONGEST, 8, 8, P, 1 << 30, None, None)
    refused(lib, unsupported, "too large", "bn_gemm_bf16_tn", P, P, P, 8, 8, LONGEST, None, None)
    refused(lib, unsupported, "too large", "bn_linear_cross_entropy_bf16", *[P] * 5, LONGEST, 100, 8, P, 1 << 30, None, None, None)
    refused(lib, unsupported, "too large", "bn_linear_cross_entropy_backward_bf16", *[P] * 7, 8, LONGEST, 8, P, 1 << 30, None, None)
    refused(lib, unsupported, "too large", "bn_gated_ff_backward_bf16", *[P] * 9, LONGEST, 8, 8, _lib.BN_ACT_SILU, P, 1 << 30, None, None)
    attn, tail = "bn_attn_prefill_bf16_backward", (P, 1 << 30, None, None)
    refused(lib, unsupported, "too large", attn, *[P] * 9, 1, LONGEST, 1, 1, 64, 0.125, 1e4, 0, 1, *tail)
    refused(lib, unsupported, "too large", attn, *[P] * 9, 65536, 1, 1, 1, 64, 0.125, 1e4, 0, 1, *tail)
    refused(lib, unsupported, "too large", attn, *[P] * 9, 1, 10, 1, 1, 64, 0.125, 1e4, LONGEST - 100, 1, *tail)
    assert lib.bn_gemm_bf16_nn_workspace_bytes(LONGEST, 8, 8) == 0
    assert lib.bn_linear_cross_entropy_bf16_workspace_bytes(LONGEST, 8, 8) == lib.bn_linear_cross_entropy_backward_bf16_workspace_bytes(8, LONGEST, 8) == 0
    assert lib.bn_gated_ff_backward_bf16_workspace_bytes(8, 8, LONGEST) == lib.bn_attn_prefill_bf16_backward_workspace_bytes(1, LONGEST, 1, 1, 64, 1) == 0
