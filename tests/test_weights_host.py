"""Checks of the gated product with its weights apart, no GPU needed: every call is refused before a launch."""
import pytest
import torch

P = 1 << 20            # an aligned address that no refused call touches


def test_gated_product_of_weights_apart(lib):
    from baranet_bdml_b200 import _lib
    call = lib.bn_gemm_swiglu_bf16_nt_separate
    for status, text, args in ((_lib.BN_ERR_INVALID_ARG, "null pointer", (P, P, None, P, 4, 64, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "null pointer", (P, None, P, P, 4, 64, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "null pointer", (None, P, P, P, 4, 64, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "16-byte aligned", (P, P, P + 8, P, 4, 64, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "bad shape", (P, P, P, P, 4, -8, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "bad shape", (P, P, P, P, 4, 2**31 - 8, 64)),
                               (_lib.BN_ERR_INVALID_ARG, "bad shape", (P, P, P, P, -4, 64, 64)),
                               (_lib.BN_ERR_UNSUPPORTED, "multiples of 8", (P, P, P, P, 4, 60, 64)),
                               (_lib.BN_ERR_UNSUPPORTED, "multiples of 8", (P, P, P, P, 4, 64, 60))):
        assert call(*args, None, None) == status, args
        assert text in _lib.last_error(), _lib.last_error()


def test_host_tensors_are_refused():
    from baranet_bdml_b200 import ops
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((104, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="only GPU implementation available"):
        ops.gemm_swiglu_bf16_nt_separate(x, w, w)
