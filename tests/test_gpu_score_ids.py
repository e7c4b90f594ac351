"""Token ids as a caller has them: on the host, as 64-bit numbers, far outside the vocabulary."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(lib):
    from baranet_bdml_b200.layers import LLaMAConfig
    from baranet_bdml_b200.model import LLaMAModelBF16
    np.random.seed(8)
    return LLaMAModelBF16(LLaMAConfig(vocab_size=504, hidden_size=256, intermediate_size=704, num_hidden_layers=1, num_attention_heads=4,
                                      num_key_value_heads=2))


def test_ids_of_the_host(model):
    ids = torch.from_numpy(np.random.default_rng(8).integers(0, 504, (3, 20)))
    on_gpu = ids.to(torch.int32).cuda()
    assert torch.equal(model.score(ids), model.score(on_gpu))
    assert torch.equal(model(ids), model(on_gpu))
    assert torch.equal(model.prefill(ids, 30), model.prefill(on_gpu, 30))
    a = model.decode_step(ids[:, 0])
    model.prefill(on_gpu, 30)
    assert torch.equal(a, model.decode_step(on_gpu[:, 0].contiguous()))


@pytest.mark.parametrize("bad", [504, -1, 2**32 + 5, -2**32 + 5, 2**31])
def test_scores_of_ids_outside_the_vocabulary(model, bad):
    ids = torch.full((2, 6), 7, dtype=torch.int64, device="cuda")
    ids[1, 3] = bad
    with pytest.raises(IndexError):
        model.score(ids)
    assert torch.isfinite(model.score(torch.full((2, 6), 7, dtype=torch.int64, device="cuda"))).all()
