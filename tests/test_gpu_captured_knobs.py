"""What a captured step keeps alive."""
import numpy as np
import pytest
import torch

import kv8_cases as K
from test_gpu_model_serving import ids_of, llama

pytestmark = pytest.mark.gpu


def test_a_captured_step_keeps_its_knobs(lib):
    """Tensors that the caller drops are still what the replay reads"""
    rng = np.random.default_rng(9)
    model = llama(2)
    model.prefill(ids_of(rng, 4, 20), 64)
    step = model.capture_decode_step(temperature=torch.full((4,), 1.5, device="cuda"), top_k=torch.full((4,), 7, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    others = [torch.zeros((4,), device="cuda") for _ in range(64)]         # (in the place of what has been given back)
    tok, u = ids_of(rng, 4), torch.tensor([0.3, 0.6, 0.8, 0.95], device="cuda")
    logits, nxt = step(tok, u)
    assert nxt.tolist() == [K.choose(x, float(w), temperature=1.5, top_k=7) for x, w in zip(logits.cpu().numpy(), u)]
    assert not any(t.any() for t in others)
