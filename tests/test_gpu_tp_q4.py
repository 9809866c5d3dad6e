"""The 4-bit KV cache of a model split over 2 GPUs: each rank's cache holds its
KV heads, whose attention gives the bits that they have in the whole model
(test_gpu_q4_paths.py, on one GPU), so that the split session's logits are the
unsplit one's at every step.  Skipped on a machine with fewer than 2 GPUs."""
import numpy as np
import pytest

from test_gpu_tp import _run, needs2

pytestmark = pytest.mark.gpu


@needs2
def test_tp2_q4_equals_the_unsplit_session():
    from model_helpers import TINY_LLAMA
    from overfit_b200 import engine
    cfg = dict(TINY_LLAMA)
    prompt = [int(x) for x in np.random.default_rng(5).integers(0, cfg["vocab"], 12)]
    (_, t0, l0, d0, mf), (_, t1, l1, d1, _) = _run(cfg, 21, "q4", prompt, 16)
    assert t0 == t1 and d0 == d1
    whole = engine.CudaLlamaInferenceEngine(cfg, mf, device=0)
    s = whole.create_session(len(prompt) + 32, "q4")
    token = s.prefill(prompt)
    for i, (t, a, b) in enumerate(zip(t0, l0, l1)):
        assert token == t
        np.testing.assert_array_equal(a, b)
        np.testing.assert_array_equal(s.get_last_logits(), a, err_msg=f"step {i}")
        if i < len(t0) - 1:
            token = s.decode(token)
    assert list(s.generate_greedy(4)) == d0
    s.close()
    whole.close()
