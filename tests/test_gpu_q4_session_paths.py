"""Sessions with the 4-bit cache beside other callers and in batches whose rows
go through different kernels than they do alone."""
import numpy as np
import pytest

from test_gpu_q4 import K, dev, device_error  # noqa: F401  (K is the fixture)
from test_gpu_q4_session import prompt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def engine():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from model_helpers import TINY_LLAMA, make_model_file
    from overfit_b200 import build, engine
    build.build()
    e = engine.CudaLlamaInferenceEngine(dict(TINY_LLAMA), make_model_file(TINY_LLAMA, seed=5), device=0)
    yield e
    e.close()


@pytest.mark.parametrize("kv", ["f32", "q4"])
def test_a_callers_bad_position_is_not_a_sessions(K, engine, kv):
    """Rows that a kernel-level caller's cache has no room for are reported to that caller, whatever session calls end in
    between, and those do not fail for it."""
    s, other = engine.create_session(100, kv), engine.create_session(100, kv)
    s.prefill(prompt(20, engine.vocabulary_size))
    kc, vc = (torch.zeros(K.KvCacheQ4.bytes(1, 64, 40), dtype=torch.uint8, device="cuda") for _ in "kv")
    x = torch.randn(1, 4, 64, device="cuda")
    assert device_error() == 0
    calls = [lambda: s.decode(3), lambda: s.verify([4, 5, 6]), lambda: s.verify_sampled([4, 5], [0.5, 0.5], 1.0),
             lambda: other.prefill(prompt(30, engine.vocabulary_size)), lambda: engine.decode_batch([s, other], [1, 2]),
             lambda: s.generate_greedy(3)]
    for call in calls:
        at = s.current_position
        K.KvCacheQ4.append(x, x, kc, vc, dev([37], torch.int32), 1, 64, 40)
        torch.cuda.synchronize()
        call()
        assert s.current_position >= at
        assert device_error() == 4 and device_error() == 0
    s.close()
    other.close()
