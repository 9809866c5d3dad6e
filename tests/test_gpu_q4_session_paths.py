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


def test_bits_of_a_batch_beside_a_long_session(engine):
    """Alone, a session's step joins its chunks in the attention's launch; beside a session of more than 12288 positions
    a kernel for many chunks joins every row, and beside many sessions one for few.  Chunks of 256 and of 512."""
    shapes = [(700, 1000), (3000, 4096), (2700, 8192), (513, 5000), (40, 12288), (1100, 13000)]
    V = engine.vocabulary_size
    alone = [engine.create_session(c, "q4") for _, c in shapes]
    batch = [engine.create_session(c, "q4") for _, c in shapes]
    for i, (n, _) in enumerate(shapes):
        for s in (alone[i], batch[i]):
            s.prefill(prompt(n, V, i))
    for step in range(3):
        t = prompt(len(shapes), V, 50 + step)
        am = engine.decode_batch(batch, t)
        for i, s in enumerate(alone):
            assert s.decode(t[i]) == am[i]
            np.testing.assert_array_equal(batch[i].get_last_logits(), s.get_last_logits())
    # 40 sessions (80 groups of rows), none of more than 12288 positions
    more = [engine.create_session(600, "q4") for _ in range(35)]
    for i, s in enumerate(more):
        s.prefill(prompt(3 + 14 * i, V, 70 + i))
    t = prompt(40, V, 90)
    am = engine.decode_batch(batch[:5] + more, t)
    for i, s in enumerate(alone[:5]):
        assert s.decode(t[i]) == am[i]
        np.testing.assert_array_equal(batch[i].get_last_logits(), s.get_last_logits())
    # and a verify of 17 rows over chunks of 512 (two parts of it) against single steps
    rows = prompt(17, V, 91)
    am, lg = batch[2].verify(rows, want_logits=True)
    for j, x in enumerate(rows):
        assert alone[2].decode(x) == am[j]
        np.testing.assert_array_equal(alone[2].get_last_logits(), lg[j])
    for s in alone + batch + more:
        s.close()


def test_calls_without_rows(K):
    """No sequences, or no rows: nothing is done."""
    A = K.CachedAttentionKernel
    kc, vc = (torch.zeros(K.KvCacheQ4.bytes(2, 64, 32), dtype=torch.uint8, device="cuda") for _ in "kv")
    scratch = torch.zeros(256, dtype=torch.uint8, device="cuda")
    for n, rows in ((0, 1), (1, 0), (0, 0)):
        pos = torch.zeros(n, dtype=torch.int32, device="cuda")
        k, v, k2, v2 = (torch.zeros(n, rows, 128, device="cuda") for _ in range(4))
        q, out = torch.zeros(n, rows, 256, device="cuda"), torch.zeros(n, rows, 256, device="cuda")
        K.KvCacheQ4.append(k, v, kc, vc, pos, 2, 64, 32)
        K.KvCacheQ4.read(kc, vc, pos, 2, 64, 32, k2, v2)
        A.compute_q4(q, kc, vc, out, pos, 4, 2, 64, 32, 0.1, scratch)
        A.compute_q4(q, kc, vc, out, pos, 4, 2, 64, 32, 0.1, scratch, k_new=k, v_new=v)
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    K.SpeculativeVerifier.verify(torch.zeros(0, 3, 100, device="cuda"), torch.zeros(0, 2, dtype=torch.int32, device="cuda"),
                                 torch.zeros(0, 3, device="cuda"), torch.zeros(0, device="cuda"), empty, empty.clone())
    assert device_error() == 0 and not kc.any() and not vc.any()
