"""Sessions that are cut back again and again: verified and sampled drafts, single
steps and batches, more of them than the session has positions."""
import numpy as np
import pytest

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
@pytest.mark.parametrize("how", ["verify", "verify_sampled", "decode", "batch"])
def test_more_cuts_than_positions(engine, kv, how):
    """The log of sampled tokens starts anew behind a cut, so that it never grows past its end, and goes on from the token
    that the session holds."""
    capacity, base = 33, 20
    prompt = np.random.default_rng(1).integers(0, engine.vocabulary_size, base).tolist()
    a, b = engine.create_session(capacity, kv), engine.create_session(capacity, kv)
    a.prefill(prompt)
    b.prefill(prompt)
    for i in range(3 * capacity):
        if how == "verify":
            a.verify([i, i + 1, i + 2])
        elif how == "verify_sampled":
            a.verify_sampled([i, i + 1, i + 2], [0.5, 0.5, 0.5], 1.0)
        elif how == "decode":
            a.decode(i)
        else:
            engine.decode_batch([a], [i])
        a.rollback_to(base)
    assert a.decode(7) == b.decode(7)
    np.testing.assert_array_equal(a.generate_greedy(capacity - base - 1), b.generate_greedy(capacity - base - 1))
    assert a.current_position == capacity
    a.close()
    b.close()


def test_a_cut_keeps_the_token_that_comes_next(engine):
    """Generation behind a cut starts with the last sampled token, as before the cut."""
    prompt = np.random.default_rng(2).integers(0, engine.vocabulary_size, 20).tolist()
    s = engine.create_session(60)
    for cut in (20, 18):
        s.reset()
        token = s.prefill(prompt)
        for t in (3, 4):
            token = s.decode(t)
        s.rollback_to(cut)
        got = s.generate_greedy(3)
        assert got[0] == token and s.current_position == cut + 3
    s.close()


def test_nothing_is_generated_behind_a_sampled_verify(engine):
    """The token that it drew is not decoded yet; the last row's greedy token is of rejected drafts."""
    prompt = np.random.default_rng(3).integers(0, engine.vocabulary_size, 20).tolist()
    s, twin = engine.create_session(60, "q4"), engine.create_session(60, "q4")
    for x in (s, twin):
        x.prefill(prompt)
    accepted, token = s.verify_sampled([5, 6, 7], [0.9, 0.9, 0.5], 1.0)
    with pytest.raises(ValueError):
        s.generate_greedy(1)
    for t in [5, 6, 7][:accepted + 1] + [token]:
        want = twin.decode(t)
    assert s.decode(token) == want
    np.testing.assert_array_equal(s.generate_greedy(5), twin.generate_greedy(5))
    s.close()
    twin.close()
