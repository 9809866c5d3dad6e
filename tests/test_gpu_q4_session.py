"""Sessions with the 4-bit KV cache, and the sampled verify, on tiny models.

A 4-bit session has no counterpart among the restatement's sessions, so its
paths are held to one another bit for bit (decode, batch decode, verify,
truncate), its attention to 64-bit forms in test_gpu_q4.py, and its logits to
those of an F32 session only so far that it is the same model: unrelated logits
have a relative distance of about 1.4, and a 4-bit cache's rounding (a step of
1/15 of a group's span, so about 5 % of an element) stays well below half.  That
does not bound a model that routes each token to some of its experts: an expert
whose score is nearly another's changes place with it for any rounding, and its
output is another matrix's.  So logits are compared where every expert is used
(mixtral_all: the same weights, no choice), and the routed model's paths are held
to one another only."""
import numpy as np
import pytest

import q4_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def engines():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from model_helpers import TINY_LLAMA, TINY_MIXTRAL, TINY_QWEN, make_model_file
    from overfit_b200 import build, engine
    build.build()
    made = {}
    for name, cfg in (("llama", TINY_LLAMA), ("qwen", TINY_QWEN), ("mixtral", TINY_MIXTRAL),
                      ("mixtral_all", dict(TINY_MIXTRAL, n_experts_used=TINY_MIXTRAL["n_experts"]))):
        made[name] = engine.CudaLlamaInferenceEngine(cfg, make_model_file(cfg, seed=5), device=0)
    yield made
    for e in made.values():
        e.close()


def prompt(n, vocab, seed=0):
    return np.random.default_rng(seed).integers(0, vocab, n).tolist()


def distance(a, b):
    return np.linalg.norm(a - b) / np.linalg.norm(b)


@pytest.mark.parametrize("name", ["llama", "qwen", "mixtral", "mixtral_all"])
@pytest.mark.parametrize("n", [5, 40, 300])
def test_prefill_and_decode(engines, name, n):
    """Short prompts take the single-token loop, longer ones the batched prefill, 300 two chunks of it."""
    e = engines[name]
    toks = prompt(n, e.vocabulary_size)
    q4, f32 = e.create_session(400, "q4"), e.create_session(400)
    loop = e.create_session(400, "q4")
    loop.disable_batched_prefill_for_parity = True
    for s in (q4, f32, loop):
        s.prefill(toks)
        assert s.current_position == n
    for t in prompt(6, e.vocabulary_size, 1):
        if name != "mixtral":
            assert distance(q4.get_last_logits(), f32.get_last_logits()) < 0.5
            # within rounding of one another until a code of the cache falls the other way, which a 4-bit step shows
            assert distance(loop.get_last_logits(), q4.get_last_logits()) < 0.5
        assert np.isfinite(q4.get_last_logits()).all()
        for s in (q4, f32, loop):
            s.decode(t)
    greedy = q4.generate_greedy(8)
    assert greedy.shape == (8,) and q4.current_position == n + 14
    for s in (q4, f32, loop):
        s.close()


@pytest.mark.parametrize("name", ["llama", "qwen", "mixtral"])
def test_verify_and_truncate_equal_decode(engines, name):
    e = engines[name]
    a, b = e.create_session(600, "q4"), e.create_session(600, "q4")
    toks, rows = prompt(280, e.vocabulary_size), prompt(20, e.vocabulary_size, 2)
    a.prefill(toks)
    b.prefill(toks)
    am, lg = a.verify(rows, want_logits=True)
    for j, t in enumerate(rows):
        assert b.decode(t) == am[j]
        np.testing.assert_array_equal(b.get_last_logits(), lg[j])
    # back to the middle of a block of eight positions, and on with other tokens
    for s in (a, b):
        s.rollback_to(283)
    other = prompt(3, e.vocabulary_size, 3)
    am, lg = a.verify(other, want_logits=True)
    for j, t in enumerate(other):
        b.decode(t)
        np.testing.assert_array_equal(b.get_last_logits(), lg[j])
    a.close()
    b.close()


def test_batch_decode_equals_decode(engines):
    """Four-bit sessions of unequal lengths and capacities in one batch; then one among sessions of other types."""
    e = engines["llama"]
    shapes = [(5, 64), (300, 600), (17, 1000), (64, 65)]
    batch = [e.create_session(c, "q4") for _, c in shapes]
    alone = [e.create_session(c, "q4") for _, c in shapes]
    for i, (n, _) in enumerate(shapes):
        for s in (batch[i], alone[i]):
            s.prefill(prompt(n, e.vocabulary_size, i))
    t = prompt(4, e.vocabulary_size, 9)
    am = e.decode_batch(batch, t)
    for i in range(4):
        assert alone[i].decode(t[i]) == am[i]
        np.testing.assert_array_equal(batch[i].get_last_logits(), alone[i].get_last_logits())
    f32, twin = e.create_session(64), e.create_session(64)
    for s in (f32, twin):
        s.prefill(prompt(9, e.vocabulary_size, 7))
    t = prompt(3, e.vocabulary_size, 10)
    am = e.decode_batch([batch[1], f32, batch[2]], t)
    for s, x, k in ((alone[1], t[0], 0), (twin, t[1], 1), (alone[2], t[2], 2)):
        assert s.decode(x) == am[k]
    np.testing.assert_array_equal(batch[2].get_last_logits(), alone[2].get_last_logits())
    np.testing.assert_array_equal(f32.get_last_logits(), twin.get_last_logits())
    with pytest.raises(ValueError):  # the last session is full
        e.decode_batch(batch, [1, 2, 3, 4])
    for s in batch + alone + [f32, twin]:
        s.close()


@pytest.mark.parametrize("kv", ["q4", "f32"])
@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_sampled(engines, kv, with_probs):
    """Accepted drafts and the drawn token are those of the rows' logits; the session goes on behind them."""
    e = engines["llama"]
    V = e.vocabulary_size
    rng = np.random.default_rng(11)
    a, b, c = (e.create_session(300, kv) for _ in range(3))
    toks = prompt(50, V)
    for s in (a, b, c):
        s.prefill(toks)
    for step, T in enumerate((0.7, 1.3, 0.0, 0.05)):
        rows = prompt(6, V, 20 + step)
        am, lg = b.verify(rows, want_logits=True)
        b.rollback_to(a.current_position)
        rows[1:4] = am[0], *(int(x) for x in rng.integers(0, V, 2))  # a likely first draft
        am, lg = b.verify(rows, want_logits=True)
        q = rng.dirichlet(np.full(V, 0.05), 5).astype(np.float32) if with_probs else None
        u = rng.random(6, dtype=np.float32)
        if step == 2:
            u[:] = 0.999
        base = a.current_position
        accepted, token = a.verify_sampled(rows, u, T, q)
        assert (accepted, token) == ref.verify(lg, rows[1:], u, np.float32(T), q, 5)
        assert a.current_position == base + 1 + accepted
        b.rollback_to(base + 1 + accepted)
        for t in rows[:1 + accepted]:
            c.decode(t)
        for s in (a, b, c):
            s.decode(token)
        np.testing.assert_array_equal(a.get_last_logits(), b.get_last_logits())
        np.testing.assert_array_equal(a.get_last_logits(), c.get_last_logits())
    assert a.verify_sampled([3], [0.5], 1.0)[0] == 0  # no drafts: one sampled step
    for s in (a, b, c):
        s.close()


def test_speculative_sampled_generation(engines):
    """Runs, commits what it returns, and is a matter of the generator alone."""
    e = engines["llama"]
    got = []
    for _ in range(2):
        s = e.create_session(200, "q4")
        history = prompt(4, e.vocabulary_size) * 6
        s.prefill(history)
        rng = np.random.default_rng(3)
        while s.current_position < 60:
            new = s.generate_speculative_sampled(history, rng, 0.8)
            assert new and all(0 <= t < e.vocabulary_size for t in new)
            history += new
            assert s.current_position == len(history)
        got.append(history)
        s.close()
    assert got[0] == got[1]


def test_refusals(engines):
    e = engines["llama"]
    s = e.create_session(40, "q4")
    s.prefill(prompt(20, e.vocabulary_size))
    with pytest.raises(NotImplementedError):
        s.save_prefix()
    with pytest.raises(ValueError):
        s.verify_sampled([1, 2], [0.5], 1.0)
    with pytest.raises(ValueError):
        s.verify_sampled([1, 2], [0.5, 0.5], 1.0, np.ones((2, 3), np.float32))
    with pytest.raises(ValueError):
        s.verify_sampled([1] * 21, [0.5] * 21, 1.0)
    with pytest.raises(ValueError):
        s.verify_sampled([e.vocabulary_size], [0.5], 1.0)
    with pytest.raises(ValueError):
        s.generate_speculative_sampled([1], np.random.default_rng(0), 0.0)
    with pytest.raises(ValueError):
        e.create_session(40, "q3")
    assert s.current_position == 20
    s.close()
