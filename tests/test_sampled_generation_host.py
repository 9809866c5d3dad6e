"""The host side of sampled verification and speculative generation, and the draw of
its first token: the library's calls are faked."""
import numpy as np
import pytest

import q4_reference as ref


@pytest.fixture
def engine():
    from overfit_b200 import build, engine
    build.build()
    return engine


class Fake:
    """A library whose sampled verify gives `status`, and whose other session calls succeed."""

    def __init__(self, status=0):
        self.status, self.position, self.rows = status, 20, []

    def ovf_session_position(self, h):
        return self.position

    def ovf_session_verify_sampled(self, h, tokens, n, probs, u, T, accepted, token):
        self.rows.append(n)
        self.position += 1
        return self.status

    def ovf_session_decode(self, h, token, logits, argmax):
        self.position += 1
        return 0

    def ovf_last_error(self):
        return b"no distribution"


def session(engine, monkeypatch, fake, logits):
    monkeypatch.setattr(engine._lib, "load", lambda: fake)
    s = engine.CudaLlamaSession.__new__(engine.CudaLlamaSession)
    s.engine = type("E", (), {"cfg": {"vocab": len(logits)}})()
    s._h, s._logits, s._have_logits, s.max_context_length = 0, np.asarray(logits, np.float32), True, 1000
    return s


def test_a_failed_verify_leaves_no_logits(engine, monkeypatch):
    """The rows behind which there is no distribution are in the cache: the logits of the step before are not the session's."""
    from overfit_b200 import _lib
    s = session(engine, monkeypatch, Fake(_lib.OVF_ESTATE), np.zeros(10))
    with pytest.raises(engine.OverfitRuntimeError):
        s.verify_sampled([1, 2], [0.5, 0.5], 1.0)
    assert s.current_position == 21
    with pytest.raises(engine.OverfitRuntimeError):
        s.get_last_logits()


def test_a_refused_verify_keeps_the_logits(engine, monkeypatch):
    s = session(engine, monkeypatch, Fake(), np.arange(10))
    with pytest.raises(ValueError):
        s.verify_sampled([1, 2], [0.5], 1.0)
    assert s.get_last_logits()[3] == 3


def test_drafts_of_any_length(engine, monkeypatch):
    """A verify takes 64 rows: a longer draft is cut, not refused."""
    fake = Fake()
    s = session(engine, monkeypatch, fake, np.r_[50.0, np.zeros(9)])
    s.generate_speculative_sampled([0] + [1, 2, 3, 4, 5, 6, 7, 8, 9] * 20, np.random.default_rng(0), 1.0, max_draft=200)
    assert fake.rows == [64]


def draws():
    rng = np.random.default_rng(3)
    big = np.finfo(np.float32).max
    for T in (1e-45, 1e-38, 1e-10, 1e-3, 0.7, 5.0, 1e10, 1e30):
        for logits in (rng.normal(0, 3, 300), rng.normal(0, 300, 300), np.full(7, 2.5), rng.normal(-200, 1, 50)):
            x = logits.astype(np.float32)
            x[2::7] = -np.inf
            x[4::9] = -big
            yield x, T


def test_the_first_token_is_drawn_as_the_others_are(engine, monkeypatch):
    """From the logits that the session holds, for every positive temperature; impossible tokens never."""
    for x, T in draws():
        for u in (0.0, 0.3, 0.999, 1 - 2.0 ** -53):
            class Rng:
                def random(self, *a, **k):
                    return u
            s = session(engine, monkeypatch, Fake(), x)
            assert s.generate_speculative_sampled([], Rng(), T) == [ref.verify(x[None], [], [u], T, None, 0)[1]]
    s = session(engine, monkeypatch, Fake(), np.r_[-np.inf, 0.0, 1.0])
    assert s.generate_speculative_sampled([], np.random.default_rng(0), 1e38)[0] in (1, 2)  # as 1e30


@pytest.mark.parametrize("bad", [[0.0, np.nan, 1.0], [0.0, np.inf, 1.0], [-np.inf] * 3, [-np.finfo(np.float32).max] * 3])
def test_logits_without_a_distribution_draw_nothing(engine, monkeypatch, bad):
    fake = Fake()
    s = session(engine, monkeypatch, fake, bad)
    with pytest.raises(engine.OverfitRuntimeError):
        s.generate_speculative_sampled([1, 2], np.random.default_rng(0), 1.0)
    assert fake.position == 20 and not fake.rows
