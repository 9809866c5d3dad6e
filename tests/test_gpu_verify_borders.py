"""The draw behind a rejected certain draft where next to nothing is left beside the
draft, and uniforms of zero and next to it."""
import numpy as np
import pytest

import q4_reference as ref
from test_gpu_q4 import K, run_verify  # noqa: F401  (K is the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n", [1, 9, 40, 300])
@pytest.mark.parametrize("vocab", [130, 300, 1003, 5000])
def test_the_least_weights_beside_a_draft(K, n, vocab):
    """Half of a row's weight is the draft's, half lies far behind it, and all other tokens weigh e^-40 or so: a uniform of
    zero draws the first of these, one of e^-41 times their number some other, and larger ones the far token."""
    rng = np.random.default_rng(vocab + n)
    logits = rng.normal(-40, 1, (n, 2, vocab)).astype(np.float32)
    drafts = rng.integers(0, 100, (n, 1)).astype(np.int32)
    logits[np.arange(n), 0, drafts[:, 0]] = 0
    logits[:, 0, vocab - 1] = 0
    u = np.full((n, 2), 0.9, np.float32)
    u[:, 1] = [(0.0, 1e-38, np.exp(-43.0) * vocab / 3, 1e-15, 1e-11, 1e-9, 1e-8, 0.5)[s % 8] for s in range(n)]
    a, t = run_verify(K, logits, drafts, u, [1.0] * n)
    want = [ref.verify(logits[s], drafts[s], u[s], np.float32(1), None, 1) for s in range(n)]
    np.testing.assert_array_equal(np.stack([a, t], 1), want)
    assert (a == 0).all() and t[0] in (0, 1)
