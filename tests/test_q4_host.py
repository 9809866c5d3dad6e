"""Host checks of the 4-bit cache's and draft verification's entry points (no
device work), and of the format itself."""
import ctypes as C

import numpy as np
import pytest

import q4_reference as ref


@pytest.fixture(scope="module")
def lib():
    from overfit_b200 import _lib, build
    build.build()
    return _lib.load()


P = C.c_void_p(4096)
P2 = C.c_void_p(8192)


def test_sizes(lib):
    assert lib.ovf_kv_q4_bytes(8, 128, 2048) == 8 * 64 * 2560
    assert lib.ovf_kv_q4_bytes(2, 64, 33) == 2 * 2 * 1280
    assert lib.ovf_kv_q4_bytes(8, 128, 1 << 20) == 8 * 32768 * 2560
    for bad in ((0, 128, 64), (8, 96, 64), (8, 128, 0), (8, 128, (1 << 20) + 1), (-1, 64, 64)):
        assert lib.ovf_kv_q4_bytes(*bad) == 0
    assert lib.ovf_attention_q4_scratch_bytes(1, 1, 32, 8, 128, 4096) > 0
    for bad in ((0, 1, 32, 8, 128, 64), (1, 0, 32, 8, 128, 64), (1, 1, 32, 8, 100, 64)):
        assert lib.ovf_attention_q4_scratch_bytes(*bad) == 0


def test_cache_refusals(lib):
    from overfit_b200 import _lib

    def append(k=P, v=P, kc=P, vc=P2, pos=P, counts=None, n=1, rows=1, kvh=8, hd=128, ctx=64, cos=None, sin=None):
        return lib.ovf_kv_q4_append(k, v, kc, vc, pos, counts, n, rows, kvh, hd, ctx, cos, sin, 0, None)

    def read(k=P, v=P2, kc=P, vc=P2, pos=P, n=1, rows=1, kvh=8, hd=128, ctx=64):
        return lib.ovf_kv_q4_read(kc, vc, pos, None, n, rows, kvh, hd, ctx, k, v, None)

    for call in (append, read):
        for bad in (dict(k=None), dict(v=None), dict(kc=None), dict(vc=None), dict(pos=None), dict(n=-1), dict(n=70000),
                    dict(rows=-1), dict(rows=65), dict(kvh=0), dict(kvh=2000), dict(hd=96), dict(hd=0), dict(ctx=0),
                    dict(ctx=(1 << 20) + 1), dict(kc=C.c_void_p(4100)), dict(vc=C.c_void_p(8))):
            assert call(**bad) == _lib.OVF_EINVAL, bad
        assert call(n=0) == _lib.OVF_OK and call(rows=0) == _lib.OVF_OK
    assert append(cos=P) == _lib.OVF_EINVAL and append(sin=P) == _lib.OVF_EINVAL
    assert append(vc=P) == _lib.OVF_EINVAL
    assert read(v=P) == _lib.OVF_EINVAL


def test_attention_refusals(lib):
    from overfit_b200 import _lib

    def call(q=P, kn=None, vn=None, kc=P, vc=P2, out=P2, pos=P, n=1, rows=1, h=32, kvh=8, hd=128, ctx=64, cos=None, sin=None,
             scratch=P):
        return lib.ovf_attention_q4(q, kn, vn, kc, vc, out, pos, None, n, rows, h, kvh, hd, ctx, cos, sin, 0, 0.1, scratch, None)

    for bad in (dict(q=None), dict(out=None), dict(scratch=None), dict(kc=None), dict(pos=None), dict(h=0), dict(h=30),
                dict(h=-8), dict(kvh=0), dict(hd=80), dict(rows=65), dict(ctx=0), dict(out=P), dict(q=C.c_void_p(4)),
                dict(scratch=C.c_void_p(8)), dict(out=C.c_void_p(20)), dict(cos=P), dict(kn=P), dict(vn=P),
                dict(kn=P, vn=P, vc=P), dict(n=-1), dict(n=70000), dict(h=65536 * 8), dict(rows=1 << 18, ctx=1 << 18),
                dict(n=65535, rows=1 << 10, ctx=1 << 10), dict(n=2, rows=1 << 18, h=8, hd=256, ctx=1 << 20)):
        assert call(**bad) == _lib.OVF_EINVAL, bad
    assert call(n=0) == _lib.OVF_OK and call(rows=0) == _lib.OVF_OK
    assert b"" != lib.ovf_last_error()


def test_verify_refusals(lib):
    from overfit_b200 import _lib

    def call(logits=P, probs=None, drafts=P, u=P, t=P, n=1, m=3, vocab=100, a=P, tok=P2):
        return lib.ovf_verify_drafts(logits, probs, drafts, None, u, t, n, m, vocab, a, tok, None)

    for bad in (dict(logits=None), dict(u=None), dict(t=None), dict(a=None), dict(tok=None), dict(drafts=None), dict(n=-1),
                dict(m=-1), dict(m=5000), dict(vocab=0), dict(vocab=1 << 25), dict(tok=P), dict(m=0, probs=P)):
        assert call(**bad) == _lib.OVF_EINVAL, bad
    assert call(n=0) == _lib.OVF_OK


def test_python_mirror_refuses_before_any_launch():
    torch = pytest.importorskip("torch")
    from overfit_b200 import kernels as K
    x = torch.zeros(1, 2, 128)
    with pytest.raises(ValueError):  # host tensors
        K.KvCacheQ4.append(x, x, torch.zeros(10), torch.zeros(10), torch.zeros(1), 1, 128, 32)
    with pytest.raises(ValueError):
        K.KvCacheQ4.append(x, x, None, None, None, 1, 96, 32)
    with pytest.raises(ValueError):
        K.SpeculativeVerifier.verify(torch.zeros(2, 3), None, None, None, None, None)


def test_values_are_near_what_they_stand_for():
    """A code's value is off by half a step of 1/15 of the group's span, and three fp16 roundings (half a step of
    2^-10 each): of D (times 1 + c/16 < 2, so 2.2 spans), of M (at most |min| + 1.1 spans) and of the value."""
    rng = np.random.default_rng(0)
    for scale in (1e-3, 1.0, 300.0):
        x = rng.normal(0, scale, (50, 128)).astype(np.float32)
        y = ref.stored(x)
        g = x.reshape(50, 4, 32).astype(np.float64)
        span = (g.max(-1) - g.min(-1))[..., None]
        tol = span / 30 + 2.0 ** -11 * (2 * np.abs(g).max(-1)[..., None] + 4 * span) + 3 * 2.0 ** -25
        assert (np.abs(y.reshape(50, 4, 32) - g) <= tol).all()


def test_layout_places_every_element_once():
    """Written one vector at a time, all 32 positions of a tile fill its bytes, and no two share a code."""
    for hd in (32, 64, 128, 256):
        for keys in (True, False):
            cache = np.zeros((1, 1, 20 * hd), np.uint8)
            for p in range(32):
                ref.put(cache, keys, 0, p, np.full(hd, 15), np.full(hd // 32, 1.0), np.full(hd // 32, 2.0))
            assert (cache[0, 0, :16 * hd] == 255).all()
            assert (cache[0, 0, 16 * hd:].view(np.float16) > 0).all()
            ref.put(cache, keys, 0, 13, np.zeros(hd, int), np.ones(hd // 32), np.ones(hd // 32))
            assert np.unpackbits(cache[0, 0, :16 * hd]).sum() == 8 * 16 * hd - 4 * hd
