"""The 4-bit KV cache, attention over it and draft verification on the GPU,
against plain 64-bit forms (q4_reference.py).

Tolerances.  The cache is compared bit for bit: its definition fixes every
rounding.  Attention is fp32: a score is a sum of products whose operands are
held to 22 bits or more, so it is off by at most 2^-21 of the sum of |q k|
scale (2^-22 for the operands, as much for the sum), an exponential by that
and 2^-20, and the output is a mean of values weighted by them: off by at most
twice that share of the largest value."""
import numpy as np
import pytest

import q4_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from overfit_b200 import build, kernels
    build.build()
    return kernels


def dev(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda() if dtype is None else torch.tensor(a, dtype=dtype, device="cuda")


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


def device_error():
    import ctypes as C
    from overfit_b200 import _lib
    code = C.c_int32()
    torch.cuda.synchronize()
    _lib.check(_lib.load().ovf_device_error(torch.cuda.current_device(), C.byref(code)))
    return code.value


def tables(ctx, hd, theta=10000.0):
    a = np.arange(ctx)[:, None] / theta ** (np.arange(0, hd, 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


class Batch:
    """Sequences of random rows in a 4-bit cache that held other bytes before, and the values that they have there."""

    def __init__(self, K, n, heads, kv_heads, hd, ctx, lengths, seed, split_half=False, rope=True, fill=None):
        self.K, self.heads, self.kv_heads, self.hd, self.ctx = K, heads, kv_heads, hd, ctx
        self.lengths, self.split_half, self.scale = lengths, split_half, 1 / np.sqrt(hd)
        rng = self.rng = np.random.default_rng(seed)
        self.cos, self.sin = tables(ctx, hd)
        self.dcos, self.dsin = (dev(self.cos), dev(self.sin)) if rope else (None, None)
        self.rope = rope
        size = n * K.KvCacheQ4.bytes(kv_heads, hd, ctx)
        before = np.full(size, fill, np.uint8) if fill is not None else rng.integers(0, 256, size, dtype=np.uint8)
        self.kc, self.vc = dev(before), dev(before[::-1].copy())
        most = max(lengths)
        self.k = rng.normal(0, 1, (n, most, kv_heads, hd)).astype(np.float32)
        self.k[..., ::17] *= 6
        self.v = rng.normal(0, 1, (n, most, kv_heads, hd)).astype(np.float32)
        if most:
            K.KvCacheQ4.append(dev(self.k.reshape(n, most, -1)), dev(self.v.reshape(n, most, -1)), self.kc, self.vc,
                               dev([0 if length else -1 for length in lengths], torch.int32), kv_heads, hd, ctx, self.dcos,
                               self.dsin, split_half, row_counts=dev(lengths, torch.int32))
        turn = [ref.rotate(self.k[s], self.cos[:most], self.sin[:most], split_half) if rope else self.k[s] for s in range(n)]
        self.kv = [(ref.stored(turn[s]), ref.stored(self.v[s])) for s in range(n)]

    def query(self, rows):
        return self.rng.normal(0, 1, (len(self.lengths), rows, self.heads, self.hd)).astype(np.float32)

    def run(self, q, positions, counts=None, out=None, sequences=slice(None), scratch=None):
        """The kernel's output for q [n, rows, heads, hd]."""
        n, rows = q.shape[:2]
        one = self.K.KvCacheQ4.bytes(self.kv_heads, self.hd, self.ctx)
        kc, vc = (c.view(-1, one)[sequences].contiguous().view(-1) for c in (self.kc, self.vc))
        out = torch.full((n, rows, self.heads * self.hd), 7.0, device="cuda") if out is None else out
        A = self.K.CachedAttentionKernel
        if scratch is None:
            scratch = torch.full((A.q4_scratch_bytes(n, rows, self.heads, self.kv_heads, self.hd, self.ctx),), 0xFF,
                                 dtype=torch.uint8, device="cuda")
            scratch[:256] = 0
        A.compute_q4(dev(q.reshape(n, rows, -1)), kc, vc, out, dev(positions, torch.int32), self.heads, self.kv_heads, self.hd,
                     self.ctx, self.scale, scratch, self.dcos, self.dsin, self.split_half,
                     row_counts=None if counts is None else dev(counts, torch.int32))
        assert not scratch[:256].any()
        return host(out).reshape(q.shape)

    def check(self, got, q, positions, counts=None):
        for s, pos in enumerate(positions):
            c = q.shape[1] if counts is None else counts[s]
            if pos < 0 or c == 0:
                assert (got[s] == 7.0).all()
                continue
            at = np.arange(pos, pos + c)
            turned = ref.rotate(q[s, :c], self.cos[at], self.sin[at], self.split_half) if self.rope else q[s, :c]
            k, v = self.kv[s]
            want, most = ref.attend(turned, k, v, pos, self.scale)
            tol = 2 * (most * 2.0 ** -21 + 2.0 ** -20) * np.abs(v[:pos + c]).max()
            np.testing.assert_allclose(got[s, :c], want, rtol=0, atol=tol)
            assert (got[s, c:] == 7.0).all()


# ------------------------------------------------------------------ the cache
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("pos,rows", [(0, 1), (5, 1), (31, 2), (3, 9), (0, 40), (26, 33)])
@pytest.mark.parametrize("split_half,rope", [(False, True), (True, True), (False, False)])
def test_append_bytes(K, hd, pos, rows, split_half, rope):
    """The bytes that an append writes, and that it leaves every other byte as it was."""
    rng = np.random.default_rng(hd + pos + rows)
    kvh, ctx = 2, 70
    one = K.KvCacheQ4.bytes(kvh, hd, ctx)
    assert one == kvh * 3 * 20 * hd
    before = rng.integers(0, 256, (2, one), dtype=np.uint8)
    k, v = rng.normal(0, 2, (2, 1, rows, kvh, hd)).astype(np.float32)
    cos, sin = tables(ctx, hd)
    kc, vc = dev(before[0]), dev(before[1])
    K.KvCacheQ4.append(dev(k.reshape(1, rows, -1)), dev(v.reshape(1, rows, -1)), kc, vc, dev([pos], torch.int32), kvh, hd, ctx,
                       dev(cos) if rope else None, dev(sin) if rope else None, split_half)
    want = before.copy().reshape(2, kvh, 3, 20 * hd)
    turned = ref.rotate(k[0], cos[pos:pos + rows], sin[pos:pos + rows], split_half) if rope else k[0]
    for side, x in ((0, turned), (1, v[0])):
        c, D, M = ref.quantise(x)
        for r in range(rows):
            for h in range(kvh):
                ref.put(want[side], side == 0, h, pos + r, c[r, h], D[r, h], M[r, h])
    np.testing.assert_array_equal(host(kc), want[0].reshape(-1))
    np.testing.assert_array_equal(host(vc), want[1].reshape(-1))


@pytest.mark.parametrize("hd", [32, 128])
def test_read_gives_the_values(K, hd):
    b = Batch(K, 3, 2, 2, hd, 100, [100, 37, 1], seed=hd)
    k, v = (torch.full((3, 50, 2 * hd), 7.0, device="cuda") for _ in "kv")
    K.KvCacheQ4.read(b.kc, b.vc, dev([50, 7, -1], torch.int32), 2, hd, 100, k, v, row_counts=dev([50, 30, 1], torch.int32))
    for got, side in ((host(k), 0), (host(v), 1)):
        got = got.reshape(3, 50, 2, hd)
        np.testing.assert_array_equal(got[0], b.kv[0][side][50:100])
        np.testing.assert_array_equal(got[1, :30], b.kv[1][side][7:37])
        assert (got[1, 30:] == 7.0).all() and (got[2] == 7.0).all()


def test_cache_of_special_values(K):
    """Groups of equal elements, zeros, NaN, infinities, numbers beyond fp16 and below it."""
    hd = 128
    x = np.random.default_rng(1).normal(0, 1, (1, 6, 1, hd)).astype(np.float32)
    x[0, 0] = 0.0
    x[0, 1, 0, :32] = 3.25
    x[0, 1, 0, 32:64] = -1e-9
    x[0, 2, 0, 5] = np.nan
    x[0, 2, 0, 40:42] = np.inf, -np.inf
    x[0, 3, 0, :32] = np.nan
    x[0, 3, 0, 64:68] = 3e38, -3e38, 1e5, 7
    x[0, 4] *= 1e-7
    x[0, 5, 0, 96:] = 60000.0
    kc, vc = (torch.zeros(K.KvCacheQ4.bytes(1, hd, 32), dtype=torch.uint8, device="cuda") for _ in "kv")
    K.KvCacheQ4.append(dev(x.reshape(1, 6, hd)), dev(x.reshape(1, 6, hd)), kc, vc, dev([0], torch.int32), 1, hd, 32)
    k, v = torch.empty(1, 6, hd, device="cuda"), torch.empty(1, 6, hd, device="cuda")
    K.KvCacheQ4.read(kc, vc, dev([0], torch.int32), 1, hd, 32, k, v)
    want = ref.stored(x[0]).reshape(6, hd)
    assert np.isfinite(want).all()
    np.testing.assert_array_equal(host(k)[0], want)
    np.testing.assert_array_equal(host(v)[0], want)
    # an element is off by half a step of its group, and the rounding of D, M and the value (fp16, half a step each)
    y = np.clip(np.nan_to_num(x[0].reshape(6, 4, 32), nan=0.0, posinf=16384, neginf=-16384), -16384, 16384).astype(np.float64)
    span = (y.max(-1) - y.min(-1))[..., None]
    tol = span / 30 + 2.0 ** -11 * (2 * np.abs(y).max(-1)[..., None] + 4 * span) + 3 * 2.0 ** -25
    assert (np.abs(want.reshape(6, 4, 32) - y) <= tol).all()


def test_rows_that_do_not_fit_are_left_out(K):
    """A position or a count in device memory that does not fit sets error 4 and writes nothing; other sequences go on."""
    hd, ctx = 64, 40
    one = K.KvCacheQ4.bytes(1, hd, ctx)
    kc, vc = (torch.zeros(3 * one, dtype=torch.uint8, device="cuda") for _ in "kv")
    x = torch.randn(3, 4, hd, device="cuda")
    assert device_error() == 0
    K.KvCacheQ4.append(x, x, kc, vc, dev([37, 36, 2 ** 31 - 1], torch.int32), 1, hd, ctx)
    assert device_error() == 4 and device_error() == 0
    for c in (kc, vc):
        a = host(c).reshape(3, one)
        assert not a[0].any() and a[1].any() and not a[2].any()
    out = torch.full((3, 4, hd), 7.0, device="cuda")
    A = K.CachedAttentionKernel
    scratch = torch.zeros(A.q4_scratch_bytes(3, 4, 1, 1, hd, ctx), dtype=torch.uint8, device="cuda")
    A.compute_q4(x, kc, vc, out, dev([37, 36, 41], torch.int32), 1, 1, hd, ctx, 0.1, scratch)
    assert device_error() == 4
    o = host(out)
    assert (o[0] == 7).all() and (o[1] != 7).all() and (o[2] == 7).all()


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (7, 1, 64), (4, 4, 32), (16, 1, 128), (4, 2, 256), (24, 2, 64)])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 64, 65, 255, 256, 257, 700])
def test_decode(K, heads, kv_heads, hd, length):
    b = Batch(K, 1, heads, kv_heads, hd, 704, [length], seed=length + hd, split_half=length % 2 == 0)
    q = b.query(1)
    b.check(b.run(q, [length - 1]), q, [length - 1])


@pytest.mark.parametrize("rows", [2, 3, 8, 9, 17, 64, 65, 130, 256])
@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (7, 1, 64), (6, 2, 32), (2, 1, 256)])
def test_rows(K, rows, heads, kv_heads, hd):
    """Several rows a sequence (verify, prefill), unequal sequences, an unused place, one without rows."""
    lengths = [rows, rows + 300, rows + 77, 0, rows]
    b = Batch(K, 5, heads, kv_heads, hd, rows + 310, lengths, seed=rows + hd, split_half=True)
    positions, counts = [0, 300, 77, -1, 0], [rows, rows, max(1, rows // 2), rows, 0]
    q = b.query(rows)
    b.check(b.run(q, positions, counts), q, positions, counts)


def test_no_rotation(K):
    b = Batch(K, 2, 4, 2, 64, 128, [100, 128], seed=3, rope=False)
    q = b.query(2)
    b.check(b.run(q, [98, 126]), q, [98, 126])


def test_long_sequence(K):
    b = Batch(K, 1, 4, 1, 128, 20000, [20000], seed=5)
    q = b.query(3)
    b.check(b.run(q, [19997]), q, [19997])


@pytest.mark.parametrize("heads,kv_heads,hd", [(6, 2, 64), (2, 1, 256)])
def test_long_sequences_of_several_rows(K, heads, kv_heads, hd):
    """More chunks than one group of lanes joins, for every (sequence, row, head)."""
    b = Batch(K, 3, heads, kv_heads, hd, 13000, [12990, 77, 12999], seed=31)
    q = b.query(3)
    at, counts = [12987, 74, 12998], [3, 2, 1]
    b.check(b.run(q, at, counts), q, at, counts)


@pytest.mark.parametrize("hd", [32, 128])
def test_long_sums_of_many_rows(K, hd):
    """Sums over 16384 positions by one CTA.  Values of 1 to 2, so that errors of one sign add up: the tensor cores cut an
    accumulator by less than 2^-23 of itself at each of at most 64 additions, the sums of these follow fp32 rounding; a
    score's error is bounded as in Batch.check."""
    heads, rows, ctx = 8, 1200, 16384
    g = torch.Generator(device="cuda").manual_seed(5)
    k = torch.randn(1, ctx, hd, generator=g, device="cuda")
    v = 1 + torch.rand(1, ctx, hd, generator=g, device="cuda")
    q = torch.randn(1, rows, heads * hd, generator=g, device="cuda") * 0.1
    kc, vc = (torch.zeros(K.KvCacheQ4.bytes(1, hd, ctx), dtype=torch.uint8, device="cuda") for _ in "kv")
    zero = dev([0], torch.int32)
    K.KvCacheQ4.append(k, v, kc, vc, zero, 1, hd, ctx)
    K.KvCacheQ4.read(kc, vc, zero, 1, hd, ctx, k, v)
    A = K.CachedAttentionKernel
    scratch = torch.zeros(A.q4_scratch_bytes(1, rows, heads, 1, hd, ctx), dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    A.compute_q4(q, kc, vc, out, dev([ctx - rows], torch.int32), heads, 1, hd, ctx, hd ** -0.5, scratch)
    k, v = k[0].double(), v[0].double()
    most, off = 0.0, torch.arange(ctx, device="cuda")
    for r in range(0, rows, 100):
        x = q[0, r:r + 100].view(-1, heads, hd).double() * hd ** -0.5
        most = max(most, (x.abs() @ k.abs().T).max().item())
        hidden = off[None] > ctx - rows + r + torch.arange(x.shape[0], device="cuda")[:, None]
        want = (x @ k.T).masked_fill(hidden[:, None], -torch.inf).softmax(-1) @ v
        tol = 2 * (64 * 2.0 ** -23 + 2 * (most * 2.0 ** -21 + 2.0 ** -20))
        torch.testing.assert_close(out[0, r:r + 100].view_as(want).double(), want, rtol=0, atol=tol)


@pytest.mark.parametrize("rows", [1, 5, 100])
def test_bytes_behind_a_sequence_do_not_matter(K, rows):
    """Stale bytes behind the last position (all ones: codes 15, D and M NaN) change no bit."""
    got = []
    for fill in (0, 0xFF):
        b = Batch(K, 1, 8, 2, 128, 420, [301], seed=9, fill=fill)
        got.append(b.run(b.query(rows), [301 - rows]))
    assert np.isfinite(got[0]).all()
    np.testing.assert_array_equal(got[0], got[1])


@pytest.mark.parametrize("rows", [4, 100])
def test_a_bad_query_stays_in_its_row(K, rows):
    b = Batch(K, 1, 8, 2, 64, 420, [400], seed=11)
    q = b.query(rows)
    clean = b.run(q, [400 - rows])
    bad = q.copy()
    bad[0, 1, 3, 5] = np.nan
    bad[0, 2, 0, 0] = np.inf
    got = b.run(bad, [400 - rows])
    assert np.isnan(got[0, 1, 3]).all() and np.isnan(got[0, 2, 0]).any()
    keep = np.ones(q.shape[1:3], bool)
    keep[1, 3] = keep[2, 0] = False
    np.testing.assert_array_equal(got[0][keep], clean[0][keep])


@pytest.mark.parametrize("factor", [0.0, 1e-30, 1e-6, 1e4])
def test_queries_of_any_size(K, factor):
    """Scores of no, little and great spread; a large query makes the softmax a choice of one position."""
    b = Batch(K, 1, 4, 2, 64, 300, [300], seed=13)
    q = (b.query(1) * np.float32(factor)).astype(np.float32)
    got = b.run(q, [299])
    if factor < 1:
        b.check(got, q, [299])
    else:
        assert np.isfinite(got).all()
        # every output is a value of the position with the largest score (the others weigh less than 2^-24)
        turned = ref.rotate(q[0], b.cos[[299]], b.sin[[299]], False)
        want, _ = ref.attend(turned, *b.kv[0], 299, b.scale)
        np.testing.assert_allclose(got[0], want, rtol=0, atol=2.0 ** -10 * np.abs(b.kv[0][1]).max())


@pytest.mark.parametrize("rows", [3, 80])
@pytest.mark.parametrize("heads,kv_heads,hd", [(4, 2, 128), (2, 2, 64), (3, 1, 32), (1, 1, 256)])
def test_maxima_that_keep_rising(K, rows, heads, kv_heads, hd):
    """Keys that grow along the sequence, so that every tile passes the maximum of the last by far, and then shrink."""
    b = Batch(K, 1, heads, kv_heads, hd, 1200, [1], seed=rows + hd)
    n = 1100
    b.k = b.rng.normal(0, 1, (1, n, kv_heads, hd)).astype(np.float32)
    b.k *= (0.05 + 3.0 * np.minimum(np.arange(n), 900) / 900).astype(np.float32)[None, :, None, None]
    b.k[:, 1000:] *= 0.1
    b.v = b.rng.normal(0, 1, (1, n, kv_heads, hd)).astype(np.float32)
    K.KvCacheQ4.append(dev(b.k.reshape(1, n, -1)), dev(b.v.reshape(1, n, -1)), b.kc, b.vc, dev([0], torch.int32), kv_heads, hd,
                       1200, b.dcos, b.dsin)
    b.kv = [(ref.stored(ref.rotate(b.k[0], b.cos[:n], b.sin[:n], False)), ref.stored(b.v[0]))]
    q = b.query(rows) * np.float32(6)
    for pos in (n - rows, 700 - rows, 129):
        b.check(b.run(q, [pos]), q, [pos])


@pytest.mark.parametrize("heads,kv_heads,hd", [(8, 2, 128), (7, 1, 64)])
def test_a_row_does_not_depend_on_its_company(K, heads, kv_heads, hd):
    """A decode step, the same row in a batch of sequences, and in a verify batch: the same bits."""
    n, rows, lengths = 5, 11, [700, 300, 11, 257, 1000]
    b = Batch(K, n, heads, kv_heads, hd, 1000, lengths, seed=17)
    q = b.query(rows)
    positions = [length - rows for length in lengths]
    whole = b.run(q, positions)
    for s in (0, 2, 4):
        for r in (0, 4, 10):
            alone = b.run(q[s:s + 1, r:r + 1], [positions[s] + r], sequences=slice(s, s + 1))
            np.testing.assert_array_equal(alone[0, 0], whole[s, r])
    batch = b.run(np.ascontiguousarray(q[:, 3:4]), [p + 3 for p in positions])
    np.testing.assert_array_equal(batch[:, 0], whole[:, 3])


@pytest.mark.parametrize("rows", [1, 6, 70])
def test_rows_appended_by_the_call(K, rows):
    """k_new / v_new: as an append and then the attention, in cache and output."""
    heads, kvh, hd, ctx = 8, 2, 128, 400
    b = Batch(K, 2, heads, kvh, hd, ctx, [250, 33], seed=19)
    one = K.KvCacheQ4.bytes(kvh, hd, ctx)
    k, v = (torch.randn(2, rows, kvh * hd, device="cuda") for _ in "kv")
    q = torch.randn(2, rows, heads * hd, device="cuda")
    pos, counts = dev([250, 33], torch.int32), dev([rows, (rows + 1) // 2], torch.int32)
    A = K.CachedAttentionKernel
    scratch = torch.zeros(A.q4_scratch_bytes(2, rows, heads, kvh, hd, ctx), dtype=torch.uint8, device="cuda")
    kc, vc, out = b.kc.clone(), b.vc.clone(), torch.zeros_like(q)
    K.KvCacheQ4.append(k, v, kc, vc, pos, kvh, hd, ctx, b.dcos, b.dsin, row_counts=counts)
    A.compute_q4(q, kc, vc, out, pos, heads, kvh, hd, ctx, 0.09, scratch, b.dcos, b.dsin, row_counts=counts)
    out2 = torch.zeros_like(q)
    A.compute_q4(q, b.kc, b.vc, out2, pos, heads, kvh, hd, ctx, 0.09, scratch, b.dcos, b.dsin, row_counts=counts, k_new=k,
                 v_new=v)
    np.testing.assert_array_equal(host(b.kc).reshape(2, one), host(kc).reshape(2, one))
    np.testing.assert_array_equal(host(b.vc), host(vc))
    np.testing.assert_array_equal(host(out2), host(out))


def test_offsets_beyond_32_bits(K):
    """A cache of more than 2^32 bytes a side: the last sequence and the last head are found."""
    hd, kvh, ctx, n = 256, 8, 1 << 18, 15
    one = K.KvCacheQ4.bytes(kvh, hd, ctx)
    assert n * one > 1 << 32
    kc, vc = (torch.zeros(n * one, dtype=torch.uint8, device="cuda") for _ in "kv")
    b = Batch(K, 1, kvh, kvh, hd, ctx, [40], seed=23, fill=0)
    kc[-one:], vc[-one:] = b.kc, b.vc
    q = b.query(1)
    out = torch.full((n, 1, kvh * hd), 7.0, device="cuda")
    qd = torch.zeros(n, 1, kvh * hd, device="cuda")
    qd[-1] = dev(q.reshape(1, -1))
    A = K.CachedAttentionKernel
    scratch = torch.zeros(A.q4_scratch_bytes(n, 1, kvh, kvh, hd, ctx), dtype=torch.uint8, device="cuda")
    A.compute_q4(qd, kc, vc, out, dev([-1] * (n - 1) + [39], torch.int32), kvh, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin)
    got = host(out).reshape(n, 1, kvh, hd)
    assert (got[:-1] == 7.0).all()
    b.check(got[-1:], q, [39])


def test_streams_and_graphs(K):
    """On a side stream, and captured once and replayed with new positions, queries and cache contents."""
    heads, kvh, hd, ctx = 8, 2, 128, 900
    b = Batch(K, 2, heads, kvh, hd, ctx, [899, 500], seed=29)
    A = K.CachedAttentionKernel
    q, out = torch.zeros(2, 1, heads * hd, device="cuda"), torch.zeros(2, 1, heads * hd, device="cuda")
    pos = dev([0, 0], torch.int32)
    scratch = torch.zeros(A.q4_scratch_bytes(2, 1, heads, kvh, hd, ctx), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        A.compute_q4(q, b.kc, b.vc, out, pos, heads, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin)
    for at in ([0, 5], [898, 499], [300, -1]):
        x = b.query(1)
        q.copy_(dev(x.reshape(2, 1, -1)))
        pos.copy_(dev(at, torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        b.check(host(out).reshape(2, 1, heads, hd), x, at)
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        out2 = torch.full_like(out, 7.0)
        A.compute_q4(q, b.kc, b.vc, out2, pos, heads, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin)
    side.synchronize()
    np.testing.assert_array_equal(host(out2), host(out))


def test_graphs_that_overlap(K):
    """Two captured steps (append and attention) with caches and scratch of their own, replayed on two streams at once,
    again and again."""
    heads, kvh, hd, ctx, rows = 8, 2, 64, 1200, 2
    A = K.CachedAttentionKernel
    steps = []
    for seed in (37, 41):
        b = Batch(K, 2, heads, kvh, hd, ctx, [1100, 600], seed=seed)
        q, k, v = (torch.randn(2, rows, h * hd, device="cuda") for h in (heads, kvh, kvh))
        pos = dev([1100, 600], torch.int32)
        scratch = torch.zeros(A.q4_scratch_bytes(2, rows, heads, kvh, hd, ctx), dtype=torch.uint8, device="cuda")
        kc, vc, want, out = b.kc.clone(), b.vc.clone(), torch.zeros_like(q), torch.zeros_like(q)
        A.compute_q4(q, kc, vc, want, pos, heads, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin, k_new=k, v_new=v)
        steps.append((b, q, k, v, pos, scratch, out, want, kc, vc, torch.cuda.Stream(), torch.cuda.CUDAGraph()))
    torch.cuda.synchronize()
    for b, q, k, v, pos, scratch, out, want, kc, vc, stream, graph in steps:
        with torch.cuda.graph(graph, stream=stream):
            A.compute_q4(q, b.kc, b.vc, out, pos, heads, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin, k_new=k, v_new=v)
    torch.cuda.synchronize()
    for _ in range(20):
        for step in steps:
            with torch.cuda.stream(step[-2]):
                step[-1].replay()
    torch.cuda.synchronize()
    for b, q, k, v, pos, scratch, out, want, kc, vc, stream, graph in steps:
        np.testing.assert_array_equal(host(out), host(want))
        np.testing.assert_array_equal(host(b.kc), host(kc))
        np.testing.assert_array_equal(host(b.vc), host(vc))
        assert not scratch[:256].any()


# ------------------------------------------------------------------ drafts
def drafted(rng, n, m, vocab, peak=2.5):
    logits = rng.normal(0, peak, (n, m + 1, vocab)).astype(np.float32)
    z = logits[:, :m] + rng.normal(0, 0.7, (n, m, vocab))
    q = np.exp(z - z.max(-1, keepdims=True))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    d = np.array([[rng.choice(vocab, p=q[s, j] / q[s, j].astype(np.float64).sum()) for j in range(m)] for s in range(n)],
                 dtype=np.int32).reshape(n, m)
    return logits, q, d, rng.random((n, m + 1), dtype=np.float32)


def run_verify(K, logits, drafts, u, T, probs=None, counts=None):
    n = logits.shape[0]
    a, t = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7, dtype=torch.int32, device="cuda")
    K.SpeculativeVerifier.verify(dev(logits), dev(drafts), dev(u), dev(np.asarray(T, np.float32)), a, t,
                                 None if probs is None else dev(probs), None if counts is None else dev(counts, torch.int32))
    return host(a), host(t)


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 1003, 32000, 128256, 151937])
@pytest.mark.parametrize("with_probs", [False, True])
def test_verify(K, vocab, with_probs):
    rng = np.random.default_rng(vocab)
    n, m = (40, 5) if vocab <= 1003 else (9, 3)
    logits, q, d, u = drafted(rng, n, m, vocab)
    T = rng.uniform(0.3, 1.6, n).astype(np.float32)
    T[-1] = 0
    counts = rng.integers(0, m + 1, n).astype(np.int32)
    counts[0] = m
    a, t = run_verify(K, logits, d, u, T, q if with_probs else None, counts)
    want = [ref.verify(logits[s], d[s], u[s], T[s], q[s] if with_probs else None, counts[s]) for s in range(n)]
    np.testing.assert_array_equal(np.stack([a, t], 1), want)


def test_verify_unusual_rows(K):
    """Tokens that are ruled out, rows without a distribution, drafts that are no tokens, equal distributions,
    temperatures near none and high, unused places."""
    rng = np.random.default_rng(3)
    n, m, vocab = 12, 3, 500
    logits, q, d, u = drafted(rng, n, m, vocab)
    T = np.ones(n, np.float32)
    counts = np.full(n, m, np.int32)
    logits[0, :, 7:] = -np.inf                      # most tokens ruled out
    logits[1, 0] = -np.inf                          # nothing left
    logits[2, 1, 40] = np.nan
    logits[2, 0, d[2, 0]] = 60                      # (its first draft is accepted)
    logits[3, 0, 5] = np.inf
    d[4, 0] = vocab
    d[5, 0] = -1
    counts[6] = -1                                  # unused
    T[7] = 1e-3
    T[8] = 50
    logits[9] = 3.0                                 # all alike
    T[10] = -1
    logits[10, 0, [4, 9]] = 50                      # two maxima: the first
    d[10, 0] = 9
    logits[11, :, 1:] = -np.inf                     # certain
    d[11] = 0
    for probs in (None, q):
        a, t = run_verify(K, logits, d, u, T, probs, counts)
        for s in range(n):
            if s == 6:
                assert (a[s], t[s]) == (-7, -7)
                continue
            want = ref.verify(logits[s], d[s], u[s], T[s], None if probs is None else probs[s], counts[s])
            assert (a[s], t[s]) == want, s
    assert run_verify(K, logits, d, u, T, None, counts)[1][1] == -1


@pytest.mark.parametrize("with_probs", [False, True])
def test_verify_of_extreme_temperatures(K, with_probs):
    """From temperatures at which neighbouring floats are worlds apart (the largest logits, which tie, share everything)
    to ones at which all tokens are alike; logits of several magnitudes and both signs, some impossible."""
    rng = np.random.default_rng(11)
    T = np.array([1e-38, 1e-20, 1e-10, 1e-9, 3e-9, 1e-8, 3e-8, 1e-7, 3e-7, 1e-6, 1e-5, 1e-3, 1e3, 1e10, 1e30], np.float32)
    n, m, vocab = 4 * T.size, 2, 700
    T = np.tile(T, 4)
    logits, q, d, u = drafted(rng, n, m, vocab)
    logits[:15] += 20
    logits[15:30] *= 300
    logits[30:45] -= 150
    for s in range(n):
        for j in range(m + 1):
            order = np.argsort(logits[s, j])
            top = logits[s, j, order[-1]]
            logits[s, j, order[-4:-1]] = top
            for i, k in enumerate(order[-8:-4]):  # the next floats below
                logits[s, j, k] = np.nextafter(logits[s, j, order[-4 - i]], np.float32(-np.inf))
            logits[s, j, order[:5]] = -np.inf
            logits[s, j, order[5:9]] = -np.finfo(np.float32).max
            if j < m and rng.random() < 0.7:
                d[s, j] = order[-1 - rng.integers(0, 3)]
    a, t = run_verify(K, logits, d, u, T, q if with_probs else None)
    want = [ref.verify(logits[s], d[s], u[s], T[s], q[s] if with_probs else None, m) for s in range(n)]
    np.testing.assert_array_equal(np.stack([a, t], 1), want)


def test_verify_at_its_borders(K):
    """u q against p where they are equal but for the last bits, and a cumulative sum that meets its target."""
    vocab, T = 4, 1.0
    logits = np.zeros((3, 2, vocab), np.float32)    # p = 1/4 each, exactly
    d = np.array([[2], [2], [2]], np.int32)
    u = np.array([[0.25, 0.5], [np.nextafter(np.float32(0.25), np.float32(0)), 0.5], [0.25, 0.0]], np.float32)
    a, t = run_verify(K, logits, d, u, [T] * 3)
    assert a.tolist() == [0, 1, 0]                  # u = p rejects, the float below accepts
    assert t.tolist() == [1, 2, 0]                  # rest (1,1,0,1)/4, target half: 2/4 > 3/8; row of 4: 3/4 > 1/2; first
    # the residual of a draft distribution that is above the target everywhere but at one token
    q = np.array([[[0.3, 0.3, 0.3, 0.1]]], np.float32)
    a, t = run_verify(K, logits[:1], np.array([[0]], np.int32), np.array([[0.99, 0.999]], np.float32), [T], q)
    assert (a[0], t[0]) == (0, 3)


def test_sampling_without_drafts(K):
    rng = np.random.default_rng(5)
    logits = rng.normal(0, 3, (64, 1, 777)).astype(np.float32)
    u = rng.random((64, 1), dtype=np.float32)
    a, t = run_verify(K, logits, np.zeros((64, 0), np.int32), u, [0.9] * 64)
    want = [ref.verify(logits[s], [], u[s], np.float32(0.9), None, 0) for s in range(64)]
    np.testing.assert_array_equal(np.stack([a, t], 1), want)


def test_verified_tokens_are_the_targets(K):
    """Over many draws the first token behind a prompt is distributed as the target says, whatever was drafted:
    each of 6 tokens within 5 standard deviations of its share."""
    n, vocab = 60000, 6
    rng = np.random.default_rng(7)
    p = np.array([.4, .25, .2, .1, .04, .01])
    q = np.array([.1, .3, .1, .3, .1, .1], np.float32)
    logits = np.broadcast_to(np.log(p).astype(np.float32), (n, 2, vocab))
    d = rng.choice(vocab, (n, 1), p=q / q.astype(np.float64).sum()).astype(np.int32)
    a, t = run_verify(K, logits, d, rng.random((n, 2), dtype=np.float32), [1.0] * n, np.broadcast_to(q, (n, 1, vocab)))
    first = np.where(a > 0, d[:, 0], t)
    share = np.bincount(first, minlength=vocab) / n
    assert (np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / n)).all()


# ------------------------------------------------------------------ together
def test_a_speculative_step(K):
    """Drafts of three sessions: their rows appended and attended, the attention's outputs projected to logits,
    the drafts verified, and the cache continued behind the accepted ones, as a run of single steps does it."""
    rng = np.random.default_rng(31)
    n, heads, kvh, hd, ctx, vocab, m = 3, 8, 2, 64, 300, 97, 4
    lengths = [200, 31, 64]
    b = Batch(K, n, heads, kvh, hd, ctx, lengths, seed=31)
    head = rng.normal(0, 1.0, (heads * hd, vocab)).astype(np.float32)
    rows = m + 1
    q, k, v = (rng.normal(0, 1, (n, rows, c * hd)).astype(np.float32) for c in (heads, kvh, kvh))
    counts = np.array([rows, rows - 2, rows], np.int32)
    A = K.CachedAttentionKernel
    scratch = torch.zeros(A.q4_scratch_bytes(n, rows, heads, kvh, hd, ctx), dtype=torch.uint8, device="cuda")
    out = torch.zeros(n, rows, heads * hd, device="cuda")
    A.compute_q4(dev(q), b.kc, b.vc, out, dev(lengths, torch.int32), heads, kvh, hd, ctx, b.scale, scratch, b.dcos, b.dsin,
                 row_counts=dev(counts), k_new=dev(k), v_new=dev(v))
    logits = (out.double() @ dev(head).double()).float().contiguous()
    drafts = rng.integers(0, vocab, (n, m)).astype(np.int32)
    greedy = host(logits).argmax(-1)
    drafts[:, :2] = greedy[:, :2]
    u = rng.random((n, rows), dtype=np.float32)
    a, t = run_verify(K, host(logits), drafts, u, [0.0, 0.5, 0.0], None, counts - 1)
    want_logits = np.zeros((n, rows, vocab), np.float32)
    for s in range(n):
        c = counts[s]
        at = np.arange(lengths[s], lengths[s] + c)
        kk = ref.stored(ref.rotate(k[s, :c].reshape(c, kvh, hd), b.cos[at], b.sin[at], False))
        vv = ref.stored(v[s, :c].reshape(c, kvh, hd))
        keys, values = (np.concatenate([old[:lengths[s]], new]) for old, new in zip(b.kv[s], (kk, vv)))
        o, _ = ref.attend(ref.rotate(q[s, :c].reshape(c, heads, hd), b.cos[at], b.sin[at], False), keys, values, lengths[s],
                          b.scale)
        want_logits[s, :c] = o.reshape(c, -1) @ head
        np.testing.assert_allclose(host(logits)[s, :c], want_logits[s, :c], rtol=0, atol=2e-3)
    want = [ref.verify(host(logits)[s], drafts[s], u[s], [0.0, 0.5, 0.0][s], None, counts[s] - 1) for s in range(n)]
    np.testing.assert_array_equal(np.stack([a, t], 1), want)
    assert a[0] >= 2 and a[2] >= 2
