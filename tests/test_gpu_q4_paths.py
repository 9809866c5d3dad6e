"""The kernels that one call of ovf_attention_q4 may take, each shown to be the
one that runs, on inputs at which it could go wrong.

Which kernel ran is read from the scratch: a call with a row that attends its
whole cache leaves that row's last partial result at the end of what the kernel
used.  attention_q4_kernel uses a place for every 256 positions (512 in long
caches, of which the first of two), attention_q4_rows_kernel one for each of its
splits, or none.

Tolerances are those of test_gpu_q4.py: a score is off by at most 2^-21 of the sum of
|q k| scale, an exponential by that and 2^-20, the output by twice that share of the
largest value.  attention_q4_rows_kernel sums a score in head_dim / 16 additions (and
as many of lo parts, 2^-11 as large) that the tensor cores each cut by less than
2^-23 of the sum of |q k|: `added` of that, in place of half of the 2^-21.  Its O is cut
by less than 2^-23 at each of the 16 additions of a tile and, in a window of two
tiles, of the one before it: 32 of that, in a mean of values times weights."""
import numpy as np
import pytest

from test_gpu_q4 import K, dev  # noqa: F401  (K is the fixture)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def used_scratch(scratch):
    """Bytes of it up to the last that a call has written (it was all ones behind the first 256)."""
    written = torch.nonzero(scratch[256:] != 0xFF)
    return 256 + (int(written[-1]) + 1 if written.numel() else 0)


def splits_of(scratch, n, rows, heads, hd, ctx):
    """Partial results of a row that attention_q4_rows_kernel left: 1 (none), or how many."""
    used, place = used_scratch(scratch) - 256, 4 * n * rows * heads * (hd + 2)
    assert used % place == 0 and used // place < -(-ctx // 256), "not the many-rows kernel's scratch"
    return max(1, used // place)


class Long:
    """Sequences of given keys and values [n, ctx, kv heads, hd] in a 4-bit cache, on the device."""

    def __init__(self, K, k, v, heads, fill=0, ctx=None):
        self.K, self.heads = K, heads
        n, length, self.kvh, self.hd = k.shape
        self.n, self.ctx = n, ctx or length
        size = n * K.KvCacheQ4.bytes(self.kvh, self.hd, self.ctx)
        self.kc, self.vc = (torch.full((size,), fill, dtype=torch.uint8, device="cuda") for _ in "kv")
        zero = dev([0] * n, torch.int32)
        k, v = k.reshape(n, length, -1).contiguous(), v.reshape(n, length, -1).contiguous()
        K.KvCacheQ4.append(k, v, self.kc, self.vc, zero, self.kvh, self.hd, self.ctx)
        ks, vs = torch.empty_like(k), torch.empty_like(v)
        K.KvCacheQ4.read(self.kc, self.vc, zero, self.kvh, self.hd, self.ctx, ks, vs)
        self.k, self.v = (x.view(n, length, self.kvh, self.hd).double() for x in (ks, vs))

    def run(self, q, positions, counts=None):
        """(output, the scratch) for q [n, rows, heads, hd]."""
        n, rows = q.shape[:2]
        A = self.K.CachedAttentionKernel
        size = A.q4_scratch_bytes(n, rows, self.heads, self.kvh, self.hd, self.ctx)
        scratch = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        scratch[:256] = 0
        out = torch.full((n, rows, self.heads * self.hd), 7.0, device="cuda")
        A.compute_q4(q.reshape(n, rows, -1).contiguous(), self.kc, self.vc, out, dev(positions, torch.int32), self.heads,
                     self.kvh, self.hd, self.ctx, self.hd ** -0.5, scratch,
                     row_counts=None if counts is None else dev(counts, torch.int32))
        torch.cuda.synchronize()
        assert not scratch[:256].any()
        return out.view(n, rows, self.heads, self.hd), scratch

    def scores(self, q, s, pos, rows):
        """Scores [row, head, position] of some rows of sequence s, in 64 bits, and the sums of |q k| scale."""
        length = pos + rows[-1] + 1
        g = self.heads // self.kvh
        x = q[s, rows].double().view(len(rows), self.kvh, g, self.hd)
        k = self.k[s, :length]
        z = torch.einsum("rhgd,phd->rhgp", x, k) * self.hd ** -0.5
        most = (torch.einsum("rhgd,phd->rhgp", x.abs(), k.abs()).amax() * self.hd ** -0.5).item()
        at = pos + torch.tensor(rows, device="cuda")
        z = z.masked_fill(torch.arange(length, device="cuda") > at[:, None, None, None], -torch.inf)
        return z, most

    def check(self, got, q, positions, rows, counts=None):
        for s, pos in enumerate(positions):
            real = [r for r in rows if counts is None or r < counts[s]]
            if not real:
                continue
            z, most = self.scores(q, s, pos, real)
            v = self.v[s, :z.shape[-1]]
            want = torch.einsum("rhgp,phd->rhgd", z.softmax(-1), v).reshape(len(real), self.heads, self.hd)
            added = max(4, self.hd // 16)
            score = most * (2.0 ** -22 + added * 2.0 ** -23)
            tol = (2 * (score + 2.0 ** -20) + 32 * 2.0 ** -23) * v.abs().max().item()
            torch.testing.assert_close(got[s, real].double(), want, rtol=0, atol=tol)


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# --------------------------------------------- attention_q4_rows_kernel
# sequences, splits that they leave room for (148 SMs)
MANY = [(4, "several"), (8, "one")]


@pytest.mark.parametrize("n,kind", MANY)
@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (8, 2, 64), (8, 2, 32)])
def test_maxima_that_rise_within_a_window(K, n, kind, heads, kvh, hd):
    """Keys that grow along the sequence: every tile of 128 passes the maximum of the last by more than 2^8 for most
    rows, odd tiles (the second of a window) too; then they shrink.  Odd and even numbers of tiles, ends inside a tile."""
    length, rows = 1500, 200
    grow = 0.02 + 8.0 * (torch.arange(length, device="cuda") / 1200).clamp(max=1)
    grow[1300:] *= 0.1
    # (keys that all point the same way, so that a row's scores rise or fall together)
    way = normal(hd, 1, 1, kvh, hd)
    k = (way + 0.1 * normal(hd + 1, n, length, kvh, hd)) * grow[None, :, None, None]
    b = Long(K, k, normal(hd + 2, n, length, kvh, hd), heads)
    q = 3 * normal(hd + 3, n, rows, heads, hd) + 2.5 * way.view(1, 1, kvh, 1, hd).expand(n, rows, kvh, heads // kvh,
                                                                                       hd).reshape(n, rows, heads, hd)
    z, _ = b.scores(q, 0, 1100 - rows, [rows - 1])
    top = z[..., :1024].unflatten(-1, (8, 128)).amax(-1) / np.log(2)
    rise = top.diff(dim=-1)  # of tiles 1 .. 7
    assert (rise[..., ::2] > 8).double().mean() > 0.5 and (rise[..., 1::2] > 8).double().mean() > 0.5
    for end in (1500, 1409, 1280, 1100, 300):
        at = [end - rows - 3 * s for s in range(n)]
        got, scratch = b.run(q, at)
        assert (splits_of(scratch, n, rows, heads, hd, b.ctx) > 1) == (kind == "several")
        b.check(got, q, at, [0, 1, 77, 127, 128, rows - 1])


@pytest.mark.parametrize("n,kind", MANY)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_bytes_behind_many_rows_do_not_matter(K, n, kind, hd):
    """Stale bytes behind the last position (all ones: codes 15, D and M NaN) change no bit."""
    length, rows, heads, kvh = 1203, 200, 8, 2
    k, v, q = normal(1, n, length, kvh, hd), normal(2, n, length, kvh, hd), normal(3, n, rows, heads, hd)
    at = [length - rows] * n
    got = []
    for fill in (0, 0xFF):
        b = Long(K, k, v, heads, fill, ctx=1500)
        out, scratch = b.run(q, at)
        assert (splits_of(scratch, n, rows, heads, hd, b.ctx) > 1) == (kind == "several")
        got.append(out)
    assert torch.isfinite(got[0]).all() and torch.equal(got[0], got[1])
    b.check(got[0], q, at, [0, 60, 199])


@pytest.mark.parametrize("n,kind", MANY)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_a_bad_query_among_many_rows(K, n, kind, hd):
    """NaN and infinities stay in the rows and heads that have them."""
    length, rows, heads, kvh = 1300, 200, 8, 2
    b = Long(K, normal(1, n, length, kvh, hd), normal(2, n, length, kvh, hd), heads)
    q = normal(3, n, rows, heads, hd)
    at = [length - rows] * n
    clean, scratch = b.run(q, at)
    assert (splits_of(scratch, n, rows, heads, hd, b.ctx) > 1) == (kind == "several")
    bad = q.clone()
    bad[0, 3, 1, 5], bad[1, 120, 7, 0], bad[2, 199, 0, 31] = torch.nan, torch.inf, -torch.inf
    got, _ = b.run(bad, at)
    hit = torch.zeros(n, rows, heads, dtype=torch.bool, device="cuda")
    hit[0, 3, 1] = hit[1, 120, 7] = hit[2, 199, 0] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize("n,kind", MANY)
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_many_rows_appended_by_the_call(K, n, kind, hd):
    """k_new / v_new: as an append and then the attention, in caches and output; ragged."""
    heads, kvh, rows, ctx = 8, 2, 200, 1500
    b = Long(K, normal(1, n, 1203, kvh, hd), normal(2, n, 1203, kvh, hd), heads, 0xFF, ctx=ctx)
    k, v, q = (normal(3 + i, n, rows, h * hd) for i, h in enumerate((kvh, kvh, heads)))
    pos = dev([1203 - 5 * s for s in range(n)], torch.int32)
    counts = dev([rows - 17 * s for s in range(n)], torch.int32)
    A = K.CachedAttentionKernel
    got = []
    for new in (False, True):
        kc, vc, out = b.kc.clone(), b.vc.clone(), torch.full((n, rows, heads * hd), 7.0, device="cuda")
        scratch = torch.full((A.q4_scratch_bytes(n, rows, heads, kvh, hd, ctx),), 0xFF, dtype=torch.uint8, device="cuda")
        scratch[:256] = 0
        if not new:
            K.KvCacheQ4.append(k, v, kc, vc, pos, kvh, hd, ctx, row_counts=counts)
        A.compute_q4(q, kc, vc, out, pos, heads, kvh, hd, ctx, 0.09, scratch, row_counts=counts,
                     k_new=k if new else None, v_new=v if new else None)
        torch.cuda.synchronize()
        assert (used_scratch(scratch) > 256) == (kind == "several")
        got.append((kc, vc, out))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    for s in range(n):
        assert (got[0][2][s, rows - 17 * s:] == 7.0).all() and (got[0][2][s, :rows - 17 * s] != 7.0).any(-1).all()


@pytest.mark.parametrize("heads,kvh,hd", [(32, 8, 128), (14, 2, 64), (8, 4, 32)])
def test_seventeen_rows(K, heads, kvh, hd):
    """The fewest rows that this kernel takes: a row group that they fill in part, unequal sequences."""
    n, rows, ctx = 6, 17, 4096
    b = Long(K, normal(1, n, ctx, kvh, hd), normal(2, n, ctx, kvh, hd), heads)
    q = normal(3, n, rows, heads, hd)
    at = [ctx - rows, 0, 111, 2000, 128, ctx - rows]
    got, scratch = b.run(q, at)
    assert 1 < splits_of(scratch, n, rows, heads, hd, b.ctx) < 16
    b.check(got, q, at, list(range(rows)))


@pytest.mark.parametrize("n,kind", MANY)
@pytest.mark.parametrize("hd", [64, 128])
def test_few_large_weights_of_many_rows(K, n, kind, hd):
    """Rows whose queries are a position's key, many times as large: its weight, and those of a few near copies of it, are
    all there is, and a score's error is theirs."""
    length, rows, heads, kvh = 2048, 200, 8, 2
    k = normal(1, n, length, kvh, hd)
    k[:, 1::2] = k[:, 0::2] + 0.02 * normal(2, n, length // 2, kvh, hd)
    b = Long(K, k, normal(3, n, length, kvh, hd), heads)
    at = [length - rows] * n
    pick = torch.randint(0, length - rows, (n, rows, heads), generator=torch.Generator(device="cuda").manual_seed(4),
                         device="cuda")
    head = torch.arange(heads, device="cuda") // (heads // kvh)
    q = b.k[torch.arange(n, device="cuda")[:, None, None], pick, head].float() * 6
    got, scratch = b.run(q, at)
    assert (splits_of(scratch, n, rows, heads, hd, b.ctx) > 1) == (kind == "several")
    b.check(got, q, at, [0, 5, 127, 128, 199])


@pytest.mark.parametrize("far", [26, 30, 31, 33, 36, 37])
def test_one_large_weight_and_a_long_flat_tail(K, far):
    """One position outweighs each of 65535 others by about 2^far: alone they are nothing, together 2^(16 - far) of the
    output.  The others' keys are zero, so that their scores are, exactly, and the output is (T - 1) / (T + 1), of
    values -1 and 1 and a tail T below 2^-9 that is off by less than 2^-16 of itself (the score's error).  The tensor cores cut
    O by less than 2^-23 at each of the 32 additions of a window, and each of the 256 windows is added in fp32, off by
    half a step of numbers below 1, 2^-25.  Weights are summed over 16 of the 512 tiles, these 32 sums to one, each
    addition off by half a step of numbers above 1, 2^-24."""
    ctx, rows, heads, kvh, hd = 65536, 320, 32, 4, 64
    k, v = torch.zeros(1, ctx, kvh, hd, device="cuda"), torch.ones(1, ctx, kvh, hd, device="cuda")
    k[:, 0], v[:, 0] = 2.0, -1.0
    b = Long(K, k, v, heads)
    assert (b.k[:, 1:] == 0).all() and (b.k[:, 0] > 1.9).all() and (b.v[:, 0] == -1).all() and (b.v[:, 1:] == 1).all()
    # weights of 2^-0.9 times 2^-far: just below half a step where 2^-far is one
    q = torch.full((1, rows, heads, hd), (far + 1.1) * np.log(2) / (b.k[0, 0, 0].sum().item() * hd ** -0.5), device="cuda")
    got, scratch = b.run(q, [ctx - rows])
    assert splits_of(scratch, 1, rows, heads, hd, ctx) == 1
    for r in (0, 150, 319):
        z, _ = b.scores(q, 0, ctx - rows, [r])
        tail = (z - z.amax(-1, keepdim=True)).exp().sum(-1) - 1
        assert (tail < 2.0 ** -9).all()
        want = ((tail - 1) / (tail + 1)).view(1, heads, 1).expand(1, heads, hd)
        tol = 2.0 ** -24 + 2 * 2.0 ** -9 * 2.0 ** -16 + 32 * 2.0 ** -23 + 256 * 2.0 ** -25 + 48 * 2.0 ** -24
        torch.testing.assert_close(got[0, r:r + 1].double(), want, rtol=0, atol=tol)


# --------------------------------------------- the same bits on every path
def bits(K, b, q, positions):
    """Rows of a call one by one (joined in the attention's launch) against the whole call."""
    whole, _ = b.run(q, positions)
    for s in range(q.shape[0]):
        one = Long.__new__(Long)
        one.__dict__.update(b.__dict__)
        size = b.kc.numel() // b.n
        one.kc, one.vc = b.kc[s * size:(s + 1) * size].clone(), b.vc[s * size:(s + 1) * size].clone()
        for r in range(q.shape[1]):
            alone, _ = one.run(q[s:s + 1, r:r + 1], [positions[s] + r])
            assert torch.equal(alone[0, 0], whole[s, r]), (s, r)
    return whole


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 128), (14, 2, 64), (4, 2, 32), (4, 2, 256)])
@pytest.mark.parametrize("ctx,rows", [(2500, 1), (2500, 5), (6000, 1), (6000, 3), (12288, 1)])
def test_bits_of_a_second_launch(K, heads, kvh, hd, ctx, rows):
    """A decode step alone joins its chunks in the attention's launch; in a call of more than 64 groups of rows a second
    one does.  Chunks of 256 and of 512 positions, the last of 1 to all of theirs."""
    n = 40
    assert n * kvh > 64
    g = torch.Generator().manual_seed(ctx + hd)
    lengths = torch.randint(rows, ctx + 1, (n,), generator=g).tolist()
    lengths[:4] = [ctx, rows, 513, 1024]
    b = Long(K, normal(1, n, ctx, kvh, hd), normal(2, n, ctx, kvh, hd), heads)
    q = normal(3, n, rows, heads, hd)
    at = [length - rows for length in lengths]
    whole = bits(K, b, q, at)
    b.check(whole, q, at, list(range(rows)))


@pytest.mark.parametrize("hd,split", [(128, 4), (64, 2), (32, 1), (256, 2)])
def test_bits_of_some_of_the_heads(K, hd, split):
    """The KV heads of a part of a model (a rank of a split one) alone give the bits that they have among all."""
    n, ctx, kvh, group = 3, 3000, 4, 4
    k, v, q = normal(1, n, ctx, kvh, hd), normal(2, n, ctx, kvh, hd), normal(3, n, 2, kvh * group, hd)
    at = [2998, 700, 0]
    whole, _ = Long(K, k, v, kvh * group).run(q, at)
    for h in range(0, kvh, split):
        part, _ = Long(K, k[:, :, h:h + split], v[:, :, h:h + split], split * group).run(
            q[:, :, h * group:(h + split) * group], at)
        assert torch.equal(part, whole[:, :, h * group:(h + split) * group])


# --------------------------------------------- every kernel
@pytest.mark.parametrize("rows,n", [(1, 2), (6, 2), (200, 4), (200, 8)])
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_scores_of_any_size(K, rows, n, hd):
    """Scores up to 2^60, between whose floats lie worlds: the softmax is a choice of the largest.  (Rows whose two largest
    are nearer than a score's error choose either, and are left out; they are few.)"""
    length, heads, kvh = 1300, 8, 2
    b = Long(K, normal(1, n, length, kvh, hd), normal(2, n, length, kvh, hd), heads)
    at = [length - rows] * n
    some = sorted({0, rows // 2, rows - 1})
    for i in range(14, 61, 2):
        q = normal(i, n, rows, heads, hd) * 2.0 ** i
        got, _ = b.run(q, at)
        assert torch.isfinite(got).all(), i
        for s in range(n):
            z, most = b.scores(q, s, at[s], some)
            top, where = z.topk(2, -1)
            clear = (top[..., 0] - top[..., 1] > 2 * most * 2.0 ** -20 + 20).flatten(1)
            assert clear.double().mean() > 0.8
            want = torch.stack([b.v[s, where[:, j, :, 0], j] for j in range(kvh)], 1).flatten(1, 2)
            torch.testing.assert_close(got[s, some].double()[clear], want[clear], rtol=0,
                                       atol=2.0 ** -20 * b.v[s].abs().max().item())
