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
