"""Cases and plain forms of the 4-bit KV cache operators and of draft verification.

The operators: appending rows of keys and values to a 4-bit cache and reading
them back, attention of query rows over that cache, and the verification of
drafted tokens against the target's probabilities.  ``run`` computes them with
elementary torch operations, or, where ``own`` is true, with the library's
entry points.

The cache of one side (keys or values) is [sequence][kv head][tile][20 * hd]
bytes, a tile holding 32 positions.  Every 32 dimensions of a head vector
share two fp16 numbers D and M; code c stands for fp16(D * (1 + c/16) + M).
Eight codes fill a 32-bit word, code i at bits 4i + 2 (mod 32).  A key tile is
[position 32][t 4][group] words (dimension 32 * group + 8 t + i) and then
[position 32][group] pairs (D, M); a value tile is [group][e 8][t 4][n 4]
words (dimension 32 * group + 8 n + e, position 8 t + i) and then
[group][D, M][t 4][8] halves, positions in the order 0 4 1 5 2 6 3 7.
"""
import math

import torch

own = False

ORDER = (0, 4, 1, 5, 2, 6, 3, 7)


def listed():
    """Llama-3-8B's heads (32 over 8, 128 wide; vocabulary 128256) and Qwen2-0.5B's (14 over 2, 64 wide; 151936)."""
    big = dict(heads=32, kv_heads=8, hd=128, split_half=False)
    small = dict(heads=14, kv_heads=2, hd=64, split_half=True)
    return [
        # one decoded token's key and value: latency alone
        dict(name="append token", op="append", seqs=1, rows=1, ctx=4096, len=2048, ragged=False, **big),
        # one token in each of 48 sessions of a small model, at odd positions
        dict(name="append sessions", op="append", seqs=48, rows=1, ctx=2500, len=2500, ragged=True, **small),
        # a prefill chunk of one prompt
        dict(name="append chunk", op="append", seqs=1, rows=256, ctx=4096, len=2048 + 37, ragged=False, **big),
        # whole prompts of eight sessions, of unequal lengths
        dict(name="append prompts", op="append", seqs=8, rows=2048, ctx=2048, len=2048, ragged=True, **big),
        # decode of one session at the benchmark's context
        dict(name="decode one", op="attend", seqs=1, rows=1, ctx=4096, len=2048, ragged=False, **big),
        # sixteen sessions of a small model, seven heads a KV head
        dict(name="decode sixteen", op="attend", seqs=16, rows=1, ctx=2500, len=2411, ragged=True, **small),
        # a full batch of sessions of unequal lengths
        dict(name="decode batch", op="attend", seqs=64, rows=1, ctx=8192, len=8192, ragged=True, **big),
        # one long context
        dict(name="decode long", op="attend", seqs=1, rows=1, ctx=131072, len=131072, ragged=False, **big),
        # verification of up to seven drafts in each of four sessions
        dict(name="verify rows", op="attend", seqs=4, rows=8, ctx=4096, len=4001, ragged=True, **big),
        # the last chunk of a long prompt
        dict(name="prefill chunk", op="attend", seqs=1, rows=256, ctx=8192, len=8192, ragged=False, **big),
        # prompt-lookup drafts of one session: the drafts are certain
        dict(name="drafts one", op="drafts", seqs=1, drafts=4, vocab=128256, probs=False, temperature=0.8),
        # a draft model's proposals in a batch of sessions
        dict(name="drafts batch", op="drafts", seqs=32, drafts=7, vocab=151936, probs=True, temperature=1.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "drafts"])
    if op == "drafts":
        drafts = rng.randint(1, 12)
        vocab = _log(rng, 1000, 151936)
        seqs = _log(rng, 1, max(1, min(64, 36_000_000 // (vocab * (drafts + 1)))))
        return dict(op=op, seqs=seqs, drafts=drafts, vocab=vocab, probs=rng.random() < 0.5,
                    temperature=round(rng.uniform(0.3, 1.5), 3))
    hd = rng.choice([32, 64, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 7, 8])
    heads = dict(heads=kv_heads * group, kv_heads=kv_heads, hd=hd, split_half=rng.random() < 0.5)
    width = kv_heads * hd
    if op == "append":
        rows = _log(rng, 1, 2048)
        seqs = _log(rng, 1, max(1, min(64, 16_000_000 // (rows * width))))
        ctx = rows + _log(rng, 1, 2048)
    else:
        rows = rng.choice([1, 1, rng.randint(2, 16), _log(rng, 17, 256)])
        each = rows * heads["heads"] * hd
        ctx = _log(rng, max(rows, 16), min(32768, 8_000_000_000 // each))
        seqs = _log(rng, 1, max(1, min(64, 500_000_000 // (ctx * width), 8_000_000_000 // (ctx * each))))
    return dict(op=op, seqs=seqs, rows=rows, ctx=ctx, len=rng.randint(rows, ctx), ragged=rng.random() < 0.7, **heads)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "drafts":
        return _prepare_drafts(case, g)
    n, rows, hkv, hd, ctx = case["seqs"], case["rows"], case["kv_heads"], case["hd"], case["ctx"]
    s = dict(case)
    # positions: how many each sequence holds before its rows; row counts: how many of its rows are real
    last = case["len"] - rows
    if case["ragged"]:
        s["positions"] = torch.randint(last // 8, last + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["counts"] = torch.randint((rows + 1) // 2, rows + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    else:
        s["positions"] = torch.full((n,), last, device="cuda", dtype=torch.int32)
        s["counts"] = None
    freq = 1.0 / 500000.0 ** (torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(ctx, device="cuda", dtype=torch.float64)[:, None] * freq
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    tiles = -(-ctx // 32)
    # keys have a few channels far larger than the others, as models' keys have
    loud = 1 + 7 * (torch.rand(hkv * hd, generator=g, device="cuda") < 0.03).float()
    if case["op"] == "append":
        s["k"] = torch.randn(n, rows, hkv * hd, generator=g, device="cuda") * loud
        s["v"] = torch.randn(n, rows, hkv * hd, generator=g, device="cuda")
        for side in ("k_cache", "v_cache"):
            s[side] = torch.zeros(n, hkv, tiles, 20 * hd, device="cuda", dtype=torch.uint8)
        s["k_read"], s["v_read"] = torch.zeros_like(s["k"]), torch.zeros_like(s["v"])
        return s
    s["q"] = torch.randn(n, rows, case["heads"] * hd, generator=g, device="cuda")
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = 1 / math.sqrt(hd)
    sides = {side: torch.empty(n, hkv, tiles, 20 * hd, device="cuda", dtype=torch.uint8) for side in ("k_cache", "v_cache")}
    for i in range(n):
        x = torch.randn(hkv, tiles * 32, hd, generator=g, device="cuda")
        sides["v_cache"][i] = _pack_values(*_quantise(x))
        x = torch.randn(hkv, tiles * 32, hd, generator=g, device="cuda") * loud.view(hkv, 1, hd)
        sides["k_cache"][i] = _pack_keys(*_quantise(x))
    s.update(sides)
    s["scratch"] = torch.zeros(_scratch_bytes(case), device="cuda", dtype=torch.uint8)
    return s


def _scratch_bytes(case):
    """Room for the partial results of every 256 positions of each (row, head)."""
    return 256 + 4 * case["seqs"] * case["rows"] * case["heads"] * (-(-case["ctx"] // 256)) * (case["hd"] + 2)


def _prepare_drafts(case, g):
    n, m, vocab = case["seqs"], case["drafts"], case["vocab"]
    s = dict(case)
    # a few hundred likely tokens over a long tail, as a trained model's logits are
    logits = torch.randn(n, m + 1, vocab, generator=g, device="cuda") * 2.5
    q = torch.softmax((logits[:, :m] + 0.7 * torch.randn(n, m, vocab, generator=g, device="cuda")) / case["temperature"], -1)
    s["logits"] = logits
    s["draft"] = torch.multinomial(q.view(n * m, vocab), 1, generator=g).view(n, m).to(torch.int32)
    s["probs"] = q if case["probs"] else None
    s["counts"] = torch.randint((m + 1) // 2, m + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    s["uniforms"] = torch.rand(n, m + 1, generator=g, device="cuda")
    s["temperatures"] = torch.full((n,), case["temperature"], device="cuda")
    s["accepted"] = torch.zeros(n, device="cuda", dtype=torch.int32)
    s["token"] = torch.zeros(n, device="cuda", dtype=torch.int32)
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin, split_half):
    """RoPE of [..., heads, hd] by cos/sin [..., 1, hd/2]: adjacent pairs, or a half with the other half."""
    if split_half:
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)


def _quantise(x):
    """Codes, D and M of [..., hd]: (codes [..., hd], D [..., hd/32], M [..., hd/32])."""
    x = torch.where(x.isnan(), torch.zeros_like(x), x).clamp(-16384.0, 16384.0)
    x = x.unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    D = ((hi - lo) * (16.0 / 15.0)).half()
    M = (lo - D.float()).half()
    inverse = torch.where(D > 0, 16.0 / D.float(), torch.zeros_like(lo))
    codes = (((x - M.float()) - D.float()) * inverse).round().clamp(0, 15).to(torch.int32)
    return codes.flatten(-2), D.squeeze(-1), M.squeeze(-1)


def _value(codes, D, M):
    """What codes [..., hd] stand for."""
    t = 1.0 + codes.unflatten(-1, (-1, 32)).float() / 16.0
    return (D.float()[..., None] * t + M.float()[..., None]).half().float().flatten(-2)


def _words(codes):
    """Eight codes of the last axis as one word, code i at bits 4i + 2 (mod 32)."""
    w = (codes.long() << (4 * torch.arange(8, device=codes.device))).sum(-1)
    w = ((w << 2) | (w >> 30)) & 0xFFFFFFFF
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _codes(words):
    w = ((words >> 2) & 0x3FFFFFFF) | (words << 30)
    return (w[..., None] >> (4 * torch.arange(8, device=words.device, dtype=torch.int32))) & 15


def _bytes(x):
    return x.contiguous().flatten(2).view(torch.uint8)


def _pack_keys(codes, D, M):
    """Tiles [kv head, tile, 20 hd] of codes [kv head, position, hd]."""
    h, p, hd = codes.shape
    w = _words(codes.view(h, p // 32, 32, hd // 32, 4, 8)).transpose(-1, -2)
    dm = torch.stack([D, M], -1).view(h, p // 32, 32, hd // 32, 2)
    return torch.cat([_bytes(w), _bytes(dm)], -1)


def _pack_values(codes, D, M):
    h, p, hd = codes.shape
    c = codes.view(h, p // 32, 4, 8, hd // 32, 4, 8).permute(0, 1, 4, 6, 2, 5, 3)  # h tile g e t n i
    dm = torch.stack([D, M], -1).view(h, p // 32, 4, 8, hd // 32, 2)[:, :, :, list(ORDER)].permute(0, 1, 4, 5, 2, 3)
    return torch.cat([_bytes(_words(c)), _bytes(dm)], -1)


def _open_keys(tiles):
    """Values [sequence, kv head, position, hd] of key tiles [sequence, kv head, tile, 20 hd]."""
    n, h, t, b = tiles.shape
    hd = b // 20
    w = tiles[..., :16 * hd].contiguous().view(torch.int32).view(n, h, t * 32, 4, hd // 32)
    codes = _codes(w).transpose(-2, -3).flatten(-3)
    dm = tiles[..., 16 * hd:].contiguous().view(torch.float16).view(n, h, t * 32, hd // 32, 2)
    return _value(codes, dm[..., 0], dm[..., 1])


def _open_values(tiles):
    n, h, t, b = tiles.shape
    hd = b // 20
    w = tiles[..., :16 * hd].contiguous().view(torch.int32).view(n, h, t, hd // 32, 8, 4, 4)
    codes = _codes(w).permute(0, 1, 2, 5, 7, 3, 6, 4).reshape(n, h, t * 32, hd)  # n h tile t i g n e
    dm = tiles[..., 16 * hd:].contiguous().view(torch.float16).view(n, h, t, hd // 32, 2, 4, 8)
    back = [ORDER.index(i) for i in range(8)]
    dm = dm[..., back].permute(0, 1, 2, 5, 6, 3, 4).reshape(n, h, t * 32, hd // 32, 2)
    return _value(codes, dm[..., 0], dm[..., 1])


def _places(s):
    """Positions of every row [sequence, row], and which rows are real."""
    r = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    p = s["positions"][:, None] + r
    real = torch.ones_like(p, dtype=torch.bool) if s["counts"] is None else r < s["counts"][:, None]
    return torch.where(real, p, torch.zeros_like(p)), real


def _append_plain(s):
    at, real = _places(s)
    k = s["k"].view(s["seqs"], s["rows"], s["kv_heads"], s["hd"])
    v = s["v"].view_as(k)
    k = _rotate(k, s["cos"][at][:, :, None], s["sin"][at][:, :, None], s["split_half"])
    real = real[:, :, None, None]
    k, v = (torch.where(real, _value(*_quantise(x)), torch.zeros_like(x)) for x in (k, v))
    return k.flatten(2), v.flatten(2)


def _attend_plain(s):
    at, real = _places(s)
    n, rows, hkv, hd = s["seqs"], s["rows"], s["kv_heads"], s["hd"]
    used = -(-s["len"] // 32)
    q = _rotate(s["q"].view(n, rows, s["heads"], hd), s["cos"][at][:, :, None], s["sin"][at][:, :, None], s["split_half"])
    q = q.view(n, rows, hkv, -1, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)  # n, kv head, (head of it, row), hd
    k, v = _open_keys(s["k_cache"][:, :, :used]), _open_values(s["v_cache"][:, :, :used])
    score = (q @ k.transpose(-1, -2)) * s["scale"]
    score = score.unflatten(2, (-1, rows))
    score = score.masked_fill(torch.arange(used * 32, device="cuda") > at[:, None, None, :, None], -math.inf)
    e = (score - score.amax(-1, keepdim=True)).exp()
    out = (e.flatten(2, 3) @ v) / e.flatten(2, 3).sum(-1, keepdim=True)
    out = out.unflatten(2, (-1, rows)).permute(0, 3, 1, 2, 4).flatten(2)
    return torch.where(real[:, :, None], out, torch.zeros_like(out))


def _drafts_plain(s):
    m, vocab = s["drafts"], s["vocab"]
    # in 64 bits: a decision next to its border must not depend on rounding
    x = s["logits"].double()
    e = ((x - x.amax(-1, keepdim=True)) / s["temperatures"].double()[:, None, None]).exp()
    p = e / e.sum(-1, keepdim=True)
    draft = s["draft"].long()
    pd = p[:, :m].gather(-1, draft[..., None]).squeeze(-1)
    qd = torch.ones_like(pd) if s["probs"] is None else s["probs"].gather(-1, draft[..., None]).squeeze(-1).double()
    u = s["uniforms"].double()
    held = (u[:, :m] * qd < pd) & (torch.arange(m, device="cuda") < s["counts"][:, None])
    accepted = held.long().cumprod(-1).sum(-1)
    last = accepted == s["counts"]
    row = p.gather(1, accepted[:, None, None].expand(-1, -1, vocab)).squeeze(1)
    at = accepted.clamp(max=m - 1)[:, None]
    if s["probs"] is None:
        other = torch.zeros_like(row).scatter(-1, draft.gather(1, at), math.inf)
    else:
        other = s["probs"].gather(1, at[..., None].expand(-1, -1, vocab)).squeeze(1).double()
    rest = (row - torch.where(last[:, None], torch.zeros_like(row), other)).clamp(min=0)
    cum = rest.cumsum(-1)
    token = (cum <= u[:, m:] * cum[:, -1:]).sum(-1)
    return accepted.to(torch.int32), token.to(torch.int32)


def run(state):
    s = state
    if own:
        from overfit_b200 import kernels
    if s["op"] == "append":
        if own:
            shape = (s["kv_heads"], s["hd"], s["ctx"])
            kernels.KvCacheQ4.append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], *shape, s["cos"], s["sin"],
                                     s["split_half"], row_counts=s["counts"])
            kernels.KvCacheQ4.read(s["k_cache"], s["v_cache"], s["positions"], *shape, s["k_read"], s["v_read"],
                                   row_counts=s["counts"])
            return s["k_read"], s["v_read"]
        return _append_plain(s)
    if s["op"] == "attend":
        if own:
            kernels.CachedAttentionKernel.compute_q4(s["q"], s["k_cache"], s["v_cache"], s["out"], s["positions"], s["heads"],
                                                     s["kv_heads"], s["hd"], s["ctx"], s["scale"], s["scratch"], s["cos"],
                                                     s["sin"], s["split_half"], row_counts=s["counts"])
            return s["out"]
        return _attend_plain(s)
    if own:
        kernels.SpeculativeVerifier.verify(s["logits"], s["draft"], s["uniforms"], s["temperatures"], s["accepted"], s["token"],
                                           draft_probs=s["probs"], draft_counts=s["counts"])
        return s["accepted"], s["token"]
    return _drafts_plain(s)


def work(case):
    n = case["seqs"]
    if case["op"] == "drafts":
        # every row of logits once, the draft's probabilities where a row is sampled from
        per = (case["drafts"] + 1 + (1 if case["probs"] else 0)) * case["vocab"]
        return dict(bytes=4 * n * (per + 4 * case["drafts"]), flops=4 * n * per)
    rows, hd = case["rows"], case["hd"]
    # what a ragged case holds on average
    share = 0.75 if case["ragged"] and rows > 1 else 1.0
    elements = n * rows * share * case["kv_heads"] * hd
    if case["op"] == "append":
        # keys and values read, 5 bits of each written and read, and the values written
        return dict(bytes=2 * elements * (4 + 2 * 0.625 + 4), flops=2 * elements * 8)
    length = case["len"] - rows * (1 - share / 2)
    before = (case["len"] - rows) * (9 / 16 if case["ragged"] else 1.0)
    length = before + rows * share
    pairs = n * rows * share * case["heads"] * (before + rows * share / 2)
    q = n * rows * share * case["heads"] * hd
    return dict(bytes=n * length * case["kv_heads"] * 1.25 * hd + 8 * q, flops=4 * pairs * hd)


# ---------------------------------------------------------------- in 64 bits
def _f32(x):
    """A sum, difference, product or quotient of two fp32 numbers, formed in 64 bits, as fp32 rounds it."""
    return x.to(torch.float32).to(torch.float64)


def _f16(x):
    return x.to(torch.float32).to(torch.float16).to(torch.float64)


def _turn(x, p, s):
    """RoPE of x [row, head, hd] (64 bits) at positions p, every step rounded as the operator's definition does."""
    c, d = s["cos"][p].double()[:, None], s["sin"][p].double()[:, None]
    half = x.shape[-1] // 2
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if s["split_half"] else (2 * i, 2 * i + 1)
    y = torch.empty_like(x)
    y[..., a] = _f32(_f32(x[..., a] * c) - _f32(x[..., b] * d))
    y[..., b] = _f32(_f32(x[..., a] * d) + _f32(x[..., b] * c))
    return y


def _stored(x):
    """The values that x [row, head, hd] has in the cache."""
    y = torch.empty_like(x)
    for g in range(x.shape[-1] // 32):
        z = x[..., 32 * g:32 * g + 32]
        lo, hi = z.min(-1, keepdim=True).values, z.max(-1, keepdim=True).values
        D = _f16(_f32(_f32(hi - lo) * torch.tensor(16 / 15, dtype=torch.float32).double().item()))
        M = _f16(_f32(lo - D))
        c = torch.round(_f32(_f32(_f32(z - M) - D) * _f32(16 / D))).clamp(0, 15)
        y[..., 32 * g:32 * g + 32] = _f16(D * (1 + c / 16) + M)
    return y


def _cached(tiles, keys):
    """Values [position, head, hd] of one sequence's tiles [head, tile, 20 hd], word by word, in 64 bits."""
    h, t, b = tiles.shape
    hd, groups = b // 20, b // 640
    words = tiles[..., :16 * hd].contiguous().view(torch.int32).long() & 0xFFFFFFFF
    halves = tiles[..., 16 * hd:].contiguous().view(torch.float16).double()
    d, p = torch.arange(hd, device="cuda")[None, :], torch.arange(32, device="cuda")[:, None]
    if keys:
        word = p * (hd // 8) + (d % 32 // 8) * groups + d // 32
        i = d % 8 + 0 * p
        first = 2 * (p * groups + d // 32)
        second = first + 1
    else:
        word = ((d // 32 * 8 + d % 8) * 4 + p // 8) * 4 + d % 32 // 8
        i = p % 8 + 0 * d
        place = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device="cuda")[p % 8]
        first = d // 32 * 64 + p // 8 * 8 + place
        second = first + 32
    w = words[:, :, word]
    code = torch.where(i == 7, (w >> 30) | ((w & 3) << 2), (w >> (4 * i + 2).clamp(max=31)) & 15)
    x = (halves[:, :, first] * (1 + code.double() / 16) + halves[:, :, second])
    return _f16(x).reshape(h, t * 32, hd).transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    n = case["seqs"]
    if case["op"] == "drafts":
        return _exact_drafts(s)
    rows, heads, hkv, hd = s["rows"], s["heads"], s["kv_heads"], s["hd"]
    at = s["positions"].tolist()
    count = [rows] * n if s["counts"] is None else s["counts"].tolist()
    if s["op"] == "append":
        k, v = (torch.zeros(n, rows, hkv, hd, device="cuda", dtype=torch.float64) for _ in "kv")
        for i in range(n):
            c = count[i]
            p = torch.arange(at[i], at[i] + c, device="cuda")
            k[i, :c] = _stored(_turn(s["k"][i, :c].double().view(c, hkv, hd), p, s))
            v[i, :c] = _stored(s["v"][i, :c].double().view(c, hkv, hd))
        return k.flatten(2), v.flatten(2)
    out = torch.zeros(n, rows, heads, hd, device="cuda", dtype=torch.float64)
    for i in range(n):
        c = count[i]
        if c == 0:
            continue
        last = at[i] + c
        p = torch.arange(at[i], last, device="cuda")
        q = s["q"][i, :c].double().view(c, heads, hd)
        co, si = s["cos"][p].double()[:, None], s["sin"][p].double()[:, None]
        j = torch.arange(hd // 2, device="cuda")
        a, b = (j, j + hd // 2) if s["split_half"] else (2 * j, 2 * j + 1)
        r = torch.empty_like(q)
        r[..., a], r[..., b] = q[..., a] * co - q[..., b] * si, q[..., a] * si + q[..., b] * co
        tiles = -(-last // 32)
        k = _cached(s["k_cache"][i, :, :tiles], True)[:last]
        v = _cached(s["v_cache"][i, :, :tiles], False)[:last]
        for h in range(heads):
            z = r[:, h] @ k[:, h * hkv // heads].T / math.sqrt(hd)
            z[torch.arange(last, device="cuda")[None, :] > p[:, None]] = -math.inf
            out[i, :c, h] = torch.softmax(z, -1) @ v[:, h * hkv // heads]
    return out.flatten(2)


def _exact_drafts(s):
    accepted, tokens = [], []
    for i in range(s["seqs"]):
        u, t = s["uniforms"][i].double(), s["temperatures"][i].double()
        k = 0
        for j in range(int(s["counts"][i])):
            p = torch.softmax(s["logits"][i, j].double() / t, 0)
            d = int(s["draft"][i, j])
            if not u[j] * (1.0 if s["probs"] is None else s["probs"][i, j, d].double()) < p[d]:
                break
            k += 1
        r = torch.softmax(s["logits"][i, k].double() / t, 0)
        if k < int(s["counts"][i]):
            d = int(s["draft"][i, k])
            if s["probs"] is None:
                r[d] = 0
            else:
                r = torch.relu(r - s["probs"][i, k].double())
        c = torch.cumsum(r, 0)
        accepted.append(k)
        tokens.append(int(torch.searchsorted(c, u[s["drafts"]] * c[-1], right=True)))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
