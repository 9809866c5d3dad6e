// ovf_attn_q4.cu — causal attention of query rows over the 4-bit KV cache.
//
// Row r of sequence s is at position p = positions[s] + r and attends the
// cache's positions [0, p]:  out = sum_j softmax_j(scale * q . K_j) V_j with
// the values that the cache's codes stand for (ovf_q4.cuh) and the query
// rotated at p.
//
// Both products run on the tensor cores (m16n8k16, fp16 operands, fp32 sums)
// without losing the query's or the weights' precision: the cached values are
// fp16 numbers by definition, and an fp32 operand x enters as two fp16 numbers,
// hi = fp16(x) and lo = fp16(x - hi), which together hold 22 bits.  The cache is
// the 16-row operand, straight from its codes (keys: 16 positions, values: 16
// dimensions), the query rows the 8-column one: 4 rows (the heads of one KV head,
// row after row) as hi and lo columns, whose two results a lane holds side by
// side and adds in fp32.  A score's products of 32 dimensions at a time go to an
// accumulator of their own, added in fp32: the tensor cores cut a sum off toward zero
// at each addition, and with one accumulator a decode step whose weights were few and
// large came out 1.9e-6 off, now 3.9e-7 (an fp32 softmax: 5.5e-7).  The shorter chains
// take a token of 32 heads at 2048 positions from 9.9 to 9.5 us, the additions 64
// sessions of 8192 from 93 to 96.
// Queries are scaled by a power of two into fp16's range, weights by 2^14, both
// exactly.  (With the query as the 16-row operand, 8 rows times hi and lo, a decode
// step of 4 heads a KV head left half of it empty: 1037 instructions a tile of 32
// positions and warp, now about half.)
//
// Work is cut into chunks of 256 positions (512 in caches of more than 4096,
// where joining less outweighs a shorter chunk's latency).  A CTA's four warps
// take 64 (two tiles) of each 256 at a time: scores, their maximum, weights,
// weighted values; a second 256 rescales once.  The four results (maximum, sum,
// weighted values) are joined in shared memory, and a second kernel joins the
// chunks of a row.  Chunks, tiles and the order of every sum go by position (and
// the cache's capacity) alone, so a row's result does not depend on what else is
// in the call, bit for bit.  CTAs stay resident and take equal runs of the chunks
// of all sequences, so that unequal lengths cost nothing; a warp's next keys load
// while it weights values, and its next values while it scores.
// Measured, 32 heads over 8, 128 wide: one token at 2048 positions 9.5 us (latency);
// 64 sessions of up to 8192, 97 us, 3.9 TB/s (60 % of the copy rate), bound by latency at
// low occupancy: 2.2 of 4 instructions a clock, half of the integer pipe (taking codes
// apart) and half of DRAM in use, 3.8 warps a scheduler, which wait for fixed latencies,
// loads and instruction fetch.  <4, 1, false> is at its 128 registers and spills some.
#include "ovf_attn_q4_rows.cu"
#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kAqWarps = 4;
static constexpr int kAqThreads = kAqWarps * 32;
static constexpr int kAqLeaf = 256;                // positions that the warps take at a time, two tiles each
static constexpr int kAqCounters = 64;             // ints at the start of the scratch, zero between calls
static_assert(4 * kAqCounters == OVF_Q4_SCRATCH_ZEROS, "what a call finds zero and leaves zero");
static constexpr int kAqWideTiles = 128;           // caches of more tiles have chunks of two leaves
static constexpr float kAqLift = 14.0f;            // weights are held times 2^14: a weight is off by 2^-22 of itself, or 2^-39 of the largest
static_assert(kAqLeaf == kAqWarps * 2 * kQ4Tile, "two tiles a warp");

// A call's shape in the template: NG groups of 32 dimensions, NT operands of 4
// query rows that share the cache's operand.
template <int NG, int NT>
struct AqShape {
    static constexpr int HD = NG * 32;
    static constexpr int kRows = 4 * NT;                 // query rows of an item
    static constexpr int kTile = q4_tile_bytes(HD);
    static constexpr int kSide = 2 * kTile;              // a warp's keys (or values) of a chunk
    static constexpr int MD = HD < 128 ? HD : 128;       // dimensions joined at a time
    static constexpr int kPad = MD + 8;                  // (rows of the join: no two lanes on one bank)
    static constexpr int kRing = kAqWarps * 2 * kSide;
    static constexpr int kMerge = kAqWarps * kRows * kPad * 4;
    static constexpr int kTotal = kRing + kMerge + kAqWarps * kRows * 8 + kAqWarps * 2 * 8;
    static constexpr int kCtas = NG == 8 ? 2 : NT == 2 ? (NG == 4 ? 2 : 3) : 4;  // per SM (registers)
};

struct AqParams {
    Q4Source src;
    int H;
    const float *q;
    float *out, *part, *part_ml;  // partial results [row][chunk][hd] and (maximum, sum)
    float scale2;                 // scale * log2(e): exponentials are powers of two
    int max_chunks;
    int splits;                   // partial results of each row (0: its chunks)
    int groups;                   // groups of rows that the counters have room for, per KV head
    int *done;                    // chunks finished of each (sequence, KV head, group of rows)
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The transpose of an 8 x 8 matrix of fp16: lane 4 e + t gives and gets row e, columns 2 t and 2 t + 1.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// hi and lo part of x, as a pair.
__device__ __forceinline__ uint32_t split1(float x) {
    const __half h = __float2half_rn(x);
    return h2_bits(__halves2half2(h, __float2half_rn(x - __half2float(h))));
}

// Positions of a chunk of a sequence.
__device__ __forceinline__ int aq_span(const Q4View &w) { return w.tiles > kAqWideTiles ? 2 * kAqLeaf : kAqLeaf; }

// The sequences' chunks as one list: per sequence [kv head][KR query rows][chunk].  An item of it:
struct AqItem {
    const uint8_t *k, *v;  // caches of its head
    const float *cos, *sin;
    int64_t head;          // bytes from one head to the next
    int s, pos, count;
    int left;              // items of this sequence behind this one
    int span, chunks, groups, chunk, mt, h;
    int last;              // last position that any of its rows attends
};

template <int KR>
__device__ __forceinline__ int aq_count(const Q4Source &src, int s, int G) {
    Q4View w;
    if (s >= src.n_seq || !q4_view(src, s, &w)) return 0;
    const int span = aq_span(w);
    return src.KVH * ((w.count * G + KR - 1) / KR) * ((w.pos + w.count + span - 1) / span);
}

template <int KR>
__device__ __forceinline__ void aq_last(AqItem *it, int G) {
    it->last = it->pos + min(it->count - 1, (it->mt * KR + KR - 1) / G);
}

// Item `target` of the list that starts with sequence `from`; false if it has fewer.
template <int KR>
__device__ __forceinline__ bool aq_locate(const Q4Source &src, int G, int tile_bytes, int from, long long target, AqItem *it) {
    const int lane = threadIdx.x & 31;
    for (int s0 = from; s0 < src.n_seq; s0 += 32) {
        const int n = aq_count<KR>(src, s0 + lane, G);
        long long sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            if (lane >= o) sum += y;
        }
        const unsigned there = __ballot_sync(0xFFFFFFFFu, target < sum);
        if (!there) {
            target -= __shfl_sync(0xFFFFFFFFu, sum, 31);
            continue;
        }
        const int l = __ffs(there) - 1;
        const int local = (int)(target - __shfl_sync(0xFFFFFFFFu, sum - n, l));
        const int items = __shfl_sync(0xFFFFFFFFu, n, l);
        Q4View w;
        it->s = s0 + l;
        q4_view(src, it->s, &w);
        it->pos = w.pos;
        it->count = w.count;
        it->cos = w.cos;
        it->sin = w.sin;
        it->head = (int64_t)w.tiles * tile_bytes;
        it->span = aq_span(w);
        it->chunks = (w.pos + w.count + it->span - 1) / it->span;
        it->groups = (w.count * G + KR - 1) / KR;
        it->left = items - 1 - local;
        it->chunk = local % it->chunks;
        it->mt = local / it->chunks % it->groups;
        it->h = local / it->chunks / it->groups;
        it->k = w.k + it->head * it->h;
        it->v = w.v + it->head * it->h;
        aq_last<KR>(it, G);
        return true;
    }
    return false;
}

template <int KR>
__device__ __forceinline__ void aq_next(const Q4Source &src, int G, int tile_bytes, AqItem *it) {
    if (it->left == 0) {
        aq_locate<KR>(src, G, tile_bytes, it->s + 1, 0, it);
        return;
    }
    --it->left;
    if (++it->chunk == it->chunks) {
        it->chunk = 0;
        if (++it->mt == it->groups) {
            it->mt = 0;
            ++it->h;
            it->k += it->head;
            it->v += it->head;
        }
        aq_last<KR>(it, G);
    }
}

// The chunks of a row to its output: weights 2^(m_c - max), sums over the chunks
// c, c + 8, .. of eight classes in ascending order, then over the classes in
// order.  Every kernel that joins forms exactly these sums.
static constexpr int kAqClasses = 8;
static constexpr int kAqJoinThreads = 256;
static constexpr int kAqJoinFew = 48;  // chunks up to which a thread takes all classes

// The row of a (row, head) of the call, its number of partial results; false if there is nothing to join.
__device__ __forceinline__ bool aq_join_of(const AqParams &p, int s, int r, int *chunks) {
    Q4View w;
    if (!q4_view(p.src, s, &w) || r >= w.count) return false;
    *chunks = p.splits ? p.splits : (w.pos + r) / aq_span(w) + 1;
    return *chunks > 1;
}

// A row by a group of GL lanes, a lane four dimensions (two fours at head_dim 256); the lanes form the weights
// together.  (A CTA a row left the 8192 rows of a prefill chunk at 17 us, a thread that reads all maxima by itself a
// decode step's 32 rows a microsecond longer.)  Groups without a row pass chunks = 0.
template <int HD>
struct AqJoin {
    static constexpr int TC = HD / 4, GL = TC < 32 ? TC : 32, E = (kAqJoinFew + GL - 1) / GL, F = TC / GL;
};
template <int HD>
__device__ __forceinline__ void aq_join_few(const AqParams &p, int64_t row, int chunks) {
    constexpr int TC = AqJoin<HD>::TC, GL = AqJoin<HD>::GL, E = AqJoin<HD>::E, F = AqJoin<HD>::F;
    const int lane = threadIdx.x & 31, l0 = lane % GL;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + row * p.max_chunks;
    const float4 *part = reinterpret_cast<const float4 *>(p.part) + row * p.max_chunks * TC + l0;
    float2 y[E];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        y[j] = j * GL + l0 < chunks ? __ldcg(ml + j * GL + l0) : make_float2(-INFINITY, 0.0f);
        top = fmaxf(top, y[j].x);
    }
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
#pragma unroll
    for (int j = 0; j < E; ++j) y[j].x = y[j].x == -INFINITY ? 0.0f : ex2(y[j].x - top);  // (0: a split without an attended position)
    float4 v[kAqClasses][F];
    float l[kAqClasses];
#pragma unroll
    for (int k = 0; k < kAqClasses; ++k) {
        l[k] = 0.0f;
#pragma unroll
        for (int f = 0; f < F; ++f) v[k][f] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    const int most = __reduce_max_sync(0xFFFFFFFFu, chunks);
#pragma unroll
    for (int c0 = 0; c0 < kAqJoinFew; c0 += kAqClasses) {
        if (c0 >= most) break;
        float4 u[kAqClasses][F];
        float w[kAqClasses], n[kAqClasses];
#pragma unroll
        for (int k = 0; k < kAqClasses; ++k) {
            const int from = lane - l0 + (c0 + k) % GL;
            w[k] = __shfl_sync(0xFFFFFFFFu, y[(c0 + k) / GL].x, from);
            n[k] = __shfl_sync(0xFFFFFFFFu, y[(c0 + k) / GL].y, from);
#pragma unroll
            for (int f = 0; f < F; ++f)
                u[k][f] = c0 + k < chunks && !(w[k] == 0.0f) ? __ldcg(part + (size_t)(c0 + k) * TC + f * GL)
                                                             : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int k = 0; k < kAqClasses; ++k) {
            l[k] += n[k] * w[k];
#pragma unroll
            for (int f = 0; f < F; ++f) {
                v[k][f].x += u[k][f].x * w[k], v[k][f].y += u[k][f].y * w[k];
                v[k][f].z += u[k][f].z * w[k], v[k][f].w += u[k][f].w * w[k];
            }
        }
    }
#pragma unroll
    for (int k = 1; k < kAqClasses; ++k) {
        l[0] += l[k];
#pragma unroll
        for (int f = 0; f < F; ++f)
            v[0][f].x += v[k][f].x, v[0][f].y += v[k][f].y, v[0][f].z += v[k][f].z, v[0][f].w += v[k][f].w;
    }
    if (chunks == 0) return;
    const float inv = 1.0f / l[0];
#pragma unroll
    for (int f = 0; f < F; ++f)
        reinterpret_cast<float4 *>(p.out)[row * TC + f * GL + l0] =
            make_float4(v[0][f].x * inv, v[0][f].y * inv, v[0][f].z * inv, v[0][f].w * inv);
}

// A warp's part of leaf `leaf` of an item: its first position, and its tiles that hold attended ones.
__device__ __forceinline__ int aq_first(const AqItem &it, int leaf, int warp) {
    return it.chunk * it.span + leaf * kAqLeaf + warp * 2 * kQ4Tile;
}
__device__ __forceinline__ int aq_tiles(const AqItem &it, int first) {
    return min(2, (it.last - first + kQ4Tile) >> 5);  // (0 or less: none)
}

template <int NG, int NT, bool Fused>
__global__ void __launch_bounds__(kAqThreads, Fused ? 2 : AqShape<NG, NT>::kCtas) attention_q4_kernel(const AqParams p) {
    using S = AqShape<NG, NT>;
    constexpr int HD = NG * 32, KR = S::kRows, TB = S::kTile, MD = S::MD, PAD = S::kPad;
    constexpr int RL = MD / 4, NP = KR * RL / kAqThreads > 0 ? KR * RL / kAqThreads : 1;  // the join: lanes a row, rows a thread
    extern __shared__ __align__(128) uint8_t smem[];
    const Q4Source &src = p.src;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = lane >> 2, t = lane & 3, G = p.H / src.KVH;
    uint8_t *keys = smem + warp * 2 * S::kSide, *values = keys + S::kSide;
    float *merge = reinterpret_cast<float *>(smem + S::kRing);                             // [warp][row][PAD]
    float2 *merge_ml = reinterpret_cast<float2 *>(merge + kAqWarps * KR * PAD);            // [warp][row]
    uint64_t *bars = reinterpret_cast<uint64_t *>(merge_ml + kAqWarps * KR) + warp * 2;    // keys, values
    __shared__ int last_one;
    if (lane < 2) mbar_init(&bars[lane], 1);
    fence_mbar_init();
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();

    // this CTA's run of the list
    long long total = 0;
    for (int s0 = 0; s0 < src.n_seq; s0 += 32) {
        int n = aq_count<KR>(src, s0 + lane, G);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
        total += n;
    }
    const long long lo = total * blockIdx.x / gridDim.x;
    int left = (int)(total * (blockIdx.x + 1) / gridDim.x - lo);
    AqItem it, next;
    if (left <= 0 || !aq_locate<KR>(src, G, TB, 0, lo, &it)) return;

    // Requests one side of this warp's part of a leaf, if it has one.
    const uint64_t policy = l2_evict_first_policy();
    auto request = [&](const AqItem &i, int leaf, bool side) {
        const int first = aq_first(i, leaf, warp), tiles = aq_tiles(i, first);
        if (tiles > 0 && lane == 0) {
            mbar_arrive_expect_tx(&bars[side], tiles * TB);
            bulk_g2s(side ? values : keys, (side ? i.v : i.k) + (size_t)(first / kQ4Tile) * TB, tiles * TB, &bars[side], policy);
        }
    };
    request(it, 0, false);
    request(it, 0, true);

    uint32_t q[NT][NG][4];  // query operand: pairs (0, 4) (1, 5) (2, 6) (3, 7) of this lane's dimensions
    float factor[NT];       // a score from its sum of products, of row 4 nt + t
    int limit[NT];          // last position that the row attends
    int row_last[NP];       // the join's rows of this thread: last position (-1: none),
    int64_t row_out[NP];    // place among the call's (row, head)s
    int have_h = -1, have_mt = -1, have_s = -1, phase = 0;
    bool dead = false;

    for (; left > 0; --left) {
        if (it.h != have_h || it.mt != have_mt || it.s != have_s) {
            have_h = it.h, have_mt = it.mt, have_s = it.s;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // column e of the operand: row e / 2, its hi (even) or lo part
                const int i = it.mt * KR + nt * 4 + (e >> 1), r = i / G;
                const bool real = r < it.count;
                float x[NG][8];
                if (real) {
                    const float4 *src4 = reinterpret_cast<const float4 *>(
                        p.q + (((size_t)it.s * src.rows + r) * p.H + it.h * G + i % G) * HD + 8 * t);
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float4 u = src4[g * 8], v = src4[g * 8 + 1];
                        x[g][0] = u.x, x[g][1] = u.y, x[g][2] = u.z, x[g][3] = u.w;
                        x[g][4] = v.x, x[g][5] = v.y, x[g][6] = v.z, x[g][7] = v.w;
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[g][k] = 0.0f;
                }
                if (it.cos) {  // Rope/RopeKernel.cs:46-93, each step rounded by itself
                    const int pos = real ? it.pos + r : 0;
                    const float *c = it.cos + (size_t)pos * (HD / 2), *sn = it.sin + (size_t)pos * (HD / 2);
                    if (!src.split_half) {
#pragma unroll
                        for (int g = 0; g < NG; ++g)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const float cc = c[g * 16 + 4 * t + k], ss = sn[g * 16 + 4 * t + k], x0 = x[g][2 * k],
                                            x1 = x[g][2 * k + 1];
                                x[g][2 * k] = fsub(fmul(x0, cc), fmul(x1, ss));
                                x[g][2 * k + 1] = fadd(fmul(x0, ss), fmul(x1, cc));
                            }
                    } else if (NG == 1) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float other = __shfl_xor_sync(0xFFFFFFFFu, x[0][k], 2);
                            const float cc = c[(8 * t + k) & 15], ss = sn[(8 * t + k) & 15];
                            x[0][k] = t < 2 ? fsub(fmul(x[0][k], cc), fmul(other, ss)) : fadd(fmul(other, ss), fmul(x[0][k], cc));
                        }
                    } else {
#pragma unroll
                        for (int g = 0; g < NG / 2; ++g)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const float cc = c[g * 32 + 8 * t + k], ss = sn[g * 32 + 8 * t + k], x0 = x[g][k],
                                            x1 = x[(g + NG / 2) % NG][k];
                                x[g][k] = fsub(fmul(x0, cc), fmul(x1, ss));
                                x[(g + NG / 2) % NG][k] = fadd(fmul(x0, ss), fmul(x1, cc));
                            }
                    }
                }
                float top = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(x[g][k]));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                // the largest element to [2^14, 2^15), by a power of two
                const int ex = min(max((__float_as_int(top) >> 23) & 255, 15), 254);
                const float up = __int_as_float((268 - ex) << 23);
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x0 = x[g][k] * up, x1 = x[g][k + 4] * up;
                        const __half2 hi = __floats2half2_rn(x0, x1);
                        const float2 f = __half22float2(hi);
                        q[nt][g][k] = h2_bits(e & 1 ? __floats2half2_rn(x0 - f.x, x1 - f.y) : hi);
                    }
                // of row 4 nt + t, whose operand the lanes of column 2 t formed
                factor[nt] = p.scale2 * __int_as_float((__shfl_sync(0xFFFFFFFFu, ex, 8 * t) - 14) << 23);
                const int row = (it.mt * KR + nt * 4 + t) / G;
                limit[nt] = row < it.count ? it.pos + row : 0x7FFFFFFF;  // (a row that is none: zeros, which nothing reads)
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int i = it.mt * KR + (threadIdx.x + n * kAqThreads) / RL, r = i / G;
                row_last[n] = r < it.count ? it.pos + r : -1;
                row_out[n] = ((int64_t)it.s * src.rows + r) * p.H + it.h * G + (i - r * G);
            }
        }
        const bool more = left > 1;
        next = it;
        if (more) aq_next<KR>(src, G, TB, &next);

        const int leaves = it.span / kAqLeaf, data_end = it.pos + it.count;
        float m[NT], l[NT], o[NT][NG * 2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = -INFINITY, l[nt] = 0.0f;
#pragma unroll
            for (int d = 0; d < NG * 2; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[nt][d][k] = 0.0f;
        }
        for (int leaf = 0; leaf < leaves; ++leaf) {
            const int first = aq_first(it, leaf, warp), tiles = aq_tiles(it, first);
            // the leaf behind this one
            const bool same = leaf + 1 < leaves;
            auto request_next = [&](bool side) {
                if (same) request(it, leaf + 1, side);
                else if (more) request(next, 0, side);
            };
            if (tiles <= 0) {
                request_next(false);
                request_next(true);
                continue;
            }
            // scores of row 4 nt + t at positions first + 32 tile + 8 (e / 2) + 4 (e % 2) + i
            float s[NT][2][4];
            if (!dead && !mbar_wait_bounded(&bars[0], phase)) dead = true;
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                if (tile < tiles) {
                    const uint8_t *kt = keys + tile * TB;
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // positions i = 2 half and 2 half + 1: the operand's rows e and e + 8
                        uint32_t w[2][NG], dm[2][NG];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const int row = 8 * (e >> 1) + 4 * (e & 1) + 2 * half + b;
                            const uint8_t *wp = kt + (row * 4 + t) * NG * 4, *dp = kt + q4_code_bytes(HD) + row * NG * 4;
                            if (NG == 1) {
                                w[b][0] = *reinterpret_cast<const uint32_t *>(wp);
                                dm[b][0] = *reinterpret_cast<const uint32_t *>(dp);
                            } else if (NG == 2) {
                                *reinterpret_cast<uint2 *>(w[b]) = *reinterpret_cast<const uint2 *>(wp);
                                *reinterpret_cast<uint2 *>(dm[b]) = *reinterpret_cast<const uint2 *>(dp);
                            } else {
#pragma unroll
                                for (int i = 0; i < NG / 4; ++i) {
                                    reinterpret_cast<uint4 *>(w[b])[i] = reinterpret_cast<const uint4 *>(wp)[i];
                                    reinterpret_cast<uint4 *>(dm[b])[i] = reinterpret_cast<const uint4 *>(dp)[i];
                                }
                            }
                        }
                        float c[NT][4] = {};
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            uint32_t v0[4], v1[4];
                            __half2 D = __low2half2(bits_h2(dm[0][g])), M = __high2half2(bits_h2(dm[0][g]));
                            q4_values(w[0][g], D, M, D, M, D, M, D, M, v0);
                            D = __low2half2(bits_h2(dm[1][g])), M = __high2half2(bits_h2(dm[1][g]));
                            q4_values(w[1][g], D, M, D, M, D, M, D, M, v1);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float part[4] = {};
                                mma_f16(part, v0[0], v1[0], v0[1], v1[1], q[nt][g][0], q[nt][g][1]);
                                mma_f16(part, v0[2], v1[2], v0[3], v1[3], q[nt][g][2], q[nt][g][3]);
#pragma unroll
                                for (int k = 0; k < 4; ++k) c[nt][k] += part[k];
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            s[nt][tile][2 * half] = (c[nt][0] + c[nt][1]) * factor[nt];
                            s[nt][tile][2 * half + 1] = (c[nt][2] + c[nt][3]) * factor[nt];
                        }
                    }
                } else {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][tile][i] = -INFINITY;
                }
            }
            uint32_t x[NT][2][4];  // weights as operands
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int at = first + 8 * (e >> 1) + 4 * (e & 1);
                if (__any_sync(0xFFFFFFFFu, first + 2 * kQ4Tile - 1 > limit[nt])) {
#pragma unroll
                    for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (at + tile * kQ4Tile + i > limit[nt]) s[nt][tile][i] = -INFINITY;
                }
                float top = m[nt];
#pragma unroll
                for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[nt][tile][i]);
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
                // (nothing attended: weights of 0.  Rounded up, so that no weight passes 2^14: with scores of 2^25 and more
                // the nearest float to top - 14 may lie 16 below top, whose weight of 2^16 fp16 does not hold)
                const float zero = top == -INFINITY ? 0.0f : top, base = __fsub_ru(zero, kAqLift);
                if (leaf > 0) {
                    const float keep = ex2(m[nt] - zero);
                    l[nt] *= keep;
#pragma unroll
                    for (int d = 0; d < NG * 2; ++d)
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[nt][d][k] *= keep;
                }
                m[nt] = top;
#pragma unroll
                for (int tile = 0; tile < 2; ++tile)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float w = ex2(s[nt][tile][i] - base);
                        l[nt] += w;
                        x[nt][tile][i] = transpose8(split1(w));
                    }
            }

            // (the maxima stand: every read of the keys is behind this warp)
            request_next(false);
            if (!dead && !mbar_wait_bounded(&bars[1], phase)) dead = true;
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                if (tile >= tiles) break;
                uint8_t *vt = values + tile * TB;
                if (first + (tile + 1) * kQ4Tile > data_end) {
                    // what lies behind the sequence's data may be anything: its weights
                    // are 0, and its values must be numbers for that
                    if (first + tile * kQ4Tile + lane >= data_end) {
                        __half *vp = reinterpret_cast<__half *>(vt + q4_code_bytes(HD));
#pragma unroll
                        for (int g = 0; g < NG; ++g) {
                            vp[q4_value_param(g, lane >> 3, lane & 7)] = __half(0.0f);
                            vp[q4_value_param(g, lane >> 3, lane & 7) + 32] = __half(0.0f);
                        }
                        fence_proxy_async_smem();
                    }
                    __syncwarp();
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint4 d = *reinterpret_cast<const uint4 *>(vt + q4_code_bytes(HD) + g * 128 + t * 16);
                    const uint4 b = *reinterpret_cast<const uint4 *>(vt + q4_code_bytes(HD) + g * 128 + 64 + t * 16);
                    const uint4 w = *reinterpret_cast<const uint4 *>(vt + ((g * 8 + e) * 4 + t) * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int half = 0; half < 2; ++half) {  // dimensions 32 g + 16 half + e and + 8
                        uint32_t v0[4], v1[4];
                        q4_values(words[2 * half], bits_h2(d.x), bits_h2(b.x), bits_h2(d.y), bits_h2(b.y), bits_h2(d.z),
                                  bits_h2(b.z), bits_h2(d.w), bits_h2(b.w), v0);
                        q4_values(words[2 * half + 1], bits_h2(d.x), bits_h2(b.x), bits_h2(d.y), bits_h2(b.y), bits_h2(d.z),
                                  bits_h2(b.z), bits_h2(d.w), bits_h2(b.w), v1);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16(o[nt][2 * g + half], v0[0], v1[0], v0[1], v1[1], x[nt][tile][0], x[nt][tile][1]);
                            mma_f16(o[nt][2 * g + half], v0[2], v1[2], v0[3], v1[3], x[nt][tile][2], x[nt][tile][3]);
                        }
                    }
                }
            }
            // (the last product has been issued, so its operands have arrived: every read of the values is behind this warp)
            request_next(true);
            phase ^= 1;
        }

        // the four warps' results to one
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[nt] += __shfl_xor_sync(0xFFFFFFFFu, l[nt], w);
            if (e == 0) merge_ml[warp * KR + nt * 4 + t] = make_float2(m[nt], l[nt]);
        }
        __syncthreads();
        float share[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kAqWarps; ++w) top = fmaxf(top, merge_ml[w * KR + nt * 4 + t].x);
            share[nt] = m[nt] == -INFINITY ? 0.0f : ex2(m[nt] - top);
        }
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += MD) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int d = 0; d < MD / 16; ++d) {
                    const float(&c)[4] = o[nt][d0 / 16 + d];
                    float *to = &merge[(warp * KR + nt * 4 + t) * PAD + 16 * d + e];
                    to[0] = (c[0] + c[1]) * share[nt];
                    to[8] = (c[2] + c[3]) * share[nt];
                }
            __syncthreads();
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int row = (threadIdx.x + n * kAqThreads) / RL, d = threadIdx.x % RL * 4;
                if (row >= KR || row_last[n] < it.chunk * it.span) continue;  // no row, or one that ends before
                float mm = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kAqWarps; ++w) mm = fmaxf(mm, merge_ml[w * KR + row].x);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kAqWarps; ++w) {
                    const float2 ml = merge_ml[w * KR + row];
                    sum += ml.x == -INFINITY ? 0.0f : ml.y * ex2(ml.x - mm);
                    const float4 u = *reinterpret_cast<const float4 *>(&merge[(w * KR + row) * PAD + d]);
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                }
                if (row_last[n] < it.span) {  // the row's only chunk
                    const float inv = 1.0f / sum;
                    *reinterpret_cast<float4 *>(p.out + row_out[n] * HD + d0 + d) =
                        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                } else {
                    const int64_t pc = row_out[n] * p.max_chunks + it.chunk;
                    *reinterpret_cast<float4 *>(p.part + pc * HD + d0 + d) = v;
                    if (d0 == 0 && d == 0) *reinterpret_cast<float2 *>(p.part_ml + pc * 2) = make_float2(mm, sum);
                }
            }
            __syncthreads();
        }
        if (Fused && it.chunks > 1) {
            // the CTA that finishes the last chunk of these rows joins them
            __threadfence();
            __syncthreads();
            int *done = p.done + (it.s * src.KVH + it.h) * p.groups + it.mt;
            if (threadIdx.x == 0) last_one = atomicAdd(done, 1) == it.chunks - 1;
            __syncthreads();
            if (last_one) {
                if (threadIdx.x == 0) *done = 0;  // as it was found
                __threadfence();
                constexpr int GL = AqJoin<HD>::GL;
#pragma unroll 1
                for (int g = threadIdx.x / GL; g < (KR * GL + 31) / 32 * 32 / GL; g += kAqThreads / GL) {
                    const int i = it.mt * KR + g, r = i / G;
                    const int chunks = g < KR && r < it.count ? (it.pos + r) / it.span + 1 : 0;
                    aq_join_few<HD>(p, ((int64_t)it.s * src.rows + r) * p.H + it.h * G + (i - r * G), chunks > 1 ? chunks : 0);
                }
            }
        }
        it = next;
    }
}

// Few chunks: the rows of a call, a group of lanes each.
template <int HD>
__global__ void __launch_bounds__(kAqJoinThreads) attention_q4_join_few_kernel(const AqParams p) {
    constexpr int GL = AqJoin<HD>::GL;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row = ((int64_t)blockIdx.x * kAqJoinThreads + threadIdx.x) / GL;
    const int rows = p.src.rows;
    int chunks = 0;
    if (row < (int64_t)p.src.n_seq * rows * p.H) {
        const int s = (int)(row / ((int64_t)rows * p.H)), r = (int)(row / p.H % rows);
        if (!aq_join_of(p, s, r, &chunks)) chunks = 0;
    }
    aq_join_few<HD>(p, row, chunks);
}

// Many chunks: a CTA a row, a group of threads a class.
template <int HD>
__global__ void __launch_bounds__(HD / 4 * kAqClasses) attention_q4_join_kernel(const AqParams p) {
    constexpr int TC = HD / 4;
    __shared__ float4 sv[kAqClasses][TC];
    __shared__ float sl[kAqClasses];
    pdl_wait();
    pdl_launch_dependents();
    const int rows = p.src.rows, c0 = threadIdx.x / TC, d = threadIdx.x % TC;
    const size_t row = blockIdx.x;
    const int s = (int)(row / ((size_t)rows * p.H)), r = (int)(row / p.H % rows);
    int chunks;
    if (!aq_join_of(p, s, r, &chunks)) return;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + row * p.max_chunks;
    const float4 *part = reinterpret_cast<const float4 *>(p.part) + row * p.max_chunks * TC + d;
    float top = -INFINITY;
    for (int c = threadIdx.x & 31; c < chunks; c += 32) top = fmaxf(top, ml[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 8
    for (int c = c0; c < chunks; c += kAqClasses) {
        const float2 x = ml[c];
        const float4 u = part[(size_t)c * TC];
        const float k = ex2(x.x - top);
        l += x.y * k;
        v.x += u.x * k, v.y += u.y * k, v.z += u.z * k, v.w += u.w * k;
    }
    sv[c0][d] = v;
    if (d == 0) sl[c0] = l;
    __syncthreads();
    if (c0 == 0) {
        for (int i = 1; i < kAqClasses; ++i) {
            const float4 u = sv[i][d];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            l += sl[i];
        }
        const float inv = 1.0f / l;
        reinterpret_cast<float4 *>(p.out)[row * TC + d] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

template <int HD>
static cudaError_t launch_aq_join(const AqParams &p, cudaStream_t st) {
    if (p.max_chunks <= kAqJoinFew) {
        const int64_t threads = (int64_t)p.src.n_seq * p.src.rows * p.H * (HD < 128 ? HD / 4 : 32);
        return launch_pdl(attention_q4_join_few_kernel<HD>, dim3((unsigned)((threads + kAqJoinThreads - 1) / kAqJoinThreads)),
                          dim3(kAqJoinThreads), 0, st, true, p);
    }
    return launch_pdl(attention_q4_join_kernel<HD>, dim3((unsigned)((int64_t)p.src.n_seq * p.src.rows * p.H)),
                      dim3(HD / 4 * kAqClasses), 0, st, true, p);
}

static int aq_max_chunks(int max_ctx) { return (max_ctx + kAqLeaf - 1) / kAqLeaf; }

int64_t attn_q4_scratch_bytes(int n_seq, int rows, int H, int hd, int max_ctx) {
    return 4 * kAqCounters + (int64_t)4 * n_seq * rows * H * aq_max_chunks(max_ctx) * (hd + 2);
}

// Scratch of launch_attention_q4_rows for up to `rows` rows, `few` at a time where they go to attention_q4_kernel.
int64_t attn_q4_rows_scratch_bytes(int rows, int few, int H, int KVH, int hd, int max_ctx, int sms) {
    int64_t most = attn_q4_scratch_bytes(1, std::min(rows, few), H, hd, max_ctx);
    for (int r = OVF_Q4_EXACT_ROWS + 1; r <= rows && hd <= 128; ++r)
        most = std::max(most, attn_q4_many_rows(1, r, H, KVH, hd, max_ctx, sms)
                                  ? 4 * kAqCounters + (int64_t)4 * r * H * attn_q4_rows_splits(1, r, H, KVH, max_ctx, sms) * (hd + 2)
                                  : attn_q4_scratch_bytes(1, r, H, hd, max_ctx));
    return most;
}

template <int NG, int NT>
static cudaError_t launch_aq(AqParams p, cudaStream_t st, bool pdl) {
    using S = AqShape<NG, NT>;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (once.pending(dev)) {
        cudaError_t e = cudaFuncSetAttribute(attention_q4_kernel<NG, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             S::kTotal);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attention_q4_kernel<NG, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal);
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    const int64_t rows = (int64_t)p.src.rows * (p.H / p.src.KVH);
    const int64_t most = (int64_t)p.src.n_seq * p.src.KVH * ((rows + S::kRows - 1) / S::kRows) * p.max_chunks;
    // One launch where the counters have room for every group of rows and a row has few chunks: calls so small that
    // launching takes the host longer than they take the device (one decoded token of 32 heads over 8 at 2048
    // positions, called from Python: 13.7 us with a second kernel, 11.5 us without; on the device they are alike).
    p.groups = (int)((rows + S::kRows - 1) / S::kRows);
    const bool fused = p.max_chunks > 1 && p.max_chunks <= kAqJoinFew &&
                       (int64_t)p.src.n_seq * p.src.KVH * p.groups <= kAqCounters;
    const int64_t room = (int64_t)sm_count(dev) * (fused ? 2 : S::kCtas);
    const dim3 grid((unsigned)std::min(most, room));
    if (fused) return launch_pdl(attention_q4_kernel<NG, NT, true>, grid, dim3(kAqThreads), S::kTotal, st, pdl, p);
    const cudaError_t e = launch_pdl(attention_q4_kernel<NG, NT, false>, grid, dim3(kAqThreads), S::kTotal, st, pdl, p);
    if (e != cudaSuccess || p.max_chunks == 1) return e;
    return launch_aq_join<NG * 32>(p, st);
}

ovf_status launch_attention_q4(const Q4Source &src, int H, int hd, const float *q, float *out, float scale,
                               void *scratch, cudaStream_t st, bool pdl) {
    AqParams p{};
    p.src = src;
    p.H = H;
    p.q = q;
    p.out = out;
    p.scale2 = scale * 1.44269504088896340736f;
    p.max_chunks = aq_max_chunks(src.max_ctx);
    p.done = static_cast<int *>(scratch);
    p.part = static_cast<float *>(scratch) + kAqCounters;
    p.part_ml = p.part + (size_t)src.n_seq * src.rows * H * p.max_chunks * hd;
    cudaError_t e = cudaSuccess;
    const int sms = sm_count(current_device());
    if (attn_q4_many_rows(src.n_seq, src.rows, H, src.KVH, hd, src.max_ctx, sms)) {
        p.splits = attn_q4_rows_splits(src.n_seq, src.rows, H, src.KVH, src.max_ctx, sms);
        p.max_chunks = p.splits;
        p.part_ml = p.part + (size_t)src.n_seq * src.rows * H * p.splits * hd;
        const ArParams a{src, H, q, out, p.part, p.part_ml, p.scale2, p.splits};
        e = hd == 32 ? launch_ar<1>(a, st) : hd == 64 ? launch_ar<2>(a, st) : launch_ar<4>(a, st);
        if (e != cudaSuccess || p.splits == 1) return cuda_status(e, "attention_q4");
        e = hd == 32 ? launch_aq_join<32>(p, st) : hd == 64 ? launch_aq_join<64>(p, st) : launch_aq_join<128>(p, st);
        return cuda_status(e, "attention_q4");
    }
    // two operands share the cache's where there are rows for them (and registers)
    const bool two = (int64_t)src.rows * (H / src.KVH) > 4 && hd < 256;
#define OVF_CALL(NG) e = two ? launch_aq<NG, NG < 8 ? 2 : 1>(p, st, pdl) : launch_aq<NG, 1>(p, st, pdl)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(e, "attention_q4");
}

ovf_status launch_attention_q4_rows(const Q4Source &src, int H, int hd, const float *q, float *out, float scale,
                                    void *scratch, int scratch_rows, bool exact, cudaStream_t st) {
    if (!exact && hd <= 128) return launch_attention_q4(src, H, hd, q, out, scale, scratch, st, false);
    for (int r = 0; r < src.rows; r += scratch_rows) {
        Q4Source part = src;
        part.pos0 = src.pos0 + r;
        part.rows = std::min(scratch_rows, src.rows - r);
        const size_t at = (size_t)r * H * hd;
        const ovf_status e = launch_attention_q4(part, H, hd, q + at, out + at, scale, scratch, st, false);
        if (e) return e;
    }
    return OVF_OK;
}

}  // namespace ovf

extern "C" {

int64_t ovf_attention_q4_scratch_bytes(int32_t n_seq, int32_t rows, int32_t n_heads, int32_t n_kv_heads,
                                       int32_t head_dim, int32_t max_ctx) {
    if (n_seq <= 0 || rows <= 0 || n_heads <= 0 || n_kv_heads <= 0 || max_ctx <= 0 || !ovf::q4_supported(head_dim)) return 0;
    return ovf::attn_q4_scratch_bytes(n_seq, rows, n_heads, head_dim, max_ctx);
}

ovf_status ovf_attention_q4(const float *q, const float *k_new, const float *v_new, void *k_cache, void *v_cache,
                            float *out, const int32_t *positions, const int32_t *row_counts, int32_t n_seq,
                            int32_t rows, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_ctx,
                            const float *rope_cos, const float *rope_sin, int32_t split_half, float scale,
                            void *scratch, void *stream) {
    using namespace ovf;
    Q4Source src;
    ovf_status st = q4_source("attention_q4", k_cache, v_cache, positions, row_counts, n_seq, rows, n_kv_heads,
                              head_dim, max_ctx, rope_cos, rope_sin, split_half, &src);
    if (st) return st;
    OVF_CHECK_ARG(n_heads > 0 && n_heads <= 65535 && n_heads % n_kv_heads == 0,
                  "attention_q4: n_heads %d must be a multiple of n_kv_heads %d (at most 65535)", n_heads, n_kv_heads);
    if (n_seq == 0 || rows == 0) return OVF_OK;
    OVF_CHECK_ARG(q && out && scratch, "attention_q4: null buffer");
    OVF_CHECK_ARG(aligned16(q) && aligned16(out) && aligned16(scratch), "attention_q4: buffers must be 16-byte aligned");
    OVF_CHECK_ARG(q != out, "attention_q4: the output must not be the query");
    OVF_CHECK_ARG(!k_new == !v_new, "attention_q4: k_new and v_new go together");
    OVF_CHECK_ARG((int64_t)rows * n_heads <= (1 << 22), "attention_q4: %d rows of %d heads in one call (at most 2^22 in all)",
                  rows, n_heads);
    // (as many partial results as an int counts: more need hundreds of GB of scratch)
    OVF_CHECK_ARG((int64_t)n_seq * rows * n_heads <= INT32_MAX / aq_max_chunks(max_ctx),
                  "attention_q4: %d sequences of %d rows of %d heads over %d positions are too many for one call", n_seq, rows,
                  n_heads, max_ctx);
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (k_new) {
        OVF_CHECK_ARG(k_cache != v_cache, "attention_q4: keys and values need caches of their own");
        OVF_CHECK_ARG(aligned16(k_new) && aligned16(v_new) && aligned16(rope_cos) && aligned16(rope_sin),
                      "attention_q4: new rows and rope tables must be 16-byte aligned");
        if ((st = launch_kv_q4_append(src, head_dim, k_new, v_new, s, false))) return st;
    }
    return launch_attention_q4(src, n_heads, head_dim, q, out, scale, scratch, s, false);
}

}  // extern "C"
