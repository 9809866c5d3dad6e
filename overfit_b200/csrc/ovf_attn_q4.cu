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
// hi = fp16(x) and lo = fp16(x - hi), which together hold 22 bits.  The 16 rows
// of an operand are the hi and the lo parts of 8 query rows (the heads of one KV
// head, row after row), so a decode step of up to 8 heads per KV head needs no
// product twice; the two halves of a result are added in fp32.  Queries are
// scaled by a power of two into fp16's range, weights by 2^14, both exactly.
//
// Work is cut into chunks of 256 positions, each one softmax pass with a running
// maximum: a CTA's four warps take two tiles of 32 positions each, their partial
// results (maximum, sum, weighted values) are joined in shared memory, and a
// second kernel joins the chunks of a row.  Chunks, tiles and the order of every
// sum go by position alone, so a row's result does not depend on what else is in
// the call, bit for bit.  CTAs stay resident and take equal runs of the chunks
// of all sequences, so that unequal lengths cost nothing.
#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kAqWarps = 4;
static constexpr int kAqThreads = kAqWarps * 32;
static constexpr int kAqChunk = 256;               // positions of a chunk: kAqWarps warps x 2 tiles
static constexpr int kAqRows = 8;                  // query rows of an operand (hi and lo parts)
static constexpr float kAqLift = 14.0f;            // weights are held times 2^14: lo parts stay normal fp16 numbers
static_assert(kAqChunk == kAqWarps * 2 * kQ4Tile, "two tiles a warp");

// CTAs per SM and stages of the tile ring of a warp, by head_dim.
__host__ __device__ constexpr int aq_ctas(int ng) { return ng <= 4 ? 3 : 2; }
__host__ __device__ constexpr int aq_stages(int ng) { return ng <= 2 ? 4 : ng == 4 ? 2 : 2; }

template <int NG>
struct AqSmem {
    static constexpr int HD = NG * 32;
    static constexpr int kTile = 2 * q4_tile_bytes(HD);  // keys, then values
    static constexpr int kRing = kAqWarps * aq_stages(NG) * kTile;
    static constexpr int MD = HD < 128 ? HD : 128;       // dimensions joined at a time
    static constexpr int kMerge = kAqWarps * kAqRows * MD * 4;
    static constexpr int kTotal = kRing + kMerge + kAqWarps * kAqRows * 8 + kAqWarps * aq_stages(NG) * 8;
};

struct AqParams {
    Q4Source src;
    int H;
    const float *q;
    float *out, *part, *part_ml;  // partial results [row][chunk][hd] and (maximum, sum)
    float scale2;                 // scale * log2(e): exponentials are powers of two
    int max_chunks;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Pair i (codes i and i + 4) of a word as two fp16 numbers 1 + c / 16.
template <int I>
__device__ __forceinline__ __half2 q4_pair(uint32_t w) {
    const uint32_t s = I == 0 ? w << 4 : I == 1 ? w : I == 2 ? w >> 4 : __funnelshift_r(w, w, 8);
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x03C003C0, 0x3C003C00, 0xEA;" : "=r"(r) : "r"(s));  // (s & mask) | ones
    return bits_h2(r);
}

// x and y as hi and lo parts, each a pair of fp16.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// The sequences' chunks as one list: per sequence [kv head][operand of 8 rows][chunk].
struct AqItem {
    Q4View w;
    int s, left;               // items of this sequence behind this one
    int chunks, tiles8, chunk, mt, h;  // chunks and operands of the sequence; this item's
};

__device__ __forceinline__ int aq_count(const Q4Source &src, int s, int G) {
    Q4View w;
    if (s >= src.n_seq || !q4_view(src, s, &w)) return 0;
    return src.KVH * ((w.count * G + kAqRows - 1) / kAqRows) * ((w.pos + w.count + kAqChunk - 1) / kAqChunk);
}

// Item `target` of the list that starts with sequence `from`; false if it has fewer.
__device__ __forceinline__ bool aq_locate(const Q4Source &src, int G, int from, long long target, AqItem *it) {
    const int lane = threadIdx.x & 31;
    for (int s0 = from; s0 < src.n_seq; s0 += 32) {
        const int n = aq_count(src, s0 + lane, G);
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
        it->s = s0 + l;
        q4_view(src, it->s, &it->w);
        it->chunks = (it->w.pos + it->w.count + kAqChunk - 1) / kAqChunk;
        it->tiles8 = (it->w.count * G + kAqRows - 1) / kAqRows;
        it->left = items - 1 - local;
        it->chunk = local % it->chunks;
        it->mt = local / it->chunks % it->tiles8;
        it->h = local / it->chunks / it->tiles8;
        return true;
    }
    return false;
}

__device__ __forceinline__ bool aq_next(const Q4Source &src, int G, AqItem *it) {
    if (it->left == 0) return aq_locate(src, G, it->s + 1, 0, it);
    --it->left;
    if (++it->chunk == it->chunks) {
        it->chunk = 0;
        if (++it->mt == it->tiles8) {
            it->mt = 0;
            ++it->h;
        }
    }
    return true;
}

// Positions of the item that any of its rows attends: [256 chunk, end).
__device__ __forceinline__ int aq_end(const AqItem &it, int G) {
    const int last_row = min(it.w.count - 1, (it.mt * kAqRows + kAqRows - 1) / G);
    return min((it.chunk + 1) * kAqChunk, it.w.pos + last_row + 1);
}

template <int NG>
__global__ void __launch_bounds__(kAqThreads, aq_ctas(NG)) attention_q4_kernel(const AqParams p) {
    constexpr int HD = NG * 32, NS = aq_stages(NG), TB = q4_tile_bytes(HD), MD = AqSmem<NG>::MD;
    extern __shared__ __align__(128) uint8_t smem[];
    const Q4Source &src = p.src;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = lane >> 2, t = lane & 3, G = p.H / src.KVH;
    uint8_t *ring = smem + warp * NS * 2 * TB;
    float *merge = reinterpret_cast<float *>(smem + AqSmem<NG>::kRing);                   // [warp][row][MD]
    float2 *merge_ml = reinterpret_cast<float2 *>(merge + kAqWarps * kAqRows * MD);       // [warp][row]
    uint64_t *bars = reinterpret_cast<uint64_t *>(merge_ml + kAqWarps * kAqRows) + warp * NS;
    if (lane < NS) mbar_init(&bars[lane], 1);
    fence_mbar_init();
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();

    // this CTA's run of the list
    long long total = 0;
    for (int s0 = 0; s0 < src.n_seq; s0 += 32) {
        int n = aq_count(src, s0 + lane, G);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
        total += n;
    }
    const long long lo = total * blockIdx.x / gridDim.x;
    int left = (int)(total * (blockIdx.x + 1) / gridDim.x - lo);  // items to compute
    AqItem it, ahead;
    if (left <= 0 || !aq_locate(src, G, 0, lo, &it)) return;
    ahead = it;
    int ahead_left = left, ahead_tile = warp * 2, issued = 0, used = 0;
    bool dead = false;

    // requests this warp's next tile, if its run has one
    auto request = [&]() {
        while (ahead_left > 0) {
            const int p0 = ahead.chunk * kAqChunk + ahead_tile * kQ4Tile;
            if (ahead_tile < warp * 2 + 2 && p0 < aq_end(ahead, G)) break;
            ahead_tile = warp * 2;
            --ahead_left;
            if (ahead_left > 0 && !aq_next(src, G, &ahead)) ahead_left = 0;
        }
        if (ahead_left <= 0) return;
        const int st = issued % NS;
        if (lane == 0) {
            const size_t at = ((size_t)ahead.h * ahead.w.tiles + ahead.chunk * (kAqChunk / kQ4Tile) + ahead_tile) * TB;
            const uint64_t pol = l2_evict_first_policy();
            mbar_arrive_expect_tx(&bars[st], 2 * TB);
            bulk_g2s(ring + st * 2 * TB, ahead.w.k + at, TB, &bars[st], pol);
            bulk_g2s(ring + st * 2 * TB + TB, ahead.w.v + at, TB, &bars[st], pol);
        }
        ++issued;
        ++ahead_tile;
    };
#pragma unroll
    for (int i = 0; i < NS; ++i) request();

    uint32_t a[NG][2][4];  // query operand: [group][step]
    float factor = 0.0f;   // score of this lane's row from its sum of products
    int limit = 0;         // last position that the row attends
    int have_h = -1, have_mt = -1, have_s = -1;

    for (; left > 0; --left) {
        if (it.h != have_h || it.mt != have_mt || it.s != have_s) {
            have_h = it.h, have_mt = it.mt, have_s = it.s;
            const int i = it.mt * kAqRows + e, r = i / G;
            const bool real = r < it.w.count;
            limit = real ? it.w.pos + r : 0x7FFFFFFF;  // (a row that is none: zeros, which nothing reads)
            float x[NG][8];
            if (real) {
                const float4 *q = reinterpret_cast<const float4 *>(
                    p.q + (((size_t)it.s * src.rows + r) * p.H + it.h * G + i % G) * HD + 8 * t);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float4 u = q[g * 8], v = q[g * 8 + 1];
                    x[g][0] = u.x, x[g][1] = u.y, x[g][2] = u.z, x[g][3] = u.w;
                    x[g][4] = v.x, x[g][5] = v.y, x[g][6] = v.z, x[g][7] = v.w;
                }
            } else {
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[g][k] = 0.0f;
            }
            if (it.w.cos) {  // Rope/RopeKernel.cs:46-93, each step rounded by itself
                const int pos = real ? limit : 0;
                const float *c = it.w.cos + (size_t)pos * (HD / 2), *sn = it.w.sin + (size_t)pos * (HD / 2);
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
            factor = p.scale2 * __int_as_float((ex - 14) << 23);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k)  // pair (k, k + 4): registers 0 and 2 of step 0, then of step 1
                    split2(x[g][k] * up, x[g][k + 4] * up, a[g][k >> 1][2 * (k & 1)], a[g][k >> 1][2 * (k & 1) + 1]);
        }

        float m = -INFINITY, l = 0.0f, o[NG * 4][4];
#pragma unroll
        for (int n = 0; n < NG * 4; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[n][k] = 0.0f;
        const int end = aq_end(it, G), data_end = it.w.pos + it.w.count;
        for (int tile = warp * 2; tile < warp * 2 + 2; ++tile) {
            const int p0 = it.chunk * kAqChunk + tile * kQ4Tile;
            if (p0 >= end) break;
            const int st = used % NS;
            if (!dead && !mbar_wait_sleep_bounded(&bars[st], (used / NS) & 1)) dead = true;
            uint8_t *kt = ring + st * 2 * TB, *vt = kt + TB;
            if (p0 + kQ4Tile > data_end) {
                // what lies behind the sequence's data may be anything: its weights
                // are 0, and its values must be numbers for that
                if (p0 + lane >= data_end) {
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
            // scores of this lane's row at positions p0 + 8 t + 2 j and + 1
            float s[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = 8 * (e >> 1) + 2 * j + (e & 1);
                uint32_t kw[NG], kp[NG];
                if (NG == 1) {
                    kw[0] = *reinterpret_cast<const uint32_t *>(kt + (row * 4 + t) * 4);
                    kp[0] = *reinterpret_cast<const uint32_t *>(kt + q4_code_bytes(HD) + row * 4);
                } else if (NG == 2) {
                    *reinterpret_cast<uint2 *>(kw) = *reinterpret_cast<const uint2 *>(kt + (row * 4 + t) * 8);
                    *reinterpret_cast<uint2 *>(kp) = *reinterpret_cast<const uint2 *>(kt + q4_code_bytes(HD) + row * 8);
                } else {
#pragma unroll
                    for (int i = 0; i < NG / 4; ++i) {
                        reinterpret_cast<uint4 *>(kw)[i] = reinterpret_cast<const uint4 *>(kt + (row * 4 + t) * NG * 4)[i];
                        reinterpret_cast<uint4 *>(kp)[i] =
                            reinterpret_cast<const uint4 *>(kt + q4_code_bytes(HD) + row * NG * 4)[i];
                    }
                }
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const __half2 dm = bits_h2(kp[g]), D = __low2half2(dm), M = __high2half2(dm);
                    mma_f16(c, a[g][0], h2_bits(__hfma2(D, q4_pair<0>(kw[g]), M)), h2_bits(__hfma2(D, q4_pair<1>(kw[g]), M)));
                    mma_f16(c, a[g][1], h2_bits(__hfma2(D, q4_pair<2>(kw[g]), M)), h2_bits(__hfma2(D, q4_pair<3>(kw[g]), M)));
                }
                s[j][0] = (c[0] + c[2]) * factor;
                s[j][1] = (c[1] + c[3]) * factor;
            }
            if (__any_sync(0xFFFFFFFFu, p0 + kQ4Tile - 1 > limit)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (p0 + 8 * t + 2 * j + i > limit) s[j][i] = -INFINITY;
            }
            float top = m;
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const float base = top == -INFINITY ? 0.0f : top;  // nothing attended so far: weights of 0
            const float keep = ex2(m - base);
            m = top;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    s[j][i] = ex2(s[j][i] - base + kAqLift);
                    sum += s[j][i];
                }
            l = l * keep + sum;
            if (__any_sync(0xFFFFFFFFu, keep != 1.0f)) {
#pragma unroll
                for (int n = 0; n < NG * 4; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) o[n][k] *= keep;
            }
            // weights as operands: pairs (0, 4) (1, 5), then (2, 6) (3, 7) of positions 8 t ..
            uint32_t w0[4], w1[4];
            split2(s[0][0], s[2][0], w0[0], w0[1]);
            split2(s[0][1], s[2][1], w0[2], w0[3]);
            split2(s[1][0], s[3][0], w1[0], w1[1]);
            split2(s[1][1], s[3][1], w1[2], w1[3]);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint4 dw = *reinterpret_cast<const uint4 *>(vt + q4_code_bytes(HD) + g * 128 + t * 16);
                const uint4 mw = *reinterpret_cast<const uint4 *>(vt + q4_code_bytes(HD) + g * 128 + 64 + t * 16);
                const uint4 cw = *reinterpret_cast<const uint4 *>(vt + ((g * 8 + e) * 4 + t) * 16);
                const uint32_t words[4] = {cw.x, cw.y, cw.z, cw.w};
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    mma_f16(o[g * 4 + n], w0, h2_bits(__hfma2(bits_h2(dw.x), q4_pair<0>(words[n]), bits_h2(mw.x))),
                            h2_bits(__hfma2(bits_h2(dw.y), q4_pair<1>(words[n]), bits_h2(mw.y))));
                    mma_f16(o[g * 4 + n], w1, h2_bits(__hfma2(bits_h2(dw.z), q4_pair<2>(words[n]), bits_h2(mw.z))),
                            h2_bits(__hfma2(bits_h2(dw.w), q4_pair<3>(words[n]), bits_h2(mw.w))));
                }
            }
            __syncwarp();
            ++used;
            request();
        }

        // the four warps' results to one
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
        l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
        if (t == 0) merge_ml[warp * kAqRows + e] = make_float2(m, l);
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAqWarps; ++w) top = fmaxf(top, merge_ml[w * kAqRows + e].x);
        const float share = m == -INFINITY ? 0.0f : ex2(m - top);
#pragma unroll
        for (int d0 = 0; d0 < HD; d0 += MD) {
#pragma unroll
            for (int n = 0; n < MD / 8; ++n) {
                // lane 4 e + t: dimensions 8 n + 2 t and + 1 of row e
                const float(&c)[4] = o[d0 / 8 + n];
                *reinterpret_cast<float2 *>(&merge[(warp * kAqRows + e) * MD + 8 * n + 2 * t]) =
                    make_float2((c[0] + c[2]) * share, (c[1] + c[3]) * share);
            }
            __syncthreads();
            for (int x = threadIdx.x; x < kAqRows * MD / 4; x += kAqThreads) {
                const int row = x / (MD / 4), d = x % (MD / 4) * 4, i = it.mt * kAqRows + row, r = i / G;
                const int row_last = it.w.pos + r;
                if (r >= it.w.count || row_last < it.chunk * kAqChunk) continue;  // no row, or one that ends before
                float mm = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kAqWarps; ++w) mm = fmaxf(mm, merge_ml[w * kAqRows + row].x);
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kAqWarps; ++w) {
                    const float2 ml = merge_ml[w * kAqRows + row];
                    sum += ml.x == -INFINITY ? 0.0f : ml.y * ex2(ml.x - mm);
                    const float4 u = *reinterpret_cast<const float4 *>(&merge[(w * kAqRows + row) * MD + d]);
                    v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
                }
                const size_t orow = ((size_t)it.s * src.rows + r) * p.H + it.h * G + i % G;
                if (row_last < kAqChunk) {  // the row's only chunk
                    const float inv = 1.0f / sum;
                    *reinterpret_cast<float4 *>(p.out + orow * HD + d0 + d) =
                        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                } else {
                    const size_t pc = orow * p.max_chunks + it.chunk;
                    *reinterpret_cast<float4 *>(p.part + pc * HD + d0 + d) = v;
                    if (d0 == 0 && d == 0) *reinterpret_cast<float2 *>(p.part_ml + pc * 2) = make_float2(mm, sum);
                }
            }
            __syncthreads();
        }
        if (left > 1 && !aq_next(src, G, &it)) break;
    }
}

// The chunks of a row to its output: weights 2^(m_c - max), sums over the
// chunks c, c + C, .. by C groups of threads, then over the groups in order.
static constexpr int kAqJoinThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kAqJoinThreads) attention_q4_join_kernel(const AqParams p) {
    constexpr int TC = HD / 4, C = kAqJoinThreads / TC;
    __shared__ float4 sv[C][TC];
    __shared__ float sl[C];
    pdl_wait();
    pdl_launch_dependents();
    const int h = blockIdx.x, r = blockIdx.y, s = blockIdx.z, c0 = threadIdx.x / TC, d = threadIdx.x % TC;
    Q4View w;
    if (!q4_view(p.src, s, &w) || r >= w.count) return;
    const int chunks = (w.pos + r) / kAqChunk + 1;
    if (chunks == 1) return;
    const size_t row = ((size_t)s * p.src.rows + r) * p.H + h;
    const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + row * p.max_chunks;
    const float4 *part = reinterpret_cast<const float4 *>(p.part) + row * p.max_chunks * TC + d;
    float top = -INFINITY;
    for (int c = threadIdx.x & 31; c < chunks; c += 32) top = fmaxf(top, ml[c].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll 4
    for (int c = c0; c < chunks; c += C) {
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
        for (int i = 1; i < C; ++i) {
            const float4 u = sv[i][d];
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
            l += sl[i];
        }
        const float inv = 1.0f / l;
        reinterpret_cast<float4 *>(p.out)[row * TC + d] = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
}

static int aq_max_chunks(int max_ctx) { return (max_ctx + kAqChunk - 1) / kAqChunk; }

int64_t attn_q4_scratch_bytes(int n_seq, int rows, int H, int hd, int max_ctx) {
    return 256 + (int64_t)4 * n_seq * rows * H * aq_max_chunks(max_ctx) * (hd + 2);
}

template <int NG>
static cudaError_t launch_aq(const AqParams &p, cudaStream_t st, bool pdl) {
    constexpr int smem = AqSmem<NG>::kTotal;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (once.pending(dev)) {
        const cudaError_t e =
            cudaFuncSetAttribute(attention_q4_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    const int G = p.H / p.src.KVH;
    const int64_t most = (int64_t)p.src.n_seq * p.src.KVH * ((p.src.rows * (int64_t)G + kAqRows - 1) / kAqRows) * p.max_chunks;
    const int grid = (int)std::min<int64_t>(most, (int64_t)sm_count(dev) * aq_ctas(NG));
    cudaError_t e = launch_pdl(attention_q4_kernel<NG>, dim3(grid), dim3(kAqThreads), smem, st, pdl, p);
    if (e != cudaSuccess || p.max_chunks == 1) return e;
    return launch_pdl(attention_q4_join_kernel<NG * 32>, dim3(p.H, p.src.rows, p.src.n_seq), dim3(kAqJoinThreads), 0, st,
                      true, p);
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
    p.part = static_cast<float *>(scratch);
    p.part_ml = p.part + (size_t)src.n_seq * src.rows * H * p.max_chunks * hd;
    cudaError_t e = cudaSuccess;
#define OVF_CALL(NG) e = launch_aq<NG>(p, st, pdl)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(e, "attention_q4");
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
    OVF_CHECK_ARG(q && out && scratch, "attention_q4: null buffer");
    OVF_CHECK_ARG(aligned16(q) && aligned16(out) && aligned16(scratch), "attention_q4: buffers must be 16-byte aligned");
    OVF_CHECK_ARG(q != out, "attention_q4: the output must not be the query");
    OVF_CHECK_ARG(!k_new == !v_new, "attention_q4: k_new and v_new go together");
    if (n_seq == 0 || rows == 0) return OVF_OK;
    OVF_CHECK_ARG((int64_t)rows * n_heads <= (1 << 22), "attention_q4: %d rows of %d heads in one call (at most 2^22 in all)",
                  rows, n_heads);
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
