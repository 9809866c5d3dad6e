// ovf_kv_q4.cu — rows of keys and values into the 4-bit cache, and back.
//
// Append: RoPE of the keys (Rope/RopeKernel.cs:46-93), then every group of 32
// dimensions is quantised (ovf_q4.cuh).  Keys: a word holds eight dimensions of
// one position, so a lane takes those, the lanes of a group agree on its range
// with two shuffles, and nothing else is shared.  Values: a word holds eight
// positions of one dimension, so a warp takes a group of a block of eight
// positions, a lane a dimension; the range of each position is one redux.  A
// block that the rows fill in part keeps the codes of its other positions.  No
// two warps write the same word.
// Bound by memory: 4 bytes read and 0.625 written per element (reading back: the
// other way round).  Measured, both calls, 8 KV heads of 128: 3.7 us for one row,
// 4.7 for 256, 65 for eight prompts of 2048 (3.6 TB/s, 55 % of the copy rate: the
// quantising and packing instructions, half an SM's issue slots, come first).
#include <algorithm>

#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kKvQ4Threads = 256;

__device__ __forceinline__ float redux_min(float x) {
    float y;
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float redux_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// Whether any of eight elements is NaN or beyond the limit, so that they need q4_clean.
__device__ __forceinline__ bool q4_unclean(const float (&x)[8]) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) bad |= !(fabsf(x[j]) <= kQ4Limit);
    return bad;
}

// The word of eight codes, with the parameters of element j's group from params(j).  A number of 0..15 is rounded to
// an integer (half to even) by adding 1.5 * 2^23, which leaves it in the low bits; what the addend leaves above is
// taken off at the end.
template <class P>
__device__ __forceinline__ uint32_t q4_word(const float (&x)[8], P params) {
    uint32_t word = 0, extra = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float3 p = params(j);  // M, D, 16 / D
        const float c = fminf(fmaxf(fmul(fsub(fsub(x[j], p.x), p.y), p.z), 0.0f), 15.0f);
        word += __float_as_uint(fadd(c, 12582912.0f)) << (4 * j);
        extra += 0x4B400000u << (4 * j);
    }
    word -= extra;
    return __funnelshift_l(word, word, 2);
}

// Keys: a thread takes one word (dimensions 32 g + 8 t ..) of one row of head h.
template <int NG>
__device__ __forceinline__ void append_key(const Q4Source &src, const float *k, const Q4View &w, int s, int h) {
    constexpr int HD = NG * 32;
    const int i = blockIdx.x * kKvQ4Threads + threadIdx.x, r = i / (4 * NG), d = i % (4 * NG) * 8, g = d / 32, t = d / 8 % 4;
    const bool real = r < w.count;
    if (!__any_sync(0xFFFFFFFFu, real)) return;
    const int pos = w.pos + (real ? r : 0);
    float x[8] = {};
    if (real) {
        const float4 *p = reinterpret_cast<const float4 *>(k + (((size_t)s * src.rows + r) * src.KVH + h) * HD + d);
        const float4 u = p[0], v = p[1];
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    }
    if (w.cos) {
        const float *c = w.cos + (size_t)pos * (HD / 2), *sn = w.sin + (size_t)pos * (HD / 2);
        if (!src.split_half) {
            const float4 cc = *reinterpret_cast<const float4 *>(c + d / 2), ss = *reinterpret_cast<const float4 *>(sn + d / 2);
            const float cv[4] = {cc.x, cc.y, cc.z, cc.w}, sv[4] = {ss.x, ss.y, ss.z, ss.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x0 = x[2 * j], x1 = x[2 * j + 1];
                x[2 * j] = fsub(fmul(x0, cv[j]), fmul(x1, sv[j]));
                x[2 * j + 1] = fadd(fmul(x0, sv[j]), fmul(x1, cv[j]));
            }
        } else {
            const int at = d % (HD / 2);
            float cv[8], sv[8];
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
                *reinterpret_cast<float4 *>(cv + j) = *reinterpret_cast<const float4 *>(c + at + j);
                *reinterpret_cast<float4 *>(sv + j) = *reinterpret_cast<const float4 *>(sn + at + j);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float other = __shfl_xor_sync(0xFFFFFFFFu, x[j], NG * 2);  // half a head further
                x[j] = d < HD / 2 ? fsub(fmul(x[j], cv[j]), fmul(other, sv[j])) : fadd(fmul(other, sv[j]), fmul(x[j], cv[j]));
            }
        }
    }
    if (q4_unclean(x)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = q4_clean(x[j]);
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) lo = fminf(lo, x[j]), hi = fmaxf(hi, x[j]);
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {  // the lanes of a group
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
    }
    const Q4Params q = q4_params(lo, hi);
    const uint32_t word = q4_word(x, [&](int) { return make_float3(q.m, q.d, q.inv); });
    if (!real) return;
    uint8_t *tile = w.k + ((size_t)h * w.tiles + pos / kQ4Tile) * q4_tile_bytes(HD);
    reinterpret_cast<uint32_t *>(tile)[q4_key_word(NG, pos & 31, t, g)] = word;
    if (t == 0)
        *reinterpret_cast<__half2 *>(reinterpret_cast<__half *>(tile + q4_code_bytes(HD)) + q4_key_param(NG, pos & 31, g)) =
            __halves2half2(q.D, q.M);
}

// Values: a warp takes group g of the block b of eight positions of head h: rows r0 .. r0 + 7, of which [j0, j1) are real.
struct Q4ValueBlock {
    int b, g, r0, j0, j1;
};
template <int NG>
__device__ __forceinline__ bool q4_value_of(const Q4View &w, Q4ValueBlock *v) {
    const int i = blockIdx.x * (kKvQ4Threads / 32) + (threadIdx.x >> 5);
    v->g = i % NG;
    v->b = (w.pos >> 3) + i / NG;
    v->r0 = v->b * 8 - w.pos;
    v->j0 = max(0, -v->r0);
    v->j1 = min(8, w.count - v->r0);
    return v->r0 < w.count;
}

template <int NG>
__device__ __forceinline__ void append_value(const Q4Source &src, const float *v, const Q4View &w, int s, int h) {
    constexpr int HD = NG * 32;
    __shared__ float4 params[kKvQ4Threads / 32][8];  // M, D, 16 / D of each position
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Q4ValueBlock a;
    if (!q4_value_of<NG>(w, &a)) return;
    const int t = a.b & 3;
    const bool whole = a.j0 == 0 && a.j1 == 8;
    uint8_t *tile = w.v + ((size_t)h * w.tiles + a.b / 4) * q4_tile_bytes(HD);
    uint32_t *word = reinterpret_cast<uint32_t *>(tile) + q4_value_word(a.g, lane & 7, t, lane >> 3);
    const float *x0 = v + (((long long)s * src.rows + a.r0) * src.KVH + h) * HD + a.g * 32 + lane;
    const size_t step = (size_t)src.KVH * HD;
    float x[8];
    if (whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = x0[j * step];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j >= a.j0 && j < a.j1 ? x0[j * step] : 0.0f;
    }
    uint32_t old = 0;
    if (!whole) old = *word;
    if (q4_unclean(x)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = q4_clean(x[j]);
    }
    __syncwarp();
    float lo = 0.0f, hi = 0.0f;  // of position `lane`
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float l = redux_min(x[j]), m = redux_max(x[j]);
        if (lane == j) lo = l, hi = m;
    }
    if (lane < 8) {
        const Q4Params q = q4_params(lo, hi);
        params[warp][lane] = make_float4(q.m, q.d, q.inv, 0.0f);
        if (lane >= a.j0 && lane < a.j1) {
            __half *to = reinterpret_cast<__half *>(tile + q4_code_bytes(HD)) + q4_value_param(a.g, t, lane);
            to[0] = q.D;
            to[32] = q.M;
        }
    }
    __syncwarp();
    uint32_t codes = q4_word(x, [&](int j) {
        const float4 q = params[warp][j];
        return make_float3(q.x, q.y, q.z);
    });
    if (!whole) {
        // the codes of the block's other positions stay: nibbles j0 .. j1 - 1 are ours
        uint32_t ours = (a.j1 == 8 ? 0xFFFFFFFFu : (1u << (4 * a.j1)) - 1u) & ~((1u << (4 * a.j0)) - 1u);
        ours = __funnelshift_l(ours, ours, 2);
        codes = (codes & ours) | (old & ~ours);
    }
    *word = codes;
}

// blockIdx.y: KV head and side
template <int NG>
__global__ void __launch_bounds__(kKvQ4Threads) kv_q4_append_kernel(const Q4Source src, const float *k, const float *v) {
    Q4View w;
    pdl_wait();
    pdl_launch_dependents();
    if (!q4_view(src, blockIdx.z, &w)) return;
    if (blockIdx.y & 1) append_value<NG>(src, v, w, blockIdx.z, blockIdx.y >> 1);
    else append_key<NG>(src, k, w, blockIdx.z, blockIdx.y >> 1);
}

template <int NG>
__global__ void __launch_bounds__(kKvQ4Threads) kv_q4_read_kernel(const Q4Source src, float *k, float *v) {
    constexpr int HD = NG * 32;
    const int s = blockIdx.z, h = blockIdx.y >> 1;
    Q4View w;
    if (!q4_view(src, s, &w)) return;
    uint32_t x[4];  // pairs (i, i + 4)
    if (!(blockIdx.y & 1)) {
        const int i = blockIdx.x * kKvQ4Threads + threadIdx.x, r = i / (4 * NG), d = i % (4 * NG) * 8;
        if (r >= w.count) return;
        const int p = (w.pos + r) & 31;
        const uint8_t *tile = w.k + ((size_t)h * w.tiles + (w.pos + r) / kQ4Tile) * q4_tile_bytes(HD);
        const uint32_t word = reinterpret_cast<const uint32_t *>(tile)[q4_key_word(NG, p, d / 8 % 4, d / 32)];
        const __half2 dm = *reinterpret_cast<const __half2 *>(reinterpret_cast<const __half *>(tile + q4_code_bytes(HD)) +
                                                              q4_key_param(NG, p, d / 32));
        const __half2 D = __low2half2(dm), M = __high2half2(dm);
        q4_values(word, D, M, D, M, D, M, D, M, x);
        const float2 a = __half22float2(bits_h2(x[0])), b = __half22float2(bits_h2(x[1])), c = __half22float2(bits_h2(x[2])),
                     e = __half22float2(bits_h2(x[3]));
        float4 *y = reinterpret_cast<float4 *>(k + (((size_t)s * src.rows + r) * src.KVH + h) * HD + d);
        y[0] = make_float4(a.x, b.x, c.x, e.x);
        y[1] = make_float4(a.y, b.y, c.y, e.y);
        return;
    }
    const int lane = threadIdx.x & 31;
    Q4ValueBlock a;
    if (!q4_value_of<NG>(w, &a)) return;
    const int t = a.b & 3;
    const uint8_t *tile = w.v + ((size_t)h * w.tiles + a.b / 4) * q4_tile_bytes(HD);
    const uint32_t word = reinterpret_cast<const uint32_t *>(tile)[q4_value_word(a.g, lane & 7, t, lane >> 3)];
    const uint4 d = *reinterpret_cast<const uint4 *>(tile + q4_code_bytes(HD) + a.g * 128 + t * 16);
    const uint4 m = *reinterpret_cast<const uint4 *>(tile + q4_code_bytes(HD) + a.g * 128 + 64 + t * 16);
    q4_values(word, bits_h2(d.x), bits_h2(m.x), bits_h2(d.y), bits_h2(m.y), bits_h2(d.z), bits_h2(m.z), bits_h2(d.w),
              bits_h2(m.w), x);
    float *y = v + (((long long)s * src.rows + a.r0) * src.KVH + h) * HD + a.g * 32 + lane;
    const size_t step = (size_t)src.KVH * HD;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(bits_h2(x[j]));
        if (j >= a.j0 && j < a.j1) y[j * step] = f.x;
        if (j + 4 >= a.j0 && j + 4 < a.j1) y[(j + 4) * step] = f.y;
    }
}

bool q4_supported(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

static dim3 kv_q4_grid(const Q4Source &src, int hd) {
    const int64_t keys = (int64_t)src.rows * (hd / 8);                       // words of a head
    const int64_t values = (int64_t)((src.rows + 14) / 8) * (hd / 32) * 32;  // rows may start anywhere in a block
    return dim3((unsigned)((std::max(keys, values) + kKvQ4Threads - 1) / kKvQ4Threads), src.KVH * 2, src.n_seq);
}

#define OVF_Q4_HD(hd, CALL)              \
    switch (hd) {                        \
        case 32: CALL(1); break;         \
        case 64: CALL(2); break;         \
        case 128: CALL(4); break;        \
        default: CALL(8); break;         \
    }

ovf_status launch_kv_q4_append(const Q4Source &src, int hd, const float *k, const float *v, cudaStream_t st, bool pdl) {
    cudaError_t e = cudaSuccess;
#define OVF_CALL(NG) \
    e = launch_pdl(kv_q4_append_kernel<NG>, kv_q4_grid(src, hd), dim3(kKvQ4Threads), 0, st, pdl, src, k, v)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(e, "kv_q4_append");
}

ovf_status launch_kv_q4_read(const Q4Source &src, int hd, float *k, float *v, cudaStream_t st) {
    const dim3 grid = kv_q4_grid(src, hd);
#define OVF_CALL(NG) kv_q4_read_kernel<NG><<<grid, kKvQ4Threads, 0, st>>>(src, k, v)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(cudaGetLastError(), "kv_q4_read");
}

// The checks that the entry points of the 4-bit cache share, and their source.
ovf_status q4_source(const char *what, const void *k_cache, const void *v_cache, const int32_t *positions,
                     const int32_t *row_counts, int32_t n_seq, int32_t rows, int32_t n_kv_heads, int32_t head_dim,
                     int32_t max_ctx, const float *rope_cos, const float *rope_sin, int32_t split_half, Q4Source *src) {
    OVF_CHECK_ARG(q4_supported(head_dim), "%s: head_dim %d unsupported (32, 64, 128 or 256)", what, head_dim);
    OVF_CHECK_ARG(n_seq >= 0 && n_seq <= 65535, "%s: n_seq %d outside [0, 65535]", what, n_seq);
    OVF_CHECK_ARG(n_kv_heads > 0 && n_kv_heads <= 1024, "%s: n_kv_heads %d outside [1, 1024]", what, n_kv_heads);
    OVF_CHECK_ARG(max_ctx > 0 && max_ctx <= (1 << 20), "%s: max_ctx %d outside [1, 2^20]", what, max_ctx);
    OVF_CHECK_ARG(rows >= 0 && rows <= max_ctx, "%s: %d rows do not fit max_ctx %d", what, rows, max_ctx);
    // (a call without rows needs no buffers: empty arrays may have no address)
    OVF_CHECK_ARG(n_seq == 0 || rows == 0 || (k_cache && v_cache && positions), "%s: null buffer", what);
    OVF_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache), "%s: caches must be 16-byte aligned", what);
    OVF_CHECK_ARG((int64_t)rows * n_kv_heads <= (1 << 22), "%s: %d rows of %d heads in one call (at most 2^22 in all)", what,
                  rows, n_kv_heads);
    OVF_CHECK_ARG(!rope_cos == !rope_sin, "%s: rope_cos and rope_sin go together", what);
    Q4Source s{};
    s.k = static_cast<uint8_t *>(const_cast<void *>(k_cache));
    s.v = static_cast<uint8_t *>(const_cast<void *>(v_cache));
    s.seq_bytes = ovf_kv_q4_bytes(n_kv_heads, head_dim, max_ctx);
    s.positions = positions;
    s.counts = row_counts;
    s.cos = rope_cos;
    s.sin = rope_sin;
    s.split_half = split_half != 0;
    s.max_ctx = max_ctx;
    s.rows = rows;
    s.n_seq = n_seq;
    s.KVH = n_kv_heads;
    s.callers = true;
    *src = s;
    return OVF_OK;
}

}  // namespace ovf

extern "C" {

int64_t ovf_kv_q4_bytes(int32_t n_kv_heads, int32_t head_dim, int32_t max_ctx) {
    if (!ovf::q4_supported(head_dim) || n_kv_heads <= 0 || max_ctx <= 0 || max_ctx > (1 << 20)) return 0;
    return (int64_t)n_kv_heads * ovf::q4_tiles(max_ctx) * ovf::q4_tile_bytes(head_dim);
}

ovf_status ovf_kv_q4_append(const float *k, const float *v, void *k_cache, void *v_cache, const int32_t *positions,
                            const int32_t *row_counts, int32_t n_seq, int32_t rows, int32_t n_kv_heads,
                            int32_t head_dim, int32_t max_ctx, const float *rope_cos, const float *rope_sin,
                            int32_t split_half, void *stream) {
    using namespace ovf;
    Q4Source src;
    ovf_status st = q4_source("kv_q4_append", k_cache, v_cache, positions, row_counts, n_seq, rows, n_kv_heads,
                              head_dim, max_ctx, rope_cos, rope_sin, split_half, &src);
    if (st || n_seq == 0 || rows == 0) return st;
    OVF_CHECK_ARG(k && v, "kv_q4_append: null buffer");
    OVF_CHECK_ARG(aligned16(k) && aligned16(v) && aligned16(rope_cos) && aligned16(rope_sin),
                  "kv_q4_append: buffers must be 16-byte aligned");
    OVF_CHECK_ARG(k_cache != v_cache, "kv_q4_append: keys and values need caches of their own");
    return launch_kv_q4_append(src, head_dim, k, v, reinterpret_cast<cudaStream_t>(stream), false);
}

ovf_status ovf_kv_q4_read(const void *k_cache, const void *v_cache, const int32_t *positions, const int32_t *row_counts,
                          int32_t n_seq, int32_t rows, int32_t n_kv_heads, int32_t head_dim, int32_t max_ctx, float *k,
                          float *v, void *stream) {
    using namespace ovf;
    Q4Source src;
    ovf_status st = q4_source("kv_q4_read", k_cache, v_cache, positions, row_counts, n_seq, rows, n_kv_heads, head_dim,
                              max_ctx, nullptr, nullptr, 0, &src);
    if (st || n_seq == 0 || rows == 0) return st;
    OVF_CHECK_ARG(k && v && k != v, "kv_q4_read: null buffer, or one for both sides");
    OVF_CHECK_ARG(aligned16(k) && aligned16(v), "kv_q4_read: buffers must be 16-byte aligned");
    return launch_kv_q4_read(src, head_dim, k, v, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
