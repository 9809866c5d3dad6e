// ovf_kv_q4.cu — rows of keys and values into the 4-bit cache, and back.
//
// Append: RoPE of the keys (Rope/RopeKernel.cs:46-93), then every group of 32
// dimensions is quantised (ovf_q4.cuh).  A value word holds eight positions of
// one dimension, so a warp owns a block of eight positions of one head: it
// reads the block's words, replaces the codes of the positions that are
// appended and writes them once, and no two warps write the same word.
// Positions outside the rows keep their codes and parameters.
// Bound by memory: 8 bytes read and 1.25 written per element pair.
#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kKvQ4Warps = 4;

// Rows of sequence `s` that lie in the 8-position block of this warp:
// positions [p0, p1), block first position b0.
struct Q4Block {
    int b0, p0, p1;
};
__device__ __forceinline__ bool q4_block(const Q4View &w, int blk, Q4Block *b) {
    b->b0 = ((w.pos >> 3) + blk) * 8;
    b->p0 = max(w.pos, b->b0);
    b->p1 = min(w.pos + w.count, b->b0 + 8);
    return b->p0 < b->p1;
}

template <int NG>
__global__ void __launch_bounds__(kKvQ4Warps * 32) kv_q4_append_kernel(const Q4Source src, const float *k,
                                                                      const float *v) {
    constexpr int HD = NG * 32;
    const int lane = threadIdx.x & 31;
    const int h = blockIdx.y >> 1, s = blockIdx.z;
    const bool values = blockIdx.y & 1;
    Q4View w;
    Q4Block b;
    if (!q4_view(src, s, &w) || !q4_block(w, blockIdx.x * kKvQ4Warps + (threadIdx.x >> 5), &b)) return;
    uint8_t *tile = (values ? w.v : w.k) + ((size_t)h * w.tiles + b.b0 / kQ4Tile) * q4_tile_bytes(HD);
    uint32_t *words = reinterpret_cast<uint32_t *>(tile);
    __half *params = reinterpret_cast<__half *>(tile + q4_code_bytes(HD));
    const int t = (b.b0 & 31) >> 3;
    const float *x0 = (values ? v : k) + ((size_t)s * src.rows * src.KVH + h) * HD + lane;
    uint32_t old[NG];
    if (values) {
#pragma unroll
        for (int g = 0; g < NG; ++g) old[g] = words[q4_value_word(g, lane & 7, t, lane >> 3)];
    }
    for (int p = b.p0; p < b.p1; ++p) {
        float x[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) x[g] = x0[(size_t)(p - w.pos) * src.KVH * HD + g * 32];
        if (!values && w.cos)
            q4_rotate<NG>(x, w.cos + (size_t)p * (HD / 2), w.sin + (size_t)p * (HD / 2), src.split_half, lane);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float y = q4_clean(x[g]);
            float lo = y, hi = y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
            }
            const Q4Params q = q4_params(lo, hi);
            const uint32_t c = q4_encode(y, q);
            if (values) {
                old[g] = q4_with_code(old[g], p & 7, c);
                if (lane == 0) {
                    const int i = q4_value_param(g, t, p & 7);
                    params[i] = q.D;
                    params[i + 32] = q.M;
                }
            } else {
                // lanes 8 t .. 8 t + 7 hold the codes of one word
                uint32_t u = __funnelshift_l(c, c, q4_shift(lane & 7));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) u |= __shfl_xor_sync(0xFFFFFFFFu, u, o);
                if ((lane & 7) == 0) words[q4_key_word(NG, p & 31, lane >> 3, g)] = u;
                if (lane == 0) *reinterpret_cast<__half2 *>(params + q4_key_param(NG, p & 31, g)) = __halves2half2(q.D, q.M);
            }
        }
    }
    if (values) {
#pragma unroll
        for (int g = 0; g < NG; ++g) words[q4_value_word(g, lane & 7, t, lane >> 3)] = old[g];
    }
}

template <int NG>
__global__ void __launch_bounds__(kKvQ4Warps * 32) kv_q4_read_kernel(const Q4Source src, float *k, float *v) {
    constexpr int HD = NG * 32;
    const int lane = threadIdx.x & 31;
    const int h = blockIdx.y >> 1, s = blockIdx.z;
    const bool values = blockIdx.y & 1;
    Q4View w;
    Q4Block b;
    if (!q4_view(src, s, &w) || !q4_block(w, blockIdx.x * kKvQ4Warps + (threadIdx.x >> 5), &b)) return;
    const uint8_t *tile = (values ? w.v : w.k) + ((size_t)h * w.tiles + b.b0 / kQ4Tile) * q4_tile_bytes(HD);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(tile);
    const __half *params = reinterpret_cast<const __half *>(tile + q4_code_bytes(HD));
    const int t = (b.b0 & 31) >> 3;
    float *y0 = (values ? v : k) + ((size_t)s * src.rows * src.KVH + h) * HD + lane;
    for (int p = b.p0; p < b.p1; ++p) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t c;
            __half D, M;
            if (values) {
                c = q4_code(words[q4_value_word(g, lane & 7, t, lane >> 3)], p & 7);
                D = params[q4_value_param(g, t, p & 7)];
                M = params[q4_value_param(g, t, p & 7) + 32];
            } else {
                c = q4_code(words[q4_key_word(NG, p & 31, lane >> 3, g)], lane & 7);
                D = params[q4_key_param(NG, p & 31, g)];
                M = params[q4_key_param(NG, p & 31, g) + 1];
            }
            y0[(size_t)(p - w.pos) * src.KVH * HD + g * 32] = q4_value(c, D, M);
        }
    }
}

bool q4_supported(int hd) { return hd == 32 || hd == 64 || hd == 128 || hd == 256; }

static dim3 kv_q4_grid(const Q4Source &src) {
    const int blocks = (src.rows + 14) / 8;  // rows that start anywhere in a block
    return dim3((blocks + kKvQ4Warps - 1) / kKvQ4Warps, src.KVH * 2, src.n_seq);
}

#define OVF_Q4_HD(hd, CALL)              \
    switch (hd) {                        \
        case 32: CALL(1); break;         \
        case 64: CALL(2); break;         \
        case 128: CALL(4); break;        \
        default: CALL(8); break;         \
    }

ovf_status launch_kv_q4_append(const Q4Source &src, int hd, const float *k, const float *v, cudaStream_t st) {
    const dim3 grid = kv_q4_grid(src);
#define OVF_CALL(NG) kv_q4_append_kernel<NG><<<grid, kKvQ4Warps * 32, 0, st>>>(src, k, v)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(cudaGetLastError(), "kv_q4_append");
}

ovf_status launch_kv_q4_read(const Q4Source &src, int hd, float *k, float *v, cudaStream_t st) {
    const dim3 grid = kv_q4_grid(src);
#define OVF_CALL(NG) kv_q4_read_kernel<NG><<<grid, kKvQ4Warps * 32, 0, st>>>(src, k, v)
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
    OVF_CHECK_ARG(k_cache && v_cache && positions, "%s: null buffer", what);
    OVF_CHECK_ARG(aligned16(k_cache) && aligned16(v_cache), "%s: caches must be 16-byte aligned", what);
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
    if (st) return st;
    OVF_CHECK_ARG(k && v, "kv_q4_append: null buffer");
    OVF_CHECK_ARG(k_cache != v_cache, "kv_q4_append: keys and values need caches of their own");
    if (n_seq == 0 || rows == 0) return OVF_OK;
    return launch_kv_q4_append(src, head_dim, k, v, reinterpret_cast<cudaStream_t>(stream));
}

ovf_status ovf_kv_q4_read(const void *k_cache, const void *v_cache, const int32_t *positions, const int32_t *row_counts,
                          int32_t n_seq, int32_t rows, int32_t n_kv_heads, int32_t head_dim, int32_t max_ctx, float *k,
                          float *v, void *stream) {
    using namespace ovf;
    Q4Source src;
    ovf_status st = q4_source("kv_q4_read", k_cache, v_cache, positions, row_counts, n_seq, rows, n_kv_heads, head_dim,
                              max_ctx, nullptr, nullptr, 0, &src);
    if (st) return st;
    OVF_CHECK_ARG(k && v && k != v, "kv_q4_read: null buffer, or one for both sides");
    if (n_seq == 0 || rows == 0) return OVF_OK;
    return launch_kv_q4_read(src, head_dim, k, v, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
