// ovf_q4.cuh — the 4-bit KV cache: its format, and the device helpers that
// the kernels which write, read and attend over it share.
//
// Every 32 consecutive dimensions of a head vector (a group) share two fp16
// numbers D and M, and an element is a code c of 0..15 that stands for
//     value(c) = fp16(D * (1 + c / 16) + M),                 rounded once.
// 1 + c / 16 is the fp16 whose exponent is that of 1 and whose top four
// mantissa bits are c, so a pair of codes becomes a pair of values with one
// logic operation and one fused multiply-add; with the usual "d * c + m" the
// code would first have to be converted.  D spans the group's range
// (16/15 * (max - min)) and M is min - D; 5 bits per element in all.  The
// values are fp16 numbers by definition, so they enter the tensor cores
// exactly.
//
// A cache holds one side (keys or values) of one layer of one sequence:
// [kv head][tile of 32 positions][20 * head_dim bytes].  A tile is one
// contiguous piece, so that it moves with one bulk copy, and its words are in
// the order in which the lanes of a warp take them as matrix operands:
//   word    eight codes, code i at bits 4 i + 2 (mod 32): pair (i, i + 4) is
//           shifted into the two halves' mantissas together;
//   key     [position 32][t 4][group] words, dimension 32 group + 8 t + i,
//           then [position 32][group] pairs (D, M): lane 4 e + t reads its
//           words of one position in one load;
//   value   [group][e 8][t 4][n 4] words, dimension 32 group + 8 n + e,
//           position 8 t + i, then [group][D, M][t 4][8] halves, positions in
//           the order 0 4 1 5 2 6 3 7 (the order of the pairs).
#pragma once

#include "ovf_internal.cuh"

namespace ovf {

constexpr int kQ4Tile = 32;    // positions of a tile
constexpr int kQ4Group = 32;   // dimensions that share D and M
constexpr float kQ4Limit = 16384.0f;  // larger magnitudes saturate: D and M stay finite in fp16

__host__ __device__ constexpr int q4_tile_bytes(int hd) { return 20 * hd; }
__host__ __device__ constexpr int q4_code_bytes(int hd) { return 16 * hd; }  // D and M follow the codes of a tile
__host__ __device__ constexpr int q4_tiles(int max_ctx) { return (max_ctx + kQ4Tile - 1) / kQ4Tile; }

// Word index of a key's codes: position p of the tile, dimensions 32 g + 8 t ..
__device__ __forceinline__ int q4_key_word(int ng, int p, int t, int g) { return (p * 4 + t) * ng + g; }
// Half index (behind the codes) of a key's D; M follows.
__device__ __forceinline__ int q4_key_param(int ng, int p, int g) { return 2 * (p * ng + g); }
// Word index of a value's codes: dimension 32 g + 8 n + e, positions 8 t ..
__device__ __forceinline__ int q4_value_word(int g, int e, int t, int n) { return ((g * 8 + e) * 4 + t) * 4 + n; }
// Half index of a value's D at position 8 t + i; M is 32 halves further.
__device__ __forceinline__ int q4_value_param(int g, int t, int i) { return g * 64 + t * 8 + 2 * (i & 3) + (i >> 2); }

// D and M of a group of smallest and largest element lo and hi.  Each step is
// rounded by itself (no contraction), so that they, and the codes
// clamp(rint(((x - M) - D) * inv), 0, 15), are the same wherever the definition
// is computed in fp32.
struct Q4Params {
    __half D, M;
    float d, m, inv;
};
__device__ __forceinline__ float q4_clean(float x) {  // NaN is stored as 0; large magnitudes saturate
    return x != x ? 0.0f : fminf(fmaxf(x, -kQ4Limit), kQ4Limit);
}
__device__ __forceinline__ Q4Params q4_params(float lo, float hi) {
    Q4Params p;
    p.D = __float2half_rn(fmul(fsub(hi, lo), 16.0f / 15.0f));
    p.d = __half2float(p.D);
    p.M = __float2half_rn(fsub(lo, p.d));
    p.m = __half2float(p.M);
    p.inv = p.d > 0.0f ? fdiv(16.0f, p.d) : 0.0f;
    return p;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// Pair i (codes i and i + 4) of a word as two fp16 numbers 1 + c / 16.
template <int I>
__device__ __forceinline__ __half2 q4_pair(uint32_t w) {
    const uint32_t s = I == 0 ? w << 4 : I == 1 ? w : I == 2 ? w >> 4 : __funnelshift_r(w, w, 8);
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x03C003C0, 0x3C003C00, 0xEA;" : "=r"(r) : "r"(s));  // (s & mask) | ones
    return bits_h2(r);
}

// The values of eight codes that share D and M (keys) or have a pair each (values).
__device__ __forceinline__ void q4_values(uint32_t w, __half2 d0, __half2 m0, __half2 d1, __half2 m1, __half2 d2, __half2 m2,
                                          __half2 d3, __half2 m3, uint32_t (&v)[4]) {
    v[0] = h2_bits(__hfma2(d0, q4_pair<0>(w), m0));
    v[1] = h2_bits(__hfma2(d1, q4_pair<1>(w), m1));
    v[2] = h2_bits(__hfma2(d2, q4_pair<2>(w), m2));
    v[3] = h2_bits(__hfma2(d3, q4_pair<3>(w), m3));
}

// The cache of one sequence, for a batch of sessions whose caches are apart.
struct Q4Seq {
    uint8_t *k, *v;       // layer 0
    int64_t layer_bytes;  // from one layer to the next
    const float *cos, *sin;
    int32_t pos, max_ctx;
};

// Where the sequences of a launch are: `seqs` (device memory) for sessions, or
// caches one behind the other.  positions[s] (pos0 where there are none) is what
// sequence s holds before its rows, counts[s] (or all `rows`) how many of its
// rows are real; a negative position marks an unused place.
struct Q4Source {
    const Q4Seq *seqs;
    int layer;
    uint8_t *k, *v;
    int64_t seq_bytes;
    const int32_t *positions, *counts;
    const float *cos, *sin;  // [max_ctx][hd / 2] or null
    int split_half, max_ctx, rows, n_seq, KVH, pos0;
    bool callers;  // positions and counts are a kernel-level caller's data
};

struct Q4View {
    uint8_t *k, *v;
    const float *cos, *sin;
    int pos, count, tiles;  // tiles of one head
};

// Sequence s; false if nothing is to be done for it.  Rows that do not fit
// the cache set the caller's error word (a session's, which the host has checked,
// the library's own) and are left out.
__device__ __forceinline__ bool q4_view(const Q4Source &p, int s, Q4View *w) {
    int max_ctx = p.max_ctx;
    if (p.seqs) {
        const Q4Seq q = p.seqs[s];
        w->k = q.k + q.layer_bytes * p.layer;
        w->v = q.v + q.layer_bytes * p.layer;
        w->cos = q.cos;
        w->sin = q.sin;
        w->pos = q.pos;
        max_ctx = q.max_ctx;
    } else {
        w->k = p.k + p.seq_bytes * s;
        w->v = p.v + p.seq_bytes * s;
        w->cos = p.cos;
        w->sin = p.sin;
        w->pos = p.positions ? p.positions[s] : p.pos0;
    }
    w->tiles = q4_tiles(max_ctx);
    w->count = p.counts ? min(max(p.counts[s], 0), p.rows) : p.rows;
    if (w->pos < 0 || w->count == 0) return false;
    if (w->pos > max_ctx - w->count) {
        if (p.callers) raise_caller_error(DEVERR_POSITION);
        else raise_dev_error(DEVERR_POSITION);
        return false;
    }
    return true;
}

// ovf_kv_q4.cu
bool q4_supported(int hd);
ovf_status q4_source(const char *what, const void *k_cache, const void *v_cache, const int32_t *positions,
                     const int32_t *row_counts, int32_t n_seq, int32_t rows, int32_t n_kv_heads, int32_t head_dim,
                     int32_t max_ctx, const float *rope_cos, const float *rope_sin, int32_t split_half, Q4Source *src);
ovf_status launch_kv_q4_append(const Q4Source &src, int hd, const float *k, const float *v, cudaStream_t st, bool pdl);
ovf_status launch_kv_q4_read(const Q4Source &src, int hd, float *k, float *v, cudaStream_t st);
// ovf_attn_q4.cu: rows of queries over the 4-bit cache; `scratch` of
// attn_q4_scratch_bytes.
int64_t attn_q4_scratch_bytes(int n_seq, int rows, int H, int hd, int max_ctx);
ovf_status launch_attention_q4(const Q4Source &src, int H, int hd, const float *q, float *out, float scale,
                               void *scratch, cudaStream_t st, bool pdl);
// Rows of one sequence at pos0 ..; `exact`, or at head_dim 256, `scratch_rows`
// (OVF_Q4_EXACT_ROWS at most) at a time, so that they get the results of single
// rows, bit for bit, and a long context's scratch (attn_q4_rows_scratch_bytes)
// stays small.
int64_t attn_q4_rows_scratch_bytes(int rows, int few, int H, int KVH, int hd, int max_ctx, int sms);
ovf_status launch_attention_q4_rows(const Q4Source &src, int H, int hd, const float *q, float *out, float scale,
                                    void *scratch, int scratch_rows, bool exact, cudaStream_t st);

}  // namespace ovf
