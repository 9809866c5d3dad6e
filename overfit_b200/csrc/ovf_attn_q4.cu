// ovf_attn_q4.cu — causal attention of query rows over the 4-bit KV cache.
//
// Row r of sequence s is at position p = positions[s] + r and attends the
// cache's positions [0, p]:  out = sum_j softmax_j(scale * q . K_j) V_j with
// the values that the cache's codes stand for (ovf_q4.cuh) and the query
// rotated at p.  One pass: a running maximum m and sum l of exp(score - m),
// the output rescaled whenever m grows.
#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kAttnQ4Warps = 4;

// One CTA per (row, head, sequence); warp w takes the positions w, w + 4, ..
template <int NG>
__global__ void __launch_bounds__(kAttnQ4Warps * 32) attention_q4_kernel(const Q4Source src, int H, const float *q,
                                                                        float *out, float scale) {
    constexpr int HD = NG * 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.x, h = blockIdx.y, s = blockIdx.z;
    Q4View w;
    if (!q4_view(src, s, &w) || r >= w.count) return;
    const int pos = w.pos + r, g_head = h / (H / src.KVH);
    float x[NG];
    const size_t row = ((size_t)s * src.rows + r) * H * HD + (size_t)h * HD;
#pragma unroll
    for (int g = 0; g < NG; ++g) x[g] = q[row + g * 32 + lane];
    if (w.cos) q4_rotate<NG>(x, w.cos + (size_t)pos * (HD / 2), w.sin + (size_t)pos * (HD / 2), src.split_half, lane);
    float m = -INFINITY, l = 0.0f, o[NG] = {};
    for (int p = warp; p <= pos; p += kAttnQ4Warps) {
        const size_t at = ((size_t)g_head * w.tiles + p / kQ4Tile) * q4_tile_bytes(HD);
        const uint32_t *kw = reinterpret_cast<const uint32_t *>(w.k + at), *vw = reinterpret_cast<const uint32_t *>(w.v + at);
        const __half *kp = reinterpret_cast<const __half *>(w.k + at + q4_code_bytes(HD)),
                     *vp = reinterpret_cast<const __half *>(w.v + at + q4_code_bytes(HD));
        const int i = p & 31;
        float dot = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int kq = q4_key_param(NG, i, g);
            dot += x[g] * q4_value(q4_code(kw[q4_key_word(NG, i, lane >> 3, g)], lane & 7), kp[kq], kp[kq + 1]);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, d);
        const float score = dot * scale, top = fmaxf(m, score);
        const float keep = expf(m - top), e = expf(score - top);
        m = top;
        l = l * keep + e;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int vq = q4_value_param(g, i >> 3, i & 7);
            o[g] = o[g] * keep +
                   e * q4_value(q4_code(vw[q4_value_word(g, lane & 7, i >> 3, lane >> 3)], i & 7), vp[vq], vp[vq + 32]);
        }
    }
    __shared__ float sm[kAttnQ4Warps], sl[kAttnQ4Warps], so[kAttnQ4Warps][HD];
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) so[warp][g * 32 + lane] = o[g];
    __syncthreads();
    float top = sm[0], sum = 0.0f;
    for (int i = 1; i < kAttnQ4Warps; ++i) top = fmaxf(top, sm[i]);
    for (int i = 0; i < kAttnQ4Warps; ++i) sum += sl[i] > 0.0f || sl[i] != sl[i] ? sl[i] * expf(sm[i] - top) : 0.0f;
    for (int d = threadIdx.x; d < HD; d += blockDim.x) {
        float y = 0.0f;
        for (int i = 0; i < kAttnQ4Warps; ++i)
            if (sl[i] > 0.0f || sl[i] != sl[i]) y += so[i][d] * expf(sm[i] - top);
        out[row + d] = y / sum;
    }
}

int64_t attn_q4_scratch_bytes(int n_seq, int rows, int H, int hd, int max_ctx) {
    return 256 + (int64_t)4 * n_seq * rows * H * ((max_ctx + 255) / 256) * (hd + 2);
}

ovf_status launch_attention_q4(const Q4Source &src, int H, int hd, const float *q, float *out, float scale,
                               void *scratch, cudaStream_t st, bool pdl) {
    const dim3 grid(src.rows, H, src.n_seq);
#define OVF_CALL(NG) attention_q4_kernel<NG><<<grid, kAttnQ4Warps * 32, 0, st>>>(src, H, q, out, scale)
    OVF_Q4_HD(hd, OVF_CALL)
#undef OVF_CALL
    return cuda_status(cudaGetLastError(), "attention_q4");
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
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (k_new) {
        OVF_CHECK_ARG(k_cache != v_cache, "attention_q4: keys and values need caches of their own");
        if ((st = launch_kv_q4_append(src, head_dim, k_new, v_new, s))) return st;
    }
    return launch_attention_q4(src, n_heads, head_dim, q, out, scale, scratch, s, false);
}

}  // extern "C"
