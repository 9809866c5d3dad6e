// ovf_verify.cu — verification of drafted tokens against the target's
// probabilities, from given random numbers.
//
// Row j of a sequence's logits gives the target's distribution after its
// first j drafts, p_j = softmax(logits_j / T); q_j is the distribution that
// draft d_j was drawn from (one-hot where the drafter is certain).  Draft j is
// accepted iff u_j q_j(d_j) < p_j(d_j).  At the first that is not, the next
// token is drawn from max(p_j - q_j, 0); if all are accepted, from the row
// behind them: the first index whose cumulative sum exceeds u_n times the
// total.  So the tokens are distributed as if the target had drawn them one by
// one.  T <= 0 is greedy: a draft is accepted iff it is its row's first
// maximum, which is also the next token.
//
// Exponentials and sums are formed in 64 bits: a decision that falls the other
// way because of a rounding changes a token, and a vocabulary has 10^5 borders.
#include "ovf_internal.cuh"

namespace ovf {

struct VerifyParams {
    const float *logits, *probs, *uniforms, *temperatures;
    const int32_t *drafts, *counts;
    int32_t *accepted, *token;
    int max_drafts, vocab;
};

static constexpr int kVerifyThreads = 1024;

// One CTA per sequence, row after row.
__global__ void __launch_bounds__(kVerifyThreads) verify_drafts_kernel(const VerifyParams p) {
    __shared__ double sd[32];
    __shared__ float sf[32];
    __shared__ int si[32];
    __shared__ int s_next;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x, V = p.vocab;
    const int n = p.counts ? min(p.counts[s], p.max_drafts) : p.max_drafts;
    if (n < 0) return;  // an unused place
    const float T = p.temperatures[s];
    const bool greedy = !(T > 0.0f);
    const int32_t *d = p.drafts ? p.drafts + (size_t)s * p.max_drafts : nullptr;
    const float *u = p.uniforms ? p.uniforms + (size_t)s * (p.max_drafts + 1) : nullptr;
    int acc = 0, next = -1;
    for (int j = 0; j <= n; ++j) {
        const float *x = p.logits + ((size_t)s * (p.max_drafts + 1) + j) * V;
        // largest logit and its first place
        float m = -INFINITY;
        int at = V;
        bool bad = false;
        for (int i = tid; i < V; i += kVerifyThreads) {
            const float y = x[i];
            bad |= y != y;
            if (y > m) m = y, at = i;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, o);
            const int a2 = __shfl_xor_sync(0xFFFFFFFFu, at, o);
            if (m2 > m || (m2 == m && a2 < at)) m = m2, at = a2;
        }
        __syncthreads();
        if (lane == 0) sf[warp] = m, si[warp] = at;
        bad = __syncthreads_or(bad);
        for (int w = 0; w < 32; ++w)
            if (sf[w] > m || (sf[w] == m && si[w] < at)) m = sf[w], at = si[w];
        bad |= !(fabsf(m) < INFINITY);
        if (bad) break;  // a row without a distribution: no token
        const int dj = j < n ? d[j] : -1;
        if (greedy) {
            if (dj == at) {
                ++acc;
                continue;
            }
            next = at;
            break;
        }
        double sum = 0.0;
        for (int i = tid; i < V; i += kVerifyThreads) sum += exp(((double)x[i] - m) / T);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        __syncthreads();
        if (lane == 0) sd[warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < 32; ++w) sum += sd[w];
        const float *q = p.probs && j < n ? p.probs + ((size_t)s * p.max_drafts + j) * V : nullptr;
        const bool known = dj >= 0 && dj < V;
        if (j < n && known) {
            const double e = exp(((double)x[dj] - m) / T), qd = q ? (double)q[dj] : 1.0;
            if ((double)u[j] * qd * sum < e) {
                ++acc;
                continue;
            }
        }
        // the residual's cumulative sum: every thread takes a run of the row
        const int per = (V + kVerifyThreads - 1) / kVerifyThreads, i0 = min(V, tid * per), i1 = min(V, i0 + per);
        auto rest = [&](int i) {
            const double e = exp(((double)x[i] - m) / T) / sum;
            if (j >= n) return e;
            if (q) return fmax(e - (double)q[i], 0.0);
            return i == dj ? 0.0 : e;
        };
        double run = 0.0;
        int last = -1;
        for (int i = i0; i < i1; ++i) {
            const double r = rest(i);
            run += r;
            if (r > 0.0) last = i;
        }
        double before = run;  // inclusive sum over the threads
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += y;
        }
        __syncthreads();
        if (lane == 31) sd[warp] = before;
        if (tid == 0) s_next = V;
        for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xFFFFFFFFu, last, o));
        if (lane == 0) si[warp] = last;
        __syncthreads();
        double base = 0.0, total = 0.0;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) base += sd[w];
            total += sd[w];
        }
        const double target = (double)u[p.max_drafts] * total;
        double c = base + before - run;
        for (int i = i0; i < i1; ++i) {
            const double r = rest(i);
            c += r;
            if (r > 0.0 && c > target) {
                atomicMin(&s_next, i);
                break;
            }
        }
        __syncthreads();
        next = s_next;
        if (next == V) {  // u of 1 or more, or no residual at all
            next = -1;
            for (int w = 0; w < 32; ++w) next = max(next, si[w]);
            if (next < 0) next = at;
        }
        break;
    }
    if (tid == 0) {
        p.accepted[s] = acc;
        p.token[s] = next;
    }
}

ovf_status launch_verify_drafts(const VerifyParams &p, int n_seq, cudaStream_t st) {
    verify_drafts_kernel<<<n_seq, kVerifyThreads, 0, st>>>(p);
    return cuda_status(cudaGetLastError(), "verify_drafts");
}

}  // namespace ovf

extern "C" ovf_status ovf_verify_drafts(const float *logits, const float *draft_probs, const int32_t *drafts,
                                        const int32_t *draft_counts, const float *uniforms, const float *temperatures,
                                        int32_t n_seq, int32_t max_drafts, int32_t vocab, int32_t *accepted,
                                        int32_t *next_token, void *stream) {
    using namespace ovf;
    OVF_CHECK_ARG(n_seq >= 0 && n_seq <= 65535, "verify_drafts: n_seq %d outside [0, 65535]", n_seq);
    OVF_CHECK_ARG(max_drafts >= 0 && max_drafts <= 1023, "verify_drafts: max_drafts %d outside [0, 1023]", max_drafts);
    OVF_CHECK_ARG(vocab > 0 && vocab <= (1 << 24), "verify_drafts: vocab %d outside [1, 2^24]", vocab);
    OVF_CHECK_ARG(logits && uniforms && temperatures && accepted && next_token, "verify_drafts: null buffer");
    OVF_CHECK_ARG(max_drafts == 0 || drafts, "verify_drafts: drafts are missing");
    OVF_CHECK_ARG(max_drafts > 0 || !draft_probs, "verify_drafts: probabilities without drafts");
    OVF_CHECK_ARG(accepted != next_token, "verify_drafts: one buffer for both results");
    if (n_seq == 0) return OVF_OK;
    VerifyParams p{logits, draft_probs, uniforms, temperatures, drafts, draft_counts, accepted, next_token, max_drafts, vocab};
    return launch_verify_drafts(p, n_seq, reinterpret_cast<cudaStream_t>(stream));
}
