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
// A decision must not depend on rounding: a vocabulary has 10^5 borders, and one
// that falls the other way changes a token.  The rows' sums are first formed from
// fp32 exponentials.  A lane rescales its sum when it meets a larger logit, at
// most once per 16 elements, 256 times in the longest row (2^24 over 8 x 512
// lanes), each time off by 2^-21.4 at most, so a sum is off by less than 2^-12;
// where a draft's decision is nearer to its border than that, its row is summed
// again in 64 bits.  The row that a token is drawn from is summed in 64 bits always.
//
// A cluster of 8 or 16 CTAs takes a sequence: every CTA a part of each row, all
// rows one behind the other, so that memory streams while sums are formed; the
// partial sums meet in distributed shared memory.  Bound by the logits' bytes for
// a batch, by the cluster's barriers and the drawing for one sequence.
#include <float.h>

#include "ovf_internal.cuh"

namespace ovf {

struct VerifyParams {
    const float *logits, *probs, *uniforms, *temperatures;
    const int32_t *drafts, *counts;
    int32_t *accepted, *token;
    int max_drafts, vocab;
};

static constexpr int kVfThreads = 512, kVfWarps = kVfThreads / 32;
static constexpr int kVfRows = 1024;        // max_drafts + 1
static constexpr int kVfCluster = 16;       // at most

// e^x in 64 bits, off by about 2^-48: x = n ln 2 / 32 + r, the series of e^r (|r| < 0.011), and 2^(n / 32) from
// the table of 2^(i / 32) that exp_libm (ovf_common.cuh) has.  ln 2 is taken in two parts, the first of 24 bits, so
// that its product with n is exact.
__device__ __forceinline__ double vf_exp(double x, const unsigned long long *tab) {
    if (!(x > -700.0)) return x < -746.0 ? 0.0 : exp(x);  // results below the normal numbers, and NaN
    const double shift = 0x1.8p52;  // its sum with a number ends in that number's nearest integer
    const double kd = fma(x, 32.0 / 0.693147180559945309417, shift), n = kd - shift;
    double r = fma(n, -0x1.62e4300000000p-1 / 32.0, x);
    r = fma(n, 0x1.05c610ca86c39p-29 / 32.0, r);
    double y = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    y = fma(y, r, 1.0 / 6.0);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    const int k = __double2loint(kd);
    return y * __longlong_as_double((long long)(tab[k & 31] + ((unsigned long long)(long long)k << 47)));
}

__device__ __forceinline__ float vf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <class T>
__device__ __forceinline__ T cluster_read(const T *p, int rank) {
    T v;
    const uint32_t at = mapa_shared(smem_u32(p), (uint32_t)rank);
    if (sizeof(T) == 8) {
        double d;
        asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(d) : "r"(at) : "memory");
        memcpy(&v, &d, sizeof(T));
    } else {
        uint32_t u;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(u) : "r"(at) : "memory");
        memcpy(&v, &u, sizeof(T));
    }
    return v;
}

// Elements 4 g - shift .. + 3 of a row (shift: what its address lies behind a
// 16-byte boundary); those outside the row are `none`.
__device__ __forceinline__ float4 vf_load4(const float *row, int V, int shift, int g, float none) {
    const int i = 4 * g - shift;
    if (i >= 0 && i + 4 <= V) return __ldg(reinterpret_cast<const float4 *>(row + i));
    float4 v;
    v.x = i >= 0 && i < V ? row[i] : none;
    v.y = i + 1 >= 0 && i + 1 < V ? row[i + 1] : none;
    v.z = i + 2 >= 0 && i + 2 < V ? row[i + 2] : none;
    v.w = i + 3 >= 0 && i + 3 < V ? row[i + 3] : none;
    return v;
}
__device__ __forceinline__ int vf_shift(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) >> 2) & 3; }

static constexpr int kVfBlock = 32;         // rows whose warps' results are joined at a time
static_assert(kVfBlock * kVfWarps == kVfThreads, "a thread joins one warp's result of one row");

struct VfShared {
    float m[kVfRows];          // this CTA's part of every row: largest logit,
    int at[kVfRows];           // its first place (greedy),
    float sum[kVfRows];        // sum of exponentials (NaN: a row with a NaN or +infinity)
    float row_m[kVfRows];      // the same of the whole rows
    int row_at[kVfRows];
    float wm[kVfBlock][kVfWarps];  // of a block of rows, the warps' parts
    int wat[kVfBlock][kVfWarps];
    float wsum[kVfBlock][kVfWarps];
    double part[2][kVfWarps];            // the drawing: sums of this CTA's warps' parts (two calls of vf_gather)
    double all[kVfCluster * kVfWarps];   // of all CTAs'
    unsigned long long tab[32];
    int first, token;
};

// The (largest, first place of it, sum) of N lanes as one, in every lane.
template <int N>
__device__ __forceinline__ void vf_join(float &m, int &at, float &sum, bool greedy, float c) {
    float top = m;
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    if (greedy) {
        if (m != top) at = 0x7FFFFFFF;
#pragma unroll
        for (int o = N / 2; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xFFFFFFFFu, at, o));
    } else {
        sum *= vf_ex2((m - top) * c);
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    m = top;
}

enum : int { VF_ACCEPT = 0, VF_REJECT = 1, VF_NEAR = 2, VF_BAD = 3 };

// The sum over the cluster of a value of every warp's part, in the order of the parts; all[] holds them.
// Calls take turns with the two sets of part: a CTA that writes one again has passed a barrier that all its
// readers have reached behind their reads.
__device__ __forceinline__ double vf_gather(VfShared &sh, double mine, int size, int warp, int lane, int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
    if (lane == 0) sh.part[turn][warp] = mine;
    cluster_barrier();
    for (int i = threadIdx.x; i < size * kVfWarps; i += kVfThreads)
        sh.all[i] = cluster_read(&sh.part[turn][i % kVfWarps], i / kVfWarps);
    turn ^= 1;
    __syncthreads();
    double s = 0.0;
    for (int i = lane; i < size * kVfWarps; i += 32) s += sh.all[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    return s;
}

__global__ void __launch_bounds__(kVfThreads, 2) verify_drafts_kernel(const VerifyParams p) {
    extern __shared__ __align__(16) unsigned char vf_smem[];
    VfShared &sh = *reinterpret_cast<VfShared *>(vf_smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.vocab;
    uint32_t rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int s = blockIdx.x / size;
    if (tid < 32) sh.tab[tid] = kExp2Tab32[tid];
    const int n = p.counts ? min(p.counts[s], p.max_drafts) : p.max_drafts;
    if (n < 0) return;  // an unused place (all CTAs of the cluster leave)
    const float T = p.temperatures[s];
    const bool greedy = !(T > 0.0f);
    const int32_t *drafts = p.drafts + (size_t)s * p.max_drafts;
    const float *u = p.uniforms + (size_t)s * (p.max_drafts + 1);
    const float *logits = p.logits + (size_t)s * (p.max_drafts + 1) * V;
    const float c = fminf(1.44269504088896340736f / T, FLT_MAX);
    const double inv = 1.0 / (double)T;
    __syncthreads();

    // Every row's largest logit and sum (greedy: and the first place of it), this CTA's part.  A warp takes its
    // part of one row behind the other, four loads a lane at a time and the next four under way.
    {
        const int step = size * kVfThreads, first = rank * kVfThreads + tid;
        float4 v[4];
        auto load = [&](int j, int g) {
            const float *x = logits + (size_t)j * V;
            const int shift = vf_shift(x);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = vf_load4(x, V, shift, g + i * step, -INFINITY);
        };
        load(0, first);
        for (int j0 = 0; j0 <= n; j0 += kVfBlock) {
            const int j1 = min(n + 1, j0 + kVfBlock);
            for (int j = j0; j < j1; ++j) {
                const int shift = vf_shift(logits + (size_t)j * V), groups = (V + shift + 3) / 4;
                float m = -FLT_MAX;
                int at = 0x7FFFFFFF;
                double sum = 0.0;
                bool bad = false;
                for (int g = first; g - first < groups; g += 4 * step) {
                    float4 w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = v[i];
                    if (g - first + 4 * step < groups) load(j, g + 4 * step);
                    else if (j < n) load(j + 1, first);
                    float top = w[0].x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fmaxf(w[i].x, w[i].y), fmaxf(w[i].z, w[i].w)));
                    if (greedy) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                bad |= e[k] != e[k];
                                const int place = 4 * (g + i * step) - shift + k;
                                if (e[k] > m || (e[k] == m && place < at)) m = e[k], at = place;
                            }
                        }
                    } else {
                        if (top > m) {
                            sum *= (double)vf_ex2((m - top) * c);
                            m = top;
                        }
                        float part = 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            part += (vf_ex2((w[i].x - m) * c) + vf_ex2((w[i].y - m) * c)) +
                                    (vf_ex2((w[i].z - m) * c) + vf_ex2((w[i].w - m) * c));
                        sum += (double)part;
                    }
                }
                float fsum = bad ? __int_as_float(0x7fc00000) : (float)sum;
                vf_join<32>(m, at, fsum, greedy, c);
                if (lane == 0) sh.wm[j - j0][warp] = m, sh.wat[j - j0][warp] = at, sh.wsum[j - j0][warp] = fsum;
            }
            __syncthreads();
            const int r = tid / kVfWarps, w = tid % kVfWarps;
            if (j0 + (warp * 32) / kVfWarps < j1) {  // (whole warps: two rows each)
                float m = sh.wm[r][w], sum = sh.wsum[r][w];
                int at = sh.wat[r][w];
                vf_join<kVfWarps>(m, at, sum, greedy, c);
                if (w == 0 && j0 + r < j1) sh.m[j0 + r] = m, sh.at[j0 + r] = at, sh.sum[j0 + r] = sum;
            }
            __syncthreads();
        }
    }
    cluster_barrier();

    // the whole rows, and what becomes of every draft (each CTA forms the same)
    int state[kVfRows / kVfThreads];
#pragma unroll
    for (int i = 0; i < kVfRows / kVfThreads; ++i) {
        const int j = tid + i * kVfThreads;
        state[i] = VF_ACCEPT;
        if (j > n) continue;
        float m = -FLT_MAX, sum = 0.0f;
        int at = 0x7FFFFFFF;
        for (int w = 0; w < (int)size; ++w) m = fmaxf(m, cluster_read(&sh.m[j], w));
        for (int w = 0; w < (int)size; ++w) {
            const float m2 = cluster_read(&sh.m[j], w), sum2 = cluster_read(&sh.sum[j], w);
            sum += greedy ? sum2 : sum2 * vf_ex2((m2 - m) * c);
            if (greedy && m2 == m) at = min(at, cluster_read(&sh.at[j], w));
        }
        sh.row_m[j] = m;
        sh.row_at[j] = at;
        const int d = j < n ? drafts[j] : -1;
        if (sum != sum || !(m < INFINITY) || (greedy ? at == 0x7FFFFFFF : sum == 0.0f)) {
            state[i] = VF_BAD;
        } else if (j == n) {
            state[i] = VF_REJECT;  // the row behind the last draft
        } else if (greedy) {
            state[i] = d == at ? VF_ACCEPT : VF_REJECT;
        } else if (d < 0 || d >= V) {
            state[i] = VF_REJECT;
        } else {
            const double e = vf_exp(((double)logits[(size_t)j * V + d] - (double)m) * inv, sh.tab);
            const double q = p.probs ? (double)p.probs[((size_t)s * p.max_drafts + j) * V + d] : 1.0;
            const double limit = (double)u[j] * q * (double)sum;
            state[i] = fabs(limit - e) <= 0x1p-12 * fmax(limit, e) ? VF_NEAR : limit < e ? VF_ACCEPT : VF_REJECT;
        }
    }

    // the first row that is not an accepted draft
    int k = -1, st = VF_ACCEPT, turn = 0;
    const int per = (int)(((size_t)V + 3 + size * kVfWarps * 128 - 1) / (size * kVfWarps * 128));  // 128 elements a step
    const int steps0 = (int)(rank * kVfWarps + warp) * per;  // this warp's part of a row: steps [steps0, steps0 + per)
    while (true) {
        __syncthreads();
        if (tid == 0) sh.first = 0x7FFFFFFF;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kVfRows / kVfThreads; ++i) {
            const int j = tid + i * kVfThreads;
            if (j <= n && j > k && state[i] != VF_ACCEPT) atomicMin(&sh.first, j * 4 + state[i]);
        }
        __syncthreads();
        k = sh.first >> 2;
        st = sh.first & 3;
        if (st != VF_NEAR) break;
        // too near to tell: the row's sum in 64 bits
        const float *x = logits + (size_t)k * V;
        const double m = (double)sh.row_m[k];
        const int shift = vf_shift(x);
        double sum = 0.0;
        for (int i = steps0; i < steps0 + per; ++i) {
            const float4 v = vf_load4(x, V, shift, i * 32 + lane, -INFINITY);
            sum += (vf_exp(((double)v.x - m) * inv, sh.tab) + vf_exp(((double)v.y - m) * inv, sh.tab)) +
                   (vf_exp(((double)v.z - m) * inv, sh.tab) + vf_exp(((double)v.w - m) * inv, sh.tab));
        }
        const double total = vf_gather(sh, sum, size, warp, lane, turn);
        const int d = drafts[k];
        const double q = p.probs ? (double)p.probs[((size_t)s * p.max_drafts + k) * V + d] : 1.0;
        if (!((double)u[k] * q * total < vf_exp(((double)x[d] - m) * inv, sh.tab))) {
            st = VF_REJECT;
            break;
        }
    }

    int token = -1;
    if (st == VF_REJECT && greedy) {
        token = sh.row_at[k];
    } else if (st == VF_REJECT) {
        const float *x = logits + (size_t)k * V;
        const float *q = p.probs && k < n ? p.probs + ((size_t)s * p.max_drafts + k) * V : nullptr;
        const int out = !q && k < n ? drafts[k] : -1;  // a certain draft has no weight left
        const double m = (double)sh.row_m[k];
        const int shift = vf_shift(x);
        auto weight4 = [&](int i, double scale, double (&w)[4]) {
            const float4 v = vf_load4(x, V, shift, i * 32 + lane, -INFINITY);
            w[0] = vf_exp(((double)v.x - m) * inv, sh.tab) * scale;
            w[1] = vf_exp(((double)v.y - m) * inv, sh.tab) * scale;
            w[2] = vf_exp(((double)v.z - m) * inv, sh.tab) * scale;
            w[3] = vf_exp(((double)v.w - m) * inv, sh.tab) * scale;
            const int at = 4 * (i * 32 + lane) - shift;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (q && at + b >= 0 && at + b < V) w[b] = fmax(w[b] - (double)q[at + b], 0.0);
                if (at + b == out) w[b] = 0.0;
            }
        };
        double scale = 1.0, w[4];
        if (q) {  // p and q are compared: p needs its sum
            double sum = 0.0;
            const float *q0 = q;
            q = nullptr;
            for (int i = steps0; i < steps0 + per; ++i) {
                weight4(i, 1.0, w);
                sum += (w[0] + w[1]) + (w[2] + w[3]);
            }
            q = q0;
            scale = 1.0 / vf_gather(sh, sum, size, warp, lane, turn);
        }
        double sum = 0.0;
        for (int i = steps0; i < steps0 + per; ++i) {
            weight4(i, scale, w);
            sum += (w[0] + w[1]) + (w[2] + w[3]);
        }
        const double rest = vf_gather(sh, sum, size, warp, lane, turn);
        const double target = (double)u[p.max_drafts] * rest;
        // the part that holds the token, and what lies before it (every warp finds the same)
        const int entries = (int)size * kVfWarps / 32;  // of a lane, one behind the other
        double own = 0.0, base = 0.0;
        for (int i = 0; i < entries; ++i) own += sh.all[lane * entries + i];
        double before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += y;
        }
        before -= own;
        int part = 0x7FFFFFFF, last = -1;
        for (int i = 0; i < entries; ++i) {
            const double y = sh.all[lane * entries + i];
            if (y > 0.0) {
                last = lane * entries + i;
                if (part == 0x7FFFFFFF && before + y > target) part = last, base = before;
            }
            before += y;
        }
        const int mine = part;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            part = min(part, __shfl_xor_sync(0xFFFFFFFFu, part, o));
            last = max(last, __shfl_xor_sync(0xFFFFFFFFu, last, o));
        }
        const unsigned holder = __ballot_sync(0xFFFFFFFFu, mine == part);
        base = __shfl_sync(0xFFFFFFFFu, base, __ffs(holder) - 1);
        if (part == 0x7FFFFFFF) part = -1;
        const bool over = part >= 0;
        if (!over) part = last;  // (u of 1 or more): the last token of any weight
        if (part == (int)rank * kVfWarps + warp) {
            int found = -1, some = -1;
            double run = base;
            for (int i = steps0; i < steps0 + per && found < 0; ++i) {
                weight4(i, scale, w);
                const double four = (w[0] + w[1]) + (w[2] + w[3]);
                double incl = four;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                    if (lane >= o) incl += y;
                }
                double cum = run + (incl - four);
                int hit = 0x7FFFFFFF, any = -1;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    cum += w[b];
                    const int at = 4 * (i * 32 + lane) - shift + b;
                    if (w[b] > 0.0) {
                        any = at;
                        if (over && cum > target) hit = min(hit, at);
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    hit = min(hit, __shfl_xor_sync(0xFFFFFFFFu, hit, o));
                    any = max(any, __shfl_xor_sync(0xFFFFFFFFu, any, o));
                }
                some = max(some, any);
                if (hit != 0x7FFFFFFF) found = hit;
                run += __shfl_sync(0xFFFFFFFFu, incl, 31);
            }
            if (lane == 0) p.token[s] = found >= 0 ? found : some;
        }
        token = -2;  // written by the part's warp
        if (part < 0) {
            // nothing has weight: the row's first maximum
            if (tid == 0) sh.token = 0x7FFFFFFF;
            __syncthreads();
            for (int i = steps0; i < steps0 + per; ++i) {
                const float4 v = vf_load4(x, V, shift, i * 32 + lane, -INFINITY);
                const int at = 4 * (i * 32 + lane) - shift;
                const float mm = sh.row_m[k];
                const int hit = v.x == mm ? at : v.y == mm ? at + 1 : v.z == mm ? at + 2 : v.w == mm ? at + 3 : 0x7FFFFFFF;
                if (hit != 0x7FFFFFFF) atomicMin(&sh.token, hit);
            }
            cluster_barrier();
            token = 0x7FFFFFFF;
            for (int w2 = 0; w2 < (int)size; ++w2) token = min(token, cluster_read(&sh.token, w2));
        }
    }
    if (rank == 0 && tid == 0) {
        p.accepted[s] = k;
        if (token != -2) p.token[s] = token;
    }
    cluster_barrier();  // nobody reads another CTA's memory any more
}

ovf_status launch_verify_drafts(const VerifyParams &p, int n_seq, cudaStream_t st) {
    static PerDeviceOnce once;
    const int dev = current_device();
    if (once.pending(dev)) {
        cudaError_t e = cudaFuncSetAttribute(verify_drafts_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(verify_drafts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)sizeof(VfShared));
        if (e != cudaSuccess) return cuda_status(e, "verify_drafts");
        once.mark(dev);
    }
    const int cluster = n_seq * kVfCluster <= sm_count(dev) ? kVfCluster : 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_seq * cluster);
    cfg.blockDim = dim3(kVfThreads);
    cfg.dynamicSmemBytes = sizeof(VfShared);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, verify_drafts_kernel, p), "verify_drafts");
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
