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
// All exponentials and sums are formed in 64 bits: a decision must not depend on
// rounding, a vocabulary has 10^5 borders, and one that falls the other way changes
// a token.  The device does 64 such products a clock and SM, so an exponential of
// ten of them (a table and a short series) keeps pace with memory.
//
// A cluster of up to 16 CTAs takes a sequence, as many as let all sequences' run at
// once.  Its warps cut all rows, one behind
// the other, into equal runs of steps (128 elements), so that a warp meets one or
// two rows and reduces as often; the partial sums meet in distributed shared
// memory, and every CTA forms the same decisions.  Where the drawn row's weights
// are its exponentials, the partial sums serve the drawing too; where a draft's
// distribution is taken away, the row is passed once more.
// Measured: 4 drafts of one sequence over 128256 tokens, 15.0 us (five chained
// phases: a maximum pass, sums, decisions, search); 32 sequences of 7 drafts over
// 151936, 78 us, 2.24 TB/s (34 % of the copy rate): the exponentials alone take 16 us
// of all SMs, the rest is the waits of each phase's loads, with 32 warps an SM.
#include <float.h>

#include "ovf_internal.cuh"

namespace ovf {

static constexpr int kVfThreads = 512, kVfWarps = kVfThreads / 32;
static constexpr int kVfRows = 1024;        // max_drafts + 1
static constexpr int kVfCluster = 16;       // at most
static constexpr int kVfStep = 128;         // elements that a warp takes at once
// rows that a warp's run meets: the run is ceil(rows * steps / warps) steps of `steps` a row
static constexpr int kVfSlots = kVfRows / kVfWarps + 2;  // (a cluster of one CTA)

// e^x in 64 bits for x of -700 to 700, off by less than 2^-43.8 (2^-44.4 for |x| < 40: the series' rest is 2^-44.5 at
// most, the double of ln 2 / 64, n times, up to 2^-45.2).  x = n ln 2 / 64 + r, the series of e^r to r^4 (|r| <
// 0.0055), and 2^(n / 64) from `tab`, this lane's column of the table: entry 16 i holds the bits of 2^(i / 64) less
// i << 46 (the lanes of half a warp have a copy each, for indices are as good as random).  NaN stays NaN.
// A branch for other x would double its time (3.8 clocks a warp and SM): its callers raise smaller logits to
// a floor of weight e^-690 instead, in 32 bits.
__device__ __forceinline__ double vf_exp(double x, const unsigned long long *tab) {
    const double shift = 0x1.8p52;  // its sum with a number ends in that number's nearest integer
    const double kd = fma(x, 64.0 / 0.693147180559945309417, shift), n = kd - shift;
    const double r = fma(n, -0.693147180559945309417 / 64.0, x);  // (|n| < 2^16)
    double y = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    y = fma(y, r, 0.5);
    y = fma(y, r, 1.0);
    y = fma(y, r, 1.0);
    const int k = __double2loint(kd);
    return y * __longlong_as_double((long long)(tab[(k & 63) * 16] + ((unsigned long long)(long long)k << 46)));
}
// The same for any x up to 0 (0 below e^-690).
__device__ __forceinline__ double vf_exp0(double x, const unsigned long long *tab) {
    return x < -690.0 ? 0.0 : vf_exp(x, tab);
}
// The temperature for a row of largest logit m: at least 2^-31 of |m|.  (The next float is 2^-25 |m| below m or more, so
// that all that is smaller has a weight below e^-64 at that temperature and at any lower one, which no sum of 2^24 in
// 64 bits holds; and the floor lies a few floats below m, not on it.)
__device__ __forceinline__ float vf_temperature(float m, float T) { return fmaxf(T, fabsf(m) * 0x1p-31f); }
// Logits up to this have no weight: rounded up, so that its own weight stays in vf_exp's range.
__device__ __forceinline__ float vf_floor(float m, float T) {
    return fmaxf(__fsub_ru(m, __fmul_rd(690.0f, vf_temperature(m, T))), -FLT_MAX);
}
// 1 / the row's temperature, from 1 / T.
__device__ __forceinline__ double vf_inverse(float m, float T, double inv) {
    const float t = vf_temperature(m, T);
    return t == T ? inv : 1.0 / (double)t;
}
__device__ __forceinline__ float vf_raise(float x, float floor) {  // the larger; NaN stays NaN
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(floor));
    return y;
}
// The table from that of 2^(i / 32) which exp_libm (ovf_common.cuh) has.
__device__ __forceinline__ unsigned long long vf_tab(int i) {
    const unsigned long long half = kExp2Tab32[i >> 1] + ((unsigned long long)(i >> 1) << 47);  // bits of 2^((i >> 1) / 32)
    const double v = __longlong_as_double((long long)half) * (i & 1 ? 0x1.02c9a3e778061p+0 : 1.0);  // 2^(1 / 64)
    return (unsigned long long)__double_as_longlong(v) - ((unsigned long long)i << 46);
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float cluster_read(const float *p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(p), (uint32_t)rank)));
    return v;
}
__device__ __forceinline__ int cluster_read(const int *p, int rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), (uint32_t)rank)));
    return v;
}
__device__ __forceinline__ double cluster_read(const double *p, int rank) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(smem_u32(p), (uint32_t)rank)));
    return v;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    return x;
}

// What a row's address lies behind a 16-byte boundary, in elements.  Lane l's
// elements of step i are 4 (32 i + l) - shift .. + 3; those outside the row are `none`.
__device__ __forceinline__ int vf_shift(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) >> 2) & 3; }
__device__ __forceinline__ float4 vf_load4(const float *row, int V, int at, float none) {
    if (at >= 0 && at + 4 <= V) return __ldg(reinterpret_cast<const float4 *>(row + at));
    float4 v;
    v.x = at >= 0 && at < V ? row[at] : none;
    v.y = at + 1 >= 0 && at + 1 < V ? row[at + 1] : none;
    v.z = at + 2 >= 0 && at + 2 < V ? row[at + 2] : none;
    v.w = at + 3 >= 0 && at + 3 < V ? row[at + 3] : none;
    return v;
}

enum : int { VF_ACCEPT = 0, VF_REJECT = 1, VF_BAD = 2 };

struct VfShared {
    // this CTA's warps' parts of the rows: largest logit, its first place (greedy), sum of exponentials (NaN: a
    // row with a NaN or +infinity)
    double sum[kVfWarps][kVfSlots];
    float m[kVfWarps][kVfSlots];
    int at[kVfWarps][kVfSlots];
    // of every row: the drafted token, the whole row's sum, largest logit and its place, the decision
    double row_sum[kVfRows];
    float row_m[kVfRows];
    int draft[kVfRows], row_at[kVfRows], state[kVfRows];
    double part[kVfWarps];               // the drawing: sums of this CTA's warps' parts
    double all[kVfCluster * kVfWarps];   // of all parts
    double step[kVfWarps];               // of the steps of the part that holds the token
    unsigned long long tab[64 * 16];
    int token, last;
};

// The row that a token is drawn from.
struct VfRow {
    const float *x, *q;  // logits; probabilities to take away, or null
    double m, inv, scale;
    float floor;         // logits up to here have no weight
    int V, shift, out;   // `out`: a token without weight, or -1
};
struct VfFour {
    double w[4];
};

// This lane's four elements of a step: logits and, where they count, probabilities to take away.
struct VfLoad {
    float x[4], q[4];
};
__device__ __forceinline__ void vf_load(const VfRow &r, int i, VfLoad *l) {
    const int at = 4 * (32 * i + (threadIdx.x & 31)) - r.shift, a0 = 128 * i - r.shift;
    if (a0 >= 0 && a0 + kVfStep <= r.V) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(r.x + at));
        l->x[0] = v.x, l->x[1] = v.y, l->x[2] = v.z, l->x[3] = v.w;
        if (r.q) {
#pragma unroll
            for (int b = 0; b < 4; ++b) l->q[b] = __ldg(r.q + at + b);
        }
        return;
    }
    const float4 v = vf_load4(r.x, r.V, at, -INFINITY);
    l->x[0] = v.x, l->x[1] = v.y, l->x[2] = v.z, l->x[3] = v.w;
    if (r.q) {
#pragma unroll
        for (int b = 0; b < 4; ++b) l->q[b] = at + b >= 0 && at + b < r.V ? r.q[at + b] : 0.0f;
    }
}

// Their weights: max(scale e^((x - m) / T) - q, 0).
__device__ __forceinline__ VfFour vf_weights(const VfRow &r, const VfLoad &l, int i, const unsigned long long *tab) {
    const int at = 4 * (32 * i + (threadIdx.x & 31)) - r.shift;
    VfFour f;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const double e = vf_exp(((double)fmaxf(l.x[b], r.floor) - r.m) * r.inv, tab) * r.scale;
        f.w[b] = at + b == r.out || !(l.x[b] > r.floor) ? 0.0 : r.q ? fmax(e - (double)l.q[b], 0.0) : e;
    }
    return f;
}

// Steps: loads of a lane that are under way together.
template <int Steps, int Ctas>
__global__ void __launch_bounds__(kVfThreads, Ctas) verify_drafts_kernel(const VerifyParams p) {
    extern __shared__ __align__(16) unsigned char vf_smem[];
    VfShared &sh = *reinterpret_cast<VfShared *>(vf_smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = p.vocab;
    int rank, size;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    const int s = blockIdx.x / size, warps = size * kVfWarps, me = rank * kVfWarps + warp;
    const int n = p.counts ? min(p.counts[s], p.max_drafts) : p.max_drafts;
    if (n < 0) return;  // an unused place (all CTAs of the cluster leave)
    const bool greedy = !(p.temperatures[s] > 0.0f);
    const float T = fminf(p.temperatures[s], 1e30f);  // (impossible tokens stay impossible)
    const float *u = p.uniforms + (size_t)s * (p.max_drafts + 1);
    const float *logits = p.logits + (size_t)s * (p.max_drafts + 1) * V;
    const double inv = 1.0 / (double)T;
    const float last_u = u[p.max_drafts];
    for (int i = tid; i < 64 * 16; i += kVfThreads) sh.tab[i] = vf_tab(i / 16);
    const unsigned long long *tab = sh.tab + (lane & 15);
    for (int j = tid; j < n; j += kVfThreads) sh.draft[j] = p.drafts[(size_t)s * p.max_drafts + j];

    __syncthreads();

    // the warps' runs of the rows' steps
    const unsigned steps = (V + 3 + kVfStep - 1) / kVfStep;  // of a row, wherever it starts
    const unsigned all_steps = (unsigned)(n + 1) * steps, run = (all_steps + warps - 1) / warps;  // (below 2^28)
    const unsigned run1 = min(all_steps, (me + 1) * run);
    const int first_row = (int)(me * run / steps);
    for (unsigned st = me * run; st < run1;) {
        const int j = (int)(st / steps);
        const unsigned stop = min(run1, (unsigned)(j + 1) * steps);
        const float *x = logits + (size_t)j * V;
        int at = 4 * (32 * (int)(st - j * steps) + lane) - vf_shift(x);
        float m = -FLT_MAX, floor = -FLT_MAX;
        double scale = inv;  // 1 / temperature, for that m
        int place = 0x7FFFFFFF;
        double sum = 0.0;
        bool bad = false;
        const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        float4 v[Steps];
        auto load = [&](unsigned from, int place0) {
            // (a branch of the whole warp: one per load would keep them from being under way together)
            const int a0 = place0 - 4 * lane;
            if (a0 >= 0 && a0 + Steps * kVfStep <= V && from + Steps <= stop) {
#pragma unroll
                for (int i = 0; i < Steps; ++i) v[i] = __ldg(reinterpret_cast<const float4 *>(x + place0 + i * kVfStep));
            } else {
#pragma unroll
                for (int i = 0; i < Steps; ++i) v[i] = from + i < stop ? vf_load4(x, V, place0 + i * kVfStep, -INFINITY) : none;
            }
        };
        load(st, at);
        for (; st < stop; st += Steps, at += Steps * kVfStep) {
            float4 w[Steps];
#pragma unroll
            for (int i = 0; i < Steps; ++i) w[i] = v[i];
            if (st + Steps < stop) load(st + Steps, at + Steps * kVfStep);  // under way meanwhile
            float e[4 * Steps];
#pragma unroll
            for (int i = 0; i < Steps; ++i) e[4 * i] = w[i].x, e[4 * i + 1] = w[i].y, e[4 * i + 2] = w[i].z, e[4 * i + 3] = w[i].w;
            if (greedy) {
#pragma unroll
                for (int i = 0; i < 4 * Steps; ++i) {
                    bad |= e[i] != e[i];
                    const int here = at + (i >> 2) * kVfStep + (i & 3);
                    if (e[i] > m || (e[i] == m && here < place)) m = e[i], place = here;
                }
            } else {
                float top = m;
#pragma unroll
                for (int i = 0; i < 4 * Steps; ++i) top = fmaxf(top, e[i]);
                if (top > m) {
                    sum *= vf_exp0(((double)m - (double)top) * inv, tab);
                    m = top;
                    floor = vf_floor(m, T);
                    scale = vf_inverse(m, T, inv);
                }
                const double md = (double)m;
                double part[4];
#pragma unroll
                for (int i = 0; i < 4 * Steps; ++i) {
                    const double y = vf_exp(((double)vf_raise(e[i], floor) - md) * scale, tab);
                    part[i & 3] = i < 4 ? y : part[i & 3] + y;
                }
                sum += (part[0] + part[1]) + (part[2] + part[3]);
            }
        }
        st = stop;
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        if (greedy) {
            place = (int)__reduce_min_sync(0xFFFFFFFFu, m == top ? (unsigned)place : 0x7FFFFFFFu);
            if (__any_sync(0xFFFFFFFFu, bad)) sum = __longlong_as_double(0x7ff8000000000000ll);
        } else {
            sum = warp_sum(sum * vf_exp0(((double)m - (double)top) * inv, tab));
        }
        if (lane == 0) {
            sh.m[warp][j - first_row] = top;
            sh.sum[warp][j - first_row] = sum;
            sh.at[warp][j - first_row] = place;
        }
    }
    cluster_barrier();

    // the whole rows, and what becomes of every draft: a warp a row, a lane a part of it
    for (int j = warp; j <= n; j += kVfWarps) {
        const int w0 = (int)(j * steps / run), w1 = (int)(((j + 1) * steps - 1) / run);
        const int d = j < n ? sh.draft[j] : -1;
        float draft_x = -INFINITY, draft_q = 1.0f, draft_u = 0.0f;
        if (lane == 0 && d >= 0 && d < V) {
            draft_x = logits[(size_t)j * V + d];
            draft_u = u[j];
            if (p.probs) draft_q = p.probs[((size_t)s * p.max_drafts + j) * V + d];
        }
        float m = -FLT_MAX;
        double sum = 0.0;
        int at = 0x7FFFFFFF;
        for (int w = w0 + lane; w <= w1; w += 32) {
            const int slot = j - (int)(w * run / steps), from = w / kVfWarps;
            const float m2 = cluster_read(&sh.m[w % kVfWarps][slot], from);
            const double sum2 = cluster_read(&sh.sum[w % kVfWarps][slot], from);
            const int at2 = cluster_read(&sh.at[w % kVfWarps][slot], from);
            const float top = fmaxf(m, m2);
            sum = greedy ? sum + sum2
                         : sum * vf_exp0(((double)m - (double)top) * inv, tab) +
                               sum2 * vf_exp0(((double)m2 - (double)top) * inv, tab);
            if (m2 > m || (m2 == m && at2 < at)) at = at2;
            m = top;
        }
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        if (!greedy) sum *= vf_exp0(((double)m - (double)top) * inv, tab);
        sum = warp_sum(sum);
        at = (int)__reduce_min_sync(0xFFFFFFFFu, m == top ? (unsigned)at : 0x7FFFFFFFu);
        if (lane) continue;
        int state = VF_REJECT;  // (the row behind the last draft, a draft that is no token)
        if (sum != sum || !(top < INFINITY) || top == -FLT_MAX) {
            state = VF_BAD;
        } else if (greedy) {
            if (j < n && d == at) state = VF_ACCEPT;
        } else if (d >= 0 && d < V) {
            const double e = vf_exp0(((double)draft_x - (double)top) * inv, tab);
            if ((double)draft_u * (double)draft_q * sum < e) state = VF_ACCEPT;
        }
        sh.row_sum[j] = sum;
        sh.row_m[j] = top;
        sh.row_at[j] = at;
        sh.state[j] = state;
    }
    __syncthreads();

    // the first row that is not an accepted draft (every warp of the cluster finds the same)
    int k = 0;
    for (int j = 0;; j += 32) {
        const unsigned stop = __ballot_sync(0xFFFFFFFFu, j + lane <= n && sh.state[min(j + lane, n)] != VF_ACCEPT);
        if (stop) {
            k = j + __ffs(stop) - 1;
            break;
        }
    }
    int token = -1;
    if (sh.state[k] == VF_REJECT && greedy) {
        token = sh.row_at[k];
    } else if (sh.state[k] == VF_REJECT) {
        VfRow row;
        row.x = logits + (size_t)k * V;
        row.q = nullptr;
        row.m = (double)sh.row_m[k];
        row.inv = vf_inverse(sh.row_m[k], T, inv);
        row.scale = 1.0;
        row.floor = vf_floor(sh.row_m[k], T);
        row.V = V;
        row.shift = vf_shift(row.x);
        row.out = -1;
        double drafted = 0.0;  // the weight of a certain draft, which is taken away
        if (k < n && !p.probs && sh.draft[k] >= 0 && sh.draft[k] < V) {
            row.out = sh.draft[k];
            drafted = vf_exp0(((double)row.x[row.out] - row.m) * inv, tab);
        }
        // The row's parts and their weights.  Without a distribution to take away they are the runs above and their
        // sums (less a draft's, unless little were left: a difference of nearly equal sums would be inexact, and a
        // uniform so small asks for the least of what is left); else the row is passed once more.
        int parts, part0, per = 0;
        const bool again = (k < n && p.probs) || drafted > 0.99 * sh.row_sum[k] || (row.out >= 0 && last_u < 1e-8f);
        if (again) {
            if (k < n && p.probs) {
                row.q = p.probs + ((size_t)s * p.max_drafts + k) * V;
                row.scale = 1.0 / sh.row_sum[k];
            }
            parts = warps, part0 = 0, per = ((int)steps + warps - 1) / warps;
            const int i0 = min((int)steps, me * per), i1 = min((int)steps, i0 + per);
            double mine = 0.0;
            VfLoad a, b;
            vf_load(row, i0, &a);
            vf_load(row, i0 + 1, &b);  // (behind the row nothing is read)
            for (int i = i0; i < i1; ++i) {
                const VfLoad now = a;
                a = b;
                vf_load(row, i + 2, &b);
                const VfFour f = vf_weights(row, now, i, tab);
                mine += (f.w[0] + f.w[1]) + (f.w[2] + f.w[3]);
            }
            mine = warp_sum(mine);
            if (lane == 0) sh.part[warp] = mine;
            cluster_barrier();
        } else {
            part0 = (int)(k * steps / run);
            parts = (int)(((k + 1) * steps - 1) / run) - part0 + 1;
        }
        const int entries = (parts + 31) / 32;  // of a lane, one behind the other: they lie 32 apart
        for (int i = tid; i < entries * 32; i += kVfThreads) {
            double y = 0.0;
            if (i < parts) {
                const int w = part0 + i, from = w / kVfWarps;
                if (again) {
                    y = cluster_read(&sh.part[w % kVfWarps], from);
                } else {
                    const int slot = k - (int)(w * run / steps);
                    const double m2 = (double)cluster_read(&sh.m[w % kVfWarps][slot], from);
                    y = cluster_read(&sh.sum[w % kVfWarps][slot], from) * vf_exp0((m2 - row.m) * inv, tab);
                    if (row.out >= 0 && (unsigned)((row.out + row.shift) / kVfStep + k * steps) / run == (unsigned)w) {
                        y -= drafted;
                        if (y < 1e-12 * sh.row_sum[k]) y = 0.0;  // rounding, if the part had nothing else
                    }
                }
            }
            sh.all[i % entries * 32 + i / entries] = y;
        }
        __syncthreads();
        // the part that holds the token, and what lies before it
        double own = 0.0, base = 0.0;
        for (int i = 0; i < entries; ++i) own += sh.all[i * 32 + lane];
        double before = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xFFFFFFFFu, before, o);
            if (lane >= o) before += y;
        }
        const double target = (double)last_u * __shfl_sync(0xFFFFFFFFu, before, 31);
        before = __shfl_up_sync(0xFFFFFFFFu, before, 1);  // (not by a subtraction, which loses small weights before a large one)
        if (lane == 0) before = 0.0;
        int part = 0x7FFFFFFF, last = -1;
        for (int i = 0; i < entries; ++i) {
            const double y = sh.all[i * 32 + lane];
            if (y > 0.0) {
                last = lane * entries + i;
                if (part == 0x7FFFFFFF && before + y > target) part = last, base = before;
            }
            before += y;
        }
        const int mine = part;
        part = (int)__reduce_min_sync(0xFFFFFFFFu, (unsigned)part);
        last = __reduce_max_sync(0xFFFFFFFFu, last);
        base = __shfl_sync(0xFFFFFFFFu, base, __ffs(__ballot_sync(0xFFFFFFFFu, mine == part)) - 1);
        const bool over = part != 0x7FFFFFFF;
        if (!over) part = last;  // (u of 1 or more): the last token of any weight
        token = -2;              // written by the part's CTA
        if (part >= 0 && (part0 + part) / kVfWarps == rank) {
            // this CTA has the part: its warps take its steps side by side
            const int w = part0 + part, at0 = again ? w * per : (int)max(w * run, k * steps) - (int)(k * steps),
                      at1 = again ? at0 + per : (int)min((w + 1) * run, (k + 1) * steps) - (int)(k * steps);
            const int p0 = min((int)steps, at0), p1 = min((int)steps, at1);
            int found = -1, some = -1;
            for (int i = p0; i < p1 && found < 0; i += kVfWarps) {
                VfLoad l;
                vf_load(row, min(i + warp, p1), &l);
                VfFour f = vf_weights(row, l, i + warp, tab);
                if (i + warp >= p1) f.w[0] = f.w[1] = f.w[2] = f.w[3] = 0.0;
                const double four = (f.w[0] + f.w[1]) + (f.w[2] + f.w[3]);
                double incl = four;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                    if (lane >= o) incl += y;
                }
                double excl = __shfl_up_sync(0xFFFFFFFFu, incl, 1);
                if (lane == 0) excl = 0.0;
                __syncthreads();
                if (lane == 31) sh.step[warp] = incl;
                if (tid == 0) sh.token = 0x7FFFFFFF, sh.last = -1;
                __syncthreads();
                double cum = base;
#pragma unroll
                for (int w = 0; w < kVfWarps; ++w) {
                    if (w < warp) cum += sh.step[w];
                    base += sh.step[w];
                }
                cum += excl;
                unsigned hit = 0x7FFFFFFFu;
                int any = -1;
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    cum += f.w[b];
                    const int at = 4 * (32 * (i + warp) + lane) - row.shift + b;
                    if (f.w[b] > 0.0) {
                        any = at;
                        if (over && cum > target) hit = min(hit, (unsigned)at);
                    }
                }
                hit = __reduce_min_sync(0xFFFFFFFFu, hit);
                any = __reduce_max_sync(0xFFFFFFFFu, any);
                if (lane == 0) {
                    atomicMin(&sh.token, (int)hit);
                    atomicMax(&sh.last, any);
                }
                __syncthreads();
                if (sh.token != 0x7FFFFFFF) found = sh.token;
                some = max(some, sh.last);
            }
            if (tid == 0) p.token[s] = found >= 0 ? found : some;
        } else if (part < 0) {
            // nothing has weight: the row's first maximum
            if (tid == 0) sh.token = 0x7FFFFFFF;
            __syncthreads();
            for (int i = me; i < (int)steps; i += warps) {
                const int at = 4 * (32 * i + lane) - row.shift;
                const float4 v = vf_load4(row.x, V, at, -INFINITY);
                const float top = sh.row_m[k];
                const int hit = v.x == top ? at : v.y == top ? at + 1 : v.z == top ? at + 2 : v.w == top ? at + 3 : 0x7FFFFFFF;
                if (hit != 0x7FFFFFFF) atomicMin(&sh.token, hit);
            }
            cluster_barrier();
            token = 0x7FFFFFFF;
            for (int w = 0; w < size; ++w) token = min(token, cluster_read(&sh.token, w));
        }
    }
    if (rank == 0 && tid == 0) {
        p.accepted[s] = k;
        if (token != -2) p.token[s] = token;
    }
    cluster_barrier();  // nobody reads another CTA's memory any more
}

template <int Steps, int Ctas>
static void vf_config(int n_seq, int cluster, cudaStream_t st, cudaLaunchAttribute *attr, cudaLaunchConfig_t *cfg) {
    *cfg = {};
    cfg->gridDim = dim3(n_seq * cluster);
    cfg->blockDim = dim3(kVfThreads);
    cfg->dynamicSmemBytes = sizeof(VfShared);
    cfg->stream = st;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = cluster;
    attr->val.clusterDim.y = attr->val.clusterDim.z = 1;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

// Prepares the kernel on this device, and gives how many of its clusters of 1 to kVfCluster CTAs run there at once.
template <int Steps, int Ctas>
static cudaError_t vf_prepare(const int **fit) {
    static PerDeviceOnce once;
    static int fits[65][kVfCluster + 1];  // (the last for a device that PerDeviceOnce does not keep)
    const int dev = current_device(), at = dev >= 0 && dev < 64 ? dev : 64;
    const auto kernel = verify_drafts_kernel<Steps, Ctas>;
    if (once.pending(dev)) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(VfShared));
        for (int c = 1; c <= kVfCluster && e == cudaSuccess; ++c) {
            cudaLaunchAttribute attr[1];
            cudaLaunchConfig_t cfg;
            vf_config<Steps, Ctas>(1, c, nullptr, attr, &cfg);
            e = cudaOccupancyMaxActiveClusters(&fits[at][c], kernel, &cfg);
        }
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    *fit = fits[at];
    return cudaSuccess;
}

template <int Steps, int Ctas>
static cudaError_t launch_vf(const VerifyParams &p, int n_seq, int cluster, cudaStream_t st) {
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg;
    vf_config<Steps, Ctas>(n_seq, cluster, st, attr, &cfg);
    return cudaLaunchKernelEx(&cfg, verify_drafts_kernel<Steps, Ctas>, p);
}

ovf_status launch_verify_drafts(const VerifyParams &p, int n_seq, cudaStream_t st) {
    const int *alone, *shared;
    cudaError_t e = vf_prepare<4, 1>(&alone);
    if (e == cudaSuccess) e = vf_prepare<2, 2>(&shared);
    if (e != cudaSuccess) return cuda_status(e, "verify_drafts");
    // Clusters of 16 with an SM a CTA and more loads a lane, if all sequences' run at once; else the largest of which all
    // do, two CTAs an SM.  (A cluster stays within a group of SMs, so that fewer run than the SMs have room for; the
    // largest power of two for which these would do took 29.5 us for 8 sequences of 5 x 128256 logits, now 22.8, and
    // 45.0 for 36 of 8 x 50000, now 35.0.)
    int cluster = kVfCluster;
    while (cluster > 1 && shared[cluster] < n_seq) --cluster;
    e = alone[kVfCluster] >= n_seq ? launch_vf<4, 1>(p, n_seq, kVfCluster, st) : launch_vf<2, 2>(p, n_seq, cluster, st);
    return cuda_status(e, "verify_drafts");
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
    if (n_seq == 0) return OVF_OK;
    OVF_CHECK_ARG(logits && uniforms && temperatures && accepted && next_token, "verify_drafts: null buffer");
    OVF_CHECK_ARG(max_drafts == 0 || drafts, "verify_drafts: drafts are missing");
    OVF_CHECK_ARG(max_drafts > 0 || !draft_probs, "verify_drafts: probabilities without drafts");
    OVF_CHECK_ARG(accepted != next_token, "verify_drafts: one buffer for both results");
    VerifyParams p{logits, draft_probs, uniforms, temperatures, drafts, draft_counts, accepted, next_token, max_drafts, vocab};
    return launch_verify_drafts(p, n_seq, reinterpret_cast<cudaStream_t>(stream));
}
