// ovf_attn_q4_rows.cu — attention of many query rows (a prefill chunk) over the
// 4-bit KV cache on the 5th-generation tensor cores.
//
// The function is ovf_attn_q4.cu's.  A CTA owns 128 query rows of one KV head (its
// query heads, row after row) and a run of the sequence's 128-position tiles:
//     S = Q K^T,  P = 2^(S - max),  O += P V,
// Q, S, P and O in TMEM (Q and P as the left operand, from TMEM), K and V expanded
// from their codes into shared memory in the UMMA layout.  As there, an fp32
// operand enters as two fp16 numbers (hi + lo, 22 bits; small weights fewer, see below),
// here as two products into one accumulator, and the cached values are fp16 numbers by definition.
//
// The tensor cores cut an accumulator's lower bits off at each addition, toward zero,
// so that a long sum falls short (measured: 3e-7 of O per 128 positions, 1.9e-5 at
// 8192), where fp32's rounding would average out.  An accumulator in TMEM therefore
// sums kArWindow tiles at most; the windows are added in fp32 in shared memory.  Two tiles:
// 1.2e-6 off at 8192 positions (a plain fp32 softmax 2.1e-6), four: 1.7e-6 and 7 %
// faster; at 1024 positions 0.95e-6 and 1.4e-6 (fp32 1.1e-6), so two.  S takes its
// small lo products first.
//
// The maximum that P refers to is raised at each window's first tile, where O begins
// anew, and inside a window only when a row's scores pass it by more than 2^3.5; until
// then P is at most 2^(12 + 3.5), inside fp16, and O needs no rescaling.  (Both steps
// from the maximum are rounded so that the bound holds for scores of 2^24 and more,
// between whose floats lie more.)  Weights are held times 2^12, so that fp16's
// smallest step is 2^-36 of the maximum's: what smaller weights lose is at most
// 2^-37 a position, 1e-6 of the values at 131072 of them (with 2^6, and 2^8 in place of
// 2^3.5, 6e-5, in all of one sign under a long flat tail; 1 % faster.  2^14 and 2^1.5
// rescale so often that they take 4 % longer).  Weights are summed in two steps, of 16
// tiles and of those sums, for the same reason.
//
// Codes lie in the pairs that their expansion yields: eight elements come out as
// 0 4 1 5 2 6 3 7, along dimensions for K and along positions for V.  Q's columns
// and S's columns (the order of K's rows) follow that order, so that products
// pair up and nothing is ever moved.
//
// Warps, linked by mbarriers (each wait is bounded; a role that gives up goes on
// without waiting, so that every barrier is met and TMEM is freed):
//   0-7    softmax: a thread per row and half of a tile's columns;
//   8-15   expansion of K and V, two stages each;
//   16     TMEM allocation, and the thread that issues the MMAs: S of the next
//          tile before O of this one.
// Per tile at head_dim 128 the tensor cores need 2048 clocks (32 MMAs of 64: two
// products each way), shared memory about 2000 (K and V read twice and written once,
// O of a window every other tile), the schedulers about 1400 each (7 instructions per
// score, 15 per eight codes); 3600 are measured, about half of the tensor cores' time.
// Single operands would halve their part at the price of an fp16 softmax's precision.
// No cluster, no multicast; tensor operands are this GPU's own.
#include "ovf_q4.cuh"

namespace ovf {

static constexpr int kArM = 128;        // query rows of a CTA
static constexpr int kArN = 128;        // positions of a tile
static constexpr int kArExpand = 8;      // expanding warps
static constexpr int kArMma = 8 + kArExpand;
static constexpr int kArThreads = (kArMma + 1) * 32;
static constexpr int kArStages = 2;
static constexpr int kArWindow = 2;      // tiles that one accumulator in TMEM sums (a power of 2)
static constexpr int kArSums = 16;       // tiles whose weights are summed before they are added to the others' (a power of 2)
static constexpr float kArLift = 12.0f; // weights times 2^12
static constexpr float kArSlack = 3.5f; // inside a window the maximum is raised when it is passed by 2^3.5

template <int NG>
struct ArSmem {
    static constexpr int HD = NG * 32;
    static constexpr int kTile = kArN * HD * 2;                  // K or V, fp16
    static constexpr int k_off = 0;
    static constexpr int v_off = k_off + kArStages * kTile;
    static constexpr int q_pitch = HD + 4;                       // rows of Q on its way to TMEM (in K's and V's place)
    static constexpr int q_bytes = kArM * q_pitch * 4;
    static constexpr int main_bytes = 2 * kArStages * kTile > q_bytes ? 2 * kArStages * kTile : q_bytes;
    static constexpr int acc_off = main_bytes;                   // [half][dimension / 4][row] float4: O of earlier windows
    static constexpr int x_off = acc_off + kArM * HD * 4;        // [2][2][128] floats: halves' maxima, sums
    static constexpr int bar_off = x_off + 2 * 2 * kArM * 4;
    static constexpr int total = bar_off + 256 + 128;
    // TMEM columns
    static constexpr int q_col = 0, o_col = HD, s_col = 2 * HD;
};

struct ArParams {
    Q4Source src;
    int H;
    const float *q;
    float *out, *part, *part_ml;
    float scale2;
    int splits;  // partial results lie [row][split]
};

// D[tmem] (+)= A[tmem] B[shared memory]: kind::f16, fp16 operands, fp32 accumulator, M = 128.
template <bool Accumulate>
__device__ __forceinline__ void ar_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "n"(Accumulate ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ constexpr uint32_t ar_idesc(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kArM >> 4) << 24);
}
__device__ __forceinline__ void ar_pair_sync(int pair) { asm volatile("bar.sync %0, 64;" ::"r"(1 + pair) : "memory"); }

// Two fp32 operations in one instruction (each rounded as the single ones are).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, w;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
        " fma.rn.f32x2 w, x, y, z;\n mov.b64 {%0, %1}, w;\n}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 z, x, y;\n"
        " mov.b64 {%0, %1}, z;\n}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// Two fp32 numbers as pairs of hi and of lo parts.
__device__ __forceinline__ void ar_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h), r = fma2(f, make_float2(-1.0f, -1.0f), make_float2(x, y));
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(r.x, r.y));
}

template <int NG>
__global__ void __launch_bounds__(kArThreads, 1) attention_q4_rows_kernel(const ArParams p) {
    using SM = ArSmem<NG>;
    constexpr int HD = NG * 32;
    extern __shared__ uint8_t ar_raw[];
    uint8_t *sm = ar_raw + ((128u - (smem_u32(ar_raw) & 127u)) & 127u);
    __shared__ uint32_t tmem_slot;
    const Q4Source &src = p.src;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.H / src.KVH;
    const int s = blockIdx.z, h = blockIdx.y % src.KVH, mt = blockIdx.y / src.KVH, split = blockIdx.x;
    Q4View w;
    if (!q4_view(src, s, &w) || mt * kArM >= w.count * G) return;
    const int last_row = min(w.count - 1, (mt * kArM + kArM - 1) / G);
    const int tiles = (w.pos + last_row + kArN) / kArN;
    const int t0 = (int)((int64_t)tiles * split / p.splits), t1 = (int)((int64_t)tiles * (split + 1) / p.splits), nt = t1 - t0;
    // row i of the CTA: query head i % G of row i / G
    auto out_row = [&](int i) { return ((size_t)s * src.rows + i / G) * p.H + h * G + i % G; };
    if (nt <= 0) {  // fewer tiles than splits: nothing to add
        const int i = mt * kArM + threadIdx.x;
        if (threadIdx.x < kArM && i / G < w.count)
            *reinterpret_cast<float2 *>(p.part_ml + (out_row(i) * p.splits + split) * 2) = make_float2(-INFINITY, 0.0f);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + SM::bar_off);
    uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *s_full = bars + 8, *p_full = bars + 10,
             *o_done = bars + 12;
    float *xch = reinterpret_cast<float *>(sm + SM::x_off);  // [parity][half][row]
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], kArExpand);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], kArExpand);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 8);
        }
        mbar_init(o_done, 1);
        fence_mbar_init();
    }
    if (warp == kArMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // The queries, rotated (Rope/RopeKernel.cs:46-93, each step rounded by itself) and times the scale, to shared memory.
    // (A warp takes four rows at a time, so that their loads are under way together.)
    float *qs = reinterpret_cast<float *>(sm);
    constexpr int PL = HD >= 64 ? HD / 64 : 1;  // pairs of a lane
    for (int i0 = warp * 4; i0 < kArM; i0 += kArThreads / 32 * 4) {
        float v0[4][PL], v1[4][PL], c[4][PL], sn[4][PL];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int g = mt * kArM + i0 + k, r = g / G;
            const float *q = p.q + (((size_t)s * src.rows + r) * p.H + h * G + (g - r * G)) * HD;
#pragma unroll
            for (int b = 0; b < PL; ++b) {
                const int j = lane + 32 * b;
                v0[k][b] = v1[k][b] = c[k][b] = sn[k][b] = 0.0f;
                if (r < w.count && j < HD / 2) {
                    if (src.split_half) {
                        v0[k][b] = q[j];
                        v1[k][b] = q[j + HD / 2];
                    } else {
                        const float2 v = *reinterpret_cast<const float2 *>(q + 2 * j);
                        v0[k][b] = v.x;
                        v1[k][b] = v.y;
                    }
                    if (w.cos) {
                        c[k][b] = w.cos[(size_t)(w.pos + r) * (HD / 2) + j];
                        sn[k][b] = w.sin[(size_t)(w.pos + r) * (HD / 2) + j];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int b = 0; b < PL; ++b) {
                const int j = lane + 32 * b;
                if (j >= HD / 2) continue;
                const float x0 = v0[k][b], x1 = v1[k][b], cc = c[k][b], ss = sn[k][b];
                const float y0 = w.cos ? fsub(fmul(x0, cc), fmul(x1, ss)) : x0;
                const float y1 = w.cos ? fadd(fmul(x0, ss), fmul(x1, cc)) : x1;
                float *to = qs + (i0 + k) * SM::q_pitch;
                if (src.split_half) {
                    to[j] = y0 * p.scale2;
                    to[j + HD / 2] = y1 * p.scale2;
                } else {
                    *reinterpret_cast<float2 *>(to + 2 * j) = make_float2(y0 * p.scale2, y1 * p.scale2);
                }
            }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t lane_addr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    const int row = 32 * (warp & 3) + lane, half = (warp >> 2) & 1;  // (softmax warps)
    float factor = 1.0f;
    int limit = 0x7FFFFFFF;
    if (warp < 8) {
        // a thread takes half of its row's dimensions to TMEM
        const float *x = qs + row * SM::q_pitch;
        float top = 0.0f;
        for (int j = 0; j < HD; j += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(x + j);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        const int ex = min(max((__float_as_int(top) >> 23) & 255, 15), 254);
        const float up = __int_as_float((268 - ex) << 23);  // the largest element to [2^14, 2^15)
        factor = __int_as_float((ex - 14) << 23);
        const int r = (mt * kArM + row) / G;
        if (r < w.count) limit = w.pos + r;
#pragma unroll
        for (int b = 0; b < HD / 16; b += (HD >= 64 ? 4 : 2)) {  // blocks of eight dimensions, 16 (8) columns at a time
            constexpr int NB = HD >= 64 ? 4 : 2;
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const float *y = x + half * (HD / 2) + (b + i) * 8;
                const float4 u = *reinterpret_cast<const float4 *>(y), v = *reinterpret_cast<const float4 *>(y + 4);
                ar_split(u.x * up, v.x * up, hi[4 * i], lo[4 * i]);
                ar_split(u.y * up, v.y * up, hi[4 * i + 1], lo[4 * i + 1]);
                ar_split(u.z * up, v.z * up, hi[4 * i + 2], lo[4 * i + 2]);
                ar_split(u.w * up, v.w * up, hi[4 * i + 3], lo[4 * i + 3]);
            }
            const uint32_t col = lane_addr + SM::q_col + half * (HD / 4) + b * 4;
            if (NB == 4) {
                tmem_st16(col, reinterpret_cast<const float *>(hi));
                tmem_st16(col + HD / 2, reinterpret_cast<const float *>(lo));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(col + i), "r"(hi[i]) : "memory");
                    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(col + HD / 2 + i), "r"(lo[i]) : "memory");
                }
            }
        }
        tmem_st_wait();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    bool ok = true;
    auto wait = [&](uint64_t *bar, int parity) { ok = ok && mbar_wait_bounded(bar, (uint32_t)parity); };
    if (warp < 8) {
        // ------------------------------------------------------- softmax
        // l: the sum of the weights of up to kArSums tiles, l_acc: of those before; m_acc: what O of the earlier windows refers to
        float m = -INFINITY, l = 0.0f, l_acc = 0.0f, m_acc = -INFINITY;
        float4 *acc = reinterpret_cast<float4 *>(sm + SM::acc_off) + half * (HD / 8) * kArM + row;
        for (int i = 0; i < nt; ++i) {
            const bool fresh = (i & (kArWindow - 1)) == 0;  // O begins anew with this tile
            const uint32_t s_at = lane_addr + SM::s_col + (i & 1) * kArN + half * (kArN / 2);
            const int p0 = (t0 + i) * kArN + half * (kArN / 2);
            wait(&s_full[i & 1], (i >> 1) & 1);
            tc_fence_after();
            // two passes over the columns, a few at a time: the registers of 64 would not leave room for 17 warps
            const bool masked = __any_sync(0xFFFFFFFFu, p0 + kArN / 2 - 1 > limit);
            float x[2][16];
            auto hide = [&](int c0, float *y) {
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 16; ++c)  // columns in the order 0 4 1 5 2 6 3 7 of positions
                        if (p0 + c0 + (c & ~7) + ((c & 7) >> 1) + 4 * (c & 1) > limit) y[c] = -INFINITY;
                }
            };
            auto load = [&](int c0, float *y) { tmem_ld16_nowait(s_at + c0, reinterpret_cast<uint32_t *>(y)); };
            float top = -INFINITY;
#pragma unroll
            for (int c0 = 32; c0 >= 0; c0 -= 32) {
                load(c0, x[0]);
                load(c0 + 16, x[1]);
                tmem_ld_wait();
                hide(c0, x[0]);
                hide(c0 + 16, x[1]);
#pragma unroll
                for (int c = 0; c < 16; ++c) top = fmaxf(top, fmaxf(x[0][c], x[1][c]));
            }
            top *= factor;
            float *mine = xch + (i & 1) * 2 * kArM + half * kArM + row;
            *mine = top;
            ar_pair_sync(warp & 3);
            top = fmaxf(top, xch[(i & 1) * 2 * kArM + (half ^ 1) * kArM + row]);
            const float m_before = m, most = __fadd_rd(m, kArSlack);
            if (fresh) {
                m = fmaxf(m, top);
                if ((i & (kArSums - 1)) == 0) {
                    l_acc += l;
                    l = 0.0f;
                }
                const float k = m_before == m ? 1.0f : ex2(m_before - m);
                l *= k;
                l_acc *= k;
            } else {
                const bool raise = top > most || (m == -INFINITY && top > m);
                if (__any_sync(0xFFFFFFFFu, raise)) {
                    // O so far, to the new maximum (this half of its columns)
                    wait(o_done, (i - 1) & 1);
                    tc_fence_after();
                    const float k = raise ? ex2(m - top) : 1.0f;
                    l *= k;
                    l_acc *= k;
                    if (raise) m = top;
#pragma unroll
                    for (int c = 0; c < HD / 2; c += 16) {
                        float o[16];
                        const uint32_t at = lane_addr + SM::o_col + half * (HD / 2) + c;
                        tmem_ld16_nowait(at, reinterpret_cast<uint32_t *>(o));
                        tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] *= k;
                        tmem_st16(at, o);
                    }
                    tmem_st_wait();
                }
            }
            const float base = __fsub_ru(m == -INFINITY ? 0.0f : m, kArLift);
            float2 sum = make_float2(0.0f, 0.0f);
            const float2 factor2 = make_float2(factor, factor), base2 = make_float2(-base, -base);
            // (P of 16 columns goes where those scores were: 8 columns of hi, 8 of lo parts)
            auto weights = [&](int c0, const float *y) {
                uint32_t p16[16];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float2 w = fma2(make_float2(y[2 * j], y[2 * j + 1]), factor2, base2);
                    w = make_float2(ex2(w.x), ex2(w.y));
                    sum = add2(sum, w);
                    ar_split(w.x, w.y, p16[j], p16[8 + j]);
                }
                tmem_st16(s_at + c0, reinterpret_cast<const float *>(p16));
            };
            // (the first 32 columns are still there)
            weights(0, x[0]);
            load(32, x[0]);
            weights(16, x[1]);
            load(48, x[1]);
            tmem_ld_wait();
            hide(32, x[0]);
            hide(48, x[1]);
            weights(32, x[0]);
            weights(48, x[1]);
            l += sum.x + sum.y;
            tmem_st_wait();
            // O of the last tile is done by now; a phase that nobody waited for could not be told from the next but one
            if (i > 0) wait(o_done, (i - 1) & 1);
            if (fresh && i > 0) {
                tc_fence_after();
                const float k = m_before == -INFINITY ? 0.0f : ex2(m_before - m), ka = m_acc == -INFINITY ? 0.0f : ex2(m_acc - m);
                constexpr int W = HD >= 64 ? 32 : 16;  // columns at a time
#pragma unroll
                for (int c = 0; c < HD / 2; c += W) {
                    float o[W];
#pragma unroll
                    for (int j = 0; j < W; j += 16)
                        tmem_ld16_nowait(lane_addr + SM::o_col + half * (HD / 2) + c + j, reinterpret_cast<uint32_t *>(o + j));
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < W; j += 4) {
                        float4 *at = acc + (c + j) / 4 * kArM, a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (i > kArWindow) a = *at;
                        *at = make_float4(fmaf(a.x, ka, o[j] * k), fmaf(a.y, ka, o[j + 1] * k), fmaf(a.z, ka, o[j + 2] * k),
                                          fmaf(a.w, ka, o[j + 3] * k));
                    }
                }
                m_acc = m;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[i & 1]);
        }
        l += l_acc;
        // the rows' results (the slot of the last tile but one: its readers have passed a barrier since)
        xch[(nt & 1) * 2 * kArM + half * kArM + row] = l;
        wait(o_done, (nt - 1) & 1);
        tc_fence_after();
        ar_pair_sync(warp & 3);
        l = xch[(nt & 1) * 2 * kArM + row] + xch[(nt & 1) * 2 * kArM + kArM + row];
        const int g = mt * kArM + row;
        const bool real = g / G < w.count;
        const size_t orow = real ? out_row(g) : 0;
        const float inv = p.splits == 1 ? 1.0f / l : 1.0f;
        float *dst = p.splits == 1 ? p.out + orow * HD : p.part + (orow * p.splits + split) * HD;
        if (real && half == 0 && p.splits > 1)
            *reinterpret_cast<float2 *>(p.part_ml + (orow * p.splits + split) * 2) = make_float2(m, l);
        const float ka = m_acc == -INFINITY ? 0.0f : ex2(m_acc - m);
#pragma unroll
        for (int c = 0; c < HD / 2; c += 16) {
            float o[16];
            tmem_ld16_nowait(lane_addr + SM::o_col + half * (HD / 2) + c, reinterpret_cast<uint32_t *>(o));
            tmem_ld_wait();
            if (nt > kArWindow) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 a = acc[(c / 4 + j) * kArM];
                    o[4 * j] = fmaf(a.x, ka, o[4 * j]);
                    o[4 * j + 1] = fmaf(a.y, ka, o[4 * j + 1]);
                    o[4 * j + 2] = fmaf(a.z, ka, o[4 * j + 2]);
                    o[4 * j + 3] = fmaf(a.w, ka, o[4 * j + 3]);
                }
            }
            if (real) {
#pragma unroll
                for (int j = 0; j < 16; j += 4)
                    *reinterpret_cast<float4 *>(dst + half * (HD / 2) + c + j) =
                        make_float4(o[j] * inv, o[j + 1] * inv, o[j + 2] * inv, o[j + 3] * inv);
            }
        }
    } else if (warp < kArMma) {
        // ----------------------------------------------------- expansion
        const int me = warp - 8, t = lane >> 3, e = lane & 7;
        const int data_end = w.pos + w.count;
        // K: a unit is 8 positions (a lane a position and the words t of its groups), two units a warp;
        // V: a unit is a group of 32 dimensions of a cache tile (a lane 8 positions of the dimensions 8 n + e)
        constexpr int KU = kArN / 8 / kArExpand, VU = 4 * NG > kArExpand ? 4 * NG / kArExpand : 1;  // units a warp and tile
        struct Codes {
            uint32_t w[NG], dm[NG];
        } kc[KU];
        struct VCodes {
            uint4 w, d, m;
        } vc[VU];
        // this lane's places in the head's cache, from the tile that is loaded next on; a tile inside the data (all but
        // the last) needs no checks
        const uint8_t *kp[KU], *vp[VU];
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            const int pos = (me * KU + u) * 8 + (e >> 1) + 4 * (e & 1);
            kp[u] = w.k + ((size_t)h * w.tiles + (size_t)t0 * (kArN / kQ4Tile) + pos / kQ4Tile) * q4_tile_bytes(HD) +
                    q4_key_word(NG, pos & 31, t, 0) * 4;
        }
#pragma unroll
        for (int u = 0; u < VU; ++u) {
            const int unit = me * VU + u;
            vp[u] = w.v + ((size_t)h * w.tiles + (size_t)t0 * (kArN / kQ4Tile) + unit / NG) * q4_tile_bytes(HD);
        }
        constexpr int kStep = kArN / kQ4Tile * q4_tile_bytes(HD);
        auto load_keys = [&](int i) {
            const bool inside = (t0 + i + 1) * kArN <= data_end;
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                const int row = ((me * KU + u) * 8 + (e >> 1) + 4 * (e & 1)) & 31;  // of its cache tile
                const uint8_t *wp = kp[u], *dp = kp[u] + q4_code_bytes(HD) + row * NG * 4 - q4_key_word(NG, row, t, 0) * 4;
                if (inside || (t0 + i) * kArN + (me * KU + u) * 8 < data_end) {
                    if (NG == 1) {
                        kc[u].w[0] = *reinterpret_cast<const uint32_t *>(wp);
                        kc[u].dm[0] = *reinterpret_cast<const uint32_t *>(dp);
                    } else if (NG == 2) {
                        *reinterpret_cast<uint2 *>(kc[u].w) = *reinterpret_cast<const uint2 *>(wp);
                        *reinterpret_cast<uint2 *>(kc[u].dm) = *reinterpret_cast<const uint2 *>(dp);
                    } else {
                        *reinterpret_cast<uint4 *>(kc[u].w) = *reinterpret_cast<const uint4 *>(wp);
                        *reinterpret_cast<uint4 *>(kc[u].dm) = *reinterpret_cast<const uint4 *>(dp);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < NG; ++g) kc[u].w[g] = kc[u].dm[g] = 0;
                }
                kp[u] += kStep;
            }
        };
        auto load_values = [&](int i) {
            const bool inside = (t0 + i + 1) * kArN <= data_end;
#pragma unroll
            for (int u = 0; u < VU; ++u) {
                const int unit = me * VU + u, j = unit / NG, g = unit % NG, pos = (t0 + i) * kArN + j * kQ4Tile;
                if (unit < 4 * NG && (inside || pos < data_end)) {
                    vc[u].w = *reinterpret_cast<const uint4 *>(vp[u] + ((g * 8 + e) * 4 + t) * 16);
                    vc[u].d = *reinterpret_cast<const uint4 *>(vp[u] + q4_code_bytes(HD) + g * 128 + t * 16);
                    vc[u].m = *reinterpret_cast<const uint4 *>(vp[u] + q4_code_bytes(HD) + g * 128 + 64 + t * 16);
                    if (!inside) {
                        // what lies behind the data may be anything: its weights are 0, and its values must be numbers
                        const int have = data_end - (pos + 8 * t);  // of these 8 positions
                        uint32_t *d = &vc[u].d.x, *m = &vc[u].m.x;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t keep = (k < have ? 0xFFFFu : 0u) | (k + 4 < have ? 0xFFFF0000u : 0u);
                            d[k] &= keep;
                            m[k] &= keep;
                        }
                    }
                } else {
                    vc[u].w = vc[u].d = vc[u].m = make_uint4(0, 0, 0, 0);
                }
                vp[u] += kStep;
            }
        };
        load_keys(0);
        for (int i = 0; i < nt; ++i) {
            const int st = i & 1;
            load_values(i);
            if (i >= kArStages) wait(&k_empty[st], ((i >> 1) - 1) & 1);
            uint8_t *kf = sm + SM::k_off + st * SM::kTile, *vf = sm + SM::v_off + st * SM::kTile;
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                uint8_t *to = kf + (me * KU + u) * (HD / 8 * 128) + e * 16 + t * 128;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const __half2 D = __low2half2(bits_h2(kc[u].dm[g])), M = __high2half2(bits_h2(kc[u].dm[g]));
                    uint32_t v[4];
                    q4_values(kc[u].w[g], D, M, D, M, D, M, D, M, v);
                    *reinterpret_cast<uint4 *>(to + g * 512) = make_uint4(v[0], v[1], v[2], v[3]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[st]);
            if (i + 1 < nt) load_keys(i + 1);
            if (i >= kArStages) wait(&v_empty[st], ((i >> 1) - 1) & 1);
#pragma unroll
            for (int u = 0; u < VU; ++u) {
                const int unit = me * VU + u, j = unit / NG, g = unit % NG;
                if (unit < 4 * NG) {
                    const uint32_t words[4] = {vc[u].w.x, vc[u].w.y, vc[u].w.z, vc[u].w.w};
#pragma unroll
                    for (int n = 0; n < 4; ++n) {  // dimensions 32 g + 8 n + e
                        uint32_t v[4];
                        q4_values(words[n], bits_h2(vc[u].d.x), bits_h2(vc[u].m.x), bits_h2(vc[u].d.y), bits_h2(vc[u].m.y),
                                  bits_h2(vc[u].d.z), bits_h2(vc[u].m.z), bits_h2(vc[u].d.w), bits_h2(vc[u].m.w), v);
                        *reinterpret_cast<uint4 *>(vf + (4 * g + n) * (kArN / 8 * 128) + (4 * j + t) * 128 + e * 16) =
                            make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
        }
    } else {
        // ---------------------------------------------------------- MMA
        // (the warp goes through the loop together; one elected lane issues)
        const uint32_t base = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint32_t kb = smem_u32(sm + SM::k_off), vb = smem_u32(sm + SM::v_off);
        auto scores = [&](int i) {
            const int st = i & 1;
            wait(&k_full[st], (i >> 1) & 1);
            tc_fence_after();
            if (elect_one()) {
                const uint64_t b = umma_desc(kb + st * SM::kTile, 128, HD / 8 * 128);
                const uint32_t d = base + SM::s_col + st * kArN;
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {  // (a step of 16: 256 bytes, 16 in the descriptor's units)
                    if (k == 0) ar_mma<false>(d, base + SM::q_col + HD / 2, b, ar_idesc(kArN));
                    else ar_mma<true>(d, base + SM::q_col + HD / 2 + 8 * k, b + 16 * k, ar_idesc(kArN));
                }
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) ar_mma<true>(d, base + SM::q_col + 8 * k, b + 16 * k, ar_idesc(kArN));
                tc_commit(&k_empty[st]);
                tc_commit(&s_full[st]);
            }
            __syncwarp();
        };
        scores(0);
        for (int i = 0; i < nt; ++i) {
            const int st = i & 1;
            // S of the next tile goes where P of the last one was: the MMAs that read it are ahead in the same queue
            if (i + 1 < nt) scores(i + 1);
            wait(&v_full[st], (i >> 1) & 1);
            wait(&p_full[st], (i >> 1) & 1);
            tc_fence_after();
            if (elect_one()) {
                const uint64_t b = umma_desc(vb + st * SM::kTile, 128, kArN / 8 * 128);
                const uint32_t pa = base + SM::s_col + st * kArN, d = base + SM::o_col;
                if ((i & (kArWindow - 1)) == 0) ar_mma<false>(d, pa, b, ar_idesc(HD));
                else ar_mma<true>(d, pa, b, ar_idesc(HD));
                ar_mma<true>(d, pa + 8, b, ar_idesc(HD));
#pragma unroll
                for (int k = 1; k < kArN / 16; ++k) {
                    const uint32_t at = pa + k * 16;  // 16 positions: 8 columns of hi, 8 of lo parts
                    ar_mma<true>(d, at, b + 16 * k, ar_idesc(HD));
                    ar_mma<true>(d, at + 8, b + 16 * k, ar_idesc(HD));
                }
                tc_commit(&v_empty[st]);
                tc_commit(o_done);
            }
            __syncwarp();
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kArMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Whether a call is for attention_q4_rows_kernel: more than OVF_Q4_EXACT_ROWS rows (its accumulators fill TMEM at
// head_dim 128), and more chunks of 8 query rows than attention_q4_kernel has CTAs under way, 2 a SM.  That kernel's
// time goes with their number; this one needs 13 us for the first.  (17, 32 and 64 rows of 32 heads over 8, 128 wide,
// in 4 sequences of 4096 positions: 84, 144 and 280 us there, 30, 34 and 54 us here; 17 rows of 14 heads over 2, 64
// wide, in one of 2048, 240 chunks: 10.8 and 14.2 us; 32 rows, 448 chunks: 16.0 and 14.6 us.)
bool attn_q4_many_rows(int n_seq, int rows, int H, int KVH, int hd, int max_ctx, int sms) {
    const int64_t chunks = ((int64_t)rows * (H / KVH) + 7) / 8 * ((max_ctx + 255) / 256);
    return rows > OVF_Q4_EXACT_ROWS && hd <= 128 && chunks * KVH * n_seq > 2 * sms;
}

// Splits of a row's tiles: as many as give each SM a CTA, no more than there are places for partial results.
int attn_q4_rows_splits(int n_seq, int rows, int H, int KVH, int max_ctx, int sms) {
    const int64_t ctas = (int64_t)n_seq * KVH * (((int64_t)rows * (H / KVH) + kArM - 1) / kArM);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min((max_ctx + 255) / 256, 16), sms / ctas));
}

template <int NG>
static cudaError_t launch_ar(const ArParams &p, cudaStream_t st) {
    constexpr int smem = ArSmem<NG>::total;
    static PerDeviceOnce once;
    const int dev = current_device();
    if (once.pending(dev)) {
        const cudaError_t e =
            cudaFuncSetAttribute(attention_q4_rows_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        once.mark(dev);
    }
    const int mtiles = (int)(((int64_t)p.src.rows * (p.H / p.src.KVH) + kArM - 1) / kArM);
    attention_q4_rows_kernel<NG><<<dim3(p.splits, p.src.KVH * mtiles, p.src.n_seq), kArThreads, smem, st>>>(p);
    return cudaGetLastError();
}

}  // namespace ovf
