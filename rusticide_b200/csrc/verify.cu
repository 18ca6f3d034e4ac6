// Verification of drafted tokens (no counterpart in the reference, whose
// generation loop draws one token per forward pass,
// crates/rusticide-model/src/generate.rs:60-110): the target model has scored
// a sequence's drafted tokens t_0 .. t_{n-1} in one pass, and the longest
// prefix that keeps the output distributed as if the target had been sampled
// token by token is accepted.
//
//   test i, in order:  accept  iff  u_i * q_i(t_i) < p_i(t_i)
//   a = the first refused test, or n
//   token a is drawn from  max(p_a - q_a, 0)  where a was refused (from p_a
//   without t_a where the draft has no distribution, q = 1 at t), from p_n
//   where every token was accepted
//
// p_i and q_i are the softmax of the sampler's scaled logits (fl(x * fl(1/T)),
// NaN read as -inf) over the whole vocabulary, or the lists of survivors that
// a filtered sampling call wrote. Every decision is the one exact arithmetic
// on the given binary32 numbers takes, up to 1e-13 relative.
//
// Whole vocabulary, two launches:
//  1. verify_rows_kernel reads the rows of every test once (HBM-bound) and
//     leaves a binary32 (maximum, sum) per row part. (Ending a sequence's
//     rows at a refusal seen meanwhile was tried: its flags and counters cost
//     what it saved, 126 us against 123 at 96 x 7 x 128256. So was one launch
//     whose clusters sum their sequence's rows position by position and read
//     none behind a refusal: 140 us against 119, and 40 against 27 at 8 x 5 x
//     151936, since so few CTAs keep too few bytes in flight.)
//  2. verify_draw_kernel, one cluster per sequence: decides the tests from
//     those sums where their error bound allows it, sums the first undecided
//     or refused position's rows once more in binary64, decides it exactly, and
//     draws the last token from binary64 running sums.
#include <algorithm>

#include <cooperative_groups.h>

#include "rsc_common.cuh"
#include "rsc_kernels.h"
#include "rsc_rowsum.cuh"

namespace cg = cooperative_groups;

namespace rsc {

namespace {

constexpr int kRowThreads = 256;
constexpr int kDrawThreads = 256;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr uint32_t kDrawMaxCtas = 16;  // the largest cluster (8 is the largest portable one)

// Part of a row, as the first launch leaves it: (m, sum of exp(v - m)) with m
// the largest v (rsc_rowsum.cuh), or for greedy calls the packed
// (total-order key, index) of the largest logit and whether any logit is finite.
struct RowPart {
    union {
        float max;
        unsigned long long best;
    };
    union {
        float sum;
        uint32_t any_finite;
    };
};
static_assert(sizeof(RowPart) == 16, "workspace layout");

// The drafted tokens of sequence b: at least 0, at most max_drafts.
__device__ __forceinline__ uint32_t drafts_of(const VerifyCall &c, uint32_t b) {
    if (!c.n_draft) return c.max_drafts;
    const int32_t n = c.n_draft[b];
    return n <= 0 ? 0u : min(static_cast<uint32_t>(n), c.max_drafts);
}

// Uniform k of sequence b's call: the tests take 0, 1, ..., the last draw
// takes the one behind them (from the caller's array: always its last column).
__device__ __forceinline__ float uniform_of(const VerifyCall &c, uint32_t b, uint32_t k,
                                            bool last_draw) {
    if (c.uniforms)
        return c.uniforms[static_cast<size_t>(b) * (c.max_drafts + 1) + (last_draw ? c.max_drafts : k)];
    uint64_t st = c.rng_states[b] + static_cast<uint64_t>(k) * kWyInc;
    return wyrand_f32(&st);
}

__device__ __forceinline__ const float *target_row(const VerifyCall &c, uint32_t b, uint32_t i) {
    return c.target + b * c.target_seq_stride + i * c.target_row_stride;
}
__device__ __forceinline__ const float *draft_row(const VerifyCall &c, uint32_t b, uint32_t i) {
    return c.draft + b * c.draft_seq_stride + i * c.draft_row_stride;
}

__device__ __forceinline__ float masked_scaled(float x, float scale) {
    return __fmul_rn(fmaxf(x, kNegInf), scale);  // fmaxf(NaN, -inf) = -inf; scale > 0
}

// Calls f(index, logit) for this thread's share of p[lo, hi) in ascending order:
// 16-byte loads between the alignment head and tail, kLoads of them in flight.
template <int kThreads, int kLoads, typename BatchF, typename OneF>
__device__ __forceinline__ void visit_segment(const float *p, uint32_t lo, uint32_t hi, BatchF batch,
                                              OneF one) {
    const uint32_t mis = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(p + lo) >> 2) & 3u);
    const uint32_t body = lo + min(hi - lo, (4u - mis) & 3u);
    const uint32_t n4 = (hi - body) / 4u;
    const uint32_t tail = body + 4u * n4;
    const bool in_tail = threadIdx.x >= 32 && threadIdx.x - 32 < hi - tail;
    const float last = in_tail ? p[tail + threadIdx.x - 32] : kNegInf;
    if (threadIdx.x < body - lo) one(lo + threadIdx.x, p[lo + threadIdx.x]);
    const float4 *p4 = reinterpret_cast<const float4 *>(p + body);
    for (uint32_t q0 = threadIdx.x; q0 < n4; q0 += kThreads * kLoads) {
        float4 x[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const uint32_t q = q0 + k * kThreads;
            x[k] = q < n4 ? __ldg(p4 + q) : make_float4(kNegInf, kNegInf, kNegInf, kNegInf);
        }
        batch(body, q0, x);
    }
    if (in_tail) one(tail + threadIdx.x - 32, last);
}

// ---------------------------------------------------------------------------
// Launch 1: a CTA per row part. Bound by HBM, with sixteen exponentials' worth
// of loads in flight a thread: 96 x 7 x 128256 with ragged drafts (383 of them)
// reads 393 MB in 68 us under a profiler (5.8 TB/s); the greedy form of 64 x 4 x 151936, 195 MB, in 39 us (5.0
// TB/s, the same with 2, 4 and 8 loads in flight and with 4 to 16 parts a row).
// ---------------------------------------------------------------------------
struct RowItem {
    uint32_t b, i, part;
    bool draft;
};

// Block index -> (position, sequence, row kind, part).
__device__ __forceinline__ RowItem row_item(const VerifyCall &c, uint32_t kinds) {
    uint32_t x = blockIdx.x;
    RowItem r;
    r.part = x % c.parts;
    x /= c.parts;
    r.draft = kinds == 2 && (x & 1u);
    x /= kinds;
    r.b = x % c.n_seqs;
    r.i = x / c.n_seqs;
    return r;
}

__device__ __forceinline__ void part_bounds(const VerifyCall &c, uint32_t part, uint32_t &lo,
                                            uint32_t &hi) {
    const uint32_t seg = ((c.vocab + c.parts - 1) / c.parts + 3u) & ~3u;
    lo = min(c.vocab, part * seg);
    hi = min(c.vocab, lo + seg);
}

// Row slots: sequence b's target rows 0..D, then its draft rows 0..D-1.
__device__ __forceinline__ size_t row_slot(const VerifyCall &c, uint32_t b, uint32_t i, bool draft) {
    return static_cast<size_t>(b) * (2u * c.max_drafts + 1u) + (draft ? c.max_drafts + 1u + i : i);
}

__global__ void __launch_bounds__(kRowThreads)
verify_rows_kernel(const __grid_constant__ VerifyCall c) {
    __shared__ float red_m[kRowThreads / 32];
    __shared__ double red_s[kRowThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const RowItem r = row_item(c, c.draft ? 2u : 1u);
    if (r.i >= drafts_of(c, r.b)) return;
    uint32_t lo, hi;
    part_bounds(c, r.part, lo, hi);
    const float *p = r.draft ? draft_row(c, r.b, r.i) : target_row(c, r.b, r.i);

    float m = kNegInf, top = kNegInf;
    double s = 0.0;
    visit_segment<kRowThreads, 4>(
        p, lo, hi,
        [&](uint32_t, uint32_t, const float4 *x) {
            float v[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[4 * k] = masked_scaled(x[k].x, c.scale);
                v[4 * k + 1] = masked_scaled(x[k].y, c.scale);
                v[4 * k + 2] = masked_scaled(x[k].z, c.scale);
                v[4 * k + 3] = masked_scaled(x[k].w, c.scale);
            }
            sum_batch<16>(m, top, s, v);
        },
        [&](uint32_t, float x) {
            const float v = masked_scaled(x, c.scale);
            sum_batch<1>(m, top, s, &v);
        });
    sum_to_top(m, top, s);
    sum_join_lanes(m, s, 32);
    if ((threadIdx.x & 31) == 0) {
        red_m[threadIdx.x >> 5] = m;
        red_s[threadIdx.x >> 5] = s;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        m = threadIdx.x < kRowThreads / 32 ? red_m[threadIdx.x] : kNegInf;
        s = threadIdx.x < kRowThreads / 32 ? red_s[threadIdx.x] : 0.0;
        sum_join_lanes(m, s, kRowThreads / 32);
        if (threadIdx.x == 0) {
            RowPart &out = static_cast<RowPart *>(c.row_parts)[row_slot(c, r.b, r.i, r.draft) * c.parts + r.part];
            out.max = m;
            out.sum = static_cast<float>(s);
        }
    }
}

__global__ void __launch_bounds__(kRowThreads)
verify_greedy_rows_kernel(const __grid_constant__ VerifyCall c) {
    __shared__ unsigned long long red_b[kRowThreads / 32];
    __shared__ uint32_t red_f[kRowThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;");
    const RowItem r = row_item(c, 1u);
    if (r.i > drafts_of(c, r.b)) return;
    uint32_t lo, hi;
    part_bounds(c, r.part, lo, hi);
    unsigned long long best = 0;
    uint32_t best_key = 0, finite = 0;
    auto visit = [&](uint32_t j, float x) {
        // A thread's elements come in ascending order: the last of equal ones stays.
        const uint32_t key = total_key(masked_scaled(x, c.scale));
        if (key >= best_key) best_key = key, best = pack_key_index(key, j);
        finite |= fabsf(x) < kPosInf ? 1u : 0u;
    };
    const float *p = target_row(c, r.b, r.i);
    visit_segment<kRowThreads, 4>(
        p, lo, hi,
        [&](uint32_t body, uint32_t q0, const float4 *x) {
            // The batch's largest key first: few batches hold a new maximum. A
            // thread whose maximum is +inf looks on for finite logits; any other
            // maximum above -inf is one.
            uint32_t top = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t a = max(total_key(masked_scaled(x[k].x, c.scale)),
                                       total_key(masked_scaled(x[k].y, c.scale)));
                const uint32_t b = max(total_key(masked_scaled(x[k].z, c.scale)),
                                       total_key(masked_scaled(x[k].w, c.scale)));
                top = max(top, max(a, b));
            }
            if (top < best_key && best_key < kKeyPosInf) return;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t j = body + 4u * (q0 + k * kRowThreads);
                if (j + 3u >= hi) continue;  // behind the body: nothing was loaded
                visit(j, x[k].x);
                visit(j + 1, x[k].y);
                visit(j + 2, x[k].z);
                visit(j + 3, x[k].w);
            }
        },
        visit);
    best = warp_max(best);
    finite = __reduce_or_sync(0xffffffffu, finite);
    if ((threadIdx.x & 31) == 0) {
        red_b[threadIdx.x >> 5] = best;
        red_f[threadIdx.x >> 5] = finite;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kRowThreads / 32; ++w) {
            best = red_b[w] > best ? red_b[w] : best;
            finite |= red_f[w];
        }
        RowPart &out = static_cast<RowPart *>(c.row_parts)[row_slot(c, r.b, r.i, false) * c.parts + r.part];
        out.best = best;
        out.any_finite = finite;
    }
}

// ---------------------------------------------------------------------------
// Greedy verification, launch 2: one warp per sequence. It reads a few words a
// row and is bound by their latency. What a row answers, and whether it answers, is
// as rsc_pick has it: T = 0 goes by the logits and wants one finite among them, as
// rsc_greedy does; top_k = 1 at another T goes by the scaled logits, as rsc_sample
// does, whose softmax has no value where the largest of them is infinite.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128)
verify_greedy_kernel(const __grid_constant__ VerifyCall c) {
    const uint32_t b = blockIdx.x * 4u + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u;
    if (b >= c.n_seqs) return;
    const uint32_t n = drafts_of(c, b);
    const uint32_t *drafts = c.draft_tokens + static_cast<size_t>(b) * c.max_drafts;
    uint32_t *out = c.out_tokens + static_cast<size_t>(b) * (c.max_drafts + 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t a = 0, token = 0xffffffffu;
    int32_t status = RSC_ROW_OK;
    for (;; ++a) {
        const RowPart *parts = static_cast<const RowPart *>(c.row_parts) + row_slot(c, b, a, false) * c.parts;
        unsigned long long best = lane < c.parts ? parts[lane].best : 0ull;
        const uint32_t finite =
            __reduce_or_sync(0xffffffffu, lane < c.parts ? parts[lane].any_finite : 0u);
        best = warp_max(best);
        const uint32_t key = static_cast<uint32_t>(best >> 32);
        if (c.finite_max ? key <= kKeyNegInf || key >= kKeyPosInf : !finite) {
            status = RSC_ROW_NO_VALID_TOKENS;
            break;
        }
        token = static_cast<uint32_t>(best & 0xffffffffull);
        if (a == n || drafts[a] != token) break;
        if (lane == 0) out[a] = token;
    }
    if (lane == 0) {
        out[a] = status == RSC_ROW_OK ? token : 0xffffffffu;
        c.out_accepted[b] = a;
        c.out_status[b] = status;
    }
    for (uint32_t i = a + 1 + lane; i <= c.max_drafts; i += 32) out[i] = 0xffffffffu;
}

// ---------------------------------------------------------------------------
// Launch 2: decisions and the last token.
// ---------------------------------------------------------------------------

// What exp(v - max) of a row is taken with; `max` is its maximum, or a reference
// that v exceeds by 500 at most. Scaled logits more than 512 below it (-inf and NaN among them)
// are raised to that floor, so that no term needs a branch and none leaves the
// normal numbers. A token whose weight is kNoWeight of the largest or less, 460.5
// or more below it, the floor's 4e-223 among them, is none that a test accepts or a
// draw takes; up to 2^31 of them add up to kNoSum at most.
//
// max - 512 is a binary32 number as long as those below max are 512 apart at
// most, up to 2^33. Beyond, every other token of the row is 512 or more below its
// largest, out of reach of binary64's weights as it is: such a row is scaled down
// by the power of two that leaves exactly 512 between the largest and what is
// next below it, the floor. (Below a power of two itself numbers are half as far
// apart as above it.)
struct RowBase {
    float scale, max32, floor;
    double max;
    __device__ __forceinline__ RowBase() {}
    __device__ __forceinline__ RowBase(float scale_, float max_) : scale(scale_), max32(max_) {
        if (fabsf(max_) >= 0x1p+33f) {
            const int at = ilogbf(max_ > 0.0f ? nextafterf(max_, 0.0f) : max_);
            const float down = scalbnf(1.0f, 32 - at);
            scale *= down;
            max32 *= down;
        }
        floor = max32 - 512.0f;
        max = max32;
    }
};
constexpr double kNoWeight = 1e-200;
constexpr double kNoSum = 1e-190;

constexpr uint32_t kExpSteps = 512;  // entries of the table 2^(j / kExpSteps)

// exp(v - max) in binary64, v = x * scale. With d = v - max = k ln2 / 512 + r
// it is 2^(k/512) * (1 + r + r^2/2 + r^3/6); k comes from d in binary32, which
// leaves |r| below 0.6 ln2 / 512 = 8.2e-4, and the first neglected term, r^4/24,
// below 2e-14. What bounds a pass is the count of instructions (25 with the
// load), then the binary64 rate (six operations at 16 lanes a cycle and
// scheduler), so k is found beside them and the polynomial is two deep.
__device__ __forceinline__ double exp64(float x, const RowBase &b, const double *tab) {
    const float v = fmaxf(__fmul_rn(x, b.scale), b.floor);  // NaN gives the floor
    const float kf = __fmaf_rn(__fsub_rn(v, b.max32), kExpSteps * 1.44269504f, 0x1.8p+23f);
    const uint32_t k = __float_as_uint(kf) - 0x4b400000u;
    const double kd = static_cast<double>(__fsub_rn(kf, 0x1.8p+23f));
    const double d = __dsub_rn(static_cast<double>(v), b.max);
    const double r = __fma_rn(kd, -0.69314718055994530942 / kExpSteps, d);
    const double p = __fma_rn(__dmul_rn(r, r), __fma_rn(r, 1.0 / 6.0, 0.5), r);
    const double t = tab[k % kExpSteps];
    const double scaled = __hiloint2double(
        __double2hiint(t) + static_cast<int>((k & ~(kExpSteps - 1u)) << 11), __double2loint(t));
    return __fma_rn(scaled, p, scaled);
}
static_assert(kExpSteps == 512, "k / 512 goes to bit 20 of the high word");

// The same with the floor's terms as the zeros they stand for.
__device__ __forceinline__ double exp64_or_zero(float x, const RowBase &b, const double *tab) {
    const double e = exp64(x, b, tab);
    return e > kNoWeight ? e : 0.0;
}

enum Weight : int {
    kWeightRow = 0,       // p
    kWeightWithout = 1,   // p without one token
    kWeightResidual = 2,  // max(p - q, 0)
};

// The weights a draw runs over: P = exp(v - max) of the target row, or P -
// kappa Q with Q the same of the draft row and kappa = sum P / sum Q.
struct Draw {
    const float *p;
    const float *q;
    RowBase base_p, base_q;
    double kappa;
    uint32_t without;
    int weight;
};

__device__ __forceinline__ double weight_of(const Draw &d, uint32_t j, float x, float y,
                                            const double *tab) {
    const double e = exp64(x, d.base_p, tab);
    if (d.weight == kWeightResidual) return fmax(e - d.kappa * exp64(y, d.base_q, tab), 0.0);
    return d.weight == kWeightWithout && j == d.without ? 0.0 : e;
}

// The residual in one pass. Its weights need kappa, the quotient of the very
// sums that the pass makes; what is there beforehand is the binary32 sums'
// quotient, within 1.5e-5 of it. That settles for nearly every token whether
// P > kappa Q, so the pass adds up, over the tokens above it, D = P - kappa~ Q
// and Q, and their weight is D + (kappa~ - kappa) Q once kappa is known. The few
// tokens with |P - kappa~ Q| below 2^-16 of kappa~ Q (four of 151936, where the
// rows differ by a normal of width 1/2) are kept apart. A cluster that finds
// more of them than it keeps, as where the rows are equal, sums the weights in
// a second pass.
constexpr uint32_t kNearWarp = 4;  // kept by a warp
constexpr uint32_t kNearCta = 16;  // and by its CTA

// A CTA's sums, as the cluster sees them.
struct CtaSums {
    // Row: sum, reference, maximum. Without: sum, sum without the token.
    // Residual: sum of P, of Q, of D, of Q where D counts. Weights: the sum.
    double s[4];
    uint32_t n_near;  // above kNearCta: too many
    double near[kNearCta][2];
};

struct DrawShared {
    double tab[kExpSteps];
    double warp_sum[kDrawWarps][4];
    double warp_near[kDrawWarps][kNearWarp][2];
    uint32_t warp_n_near[kDrawWarps];
    double cta_near[kNearCta][2];
    double warp_weight[kDrawWarps];
    // Two sets, used in turn: a CTA may write the next sums while a peer still
    // reads the last ones.
    CtaSums cta[2][kDrawMaxCtas];
    // The position at hand, decided by every CTA of the cluster alike.
    uint32_t first;
    float max_p[kDrawWarps], max_q[kDrawWarps];
    double kappa[kDrawWarps];
    // What each warp's position was tested with: u, and both rows' logits of the token.
    float test_u[kDrawWarps], test_p[kDrawWarps], test_q[kDrawWarps];
    uint32_t test_token[kDrawWarps];
    // Weights up to this are none: of CTAs on the row's scale, of tokens on the CTA's.
    double none_row, none;
    float bonus_max;  // the largest scaled logit of the row behind the last test, when that is drawn from
};

// [lo, hi) cut into kDrawWarps runs whose length is a multiple of 32.
__device__ __forceinline__ void warp_run(uint32_t lo, uint32_t hi, uint32_t w, uint32_t &wlo,
                                         uint32_t &whi) {
    const uint32_t len = ((hi - lo + kDrawWarps - 1) / kDrawWarps + 31u) & ~31u;
    wlo = min(hi, lo + w * len);
    whi = min(hi, wlo + len);
}

// Calls f(first index, target logits, draft logits) for the blocks of 32 *
// kLoads elements of a warp's run, lane l holding elements first + 32 k + l
// (single words: the two rows need not share an alignment). Behind the run's
// end the logits read -inf.
template <bool kPair, int kLoads, typename F>
__device__ __forceinline__ void visit_run(const float *p, const float *q, uint32_t wlo, uint32_t whi,
                                          F f) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t j0 = wlo;
    float x[kLoads], y[kLoads];
#pragma unroll 1
    for (; j0 + 32 * kLoads <= whi; j0 += 32 * kLoads) {
        const float *pj = p + j0 + lane;
        const float *qj = q + j0 + lane;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            x[k] = __ldg(pj + 32 * k);
            y[k] = kPair ? __ldg(qj + 32 * k) : kNegInf;
        }
        f(j0, x, y);
    }
    if (j0 < whi) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const uint32_t j = j0 + 32 * k + lane;
            x[k] = j < whi ? __ldg(p + j) : kNegInf;
            y[k] = kPair && j < whi ? __ldg(q + j) : kNegInf;
        }
        f(j0, x, y);
    }
}
constexpr int kRowLoads = 16;  // sixteen exponentials at a time
constexpr int kPairLoads = 8;  // likewise

// This warp's sum of the weights over its run.
__device__ __forceinline__ double run_sum(const Draw &d, uint32_t wlo, uint32_t whi,
                                          const double *tab) {
    double s = 0.0;
    auto add = [&](uint32_t j0, const float *x, const float *y) {
#pragma unroll
        for (int k = 0; k < kPairLoads; ++k)
            s += weight_of(d, j0 + 32 * k + (threadIdx.x & 31u), x[k], y[k], tab);
    };
    if (d.weight == kWeightResidual)
        visit_run<true, kPairLoads>(d.p, d.q, wlo, whi, add);
    else
        visit_run<false, kPairLoads>(d.p, d.q, wlo, whi, add);
    return warp_sum(s);
}

// Inclusive sums over the lanes.
__device__ __forceinline__ double warp_scan(double s) {
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const double up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= static_cast<uint32_t>(o)) s += up;
    }
    return s;
}

// Of the lanes' sums of weights, the first whose running total exceeds `rest`;
// `rest` becomes what is wanted within it. Where rounding leaves none, the last
// lane of any weight, with all of it wanted. The same in every lane.
__device__ __forceinline__ uint32_t locate(double s, double none, double &rest) {
    const bool some = s > none;
    const double upto = warp_scan(s);
    const uint32_t hit = __ballot_sync(0xffffffffu, some && upto > rest);
    const uint32_t any = __ballot_sync(0xffffffffu, some);
    if (hit == 0) {
        rest = __longlong_as_double(0x7ff0000000000000ll);
        return any ? 31u - __clz(any) : 0u;
    }
    const uint32_t at = __ffs(hit) - 1u;
    const double before = __shfl_sync(0xffffffffu, upto, at ? at - 1u : 0u);
    if (at) rest -= before;
    return at;
}

// The weight of a run or a CTA from its residual sums, kappa known.
__device__ __forceinline__ double residual_weight(double sum_d, double sum_q, double slip,
                                                  double kappa, const double (*near)[2],
                                                  uint32_t n_near) {
    double s = sum_d + slip * sum_q;
    for (uint32_t k = 0; k < n_near; ++k) s += fmax(near[k][0] - kappa * near[k][1], 0.0);
    return s;
}

// The first token of weight at `hi` or behind it, else the last one before `lo`; the
// whole block, apart from the draw (whose registers it would cost).
__device__ __noinline__ uint32_t nearest_token(Draw d, uint32_t lo, uint32_t hi, uint32_t vocab, DrawShared &sh) {
    auto counts = [&](uint32_t j) {
        return j < vocab &&
               weight_of(d, j, d.p[j], d.weight == kWeightResidual ? d.q[j] : 0.0f, sh.tab) > kNoWeight;
    };
    if (threadIdx.x == 0) sh.first = vocab;
    bool any = false;
    for (uint32_t k = hi; !any && k < vocab; k += kDrawThreads) {
        const bool hit = counts(k + threadIdx.x);
        any = __syncthreads_or(hit);
        if (hit) atomicMin(&sh.first, k + threadIdx.x);
    }
    if (!any) {
        __syncthreads();
        if (threadIdx.x == 0) sh.first = 0;
        for (uint32_t k = (lo + kDrawThreads - 1) / kDrawThreads; !any && k-- > 0;) {
            const uint32_t j = k * kDrawThreads + threadIdx.x;
            const bool hit = j < lo && counts(j);
            any = __syncthreads_or(hit);
            if (hit) atomicMax(&sh.first, j);
        }
    }
    __syncthreads();
    return sh.first;
}

// 96 x 7 x 128256: 67 us for the 72 MB of rows that it reads a second time. It is
// bound by the latency of its chains of binary64 and table operations at two CTAs
// an SM (issue slots 42 % busy, the binary64 pipe 21 %, DRAM 16 %); more threads,
// CTAs or unrolling, with fewer registers each, took 116-125 us a call alike.
__global__ void __launch_bounds__(kDrawThreads, 2)
verify_draw_kernel(const __grid_constant__ VerifyCall c, uint32_t ctas) {
    extern __shared__ __align__(16) unsigned char draw_smem[];
    DrawShared &sh = *reinterpret_cast<DrawShared *>(draw_smem);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank();
    const uint32_t b = blockIdx.x / ctas;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    for (uint32_t j = threadIdx.x; j < kExpSteps; j += kDrawThreads)
        sh.tab[j] = exp2(static_cast<double>(j) / kExpSteps);
    if (threadIdx.x == 0) {
        sh.none_row = sh.none = kNoWeight;
        sh.bonus_max = kNegInf;
    }
    const uint32_t n = drafts_of(c, b);
    const uint32_t *drafts = c.draft_tokens + static_cast<size_t>(b) * c.max_drafts;
    const uint32_t seg = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const uint32_t lo = min(c.vocab, rank * seg), hi = min(c.vocab, lo + seg);
    uint32_t wlo, whi;
    warp_run(lo, hi, warp, wlo, whi);
    // What a test needs besides the row sums, fetched while those are still
    // being made. A warp looks at one position, lanes 0-15 at its target row,
    // lanes 16-31 at its draft row.
    const bool drafted = lane >= 16;
    auto fetch = [&](uint32_t i, uint32_t &t, float &u, float &x) {
        t = drafts[i];
        u = uniform_of(c, b, i, false);
        x = kNegInf;
        if (t < c.vocab && (c.draft || !drafted))
            x = (drafted ? draft_row(c, b, i) : target_row(c, b, i))[t];
    };
    uint32_t test_token = 0;
    float test_u = 0.0f, test_x = 0.0f;
    if (warp < n) fetch(warp, test_token, test_u, test_x);
    const float last_u = c.uniforms ? uniform_of(c, b, 0, true) : 0.0f;
    cluster.sync();  // every CTA of the cluster runs before its memory is written
    asm volatile("griddepcontrol.wait;" ::: "memory");

    uint32_t set = 1;  // the set of sums in use
    // The CTA's sums (this warp's, every lane alike) to the whole cluster.
    auto share = [&](double s0, double s1, double s2, double s3, uint32_t n_near) {
        set ^= 1u;
        if (lane == 0) {
            sh.warp_sum[warp][0] = s0;
            sh.warp_sum[warp][1] = s1;
            sh.warp_sum[warp][2] = s2;
            sh.warp_sum[warp][3] = s3;
            sh.warp_n_near[warp] = n_near;
        }
        __syncthreads();
        if (warp == 0) {
            const bool in = lane < kDrawWarps;
            double s[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = warp_sum(in ? sh.warp_sum[lane][k] : 0.0);
            // The kept tokens in the order of the warps.
            const uint32_t mine = in ? sh.warp_n_near[lane] : 0u;
            uint32_t upto = min(mine, kNearWarp);
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= static_cast<uint32_t>(o)) upto += up;
            }
            uint32_t count = __shfl_sync(0xffffffffu, upto, 31);
            if (__any_sync(0xffffffffu, mine > kNearWarp) || count > kNearCta) count = kNearCta + 1u;
            if (count <= kNearCta)
                for (uint32_t k = 0; k < min(mine, kNearWarp); ++k) {
                    sh.cta_near[upto - mine + k][0] = sh.warp_near[lane][k][0];
                    sh.cta_near[upto - mine + k][1] = sh.warp_near[lane][k][1];
                }
            __syncwarp();
            if (lane < ctas) {
                CtaSums &to = cluster.map_shared_rank(&sh, lane)->cta[set][rank];
#pragma unroll
                for (int k = 0; k < 4; ++k) to.s[k] = s[k];
                to.n_near = count;
                for (uint32_t k = 0; count <= kNearCta && k < count; ++k) {
                    to.near[k][0] = sh.cta_near[k][0];
                    to.near[k][1] = sh.cta_near[k][1];
                }
            }
        }
        cluster.sync();
    };
    auto cta_sum = [&](int k) { return lane < ctas ? sh.cta[set][lane].s[k] : 0.0; };

    uint32_t a = 0;
    int32_t status = RSC_ROW_OK;
    Draw d{};
    // Filled once the last token's row is settled: the weight of lane r's CTA and
    // their sum, and the weights of this CTA's runs (warp_weight) on its own scale.
    double cta_weight = 0.0, total = 0.0, own_scale = 1.0;
    bool refused = false;
    while (true) {
        // The first position at or behind `a` that the binary32 sums do not
        // accept for certain. A half-warp joins the parts of its row.
        if (threadIdx.x == 0) sh.first = n;
        __syncthreads();
        uint32_t at = 0;  // its warp
        for (uint32_t i0 = a; i0 < n; i0 += kDrawWarps) {
            const uint32_t i = i0 + warp;
            const bool mine = i < n;
            float m = kNegInf;
            double s = 0.0;
            if (mine && (c.draft || !drafted) && (lane & 15u) < c.parts) {
                const RowPart &part = static_cast<const RowPart *>(
                    c.row_parts)[row_slot(c, b, i, drafted) * c.parts + (lane & 15u)];
                m = part.max;
                s = part.sum;
            }
            sum_join_lanes(m, s, 16);
            if (mine && i != warp) fetch(i, test_token, test_u, test_x);
            const double e = fabsf(m) < kPosInf
                                 ? exp64_or_zero(test_x, RowBase(c.scale, m), sh.tab)
                                 : 0.0;
            const float mq = __shfl_sync(0xffffffffu, m, 16);
            const double sq = __shfl_sync(0xffffffffu, s, 16), eq = __shfl_sync(0xffffffffu, e, 16);
            if (mine && lane == 0) {
                bool certain = false;
                const bool valid = fabsf(m) < kPosInf && (!c.draft || fabsf(mq) < kPosInf);
                if (valid && test_token < c.vocab) {
                    const double left = test_u * s * (c.draft ? eq : 1.0);
                    const double right = e * (c.draft ? sq : 1.0);
                    // Each sum is within 7e-6 of its value.
                    certain = left * (1.0 + 3e-5) < right;
                }
                if (!certain) atomicMin(&sh.first, i);
                sh.max_p[warp] = m;
                sh.max_q[warp] = mq;
                sh.kappa[warp] = s / sq;
                sh.test_u[warp] = test_u;
                sh.test_p[warp] = test_x;
                sh.test_token[warp] = test_token;
            }
            if (mine && lane == 16) sh.test_q[warp] = test_x;
            __syncthreads();
            const uint32_t f = sh.first;
            if (f < n) {
                at = f - i0;
                break;
            }
            __syncthreads();  // everyone has read sh.first
        }
        a = sh.first;
        refused = a < n;
        d.p = target_row(c, b, a);
        if (!refused) {
            // The row behind the last test, of which nothing is known yet: each
            // warp sums against the maximum of its first block; binary64 holds
            // terms up to 500 above that, a run with larger ones is summed again (as
            // is any beyond 2^33, whose maximum RowBase has to know).
            float ref = kNegInf, top = kNegInf;
            double s = 0.0;
            while (true) {
                visit_run<false, kRowLoads>(d.p, d.p, wlo, whi, [&](uint32_t, const float *x, const float *) {
                    float m = x[0];
#pragma unroll
                    for (int k = 1; k < kRowLoads; ++k) m = fmaxf(m, x[k]);
                    m = masked_scaled(m, c.scale);
                    top = fmaxf(top, m);
                    if (ref == kNegInf) ref = warp_max(m);
                    if (ref == kNegInf) return;  // nothing but -inf so far
                    const RowBase base(c.scale, ref);
#pragma unroll
                    for (int k = 0; k < kRowLoads; ++k) s += exp64(x[k], base, sh.tab);
                });
                top = warp_max(top);
                if (top == ref || !(top < kPosInf) || static_cast<double>(top) - ref <= 500.0) break;
                ref = top;
                s = 0.0;
            }
            s = warp_sum(s);
            // On the CTA's largest reference.
            if (lane == 0) {
                sh.max_p[warp] = ref;
                sh.max_q[warp] = top;
            }
            __syncthreads();
            const float cta_ref = warp_max(lane < kDrawWarps ? sh.max_p[lane] : kNegInf);
            const float cta_top = warp_max(lane < kDrawWarps ? sh.max_q[lane] : kNegInf);
            s = ref == kNegInf ? 0.0 : s * exp(static_cast<double>(ref) - static_cast<double>(cta_ref));
            share(s, warp == 0 ? static_cast<double>(cta_ref) : 0.0,
                  warp == 0 ? static_cast<double>(cta_top) : 0.0, 0.0, 0u);
            const double refs = lane < ctas ? sh.cta[set][lane].s[1] : -__longlong_as_double(0x7ff0000000000000ll);
            const double row_ref = warp_max(refs);
            const double row_top = warp_max(lane < ctas ? sh.cta[set][lane].s[2] : refs);
            if (!(fabs(row_top) < __longlong_as_double(0x7ff0000000000000ll))) {
                status = RSC_ROW_NO_VALID_TOKENS;
                break;
            }
            d.weight = kWeightRow;
            cta_weight = cta_sum(0) * (lane < ctas ? exp(refs - row_ref) : 0.0);
            d.base_p = RowBase(c.scale, cta_ref);
            own_scale = exp(row_ref - static_cast<double>(cta_ref));
            // References may lie below the row's maximum, which has the say on weights.
            if (threadIdx.x == 0) {
                sh.bonus_max = static_cast<float>(row_top);
                const double none_row = kNoWeight * exp(row_top - row_ref);
                sh.none_row = none_row;
                sh.none = none_row * own_scale;
            }
            if (threadIdx.x < kDrawWarps) sh.warp_weight[threadIdx.x] = sh.warp_sum[threadIdx.x][0];
            total = warp_sum(cta_weight);
            break;
        }
        const float max_p = sh.max_p[at], max_q = sh.max_q[at];
        const double guess = sh.kappa[at];
        const bool paired = c.draft != nullptr;
        if (!(fabsf(max_p) < kPosInf) || (paired && !(fabsf(max_q) < kPosInf))) {
            status = RSC_ROW_NO_VALID_TOKENS;
            break;
        }
        // The rows' own maxima: the same for rows that are the same, which leave
        // nothing of one another, and a row's only likely token has a term of 1.
        d.base_p = RowBase(c.scale, max_p);
        d.base_q = RowBase(c.scale, max_q);
        const uint32_t t = sh.test_token[at];
        const float test_p = sh.test_p[at], test_q = sh.test_q[at];
        const double u = sh.test_u[at];
        d.without = t;
        double s0 = 0.0, s1 = 0.0, s2 = 0.0, s3 = 0.0;
        uint32_t n_near = 0;
        if (paired) {
            d.q = draft_row(c, b, a);
            visit_run<true, kPairLoads>(d.p, d.q, wlo, whi, [&](uint32_t, const float *x, const float *y) {
                double e[kPairLoads], f[kPairLoads];
                bool any = false;
#pragma unroll
                for (int k = 0; k < kPairLoads; ++k) {
                    e[k] = exp64(x[k], d.base_p, sh.tab);
                    f[k] = exp64(y[k], d.base_q, sh.tab);
                }
#pragma unroll
                for (int k = 0; k < kPairLoads; ++k) {
                    s0 += e[k];
                    s1 += f[k];
                    const double g = guess * f[k], over = e[k] - g;
                    // |over| <= 2^-16 g by the high words (up to their last bit).
                    const int32_t high = __double2hiint(over);
                    const bool near = (high & 0x7fffffff) + (16 << 20) <= __double2hiint(g) + 1;
                    any |= near;
                    if (high > 0 && !near) {
                        s2 += over;
                        s3 += f[k];
                    }
                }
                if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                    for (int k = 0; k < kPairLoads; ++k) {
                        const double g = guess * f[k], over = e[k] - g;
                        const bool near = e[k] > kNoWeight && (__double2hiint(over) & 0x7fffffff) + (16 << 20) <=
                                                                  __double2hiint(g) + 1;
                        const uint32_t who = __ballot_sync(0xffffffffu, near);
                        const uint32_t slot = n_near + __popc(who & ((1u << lane) - 1u));
                        if (near && slot < kNearWarp) {
                            sh.warp_near[warp][slot][0] = e[k];
                            sh.warp_near[warp][slot][1] = f[k];
                        }
                        n_near += __popc(who);
                    }
                }
            });
            s2 = warp_sum(s2);
            s3 = warp_sum(s3);
        } else {
            visit_run<false, kRowLoads>(d.p, d.p, wlo, whi, [&](uint32_t j0, const float *x, const float *) {
#pragma unroll
                for (int k = 0; k < kRowLoads; ++k) {
                    const double e = exp64(x[k], d.base_p, sh.tab);
                    s0 += e;
                    s1 += j0 + 32 * k + lane == t ? 0.0 : e;
                }
            });
        }
        s0 = warp_sum(s0);
        s1 = warp_sum(s1);
        share(s0, s1, s2, s3, n_near);
        const double sum_p = warp_sum(cta_sum(0)), sum_1 = warp_sum(cta_sum(1));
        // The exact decision.
        bool accept = false;
        if (t < c.vocab) {
            double left = u * sum_p;
            double right = exp64_or_zero(test_p, d.base_p, sh.tab);
            if (paired) {
                left *= exp64_or_zero(test_q, d.base_q, sh.tab);
                right *= sum_1;
            }
            accept = left < right;
        }
        if (accept) {
            ++a;
            continue;
        }
        if (!paired) {
            d.weight = kWeightWithout;
            cta_weight = cta_sum(1);
            if (threadIdx.x < kDrawWarps) sh.warp_weight[threadIdx.x] = sh.warp_sum[threadIdx.x][1];
            total = warp_sum(cta_weight);
        } else {
            d.weight = kWeightResidual;
            d.kappa = sum_p / sum_1;
            const bool many = lane < ctas && sh.cta[set][lane].n_near > kNearCta;
            if (!__any_sync(0xffffffffu, many)) {
                const double slip = guess - d.kappa;
                cta_weight = lane < ctas ? residual_weight(cta_sum(2), cta_sum(3), slip, d.kappa,
                                                           sh.cta[set][lane].near, sh.cta[set][lane].n_near)
                                         : 0.0;
                if (threadIdx.x < kDrawWarps)
                    sh.warp_weight[threadIdx.x] = residual_weight(
                        sh.warp_sum[threadIdx.x][2], sh.warp_sum[threadIdx.x][3], slip, d.kappa,
                        sh.warp_near[threadIdx.x], sh.warp_n_near[threadIdx.x]);
            } else {
                share(run_sum(d, wlo, whi, sh.tab), 0.0, 0.0, 0.0, 0u);
                cta_weight = cta_sum(0);
                if (threadIdx.x < kDrawWarps) sh.warp_weight[threadIdx.x] = sh.warp_sum[threadIdx.x][0];
            }
            total = warp_sum(cta_weight);
        }
        if (!(total > kNoSum)) {
            // Nothing is left (p and q are equal, the token was outside both): p itself.
            d.weight = kWeightRow;
            share(run_sum(d, wlo, whi, sh.tab), 0.0, 0.0, 0.0, 0u);
            cta_weight = cta_sum(0);
            if (threadIdx.x < kDrawWarps) sh.warp_weight[threadIdx.x] = sh.warp_sum[threadIdx.x][0];
            total = warp_sum(cta_weight);
        }
        break;
    }
    __syncthreads();  // warp_weight and none are complete

    uint32_t *out = c.out_tokens + static_cast<size_t>(b) * (c.max_drafts + 1);
    if (rank == 0) {
        for (uint32_t i = threadIdx.x; i <= c.max_drafts; i += kDrawThreads)
            if (i != a) out[i] = i < a ? drafts[i] : 0xffffffffu;
        if (threadIdx.x == 0) {
            if (status != RSC_ROW_OK) out[a] = 0xffffffffu;
            c.out_accepted[b] = a;
            c.out_status[b] = status;
        }
    }
    // The draw: the first index whose running weight exceeds u * total. The CTA
    // whose share of the row holds it goes on alone: the run of one of its
    // warps, cut again while it is longer than kTail elements a thread.
    const uint32_t tests = a + (refused ? 1u : 0u);
    if (status == RSC_ROW_OK) {
        constexpr uint32_t kTail = 8;
        double rest = static_cast<double>(c.uniforms ? last_u : uniform_of(c, b, tests, true)) * total;
        if (locate(cta_weight, sh.none_row, rest) == rank) {
            rest *= own_scale;
            uint32_t flo = lo, fhi = hi;
            while (true) {
                const uint32_t w = locate(lane < kDrawWarps ? sh.warp_weight[lane] : 0.0, sh.none, rest);
                uint32_t nlo, nhi;
                warp_run(flo, fhi, w, nlo, nhi);
                flo = nlo;
                fhi = nhi;
                if (fhi - flo <= kTail * kDrawThreads) break;
                warp_run(flo, fhi, warp, nlo, nhi);
                const double s = run_sum(d, nlo, nhi, sh.tab);
                __syncthreads();
                if (lane == 0) sh.warp_weight[warp] = s;
                __syncthreads();
            }
            const uint32_t each = (fhi - flo + kDrawThreads - 1) / kDrawThreads;
            const uint32_t j0 = flo + threadIdx.x * each;
            double w[kTail], sum = 0.0;
#pragma unroll
            for (uint32_t k = 0; k < kTail; ++k) {
                const uint32_t j = j0 + k;
                w[k] = 0.0;
                if (k < each && j < fhi) {
                    w[k] = weight_of(d, j, d.p[j], d.weight == kWeightResidual ? d.q[j] : 0.0f, sh.tab);
                    if (!(w[k] > sh.none)) w[k] = 0.0;
                }
                sum += w[k];
            }
            const double upto = warp_scan(sum);
            if (__syncthreads_or(sum > 0.0)) {
                if (lane == 31) sh.warp_weight[warp] = upto;
                __syncthreads();
                if (locate(lane < kDrawWarps ? sh.warp_weight[lane] : 0.0, 0.0, rest) == warp &&
                    locate(sum, 0.0, rest) == lane) {
                    double run = 0.0;
                    uint32_t token = j0;
                    bool found = false;
#pragma unroll
                    for (uint32_t k = 0; k < kTail; ++k) {
                        if (found || w[k] == 0.0) continue;
                        run += w[k];
                        token = j0 + k;
                        found = run > rest;
                    }
                    out[a] = token;
                }
            } else {
                // The run was found for the sum of tokens that are none by themselves: a
                // draw of u = 0, or the sums' rounding at a row's end. The first
                // token of weight behind it is meant, or the last one before it (one of
                // them exists, the total being above kNoSum).
                if (sh.bonus_max != kNegInf) d.base_p = RowBase(c.scale, sh.bonus_max);
                const uint32_t token = nearest_token(d, flo, fhi, c.vocab, sh);
                if (threadIdx.x == 0) out[a] = token;
            }
        }
    }
    if (c.rng_states) {
        // Every CTA has taken its draws from the state.
        cluster.sync();
        if (rank == 0 && threadIdx.x == 0)
            c.rng_states[b] += kWyInc * static_cast<uint64_t>(status == RSC_ROW_OK ? tests + 1u : a);
    }
}

// ---------------------------------------------------------------------------
// Survivor records: one block per sequence, a warp per test, then one warp that
// draws. The lists are short (top_k and its ties), so the call is bound by the
// chain of dependent loads (token, list, bisection in the draft's list) and the
// launch: one sequence of 4 drafts over 64 slots 5.8 us, 512 of 6 over 152 slots
// 14.9 us.
// ---------------------------------------------------------------------------
constexpr int kListThreads = 128;
constexpr int kListWarps = kListThreads / 32;

// The probability of `token` in a record (0 when it is not listed): a warp
// looks through the list.
__device__ __forceinline__ float record_prob(const uint32_t *ids, const float *probs, uint32_t n,
                                             uint32_t token) {
    float found = 0.0f;
    for (uint32_t j0 = 0; j0 < n; j0 += 32) {
        const uint32_t j = j0 + (threadIdx.x & 31u);
        const bool hit = j < n && ids[j] == token;
        const uint32_t who = __ballot_sync(0xffffffffu, hit);
        if (who) {
            found = __shfl_sync(0xffffffffu, hit ? probs[j] : 0.0f, __ffs(who) - 1);
            break;
        }
    }
    return found;
}

// The probability of `token` in a record by bisection (ids ascending).
__device__ __forceinline__ float record_find(const uint32_t *ids, const float *probs, uint32_t n,
                                             uint32_t token) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (ids[mid] < token)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo < n && ids[lo] == token ? probs[lo] : 0.0f;
}

__global__ void __launch_bounds__(kListThreads)
verify_records_kernel(const __grid_constant__ VerifyCall c) {
    __shared__ uint32_t first;
    const uint32_t b = blockIdx.x;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t n = drafts_of(c, b);
    const uint32_t *drafts = c.draft_tokens + static_cast<size_t>(b) * c.max_drafts;
    if (threadIdx.x == 0) first = n;
    __syncthreads();
    // The row's status: the record must hold a whole distribution.
    auto row_status = [&](const VerifyRecords &rec, size_t row) -> int32_t {
        if (rec.status && (rec.status[row] & 0xff) != RSC_ROW_OK) return rec.status[row] & 0xff;
        if (rec.n[row] > rec.cap) return RSC_ROW_INTERNAL;
        return rec.n[row] == 0 ? RSC_ROW_NO_VALID_TOKENS : RSC_ROW_OK;
    };
    for (uint32_t i0 = 0; i0 < n; i0 += kListWarps) {
        const uint32_t i = i0 + warp;
        if (i < n) {
            const size_t row = static_cast<size_t>(b) * (c.max_drafts + 1) + i;
            const size_t row_q = static_cast<size_t>(b) * c.max_drafts + i;
            bool accept = row_status(c.target_rec, row) == RSC_ROW_OK &&
                          (!c.draft_rec.n || row_status(c.draft_rec, row_q) == RSC_ROW_OK);
            if (accept) {
                const uint32_t t = drafts[i];
                const float p = record_prob(c.target_rec.ids + row * c.target_rec.cap,
                                            c.target_rec.probs + row * c.target_rec.cap,
                                            c.target_rec.n[row], t);
                const float q = c.draft_rec.n ? record_prob(c.draft_rec.ids + row_q * c.draft_rec.cap,
                                                            c.draft_rec.probs + row_q * c.draft_rec.cap,
                                                            c.draft_rec.n[row_q], t)
                                              : 1.0f;
                // A product of two binary32 numbers is exact in binary64.
                accept = static_cast<double>(uniform_of(c, b, i, false)) * q < static_cast<double>(p);
            }
            if (!accept && lane == 0) atomicMin(&first, i);
        }
        __syncthreads();
        if (first < n) break;
        __syncthreads();
    }
    __syncthreads();
    const uint32_t a = first;
    const bool refused = a < n;
    const size_t row = static_cast<size_t>(b) * (c.max_drafts + 1) + a;
    const size_t row_q = static_cast<size_t>(b) * c.max_drafts + a;
    const bool paired = refused && c.draft_rec.n;
    int32_t status = row_status(c.target_rec, row);
    if (status == RSC_ROW_OK && paired) status = row_status(c.draft_rec, row_q);
    uint32_t *out = c.out_tokens + static_cast<size_t>(b) * (c.max_drafts + 1);
    for (uint32_t i = threadIdx.x; i <= c.max_drafts; i += kListThreads)
        if (i != a) out[i] = i < a ? drafts[i] : 0xffffffffu;
    if (warp != 0) return;
    // One warp draws: 32 entries at a time, twice over the list (the sum,
    // then the running sum).
    const uint32_t *ids = c.target_rec.ids + row * c.target_rec.cap;
    const float *probs = c.target_rec.probs + row * c.target_rec.cap;
    const uint32_t len = status == RSC_ROW_OK ? c.target_rec.n[row] : 0u;
    const uint32_t without = refused ? drafts[a] : 0xffffffffu;
    bool whole = !refused;
    auto weight = [&](uint32_t j) -> double {
        const double p = static_cast<double>(probs[j]);
        if (whole) return p;
        if (!paired) return ids[j] == without ? 0.0 : p;
        const double q = record_find(c.draft_rec.ids + row_q * c.draft_rec.cap,
                                     c.draft_rec.probs + row_q * c.draft_rec.cap,
                                     c.draft_rec.n[row_q], ids[j]);
        return fmax(p - q, 0.0);
    };
    double total = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
        double s = 0.0;
        for (uint32_t j = lane; j < len; j += 32) s += weight(j);
        total = warp_sum(s);
        if (total > 0.0) break;
        whole = true;  // nothing is left of p - q: p itself
    }
    const uint32_t tests = a + (refused ? 1u : 0u);
    uint32_t token = 0xffffffffu, positive = 0xffffffffu;
    if (status == RSC_ROW_OK) {
        const double want = static_cast<double>(uniform_of(c, b, tests, true)) * total;
        double run = 0.0;
        for (uint32_t j0 = 0; j0 < len && token == 0xffffffffu; j0 += 32) {
            const uint32_t j = j0 + lane;
            const double w = j < len ? weight(j) : 0.0;
            double cum = w;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double up = __shfl_up_sync(0xffffffffu, cum, o);
                if (lane >= static_cast<uint32_t>(o)) cum += up;
            }
            cum += run;
            const uint32_t pos = __ballot_sync(0xffffffffu, w > 0.0);
            const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && cum > want);
            if (pos) positive = ids[j0 + 31u - __clz(pos)];
            if (hit) token = ids[j0 + __ffs(hit) - 1u];
            run = __shfl_sync(0xffffffffu, cum, 31);
        }
        if (token == 0xffffffffu) token = positive;
        if (token == 0xffffffffu) status = RSC_ROW_NO_VALID_TOKENS;  // a record without weight
    }
    if (lane == 0) {
        out[a] = token;
        c.out_accepted[b] = a;
        c.out_status[b] = status;
        if (c.rng_states && !c.uniforms)
            c.rng_states[b] += kWyInc * static_cast<uint64_t>(status == RSC_ROW_OK ? tests + 1u : a);
    }
}

}  // namespace

// Parts of a row. A batch whose rows are fewer than the CTAs that fit the GPU
// at once (six per SM) is spread over one wave of them, in parts of at least
// 2048 logits; a larger one is cut into parts of about 32768.
uint32_t verify_parts(size_t rows, uint32_t vocab, int num_sms) {
    const size_t wave = static_cast<size_t>(num_sms) * 6;
    size_t parts = rows < wave ? wave / (rows ? rows : 1) : 1;
    parts = std::max<size_t>(parts, (static_cast<size_t>(vocab) + 32767) / 32768);
    parts = std::min<size_t>(parts, std::max<uint32_t>(1u, vocab / 2048));
    return static_cast<uint32_t>(std::min<size_t>(parts, kVerifyMaxParts));
}

size_t verify_workspace_bytes(size_t n_seqs, size_t max_drafts, size_t vocab) {
    const size_t parts = std::min<size_t>(kVerifyMaxParts, std::max<size_t>(1, vocab / 2048));
    return n_seqs * (2 * max_drafts + 1) * parts * sizeof(RowPart);
}

// CTAs a sequence is drawn by. Few sequences take as many as leave the GPU's
// SMs one or two each (16 is the largest cluster, above 8 only where the whole
// of it finds room); more take slices of about 24576 tokens, whose uneven
// lengths (a refused token reads two rows, an accepted draft one) even out.
// Measured, us a call: 8 x 5 x 151936 27.5 with 16 CTAs, 35.7 with 8; 32 x 8 x
// 50001 20.3 with 6, 25.8 with 8; 96 x 7 x 128256 120 with 6, 138 with 2.
uint32_t draw_ctas(uint32_t n_seqs, uint32_t vocab, int num_sms) {
    const uint32_t room = static_cast<uint32_t>(num_sms) * 4u / 3u / n_seqs;
    uint32_t ctas = room >= 16 ? 16u : std::min(room, 8u);
    ctas = std::max(ctas, std::min(8u, (vocab + 24575u) / 24576u));
    return std::max(1u, std::min(ctas, vocab / 1024u));
}

cudaError_t launch_verify(const VerifyCall &call, bool greedy, int num_sms, uint64_t *launches,
                          cudaStream_t stream) {
    VerifyCall c = call;
    const size_t row_count = static_cast<size_t>(c.n_seqs) *
                             (greedy ? c.max_drafts + 1 : c.max_drafts * (c.draft ? 2u : 1u));
    c.parts = verify_parts(row_count, c.vocab, num_sms);
    cudaError_t e = cudaSuccess;
    if (row_count > 0) {
        const unsigned grid = static_cast<unsigned>(row_count * c.parts);
        if (greedy)
            verify_greedy_rows_kernel<<<grid, kRowThreads, 0, stream>>>(c);
        else
            verify_rows_kernel<<<grid, kRowThreads, 0, stream>>>(c);
        ++*launches;
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
    }
    // The second launch may become resident while the first drains; it reads
    // the first's results behind griddepcontrol.wait.
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = stream;
    cfg.attrs = attr;
    ++*launches;
    if (greedy) {
        cfg.gridDim = dim3((c.n_seqs + 3) / 4, 1, 1);
        cfg.blockDim = dim3(128, 1, 1);
        cfg.numAttrs = row_count > 0 ? 1 : 0;
        return cudaLaunchKernelEx(&cfg, verify_greedy_kernel, c);
    }
    const uint32_t ctas = draw_ctas(c.n_seqs, c.vocab, num_sms);
    cfg.gridDim = dim3(c.n_seqs * ctas, 1, 1);
    cfg.blockDim = dim3(kDrawThreads, 1, 1);
    cfg.dynamicSmemBytes = sizeof(DrawShared);
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    if (row_count > 0) {
        cfg.numAttrs = 2;
    } else {
        cfg.attrs = attr + 1;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, verify_draw_kernel, c, ctas);
}

cudaError_t verify_setup() {
    return cudaFuncSetAttribute(verify_draw_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

cudaError_t launch_verify_records(const VerifyCall &c, cudaStream_t stream) {
    verify_records_kernel<<<c.n_seqs, kListThreads, 0, stream>>>(c);
    return cudaGetLastError();
}

}  // namespace rsc
