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
//     leaves a binary32 (maximum, sum) per row part; position-major, so that
//     large batches can skip the rows behind a refused token.
//  2. verify_draw_kernel, one cluster per sequence: decides the tests from
//     those sums where their error bound allows it, sums the first undecided
//     or refused position's rows once more in binary64, decides it exactly, and
//     draws the last token from binary64 running sums.
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
constexpr uint32_t kDrawMaxCtas = 8;  // the largest portable cluster

// Part of a row, as the first launch leaves it: (maximum, sum of exp(v -
// maximum)), or for greedy calls the packed (total-order key, index) of the
// largest logit and whether any logit is finite.
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

// Calls f(index, logit) for this thread's share of p[lo, hi): 16-byte loads
// between the alignment head and tail, kLoads of them in flight.
template <int kThreads, int kLoads, typename BatchF, typename OneF>
__device__ __forceinline__ void visit_segment(const float *p, uint32_t lo, uint32_t hi, BatchF batch,
                                              OneF one) {
    const uint32_t mis = static_cast<uint32_t>((reinterpret_cast<uintptr_t>(p + lo) >> 2) & 3u);
    const uint32_t body = lo + min(hi - lo, (4u - mis) & 3u);
    const uint32_t n4 = (hi - body) / 4u;
    const uint32_t tail = body + 4u * n4;
    if (threadIdx.x < body - lo) one(lo + threadIdx.x, p[lo + threadIdx.x]);
    if (threadIdx.x >= 32 && threadIdx.x - 32 < hi - tail)
        one(tail + threadIdx.x - 32, p[tail + threadIdx.x - 32]);
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
}

// ---------------------------------------------------------------------------
// Launch 1: a CTA per row part.
// ---------------------------------------------------------------------------
struct RowItem {
    uint32_t b, i, part;
    bool draft;
};

// Block index -> (position, sequence, row kind, part), positions slowest.
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

    float m = kNegInf;
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
            sum_batch<16>(m, s, v);
        },
        [&](uint32_t, float x) {
            const float v = masked_scaled(x, c.scale);
            sum_batch<1>(m, s, &v);
        });
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
    uint32_t finite = 0;
    auto visit = [&](uint32_t j, float x) {
        const float v = masked_scaled(x, c.scale);
        const unsigned long long cand = pack_key_index(total_key(v), j);
        best = cand > best ? cand : best;
        finite |= fabsf(x) < kPosInf ? 1u : 0u;
    };
    const float *p = target_row(c, r.b, r.i);
    visit_segment<kRowThreads, 4>(
        p, lo, hi,
        [&](uint32_t body, uint32_t q0, const float4 *x) {
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
// Greedy verification, launch 2: one warp per sequence.
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
        if (!finite) {
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

// exp(d) in binary64 for d <= 0: d = k ln2 / 256 + r with |r| <= ln2 / 512,
// exp(d) = 2^(k/256) * (1 + r + r^2/2 + r^3/6 + r^4/24). The first neglected
// term, r^5/120, is below 4e-17. `tab` holds 2^(j/256). Below -700 the result
// is 0: no such term changes a sum whose largest is 1.
__device__ __forceinline__ double exp64(double d, const double *tab) {
    constexpr double kMagic = 0x1.8p+52;
    if (!(d > -700.0)) return 0.0;
    const double k0 = __fma_rn(d, 256.0 * 1.4426950408889634074, kMagic);
    const int32_t k = __double2loint(k0);
    const double kd = __dsub_rn(k0, kMagic);
    const double r = __fma_rn(kd, -0.69314718055994530942 / 256.0, d);
    double p = __fma_rn(r, 1.0 / 24.0, 1.0 / 6.0);
    p = __fma_rn(p, r, 0.5);
    p = __fma_rn(p, r, 1.0);
    const double t = tab[k & 255];
    const double scaled = __hiloint2double(__double2hiint(t) + ((k >> 8) << 20), __double2loint(t));
    return __fma_rn(scaled, __dmul_rn(p, r), scaled);
}

enum Weight : int {
    kWeightRow = 0,       // p
    kWeightWithout = 1,   // p without one token
    kWeightResidual = 2,  // max(p - q, 0)
};

// What a draw sums over: v of the target row against its maximum, and for the
// residual the draft row's and both reciprocal sums.
struct Draw {
    const float *p;
    const float *q;
    double max_p, max_q;
    double inv_p, inv_q;
    uint32_t without;
    int weight;
};

struct DrawShared {
    double tab[256];
    double warp_sum[kDrawWarps][2];
    // Two sets, used in turn: a CTA may write the next sums while a peer still
    // reads the last ones.
    double cta_sum[2][kDrawMaxCtas][2];
    float warp_max[kDrawWarps];
    float cta_max[kDrawMaxCtas];
    // The position at hand, decided by every CTA of the cluster alike.
    uint32_t first;
    float max_p[kDrawWarps], max_q[kDrawWarps];
    float pos_max_p, pos_max_q;
};

__device__ __forceinline__ double weight_at(const Draw &d, uint32_t j, float scale,
                                            const double *tab) {
    const double e = exp64(static_cast<double>(masked_scaled(d.p[j], scale)) - d.max_p, tab);
    if (d.weight == kWeightResidual) {
        const double f = exp64(static_cast<double>(masked_scaled(d.q[j], scale)) - d.max_q, tab);
        return fmax(e * d.inv_p - f * d.inv_q, 0.0);
    }
    return d.weight == kWeightWithout && j == d.without ? 0.0 : e;
}

// [lo, hi) cut into kDrawWarps runs whose length is a multiple of 32.
__device__ __forceinline__ void warp_run(uint32_t lo, uint32_t hi, uint32_t w, uint32_t &wlo,
                                         uint32_t &whi) {
    const uint32_t len = ((hi - lo + kDrawWarps - 1) / kDrawWarps + 31u) & ~31u;
    wlo = min(hi, lo + w * len);
    whi = min(hi, wlo + len);
}

// This warp's sum of the weights over its run of [lo, hi) into warp_sum[w][0].
__device__ __forceinline__ double run_sum(const Draw &d, uint32_t wlo, uint32_t whi, float scale,
                                          const double *tab) {
    double s = 0.0;
    for (uint32_t j = wlo + (threadIdx.x & 31u); j < whi; j += 32) s += weight_at(d, j, scale, tab);
    return warp_sum(s);
}

__global__ void __launch_bounds__(kDrawThreads)
verify_draw_kernel(const __grid_constant__ VerifyCall c, uint32_t ctas) {
    __shared__ DrawShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank();
    const uint32_t b = blockIdx.x / ctas;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    for (uint32_t j = threadIdx.x; j < 256; j += kDrawThreads) sh.tab[j] = exp2(j / 256.0);
    const uint32_t n = drafts_of(c, b);
    const uint32_t *drafts = c.draft_tokens + static_cast<size_t>(b) * c.max_drafts;
    const uint32_t seg = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const uint32_t lo = min(c.vocab, rank * seg), hi = min(c.vocab, lo + seg);
    uint32_t wlo, whi;
    warp_run(lo, hi, warp, wlo, whi);
    // A CTA's partial sums to every CTA of the cluster, and their total in
    // rank order.
    uint32_t set = 1;
    auto share_sums = [&](double a0, double a1, double &t0, double &t1) {
        set ^= 1u;
        __syncthreads();
        if (lane == 0) {
            sh.warp_sum[warp][0] = a0;
            sh.warp_sum[warp][1] = a1;
        }
        __syncthreads();
        if (threadIdx.x < ctas) {
            double s0 = 0.0, s1 = 0.0;
            for (int w = 0; w < kDrawWarps; ++w) {
                s0 += sh.warp_sum[w][0];
                s1 += sh.warp_sum[w][1];
            }
            double *to = &cluster.map_shared_rank(&sh, threadIdx.x)->cta_sum[set][rank][0];
            to[0] = s0;
            to[1] = s1;
        }
        cluster.sync();
        t0 = t1 = 0.0;
        for (uint32_t r = 0; r < ctas; ++r) {
            t0 += sh.cta_sum[set][r][0];
            t1 += sh.cta_sum[set][r][1];
        }
    };
    cluster.sync();  // every CTA of the cluster runs before its memory is written
    asm volatile("griddepcontrol.wait;" ::: "memory");

    uint32_t a = 0;
    int32_t status = RSC_ROW_OK;
    Draw d{};
    // The weights' sums are left in warp_sum[.][1] and cta_sum[set][.][1].
    double total = 0.0;
    bool refused = false;
    while (true) {
        // The first position at or behind `a` that the binary32 sums do not
        // accept for certain. A warp looks at one position; lanes 0-15 join
        // the target row's parts, lanes 16-31 the draft row's.
        if (threadIdx.x == 0) sh.first = n;
        __syncthreads();
        for (uint32_t i0 = a; i0 < n; i0 += kDrawWarps) {
            const uint32_t i = i0 + warp;
            const bool mine = i < n;
            const bool drafted = lane >= 16;
            float m = kNegInf;
            double s = 0.0;
            if (mine && (c.draft || !drafted) && (lane & 15u) < c.parts) {
                const RowPart &part = static_cast<const RowPart *>(
                    c.row_parts)[row_slot(c, b, i, drafted) * c.parts + (lane & 15u)];
                m = part.max;
                s = part.sum;
            }
            sum_join_lanes(m, s, 16);
            const float mq = __shfl_sync(0xffffffffu, m, 16);
            const double sq = __shfl_sync(0xffffffffu, s, 16);
            if (mine && lane == 0) {
                const uint32_t t = drafts[i];
                bool certain = false;
                const bool valid = fabsf(m) < kPosInf && (!c.draft || fabsf(mq) < kPosInf);
                if (valid && t < c.vocab) {
                    const double u = uniform_of(c, b, i, false);
                    double left = u * s;
                    double right = exp(static_cast<double>(masked_scaled(target_row(c, b, i)[t], c.scale)) - m);
                    if (c.draft) {
                        left *= exp(static_cast<double>(masked_scaled(draft_row(c, b, i)[t], c.scale)) - mq);
                        right *= sq;
                    }
                    // Both sums are within 4e-6 of their values.
                    certain = left * (1.0 + 3e-5) < right;
                }
                if (!certain) atomicMin(&sh.first, i);
                sh.max_p[warp] = m;
                sh.max_q[warp] = mq;
            }
            __syncthreads();
            const uint32_t f = sh.first;
            if (f < n) {
                if (threadIdx.x == 0) {
                    sh.pos_max_p = sh.max_p[f - i0];
                    sh.pos_max_q = sh.max_q[f - i0];
                }
                break;
            }
            __syncthreads();  // everyone has read sh.first
        }
        __syncthreads();
        a = sh.first;
        refused = a < n;
        d.p = target_row(c, b, a);
        float max_p = sh.pos_max_p, max_q = sh.pos_max_q;
        if (!refused) {
            // The row behind the last test has no sums yet: its maximum first.
            float m = kNegInf;
            visit_segment<kDrawThreads, 4>(
                d.p, lo, hi,
                [&](uint32_t, uint32_t, const float4 *x) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        m = fmaxf(fmaxf(m, fmaxf(x[k].x, x[k].y)), fmaxf(x[k].z, x[k].w));
                },
                [&](uint32_t, float x) { m = fmaxf(m, x); });
            m = warp_max(masked_scaled(m, c.scale));
            if (lane == 0) sh.warp_max[warp] = m;
            __syncthreads();
            if (threadIdx.x < ctas) {
                for (int w = 0; w < kDrawWarps; ++w) m = fmaxf(m, sh.warp_max[w]);
                cluster.map_shared_rank(&sh, threadIdx.x)->cta_max[rank] = m;
            }
            cluster.sync();
            max_p = kNegInf;
            for (uint32_t r = 0; r < ctas; ++r) max_p = fmaxf(max_p, sh.cta_max[r]);
        }
        const bool paired = refused && c.draft;
        if (!(fabsf(max_p) < kPosInf) || (paired && !(fabsf(max_q) < kPosInf))) {
            status = RSC_ROW_NO_VALID_TOKENS;
            break;
        }
        d.max_p = max_p;
        d.max_q = max_q;
        d.without = refused ? drafts[a] : 0xffffffffu;
        // Both rows' sums in binary64; without a draft row the second sum is
        // that of the weights.
        double s0 = 0.0, s1 = 0.0;
        if (paired) d.q = draft_row(c, b, a);
        for (uint32_t j = wlo + lane; j < whi; j += 32) {
            const double e = exp64(static_cast<double>(masked_scaled(d.p[j], c.scale)) - d.max_p, sh.tab);
            s0 += e;
            if (paired)
                s1 += exp64(static_cast<double>(masked_scaled(d.q[j], c.scale)) - d.max_q, sh.tab);
            else
                s1 += j == d.without ? 0.0 : e;
        }
        s0 = warp_sum(s0);
        s1 = warp_sum(s1);
        double sum_p, sum_1;
        share_sums(s0, s1, sum_p, sum_1);
        if (!refused) {
            d.weight = kWeightRow;
            total = sum_1;
            break;
        }
        // The exact decision.
        const uint32_t t = drafts[a];
        bool accept = false;
        if (t < c.vocab) {
            const double u = uniform_of(c, b, a, false);
            double left = u * sum_p;
            double right = exp64(static_cast<double>(masked_scaled(d.p[t], c.scale)) - d.max_p, sh.tab);
            if (paired) {
                left *= exp64(static_cast<double>(masked_scaled(d.q[t], c.scale)) - d.max_q, sh.tab);
                right *= sum_1;
            }
            accept = left < right;
        }
        if (accept) {
            ++a;
            continue;
        }
        if (paired) {
            d.weight = kWeightResidual;
            d.inv_p = 1.0 / sum_p;
            d.inv_q = 1.0 / sum_1;
            double unused;
            s1 = run_sum(d, wlo, whi, c.scale, sh.tab);
            share_sums(0.0, s1, unused, total);
        } else {
            d.weight = kWeightWithout;
            total = sum_1;
        }
        if (!(total > 0.0)) {
            // p and q are equal and the token was outside both: p itself.
            d.weight = kWeightRow;
            double unused;
            s1 = run_sum(d, wlo, whi, c.scale, sh.tab);
            share_sums(0.0, s1, unused, total);
        }
        break;
    }

    // The draw: the first index whose running weight exceeds u * total. The
    // CTA whose share of the row holds it goes on alone: its warps' runs, then
    // that run cut again, then one warp over what is left.
    if (rank == 0) {
        uint32_t *out = c.out_tokens + static_cast<size_t>(b) * (c.max_drafts + 1);
        for (uint32_t i = threadIdx.x; i <= c.max_drafts; i += kDrawThreads)
            if (i != a) out[i] = i < a ? drafts[i] : 0xffffffffu;
        if (threadIdx.x == 0) {
            if (status != RSC_ROW_OK) out[a] = 0xffffffffu;
            c.out_accepted[b] = a;
            c.out_status[b] = status;
        }
    }
    const uint32_t tests = a + (refused ? 1u : 0u);
    double want = 0.0;
    if (status == RSC_ROW_OK) {
        want = static_cast<double>(uniform_of(c, b, tests, true)) * total;
        double before = 0.0;
        uint32_t owner = ctas, last = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            const double s = sh.cta_sum[set][r][1];
            if (s > 0.0) last = r;
            if (owner == ctas) {
                if (before + s > want)
                    owner = r;
                else
                    before += s;
            }
        }
        // Rounding can leave u * total at the whole sum: then the last index
        // of positive weight.
        const bool past = owner == ctas;
        if (past) owner = last;
        if (owner == rank) {
            double rest = past ? __longlong_as_double(0x7ff0000000000000ll) : want - before;
            uint32_t flo = lo, fhi = hi;
            while (true) {
                uint32_t w = kDrawWarps, end = 0;
                double prior = 0.0;
                for (int k = 0; k < kDrawWarps; ++k) {
                    const double s = sh.warp_sum[k][1];
                    if (s > 0.0) end = k;
                    if (w == kDrawWarps) {
                        if (prior + s > rest)
                            w = k;
                        else
                            prior += s;
                    }
                }
                if (w == kDrawWarps) {
                    w = end;
                    rest = __longlong_as_double(0x7ff0000000000000ll);
                } else {
                    rest -= prior;
                }
                uint32_t nlo, nhi;
                warp_run(flo, fhi, w, nlo, nhi);
                flo = nlo;
                fhi = nhi;
                if (fhi - flo <= 256) break;
                warp_run(flo, fhi, warp, nlo, nhi);
                const double s = run_sum(d, nlo, nhi, c.scale, sh.tab);
                __syncthreads();
                if (lane == 0) sh.warp_sum[warp][1] = s;
                __syncthreads();
            }
            if (warp == 0) {
                uint32_t token = 0xffffffffu, positive = 0xffffffffu;
                double run = 0.0;
                for (uint32_t j0 = flo; j0 < fhi && token == 0xffffffffu; j0 += 32) {
                    const uint32_t j = j0 + lane;
                    const double w = j < fhi ? weight_at(d, j, c.scale, sh.tab) : 0.0;
                    double cum = w;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const double up = __shfl_up_sync(0xffffffffu, cum, o);
                        if (lane >= static_cast<uint32_t>(o)) cum += up;
                    }
                    cum += run;
                    const uint32_t pos = __ballot_sync(0xffffffffu, w > 0.0);
                    const uint32_t hit = __ballot_sync(0xffffffffu, w > 0.0 && cum > rest);
                    if (pos) positive = j0 + 31u - __clz(pos);
                    if (hit) token = j0 + __ffs(hit) - 1u;
                    run = __shfl_sync(0xffffffffu, cum, 31);
                }
                if (lane == 0)
                    c.out_tokens[static_cast<size_t>(b) * (c.max_drafts + 1) + a] =
                        token != 0xffffffffu ? token : positive;
            }
        }
    }
    // Every CTA has taken its uniforms and its peers' sums.
    cluster.sync();
    if (c.rng_states && !c.uniforms && rank == 0 && threadIdx.x == 0)
        c.rng_states[b] += kWyInc * static_cast<uint64_t>(status == RSC_ROW_OK ? tests + 1u : a);
}

// ---------------------------------------------------------------------------
// Survivor records: one block per sequence.
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

uint32_t verify_parts(size_t rows, uint32_t vocab, int num_sms) {
    // Enough CTAs for six per SM, in parts of at least 2048 logits.
    const size_t want = static_cast<size_t>(num_sms) * 6;
    uint32_t parts = 1;
    while (parts < kVerifyMaxParts && rows * parts < want && vocab / (parts * 2) >= 2048) parts *= 2;
    return parts;
}

size_t verify_workspace_bytes(size_t n_seqs, size_t max_drafts, size_t vocab) {
    size_t parts = 1;
    while (parts < kVerifyMaxParts && vocab / (parts * 2) >= 2048) parts *= 2;
    return n_seqs * (2 * max_drafts + 1) * parts * sizeof(RowPart);
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
    uint32_t ctas = 1;
    while (ctas < kDrawMaxCtas && static_cast<size_t>(c.n_seqs) * ctas < 2u * num_sms &&
           c.vocab / (ctas * 2) >= 2048)
        ctas *= 2;
    cfg.gridDim = dim3(c.n_seqs * ctas, 1, 1);
    cfg.blockDim = dim3(kDrawThreads, 1, 1);
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

cudaError_t launch_verify_records(const VerifyCall &c, cudaStream_t stream) {
    verify_records_kernel<<<c.n_seqs, kListThreads, 0, stream>>>(c);
    return cudaGetLastError();
}

}  // namespace rsc
