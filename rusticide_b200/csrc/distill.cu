// Distillation from a teacher's top tokens (no counterpart in the reference,
// which serves only): the loss of a student's logits against the teacher's
// listed log-probabilities, and its gradient.
//
// With v = x * s (s = fl(1/T)), S = sum_j exp(v_j), p_j = exp(v_j) / S, and the
// row's teacher entries (id_k, y_k):
//   renormalised   t_k = exp(y_k) / sum exp(y),  r = 0,                M = 1
//   with the tail  t_k = exp(y_k),  r = max(0, 1 - sum t),  M = max(1, sum t)
//   loss = sum_k t_k (log t_k - log p_k) + r (log r - log(S_tail / S))
//   d loss / d x_j = s (p_j M - t_j) on a listed token,
//                    s (p_j M - r exp(v_j) / S_tail) on any other,
// S_tail being the sum over the tokens that are not listed. Both terms of the
// second are multiples of exp(v_j - m), m the largest unlisted v: one
// exponential a token, and none that vanishes where the tail's share does.
//
// A row is spread over a cluster of CTAs that join their sums through
// distributed shared memory. S_tail is summed over the unlisted tokens as such
// (a bitmap of the listed ones masks them out): S minus the listed terms would
// lose it where the listed tokens hold nearly all of the mass. Sums leave a
// thread's batch of 16 in binary64 (rsc_rowsum.cuh), what is computed per row
// or per entry is binary64 throughout.
#include <cooperative_groups.h>

#include "rsc_common.cuh"
#include "rsc_kernels.h"
#include "rsc_rowsum.cuh"

namespace cg = cooperative_groups;

namespace rsc {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kMaxCtas = 8;  // the largest portable cluster
constexpr uint32_t kLoads = 4;    // 16-byte loads in flight per thread

// One CTA's contribution to its row, shared with the whole cluster.
struct RowShare {
    float max_rest, max_listed;  // over the tokens summed in the pass; over the listed ones
    double sum_rest, sum_listed;
    double cross, held;  // sums of t (log t - v) and of t over the CTA's entries
};

struct DistillShared {
    uint32_t id[kDistillMaxTop];
    float t[kDistillMaxTop];  // teacher probability
    float v[kDistillMaxTop];  // scaled student logit (entries of this CTA's segment)
    float y[kDistillMaxTop];  // teacher log-probability as given
    float red_m[kWarps];
    double red_s[kWarps];
    RowShare share[kMaxCtas];
    double log_norm;  // log t = y - log_norm
    double r, mass;
    uint32_t some, unordered;
    // The row as the gradient needs it: p = exp(v - max) * inv on the listed
    // tokens, exp(v - rest_max) * rest_factor the whole term on the others.
    float max, inv, rest_max, rest_factor;
};

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// The id of an absent entry: one outside the vocabulary, or of no probability.
constexpr uint32_t kAbsent = 0xffffffffu;

// The teacher's list of a row: ids, t and the sums over them.
__device__ __forceinline__ uint32_t load_teacher(const DistillCall &c, size_t row, DistillShared &sh) {
    uint32_t n = static_cast<uint32_t>(c.cap);
    if (c.n) n = min(n, c.n[row]);
    for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
        const uint32_t id = c.ids[row * c.cap + k];
        const float y = c.logprobs[row * c.cap + k];
        sh.id[k] = id < c.vocab && y != kNegInf ? id : kAbsent;
        sh.y[k] = y;
    }
    if (threadIdx.x == 0) sh.unordered = 0;
    __syncthreads();
    // Lists in ascending order hold no id twice.
    for (uint32_t k = threadIdx.x; k + 1 < n; k += kThreads)
        if (!(sh.id[k] < sh.id[k + 1]) && sh.id[k + 1] != kAbsent) sh.unordered = 1;
    if (threadIdx.x < 32) {
        float top = kNegInf;
        bool some = false;
        for (uint32_t k = threadIdx.x; k < n; k += 32)
            if (sh.id[k] != kAbsent) {
                top = fmaxf(top, sh.y[k]);
                some = true;
            }
        top = warp_max(top);
        some = __any_sync(0xffffffffu, some);
        // With the tail the values are log-probabilities as such.
        const double ref = c.tail || !(fabsf(top) < kPosInf) ? 0.0 : static_cast<double>(top);
        double sum = 0.0;
        for (uint32_t k = threadIdx.x; k < n; k += 32)
            if (sh.id[k] != kAbsent) sum += exp(static_cast<double>(sh.y[k]) - ref);
        sum = warp_sum(sum);
        if (threadIdx.x == 0) {
            sh.some = some ? 1u : 0u;
            if (c.tail) {
                sh.log_norm = 0.0;
                sh.r = sum < 1.0 ? 1.0 - sum : 0.0;
                sh.mass = sum > 1.0 ? sum : 1.0;
            } else {
                sh.log_norm = ref + log(sum);
                sh.r = 0.0;
                sh.mass = 1.0;
            }
        }
    }
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n; k += kThreads)
        sh.t[k] = sh.id[k] != kAbsent
                      ? static_cast<float>(exp(static_cast<double>(sh.y[k]) - sh.log_norm))
                      : 0.0f;
    return n;
}

// Entry k is the first of its id, and the sum of t over the entries of that
// id in list order (ids may repeat: each entry counts).
__device__ __forceinline__ bool first_of_id(const DistillShared &sh, uint32_t n, uint32_t k,
                                            float &t_sum) {
    t_sum = sh.t[k];
    if (!sh.unordered) return true;
    const uint32_t id = sh.id[k];
    double sum = 0.0;
    bool first = true;
    for (uint32_t q = 0; q < n; ++q) {
        if (sh.id[q] != id) continue;
        first &= q >= k;
        sum += static_cast<double>(sh.t[q]);
    }
    t_sum = static_cast<float>(sum);
    return first;
}

// A row segment of T cut at 16-byte boundaries: [lo, body) and [tail, hi)
// element by element, n_vec 16-byte words from body on.
template <typename T>
struct Segment {
    uint32_t lo, hi, body, tail, n_vec;
    __device__ __forceinline__ Segment(const T *p, uint32_t lo_, uint32_t hi_) : lo(lo_), hi(hi_) {
        constexpr uint32_t kE = kVecElems<T>;
        const uint32_t off =
            static_cast<uint32_t>((reinterpret_cast<uintptr_t>(p + lo) / sizeof(T)) % kE);
        body = lo + min(hi - lo, (kE - off) % kE);
        n_vec = (hi - body) / kE;
        tail = body + n_vec * kE;
    }
};

template <typename T, bool kForward, bool kGrad>
__global__ void __launch_bounds__(kThreads)
distill_kernel(const __grid_constant__ DistillCall c, uint32_t ctas) {
    extern __shared__ uint32_t bits[];  // one per element of the segment, set where it is listed
    __shared__ DistillShared sh;
    constexpr uint32_t kE = kVecElems<T>;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank();
    const size_t row = blockIdx.x / ctas;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const T *x = static_cast<const T *>(c.logits) + row * c.row_stride;
    const uint32_t seg_len = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const uint32_t lo = min(c.vocab, rank * seg_len), hi = min(c.vocab, lo + seg_len);
    const Segment<T> seg(x, lo, hi);
    const uint32_t n = load_teacher(c, row, sh);
    // Every CTA of the cluster runs before its memory is written (the row is
    // empty for all of them or for none).
    if (kForward && sh.some) cluster.barrier_arrive();
    auto here = [&](uint32_t id) { return id >= lo && id < hi; };
    const bool empty = sh.some == 0;
    const bool masked = kForward && c.tail;
    float *state = c.state ? c.state + row * 4 : nullptr;

    // The entries' student logits, before anything is written (the gradient
    // may replace the logits).
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n; k += kThreads)
        sh.v[k] = here(sh.id[k]) ? __fmul_rn(elem_to_float<T>(x[sh.id[k]]), c.scale) : kNegInf;

    if (kForward && !empty) {
        // Bit b stands for element body - pad + b, so that a word's elements
        // start at a multiple of kE.
        const uint32_t pad = (32u - ((seg.body - lo) & 31u)) & 31u;
        if (masked) {
            for (uint32_t w = threadIdx.x; w < (hi - lo + pad + 31u) / 32u; w += kThreads) bits[w] = 0;
            __syncthreads();
            for (uint32_t k = threadIdx.x; k < n; k += kThreads)
                if (here(sh.id[k])) {
                    const uint32_t b = sh.id[k] - lo + pad;
                    atomicOr(&bits[b / 32u], 1u << (b % 32u));
                }
        }
        __syncthreads();
        float m = kNegInf;
        double s = 0.0;
        auto one = [&](uint32_t j) {
            const uint32_t b = j - lo + pad;
            if (masked && (bits[b / 32u] >> (b % 32u) & 1u)) return;
            const float v = __fmul_rn(elem_to_float<T>(x[j]), c.scale);
            sum_batch<1>(m, s, &v);
        };
        if (threadIdx.x < seg.body - lo) one(lo + threadIdx.x);
        if (threadIdx.x >= 32 && threadIdx.x - 32 < hi - seg.tail) one(seg.tail + threadIdx.x - 32);
        const uint4 *words = reinterpret_cast<const uint4 *>(x + seg.body);
        for (uint32_t q0 = threadIdx.x; q0 < seg.n_vec; q0 += kThreads * kLoads) {
            uint4 w[kLoads];
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) {
                const uint32_t q = q0 + k * kThreads;
                w[k] = q < seg.n_vec ? words[q] : make_uint4(0, 0, 0, 0);
            }
            float v[kLoads * kE];
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) {
                const uint32_t q = q0 + k * kThreads;
                unpack<T>(w[k], v + k * kE);
#pragma unroll
                for (uint32_t i = 0; i < kE; ++i)
                    v[k * kE + i] = q < seg.n_vec ? __fmul_rn(v[k * kE + i], c.scale) : kNegInf;
                if (masked && q < seg.n_vec) {
                    const uint32_t b = seg.body - lo + pad + q * kE;
                    const uint32_t set = bits[b / 32u] >> (b % 32u) & ((1u << kE) - 1u);
                    if (set) {
#pragma unroll
                        for (uint32_t i = 0; i < kE; ++i)
                            if (set >> i & 1u) v[k * kE + i] = kNegInf;
                    }
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < kLoads * kE; k += 16) sum_batch<16>(m, s, v + k);
        }
        sum_join_lanes(m, s, 32);
        if (lane == 0) {
            sh.red_m[warp] = m;
            sh.red_s[warp] = s;
        }
        __syncthreads();
        cluster.barrier_wait();
        if (warp == 0) {
            m = lane < kWarps ? sh.red_m[lane] : kNegInf;
            s = lane < kWarps ? sh.red_s[lane] : 0.0;
            sum_join_lanes(m, s, kWarps);
            // The entries of this segment: their part of the loss, and with the
            // tail their own sum, each id once.
            float ml = kNegInf;
            double sl = 0.0, cross = 0.0, held = 0.0;
            for (uint32_t k = lane; k < n; k += 32) {
                if (!here(sh.id[k])) continue;
                const double v = sh.v[k];
                float t_sum;
                if (masked && first_of_id(sh, n, k, t_sum)) sum_join(ml, sl, sh.v[k], sh.v[k] == kNegInf ? 0.0 : 1.0);
                if (sh.t[k] == 0.0f) continue;
                cross += static_cast<double>(sh.t[k]) * (static_cast<double>(sh.y[k]) - sh.log_norm - v);
                held += static_cast<double>(sh.t[k]);
            }
            sum_join_lanes(ml, sl, 32);
            cross = warp_sum(cross);
            held = warp_sum(held);
            if (lane < ctas) {
                RowShare &to = cluster.map_shared_rank(&sh, lane)->share[rank];
                to.max_rest = m;
                to.sum_rest = s;
                to.max_listed = ml;
                to.sum_listed = sl;
                to.cross = cross;
                to.held = held;
            }
        }
        cluster.sync();
        if (threadIdx.x == 0) {
            float mr = kNegInf, ma = kNegInf;
            double sr = 0.0, sa = 0.0, loss = 0.0, held = 0.0;
            for (uint32_t r = 0; r < ctas; ++r) {
                sum_join(mr, sr, sh.share[r].max_rest, sh.share[r].sum_rest);
                sum_join(ma, sa, sh.share[r].max_listed, sh.share[r].sum_listed);
                loss += sh.share[r].cross;
                held += sh.share[r].held;
            }
            sum_join(ma, sa, mr, sr);
            // A row of -inf alone has no distribution: NaN, as a NaN or +inf
            // logit gives through the sum.
            if (!(sa > 0.0)) sa = __longlong_as_double(0x7ff8000000000000ll);
            const double lse = static_cast<double>(ma) + log(sa);
            loss += held * lse;
            // The unlisted tokens' factor against their own maximum. Without any
            // mass there (mr = -inf) it is 0.
            double factor = 0.0;
            if (sr != 0.0)
                factor = sh.mass * exp(static_cast<double>(mr) - static_cast<double>(ma)) / sa;
            if (sh.r > 0.0) {
                loss += sh.r * (log(sh.r) + lse);
                loss -= sh.r * (sr != 0.0 ? static_cast<double>(mr) + log(sr) : static_cast<double>(kNegInf));
                if (sr != 0.0) factor -= sh.r / sr;
            }
            sh.max = ma;
            sh.inv = static_cast<float>(1.0 / sa);
            sh.rest_max = mr == kNegInf ? 0.0f : mr;
            sh.rest_factor = static_cast<float>(sa == sa ? factor : sa);
            if (rank == 0) {
                c.loss[row] = static_cast<float>(loss);
                if (state) {
                    state[0] = sh.max;
                    state[1] = sh.inv;
                    state[2] = sh.rest_max;
                    state[3] = sh.rest_factor;
                }
            }
        }
    } else if (kForward && rank == 0 && threadIdx.x == 0) {
        c.loss[row] = 0.0f;
        if (state) state[0] = state[1] = state[2] = state[3] = 0.0f;
    }
    if (!kForward && threadIdx.x == 0) {
        sh.max = state[0];
        sh.inv = state[1];
        sh.rest_max = state[2];
        sh.rest_factor = state[3];
    }
    if (kGrad) {
        __syncthreads();
        T *g = static_cast<T *>(c.dlogits) + row * c.grad_stride;
        const float up = c.row_grads[row];
        // An empty row, or one whose loss does not count, has no gradient,
        // whatever its logits hold.
        const bool none = empty || up == 0.0f;
        const float by = __fmul_rn(up, c.scale);
        const float rest_max = sh.rest_max;
        const float factor = none ? 0.0f : __fmul_rn(by, sh.rest_factor);
        auto grad = [&](float xv) {
            return none ? 0.0f
                        : __fmul_rn(exp_fast(__fsub_rn(__fmul_rn(xv, c.scale), rest_max)), factor);
        };
        const Segment<T> to(g, lo, hi);
        if (to.body == seg.body) {
            auto one = [&](uint32_t j) { g[j] = from_float<T>(grad(none ? 0.0f : elem_to_float<T>(x[j]))); };
            if (threadIdx.x < seg.body - lo) one(lo + threadIdx.x);
            if (threadIdx.x >= 32 && threadIdx.x - 32 < hi - seg.tail) one(seg.tail + threadIdx.x - 32);
            const uint4 *words = reinterpret_cast<const uint4 *>(x + seg.body);
            uint4 *out = reinterpret_cast<uint4 *>(g + seg.body);
            for (uint32_t q0 = threadIdx.x; q0 < seg.n_vec; q0 += kThreads * kLoads) {
                uint4 w[kLoads];
#pragma unroll
                for (uint32_t k = 0; k < kLoads; ++k) {
                    const uint32_t q = q0 + k * kThreads;
                    w[k] = q < seg.n_vec && !none ? words[q] : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (uint32_t k = 0; k < kLoads; ++k) {
                    const uint32_t q = q0 + k * kThreads;
                    float v[kE];
                    unpack<T>(w[k], v);
                    union {
                        uint4 word;
                        T elem[kE];
                    } o;
#pragma unroll
                    for (uint32_t i = 0; i < kE; ++i) o.elem[i] = from_float<T>(grad(v[i]));
                    if (q < seg.n_vec) out[q] = o.word;
                }
            }
        } else {
            // The gradient's rows start at another 16-byte phase than the logits'.
            for (uint32_t j = lo + threadIdx.x; j < hi; j += kThreads)
                g[j] = from_float<T>(grad(none ? 0.0f : elem_to_float<T>(x[j])));
        }
        // The listed tokens' gradients replace what the loop wrote there.
        __syncthreads();
        if (!none) {
            const float mass = static_cast<float>(sh.mass);
            for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
                float t_sum;
                if (!here(sh.id[k]) || !first_of_id(sh, n, k, t_sum)) continue;
                const float p = __fmul_rn(exp_fast(__fsub_rn(sh.v[k], sh.max)), sh.inv);
                g[sh.id[k]] = from_float<T>(__fmul_rn(by, __fsub_rn(__fmul_rn(p, mass), t_sum)));
            }
        }
    }
    // A CTA's shared memory outlives its peers' writes to it.
    if (kForward && !empty) cluster.sync();
}

template <typename T, bool kForward, bool kGrad>
cudaError_t launch(const DistillCall &c, uint32_t ctas, cudaStream_t stream) {
    const uint32_t seg = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const size_t smem = kForward && c.tail ? (seg / 32u + 2u) * sizeof(uint32_t) : 0;
    auto kernel = distill_kernel<T, kForward, kGrad>;
    if (smem > (24u << 10)) {  // above the default limit, together with the static part
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c.rows * ctas, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, c, ctas);
}

template <typename T>
cudaError_t launch_typed(const DistillCall &c, bool forward, bool grad, uint32_t ctas,
                         cudaStream_t stream) {
    if (forward)
        return grad ? launch<T, true, true>(c, ctas, stream) : launch<T, true, false>(c, ctas, stream);
    return launch<T, false, true>(c, ctas, stream);
}

}  // namespace

cudaError_t launch_distill(const DistillCall &c, rsc_dtype dtype, bool forward, bool grad, int num_sms,
                           cudaStream_t stream) {
    // Four CTAs per SM, in segments of at least 2048 logits.
    uint32_t ctas = 1;
    while (ctas < kMaxCtas && static_cast<size_t>(c.rows) * ctas < 4u * static_cast<size_t>(num_sms) &&
           c.vocab / (ctas * 2) >= 2048)
        ctas *= 2;
    // The bitmap of a segment fits in shared memory.
    while (ctas < kMaxCtas && c.vocab / ctas > (1u << 20)) ctas *= 2;
    switch (dtype) {
        case RSC_F32: return launch_typed<float>(c, forward, grad, ctas, stream);
        case RSC_BF16: return launch_typed<__nv_bfloat16>(c, forward, grad, ctas, stream);
        case RSC_F16: return launch_typed<__half>(c, forward, grad, ctas, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace rsc
