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
// A row is cut into segments for a cluster of CTAs that join their sums through
// distributed shared memory. The pass is bound by HBM (the loss alone: one
// read), next by the exponentials (one MUFU operation each, 16 a cycle and SM)
// and the instructions around them, so exponents and sums are taken two at a
// time (f32x2) and a 16-byte word's maximum on its packed halves; the lists'
// binary64 work runs while the cluster's CTAs wait for one another. S_tail is
// summed over the unlisted tokens as such (a bitmap of the listed ones masks
// them out): S minus the listed terms would lose it where the listed tokens
// hold nearly all of the mass. Measured (B200, GPU time): loss of 4096 x 128256
// bf16 with 128 entries and the tail 190 us (5.5 TB/s), loss and gradient of 2048
// x 151936 bf16 234 us (5.3 TB/s of one read and one write). Figures of variants
// below are differences to these, each measured beside the kernel as it then was. Keeping the segment
// in shared memory between the passes (TMA copies, four CTAs of 52 KB an SM)
// took 305-322 us: the phases of so few CTAs do not overlap.
#include <algorithm>
#include <cmath>
#include <type_traits>

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
struct __align__(16) RowShare {
    float max_rest, sum_rest;      // over the tokens of the pass
    float max_listed, sum_listed;  // over the listed ones, with the tail
    double cross, held;            // sums of t (y - y_ref - (v - v_ref)) and of t over the CTA's entries
};

struct DistillShared {
    float red_m[kWarps], red_s[kWarps];
    float list_m[kWarps], list_s[kWarps];
    float red_y[kWarps];
    double red_t[kWarps];
    RowShare share[kMaxCtas];
    uint32_t unordered;
    float v_ref;  // v of the row's first entry: what a loss is put together against
    float4 row;  // maximum, 1 / sum, unlisted maximum, unlisted factor
};

// A row's teacher entries in shared memory (cap of each).
struct Entries {
    uint32_t *id;
    float *y;  // log-probability as given
    float *t;  // probability
    float *v;  // scaled student logit (entries of this CTA's segment)
};
__device__ __forceinline__ uint32_t list_warps(uint32_t n) { return min(static_cast<uint32_t>(kWarps), (n + 31u) / 32u); }
constexpr size_t kEntryBytes = 16;

// What is known of a row's list as a whole, in every thread.
struct Teacher {
    bool some;     // it has an entry
    float y_ref;   // what exponents were taken against
    double sum;    // of exp(y - y_ref)
    double r, mass;
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

// Exponentials of a row against a reference value `ref` (any number near its
// largest v): exp(v - ref) = 2^(v c - mc) * 2^-slip with c = fl(log2 e) and mc =
// fl(ref c), one packed multiply-add for two of them. v = x s is rounded as the
// listed tokens' is; where s is a power of two that product is exact and goes into
// c (kExact, 2048 x 151936 bf16: up to 7 us less than with the product). The exponent is
// rounded once (2^-24) and c is 1.3e-8 off, |v - ref| 2^-23 in all; exponentials
// below 2^-126 are 0. What mc makes the reference off by is the same factor for the
// whole row, slip (log2, binary64), and is taken out of sums and factors. It grows
// with ref; beyond 2^24 (`wide`) the exponent is (v - ref) log2 e instead.
constexpr float kLog2e = 1.44269504f;
struct ExpRef {
    float ref, mc;
    bool wide;
    __device__ __forceinline__ explicit ExpRef(float ref_) : ref(ref_), mc(ref_ * kLog2e) {
        wide = !(fabsf(mc) < 0x1p+24f) && fabsf(ref) < kPosInf;
    }
    // 2^-slip, which a sum or factor of these exponentials is to be multiplied by.
    __device__ __forceinline__ double correction() const {
        if (wide) return 1.0;
        const double z = -0.6931471805599453 * __fma_rn(static_cast<double>(ref), static_cast<double>(kLog2e),
                                                        -static_cast<double>(mc));
        // |z| is 1e-7 of |ref|; its cube / 6 is below 2e-13 in the short form.
        return fabs(z) < 1e-4 ? __fma_rn(z, __fma_rn(z, 0.5, 1.0), 1.0) : exp(z);
    }
};

__device__ __forceinline__ float ex2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Two binary32 values in one 64-bit register pair, as the packed operations
// take them.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float low_of(uint64_t p) {
    float a;
    asm("mov.b64 {%0, _}, %1;" : "=f"(a) : "l"(p));
    return a;
}
__device__ __forceinline__ float high_of(uint64_t p) {
    float a;
    asm("mov.b64 {_, %0}, %1;" : "=f"(a) : "l"(p));
    return a;
}
// The largest of a warp's values (NaN passed over), in every lane.
__device__ __forceinline__ float warp_top(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// Two neighbouring exponentials.
template <bool kExact>
__device__ __forceinline__ uint64_t exp_pair(float x0, float x1, float scale, float mc) {
    uint64_t v = pair_of(x0, x1);
    float c = kLog2e;
    if (kExact)
        c = __fmul_rn(c, scale);
    else
        v = mul_pair(v, pair_of(scale, scale));
    const uint64_t t = fma_pair(v, pair_of(c, c), pair_of(-mc, -mc));
    return pair_of(ex2_fast(low_of(t)), ex2_fast(high_of(t)));
}
__device__ __forceinline__ float exp_one(float x, float scale, const ExpRef &r) {
    const float v = __fmul_rn(x, scale);
    return r.wide ? exp_fast(__fsub_rn(v, r.ref)) : ex2_fast(__fmaf_rn(v, kLog2e, -r.mc));
}

// The largest element of a 16-byte word (NaN passed over).
template <typename T>
__device__ __forceinline__ float word_max(const uint4 &w);
template <>
__device__ __forceinline__ float word_max<float>(const uint4 &w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)),
                 fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
}
template <>
__device__ __forceinline__ float word_max<__nv_bfloat16>(const uint4 &w) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&w);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
template <>
__device__ __forceinline__ float word_max<__half>(const uint4 &w) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&w);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// A 16-byte word of the gradient from one of the logits: exp(v - ref) * factor.
template <typename T, bool kWide, bool kExact>
__device__ __forceinline__ uint4 grad_word(const uint4 &w, float scale, const ExpRef &r, float factor) {
    constexpr int kE = kVecElems<T>;
    float v[kE];
    unpack<T>(w, v);
    union {
        uint4 word;
        T elem[kE];
    } o;
#pragma unroll
    for (int i = 0; i < kE; i += 2) {
        if (kWide) {
            o.elem[i] = from_float<T>(__fmul_rn(exp_one(v[i], scale, r), factor));
            o.elem[i + 1] = from_float<T>(__fmul_rn(exp_one(v[i + 1], scale, r), factor));
        } else {
            const uint64_t g = mul_pair(exp_pair<kExact>(v[i], v[i + 1], scale, r.mc), pair_of(factor, factor));
            o.elem[i] = from_float<T>(low_of(g));
            o.elem[i + 1] = from_float<T>(high_of(g));
        }
    }
    return o.word;
}

// The id of an absent entry: one outside the vocabulary, or of no probability.
constexpr uint32_t kAbsent = 0xffffffffu;

// The ids and log-probabilities of a row's list (one entry a thread for lists of
// up to a block), absent ones marked.
__device__ __forceinline__ void load_entries(const DistillCall &c, size_t row, uint32_t n,
                                             const Entries &e, DistillShared &sh) {
    const uint32_t *ids = c.ids + row * c.cap;
    bool unordered = false;
    for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
        const uint32_t id = ids[k], next = k + 1 < n ? ids[k + 1] : kAbsent;
        const float y = c.logprobs[row * c.cap + k];
        e.id[k] = id < c.vocab && y != kNegInf ? id : kAbsent;
        e.y[k] = y;
        // Lists in ascending order (padding aside) hold no id twice.
        unordered |= !(id < next) && next < c.vocab;
    }
    if (unordered) sh.unordered = 1;
}

// The entries' probabilities, from what this thread loaded. The exponentials
// are binary64: with the tail, r is what they leave of 1. Called by the whole
// block; it has passed a barrier before e.t is read by others.
__device__ __forceinline__ Teacher weigh_entries(const DistillCall &c, uint32_t n, const Entries &e,
                                                 DistillShared &sh) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t warps = list_warps(n);
    Teacher te;
    // With the tail the values are log-probabilities as such.
    te.y_ref = 0.0f;
    bool some = false;
    if (!c.tail) {
        if (warp < warps) {
            float top = kNegInf;
            for (uint32_t k = threadIdx.x; k < n; k += kThreads)
                if (e.id[k] != kAbsent) top = fmaxf(top, e.y[k]);
            top = warp_top(top);
            if (lane == 0) sh.red_y[warp] = top;
        }
        __syncthreads();
        float top = kNegInf;
        for (uint32_t w = 0; w < warps; ++w) top = fmaxf(top, sh.red_y[w]);
        if (fabsf(top) < kPosInf) te.y_ref = top;
    }
    if (warp < warps) {
        double part = 0.0;
        for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
            const bool there = e.id[k] != kAbsent;
            const double p =
                there ? exp(static_cast<double>(e.y[k]) - static_cast<double>(te.y_ref)) : 0.0;
            e.t[k] = static_cast<float>(p);
            part += p;
            some |= there;
        }
        part = warp_sum(part);
        if (lane == 0) sh.red_t[warp] = part;
    }
    te.some = __syncthreads_or(some);
    te.sum = 0.0;
    for (uint32_t w = 0; w < warps; ++w) te.sum += sh.red_t[w];
    te.r = 0.0;
    te.mass = 1.0;
    if (c.tail) {
        if (te.sum < 1.0) te.r = 1.0 - te.sum;
        if (te.sum > 1.0) te.mass = te.sum;
    } else if (warp < warps) {
        const float inv = __fdiv_rn(1.0f, static_cast<float>(te.sum));
        for (uint32_t k = threadIdx.x; k < n; k += kThreads) e.t[k] = __fmul_rn(e.t[k], inv);
    }
    return te;
}

// Entry k is the first of its id (ids may repeat: each entry counts).
__device__ __forceinline__ bool first_of_id(const Entries &e, bool unordered, uint32_t k) {
    if (unordered)
        for (uint32_t q = 0; q < k; ++q)
            if (e.id[q] == e.id[k]) return false;
    return true;
}

// The sum of t over the entries of k's id, in list order.
__device__ __forceinline__ float sum_of_id(const Entries &e, uint32_t n, uint32_t k) {
    double sum = 0.0;
    for (uint32_t q = 0; q < n; ++q)
        if (e.id[q] == e.id[k]) sum += static_cast<double>(e.t[q]);
    return static_cast<float>(sum);
}

// The (m, s) pairs of a warp's lanes joined in binary32, in all of them. A sum
// against -inf is 0 or NaN and stays.
__device__ __forceinline__ void join_lanes(float &m, float &s) {
    const float top = warp_top(m);
    if (m != kNegInf) s = __fmul_rn(s, exp_fast(__fsub_rn(m, top)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
    m = top;
}

// Loss and gradient together: a thread's own words of a segment on their way
// through shared memory, kDepth batches of kBatch 16-byte words copied
// asynchronously, so that the next ones travel while one is worked on. No other
// thread reads them. The second pass goes from the segment's end, whose last
// batches are still there. 48 KB a CTA leave four on an SM: 2048 x 151936 bf16
// takes 25 us more with plain loads and six CTAs, 12 with six of 32 KB, 21 with three
// of 64 KB, 7 with twelve words in batches of two. (The loss alone has no second
// pass that stalls: six CTAs of plain loads, 8 us less than the ring at 4096 x
// 128256 bf16.)
constexpr uint32_t kBatch = 4;
constexpr uint32_t kDepth = 3;
constexpr uint32_t kRingBytes = kThreads * kBatch * kDepth * 16;
struct Ring {
    const uint4 *from;  // this thread's first word
    uint32_t slots;     // shared-memory address of its first slot
    uint32_t full;      // whole batches of this thread

    __device__ __forceinline__ Ring(const uint4 *words, uint32_t n_vec, unsigned char *smem)
        : from(words + threadIdx.x),
          slots(static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + threadIdx.x * 16u) {
        const uint32_t last = threadIdx.x + kThreads * (kBatch - 1);
        full = n_vec > last ? (n_vec - last + kThreads * kBatch - 1) / (kThreads * kBatch) : 0u;
    }
    __device__ __forceinline__ uint32_t slot(uint32_t b) const {
        return slots + (b % kDepth) * (kThreads * kBatch * 16u);
    }
    __device__ __forceinline__ void fetch(uint32_t b) const {
        const uint4 *src = from + static_cast<size_t>(b) * (kThreads * kBatch);
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot(b) + k * kThreads * 16u),
                         "l"(src + k * kThreads)
                         : "memory");
    }
    static __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    static __device__ __forceinline__ void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
    }
    __device__ __forceinline__ void take(uint32_t b, uint4 *w) const {
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[k].x), "=r"(w[k].y), "=r"(w[k].z), "=r"(w[k].w)
                         : "r"(slot(b) + k * kThreads * 16u)
                         : "memory");
    }
};

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

// The exponentials of kN 16-byte words added up as a tree.
template <typename T, int kN, bool kExact>
__device__ __forceinline__ float batch_sum(const uint4 *w, float scale, float mc) {
    constexpr int kE = kVecElems<T>, kPairs = kN * kE / 2;
    uint64_t e[kPairs];
#pragma unroll
    for (int k = 0; k < kN; ++k) {
        float v[kE];
        unpack<T>(w[k], v);
#pragma unroll
        for (int i = 0; i < kE; i += 2) e[(k * kE + i) / 2] = exp_pair<kExact>(v[i], v[i + 1], scale, mc);
    }
#pragma unroll
    for (int d = 1; d < kPairs; d *= 2) {
#pragma unroll
        for (int i = 0; i + d < kPairs; i += 2 * d) e[i] = add_pair(e[i], e[i + d]);
    }
    return __fadd_rn(low_of(e[0]), high_of(e[0]));
}

// (m, s) of this thread's share of a segment: a batch of 16-byte words at a time
// against one reference, as in rsc_rowsum.cuh. Where the tail is wanted by itself
// the listed elements are left out by their bit.
template <typename T, bool kRinged>
__device__ __forceinline__ void sum_segment(const DistillCall &c, const T *x, const Segment<T> &seg,
                                             uint32_t *bits, const Entries &en, uint32_t n, const Ring &ring,
                                             float &m, double &s) {
    constexpr uint32_t kE = kVecElems<T>;
    const uint32_t lo = seg.lo, hi = seg.hi;
    const bool masked = c.tail;
    if (kRinged) {
#pragma unroll
        for (uint32_t b = 0; b < kDepth; ++b) {
            if (b < ring.full) ring.fetch(b);
            Ring::commit();
        }
    }
    // Bit b stands for element lo - pad + b, so that the words' elements start at
    // bit 32 * first.
    const uint32_t first = (seg.body - lo + 31u) / 32u;
    const uint32_t pad = first * 32u - (seg.body - lo);
    if (masked) {
        for (uint32_t w = threadIdx.x; w < (hi - lo + pad + 31u) / 32u; w += kThreads) bits[w] = 0;
        __syncthreads();
        for (uint32_t k = threadIdx.x; k < n; k += kThreads)
            if (en.id[k] >= lo && en.id[k] < hi) {
                const uint32_t b = en.id[k] - lo + pad;
                atomicOr(&bits[b / 32u], 1u << (b % 32u));
            }
        __syncthreads();
    }
    const unsigned char *bytes = reinterpret_cast<const unsigned char *>(bits + first);
    // This thread's element of the head or tail, if it has one.
    float one = kNegInf;
    uint32_t j = hi;
    if (threadIdx.x < seg.body - lo) j = lo + threadIdx.x;
    if (threadIdx.x >= 32 && threadIdx.x - 32 < hi - seg.tail) j = seg.tail + threadIdx.x - 32;
    if (j < hi && !(masked && (bits[(j - lo + pad) / 32u] >> ((j - lo + pad) % 32u) & 1u)))
        one = elem_to_float<T>(x[j]);
    // m stays -inf until there is a logit above it; the exponents' reference is
    // then 0, against which -inf gives 0 and NaN gives NaN.
    if (one > kNegInf) m = __fmul_rn(one, c.scale);
    ExpRef r(m > kNegInf ? m : 0.0f);
    double correction = r.correction();
    s = static_cast<double>(exp_one(one, c.scale, r)) * correction;
    const uint4 *words = reinterpret_cast<const uint4 *>(x + seg.body);
    // A batch of words, the listed elements among them taken out.
    auto add = [&](uint4 *w, const uint32_t *set, auto count) {
        constexpr int kN = decltype(count)::value;
        uint32_t any = 0;
#pragma unroll
        for (int k = 0; k < kN; ++k) any |= set[k];
        if (any) {
#pragma unroll
            for (int k = 0; k < kN; ++k) {
                union {
                    uint4 word;
                    T elem[kE];
                } u;
                u.word = w[k];
#pragma unroll
                for (uint32_t i = 0; i < kE; ++i)
                    if (set[k] >> i & 1u) u.elem[i] = from_float<T>(kNegInf);
                w[k] = u.word;
            }
        }
        float b = word_max<T>(w[0]);
#pragma unroll
        for (int k = 1; k < kN; ++k) b = fmaxf(b, word_max<T>(w[k]));
        const float next = __fmul_rn(b, c.scale);
        if (next > m + kHeadroom) {
            // Before the first logit above -inf the sum is 0 or NaN.
            if (m > kNegInf) s *= static_cast<double>(exp_fast(__fsub_rn(m, next)));
            m = next;
            r = ExpRef(next);
            correction = r.correction();
        }
        if (r.wide) {
            for (int k = 0; k < kN; ++k) {
                float v[kE];
                unpack<T>(w[k], v);
                for (uint32_t i = 0; i < kE; ++i) s += static_cast<double>(exp_one(v[i], c.scale, r));
            }
        } else {
            const float sum = c.exact ? batch_sum<T, kN, true>(w, c.scale, r.mc)
                                      : batch_sum<T, kN, false>(w, c.scale, r.mc);
            s += static_cast<double>(sum) * correction;
        }
    };
    auto listed = [&](uint32_t q) -> uint32_t {
        if (!masked) return 0u;
        return kE == 8 ? bytes[q] : bytes[q / 2u] >> (4u * (q & 1u)) & 15u;
    };
    uint32_t q0 = threadIdx.x;
    if (!kRinged) {
        for (; q0 + kThreads * (kLoads - 1) < seg.n_vec; q0 += kThreads * kLoads) {
            uint4 w[kLoads];
            uint32_t set[kLoads];
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) w[k] = __ldg(words + q0 + k * kThreads);
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) set[k] = listed(q0 + k * kThreads);
            add(w, set, std::integral_constant<int, kLoads>());
        }
    }
#pragma unroll 1
    for (uint32_t b = 0; kRinged && b < ring.full; ++b, q0 += kThreads * kBatch) {
        uint4 w[kBatch];
        uint32_t set[kBatch];
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) set[k] = listed(q0 + k * kThreads);
        Ring::wait();
        ring.take(b, w);
        if (b + kDepth < ring.full) ring.fetch(b + kDepth);
        Ring::commit();
        add(w, set, std::integral_constant<int, kBatch>());
    }
    for (; q0 < seg.n_vec; q0 += kThreads) {
        uint4 w = __ldg(words + q0);
        const uint32_t set = listed(q0);
        add(&w, &set, std::integral_constant<int, 1>());
    }
}

template <typename T, bool kForward, bool kGrad>
__global__ void __launch_bounds__(kThreads, kForward ? (kGrad ? 4 : 6) : 8)
distill_kernel(const __grid_constant__ DistillCall c, uint32_t ctas, uint32_t bitmap_bytes) {
    // One bit per element of the segment (with the tail), then the entries.
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ DistillShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank();
    const size_t row = blockIdx.x / ctas;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const T *x = static_cast<const T *>(c.logits) + row * c.row_stride;
    const uint32_t seg_len = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const uint32_t lo = min(c.vocab, rank * seg_len), hi = min(c.vocab, lo + seg_len);
    const Segment<T> seg(x, lo, hi);
    constexpr uint32_t kRing = kForward && kGrad ? kRingBytes : 0;
    const Ring ring(reinterpret_cast<const uint4 *>(x + seg.body), seg.n_vec, dynamic);
    Entries e;
    e.id = reinterpret_cast<uint32_t *>(dynamic + kRing + bitmap_bytes);
    e.y = reinterpret_cast<float *>(e.id + c.cap);
    e.t = e.y + c.cap;
    e.v = e.t + c.cap;
    uint32_t n = static_cast<uint32_t>(c.cap);
    if (c.n) n = min(n, static_cast<uint32_t>(max(0, static_cast<int32_t>(c.n[row]))));
    // A row with an empty list is not looked at (for every CTA of the cluster alike).
    const bool listed = n > 0;
    float *state = c.state ? c.state + row * 4 : nullptr;
    // Every CTA of the cluster runs before its memory is written. (Warps that
    // have written nothing for their peers arrive without a fence: 235 to 231 us.)
    if (kForward && listed) asm volatile("barrier.cluster.arrive.relaxed.aligned;");
    if (threadIdx.x == 0) sh.unordered = 0;
    __syncthreads();
    load_entries(c, row, n, e, sh);
    auto here = [&](uint32_t id) { return id >= lo && id < hi; };
    const bool masked = kForward && c.tail;
    __syncthreads();
    const bool unordered = sh.unordered != 0;

    // The entries' student logits, before anything is written (the gradient
    // may replace the logits).
    for (uint32_t k = threadIdx.x; k < n; k += kThreads)
        e.v[k] = here(e.id[k]) ? __fmul_rn(elem_to_float<T>(x[e.id[k]]), c.scale) : kNegInf;
    if (kForward && threadIdx.x == 32) {
        uint32_t k = 0;
        while (k < n && e.id[k] == kAbsent) ++k;
        const float v = k < n ? __fmul_rn(elem_to_float<T>(x[e.id[k]]), c.scale) : 0.0f;
        sh.v_ref = fabsf(v) < kPosInf ? v : 0.0f;
    }

    Teacher te{};
    if (kForward && listed) {
        float m = kNegInf;
        double sum = 0.0;
        sum_segment<T, kGrad>(c, x, seg, reinterpret_cast<uint32_t *>(dynamic + kRing), e, n, ring, m, sum);
        float s = static_cast<float>(sum);
        join_lanes(m, s);
        if (lane == 0) {
            sh.red_m[warp] = m;
            sh.red_s[warp] = s;
        }
        // With the tail, the listed tokens' own sum, each id once.
        const uint32_t warps = list_warps(n);
        if (masked && warp < warps) {
            float ml = kNegInf, sl = 0.0f;
            for (uint32_t k = threadIdx.x; k < n; k += kThreads) ml = fmaxf(ml, e.v[k]);
            ml = warp_top(ml);
            for (uint32_t k = threadIdx.x; k < n; k += kThreads)
                if (here(e.id[k]) && e.v[k] != kNegInf && first_of_id(e, unordered, k))
                    sl = __fadd_rn(sl, exp_fast(__fsub_rn(e.v[k], ml)));
            sl = warp_sum(sl);
            if (lane == 0) {
                sh.list_m[warp] = ml;
                sh.list_s[warp] = sl;
            }
        }
        __syncthreads();
        cluster.barrier_wait();
        // The CTA's sums to its peers (to the first alone where the loss is all).
        if (warp == 0) {
            m = lane < kWarps ? sh.red_m[lane] : kNegInf;
            s = lane < kWarps ? sh.red_s[lane] : 0.0f;
            join_lanes(m, s);
            float ml = kNegInf, sl = 0.0f;
            if (masked) {
                ml = lane < warps ? sh.list_m[lane] : kNegInf;
                sl = lane < warps ? sh.list_s[lane] : 0.0f;
                join_lanes(ml, sl);
            }
            if (lane < (kGrad ? ctas : 1u)) {
                RowShare &to = cluster.map_shared_rank(&sh, lane)->share[rank];
                to.max_rest = m;
                to.sum_rest = s;
                to.max_listed = ml;
                to.sum_listed = sl;
            }
        }
        // The teacher's side while the cluster's other CTAs arrive.
        if (warp == 0)
            cluster.barrier_arrive();
        else
            asm volatile("barrier.cluster.arrive.relaxed.aligned;");
        te = weigh_entries(c, n, e, sh);
        __syncthreads();
        cluster.barrier_wait();
        if (warp == 1) {
            // This segment's part of the loss.
            double cross = 0.0, held_t = 0.0;
            for (uint32_t k = lane; k < n; k += 32) {
                const double t = e.t[k];
                if (!here(e.id[k]) || t == 0.0) continue;
                cross += t * (static_cast<double>(e.y[k]) - static_cast<double>(te.y_ref) -
                              (static_cast<double>(e.v[k]) - static_cast<double>(sh.v_ref)));
                held_t += t;
            }
            cross = warp_sum(cross);
            held_t = warp_sum(held_t);
            if (lane == 0) {
                RowShare &to = cluster.map_shared_rank(&sh, 0)->share[rank];
                to.cross = cross;
                to.held = held_t;
            }
        }
        if (warp == 1)
            cluster.barrier_arrive();
        else
            asm volatile("barrier.cluster.arrive.relaxed.aligned;");
        if (warp == 0 && (kGrad || rank == 0)) {
            const bool in = lane < ctas;
            float mr = in ? sh.share[lane].max_rest : kNegInf;
            float sr = in ? sh.share[lane].sum_rest : 0.0f;
            join_lanes(mr, sr);
            float ml = kNegInf, sl = 0.0f;
            if (masked) {
                ml = in ? sh.share[lane].max_listed : kNegInf;
                sl = in ? sh.share[lane].sum_listed : 0.0f;
                join_lanes(ml, sl);
            }
            const float row_max = fmaxf(mr, ml);
            float all = __fadd_rn(mr == kNegInf ? sr : __fmul_rn(sr, exp_fast(__fsub_rn(mr, row_max))),
                                  ml == kNegInf ? sl : __fmul_rn(sl, exp_fast(__fsub_rn(ml, row_max))));
            // A row of -inf alone has no distribution: NaN, as a NaN or +inf logit
            // gives through the sum.
            if (!(all > 0.0f)) all = __uint_as_float(0x7fc00000u);
            const float inv = __fdiv_rn(1.0f, all);
            // The unlisted tokens' factor against their own maximum. Without any mass
            // there (mr = -inf) it is 0.
            const float rest_max = mr == kNegInf ? 0.0f : mr;
            float factor = 0.0f;
            if (sr != 0.0f) {
                factor = __fmul_rn(__fmul_rn(static_cast<float>(te.mass), exp_fast(__fsub_rn(mr, row_max))), inv);
                if (te.r > 0.0) factor = __fsub_rn(factor, __fdiv_rn(static_cast<float>(te.r), sr));
            }
            factor = __fmul_rn(factor, static_cast<float>(ExpRef(rest_max).correction()));
            if (!(all == all)) factor = all;
            if (lane == 0) {
                sh.row = make_float4(row_max, inv, rest_max, factor);
                sh.red_m[0] = mr;
                sh.red_s[0] = sr;
                sh.red_s[1] = all;
                // (1 / sum is never 0: a state of zeros is a row without entries.)
                if (rank == 0 && state)
                    *reinterpret_cast<float4 *>(state) = te.some ? sh.row : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
        }
        __syncthreads();
    } else if (kForward && rank == 0 && threadIdx.x == 0) {
        c.loss[row] = 0.0f;
        if (state) *reinterpret_cast<float4 *>(state) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (kGrad) {
        if (!kForward) __syncthreads();  // every entry's logit is read
        // The row as the gradient needs it: p = exp(v - row_max) * inv on the listed
        // tokens, exp(v - rest_max) * rest_factor the whole term on the others.
        float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (!kForward)
            st = *reinterpret_cast<const float4 *>(state);
        else if (te.some)
            st = sh.row;
        const float row_max = st.x, inv = st.y, rest_max = st.z, rest_factor = st.w;
        T *g = static_cast<T *>(c.dlogits) + row * c.grad_stride;
        const float up = c.row_grads[row];
        // A row without an entry, or one whose loss does not count, has no
        // gradient, whatever its logits hold.
        const bool none = inv == 0.0f || up == 0.0f;
        const float by = __fmul_rn(up, c.scale);
        const ExpRef r(rest_max);
        const float factor = __fmul_rn(by, rest_factor);
        auto one = [&](uint32_t j) {
            g[j] = from_float<T>(
                none ? 0.0f : __fmul_rn(exp_one(elem_to_float<T>(x[j]), c.scale, r), factor));
        };
        const Segment<T> to(g, lo, hi);
        if (to.body == seg.body) {
            if (threadIdx.x < seg.body - lo) one(lo + threadIdx.x);
            if (threadIdx.x >= 32 && threadIdx.x - 32 < hi - seg.tail) one(seg.tail + threadIdx.x - 32);
            const uint4 *words = reinterpret_cast<const uint4 *>(x + seg.body);
            uint4 *out = reinterpret_cast<uint4 *>(g + seg.body);
            if (none) {
                for (uint32_t q = threadIdx.x; q < seg.n_vec; q += kThreads) out[q] = make_uint4(0, 0, 0, 0);
            } else if (r.wide) {
                for (uint32_t q = threadIdx.x; q < seg.n_vec; q += kThreads)
                    out[q] = grad_word<T, true, false>(words[q], c.scale, r, factor);
            } else {
                // One loop for each form of the exponent.
                auto loop = [&](auto exact) {
                    auto word = [&](const uint4 &w) {
                        return grad_word<T, false, decltype(exact)::value>(w, c.scale, r, factor);
                    };
                    uint32_t q0 = threadIdx.x;
                    if (kForward) {
                        // From the segment's end, whose last batches are still there.
#pragma unroll 1
                        for (uint32_t b = ring.full; b-- > 0;) {
                            uint4 w[kBatch];
                            Ring::wait();
                            ring.take(b, w);
                            if (b >= kDepth) ring.fetch(b - kDepth);
                            Ring::commit();
#pragma unroll
                            for (uint32_t k = 0; k < kBatch; ++k)
                                __stcs(out + q0 + (b * kBatch + k) * kThreads, word(w[k]));
                        }
                        q0 += ring.full * kThreads * kBatch;
                    }
                    for (; !kForward && q0 + kThreads * (kLoads - 1) < seg.n_vec; q0 += kThreads * kLoads) {
                        uint4 w[kLoads];
#pragma unroll
                        for (uint32_t k = 0; k < kLoads; ++k) w[k] = __ldcs(words + q0 + k * kThreads);
#pragma unroll
                        for (uint32_t k = 0; k < kLoads; ++k)
                            __stcs(out + q0 + k * kThreads, word(w[k]));
                    }
                    for (; q0 < seg.n_vec; q0 += kThreads)
                        out[q0] = word(words[q0]);
                };
                if (c.exact)
                    loop(std::true_type());
                else
                    loop(std::false_type());
            }
        } else {
            // The gradient's rows start at another 16-byte phase than the logits', as
            // dense rows beside padded ones of an odd vocabulary: element by element
            // (2048 x 151937 bf16 766 us, against 285 in place or with both dense).
            for (uint32_t j = lo + threadIdx.x; j < hi; j += kThreads) one(j);
        }
        // The listed tokens' gradients replace what the loop wrote there.
        if (!kForward && !none) te = weigh_entries(c, n, e, sh);
        __syncthreads();
        if (!none) {
            const float mass = static_cast<float>(te.mass);
            for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
                if (!here(e.id[k]) || !first_of_id(e, unordered, k)) continue;
                const float p = __fmul_rn(exp_fast(__fsub_rn(e.v[k], row_max)), inv);
                const float t = unordered ? sum_of_id(e, n, k) : e.t[k];
                g[e.id[k]] = from_float<T>(__fmul_rn(by, __fsub_rn(__fmul_rn(p, mass), t)));
            }
        }
    }
    if (kForward && listed) {
        cluster.barrier_wait();  // every CTA's part of the loss is here
        if (rank == 0 && warp == 0) {
            double loss = warp_sum(lane < ctas ? sh.share[lane].cross : 0.0);
            const double held_all = warp_sum(lane < ctas ? sh.share[lane].held : 0.0);
            if (lane == 0) {
                const float mr = sh.red_m[0], sr = sh.red_s[0];
                // log S against v_ref and against the unlisted maximum: as such it would
                // lose log of the sum where the logits are large.
                const double row_max = sh.row.x, log_sum = log(static_cast<double>(sh.red_s[1]));
                loss += held_all * (row_max - static_cast<double>(sh.v_ref) + log_sum -
                                    (c.tail ? 0.0 : log(te.sum)));
                if (te.r > 0.0)
                    loss += te.r * (sr != 0.0f ? log(te.r) + (row_max - static_cast<double>(mr)) + log_sum -
                                                     log(static_cast<double>(sr))
                                               : static_cast<double>(kPosInf));
                c.loss[row] = te.some ? static_cast<float>(loss) : 0.0f;
            }
        }
    }
}

template <typename T, bool kForward, bool kGrad>
cudaError_t launch(const DistillCall &c, uint32_t ctas, size_t bitmap, cudaStream_t stream) {
    bitmap = (bitmap + 15u) & ~size_t{15};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c.rows * ctas, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = (kForward && kGrad ? kRingBytes : 0) + bitmap + c.cap * kEntryBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, distill_kernel<T, kForward, kGrad>, c, ctas,
                              static_cast<uint32_t>(bitmap));
}

template <typename T>
cudaError_t launch_typed(const DistillCall &c, bool forward, bool grad, int num_sms,
                         cudaStream_t stream) {
    const size_t bytes = static_cast<size_t>(c.vocab) * sizeof(T);
    // A CTA's segment. The loss alone and the backward pass read a row once, and
    // every CTA of a row repeats the work on its list: whole rows up to 320 KB
    // (2 x 160 KB costs 4096 x 128256 bf16 losses 32 us). Loss and
    // gradient together read the row twice, the second time from L2, which has to
    // hold what the CTAs of the GPU (four per SM) are at: 104 KB each (2048 x
    // 151936 bf16 takes 10 us more with 152 KB, 33 with 76 KB). Small batches take
    // more CTAs, to four per SM; a batch a little above one round of the GPU's CTAs
    // (888 for the loss alone) pays for a second, nearly empty one.
    const size_t share = (forward && grad ? 104u : 320u) << 10;
    uint32_t ctas = static_cast<uint32_t>(std::min<size_t>(kMaxCtas, (bytes + share - 1) / share));
    while (ctas < kMaxCtas && static_cast<size_t>(c.rows) * ctas < 4 * static_cast<size_t>(num_sms) &&
           c.vocab / (ctas * 2) >= 2048)
        ctas = std::min(kMaxCtas, ctas * 2);
    if (!forward) return launch<T, false, true>(c, ctas, 0, stream);
    const uint32_t seg = ((c.vocab + ctas - 1) / ctas + 31u) & ~31u;
    const size_t bits = c.tail ? (seg / 32u + 2u) * sizeof(uint32_t) : 0;
    return grad ? launch<T, true, true>(c, ctas, bits, stream) : launch<T, true, false>(c, ctas, bits, stream);
}

template <typename T>
cudaError_t setup_typed() {
    // A bitmap of kDistillMaxVocab / kMaxCtas elements and the longest lists.
    const int most = static_cast<int>((kDistillMaxVocab / kMaxCtas / 32u + 3u) * sizeof(uint32_t) +
                                      kDistillMaxTop * kEntryBytes + 16u + kRingBytes);
    cudaError_t e = cudaFuncSetAttribute(distill_kernel<T, true, true>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(distill_kernel<T, true, false>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return e;
}

}  // namespace

cudaError_t distill_setup() {
    cudaError_t e = setup_typed<float>();
    if (e == cudaSuccess) e = setup_typed<__nv_bfloat16>();
    if (e == cudaSuccess) e = setup_typed<__half>();
    return e;
}

cudaError_t launch_distill(const DistillCall &call, rsc_dtype dtype, bool forward, bool grad, int num_sms,
                           cudaStream_t stream) {
    DistillCall c = call;
    int exponent = 0;
    c.exact = std::frexp(c.scale, &exponent) == 0.5f;  // a power of two
    switch (dtype) {
        case RSC_F32: return launch_typed<float>(c, forward, grad, num_sms, stream);
        case RSC_BF16: return launch_typed<__nv_bfloat16>(c, forward, grad, num_sms, stream);
        case RSC_F16: return launch_typed<__half>(c, forward, grad, num_sms, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace rsc
