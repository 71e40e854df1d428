// Softmax statistics and top lists of rows of logits, shared by the kernels
// that score logits in memory (vxk_score.cu) and those that score a product's
// tiles as they are made (vxk_head_score.cu).
//
// A set of logits is summed up by (m, s, t): m the largest, s = sum e^(l - m),
// t = sum e^(l - m) (l - m).  Then log-sum-exp = m + log s and the entropy is
// log s - t / s, in which both terms are positive: nothing cancels.  Two sets
// join at the larger m: with d = m_old - m_new <= 0,
//   s' = s e^d,  t' = (t + s d) e^d.
// All three are fp32; exponentials are ex2 of the fp32 difference l - m (not of
// l and m scaled apart: their rounding would be as large as |l|).
//
// A top list is kept as 64-bit keys: the logit's bits in unsigned order above the
// inverted index, so that the larger key is the larger logit or, among equal
// ones, the lower index.  Key 0 is below every logit's.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace vxk {

constexpr int kMaxTop = 16;           // alternatives of one row
constexpr int32_t kErrToken = 4;      // device error word: a given token outside the vocabulary

// Statistics and list of a part of a row, to be joined with the row's others.
struct ScorePart {
    float m, s, t, pad;
    unsigned long long top[kMaxTop];
};

// Where a row's scores go (vxk_head_score*); null pointers are skipped.
struct ScoreOut {
    const int32_t * tokens;
    float * logprob;
    float * entropy;
    int32_t * top_ids;
    float * top_logprobs;
    int32_t * error;
    int32_t n_top;
    int32_t vocab;
};

#ifdef __CUDACC__

constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct Stat {
    float m, s, t;
};

__device__ __forceinline__ Stat stat_empty() { return {-INFINITY, 0.0f, 0.0f}; }

// What l - m is taken from: m, or 0 while nothing but -inf was seen.
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }

// Adds e^(l - base) for one logit l <= base.
__device__ __forceinline__ void stat_add(Stat & a, float l, float base) {
    const float d = l - base;
    const float e = ex2(d * kLog2e);
    a.s += e;
    a.t = fmaf(e, fmaxf(d, -1e30f), a.t);  // l = -inf: e is 0 and the product has to be 0 too
}

// Moves the sums to a larger maximum.
__device__ __forceinline__ void stat_raise(Stat & a, float m) {
    const float d = stat_base(a.m) - stat_base(m);
    if (a.m != -INFINITY) {
        const float f = ex2(d * kLog2e);
        a.t = fmaf(a.s, fmaxf(d, -1e30f), a.t) * f;
        a.s *= f;
    }
    a.m = m;
}

__device__ __forceinline__ Stat stat_join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m);
    stat_raise(a, m);
    stat_raise(b, m);
    a.s += b.s;
    a.t += b.t;
    return a;
}

__device__ __forceinline__ Stat stat_shfl_xor(const Stat & a, int o) {
    return {__shfl_xor_sync(kAll, a.m, o), __shfl_xor_sync(kAll, a.s, o), __shfl_xor_sync(kAll, a.t, o)};
}

__device__ __forceinline__ uint32_t top_bits(float v) {
    uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals 0
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    if (v != v) u = 1u;  // a NaN stands below every number (and above an empty place)
    return u;
}

__device__ __forceinline__ unsigned long long top_key(float v, int idx) {
    return ((unsigned long long) top_bits(v) << 32) | (unsigned long long) (0xFFFFFFFFu - (uint32_t) idx);
}

__device__ __forceinline__ int top_index(unsigned long long key) {
    return (int) (0xFFFFFFFFu - (uint32_t) (key & 0xFFFFFFFFull));
}

__device__ __forceinline__ float top_value(unsigned long long key) {
    const uint32_t u = (uint32_t) (key >> 32);
    if (u == 1u) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// The next value below that of `bits` (a key's upper half), NaN where there is none: a
// comparison with it passes what the bits allow.
__device__ __forceinline__ float top_below(uint32_t bits) {
    if (bits <= 1u) return __uint_as_float(0x7fc00000u);
    --bits;
    if (bits == 0x7fffffffu) --bits;  // -0 is 0 here
    return top_value((unsigned long long) bits << 32);
}

// A list held by a warp, its j-th largest key in lane j.
struct WarpTop {
    unsigned long long key;  // this lane's
    unsigned long long low;  // the n_top-th key: what a candidate has to beat
    int n_top;

    __device__ __forceinline__ void clear(int n) {
        key = 0ull;
        low = n > 0 ? 0ull : ~0ull;
        n_top = n;
    }
    // Raises `low` before anything is listed.  Each lane holds the largest value bits
    // (a key's upper half, 0: none) of a set of its own: the n_top-th largest of them is
    // no more than the n_top-th largest of all elements, so nothing below it belongs to
    // the list, and few candidates are left to insert one by one.
    __device__ __forceinline__ void bound(uint32_t largest) {
        const int lane = threadIdx.x & 31;
        uint32_t v = 0;
        for (int i = 0; i < n_top; ++i) {
            v = __reduce_max_sync(kAll, largest);
            if (v == 0) return;  // fewer sets than places
            const unsigned who = __ballot_sync(kAll, largest == v);
            if (lane == __ffs(who) - 1) largest = 0;
        }
        raise(v);
    }
    __device__ __forceinline__ void raise(uint32_t value_bits) {
        const unsigned long long b = (unsigned long long) value_bits << 32;  // below every key of that value
        if (n_top && b > low) low = b;
    }
    // Inserts a key that every lane holds.
    __device__ __forceinline__ void insert(unsigned long long k) {
        const int lane = threadIdx.x & 31;
        const int at = __popc(__ballot_sync(kAll, key > k));
        const unsigned long long up = __shfl_up_sync(kAll, key, 1);
        if (lane == at) key = k;
        if (lane > at) key = up;
        const unsigned long long last = __shfl_sync(kAll, key, n_top - 1);
        if (last > low) low = last;
    }
    // Offers each lane's candidate (0: none).
    __device__ __forceinline__ void offer(unsigned long long cand) {
        unsigned mask = __ballot_sync(kAll, cand > low);
        while (mask) {
            const unsigned long long k = __shfl_sync(kAll, cand, __ffs(mask) - 1);
            if (k > low) insert(k);
            mask &= mask - 1;
        }
    }
};

// Writes the scores of one row by one warp: its statistics (in every lane), its
// list, and its given token's logit.
__device__ __forceinline__ void score_write(const ScoreOut & o, int64_t row, const Stat & a, unsigned long long key,
                                            int32_t token, float token_logit) {
    const int lane = threadIdx.x & 31;
    const float base = stat_base(a.m);
    const float log_s = logf(a.s);
    if (lane == 0) {
        if (o.logprob) {
            float lp = (token_logit - base) - log_s;
            if (token < 0) lp = 0.0f;
            if (token >= o.vocab) {
                lp = __uint_as_float(0x7fc00000u);
                atomicCAS(o.error, 0, kErrToken);
            }
            o.logprob[row] = lp;
        }
        if (o.entropy) o.entropy[row] = log_s - a.t / a.s;
    }
    if (lane < o.n_top) {
        if (o.top_ids) o.top_ids[row * o.n_top + lane] = top_index(key);
        if (o.top_logprobs) o.top_logprobs[row * o.n_top + lane] = (top_value(key) - base) - log_s;
    }
}

template <int DT>
__device__ __forceinline__ float logit_at(const void * p, int64_t i) {
    if constexpr (DT == 0) return static_cast<const float *>(p)[i];
    if constexpr (DT == 1) return __half2float(static_cast<const __half *>(p)[i]);
    if constexpr (DT == 30) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

#endif  // __CUDACC__

}  // namespace vxk
