// Scores of logits in memory (vxk_head_score_logits): each row's given token's
// log probability, entropy and top list in one pass (the mathematics is in
// vxk_score.h).  Bound by reading the logits once.
//
// The rows' elements are cut into strips of 4096; a CTA takes an equal, unbroken
// run of all rows' strips, so that any number of rows keeps the whole device busy
// to the end: a row that lies within one CTA's run is finished there, one that
// crosses into others' leaves a part in each, and the CTA that arrives last joins
// them in order (the result does not depend on which that is).  Rows of at most
// one strip go one to a warp instead: there the block's reductions would cost more
// than the read.
//
// A thread holds 16 elements of a strip at a time (16-byte loads), takes their
// maximum first, so that the sums are rescaled at most once a strip, and offers
// candidates to its warp's top list only where that maximum reaches the list's
// end.
#include "vxk_internal.h"
#include "vxk_score.h"

#include <algorithm>

namespace vxk {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPer = 16;  // elements of a strip in one thread

template <int DT>
struct Elem {
    static constexpr int kBytes = DT == 0 ? 4 : 2;
    static constexpr int kVec = 16 / kBytes;      // elements of a 16-byte load
    static constexpr int kLoads = kPer / kVec;    // loads of a strip in one thread
};

template <int DT>
__device__ __forceinline__ void unpack(const uint4 & u, float * v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (DT == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == 30) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
}

__device__ __forceinline__ uint4 load_stream(const void * p) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
    return u;
}

// Strips [c0, c1) of one row by TEAM warps: adds to the thread's statistics and
// the warp's list.  shared_low: the largest list end of the team's warps, which no
// warp's candidates need go below.  Elements before the row's first 16-byte boundary and behind
// its last go with strip 0.
template <int DT, int TEAM>
__device__ __forceinline__ void scan(const uint8_t * row, int32_t vocab, int64_t c0, int64_t c1, int tid, Stat & a,
                                     WarpTop & top, uint32_t * shared_low) {
    using E = Elem<DT>;
    constexpr int kTeam = TEAM * 32;
    const int lead = min(vocab, (int) ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / E::kBytes);
    const int n_vec = (vocab - lead) / E::kVec;
    const uint8_t * body = row + (int64_t) lead * E::kBytes;

    if (c0 == 0) {
        const int tail0 = lead + n_vec * E::kVec;
        int idx = -1;
        if (tid < lead) idx = tid;
        else if (tid >= 16 && tid - 16 < vocab - tail0) idx = tail0 + tid - 16;
        if (__any_sync(kAll, idx >= 0)) {
            const float v = idx >= 0 ? logit_at<DT>(row, idx) : -INFINITY;
            const float m = fmaxf(a.m, v);
            stat_raise(a, m);
            if (idx >= 0) stat_add(a, v, stat_base(m));
            if (top.n_top) top.offer(idx >= 0 ? top_key(v, idx) : 0ull);
        }
    }
    for (int64_t c = c0; c < c1; ++c) {
        const int64_t v0 = c * (kTeam * E::kLoads) + tid;
        if (c * (kTeam * E::kLoads) >= n_vec) break;
        float x[kPer];
        uint4 u[E::kLoads];
#pragma unroll
        for (int j = 0; j < E::kLoads; ++j)
            if (v0 + j * kTeam < n_vec) u[j] = load_stream(body + (v0 + j * kTeam) * 16);
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < E::kLoads; ++j) {
            if (v0 + j * kTeam < n_vec) {
                unpack<DT>(u[j], x + j * E::kVec);
            } else {
#pragma unroll
                for (int i = 0; i < E::kVec; ++i) x[j * E::kVec + i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < E::kVec; ++i) m = fmaxf(m, x[j * E::kVec + i]);
        }
        if (top.n_top) {
            // every lane's largest element, or none where it has no element
            const uint32_t largest = v0 < n_vec ? top_bits(m) : 0u;
            if (top.low == 0ull) top.bound(largest);
            if (shared_low) top.raise(*shared_low);
            if (__any_sync(kAll, largest >= (uint32_t) (top.low >> 32))) {
#pragma unroll
                for (int j = 0; j < E::kLoads; ++j) {
                    const bool in = v0 + j * kTeam < n_vec;
                    const int idx = lead + (int) (v0 + j * kTeam) * E::kVec;
#pragma unroll
                    for (int i = 0; i < E::kVec; ++i)
                        top.offer(in ? top_key(x[j * E::kVec + i], idx + i) : 0ull);
                }
                if (shared_low && (threadIdx.x & 31) == 0) atomicMax(shared_low, (uint32_t) (top.low >> 32));
            }
        }
        if (m > a.m) stat_raise(a, m);
        const float base = stat_base(a.m);
#pragma unroll
        for (int i = 0; i < kPer; ++i) stat_add(a, x[i], base);
    }
}

__device__ __forceinline__ Stat warp_join(Stat a) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a = stat_join(a, stat_shfl_xor(a, o));
    return a;
}

template <int DT>
__device__ __forceinline__ void finish(const ScoreLogitsParams & p, int64_t row, const Stat & a,
                                       unsigned long long key) {
    const int32_t token = p.out.tokens ? p.out.tokens[row] : -1;
    const uint8_t * at = static_cast<const uint8_t *>(p.logits) + row * p.ld * Elem<DT>::kBytes;
    const float l = token >= 0 && token < p.out.vocab ? logit_at<DT>(at, token) : 0.0f;
    score_write(p.out, row, a, key, token, l);
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) score_warp_kernel(const ScoreLogitsParams p) {
    const int64_t row = (int64_t) blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    Stat a = stat_empty();
    WarpTop top;
    top.clear(p.out.n_top);
    const int strips = p.out.vocab / (32 * kPer) + 1;
    scan<DT, 1>(static_cast<const uint8_t *>(p.logits) + row * p.ld * Elem<DT>::kBytes, p.out.vocab, 0, strips,
                threadIdx.x & 31, a, top, nullptr);
    finish<DT>(p, row, warp_join(a), top.key);
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 2) score_block_kernel(const ScoreLogitsParams p) {
    __shared__ Stat stats[kWarps];
    __shared__ unsigned long long lists[kWarps * kMaxTop];
    __shared__ uint32_t shared_low;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_top = p.out.n_top;
    const int64_t strips = p.strips, total = strips * p.rows, grid = gridDim.x, cta = blockIdx.x;
    const int64_t begin = cta * total / grid, end = (cta + 1) * total / grid;

    for (int64_t x = begin; x < end;) {
        const int64_t row = x / strips, c0 = x - row * strips;
        const int64_t c1 = min(strips, c0 + end - x);
        if (tid == 0) shared_low = 0;
        __syncthreads();
        Stat a = stat_empty();
        WarpTop top;
        top.clear(n_top);
        scan<DT, kWarps>(static_cast<const uint8_t *>(p.logits) + row * p.ld * Elem<DT>::kBytes, p.out.vocab, c0, c1,
                         tid, a, top, &shared_low);
        a = warp_join(a);
        if (lane == 0) stats[warp] = a;
        if (lane < n_top) lists[warp * n_top + lane] = top.key;
        __syncthreads();
        if (warp == 0) {
            a = warp_join(lane < kWarps ? stats[lane] : stat_empty());
            if (n_top) top.raise(shared_low);
            for (int i = n_top; i < kWarps * n_top; i += 32)  // the warp's own list is in place
                top.offer(i + lane < kWarps * n_top ? lists[i + lane] : 0ull);
            if (c1 - c0 == strips) {
                finish<DT>(p, row, a, top.key);
            } else {
                // the CTAs whose runs hold this row's first and last strips
                const int64_t r0 = row * strips, r1 = r0 + strips - 1;
                const int64_t first = ((r0 + 1) * grid - 1) / total, last = ((r1 + 1) * grid - 1) / total;
                ScorePart * part = p.parts + 2 * cta + (x == begin ? 0 : 1);
                if (lane == 0) {
                    part->m = a.m;
                    part->s = a.s;
                    part->t = a.t;
                }
                if (lane < n_top) part->top[lane] = top.key;
                __threadfence();
                __syncwarp();
                int seen = 0;
                if (lane == 0) seen = atomicAdd(&p.counters[first], 1);
                seen = __shfl_sync(kAll, seen, 0);
                if (seen == (int) (last - first)) {
                    __threadfence();
                    Stat sum = stat_empty();
                    top.clear(n_top);
                    for (int64_t b0 = first; b0 <= last; b0 += 32) {
                        const int64_t b = b0 + lane;
                        Stat one = stat_empty();
                        if (b <= last) {
                            const bool mid = b == first && b * total / grid != r0;
                            const ScorePart * q = p.parts + 2 * b + (mid ? 1 : 0);
                            one = {__ldcg(&q->m), __ldcg(&q->s), __ldcg(&q->t)};
                        }
                        sum = stat_join(sum, warp_join(one));
                    }
                    for (int64_t b0 = first; n_top && b0 <= last; b0 += 32) {
                        const int64_t b = b0 + lane;
                        const bool mid = b == first && b * total / grid != r0;
                        const ScorePart * q = p.parts + 2 * b + (mid ? 1 : 0);
                        for (int j = 0; j < n_top; ++j) {  // the parts' lists are in order
                            const unsigned long long k = b <= last ? __ldcg(&q->top[j]) : 0ull;
                            if (j == 0 && top.low == 0ull) top.bound((uint32_t) (k >> 32));
                            if (!__any_sync(kAll, k > top.low)) break;
                            top.offer(k);
                        }
                    }
                    if (lane == 0) p.counters[first] = 0;
                    finish<DT>(p, row, sum, top.key);
                }
            }
        }
        __syncthreads();
        x += c1 - c0;
    }
}

template <int DT>
cudaError_t launch(ScoreLogitsParams & p, int sms, cudaStream_t stream) {
    if (p.out.vocab <= kThreads * kPer) {
        score_warp_kernel<DT><<<(unsigned) ((p.rows + kWarps - 1) / kWarps), kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const int64_t n_vec = p.out.vocab / Elem<DT>::kVec;
    p.strips = (n_vec + kThreads * Elem<DT>::kLoads - 1) / (kThreads * Elem<DT>::kLoads);
    const int64_t grid = std::min<int64_t>(p.strips * p.rows, (int64_t) sms * kScoreCtasPerSm);
    score_block_kernel<DT><<<(unsigned) grid, kThreads, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_score_logits(ScoreLogitsParams p, int sms, cudaStream_t stream) {
    switch (p.dtype) {
        case 0: return launch<0>(p, sms, stream);
        case 1: return launch<1>(p, sms, stream);
        case 30: return launch<30>(p, sms, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace vxk
