// Scores of logits in memory (vxk_head_score_logits): each row's given token's
// log probability, entropy and top list in one pass (the mathematics is in
// vxk_score.h).  Bound by reading the logits once.
//
// The rows' elements are cut into strips of 4096; a CTA takes an unbroken run of all rows'
// strips.  Where the rows' number lets whole rows fill the device they stay whole;
// elsewhere the runs are equal, so that any number of rows keeps the whole device busy to
// the end: a row that lies within one CTA's run is finished there, one that crosses into
// others' leaves a part in each, and the CTA that arrives last joins them (the result does
// not depend on which that is).  Rows of at most one strip go one to a warp instead: there
// the block's reductions would cost more than the read.
//
// Strips reach shared memory by bulk copies, two ahead of the one that is read.  A thread
// takes 16 elements of each and their maximum first, so that the sums are rescaled at
// most once a strip.
//
// Measured: 600 rows of 131072 f32 logits 58 us without a list (5.4 TB/s, 83 % of a copy's
// rate; two CTAs or deeper rings were no faster) and 72 with one of 8; 333 rows of 32003
// bf16 15 and 18 us; four rows 12 us, one launch, in which a row's parts are written,
// counted in and joined behind one strip a CTA.
//
// The top list costs the scan nothing but each thread's running maximum, noted a dozen
// times a run.  Behind the run the n_top-th largest of 64 groups' maxima bounds the
// list's end from below; the few noted maxima that reach it name the elements to read
// again (from L2), and the keys found there are ranked against each other, all at once.
// Where too many reach the bound (rows of equal or masked logits) the run's strips are
// gone through once more in order, each with a bound that at most n_top groups of 64
// elements reach.
#include "vxk_internal.h"
#include "vxk_score.h"
#include "vxk_tc.h"

#include <algorithm>

namespace vxk {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kRowOfWarp = 4096;  // a row of at most so many elements is one warp's

template <int DT>
struct Elem {
    static constexpr int kBytes = DT == 0 ? 4 : 2;
    static constexpr int kVec = 16 / kBytes;      // elements of a 16-byte load
    static constexpr int kPer = 16;               // elements of a strip in one thread
    static constexpr int kLoads = kPer / kVec;    // their vectors
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

// A row in memory: elements before its first 16-byte boundary, whole 16-byte vectors, and
// those behind the last.
template <int DT>
struct Row {
    const uint8_t * at;
    const uint8_t * body;
    int vocab, lead, n_vec;
    __device__ __forceinline__ Row(const ScoreLogitsParams & p, int64_t row) {
        using E = Elem<DT>;
        at = static_cast<const uint8_t *>(p.logits) + row * p.ld * E::kBytes;
        vocab = p.out.vocab;
        lead = min(vocab, (int) ((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) / E::kBytes);
        n_vec = (vocab - lead) / E::kVec;
        body = at + (int64_t) lead * E::kBytes;
    }
    // Thread t's element of those outside the vectors, -1: none (t < 32 suffices).
    __device__ __forceinline__ int ragged(int t) const {
        const int tail = lead + n_vec * Elem<DT>::kVec;
        if (t < lead) return t;
        return t >= 16 && t - 16 < vocab - tail ? tail + t - 16 : -1;
    }
};

// A thread's elements of a strip whose vectors start at v0, `team` apart, from where they
// lie (global memory, or the strip's copy in shared memory); -inf where there is none.
// Returns the largest.
template <int DT, bool SHARED>
__device__ __forceinline__ float take_strip(const Row<DT> & r, const uint8_t * from, int v0, int team,
                                            float (&x)[Elem<DT>::kPer]) {
    using E = Elem<DT>;
    uint4 u[E::kLoads];
#pragma unroll
    for (int j = 0; j < E::kLoads; ++j)
        if (v0 + j * team < r.n_vec)
            u[j] = SHARED ? *reinterpret_cast<const uint4 *>(from + j * team * 16) : load_stream(from + (int64_t) j * team * 16);
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < E::kLoads; ++j) {
        if (v0 + j * team < r.n_vec) {
            unpack<DT>(u[j], x + j * E::kVec);
        } else {
#pragma unroll
            for (int i = 0; i < E::kVec; ++i) x[j * E::kVec + i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < E::kVec; ++i) m = fmaxf(m, x[j * E::kVec + i]);
    }
    return m;
}

template <int N>
__device__ __forceinline__ void add_strip(Stat & a, const float (&x)[N], float m) {
    if (m > a.m) stat_raise(a, m);
    const float base = stat_base(a.m);
#pragma unroll
    for (int i = 0; i < N; ++i) stat_add(a, x[i], base);
}

__device__ __forceinline__ Stat warp_join(Stat a) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a = stat_join(a, stat_shfl_xor(a, o));
    return a;
}

// A row's given token and its logit, read ahead of the row: one behind the other they take
// longer than a small row does.
struct Given {
    int32_t token;
    float logit;
};
template <int DT>
__device__ __forceinline__ Given given_of(const ScoreLogitsParams & p, int64_t row) {
    Given g = {p.out.tokens ? p.out.tokens[row] : -1, 0.0f};
    const uint8_t * at = static_cast<const uint8_t *>(p.logits) + row * p.ld * Elem<DT>::kBytes;
    if (g.token >= 0 && g.token < p.out.vocab) g.logit = logit_at<DT>(at, g.token);
    return g;
}

// A row of at most one strip by one warp, its list in the warp's lanes.
template <int DT>
__global__ void __launch_bounds__(kThreads, 2) score_warp_kernel(const ScoreLogitsParams p) {
    using E = Elem<DT>;
    const int64_t row = (int64_t) blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= p.rows) return;
    const Row<DT> r(p, row);
    const Given given = given_of<DT>(p, row);
    Stat a = stat_empty();
    WarpTop top;
    top.clear(p.out.n_top);
    const int idx = r.ragged(lane);
    if (idx >= 0) {
        const float v = logit_at<DT>(r.at, idx);
        stat_raise(a, v > a.m ? v : a.m);
        stat_add(a, v, stat_base(a.m));
    }
    if (top.n_top) top.offer(idx >= 0 ? top_key(logit_at<DT>(r.at, idx), idx) : 0ull);
    for (int first = 0; first < r.n_vec; first += 32 * E::kLoads) {
        const int v0 = first + lane;
        float x[E::kPer];
        const float m = take_strip<DT, false>(r, r.body + (int64_t) v0 * 16, v0, 32, x);
        if (top.n_top) {
            // no less than any of a lane's elements; a maximum of -inf may also be that of NaNs,
            // which stand below -inf in the list and so bound nothing
            const uint32_t largest = v0 < r.n_vec ? top_bits(m) : 0u;
            if (top.low == 0ull) top.bound(m > -INFINITY ? largest : 0u);
            if (__any_sync(kAll, largest >= (uint32_t) (top.low >> 32))) {
#pragma unroll
                for (int j = 0; j < E::kLoads; ++j) {
                    const bool in = v0 + j * 32 < r.n_vec;
                    const int at = r.lead + (int) (v0 + j * 32) * E::kVec;
#pragma unroll
                    for (int i = 0; i < E::kVec; ++i) top.offer(in ? top_key(x[j * E::kVec + i], at + i) : 0ull);
                }
            }
        }
        add_strip(a, x, m);
    }
    score_write(p.out, row, warp_join(a), top.key, given.token, given.logit);
}

constexpr int kStages = 3;     // strips of a CTA under way or being read
constexpr int kNotes = 12;     // maxima that a thread notes in a run
constexpr int kCands = 512;    // noted maxima that reach the bound
// keys at once: those of n_top groups of 64 elements, the list, and a row's ragged ends
constexpr int kKeys = kMaxTop * 64 + kMaxTop + 16;

struct Collected {
    unsigned long long key[kKeys];
    unsigned long long best[kMaxTop];
    unsigned long long group[kThreads];
    unsigned long long bound;  // a key that bounds the list's end from below
    int count;
    int n_cands;
    uint16_t cand[kCands];     // thread + 256 x note
    float note[kNotes][kThreads];
};

// Ranks `n` collected keys (all threads; n is the same for all): the n_top largest, in
// order, stay, and the list's end becomes the bound.
__device__ __forceinline__ void rank_keys(Collected & c, int n, int n_top) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long mine = c.key[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += c.key[j] > mine;
        if (above < n_top) c.best[above] = mine;
    }
    __syncthreads();
    if ((int) threadIdx.x < n_top) c.key[threadIdx.x] = (int) threadIdx.x < n ? c.best[threadIdx.x] : 0ull;
    if (threadIdx.x == 0) {
        c.count = min(n, n_top);
        if (n >= n_top) c.bound = max(c.bound, c.best[n_top - 1]);
    }
    __syncthreads();
}

// The same for all that were collected, as all threads see them behind a barrier.
__device__ __forceinline__ void rank_kept(Collected & c, int n_top) {
    const int n = c.count;
    __syncthreads();
    rank_keys(c, n, n_top);
}

// Appends a key; one that finds no room is only counted.
__device__ __forceinline__ void append(Collected & c, unsigned long long k) {
    const int place = atomicAdd(&c.count, 1);
    if (place < kKeys) c.key[place] = k;
}

// The n_top-th largest of the 64 groups' keys, of four threads each with its own largest
// (0: none), into c.bound where it is more.  Ends in front of a barrier.
__device__ __forceinline__ void group_bound(Collected & c, unsigned long long mine, int n_top) {
    unsigned long long g = max(mine, __shfl_xor_sync(kAll, mine, 1));
    g = max(g, __shfl_xor_sync(kAll, g, 2));
    if (threadIdx.x % 4 == 0) c.group[threadIdx.x / 4] = g;
    __syncthreads();
    if (threadIdx.x < kThreads / 4) {
        const unsigned long long k = c.group[threadIdx.x];
        int above = 0;
        for (int j = 0; j < kThreads / 4; ++j) above += c.group[j] > k;
        if (above == n_top - 1 && k > c.bound) c.bound = k;  // keys differ: one thread
    }
}

// The run's list (strips [c0, c1) of row r) behind its scan: c.key[0 .. n_top) on return.
// `ragged` keys are in c.key already; `most` is the thread's largest element, its maxima of
// every `span` strips are noted.
template <int DT>
__device__ __forceinline__ void select(Collected & c, const Row<DT> & r, int c0, int c1, int span, float most, int ragged,
                                       int n_top) {
    using E = Elem<DT>;
    constexpr int kStep = kThreads * E::kLoads;
    const int tid = threadIdx.x;
    // maxima as keys: the value, and who holds it
    const uint32_t bits = c0 * kStep + tid < r.n_vec ? top_bits(most) : 0u;
    if (tid == 0) {
        c.bound = 0ull;
        c.n_cands = 0;
    }
    group_bound(c, bits ? top_key(most, tid) : 0ull, n_top);
    __syncthreads();
    const float low = top_below((uint32_t) (c.bound >> 32));
    for (int e = 0; e * span < c1 - c0; ++e) {
        if ((c0 + e * span) * kStep + tid < r.n_vec && !(c.note[e][tid] <= low)) {
            const int place = atomicAdd(&c.n_cands, 1);
            if (place < kCands) c.cand[place] = (uint16_t) (tid + 256 * e);
        }
    }
    __syncthreads();
    const int n_cands = c.n_cands;
    if (n_cands <= kCands) {
        for (int i = tid; i < n_cands * span * E::kLoads; i += kThreads) {
            const int who = c.cand[i / (span * E::kLoads)], in = i % (span * E::kLoads);
            const int strip = c0 + who / 256 * span + in / E::kLoads;
            const int v = strip * kStep + in % E::kLoads * kThreads + who % 256;
            if (strip >= c1 || v >= r.n_vec) continue;
            float x[E::kVec];
            unpack<DT>(load_stream(r.body + (int64_t) v * 16), x);
#pragma unroll
            for (int j = 0; j < E::kVec; ++j)
                if (!(x[j] <= low)) append(c, top_key(x[j], r.lead + v * E::kVec + j));
        }
    }
    __syncthreads();
    const int n = c.count;
    __syncthreads();
    // (fewer than n_top where the rest is NaN)
    if (n_cands <= kCands && n <= kKeys && n >= min(n_top, (c1 - c0) * kStep * E::kVec)) {
        rank_keys(c, n, n_top);
        return;
    }
    if (tid == 0) {
        c.bound = 0ull;
        c.count = ragged;
    }
    __syncthreads();
    for (int s = c0; s < c1; ++s) {
        const int v0 = s * kStep + tid;
        float x[E::kPer];
        take_strip<DT, false>(r, r.body + (int64_t) v0 * 16, v0, kThreads, x);
        // Whole keys: the list's last may be one of the row's last elements, which are in it from
        // the start, and an element of the same value here stands before it.
        const unsigned long long last = c.bound;
        bool any = false;
#pragma unroll
        for (int i = 0; i < E::kPer; ++i) {
            const int v = v0 + i / E::kVec * kThreads;
            any |= v < r.n_vec && top_key(x[i], r.lead + v * E::kVec + i % E::kVec) > last;
        }
        if (!__syncthreads_or(any)) continue;
        int at = -1;  // the thread's first element of the largest bits
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < E::kPer; ++i) {
            const int v = v0 + i / E::kVec * kThreads;
            if (v < r.n_vec && top_bits(x[i]) > largest) {
                largest = top_bits(x[i]);
                at = r.lead + v * E::kVec + i % E::kVec;
            }
        }
        group_bound(c, largest ? ((unsigned long long) largest << 32) | (0xFFFFFFFFu - (uint32_t) at) : 0ull, n_top);
        __syncthreads();
        const unsigned long long bound = c.bound;
#pragma unroll
        for (int i = 0; i < E::kPer; ++i) {
            const int v = v0 + i / E::kVec * kThreads;
            const unsigned long long k = top_key(x[i], r.lead + v * E::kVec + i % E::kVec);
            if (v < r.n_vec && k >= bound) append(c, k);
        }
        __syncthreads();
        rank_kept(c, n_top);
    }
    rank_kept(c, n_top);
}

template <int DT, bool LIST>
__global__ void __launch_bounds__(kThreads, kScoreCtasPerSm) score_block_kernel(const ScoreLogitsParams p) {
    using E = Elem<DT>;
    __shared__ Stat stats[kWarps];
    __shared__ Collected keys;
    __shared__ int arrived;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n_top = LIST ? p.out.n_top : 0;
    const int strips = (int) p.strips;
    const int64_t total = strips * p.rows;
    const uint32_t grid = gridDim.x, cta = blockIdx.x;
    const int64_t units = total / p.unit;
    const int64_t begin = cta * units / grid * p.unit, end = (cta + 1) * units / grid * p.unit;
    constexpr int kStep = kThreads * E::kLoads;  // vectors of a strip
    constexpr int kStripBytes = kStep * 16;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t full[kStages], empty[kStages];
    __shared__ volatile int32_t abort_flag;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kWarps);
        }
        abort_flag = 0;
        mbar_fence_init();
    }
    __syncthreads();
    // Strips under way: thread 0 copies the run's next strip as soon as the warps have read
    // the one in its place.  A wait that runs out sets the error word and goes on: what
    // is then read is wrong but lies in the ring.
    __shared__ int64_t fed_row;  // thread 0's: the strip to copy next
    __shared__ int fed_strip;
    if (tid == 0) {
        fed_row = begin / strips;
        fed_strip = (int) (begin % strips);
    }
    uint32_t turn = 0;
    auto feed = [&](uint32_t nth) {  // the run's nth strip
        if (tid != 0 || (int64_t) nth >= end - begin) return;
        const int st = nth % kStages;
        tc_wait(&empty[st], ((nth / kStages) & 1) ^ 1, &abort_flag, p.out.error);
        const Row<DT> r(p, fed_row);
        const int v0 = fed_strip * kStep;
        const uint32_t bytes = (uint32_t) max(0, min(kStep, r.n_vec - v0)) * 16;
        mbar_expect_tx(&full[st], bytes);
        if (bytes) bulk_load(ring + st * kStripBytes, r.body + (int64_t) v0 * 16, bytes, &full[st]);
        if (++fed_strip == strips) {
            fed_strip = 0;
            ++fed_row;
        }
    };
    for (int i = 0; i < kStages - 1; ++i) feed(i);

    for (int64_t at = begin; at < end;) {
        const int64_t row = at / strips;
        const int c0 = (int) (at - row * strips), c1 = (int) min((int64_t) strips, c0 + end - at);
        const Row<DT> r(p, row);
        Given given = {-1, 0.0f};
        if (warp == 0) given = given_of<DT>(p, row);
        Stat a = stat_empty();
        if (tid == 0) {
            keys.bound = 0ull;
            keys.count = 0;
        }
        __syncthreads();
        if (c0 == 0) {
            const int idx = r.ragged(tid);
            if (idx >= 0) {
                const float v = logit_at<DT>(r.at, idx);
                stat_raise(a, v > a.m ? v : a.m);
                stat_add(a, v, stat_base(a.m));
                if (n_top) keys.key[atomicAdd(&keys.count, 1)] = top_key(v, idx);
            }
            __syncthreads();
        }
        const int ragged = keys.count;
        __syncthreads();
        const int span = (c1 - c0 + kNotes - 1) / kNotes;  // strips of a note
        float most = -INFINITY, note = -INFINITY;
        int noted = 0, left = span;
        for (int c = c0; c < c1; ++c) {
            const int v0 = c * kStep + tid;
            float x[E::kPer];
            const int st = turn % kStages;
            tc_wait(&full[st], (turn / kStages) & 1, &abort_flag, p.out.error);
            const float m = take_strip<DT, true>(r, ring + st * kStripBytes + tid * 16, v0, kThreads, x);
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
            ++turn;
            feed(turn + kStages - 2);
            add_strip(a, x, m);
            if constexpr (LIST) {
                note = fmaxf(note, m);
                if (--left == 0 || c + 1 == c1) {
                    keys.note[noted++][tid] = note;
                    most = fmaxf(most, note);
                    note = -INFINITY;
                    left = span;
                }
            }
        }
        a = warp_join(a);
        if (lane == 0) stats[warp] = a;
        __syncthreads();
        if (n_top) select(keys, r, c0, c1, span, most, ragged, n_top);
        if (warp == 0) {
            a = lane < kWarps ? stats[lane] : stat_empty();
            a = warp_join(a);
        }
        const unsigned long long mine = tid < n_top ? keys.key[tid] : 0ull;
        if (c1 - c0 == strips) {
            if (warp == 0) score_write(p.out, row, a, mine, given.token, given.logit);
        } else {
            // the CTAs whose runs hold this row's first and last strips
            const int64_t r0 = row * strips;
            const int from = (int) (((r0 + 1) * grid - 1) / total), upto = (int) (((r0 + strips) * grid - 1) / total);
            if (warp == 0) {
                ScorePart * part = p.parts + 2 * cta + (at == begin ? 0 : 1);
                if (lane == 0) {
                    part->m = a.m;
                    part->s = a.s;
                    part->t = a.t;
                }
                if (lane < n_top) part->top[lane] = mine;
                __threadfence();
                __syncwarp();
                if (lane == 0) arrived = atomicAdd(&p.counters[from], 1);
            }
            __syncthreads();
            if (arrived == upto - from) {
                __threadfence();
                auto part_of = [&](int b) {
                    const bool mid = b == from && b * total / grid != r0;
                    return p.parts + 2 * b + (mid ? 1 : 0);
                };
                // the n_top-th largest of the parts' largest keys bounds the list from below
                if (tid == 0) {
                    keys.bound = 0ull;
                    keys.count = 0;
                }
                Stat one = stat_empty();
                unsigned long long most = 0ull;
                for (int b0 = from; b0 <= upto; b0 += kThreads) {
                    const int b = b0 + tid;
                    if (b <= upto) {
                        const ScorePart * q = part_of(b);
                        one = stat_join(one, Stat{__ldcg(&q->m), __ldcg(&q->s), __ldcg(&q->t)});
                        if (n_top) most = max(most, __ldcg(&q->top[0]));
                    }
                }
                one = warp_join(one);
                if (lane == 0) stats[warp] = one;
                keys.group[tid] = most;
                __syncthreads();
                if (n_top && most) {
                    int above = 0;
                    const int parts = min(kThreads, upto - from + 1);
                    for (int j = 0; j < parts; ++j) above += keys.group[j] > most;
                    if (above == n_top - 1) keys.bound = most;
                }
                __syncthreads();
                // at most 1024 keys at a time
                const int step = n_top ? 1024 / kMaxTop : upto - from + 1;
                for (int b0 = from; n_top && b0 <= upto; b0 += step) {
                    for (int i = tid; i < step * n_top; i += kThreads) {
                        const int b = b0 + i / n_top;
                        if (b > upto) break;
                        const unsigned long long k = __ldcg(&part_of(b)->top[i % n_top]);
                        if (k && k >= keys.bound) keys.key[atomicAdd(&keys.count, 1)] = k;
                    }
                    __syncthreads();
                    rank_kept(keys, n_top);
                }
                if (warp == 0) {
                    one = warp_join(lane < kWarps ? stats[lane] : stat_empty());
                    if (lane == 0) p.counters[from] = 0;
                    score_write(p.out, row, one, lane < n_top ? keys.key[lane] : 0ull, given.token, given.logit);
                }
            }
        }
        __syncthreads();
        at += c1 - c0;
    }
}

template <int DT>
cudaError_t launch(ScoreLogitsParams & p, int sms, cudaStream_t stream) {
    if (p.out.vocab <= kRowOfWarp) {
        score_warp_kernel<DT><<<(unsigned) ((p.rows + kWarps - 1) / kWarps), kThreads, 0, stream>>>(p);
        return cudaGetLastError();
    }
    const int64_t n_vec = p.out.vocab / Elem<DT>::kVec;
    p.strips = (n_vec + kThreads * Elem<DT>::kLoads - 1) / (kThreads * Elem<DT>::kLoads);
    const int64_t most = (int64_t) sms * kScoreCtasPerSm;
    // Whole rows where that lengthens no run by more than six strips, what a row's parts
    // cost to write, wait for and join.  Measured on 444 CTAs, split / whole (us, bf16, no
    // list): 333 rows of 8 strips 18 / 15, 500 rows (9 or 16 strips a run) 21 / 22, 148 rows
    // of 32 strips (11 or 32) 21 / 27, 400 rows (29 or 32) 42 / 39; f32 is alike.
    const int64_t split = p.strips * p.rows / most, whole = (p.rows + most - 1) / most * p.strips;
    p.unit = whole <= split + 6 ? p.strips : 1;
    const int64_t grid = std::min(p.strips * p.rows / p.unit, most);
    constexpr int kRing = kStages * kThreads * Elem<DT>::kLoads * 16;
    auto kernel = p.out.n_top > 0 ? score_block_kernel<DT, true> : score_block_kernel<DT, false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned) grid, kThreads, kRing, stream>>>(p);
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
