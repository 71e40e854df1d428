// Scores of hidden rows (vxk_head_score): the logits W x of up to 2048 rows, their
// softmax statistics and top lists, without the logits in memory (the mathematics
// of the scores is in vxk_score.h).
//
// Bound by reading W (few rows) or by the tensor cores (many).  The rows are the M
// operand and a slice of the vocabulary the N operand of tcgen05.mma, so a thread of
// the epilogue owns one row and half of a slice's columns: it keeps the row's
// statistics in registers over all slices of its CTA and nothing crosses threads
// before the end.
//
//   up to 128 rows   one CTA per tile of 128 rows x tile_cols (cta_group::1)
//   more             a CTA pair per tile of 256 rows x tile_cols (cta_group::2):
//                    each CTA loads its own 128 rows of x and half of the slice of
//                    W, 32 KB instead of 48 KB a 64-column step, so that the L2 can
//                    feed the tensor cores
//
// The tensor cores' accumulation drops the bits below 2^-23 of the running sum at
// every step: over 4096 columns the largest logits come out 6e-6 too small, and the
// entropy 4e-5 off.  So a sum is taken out every 512 columns (bf16) or 256 (f16, whose
// products have six bits more to lose), two accumulators in turn in TMEM, and added up
// in fp32 registers: 128 columns a thread, eight epilogue warps (segment_of).  Entropies of
// 700 rows of 2048 columns are then 4.3e-6 off (bf16) or 4.9e-6 (f16), a plain fp32
// product's 5e-6.  What is dropped always makes a sum smaller in magnitude; giving its mean
// back as a factor would halve these errors or better for rows like those measured, but
// change sums of few columns or few bits, of which nothing was dropped, by up to 11
// units in the last place.
//
// Measured (bf16) in short runs (in brackets: back to back, under the power cap): 100 rows x
// 131072 x 2048 102 us with lists of 4, 5.3 TB/s of W (112; 93 without lists); 2000 rows x
// 131072 x 4096 1590 us, 1.35 PFLOP/s (1700; without lists 1450, 1.48; a plain library product
// reaches 1.66 in a burst and 1.39 under the power cap), of f16, whose segments are half as
// long, 2000 (2110: the TMEM reads); 5 rows of f16 x
// 32000 x 1280 29 us, of which three launches and the join are 14.  The lists' cost
// is the few candidates behind each row's bound, looked for by every thread of a tile.
//
// A row's top list is found by 2 n_groups threads, each over its own columns.  What
// one thread knows of the list's end bounds it for all, so they share the largest such
// bound in global memory (row_low) and few candidates are left to any of them; the
// lists do not depend on when a bound is seen, only the work does.
//
// Persistent: CTA (or pair) c takes row tile c mod n_row_tiles and the slices
// c / n_row_tiles, + n_groups, ...: CTAs of different row tiles walk the same slices
// at the same time and share them in L2.
//   warp 0      TMA producer      warp 1   tcgen05.mma issuer (the pair's first CTA)
//   warps 4-11  epilogue: TMEM lane quadrant warp % 4, columns of half (warp - 4) / 4
#include "vxk_internal.h"
#include "vxk_score.h"
#include "vxk_tc.h"

#include <algorithm>

namespace vxk {
namespace {

constexpr int kThreads = 384;
constexpr int kMostGroups = 160;                // CTAs that share a row tile, at most
// Registers a thread after the split: 128 x 40 + 256 x 232 = 128 x 24 + 256 x 240 = 384 x 168,
// the launch's; which of the two leaves no role spilling goes by the list.
template <int LIST>
constexpr int kRegsIssue = LIST ? 40 : 24;
template <int LIST>
constexpr int kRegsEpilogue = LIST ? 232 : 240;
constexpr int kChunk = 64;                      // columns of x and W in a stage (one 128-byte row)
constexpr int kXBytes = 128 * 128;              // a CTA's rows of x in a stage
constexpr int kHalfCols = 128;                  // most columns of a tile in one epilogue thread
constexpr int kTmemCols = 512;
constexpr int kRing = 192 * 1024;               // 4 stages of 48 KB, or 6 of 32 KB
constexpr int kListBytes = kMaxTop * 256 * 8;   // the epilogue threads' top lists
constexpr int kOffBar = kRing + kListBytes;
constexpr int kSmem = kOffBar + 256 + 1024;     // + alignment slack
static_assert(kSmem <= 232448, "head scoring exceeds 227 KB of shared memory");

template <int CG>
struct Shape {
    static constexpr int kStages = CG == 1 ? 4 : 6;
    static constexpr int kStageBytes = kRing / kStages;
    static constexpr int kFull = 0, kEmpty = kStages, kDFull = 2 * kStages, kDEmpty = kDFull + 2, kDrain = kDEmpty + 2;
    static constexpr int kBars = kDrain + 1;
};

// Chunks summed in TMEM before they are moved to registers: 8 (bf16) or 4 (f16).  Where a plain
// fp32 product is more exact than its usual few 1e-6 the segments are shorter.  Rows of fewer
// than 1280 columns: at 1024, 2000 rows x 30000, 6 for 8 takes 153 us for 140 and brings an
// entropy's error from 4.7e-6 to 3.2e-6 (bf16; plain 3.6e-6), 3 for 4 197 us for 170 and 5.4e-6 to
// 3.5e-6 (f16; plain 4.2e-6).  Up to 16 rows, which a plain product sums in trees: 2, no slower
// than 8, or 1 for up to four rows of f16 (2.2e-6 -> 1.2e-6, a unit or two in a logit's last
// place; one row x 131072 x 2048 104 -> 130 us, x 32000 x 1280 28.7 -> 29.9).
template <int DT>
__device__ __forceinline__ int segment_of(int n_rows, int n_chunks) {
    if (n_rows <= 16) return DT != 30 && n_rows <= 4 ? 1 : 2;
    return DT == 30 ? min(8, max(1, n_chunks * 2 / 5)) : min(4, max(1, n_chunks / 5));
}

// One thread's list of its largest keys, largest first.  LIST 0: none; up to 4 places in
// registers (an insertion is four compares and swaps); up to 16 in shared memory, the
// j-th at at[j * 256].
template <int LIST>
struct ThreadTop {
    unsigned long long key[LIST == 4 ? 4 : 1];
    unsigned long long * at;
    int n_top;

    __device__ __forceinline__ void clear(unsigned long long * place, int n) {
        at = place;
        n_top = n;
        if constexpr (LIST == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) key[j] = 0ull;
        }
        if constexpr (LIST == 16) {
            for (int j = 0; j < n_top; ++j) at[j * 256] = 0ull;
        }
    }
    __device__ __forceinline__ void insert(unsigned long long k) {
        if constexpr (LIST == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool above = k > key[j];
                const unsigned long long down = above ? key[j] : k;
                key[j] = above ? k : key[j];
                k = down;
            }
        }
        if constexpr (LIST == 16) {
            int j = n_top - 1;
            for (; j > 0; --j) {
                const unsigned long long up = at[(j - 1) * 256];
                if (up > k) break;
                at[j * 256] = up;
            }
            at[j * 256] = k;
        }
    }
    // The n_top-th key, 0 while there are fewer.
    __device__ __forceinline__ unsigned long long end() const {
        if constexpr (LIST == 4) {
            const unsigned long long a = n_top > 1 ? key[1] : key[0], b = n_top > 3 ? key[3] : key[2];
            return n_top > 2 ? b : a;
        }
        if constexpr (LIST == 16) return at[(n_top - 1) * 256];
        return 0ull;
    }
    __device__ __forceinline__ void store(unsigned long long * to) const {  // [n_top], 128 apart
        if constexpr (LIST == 4) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < n_top) to[j * 128] = key[j];
        }
        if constexpr (LIST == 16) {
            for (int j = 0; j < n_top; ++j) to[j * 128] = at[j * 256];
        }
    }
};

template <int DT, int CG, int LIST>
__global__ void __launch_bounds__(kThreads, 1) head_score_kernel(const __grid_constant__ CUtensorMap tmw,
                                                                 const __grid_constant__ CUtensorMap tmx,
                                                                 const HeadScoreParams p) {
    using S = Shape<CG>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned long long * lists = reinterpret_cast<unsigned long long *>(base + kRing);
    uint64_t * bars = reinterpret_cast<uint64_t *>(base + kOffBar);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(base + kOffBar + 8 * S::kBars);
    volatile int32_t * abort_flag = reinterpret_cast<volatile int32_t *>(base + kOffBar + 8 * S::kBars + 4);

    const int tid = threadIdx.x, warp = (int) uniform(tid >> 5), lane = tid & 31;
    const int rank = CG == 2 ? (int) cluster_rank() : 0;
    const int unit = (int) blockIdx.x / CG;
    const int row_tile = unit % p.n_row_tiles, group = unit / p.n_row_tiles;
    const int row0 = row_tile * (128 * CG) + rank * 128;  // this CTA's first row
    const int n_chunks = p.dim / kChunk;
    const int segment = segment_of<DT>(p.n_rows, n_chunks);
    const int n_segs = (n_chunks + segment - 1) / segment;

    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&bars[S::kFull + s], 1);
            mbar_init(&bars[S::kEmpty + s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bars[S::kDFull + b], 1);
            mbar_init(&bars[S::kDEmpty + b], 8 * CG);
        }
        mbar_init(&bars[S::kDrain], 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<CG>(tmem_slot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue<LIST>));
        if (warp == 0 && lane == 0) {
            const int w_rows = p.tile_cols / CG;
            const uint32_t bytes = (uint32_t) (p.x_box_rows + w_rows) * 128;
            uint32_t c = 0;
            bool ok = true;
            // W is no other launch's output: the first stages' part of it is under way while
            // the rows are still being rounded
            const int early = min(S::kStages, n_chunks);
            for (int ch = 0; ch < early; ++ch) {
                if (rank == 0) mbar_expect_tx(&bars[S::kFull + ch], bytes * CG);
                tma_load_2d<CG>(base + ch * S::kStageBytes + kXBytes, &tmw, ch * kChunk,
                                group * p.tile_cols + rank * w_rows, &bars[S::kFull + ch]);
            }
            asm volatile("griddepcontrol.wait;" ::: "memory");
            for (; (int) c < early; ++c)
                tma_load_2d<CG>(base + c * S::kStageBytes, &tmx, (int) c * kChunk, row0, &bars[S::kFull + c]);
            for (int tile = group; ok && tile < p.n_tiles; tile += p.n_groups) {
                for (int ch = tile == group ? early : 0; ch < n_chunks; ++ch, ++c) {
                    const int st = (int) (c % S::kStages);
                    if (!tc_wait(&bars[S::kEmpty + st], ((c / S::kStages) & 1) ^ 1, abort_flag, p.error)) {
                        ok = false;
                        break;
                    }
                    uint8_t * dst = base + st * S::kStageBytes;
                    if (rank == 0) mbar_expect_tx(&bars[S::kFull + st], bytes * CG);
                    tma_load_2d<CG>(dst, &tmx, ch * kChunk, row0, &bars[S::kFull + st]);
                    tma_load_2d<CG>(dst + kXBytes, &tmw, ch * kChunk, tile * p.tile_cols + rank * w_rows,
                                    &bars[S::kFull + st]);
                }
            }
            // copies in flight land before the CTA leaves (a pair's land on its first CTA's barriers)
            if (rank == 0)
                for (uint32_t d = c > (uint32_t) S::kStages ? c - S::kStages : 0; d < c; ++d)
                    tc_drain(&bars[S::kFull + d % S::kStages], (d / S::kStages) & 1);
        }
        if (warp == 1 && rank == 0) {
            constexpr uint32_t fmt = DT == 30 ? 1u : 0u;
            const uint32_t idesc = tc_idesc(fmt, 128 * CG, p.tile_cols);
            const uint32_t ring = smem_u32(base);
            uint32_t st = 0, par = 0, seg = 0;
            bool ok = true;
            for (int tile = group; ok && tile < p.n_tiles; tile += p.n_groups) {
                for (int s = 0; ok && s < n_segs; ++s, ++seg) {
                    const uint32_t b = seg & 1;
                    ok = uniform(tc_wait(&bars[S::kDEmpty + b], ((seg >> 1) & 1) ^ 1, abort_flag, p.error));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem + 256 * b;
                    const int last = min(n_chunks, (s + 1) * segment);
                    for (int ch = s * segment; ch < last; ++ch) {
                        ok = uniform(tc_wait(&bars[S::kFull + st], par, abort_flag, p.error));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t xa = ring + st * S::kStageBytes;
                        const uint64_t da = sw128_desc(xa, 16, 1024), db = sw128_desc(xa + kXBytes, 16, 1024);
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks)  // 32 bytes further: 2 in the descriptor's 16-byte units
                                tc_mma<CG>(d, da + 2 * ks, db + 2 * ks, idesc, (ch != s * segment) | (ks != 0));
                            tc_commit<CG>(&bars[S::kEmpty + st]);
                            if (ch + 1 == last) tc_commit<CG>(&bars[S::kDFull + b]);
                        }
                        __syncwarp();
                        if (++st == S::kStages) st = 0, par ^= 1;
                    }
                }
            }
            if (elect_one()) {
                tc_commit<CG>(&bars[S::kDrain]);
                tc_drain(&bars[S::kDrain], 0);
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpilogue<LIST>));
        const int q = warp & 3, half = (warp - 4) >> 2;
        const int t = half * 128 + q * 32 + lane;   // this thread's place in the lists
        const int row = row0 + q * 32 + lane;
        const int n_half = p.tile_cols / 2;
        const uint32_t lane_off = ((uint32_t) (32 * q) << 16) + (uint32_t) (half * n_half);
        const int n_top = p.n_top;
        ThreadTop<LIST> list;
        list.clear(lists + t, n_top);
        // What a candidate has to be above: NaN without a bound; the value below the bound;
        // the list's last value once it is full (a later column of that value comes after
        // it, so "above" is enough).
        float low = __uint_as_float(0x7fc00000u);
        unsigned long long low_key = 0ull;
        const bool listed = LIST != 0 && row < p.n_rows;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int32_t token = p.tokens && row < p.n_rows ? p.tokens[row] : -1;
        Stat a = stat_empty();
        uint32_t seg = 0;  // two accumulators in turn: bit 0, and the parity in bit 1
        bool have = true;
        const bool rows_here = row0 + q * 32 < p.n_rows;  // the same for a warp
        for (int tile = group; have && tile < p.n_tiles; tile += p.n_groups) {
            float acc[kHalfCols];
            for (int s = 0; s < n_segs; ++s, ++seg) {
                const int b = (int) (seg & 1);
                have = __all_sync(kAll, tc_wait(&bars[S::kDFull + b], (seg >> 1) & 1, abort_flag, p.error));
                if (!have) break;
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < kHalfCols; c0 += 32) {
                    if (!rows_here) break;
                    float v[32];
                    tmem_ld32(tmem + 256 * b + lane_off + c0, v);
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c0 + j] = s == 0 ? v[j] : acc[c0 + j] + v[j];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster<CG>(&bars[S::kDEmpty + b], 0);
            }
            if (!have) break;
            if (!rows_here) continue;
            // the row's bound so far, on its way while the statistics are taken
            uint32_t bound = listed && tile != group ? __ldcg(&p.row_low[row]) : 0u;
            const int col0 = tile * p.tile_cols + half * n_half;
            const int limit = min(n_half, p.vocab - col0);
            if (limit < kHalfCols) {
#pragma unroll
                for (int j = 0; j < kHalfCols; ++j)
                    if (j >= limit) acc[j] = -INFINITY;
            }
            const int given = token - col0;
            if (__any_sync(kAll, token >= 0 && given >= 0 && given < limit)) {
                float l = 0.0f;
#pragma unroll
                for (int j = 0; j < kHalfCols; ++j)
                    if (j == given) l = acc[j];
                if (token >= 0 && given >= 0 && given < limit) p.token_logits[row] = l;
            }
            float most[16];                         // the largest of every eight
#pragma unroll
            for (int g = 0; g < 16; ++g) {
                most[g] = acc[8 * g];
#pragma unroll
                for (int j = 1; j < 8; ++j) most[g] = fmaxf(most[g], acc[8 * g + j]);
            }
            float m = most[0];                      // the tile's
#pragma unroll
            for (int g = 1; g < 16; ++g) m = fmaxf(m, most[g]);
            if (listed && tile == group) {
                // The n_top-th largest of these maxima is no more than the n_top-th largest
                // of all the row's logits: what is below it is in no list.
                float sorted[16];
#pragma unroll
                for (int g = 0; g < 16; ++g) sorted[g] = fmaxf(most[g], -INFINITY);  // NaN: no number
#pragma unroll
                for (int size = 2; size <= 16; size *= 2)
#pragma unroll
                    for (int step = size / 2; step >= 1; step /= 2)
#pragma unroll
                        for (int g = 0; g < 16; ++g)
                            if ((g & step) == 0) {
                                const float x = sorted[g], y = sorted[g + step];
                                const bool down = (g & size) == 0;
                                sorted[g] = down ? fmaxf(x, y) : fminf(x, y);
                                sorted[g + step] = down ? fminf(x, y) : fmaxf(x, y);
                            }
#pragma unroll
                for (int g = 0; g < 16; ++g)
                    if (g == n_top - 1 && sorted[g] > -INFINITY) bound = top_bits(sorted[g]);
                if (bound) atomicMax(&p.row_low[row], bound);
            }
            if (m > a.m) stat_raise(a, m);
            const float from = stat_base(a.m);
#pragma unroll
            for (int j = 0; j < kHalfCols; ++j) stat_add(a, acc[j], from);
            if (listed) {
                if (tile == group) bound = __ldcg(&p.row_low[row]);  // the others' first bounds, as they come
                if ((unsigned long long) bound << 32 > low_key) {
                    low_key = (unsigned long long) bound << 32;
                    low = top_below(bound);
                }
                if (!(m <= low)) {
                    bool raised = false;
#pragma unroll
                    for (int g = 0; g < 16; ++g) {
                        if (!(most[g] <= low)) {
                            uint32_t mask = 0;
#pragma unroll
                            for (int j = 0; j < 8; ++j) mask |= !(acc[8 * g + j] <= low) ? 1u << j : 0u;
                            if (limit < 8 * g + 8) mask &= limit <= 8 * g ? 0u : (1u << (limit - 8 * g)) - 1u;
                            while (mask) {
                                const int at = __ffs(mask) - 1;
                                mask &= mask - 1;
                                float v = acc[8 * g];
#pragma unroll
                                for (int j = 1; j < 8; ++j)
                                    if (j == at) v = acc[8 * g + j];
                                const unsigned long long k = top_key(v, col0 + 8 * g + at);
                                if (k > low_key) {
                                    list.insert(k);
                                    const unsigned long long end = list.end();
                                    if (end > low_key) {
                                        low_key = end;
                                        low = top_value(end);
                                        raised = true;
                                    }
                                }
                            }
                        }
                    }
                    if (raised) atomicMax(&p.row_low[row], (uint32_t) (low_key >> 32));
                }
            }
        }
        // this thread's part of its row
        const int64_t slot = ((int64_t) unit * CG + rank) * 2 + half;
        const int place = q * 32 + lane;
        p.part_stats[slot * 128 + place] = make_float4(a.m, a.s, a.t, 0.0f);
        list.store(p.part_keys + slot * n_top * 128 + place);
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<CG>(tmem, kTmemCols);
    }
}

// x [n_rows][dim] fp32 -> 16 bits, four values a thread; clears the rows' bounds.
template <int DT>
__global__ void __launch_bounds__(256) head_round_kernel(const float4 * x, uint2 * xh, int64_t n, uint32_t * row_low,
                                                         int n_rows) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i < n_rows) row_low[i] = 0u;
    if (i >= n) return;
    const float4 v = x[i];
    if constexpr (DT == 30) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        xh[i] = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        xh[i] = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    }
}

__device__ __forceinline__ int64_t part_slot(const HeadScoreParams & p, int cg, int row, int i) {
    const int64_t unit = (int64_t) (i >> 1) * p.n_row_tiles + row / (128 * cg);
    return (unit * cg + row / 128 % cg) * 2 + (i & 1);
}

// Joins the parts of a row by a warp, a lane one part at a time: rows with few parts.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(kJoinWarps * 32) head_join_warp_kernel(const HeadScoreParams p, const ScoreOut out, int cg) {
    const int lane = threadIdx.x & 31, row = (int) blockIdx.x * kJoinWarps + (threadIdx.x >> 5), place = row % 128;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= p.n_rows) return;
    const int32_t token = out.tokens ? out.tokens[row] : -1;
    const float token_logit = p.token_logits[row];
    Stat a = stat_empty();
    WarpTop top;
    top.clear(p.n_top);
    if (p.n_top) top.raise(p.row_low[row]);
    for (int i0 = 0; i0 < 2 * p.n_groups; i0 += 32) {
        const int i = i0 + lane;
        const bool in = i < 2 * p.n_groups;
        const int64_t slot = part_slot(p, cg, row, i);
        unsigned long long k = in && p.n_top ? p.part_keys[slot * p.n_top * 128 + place] : 0ull;
        if (in) {
            const float4 s = p.part_stats[slot * 128 + place];
            a = stat_join(a, Stat{s.x, s.y, s.z});
        }
        for (int j = 0; j < p.n_top; ++j) {
            if (j) k = in ? p.part_keys[(slot * p.n_top + j) * 128 + place] : 0ull;
            if (j == 0 && i0 == 0) top.bound((uint32_t) (k >> 32));
            if (!__any_sync(kAll, k > top.low)) break;  // the parts' lists are in order
            top.offer(k);
        }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a = stat_join(a, stat_shfl_xor(a, o));
    score_write(out, row, a, top.key, token, token_logit);
}

// The same by a CTA, a thread one part: few rows, of many parts.  The keys that reach the
// row's bound are ranked against each other.
constexpr int kJoinKeys = 2 * kMostGroups * kMaxTop;
__global__ void __launch_bounds__(kJoinWarps * 32) head_join_block_kernel(const HeadScoreParams p, const ScoreOut out, int cg) {
    __shared__ Stat stats[kJoinWarps];
    __shared__ unsigned long long keys[kJoinKeys], best[kMaxTop], group[64], bound;
    __shared__ int count;
    constexpr int kThreadsOfRow = kJoinWarps * 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = (int) blockIdx.x, place = row % 128;
    const int n_top = p.n_top, n_parts = 2 * p.n_groups;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int32_t token = out.tokens ? out.tokens[row] : -1;
    const float token_logit = p.token_logits[row];
    const uint32_t low = n_top ? p.row_low[row] : 0u;
    Stat a = stat_empty();
    unsigned long long first[2] = {0ull, 0ull};  // its parts' largest keys
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int i = tid + t * kThreadsOfRow;
        if (i < n_parts) {
            const int64_t slot = part_slot(p, cg, row, i);
            const float4 s = p.part_stats[slot * 128 + place];
            if (n_top) first[t] = p.part_keys[slot * n_top * 128 + place];
            a = stat_join(a, Stat{s.x, s.y, s.z});
        }
    }
    if (tid == 0) {
        count = 0;
        bound = (unsigned long long) low << 32;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) a = stat_join(a, stat_shfl_xor(a, o));
    if (lane == 0) stats[warp] = a;
    if (n_top) {  // the n_top-th largest of 64 groups' keys bounds the list closer than any one part could
        unsigned long long g = max(first[0], first[1]);
        g = max(g, __shfl_xor_sync(kAll, g, 1));
        g = max(g, __shfl_xor_sync(kAll, g, 2));
        if (tid % 4 == 0) group[tid / 4] = g;
        __syncthreads();
        if (tid < 64) {
            int above = 0;
            for (int j = 0; j < 64; ++j) above += group[j] > group[tid];
            if (above == n_top - 1 && group[tid] > bound) bound = group[tid];  // keys differ: one thread
        }
    }
    __syncthreads();
    const unsigned long long least = bound;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int64_t slot = part_slot(p, cg, row, tid + t * kThreadsOfRow);
        unsigned long long k = first[t];
        for (int j = 0; k && k >= least; ) {
            keys[atomicAdd(&count, 1)] = k;
            if (++j == n_top) break;
            k = p.part_keys[(slot * n_top + j) * 128 + place];  // a part's list is in order
        }
    }
    __syncthreads();
    const int n = count;
    for (int i = tid; i < n; i += kThreadsOfRow) {
        const unsigned long long mine = keys[i];
        int above = 0;
        for (int j = 0; j < n; ++j) above += keys[j] > mine;
        if (above < n_top) best[above] = mine;
    }
    __syncthreads();
    if (warp != 0) return;
    a = lane < kJoinWarps ? stats[lane] : stat_empty();
#pragma unroll
    for (int o = kJoinWarps / 2; o >= 1; o >>= 1) a = stat_join(a, stat_shfl_xor(a, o));
    a = {__shfl_sync(kAll, a.m, 0), __shfl_sync(kAll, a.s, 0), __shfl_sync(kAll, a.t, 0)};
    score_write(out, row, a, lane < min(n, n_top) ? best[lane] : 0ull, token, token_logit);
}

template <int DT, int CG, int LIST>
cudaError_t launch_list(const HeadScoreParams & p, const CUtensorMap & tmw, const CUtensorMap & tmx, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(head_score_kernel<DT, CG, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (p.n_row_tiles * p.n_groups * CG));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CG;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, head_score_kernel<DT, CG, LIST>, tmw, tmx, p);
}

template <int DT>
cudaError_t launch(const HeadScoreParams & p, const CUtensorMap & tmw, const CUtensorMap & tmx, int cg,
                   cudaStream_t stream) {
    if (cg == 1) {
        if (p.n_top == 0) return launch_list<DT, 1, 0>(p, tmw, tmx, stream);
        if (p.n_top <= 4) return launch_list<DT, 1, 4>(p, tmw, tmx, stream);
        return launch_list<DT, 1, 16>(p, tmw, tmx, stream);
    }
    if (p.n_top == 0) return launch_list<DT, 2, 0>(p, tmw, tmx, stream);
    if (p.n_top <= 4) return launch_list<DT, 2, 4>(p, tmw, tmx, stream);
    return launch_list<DT, 2, 16>(p, tmw, tmx, stream);
}

}  // namespace

// How a pass of n_rows rows is cut: row tiles, groups of CTAs (or pairs) that share
// a row tile's vocabulary, and slices of the vocabulary as wide as keeps the groups'
// numbers of slices equal.
HeadScorePlan head_score_plan(int32_t n_rows, int32_t vocab, int sms) {
    HeadScorePlan c{};
    c.cg = n_rows <= 128 ? 1 : 2;
    c.n_row_tiles = (n_rows + 128 * c.cg - 1) / (128 * c.cg);
    const int64_t groups = std::min(kMostGroups, std::max(1, sms / c.cg / c.n_row_tiles));
    const int64_t rounds = (vocab + groups * 256 - 1) / (groups * 256);
    const int64_t cols = ((int64_t) vocab + groups * rounds - 1) / (groups * rounds);
    c.tile_cols = (int32_t) std::min<int64_t>(256, (cols + 31) / 32 * 32);
    c.n_tiles = (vocab + c.tile_cols - 1) / c.tile_cols;
    c.n_groups = (int32_t) std::min<int64_t>(groups, c.n_tiles);
    c.x_box_rows = c.cg == 2 ? 128 : (n_rows + 7) / 8 * 8;
    return c;
}

cudaError_t launch_head_score(const HeadScoreParams & p, const ScoreOut & out, const CUtensorMap & tmw,
                              const CUtensorMap & tmx, cudaStream_t stream) {
    const int64_t n4 = (int64_t) p.n_rows * p.dim / 4;
    const unsigned grid = (unsigned) ((n4 + 255) / 256);
    const int cg = p.n_rows <= 128 ? 1 : 2;
    cudaError_t e;
    if (p.dtype == 30) {
        head_round_kernel<30><<<grid, 256, 0, stream>>>(reinterpret_cast<const float4 *>(p.x),
                                                        reinterpret_cast<uint2 *>(p.xh), n4, p.row_low, p.n_rows);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        e = launch<30>(p, tmw, tmx, cg, stream);
    } else {
        head_round_kernel<1><<<grid, 256, 0, stream>>>(reinterpret_cast<const float4 *>(p.x),
                                                       reinterpret_cast<uint2 *>(p.xh), n4, p.row_low, p.n_rows);
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
        e = launch<1>(p, tmw, tmx, cg, stream);
    }
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    // a warp takes 64 parts in two turns; with more the CTA's barriers are the shorter way
    const bool many = 2 * p.n_groups > 64;
    cfg.gridDim = dim3((unsigned) (many ? p.n_rows : (p.n_rows + kJoinWarps - 1) / kJoinWarps));
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return many ? cudaLaunchKernelEx(&cfg, head_join_block_kernel, p, out, cg)
                : cudaLaunchKernelEx(&cfg, head_join_warp_kernel, p, out, cg);
}

}  // namespace vxk
