// Attention within packed sequences (vxk_prompt_attention) on the tensor cores:
//   out_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c (s_ij - m_i)),  s_ij = q_i . k_j,
// c = scale log2 e, over the rows j of i's sequence that i attends, in one pass over the
// keys with the running maximum m_i.
//
// A tile is 128 query rows: 128 / pack tokens of `pack` heads that share a kv head (pack:
// the largest power of two in n_q / n_kv), so that a key tile serves a group's heads and
// a causal tile spans few tokens.  An item is two tiles, A and B, of consecutive tokens
// of one sequence; the plan deals the items to the CTAs, longest first.
//
// One persistent CTA per SM, 12 warps:
//   warps 0-3   warp 0 TMA producer (K0, Q, V0, K1, V1, ... through a ring of 128-row
//               tiles), warp 1 tcgen05.mma issuer, warps 2-3 see to V rows that a mask hides
//   warps 4-7   softmax of tile A, one thread a row; warps 8-11 of tile B
// TMEM: S_A, S_B (128 columns each; P overwrites the first half of its S), O_A, O_B.
// The issuer's order is  P_A V, S_A of the next keys, P_B V, S_B of the next keys: while
// one tile's softmax runs, the tensor cores work for the other.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 (p is then at most
// 2^8, or 2^15 in f16, whose small p are lifted out of its subnormals): a few times a row
// instead of once a tile.  Sums are fp32 over the unrounded p; p is rounded to the 16-bit type for its
// product, which is the error that the format allows (2^-12 f16, 2^-9 bf16 on average).
//
// Bound by the waits from one step of a tile to the next: a 128 x 128 tile of head dim 128 is
// 1024 clocks of matrix instructions (512 for either product) and 1024 of ex2 (16 a clock and
// SM), and at 8192 rows both pipes are busy a little over half the time, the issue slots a third.
// Measured in short runs (in brackets: back to back, under the power cap), 32 / 8 heads of
// 128: 8192 rows causal f16 484 us, 1.14 PFLOP/s (550; the exponentials alone are 245 us, the
// products 330); sixteen ragged prompts of 9,935 rows, bf16, 138 us, 0.82 (153); 64 x 38 rows
// 24.6 us, where filling and emptying the pipeline is all; four times 1500 rows of 20 heads
// of 64, not causal, 94 us (exponentials 41).  A CTA's first scores of an item wait for
// its Q, and an item's end (the last product, the division, 64 KB of output) is 3500 clocks,
// about 2.5 us of 15 an item in the ragged case.
//
// Tried and slower: a share of the exponentials as polynomials (head dim 128 490 -> 520 us;
// 64: 3 % faster), softmax over 64 keys at a time, P in columns of its own (102 -> 104 us at
// head dim 64), the next item's first scores before this one's end (478 -> 497), four
// stages of K and V instead of five (+1 to 4 %), output turned within four lanes to
// whole lines (8192 rows 550 -> 541 us under the power cap, but 64 x 38 rows 22.6 -> 24.5).
//
// Rows that a mask hides must not reach a result, and 0 * NaN would: in key tiles where
// some row is masked, the rows of V behind the sequence are cleared, and other values
// that are not finite are cleared and marked; the epilogue then adds them to the rows that
// do attend them (a slow path that finite inputs never take).
#include "vxk_internal.h"
#include "vxk_tc.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace vxk {
namespace {

constexpr int kThreads = 384;
// Registers a thread after the split: 128 x 72 + 256 x 216 = 384 x 168, the launch's.
constexpr int kRegsIssue = 72, kRegsSoftmax = 216;
constexpr int kTile = 128;        // query rows and keys of a tile
constexpr int kFlags = 16;        // a tile's items whose V flags are kept
constexpr float kSlack = 8.0f;    // growth of c m that is let pass without a rescale
// p is made 2^kLift times as large, in the sums too: f16 then holds it to 2^-11 of itself down to
// 2^-21 of the largest and to 2^-32 of that below, and 2^(kSlack + kLift) is still inside its
// range.  Unlifted, thousands of keys at 2^-25 of the largest would come to nothing.
template <int DT>
constexpr float kLift = DT == 30 ? 0.0f : 7.0f;

template <int HD>
struct Shape {
    static constexpr int kTileBytes = kTile * HD * 2;
    static constexpr int kStages = HD == 128 ? 5 : 10;
    static constexpr int kOffRing = 2 * kTileBytes;  // after Q_A, Q_B
    static constexpr int kOffBar = kOffRing + kStages * kTileBytes;
    // barriers
    static constexpr int kFull = 0, kEmpty = kStages, kReady = 2 * kStages, kQFull = 3 * kStages, kQEmpty = kQFull + 2,
                         kSFull = kQEmpty + 2, kPFull = kSFull + 2, kODone = kPFull + 4, kDrain = kODone + 2;
    static constexpr int kBars = kDrain + 1;
    static constexpr int kOffMisc = kOffBar + 8 * kBars;  // TMEM base, abort flag, V flags
    static constexpr int kSmem = kOffMisc + 8 + 4 * kFlags * 4 + 1024;
};
// The V warps may write the flags of an item of tile s while its softmax warps have yet to read
// those of an earlier one.  Counted in items that have a tile s, the writers are never more than
// kStages / 2 + 1 ahead: the issuer passes such an item only with P, which those warps make
// behind the epilogue of the one before, and the ring lets the V warps kStages tiles, two an item at
// least, past the issuer.  (Counted in all items there would be no limit: those without a tile B do
// not wait for its warps.)
static_assert(Shape<128>::kStages / 2 + 1 < kFlags && Shape<64>::kStages / 2 + 1 < kFlags, "V flags overtake their readers");
static_assert(Shape<128>::kSmem <= 232448 && Shape<64>::kSmem <= 232448, "attention exceeds 227 KB of shared memory");

// What every role derives from an item.
struct Item {
    int row0, len;        // the sequence's first row and its rows
    int t0;               // first token of tile A
    int head;             // first query head
    int lo;               // first key tile
    int n[2];             // key tiles of A and B (0: no rows)
    __device__ __forceinline__ void set(const int4 & w, const PromptAttnParams & p) {
        row0 = w.x;
        len = w.y;
        t0 = w.z;
        head = w.w;
        lo = p.window > 0 ? max(0, t0 - p.window + 1) / kTile : 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int first = t0 + s * p.tokens;
            const int last = min(first + p.tokens, len) - 1;
            n[s] = first >= len ? 0 : (p.causal ? last / kTile : (len - 1) / kTile) + 1 - lo;
        }
    }
    __device__ __forceinline__ int tiles() const { return max(n[0], n[1]); }
    // Whether some row of the item does not attend some key of tile lo + j.
    __device__ __forceinline__ bool masked(int j, const PromptAttnParams & p) const {
        const int k0 = (lo + j) * kTile;
        if (k0 + kTile > (p.causal ? t0 + 1 : len)) return true;
        return p.window > 0 && min(t0 + 2 * p.tokens, len) - p.window > k0;
    }
};

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t r, float & a, float & b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
template <int DT>
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
    uint32_t r;
    if constexpr (DT == 30) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int DT>
__device__ __forceinline__ float from16(uint16_t v) {
    if constexpr (DT == 30) return __uint_as_float((uint32_t) v << 16);
    else return __half2float(__ushort_as_half(v));
}
// Exponent bits of a 16-bit value all ones: an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool not_finite(uint16_t v) {
    constexpr uint16_t e = DT == 30 ? 0x7f80 : 0x7c00;
    return (v & e) == e;
}

// Of two such values: all ones in each finite one's half.
template <int DT>
__device__ __forceinline__ uint32_t finite_mask(uint32_t w) {
    constexpr uint32_t e = DT == 30 ? 0x7f807f80u : 0x7c007c00u;
    return __vcmpne2(w & e, e);
}

// Shared-memory descriptors (vxk_tc.h) in halves: the upper one is the same for every
// operand here (1024 bytes from one group of eight rows to the next, 128-byte swizzle), the
// lower one holds the address and, for V, the 16 KB from one 64 dims to the next.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | ((lbo >> 4) << 16); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHi)
        : "memory");
}

// A in TMEM.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHi)
        : "memory");
}

// TMA box {64 dims, heads, tokens} at (dim, head, row).
__device__ __forceinline__ void tma_load_3d(void * dst, const CUtensorMap * map, int c0, int c1, int c2, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t taddr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// 32 bytes to a 32-byte aligned address.
__device__ __forceinline__ void store_32(void * to, const uint32_t * v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// p = 2^(c x + off) of 32 scores (off: kLift - c m), added to the sums and stored as 16 bits in TMEM.
template <int DT>
__device__ __forceinline__ void exp_chunk(const float * x, uint32_t tp, uint64_t c2, uint64_t off2, uint64_t (&total)[2]) {
    uint32_t h[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
        float a, b;
        unpair(fma2(pair(x[e], x[e + 1]), c2, off2), a, b);
        a = ex2f(a);
        b = ex2f(b);
        total[e / 2 % 2] = add2(total[e / 2 % 2], pair(a, b));
        h[e / 2] = cvt2<DT>(a, b);
    }
    tmem_store16(tp, h);
}

// O times f, a row's columns of TMEM at `to`.
template <int HD>
__device__ __forceinline__ void scale_o(uint32_t to, float f) {
#pragma unroll
    for (int k = 0; k < HD; k += 16) {
        uint32_t o[16];
        tmem_load16(to + k, o);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
        tmem_store16(to + k, o);
    }
}

// One thread's running state over the keys of its row.
struct RowState {
    float m;             // what p is taken from, in score units
    float sum;
};

// 128 scores of a row: the running maximum, p into TMEM at tp, the sum.  hi, lo: the columns
// [lo, hi) that the row attends (MASKED).  Where some row's maximum has outgrown kSlack,
// grown() multiplies O by its argument first.  half_done(k): a half of p is stored.
template <int DT, bool MASKED, typename F, typename G>
__device__ __forceinline__ void tile_step(float (&x)[128], uint32_t tp, float c, int hi, int lo, RowState & r, F && grown,
                                          G && half_done) {
    bool none[4] = {false, false, false, false};
    if constexpr (MASKED) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool whole = __all_sync(0xffffffffu, hi >= 32 * k + 32 && lo <= 32 * k);
            none[k] = __all_sync(0xffffffffu, hi <= 32 * k || lo >= 32 * k + 32);
            if (!whole && !none[k]) {
#pragma unroll
                for (int e = 32 * k; e < 32 * k + 32; ++e)
                    if (e >= hi || e < lo) x[e] = -INFINITY;
            }
        }
    }
    float mt[4] = {r.m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (MASKED && none[k]) continue;
#pragma unroll
        for (int e = 32 * k; e < 32 * k + 32; e += 2) mt[e / 2 % 4] = max3(mt[e / 2 % 4], x[e], x[e + 1]);
    }
    const float mn = fmaxf(max3(mt[0], mt[1], mt[2]), mt[3]);
    const bool grow = r.m != -INFINITY && (mn - r.m) * c > kSlack;
    if (__any_sync(0xffffffffu, grow)) {
        const float f = grow ? ex2f((r.m - mn) * c) : 1.0f;
        r.sum *= f;
        if (grow) r.m = mn;
        grown(f);
    }
    if (r.m == -INFINITY) r.m = mn;                  // nothing in O or the sum yet
    const float off = r.m == -INFINITY ? 0.0f : fmaf(-r.m, c, kLift<DT>);
    const uint64_t c2 = pair(c, c), off2 = pair(off, off);
    uint64_t total[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (MASKED && none[k]) {
            const uint32_t zero[16] = {};
            tmem_store16(tp + 16 * k, zero);
        } else {
            exp_chunk<DT>(x + 32 * k, tp + 16 * k, c2, off2, total);
        }
        if (k & 1) half_done(k >> 1);
    }
    float a, b;
    unpair(add2(total[0], total[1]), a, b);
    r.sum += a + b;
}

template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 1) prompt_attention_kernel(const __grid_constant__ CUtensorMap tmq,
                                                                       const __grid_constant__ CUtensorMap tmk,
                                                                       const __grid_constant__ CUtensorMap tmv,
                                                                       const PromptAttnParams p) {
    using S = Shape<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t * ring = base + S::kOffRing;
    uint64_t * bars = reinterpret_cast<uint64_t *>(base + S::kOffBar);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(base + S::kOffMisc);
    volatile int32_t * abort_flag = reinterpret_cast<volatile int32_t *>(base + S::kOffMisc + 4);
    volatile int32_t * v_flags = reinterpret_cast<volatile int32_t *>(base + S::kOffMisc + 8);  // [2 tiles][2 warps][kFlags]

    const int tid = threadIdx.x, warp = (int) uniform(tid >> 5), lane = tid & 31;
    const int4 head = *reinterpret_cast<const int4 *>(p.plan);
    if (head.y > p.rows) {  // a replay under a plan larger than the buffers
        if (tid == 0 && blockIdx.x == 0) atomicCAS(p.error, 0, kErrPlan);
        return;
    }
    const int32_t * offsets = reinterpret_cast<const int32_t *>(p.plan + p.off_offsets);
    const int begin = offsets[blockIdx.x], end = offsets[blockIdx.x + 1];
    if (begin == end) return;
    const int4 * items = reinterpret_cast<const int4 *>(p.plan + p.off_items);

    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&bars[S::kFull + s], 1);
            mbar_init(&bars[S::kEmpty + s], 1);
            mbar_init(&bars[S::kReady + s], 2);  // both V warps
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bars[S::kQFull + s], 1);
            mbar_init(&bars[S::kQEmpty + s], 1);
            mbar_init(&bars[S::kSFull + s], 1);
            mbar_init(&bars[S::kPFull + 2 * s], 4);  // keys 0-63
            mbar_init(&bars[S::kPFull + 2 * s + 1], 4);
            mbar_init(&bars[S::kODone + s], 1);
        }
        mbar_init(&bars[S::kDrain], 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc<1>(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_slot);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        if (warp == 0 && lane == 0) {
            // ---------------- TMA producer ----------------
            uint32_t c = 0, cq[2] = {0, 0};
            bool ok = true;
            auto load_kv = [&](const CUtensorMap * map, int kv_head, int row) {
                const uint32_t st = c % S::kStages;
                if (!tc_wait(&bars[S::kEmpty + st], ((c / S::kStages) & 1) ^ 1, abort_flag, p.error)) return false;
                mbar_expect_tx(&bars[S::kFull + st], S::kTileBytes);
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                    tma_load_3d(ring + st * S::kTileBytes + h * (kTile * 128), map, 64 * h, kv_head, row, &bars[S::kFull + st]);
                ++c;
                return true;
            };
            for (int i = begin; ok && i < end; ++i) {
                Item it;
                it.set(items[i], p);
                const int kv_head = it.head / p.group, n = it.tiles();
                for (int j = 0; ok && j < n; ++j) {
                    const int row = it.row0 + (it.lo + j) * kTile;
                    if (!(ok = load_kv(&tmk, kv_head, row))) break;
                    for (int s = 0; ok && j == 0 && s < 2; ++s) {
                        if (it.n[s] == 0) continue;
                        if (!(ok = tc_wait(&bars[S::kQEmpty + s], (cq[s] & 1) ^ 1, abort_flag, p.error))) break;
                        mbar_expect_tx(&bars[S::kQFull + s], S::kTileBytes);
#pragma unroll
                        for (int h = 0; h < HD / 64; ++h)
                            tma_load_3d(base + s * S::kTileBytes + h * (kTile * 128), &tmq, 64 * h, it.head,
                                        it.row0 + it.t0 + s * p.tokens, &bars[S::kQFull + s]);
                        ++cq[s];
                    }
                    if (ok) ok = load_kv(&tmv, kv_head, row);
                }
            }
            // copies in flight land before the CTA leaves
            for (uint32_t d = c > (uint32_t) S::kStages ? c - S::kStages : 0; d < c; ++d)
                tc_drain(&bars[S::kFull + d % S::kStages], (d / S::kStages) & 1);
            for (int s = 0; s < 2; ++s)
                if (cq[s]) tc_drain(&bars[S::kQFull + s], (cq[s] - 1) & 1);
        } else if (warp == 1) {
            // ---------------- tcgen05.mma issuer ----------------
            constexpr uint32_t fmt = DT == 30 ? 1u : 0u;
            constexpr uint32_t idesc_s = tc_idesc(fmt, kTile, kTile), idesc_o = tc_idesc(fmt, kTile, HD, 1);
            // a place in the ring and its parity; a parity bit for every other barrier waited on
            uint32_t st = 0, par = 0;
            constexpr uint32_t kBitQ = 1, kBitP = 4;
            uint32_t bits = 0;
            bool ok = true;
            auto wait_bit = [&](int bar, uint32_t bit) {
                const bool have = tc_wait(&bars[bar], (bits & bit) != 0, abort_flag, p.error);
                tc_fence_after();
                bits ^= bit;
                return (bool) uniform(have);
            };
            auto wait_tile = [&](uint32_t at, uint32_t parity) {
                const bool have = tc_wait(&bars[S::kReady + at], parity, abort_flag, p.error);
                tc_fence_after();
                return (bool) uniform(have);
            };
            const uint32_t sm_q = desc_lo(smem_u32(base), 16), sm_k = desc_lo(smem_u32(ring), 16),
                           sm_v = desc_lo(smem_u32(ring), kTile * 128);
            constexpr uint32_t kTileDesc = S::kTileBytes >> 4;
            // S of a tile from the keys in place `at`; then what the scores were the last to use
            auto scores = [&](int s, uint32_t at, bool last) {
                const uint32_t dq = sm_q + s * kTileDesc, dk = sm_k + at * kTileDesc;
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) {  // 64 dims are 16 KB of the tile
                        const uint32_t step = (uint32_t) ((ks / 4) * (kTile * 128) + (ks % 4) * 32) >> 4;
                        mma_ss(tmem + s * kTile, dq + step, dk + step, idesc_s, ks != 0);
                    }
                    tc_commit<1>(&bars[S::kSFull + s]);
                    if (last) tc_commit<1>(&bars[S::kQEmpty + s]);
                }
                __syncwarp();
            };
            auto release = [&](uint32_t at) {
                if (elect_one()) tc_commit<1>(&bars[S::kEmpty + at]);
                __syncwarp();
            };
            for (int i = begin; ok && i < end; ++i) {
                Item it;
                it.set(items[i], p);
                const int n0 = (int) uniform(it.n[0]), n1 = (int) uniform(it.n[1]), n = max(n0, n1);
                ok = wait_tile(st, par);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const int ns = s ? n1 : n0;
                    if (!ok || ns == 0) continue;
                    ok = wait_bit(S::kQFull + s, kBitQ << s);
                    if (ok) scores(s, st, ns == 1);
                }
                if (!ok) break;
                release(st);
                for (int j = 0; ok && j < n; ++j) {
                    if (++st == S::kStages) st = 0, par ^= 1;       // V of these keys
                    uint32_t st_k = st + 1, par_k = par;            // K of the next
                    if (st_k == S::kStages) st_k = 0, par_k ^= 1;
                    const uint32_t dv = sm_v + st * kTileDesc;
                    bool have_v = false, have_k = false;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int ns = s ? n1 : n0;
                        if (ok && j < ns) {
                            const uint32_t d = tmem + 2 * kTile + s * HD, a = tmem + s * kTile;
                            ok = wait_bit(S::kPFull + 2 * s, kBitP << s);
                            if (ok && !have_v) ok = wait_tile(st, par);
                            have_v = true;
                            if (!ok) break;
                            if (elect_one()) {
#pragma unroll
                                for (int ks = 0; ks < kTile / 32; ++ks)  // 16 keys: 8 columns of P, 2 KB of V
                                    mma_ts(d, a + 8 * ks, dv + 128 * ks, idesc_o, (j | ks) != 0);
                                }
                            __syncwarp();
                            bits ^= kBitP << s;  // the second half's barrier has the first's parity
                            ok = wait_bit(S::kPFull + 2 * s + 1, kBitP << s);
                            if (!ok) break;
                            if (elect_one()) {
#pragma unroll
                                for (int ks = kTile / 32; ks < kTile / 16; ++ks)
                                    mma_ts(d, a + 8 * ks, dv + 128 * ks, idesc_o, 1);
                                tc_commit<1>(&bars[S::kODone + s]);
                            }
                            __syncwarp();
                        }
                        if (ok && j + 1 < ns) {
                            if (!have_k) ok = wait_tile(st_k, par_k);
                            have_k = true;
                            if (!ok) break;
                            scores(s, st_k, j + 2 == ns);
                        }
                    }
                    if (!ok) break;
                    release(st);
                    if (j + 1 < n) release(st_k);
                    st = st_k, par = par_k;
                }
            }
            if (elect_one()) {
                tc_commit<1>(&bars[S::kDrain]);
                tc_drain(&bars[S::kDrain], 0);
            }
            __syncwarp();
        } else if (warp >= 2) {
            // ---------------- V rows under a mask ----------------
            // These warps see every tile in turn, masked or not, and pass it on to the issuer:
            // a wait by parity holds only for a reader that is never a turn of the ring away.
            const int t = (warp - 2) * 32 + lane;
            uint32_t st = 0, par = 0;
            int nth[2] = {0, 0};  // items of either tile so far
            bool ok = true;
            for (int i = begin; ok && i < end; ++i) {
                Item it;
                it.set(items[i], p);
                const int n = it.tiles();
                bool bad = false;
                for (int j = 0; ok && j < 2 * n; ++j) {  // K, V, K, V, ...
                    ok = __all_sync(0xffffffffu, tc_wait(&bars[S::kFull + st], par, abort_flag, p.error));
                    if (!ok) break;
                    if ((j & 1) && it.masked(j >> 1, p)) {
                        // 16-byte chunk q of the tile holds eight dims of row (q / 8) % 128
                        uint4 * v = reinterpret_cast<uint4 *>(ring + st * S::kTileBytes);
                        const int rows = it.len - (it.lo + (j >> 1)) * kTile;
                        for (int q = t; q < S::kTileBytes / 16; q += 64) {
                            if (q / 8 % kTile >= rows) {
                                v[q] = make_uint4(0, 0, 0, 0);
                                continue;
                            }
                            uint4 x = v[q];
                            const uint4 f = make_uint4(finite_mask<DT>(x.x), finite_mask<DT>(x.y), finite_mask<DT>(x.z),
                                                       finite_mask<DT>(x.w));
                            if ((f.x & f.y & f.z & f.w) != 0xffffffffu) {
                                bad = true;
                                v[q] = make_uint4(x.x & f.x, x.y & f.y, x.z & f.z, x.w & f.w);
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        bad = __any_sync(0xffffffffu, bad);
                        if (lane == 0) {
#pragma unroll
                            for (int s = 0; s < 2; ++s)
                                if (it.n[s]) v_flags[(2 * s + warp - 2) * kFlags + nth[s] % kFlags] = bad;
                        }
                    }
                    if (lane == 0) mbar_arrive(&bars[S::kReady + st]);
                    if (++st == S::kStages) st = 0, par ^= 1;
                }
                nth[0] += it.n[0] != 0;
                nth[1] += it.n[1] != 0;
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ---------------- softmax ----------------
        const int s = (warp - 4) >> 2;
        const int q = warp & 3, r = q * 32 + lane;          // TMEM lane = row of the tile
        const uint32_t lanes = (uint32_t) (32 * q) << 16;
        const uint32_t ts = tmem + s * kTile + lanes, to = tmem + 2 * kTile + s * HD + lanes;
        const float c = p.scale_log2;
        uint32_t cs = 0;                                     // key tiles so far
        int nth = 0;                                         // items of this tile so far
        bool ok = true;
        for (int i = begin; ok && i < end; ++i) {
            Item it;
            it.set(items[i], p);
            const int n = s ? it.n[1] : it.n[0];
            if (n == 0) continue;
            const int first = it.t0 + s * p.tokens;
            const int token = first + (r >> p.pack_shift);
            const int last = min(first + p.tokens, it.len) - 1;
            RowState row = {-INFINITY, 0.0f};
            for (int j = 0; j < n; ++j, ++cs) {
                ok = __all_sync(0xffffffffu, tc_wait(&bars[S::kSFull + s], cs & 1, abort_flag, p.error));
                if (!ok) break;
                tc_fence_after();
                float x[128];
#pragma unroll
                for (int k = 0; k < 128; k += 32) tmem_load32(ts + k, reinterpret_cast<uint32_t *>(x) + k);
                const int k0 = (it.lo + j) * kTile;
                const bool masked =
                    k0 + kTile > (p.causal ? min(first + 1, it.len) : it.len) || (p.window > 0 && last - p.window >= k0);
                const int hi = (p.causal ? min(token + 1, it.len) : it.len) - k0;
                const int lo = p.window > 0 ? token - p.window + 1 - k0 : 0;
                tmem_wait_ld();
                auto grown = [&](float f) {  // O is complete up to the last tile when S is there
                    if (j > 0) scale_o<HD>(to, f);
                };
                auto half_done = [&](int half) {
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bars[S::kPFull + 2 * s + half]);
                };
                if (masked) tile_step<DT, true>(x, ts, c, hi, lo, row, grown, half_done);
                else tile_step<DT, false>(x, ts, c, 0, 0, row, grown, half_done);
            }
            if (!ok) break;
            // epilogue: O / sum
            ok = __all_sync(0xffffffffu, tc_wait(&bars[S::kODone + s], (cs - 1) & 1, abort_flag, p.error));
            if (!ok) break;
            tc_fence_after();
            const bool bad = v_flags[2 * s * kFlags + nth % kFlags] | v_flags[(2 * s + 1) * kFlags + nth % kFlags];
            ++nth;
            const int head = it.head + (r & ((1 << p.pack_shift) - 1));
            const float f = 1.0f / row.sum;
            uint16_t * out = static_cast<uint16_t *>(p.out) + ((int64_t) (it.row0 + token) * p.n_q + head) * HD;
#pragma unroll
            for (int k = 0; k < HD; k += 32) {
                uint32_t o[32];
                tmem_load32(to + k, o);
                tmem_wait_ld();
                if (token < it.len) {
                    float y[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) y[e] = __uint_as_float(o[e]) * f;
                    if (bad) {
                        for (int t = 0; t < it.tiles(); ++t) {
                            if (!it.masked(t, p)) continue;
                            const int k0 = (it.lo + t) * kTile;
                            const int from = max(k0, p.window > 0 ? token - p.window + 1 : 0);
                            const int upto = min(k0 + kTile, p.causal ? token + 1 : it.len);
                            for (int key = from; key < upto; ++key) {
                                const uint16_t * v = static_cast<const uint16_t *>(p.v) +
                                                     ((int64_t) (it.row0 + key) * p.n_kv + it.head / p.group) * HD + k;
#pragma unroll
                                for (int e = 0; e < 32; ++e) {
                                    const uint16_t w = v[e];
                                    if (not_finite<DT>(w)) y[e] += from16<DT>(w);
                                }
                            }
                        }
                    }
                    uint32_t h[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) h[e] = cvt2<DT>(y[2 * e], y[2 * e + 1]);
                    if (p.out_32) {  // whole sectors: half the requests
                        store_32(out + k, h);
                        store_32(out + k + 16, h + 8);
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            *reinterpret_cast<uint4 *>(out + k + 2 * e) = make_uint4(h[e], h[e + 1], h[e + 2], h[e + 3]);
                    }
                }
            }
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_free<1>(tmem, 512);
    }
}

template <int DT, int HD>
cudaError_t launch(const PromptAttnParams & p, const CUtensorMap & tmq, const CUtensorMap & tmk, const CUtensorMap & tmv,
                   int ctas, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(prompt_attention_kernel<DT, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Shape<HD>::kSmem);
    if (e != cudaSuccess) return e;
    prompt_attention_kernel<DT, HD><<<(unsigned) ctas, kThreads, Shape<HD>::kSmem, stream>>>(tmq, tmk, tmv, p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_prompt_attention(const PromptAttnParams & p, const CUtensorMap & tmq, const CUtensorMap & tmk,
                                    const CUtensorMap & tmv, int ctas, cudaStream_t stream) {
    if (p.head_dim == 64)
        return p.dtype == 30 ? launch<30, 64>(p, tmq, tmk, tmv, ctas, stream) : launch<1, 64>(p, tmq, tmk, tmv, ctas, stream);
    return p.dtype == 30 ? launch<30, 128>(p, tmq, tmk, tmv, ctas, stream) : launch<1, 128>(p, tmq, tmk, tmv, ctas, stream);
}

}  // namespace vxk
