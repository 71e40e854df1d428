// Packed prompts (vxk_prompt_*): the rotary rows and the attention within each
// sequence.
#include "vxk_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace vxk {
namespace {

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (DT == 30) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (DT == 30) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
}

// ---- rotary rows ------------------------------------------------------------

// (cos, sin) of position * theta^(-2i / head_dim), in 64 bits: at position 10^5 a
// 32-bit angle is off by 4e-3 of a radian, more than a 16-bit value resolves.
__global__ void rope_table_kernel(float2 * table, int64_t n, int32_t half, double log_theta) {
    const int64_t at = (int64_t) blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= n) return;
    const int64_t pos = at / half;
    const int i = (int) (at - pos * half);
    double s, c;
    sincos((double) pos * exp(-log_theta * i / half), &s, &c);
    table[at] = make_float2((float) c, (float) s);
}

// One CTA a row; a thread turns 8 values (two 16-byte loads, one store) at a time.
// 256 threads x 8 values are a whole number of heads, so a thread's four pairs are
// the same in every head and their (cos, sin) are loaded once.  Bound by HBM: 4
// bytes read and 2 written per value, and head_dim * 4 bytes of table a row.
template <int DT>
__global__ void __launch_bounds__(256) rope_kernel(const PromptRopeParams p) {
    const int4 head = *reinterpret_cast<const int4 *>(p.plan);
    if (head.y > p.rows) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.error, 0, kErrPlan);
        return;
    }
    const int64_t row = blockIdx.x;
    if (row >= head.y) return;
    const int per_head = p.head_dim / 8;
    const int nq = p.n_q * per_head, nkv = p.n_kv * per_head;
    const int pos = p.positions[row];
    const float4 * turn = reinterpret_cast<const float4 *>(p.table + (int64_t) pos * (p.head_dim / 2)) +
                          (threadIdx.x % per_head) * 2;
    const float4 t0 = __ldg(turn), t1 = __ldg(turn + 1);
    for (int c = threadIdx.x; c < nq + 2 * nkv; c += 256) {
        const float * src;
        uint16_t * dst;
        if (c < nq) {
            src = p.q + (row * nq + c) * 8;
            dst = p.q16 + (row * nq + c) * 8;
        } else if (c < nq + nkv) {
            src = p.k + (row * nkv + c - nq) * 8;
            dst = p.k16 + (row * nkv + c - nq) * 8;
        } else {
            src = p.v + (row * nkv + c - nq - nkv) * 8;
            dst = p.v16 + (row * nkv + c - nq - nkv) * 8;
        }
        float4 a = __ldcs(reinterpret_cast<const float4 *>(src));
        float4 b = __ldcs(reinterpret_cast<const float4 *>(src) + 1);
        if (c < nq + nkv) {
            a = make_float4(a.x * t0.x - a.y * t0.y, a.x * t0.y + a.y * t0.x, a.z * t0.z - a.w * t0.w,
                            a.z * t0.w + a.w * t0.z);
            b = make_float4(b.x * t1.x - b.y * t1.y, b.x * t1.y + b.y * t1.x, b.z * t1.z - b.w * t1.w,
                            b.z * t1.w + b.w * t1.z);
        }
        *reinterpret_cast<uint4 *>(dst) =
            make_uint4(pack2<DT>(a.x, a.y), pack2<DT>(a.z, a.w), pack2<DT>(b.x, b.y), pack2<DT>(b.z, b.w));
    }
}

// ---- attention --------------------------------------------------------------

// One warp per query row and head, one key at a time: the plain form of
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q . k_j,
// with the running maximum m and sums rescaled when it grows.
template <int DT, int HD>
__global__ void __launch_bounds__(128) attention_kernel(const PromptAttnParams p) {
    const int4 head = *reinterpret_cast<const int4 *>(p.plan);
    if (head.y > p.rows) {
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.error, 0, kErrPlan);
        return;
    }
    constexpr int W = HD / 64;  // 32-bit words a lane holds
    const int64_t unit = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int64_t row = unit / p.n_q;
    const int h = (int) (unit - row * p.n_q);
    if (row >= head.y) return;
    const int4 seq = p.row_seq[row];  // first row, rows
    const int i = (int) row - seq.x;
    const int j0 = p.window > 0 ? max(0, i - p.window + 1) : 0;
    const int j1 = p.causal ? i + 1 : seq.y;
    const int hk = h / (p.n_q / p.n_kv);
    float q[2 * W], acc[2 * W];
    const uint32_t * qp = reinterpret_cast<const uint32_t *>(p.q) + (row * p.n_q + h) * (HD / 2) + lane * W;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const float2 f = unpack2<DT>(qp[w]);
        q[2 * w] = f.x * p.scale_log2;
        q[2 * w + 1] = f.y * p.scale_log2;
        acc[2 * w] = acc[2 * w + 1] = 0.0f;
    }
    float m = -INFINITY, s = 0.0f;
    for (int j = j0; j < j1; ++j) {
        const int64_t at = ((int64_t) (seq.x + j) * p.n_kv + hk) * (HD / 2) + lane * W;
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 f = unpack2<DT>(reinterpret_cast<const uint32_t *>(p.k)[at + w]);
            d = fmaf(q[2 * w], f.x, fmaf(q[2 * w + 1], f.y, d));
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const float mn = fmaxf(m, d);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float f0 = ex2(m - base), e = ex2(d - base);
        s = s * f0 + e;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 f = unpack2<DT>(reinterpret_cast<const uint32_t *>(p.v)[at + w]);
            acc[2 * w] = fmaf(acc[2 * w], f0, e * f.x);
            acc[2 * w + 1] = fmaf(acc[2 * w + 1], f0, e * f.y);
        }
        m = mn;
    }
    uint32_t * op = reinterpret_cast<uint32_t *>(p.out) + (row * p.n_q + h) * (HD / 2) + lane * W;
#pragma unroll
    for (int w = 0; w < W; ++w) op[w] = pack2<DT>(acc[2 * w] / s, acc[2 * w + 1] / s);
}

}  // namespace

cudaError_t launch_rope_table(float2 * table, int32_t rows, int32_t head_dim, double log_theta, cudaStream_t stream) {
    const int64_t n = (int64_t) rows * (head_dim / 2);
    rope_table_kernel<<<(unsigned) ((n + 255) / 256), 256, 0, stream>>>(table, n, head_dim / 2, log_theta);
    return cudaGetLastError();
}

cudaError_t launch_prompt_rope(const PromptRopeParams & p, cudaStream_t stream) {
    if (p.dtype == 30) {
        rope_kernel<30><<<(unsigned) p.rows, 256, 0, stream>>>(p);
    } else {
        rope_kernel<1><<<(unsigned) p.rows, 256, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

cudaError_t launch_prompt_attention(const PromptAttnParams & p, cudaStream_t stream) {
    const unsigned grid = (unsigned) (((int64_t) p.rows * p.n_q + 3) / 4);
    if (p.head_dim == 64) {
        if (p.dtype == 30) attention_kernel<30, 64><<<grid, 128, 0, stream>>>(p);
        else attention_kernel<1, 64><<<grid, 128, 0, stream>>>(p);
    } else {
        if (p.dtype == 30) attention_kernel<30, 128><<<grid, 128, 0, stream>>>(p);
        else attention_kernel<1, 128><<<grid, 128, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace vxk
