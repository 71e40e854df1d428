// Rotary rows of packed prompts (vxk_prompt_rope).
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
// bytes read and 2 written per value, and head_dim * 4 bytes of table a row.  13,033 rows
// of 32 / 8 heads of 128 to bf16: 77 us, 6.3 TB/s, 96 % of a plain copy's rate; 38 rows:
// 3 us of kernel, 7.5 us a call, the launch.
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
    const int pos = reinterpret_cast<const int32_t *>(p.plan + head.w)[row];
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

// Eight values a thread.
template <int DT>
__global__ void __launch_bounds__(256) widen_kernel(const uint4 * in, float4 * out, int64_t n8) {
    const int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const uint4 u = in[i];
    const float2 a = unpack2<DT>(u.x), b = unpack2<DT>(u.y), c = unpack2<DT>(u.z), d = unpack2<DT>(u.w);
    out[2 * i] = make_float4(a.x, a.y, b.x, b.y);
    out[2 * i + 1] = make_float4(c.x, c.y, d.x, d.y);
}

}  // namespace

cudaError_t launch_widen(const void * in, float * out, int64_t n, int32_t dtype, cudaStream_t stream) {
    const int64_t n8 = n / 8;
    const unsigned grid = (unsigned) ((n8 + 255) / 256);
    if (dtype == 30) {
        widen_kernel<30><<<grid, 256, 0, stream>>>(static_cast<const uint4 *>(in), reinterpret_cast<float4 *>(out), n8);
    } else {
        widen_kernel<1><<<grid, 256, 0, stream>>>(static_cast<const uint4 *>(in), reinterpret_cast<float4 *>(out), n8);
    }
    return cudaGetLastError();
}

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

}  // namespace vxk
