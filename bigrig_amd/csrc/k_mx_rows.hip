// Rows into MXFP4 and back.
#include "mx_common.h"
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kThreads = 256;

// 8 consecutive values of a row, from any address their type is aligned to.
template <int DT>
__device__ __forceinline__ void load8(const void* p, float (&v)[8]) {
    if constexpr (DT == BRX_DT_F32) {
        struct __attribute__((packed, aligned(4))) V { u32x4_t a, b; };
        const V q = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, i < 4 ? q.a[i & 3] : q.b[i & 3]);
    } else {
        struct __attribute__((packed, aligned(2))) V { u32x4_t a; };
        const V q = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = DT == BRX_DT_BF16 ? bf2f(q.a[i] & 0xFFFFu) : h2f(q.a[i] & 0xFFFFu);
            v[2 * i + 1] = DT == BRX_DT_BF16 ? bf2f(q.a[i] >> 16) : h2f(q.a[i] >> 16);
        }
    }
}

// One group of 32 per four neighbouring lanes. Bound by HBM for large matrices.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_mx_quantize(MxRows m) {
    constexpr int ES = DT == BRX_DT_F32 ? 4 : 2;
    const int64_t g = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 2;
    const int part = threadIdx.x & 3;
    const int G = m.cols / 32;
    if (g >= m.groups) return;      // whole groups of four lanes
    const int64_t row = g / G;
    const int col = (int)(g - row * G);
    const int64_t b = row / m.rows, r = row - b * m.rows;
    const uint8_t* src = (const uint8_t*)m.x + (b * m.x_batch + r * m.x_row + (int64_t)col * 32 + part * 8) * ES;
    float v[8];
    load8<DT>(src, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, mx_mag(v[i]));
    top = max(top, dpp_u<0xB1>(top));
    top = max(top, dpp_u<0x4E>(top));
    const uint32_t sb = mx_scale(top);
    const int64_t rg = r * G + col;
    struct __attribute__((packed, aligned(1))) W { uint32_t w; };
    reinterpret_cast<W*>(m.codes + b * m.codes_batch + rg * 16 + part * 4)->w = mx_codes(v, sb);
    if (part == 0) m.scales[b * m.scales_batch + rg] = (uint8_t)sb;
}

// 8 values a thread, written as one contiguous [batch, rows, cols] tensor.
template <int DT>
__global__ __launch_bounds__(kThreads) void k_mx_dequantize(MxRows m) {
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;     // 8-code chunk
    if (c >= m.groups * 4) return;
    const int64_t per = (int64_t)m.rows * (m.cols / 8);
    const int64_t b = c / per, rc = c - b * per;
    struct __attribute__((packed, aligned(1))) W { uint32_t w; };
    const uint32_t q = reinterpret_cast<const W*>(m.codes + b * m.codes_batch + rc * 4)->w;
    const float s = e8m0_f32(m.scales[b * m.scales_batch + (rc >> 2)]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e2m1_f32((q >> (4 * i)) & 15u) * s;
    if constexpr (DT == BRX_DT_F32) {
        float* o = (float*)m.x + c * 8;
        struct __attribute__((packed, aligned(4))) V { f32x4_t a, b; };
        *reinterpret_cast<V*>(o) = V{f32x4_t{v[0], v[1], v[2], v[3]}, f32x4_t{v[4], v[5], v[6], v[7]}};
    } else {
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == BRX_DT_BF16) {
                o[i] = pk_bf16(v[2 * i], v[2 * i + 1]);
            } else {
                typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                o[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * i], (_Float16)v[2 * i + 1]});
            }
        }
        struct __attribute__((packed, aligned(2))) V { u32x4_t a; };
        reinterpret_cast<V*>((uint16_t*)m.x + c * 8)->a = o;
    }
}

}  // namespace

hipError_t launch_mx_quantize(const MxRows& m, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)((m.groups * 4 + kThreads - 1) / kThreads));
    if (dtype == BRX_DT_F32) hipLaunchKernelGGL(k_mx_quantize<BRX_DT_F32>, grid, dim3(kThreads), 0, s, m);
    else if (dtype == BRX_DT_BF16) hipLaunchKernelGGL(k_mx_quantize<BRX_DT_BF16>, grid, dim3(kThreads), 0, s, m);
    else hipLaunchKernelGGL(k_mx_quantize<BRX_DT_F16>, grid, dim3(kThreads), 0, s, m);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const MxRows& m, int dtype, hipStream_t s) {
    const dim3 grid((unsigned)((m.groups * 4 + kThreads - 1) / kThreads));
    if (dtype == BRX_DT_F32) hipLaunchKernelGGL(k_mx_dequantize<BRX_DT_F32>, grid, dim3(kThreads), 0, s, m);
    else if (dtype == BRX_DT_BF16) hipLaunchKernelGGL(k_mx_dequantize<BRX_DT_BF16>, grid, dim3(kThreads), 0, s, m);
    else hipLaunchKernelGGL(k_mx_dequantize<BRX_DT_F16>, grid, dim3(kThreads), 0, s, m);
    return hipGetLastError();
}

}  // namespace brx
