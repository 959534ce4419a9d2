// Rows into MXFP4 and back.
#include "mx_common.h"
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kThreads = 256;

// Values of a run, 16 bytes: what a lane loads at once, so that a wave reads 1 KB in a row (32 bytes a lane,
// fp32's 8 values, cost a 131072 x 2048 matrix 262 instead of 237 us).
template <int DT>
constexpr int kRun = DT == BRX_DT_F32 ? 4 : 8;

// One run, from any address its type is aligned to.
template <int DT>
__device__ __forceinline__ void load_run(const void* p, float (&v)[kRun<DT>]) {
    typedef u32x4_t __attribute__((aligned(2))) V;
    // (read once: past the caches, a 131072 x 2048 fp32 matrix and back 331 -> 309 us)
    const u32x4_t q = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == BRX_DT_F32) {
            const uint32_t x = q[i];               // (a bit cast of the element itself reads the vector's first)
            v[i] = __builtin_bit_cast(float, x);
        } else {
            v[2 * i] = DT == BRX_DT_BF16 ? bf2f(q[i] & 0xFFFFu) : h2f(q[i] & 0xFFFFu);
            v[2 * i + 1] = DT == BRX_DT_BF16 ? bf2f(q[i] >> 16) : h2f(q[i] >> 16);
        }
    }
}

// A thread takes kUnit runs (its neighbours the others of a group), a wave 64 neighbouring runs at a time, all
// loads before the first use. HBM sets the time of a large matrix: 131072 x 2048 fp32 values take 195 us
// to MXFP4 (6.2 TB/s) and 94 us from there to bf16 (7.3 TB/s).
constexpr int kUnit = 2;
constexpr int kBlocksMost = 1 << 22;

// Run i of the matrices, `run` values each: matrix b, row r and run c of it. FLAT: one matrix whose rows
// follow one another, so rows need no division.
template <bool FLAT>
__device__ __forceinline__ void find_run(const MxRows& m, int run, int64_t i, int64_t& b, int64_t& r, int64_t& c) {
    if constexpr (FLAT) {
        b = r = 0;
        c = i;
    } else {
        const int64_t per = m.cols / run;
        int64_t row;
        if (m.groups < (int64_t)1 << 28) {         // (uniform: 32-bit divisions)
            row = (uint32_t)i / (uint32_t)per;
            b = (uint32_t)row / (uint32_t)m.rows;
        } else {
            row = i / per;
            b = row / m.rows;
        }
        c = i - row * per;
        r = row - b * m.rows;
    }
}

template <int DT, bool FLAT>
__global__ __launch_bounds__(kThreads) void k_mx_quantize(MxRows m) {
    constexpr int ES = DT == BRX_DT_F32 ? 4 : 2, R = kRun<DT>, L = 32 / R;      // L lanes a group
    const int64_t runs = m.groups * L;             // (a group's lanes come or go together)
    const int64_t per = (int64_t)m.cols / R;
    for (int64_t i0 = (int64_t)blockIdx.x * (kThreads * kUnit); i0 < runs; i0 += (int64_t)gridDim.x * (kThreads * kUnit)) {
        float v[kUnit][R];
        int64_t at[kUnit], b[kUnit];
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            int64_t i = i0 + u * kThreads + threadIdx.x, r, c;
            i = i < runs ? i : runs - L + (threadIdx.x & (L - 1));
            find_run<FLAT>(m, R, i, b[u], r, c);
            load_run<DT>((const uint8_t*)m.x + (b[u] * m.x_batch + r * m.x_row + c * R) * ES, v[u]);
            at[u] = r * per + c;
        }
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < R; ++i) top = max(top, mx_mag(v[u][i]));
            top = max(top, dpp_u<0xB1>(top));
            top = max(top, dpp_u<0x4E>(top));
            if constexpr (L == 8) top = max(top, dpp_u<0x141>(top));   // (row_half_mirror)
            const uint32_t sb = mx_scale(top);
            if (i0 + u * kThreads + threadIdx.x < runs) {
                uint8_t* const to = m.codes + b[u] * m.codes_batch + at[u] * (R / 2);
                if constexpr (R == 8) {
                    struct __attribute__((packed, aligned(1))) W { uint32_t w; };
                    reinterpret_cast<W*>(to)->w = mx_codes(v[u], sb);
                } else {
                    struct __attribute__((packed, aligned(1))) W { uint16_t w; };
                    reinterpret_cast<W*>(to)->w = (uint16_t)mx_codes(v[u], sb);
                }
                if ((threadIdx.x & (L - 1)) == 0) m.scales[b[u] * m.scales_batch + at[u] / L] = (uint8_t)sb;
            }
        }
    }
}

// 16 bytes to any address their values are aligned to, past the caches (as much again as the loads: the same
// matrix and back 309 -> 281 us, 1999 x 4128 10.6 -> 8.4).
__device__ __forceinline__ void put16(void* p, const u32x4_t& v) {
    typedef u32x4_t __attribute__((aligned(2))) V;
    __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
}

// The values go to one contiguous [batch, rows, cols] tensor. FLAT: one matrix.
template <int DT, bool FLAT>
__global__ __launch_bounds__(kThreads) void k_mx_dequantize(MxRows m) {
    const int64_t runs = m.groups * 4;
    const int64_t per = (int64_t)m.cols / 8;
    for (int64_t i0 = (int64_t)blockIdx.x * (kThreads * kUnit); i0 < runs; i0 += (int64_t)gridDim.x * (kThreads * kUnit)) {
        uint32_t q[kUnit], sb[kUnit];
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            int64_t i = i0 + u * kThreads + threadIdx.x, b, r, c;
            i = i < runs ? i : runs - 1;
            find_run<FLAT>(m, 8, i, b, r, c);
            const int64_t at = r * per + c;
            struct __attribute__((packed, aligned(1))) W { uint32_t w; };
            q[u] = reinterpret_cast<const W*>(m.codes + b * m.codes_batch + at * 4)->w;
            sb[u] = m.scales[b * m.scales_batch + (at >> 2)];
        }
#pragma unroll
        for (int u = 0; u < kUnit; ++u) {
            const int64_t i = i0 + u * kThreads + threadIdx.x;
            if (i >= runs) return;
            const float s = e8m0_f32(sb[u]);
            if constexpr (DT == BRX_DT_BF16) {
                uint32_t o[4];
                dq_fp4(q[u], s, o);
                const uint32_t nan = sb[u] == 255u ? 0x7FC07FC0u : 0u;
                put16((uint16_t*)m.x + i * 8, u32x4_t{o[0] | nan, o[1] | nan, o[2] | nan, o[3] | nan});
            } else {
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = e2m1_f32((q[u] >> (4 * k)) & 15u) * s;
                if constexpr (DT == BRX_DT_F32) {
                    float* const o = (float*)m.x + i * 8;
                    put16(o, __builtin_bit_cast(u32x4_t, f32x4_t{v[0], v[1], v[2], v[3]}));
                    put16(o + 4, __builtin_bit_cast(u32x4_t, f32x4_t{v[4], v[5], v[6], v[7]}));
                } else {
                    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                    u32x4_t o;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        o[k] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)v[2 * k], (_Float16)v[2 * k + 1]});
                    put16((uint16_t*)m.x + i * 8, o);
                }
            }
        }
    }
}

dim3 grid_of(const MxRows& m, int run) {
    const int64_t n = (m.groups * (32 / run) + kThreads * kUnit - 1) / (kThreads * kUnit);
    return dim3((unsigned)(n < kBlocksMost ? n : kBlocksMost));
}

}  // namespace

hipError_t launch_mx_quantize(const MxRows& m, int dtype, hipStream_t s) {
    const bool flat = m.groups == m.rows * (m.cols / 32) && (m.rows == 1 || m.x_row == m.cols);
#define BRX_Q(DT) \
    if (flat) hipLaunchKernelGGL((k_mx_quantize<DT, true>), grid_of(m, kRun<DT>), dim3(kThreads), 0, s, m); \
    else hipLaunchKernelGGL((k_mx_quantize<DT, false>), grid_of(m, kRun<DT>), dim3(kThreads), 0, s, m)
    if (dtype == BRX_DT_F32) { BRX_Q(BRX_DT_F32); }
    else if (dtype == BRX_DT_BF16) { BRX_Q(BRX_DT_BF16); }
    else { BRX_Q(BRX_DT_F16); }
#undef BRX_Q
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const MxRows& m, int dtype, hipStream_t s) {
    const bool flat = m.groups == m.rows * (m.cols / 32);
#define BRX_D(DT) \
    if (flat) hipLaunchKernelGGL((k_mx_dequantize<DT, true>), grid_of(m, 8), dim3(kThreads), 0, s, m); \
    else hipLaunchKernelGGL((k_mx_dequantize<DT, false>), grid_of(m, 8), dim3(kThreads), 0, s, m)
    if (dtype == BRX_DT_F32) { BRX_D(BRX_DT_F32); }
    else if (dtype == BRX_DT_BF16) { BRX_D(BRX_DT_BF16); }
    else { BRX_D(BRX_DT_F16); }
#undef BRX_D
    return hipGetLastError();
}

}  // namespace brx
