// MXFP4 on the device: rounding a group of 32 values to e2m1 codes under one e8m0 scale, and the
// operand layout of the scaled matrix instructions.
//
// A group's shared exponent is floor(log2(max |v|)) - 2 (2 is the exponent of e2m1's largest value,
// 6), clamped to [-127, 127]; an element is v / 2^e rounded to the nearest e2m1 value, ties to the
// even code, saturating at 6 (OCP Microscaling v1.0, section 6.3). The codes are those of
// formats.quantize_mxfp4: no negative zero. A group that holds a NaN or an infinity gets the NaN
// scale (255) and zero codes, so that every product it enters is NaN.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 with fp4 operands: lane l holds row (or column) l % 16 and the 32
// values of K group l / 16, sixteen bytes as the rows are packed, and that group's scale byte. So a
// packed row and its scale array are operands as they stand: nothing is converted. Which 128 K a step
// takes is free, the same on both sides: in a chunk of 512 K (256 bytes of a row, 16 groups), step t
// takes groups 4 g + t, so that the four scales of lane group g are one word of the row, a byte a step
// (the instruction selects it). The instruction multiplies exactly and accumulates in fp32; a scale of
// 255 makes the lane's outputs NaN.
#pragma once

#include "brx_internal.h"

namespace brx {

// Most tokens and (token, expert) pairs of a step that always runs on the few-pair kernels; of one that may, and
// whose blocks plan it themselves (a pair or two a lane) or have it bucketed first.
constexpr int kMxFewTokens = 8, kMxFewPairs = 64;
constexpr int kMxPlanPairs = 128;
constexpr int kMxMidTokens = 64, kMxMidPairs = 256;

// What the GEMM launches take beside the forward's arguments (FwdArgs::x is unused).
struct MxArgs {
    const uint8_t* xq;          // activation rows: codes [T, n_in / 2]
    const uint8_t* xs;          // ... and scales [T, n_in / 32]
    uint8_t* hq;                // intermediate rows in bucketed order: codes, `hstride` values apart
    uint8_t* hs;                // ... and scales
    const int32_t* order;
    const int32_t* tile_start;
    const int4* tinfo;
    uint16_t* y16;              // bf16 rows, a routed pair's at its row of the caller's, or null
    float* y32;                 // fp32 rows, likewise (every token's shared pair at its index), or null
    int32_t hstride;            // values between h rows
    int32_t E_ext, ntn;
    int32_t group;              // M tiles an XCD takes together
    int32_t proj;               // the projection of an expert product
};
static_assert(sizeof(FwdArgs) + sizeof(MxArgs) <= 512, "kernel argument blocks must stay under 512 bytes");

namespace {

typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

// |v|'s bits: their unsigned order is the order of the magnitudes, infinities and NaN on top.
__device__ __forceinline__ uint32_t mx_mag(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu; }

// The scale byte of a group whose largest magnitude has these bits (subnormal: floor(log2) - 2 is
// below -127).
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
    return top >= 0x7F800000u ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0);
}

// The codes of N = 4 or 8 consecutive values of a group with scale byte `sb`, the first in the low bits. The
// hardware conversion divides by the scale, rounds to nearest even and saturates; it keeps the
// sign of a zero, which is cleared here: (m + 7) of a code's magnitude m has bit 3 set unless m is 0,
// and never carries into the next code.
template <int N>
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[N], uint32_t sb) {
    const float sc = __builtin_bit_cast(float, sb == 0u ? 0x00400000u : sb << 23);
    uint32_t o = 0u;
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], sc, 0);
    o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], sc, 1);
    if constexpr (N == 8) {
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], sc, 2);
        o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], sc, 3);
    }
    const uint32_t m = o & 0x77777777u;
    o = m | (o & (m + 0x77777777u) & 0x88888888u);
    return sb == 255u ? 0u : o;
}

// The 4 x 4 transpose of 16-byte pieces over each four neighbouring lanes: lane q comes in with piece q of
// rows 0 to 3 (in[t]: row t) and goes out with pieces 0 to 3 of row q. Two rounds of exchanges, with the
// lane one away and with the lane two away.
template <int CTRL>
__device__ __forceinline__ uint32_t mx_quad(uint32_t v) {     // (every lane of a quad has a source)
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
__device__ __forceinline__ void mx_transpose(mx_u32x4 (&v)[4]) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int t = 0; t < 4; t += 2) {       // quad_perm [1, 0, 3, 2]
            const uint32_t a = v[t][i], b = v[t + 1][i], s = mx_quad<0xB1>(odd ? a : b);
            v[t][i] = odd ? s : a;
            v[t + 1][i] = odd ? b : s;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {          // quad_perm [2, 3, 0, 1]
            const uint32_t a = v[t][i], b = v[t + 2][i], s = mx_quad<0x4E>(high ? a : b);
            v[t][i] = high ? s : a;
            v[t + 2][i] = high ? b : s;
        }
    }
}

// The activation of one output: act_apply's values with the rule picked by selects (one copy of the code)
// and the limits by comparisons, which leave a NaN as it is; NaN for an absent expert.
__device__ __forceinline__ float mx_act(const FwdArgs& a, bool gated, bool clamped, float alpha, float g, float u,
                                        bool absent) {
    if (clamped) {
        g = g > a.limit ? a.limit : g;
        u = (u > a.limit ? a.limit : u < -a.limit ? -a.limit : u) + 1.0f;
    }
    const float h = x_sigmoid(g, alpha) * (gated ? u : 1.0f);
    return absent ? absent_nan() : h;
}

// acc += W (16 rows) . X (16 rows) over 128 K under byte S of each side's scales: lane l ends with W rows
// 4 (l / 16) .. + 3 of X row l % 16.
template <int S>
__device__ __forceinline__ f32x4_t mx_mfma(const mx_u32x4& w, uint32_t ws, const mx_u32x4& x, uint32_t xs,
                                           const f32x4_t& acc) {
    const mx_i32x8 a{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const mx_i32x8 b{(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, S, (int)ws, S, (int)xs);
}

}  // namespace
}  // namespace brx
