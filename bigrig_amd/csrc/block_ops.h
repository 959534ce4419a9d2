// Operators around a block's experts -- pairs sorted by expert and back (k_pairs.hip), products of sorted
// rows (k_grouped.hip), norms at both ends of the block (k_norm.hip) -- and device helpers they share.
#pragma once

#include "brx_internal.h"

namespace brx {

// Message and code of a failed call (brx_last_error), and whether brx_init was called: for entry points
// outside brx_api.hip.
int api_fail(int code, const char* fmt, ...);
int api_ready();

constexpr int kMaxExperts = 512;      // as in a layer descriptor
constexpr int kMaxTopK = 64;

inline int dtype_bytes(int dt) { return dt == BRX_DT_F32 ? 4 : 2; }

// ------------------------------------------------------------------ pairs
struct PairsPlan {
    const int32_t* idx;
    int32_t *order, *position, *offsets, *counts;
    int n, E;
};
size_t pairs_plan_workspace(int64_t n, int E);
hipError_t launch_pairs_plan(const PairsPlan& p, hipStream_t s);

struct PairRows {
    const void* x;              // [T, H] tokens or their gradients, rows `x_row` values apart
    const void* rows;           // [T k, H] sorted rows
    const int32_t* position;    // [T, k]
    const float* w;             // [T, k] or null (ones)
    void* out;
    float* dw;
    int64_t x_row;
    int T, k, H;
};
hipError_t launch_pairs_dispatch(const PairRows& p, int dtype, hipStream_t s);
hipError_t launch_pairs_combine(const PairRows& p, int dtype, hipStream_t s);
hipError_t launch_pairs_combine_backward(const PairRows& p, int dtype, hipStream_t s);

// ------------------------------------------------------------------ norms
// Gate forms: none, one value a channel, a row, an element.
enum { kGateNone = 0, kGateChannel = 1, kGateRow = 2, kGateFull = 3 };

struct NormArgs {
    const void *y, *r;                      // [T, H], rows y_row / r_row values apart; y null: enter
    const void *post, *next, *gate;         // null: none
    void *new_r, *h;                        // forward's outputs
    float *rstd_y, *rstd_n;                 // [T] (forward: may be null)
    const void *d_new, *d_h;                // backward: gradients of new_r and h, either may be null
    void *dy, *dr, *dgate;                  // backward's outputs, each may be null
    void *dpost, *dnext;
    float* partial;                         // column sums of the blocks
    int64_t y_row, r_row;
    float scale, eps;
    int T, H;
    int gate_form;
    int post_dt, next_dt, gate_dt;          // BRX_DT_*, of their gradients too
};
int norm_blocks(int T, int H);              // blocks of a backward launch
hipError_t launch_norm_forward(const NormArgs& a, int y_dt, int r_dt, hipStream_t s);
hipError_t launch_norm_backward(const NormArgs& a, int y_dt, int r_dt, hipStream_t s);

// ------------------------------------------------------------------ grouped products
struct GroupedArgs {
    const uint16_t *a, *b;        // operands (see k_grouped.hip)
    const uint16_t* bias;         // [E, N] or null
    uint16_t* out;
    const int32_t* offsets;       // [E + 1]
    int64_t b_expert, b_row;      // values between experts and rows of b (weights)
    int P, E, K, N;               // rows, experts, reduction (row products) and output widths
    bool past_cache;              // (set by the launch) the output is stored past the caches
};
hipError_t launch_grouped_rows(const GroupedArgs& g, bool transposed, int dtype, hipStream_t s);
hipError_t launch_grouped_weight(const GroupedArgs& g, int dtype, hipStream_t s);
hipError_t launch_grouped_bias(const GroupedArgs& g, int dtype, hipStream_t s);

// ------------------------------------------------------------------ device helpers
namespace {

typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));

// 16 bytes at any address their values are aligned to.
__device__ __forceinline__ v4u_t get16(const void* p) {
    typedef v4u_t __attribute__((aligned(2))) V;
    return *reinterpret_cast<const V*>(p);
}
__device__ __forceinline__ void set16(void* p, const v4u_t& v) {
    typedef v4u_t __attribute__((aligned(2))) V;
    *reinterpret_cast<V*>(p) = v;
}

template <int DT>
struct Elem;
template <>
struct Elem<BRX_DT_F32> { typedef float T; static constexpr int kVec = 4; };
template <>
struct Elem<BRX_DT_BF16> { typedef uint16_t T; static constexpr int kVec = 8; };
template <>
struct Elem<BRX_DT_F16> { typedef uint16_t T; static constexpr int kVec = 8; };

template <int DT>
__device__ __forceinline__ float to_f(typename Elem<DT>::T v) {
    if constexpr (DT == BRX_DT_F32) return v;
    else if constexpr (DT == BRX_DT_BF16) return bf2f(v);
    else return h2f(v);
}
// fp32 to a type, rounded to nearest even
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T from_f(float v) {
    if constexpr (DT == BRX_DT_F32) return v;
    else if constexpr (DT == BRX_DT_BF16) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The values of 16 bytes, and back.
template <int DT>
__device__ __forceinline__ void unpack(const v4u_t& q, float (&v)[Elem<DT>::kVec]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = q[i];
        if constexpr (DT == BRX_DT_F32) {
            v[i] = __builtin_bit_cast(float, x);
        } else {
            v[2 * i] = to_f<DT>((uint16_t)(x & 0xFFFFu));
            v[2 * i + 1] = to_f<DT>((uint16_t)(x >> 16));
        }
    }
}
template <int DT>
__device__ __forceinline__ v4u_t pack(const float (&v)[Elem<DT>::kVec]) {
    v4u_t q;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == BRX_DT_F32) q[i] = __builtin_bit_cast(uint32_t, v[i]);
        else q[i] = (uint32_t)from_f<DT>(v[2 * i]) | ((uint32_t)from_f<DT>(v[2 * i + 1]) << 16);
    }
    return q;
}

}  // namespace
}  // namespace brx
