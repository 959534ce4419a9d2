// Norms at both ends of a block, with its gate, residual scale and residual sum, and the gradients.
//
//   n(v; w) = v rstd(v) w,  rstd(v) = (mean(v^2) + eps)^(-1/2)
//   enter   h = n(r; next)
//   leave   u = n(y; post) (or y),  r' = r + scale gate u,  h = n(r'; next)
// r' is rounded to its type first and h is made of what was rounded, as a later `enter` of r' would: the two calls
// and the one give the same bits. Statistics and sums are fp32. The gradients, with D the whole gradient of r':
//   D  = d_new + rstd (g - x^ mean(g x^)),   g = d_h next,  x^ = r' rstd
//   dr = D,  dnext = sum_t d_h x^,  dgate = scale u D summed to the gate's shape
//   du = scale gate D,  dy = rstd_y (q - y^ mean(q y^)),  q = du post,  dpost = sum_t du y^
// Column sums are made in two steps, each block's over the rows it took and then those of the blocks, in a fixed
// order.
//
// Bound: memory, each input read once and each output written once; a row stays in registers, 8 values a run. 16384 x 2048,
// bf16 with an fp32 residual, both norms and a gate: 74 us (5.4 TB/s), its gradient 126 us (4.8 TB/s).
#include "block_ops.h"

namespace brx {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int V = 8;                  // values of a run

// Run c of a row: elements from `at` on; those below `own` are another lane's (the last run of a row whose width is no
// multiple of 8 overlaps the one before; a lane without a run owns none).
struct Run {
    int at, own;
};
template <int TPR>
__device__ __forceinline__ Run run_of(int H, int lane, int c) {
    const int i = (c * TPR + lane) * V;
    const int at = min(i, max(H - V, 0));
    return {at, min(i - at, V)};
}

template <int DT>
__device__ __forceinline__ void load8(const void* base, int64_t row_at, const Run& r, int H, float (&v)[V]) {
    typedef typename Elem<DT>::T ET;
    const ET* p = (const ET*)base + row_at + r.at;
    if (H >= V) {                     // uniform
        if constexpr (DT == BRX_DT_F32) {
            float lo[4], hi[4];
            unpack<DT>(get16(p), lo);
            unpack<DT>(get16(p + 4), hi);
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[i] = lo[i]; v[4 + i] = hi[i]; }
        } else {
            unpack<DT>(get16(p), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = i < H ? to_f<DT>(p[min(i, H - 1)]) : 0.f;
    }
}
// the same of a vector whose type is known at run time (uniform)
__device__ __forceinline__ void load8_any(const void* base, int dt, int64_t row_at, const Run& r, int H, float (&v)[V]) {
    if (dt == BRX_DT_BF16) load8<BRX_DT_BF16>(base, row_at, r, H, v);
    else if (dt == BRX_DT_F32) load8<BRX_DT_F32>(base, row_at, r, H, v);
    else load8<BRX_DT_F16>(base, row_at, r, H, v);
}
template <int DT>
__device__ __forceinline__ void store8(void* base, int64_t row_at, const Run& r, int H, const float (&v)[V]) {
    typedef typename Elem<DT>::T ET;
    ET* p = (ET*)base + row_at + r.at;
    if (r.own >= V) return;
    if (H >= V) {
        if constexpr (DT == BRX_DT_F32) {
            const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
            set16(p, pack<DT>(lo));
            set16(p + 4, pack<DT>(hi));
        } else {
            set16(p, pack<DT>(v));
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < H) p[i] = from_f<DT>(v[i]);
    }
}
// elements that count: owned, and inside a row of fewer than 8
__device__ __forceinline__ bool counts(const Run& r, int H, int i) { return i >= r.own && i < H; }

// v^(-1/2): the instruction's value is off by up to a step of its last place, which every value of the row would be off by; one
// Newton step on it leaves its own rounding. (An infinite v, of a sum that overflowed, keeps its 0.)
__device__ __forceinline__ float rsqrt_of(float v) {
    const float r = __builtin_amdgcn_rsqf(v), t = v * r;
    const float e = __builtin_fmaf(-t, r, 1.0f) - __builtin_fmaf(v, r, -t) * r;      // 1 - v r^2
    return v < __builtin_inff() ? __builtin_fmaf(0.5f * r, e, r) : r;
}

// Sum over the threads of a row. Across waves: one slot a wave in `s`, two sets of slots in turn, so one barrier a
// sum suffices.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float (*s)[kWaves], int& turn) {
    v = wave_sum(v);
    if constexpr (TPR == kWave) {
        return v;
    } else {
        const int wv = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) s[turn][wv] = v;
        __syncthreads();
        const float a = (s[turn][0] + s[turn][1]) + (s[turn][2] + s[turn][3]);
        turn ^= 1;
        return a;
    }
}

template <int YD, int RD, int TPR, int NC>
__global__ __launch_bounds__(kThreads) void k_norm_forward(NormArgs a) {
    __shared__ float slots[2][kWaves];
    int turn = 0;
    const int lane = threadIdx.x & (TPR - 1);
    const int t = blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
    if (t >= a.T) return;             // (whole waves, or the whole block)
    const int H = a.H;
    Run rn[NC];
    float r[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        rn[c] = run_of<TPR>(H, lane, c);
        load8<RD>(a.r, (int64_t)t * a.r_row, rn[c], H, r[c]);
    }
    if (a.y) {
        float y[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) load8<YD>(a.y, (int64_t)t * a.y_row, rn[c], H, y[c]);
        if (a.post) {
            float s = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) s = counts(rn[c], H, i) ? __builtin_fmaf(y[c][i], y[c][i], s) : s;
            const float rstd = rsqrt_of(row_sum<TPR>(s, slots, turn) / (float)H + a.eps);
            if (lane == 0 && a.rstd_y) a.rstd_y[t] = rstd;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float w[V];
                load8_any(a.post, a.post_dt, 0, rn[c], H, w);
#pragma unroll
                for (int i = 0; i < V; ++i) y[c][i] = y[c][i] * rstd * w[i];
            }
        }
        const float g_row = a.gate_form != kGateRow ? 1.0f
                            : a.gate_dt == BRX_DT_F32 ? ((const float*)a.gate)[t]
                            : a.gate_dt == BRX_DT_BF16 ? bf2f(((const uint16_t*)a.gate)[t]) : h2f(((const uint16_t*)a.gate)[t]);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float g[V];
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = g_row;
            if (a.gate_form == kGateChannel) load8_any(a.gate, a.gate_dt, 0, rn[c], H, g);
            if (a.gate_form == kGateFull) load8_any(a.gate, a.gate_dt, (int64_t)t * H, rn[c], H, g);
#pragma unroll
            for (int i = 0; i < V; ++i) r[c][i] = to_f<RD>(from_f<RD>(__builtin_fmaf(a.scale * g[i], y[c][i], r[c][i])));
            store8<RD>(a.new_r, (int64_t)t * H, rn[c], H, r[c]);
        }
    }
    if (!a.h) return;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) s = counts(rn[c], H, i) ? __builtin_fmaf(r[c][i], r[c][i], s) : s;
    const float rstd = rsqrt_of(row_sum<TPR>(s, slots, turn) / (float)H + a.eps);
    if (lane == 0 && a.rstd_n) a.rstd_n[t] = rstd;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float w[V], h[V];
        if (a.next) load8_any(a.next, a.next_dt, 0, rn[c], H, w);
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = a.next ? r[c][i] * rstd * w[i] : r[c][i] * rstd;
        store8<YD>(a.h, (int64_t)t * H, rn[c], H, h);
    }
}

// A row per TPR threads, rows one grid apart. What of dpost, dgate (one value a channel) and dnext is asked for is
// summed over a thread's rows in registers, over a block's row groups through LDS, and written to `partial`
// [3][blocks][H].
template <int YD, int RD, int TPR, int NC>
__global__ __launch_bounds__(kThreads) void k_norm_backward(NormArgs a) {
    constexpr int kRows = kThreads / TPR;
    __shared__ float slots[2][kWaves];
    extern __shared__ float merge[];  // [H], where a block has several row groups
    int turn = 0;
    const int lane = threadIdx.x & (TPR - 1), group = threadIdx.x / TPR;
    const int H = a.H;
    const float inv = 1.0f / (float)H;
    Run rn[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) rn[c] = run_of<TPR>(H, lane, c);
    float sum_post[NC][V], sum_gate[NC][V], sum_next[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) sum_post[c][i] = sum_gate[c][i] = sum_next[c][i] = 0.f;
    // the columns' weights, in registers where these suffice
    constexpr bool kKeep = NC <= 2;
    float w_post[kKeep ? NC : 1][V], w_next[kKeep ? NC : 1][V], w_gate[kKeep ? NC : 1][V];
    if constexpr (kKeep) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < V; ++i) w_post[c][i] = w_next[c][i] = w_gate[c][i] = 1.0f;
            if (a.post) load8_any(a.post, a.post_dt, 0, rn[c], H, w_post[c]);
            if (a.next) load8_any(a.next, a.next_dt, 0, rn[c], H, w_next[c]);
            if (a.gate_form == kGateChannel) load8_any(a.gate, a.gate_dt, 0, rn[c], H, w_gate[c]);
        }
    }
    for (int t = blockIdx.x * kRows + group; t < a.T; t += gridDim.x * kRows) {
        float D[NC][V], y[NC][V], x[NC][V], g[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int i = 0; i < V; ++i) D[c][i] = 0.f;
            if (a.d_new) load8<RD>(a.d_new, (int64_t)t * H, rn[c], H, D[c]);
            if (a.y) load8<YD>(a.y, (int64_t)t * a.y_row, rn[c], H, y[c]);
            if (a.d_h) {
                load8<RD>(a.r, (int64_t)t * a.r_row, rn[c], H, x[c]);
                load8<YD>(a.d_h, (int64_t)t * H, rn[c], H, g[c]);
            }
        }
        if (a.d_h) {
            float s = 0.f;
            const float rstd = a.rstd_n[t];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float w[V];
                if constexpr (!kKeep) {
                    if (a.next) load8_any(a.next, a.next_dt, 0, rn[c], H, w);
                    else
#pragma unroll
                        for (int i = 0; i < V; ++i) w[i] = 1.0f;
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[c][i] *= rstd;
                    sum_next[c][i] = __builtin_fmaf(g[c][i], x[c][i], sum_next[c][i]);
                    g[c][i] *= kKeep ? w_next[c][i] : w[i];
                    s = counts(rn[c], H, i) ? __builtin_fmaf(g[c][i], x[c][i], s) : s;
                }
            }
            const float m = row_sum<TPR>(s, slots, turn) * inv;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) D[c][i] = __builtin_fmaf(rstd, __builtin_fmaf(-x[c][i], m, g[c][i]), D[c][i]);
        }
        if (a.dr) {
#pragma unroll
            for (int c = 0; c < NC; ++c) store8<RD>(a.dr, (int64_t)t * H, rn[c], H, D[c]);
        }
        if (!a.y) continue;
        const float rstd = a.post ? a.rstd_y[t] : 1.0f;
        const float g_row = a.gate_form != kGateRow ? 1.0f
                            : a.gate_dt == BRX_DT_F32 ? ((const float*)a.gate)[t]
                            : a.gate_dt == BRX_DT_BF16 ? bf2f(((const uint16_t*)a.gate)[t]) : h2f(((const uint16_t*)a.gate)[t]);
        float s = 0.f, gs = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float w[V], g[V], dg[V];
            if constexpr (!kKeep) {
#pragma unroll
                for (int i = 0; i < V; ++i) w[i] = 1.0f;
                if (a.post) load8_any(a.post, a.post_dt, 0, rn[c], H, w);
            }
            if (a.gate_form == kGateFull) {
                load8_any(a.gate, a.gate_dt, (int64_t)t * H, rn[c], H, g);
            } else if (!kKeep && a.gate_form == kGateChannel) {
                load8_any(a.gate, a.gate_dt, 0, rn[c], H, g);
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = kKeep && a.gate_form == kGateChannel ? w_gate[c][i] : g_row;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float wp = kKeep ? w_post[c][i] : w[i];
                y[c][i] *= rstd;                                                // y^ (or y)
                dg[i] = a.scale * (y[c][i] * wp) * D[c][i];
                sum_gate[c][i] += dg[i];
                gs = counts(rn[c], H, i) ? gs + dg[i] : gs;
                const float du = a.scale * g[i] * D[c][i];
                sum_post[c][i] = __builtin_fmaf(du, y[c][i], sum_post[c][i]);
                D[c][i] = du * wp;                                              // q
                s = counts(rn[c], H, i) ? __builtin_fmaf(D[c][i], y[c][i], s) : s;
            }
            if (a.gate_form == kGateFull && a.dgate) {
                if (a.gate_dt == BRX_DT_F32) store8<BRX_DT_F32>(a.dgate, (int64_t)t * H, rn[c], H, dg);
                else if (a.gate_dt == BRX_DT_BF16) store8<BRX_DT_BF16>(a.dgate, (int64_t)t * H, rn[c], H, dg);
                else store8<BRX_DT_F16>(a.dgate, (int64_t)t * H, rn[c], H, dg);
            }
        }
        if (a.gate_form == kGateRow && a.dgate) {
            const float v = row_sum<TPR>(gs, slots, turn);
            if (lane == 0) {
                if (a.gate_dt == BRX_DT_F32) ((float*)a.dgate)[t] = v;
                else ((uint16_t*)a.dgate)[t] = a.gate_dt == BRX_DT_BF16 ? from_f<BRX_DT_BF16>(v) : from_f<BRX_DT_F16>(v);
            }
        }
        if (a.dy) {
            if (a.post) {
                const float m = row_sum<TPR>(s, slots, turn) * inv;
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int i = 0; i < V; ++i) D[c][i] = rstd * __builtin_fmaf(-y[c][i], m, D[c][i]);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) store8<YD>(a.dy, (int64_t)t * H, rn[c], H, D[c]);
        }
    }
    auto columns = [&](int which, float (&v)[NC][V]) __attribute__((always_inline)) {
        float* to = a.partial + ((int64_t)which * gridDim.x + blockIdx.x) * H;
        if constexpr (kRows > 1) {
            for (int w = 0; w < kRows; ++w) {
                __syncthreads();
                if (group == w) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            if (counts(rn[c], H, i)) {
                                const float x = w ? merge[rn[c].at + i] + v[c][i] : v[c][i];
                                if (w == kRows - 1) to[rn[c].at + i] = x;
                                else merge[rn[c].at + i] = x;
                            }
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (counts(rn[c], H, i)) to[rn[c].at + i] = v[c][i];
        }
    };
    if (a.dpost) columns(0, sum_post);
    if (a.dgate && a.gate_form == kGateChannel) columns(1, sum_gate);
    if (a.dnext) columns(2, sum_next);
}

// The blocks' column sums, summed: 64 columns a block, its waves take every 16th row each and join in order.
constexpr int kColThreads = 1024;
__global__ __launch_bounds__(kColThreads) void k_norm_columns(NormArgs a, int blocks) {
    constexpr int W = kColThreads / kWave;
    __shared__ float s[W][kWave];
    const int which = blockIdx.y, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    void* const out = which == 0 ? a.dpost : which == 1 ? (a.gate_form == kGateChannel ? a.dgate : nullptr) : a.dnext;
    if (!out) return;
    const int dt = which == 0 ? a.post_dt : which == 1 ? a.gate_dt : a.next_dt;
    const int col = blockIdx.x * kWave + lane, H = a.H;
    const float* p = a.partial + (int64_t)which * blocks * H + min(col, H - 1);
    float v = 0.f;
#pragma unroll 8
    for (int b = wv; b < blocks; b += W) v += p[(int64_t)b * H];
    s[wv][lane] = v;
    __syncthreads();
    if (wv == 0 && col < H) {
        for (int w = 1; w < W; ++w) v += s[w][lane];
        if (dt == BRX_DT_F32) ((float*)out)[col] = v;
        else ((uint16_t*)out)[col] = dt == BRX_DT_BF16 ? from_f<BRX_DT_BF16>(v) : from_f<BRX_DT_F16>(v);
    }
}

// Threads of a row: a wave up to 1024 values, else a block; of a gradient's, whose block sums columns over its rows, a wave up
// to 512 (4999 x 1001, fp16: a wave a row 26 us, a block 17.6).
constexpr int kWaveRow = 1024, kWaveRowBack = 512;
inline int threads_of(int H, int wave_row) { return H <= wave_row ? kWave : kThreads; }

// Blocks of a gradient: as many as its registers let run at once, so that none is left for a second round on a part of the
// chip: of up to 2048 values (138 registers) three a CU, up to 4096 (221) two, beyond (402) one. bf16, us, 256 / 512 / 768 / 1024
// blocks: 16384 x 2048 (fp32 residual) 206 / 136 / 129 / 156; 16384 x 2880 enter 195 / 119 / 152 / 127, leave 325 / 224 / 285 / 240;
// 16384 x 4096 207 / 129 / 164 / 138, 350 / 258 / 323 / 277; 4096 x 8192 114 / 121 / 128 / 135, 248 / 269 / 290 / 310.
inline int back_blocks(int H) { return H <= kThreads * V ? 768 : H <= 2 * kThreads * V ? 512 : 256; }

}  // namespace

int norm_blocks(int T, int H) {
    const int per = kThreads / threads_of(H, kWaveRowBack);
    const int most = (T + per - 1) / per;
    return most < back_blocks(H) ? most : back_blocks(H);
}

#define BRX_SHAPE(KERNEL, YD, RD, WAVE_ROW, GRID, LDS)                                                                 \
    do {                                                                                                               \
        if (a.H <= 512) hipLaunchKernelGGL((KERNEL<YD, RD, kWave, 1>), GRID, dim3(kThreads), LDS, s, a);               \
        else if (WAVE_ROW > 512 && a.H <= 1024)                                                                        \
            hipLaunchKernelGGL((KERNEL<YD, RD, WAVE_ROW <= 512 ? kThreads : kWave, WAVE_ROW <= 512 ? 1 : 2>), GRID,    \
                               dim3(kThreads), 0, s, a);                                                               \
        else if (a.H <= kThreads * V) hipLaunchKernelGGL((KERNEL<YD, RD, kThreads, 1>), GRID, dim3(kThreads), 0, s, a);\
        else if (a.H <= 2 * kThreads * V) hipLaunchKernelGGL((KERNEL<YD, RD, kThreads, 2>), GRID, dim3(kThreads), 0, s, a);\
        else hipLaunchKernelGGL((KERNEL<YD, RD, kThreads, 4>), GRID, dim3(kThreads), 0, s, a);                         \
    } while (0)
// (y's type, r's type: equal, or r fp32)
#define BRX_TYPES(KERNEL, W, GRID, LDS)                                                                                \
    do {                                                                                                               \
        if (y_dt == BRX_DT_F32) BRX_SHAPE(KERNEL, BRX_DT_F32, BRX_DT_F32, W, GRID, LDS);                               \
        else if (y_dt == BRX_DT_BF16 && r_dt == y_dt) BRX_SHAPE(KERNEL, BRX_DT_BF16, BRX_DT_BF16, W, GRID, LDS);       \
        else if (y_dt == BRX_DT_BF16) BRX_SHAPE(KERNEL, BRX_DT_BF16, BRX_DT_F32, W, GRID, LDS);                        \
        else if (r_dt == y_dt) BRX_SHAPE(KERNEL, BRX_DT_F16, BRX_DT_F16, W, GRID, LDS);                                \
        else BRX_SHAPE(KERNEL, BRX_DT_F16, BRX_DT_F32, W, GRID, LDS);                                                  \
    } while (0)

hipError_t launch_norm_forward(const NormArgs& a, int y_dt, int r_dt, hipStream_t s) {
    const int per = kThreads / threads_of(a.H, kWaveRow);
    const dim3 grid((a.T + per - 1) / per);
    BRX_TYPES(k_norm_forward, kWaveRow, grid, 0);
    return hipGetLastError();
}

hipError_t launch_norm_backward(const NormArgs& a, int y_dt, int r_dt, hipStream_t s) {
    const int blocks = norm_blocks(a.T, a.H);
    const dim3 grid(blocks);
    const size_t lds = (size_t)a.H * sizeof(float);     // (blocks of several rows)
    BRX_TYPES(k_norm_backward, kWaveRowBack, grid, lds);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (!a.dpost && !a.dnext && !(a.dgate && a.gate_form == kGateChannel)) return hipSuccess;
    hipLaunchKernelGGL(k_norm_columns, dim3((a.H + kWave - 1) / kWave, 3), dim3(kColThreads), 0, s, a, blocks);
    return hipGetLastError();
}

}  // namespace brx
