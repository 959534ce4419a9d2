// Grouped GEMMs of MXFP4 activations with MXFP4 experts on the scaled matrix instructions, and the
// expert layer made of them (see mx_common.h for the format).
//
//   k_mx_gemm<0>  gate/up: A rows are the pairs' token rows, weight rows the gate and up rows of 32
//                 features a wave; the epilogue applies act() in fp32 and rounds h to MXFP4 in place
//                 (a wave holds whole groups), in bucketed order.
//   k_mx_gemm<1>  down: A = h rows; + bias, each pair's bf16 row at its (token, k) position.
//   k_mx_gemm<2>  one projection of the pairs' token rows (the expert product), stored as <1>.
// The pairs are bucketed per expert and cut into M tiles by k_bucket (k_prefill.hip).
//
// y[n][m] = sum over K groups g of 2^(es_w[m][g] + es_x[n][g] - 254) * sum_k w[m][k] x[n][k], exact
// products, fp32 sums in steps of 128 K in order. A row's bits do not depend on its tile.
#include "mx_common.h"
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kMxWaves = 4;
constexpr int kMxThreads = 64 * kMxWaves;
constexpr int kMxRows = 64;                      // weight rows of a wave: four fragments
constexpr int kMxBlockN = kMxWaves * kMxRows;
// pairs of steps of weights a wave has in registers
template <int MP>
constexpr int kMxNH = 2;

// LDS bytes of a staged A row's codes and scales. One zero chunk follows the row's last: what the lanes
// of K groups past the row's end read. The code pitch is an odd number of 16-byte chunks and the scale
// pitch an odd number of words, so that 16 rows spread over the banks. A 16-bit copy into LDS fills a
// word, so a word holds two groups' scales.
__host__ __device__ inline int mx_code_pitch(int K) { return K / 2 + 16; }
__host__ __device__ inline int mx_scale_pitch(int K) { return (K / 64 | 1) * 4; }
__host__ __device__ inline int mx_row_lds(int K) { return mx_code_pitch(K) + mx_scale_pitch(K); }

__device__ __forceinline__ float mx_act(const FwdArgs& a, float g, float u) {
    return act_apply(a.act, g, u, a.alpha, a.limit);
}

template <int KIND, int MP>
__device__ __forceinline__ void mx_tile(const FwdArgs& a, const MxArgs& m, uint8_t* smem, int e, int m0, int rows,
                                        int slot, int nt) {
    const bool sh = e >= a.E;
    const Layout& L = sh ? a.lay_sh : a.lay;
    const uint8_t* base = sh ? a.shared : code_base(a, clamp_code(a, slot));
    const bool absent = slot == kAbsentCode;
    const bool gated = KIND == 0 && a.act != BRX_ACT_SILU_MLP;
    const Proj P0 = KIND == 0 ? L.p[0] : KIND == 1 ? L.p[2] : m.proj == 0 ? L.p[0] : m.proj == 1 ? L.p[1] : L.p[2];
    const Proj P1 = gated ? L.p[1] : P0;
    const int K = P0.n_in, N = P0.n_out;
    const int G = K / 32;                        // scale groups of a row, 16-byte chunks of its codes
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;

    // ---- weight rows. Fragment f's row m is row 8 (m / 4) + 4 (f % 2) + m % 4 of the 32 rows from c0 on
    // (fragments 2 and 3: the same 32 of the up matrix, or the next 32), so a lane's outputs of two
    // fragments are 8 consecutive rows. (Widths are multiples of 64: a wave's rows are all there or
    // none is; a wave with none works on the last ones and stores nothing.)
    const int c0 = nt * (gated ? kMxBlockN / 2 : kMxBlockN) + wv * (gated ? kMxRows / 2 : kMxRows);
    const int cr = min(c0, N - (gated ? kMxRows / 2 : kMxRows));
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(base, (uint32_t)L.bytes);
    // Codes: a load instruction reads 128 bytes (256 K) of 8 rows, lane (g, m) chunk 4 (m / 8) + g of row
    // m % 8: whole cache lines. Two of them (rows 0-7 and 8-15 of a fragment) hold two steps, and the
    // halves of each 16-lane group trade places to make the operands (mx_pair).
    const uint32_t vw = (uint32_t)P0.w + (uint32_t)(cr + 8 * ((l16 & 7) >> 2) + (l16 & 3)) * (uint32_t)(K / 2);
    const uint32_t dw = gated ? (uint32_t)(P1.w - P0.w) : 16u * (uint32_t)K;
    // Scales: a load reads the 16 scale bytes of 512 K of 16 rows, lane (g, m) the four of step g of row m;
    // the last four of a row where there are fewer left.
    const uint32_t vs = (uint32_t)P0.s + (uint32_t)(cr + 8 * (l16 >> 2) + (l16 & 3)) * (uint32_t)G;
    const uint32_t ds = gated ? (uint32_t)(P1.s - P0.s) : 32u * (uint32_t)G;
    struct Half {
        mx_u32x4 w[4][2];
    };
    struct Scales {
        uint32_t s[4];
    };
    // (chunks past the row's end read its last one: their A codes are zero)
    auto issue = [&](int hs, Half& q) __attribute__((always_inline)) {
        const uint32_t v = vw + 16u * (uint32_t)min(8 * hs + 4 * (l16 >> 3) + g, G - 1);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                q.w[f][i] = __builtin_amdgcn_raw_buffer_load_b128(rw, v, (f >> 1) * dw + (f & 1) * 2u * K + i * 8u * K, 0);
        }
    };
    auto issue_s = [&](int ss, Scales& q) __attribute__((always_inline)) {
        const uint32_t v = vs + (uint32_t)min(16 * ss + 4 * g, G - 4);
#pragma unroll
        for (int f = 0; f < 4; ++f)
            q.s[f] = __builtin_amdgcn_raw_buffer_load_b32(rw, v, (f >> 1) * ds + (f & 1) * 4u * G, 0);
    };
    // ---- the tile's pairs, one a lane, and what follows from them: the A row (gathered rows) and the
    // row the outputs go to (>= 0 routed, -2 - t shared)
    int arow = m0 + lane, drow = 0;
    if constexpr (KIND != 1) {
        const int pair = m.order[m0 + min(lane, rows - 1)];
        arow = pair_token(a, pair);
        if constexpr (KIND == 2) drow = pair_row(a, pair);
    } else {
        const int pair = m.order[m0 + min(lane, rows - 1)];
        drow = pair < a.P ? pair_row(a, pair) : -2 - (pair - a.P);
    }
    // the outputs' biases, and the first steps' scales and codes under the A rows' round trip
    const bool biased = P0.bias >= 0;              // uniform
    u32x4_t bias[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bias[h] = u32x4_t{0u, 0u, 0u, 0u};
        if (biased)
            bias[h] = __builtin_amdgcn_raw_buffer_load_b128(
                rw, (uint32_t)P0.bias + 2u * (uint32_t)(cr + 8 * g), gated ? h * (P1.bias - P0.bias) : 64 * h, 0);
    }
    constexpr int NH = kMxNH<MP>;
    Half q[NH];
    Scales qs[2];
    issue_s(0, qs[0]);
    issue(0, q[0]);
    asm volatile("" ::: "memory");

    // ---- A rows, whole, copied into LDS: row r by wave r % 4, a 1 KB run of codes or 64 scale pairs an
    // instruction. Lanes past the row, and rows past the tile's pairs, read past their buffer's end: zeros.
    const int PC = mx_code_pitch(K), PS = mx_scale_pitch(K);
    uint8_t* const sc = smem + 16 * MP * PC;
    const uint8_t* const srcc = KIND == 1 ? m.hq : m.xq;
    const uint8_t* const srcs = KIND == 1 ? m.hs : m.xs;
    const int64_t stride = KIND == 1 ? m.hstride : K;
#pragma unroll 1
    for (int i = 0; i < 4 * MP; ++i) {
        const int r = 4 * i + wv;
        const int64_t row = __builtin_amdgcn_readlane(arow, r);
        const __amdgpu_buffer_rsrc_t rc = make_rsrc(srcc + row * (stride / 2), r < rows ? (uint32_t)(K / 2) : 0u);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(srcs + row * (stride / 32), r < rows ? (uint32_t)G : 0u);
#pragma unroll 1
        for (int c = 0; c <= G; c += 64)
            if (c + lane <= G)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rc, (LDS_PTR)(smem + r * PC + 16 * c), 16, 16 * (c + lane), 0, 0, 0);
#pragma unroll 1
        for (int c = 0; 2 * c < G; c += 64)
            if (2 * (c + lane) < G)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_PTR)(sc + r * PS + 4 * c), 2, 2 * (c + lane), 0, 0, 0);
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int h = 1; h < NH - 1; ++h) issue(h, q[h]);
    dma_wait_barrier<8 * (NH - 2)>();

    f32x4_t acc[MP][4];
#pragma unroll
    for (int p = 0; p < MP; ++p)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[p][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const uint8_t* const ac = smem + l16 * PC;
    const uint8_t* const as = sc + l16 * PS;
    // one round: 8 steps, two loads of scales, four of codes; steps past the last multiply the zero chunk
    const int rounds = (G + 31) / 32;
    for (int r0 = 0; r0 < rounds; ++r0) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int hs = 4 * r0 + h;
            if ((h & 1) == 0) issue_s(hs / 2 + 1, qs[((h >> 1) + 1) & 1]);
            issue(hs + NH - 1, q[(h + NH - 1) % NH]);
            __builtin_amdgcn_sched_barrier(0);     // (or the loads sink to where they are used)
            mx_u32x4 w[2][4];
#pragma unroll
            for (int f = 0; f < 4; ++f) mx_pair(q[h % NH].w[f], w[0][f], w[1][f]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int s = 2 * hs + j;
                uint32_t ws[4];
                // (a mask, not a select: that becomes a branch; only the low byte counts)
                const uint32_t sh = 8u * (uint32_t)(g + max(0, 4 * s + 4 - G)), in = (uint32_t)((4 * s + g - G) >> 31);
#pragma unroll
                for (int f = 0; f < 4; ++f)
                    ws[f] = (mx_group(qs[(h >> 1) & 1].s[f], 2 * (h & 1) + j) >> (sh & 31u)) & in;
                const int gi = min(4 * s + g, G), gs = min(4 * s + g, G - 1);
#pragma unroll
                for (int p = 0; p < MP; ++p) {
                    const u32x4_t xv = *reinterpret_cast<const u32x4_t*>(ac + p * 16 * PC + 16 * gi);
                    const uint32_t xe = as[p * 16 * PS + 4 * (gs >> 1) + (gs & 1)];
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        acc[p][f] = mx_mfma(w[j][f], ws[f], mx_u32x4{xv[0], xv[1], xv[2], xv[3]}, xe, acc[p][f]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // ---- epilogue: lane (g, l16) has rows 8 g .. 8 g + 7 of each 32-row group for pair l16
    auto bias8 = [&](const u32x4_t& w, float (&b)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = bf2f((i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
    };
    if (c0 >= N) return;                           // (a wave past the last rows)
    const float nan = absent_nan();
    if constexpr (KIND == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {             // gated: one group; else fragments 2 h, 2 h + 1
            if (gated && h == 1) break;
            const int col = c0 + 32 * h + 8 * g;
            float b0[8], b1[8];
            bias8(bias[h], b0);
            bias8(bias[1], b1);
#pragma unroll
            for (int p = 0; p < MP; ++p) {
                float hv[8];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float gv = acc[p][2 * h + (i >> 2)][i & 3] + b0[i];
                    const float uv = gated ? acc[p][2 + (i >> 2)][i & 3] + b1[i] : 0.f;
                    hv[i] = absent ? nan : mx_act(a, gv, uv);
                    top = max(top, mx_mag(hv[i]));
                }
                top = max(top, lane_xor16(top));
                top = max(top, lane_xor32(top));
                const uint32_t sb = mx_scale(top);
                const int r = p * 16 + l16;
                if (r < rows) {
                    const int64_t row = m0 + r;
                    *reinterpret_cast<uint32_t*>(m.hq + row * (m.hstride / 2) + col / 2) = mx_codes(hv, sb);
                    if (g == 0) m.hs[row * (m.hstride / 32) + col / 32] = (uint8_t)sb;
                }
            }
        }
    } else {
        uint16_t* dst[MP];
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            const int d = __shfl(drow, p * 16 + l16, 64);
            dst[p] = p * 16 + l16 >= rows ? nullptr : d >= 0 ? m.y_routed + (int64_t)d * N : m.y_shared + (int64_t)(-2 - d) * N;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int col = c0 + 32 * h + 8 * g;
            float b[8];
            bias8(bias[h], b);
#pragma unroll
            for (int p = 0; p < MP; ++p) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = absent ? nan : acc[p][2 * h + (i >> 2)][i & 3] + b[i];
                if (dst[p])
                    *reinterpret_cast<u32x4_t*>(dst[p] + col) =
                        u32x4_t{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3]), pk_bf16(y[4], y[5]), pk_bf16(y[6], y[7])};
            }
        }
    }
}

// MPX: the call's tallest tiles, in 16 pairs (a launch of low tiles takes fewer registers).
template <int KIND, int MPX>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(MPX == 4 ? 2 : 3)))
void k_mx_gemm(FwdArgs a, MxArgs m) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    prefetch_args(a);
    const int blk = blockIdx.x;
    const int loc = blk / kXcd;
    const int nt = loc % m.ntn;
    const int mt = (loc / m.ntn) * kXcd + blk % kXcd;
    const int total = m.tile_start[m.E_ext];
    const int4 ti = m.tinfo[mt];
    if (mt >= total) return;
    const int e = ti.x, m0 = ti.y, rows = ti.z;
    const Layout& L = e >= a.E ? a.lay_sh : a.lay;
    const int pj = KIND == 0 ? 0 : KIND == 1 ? 2 : m.proj;
    const int N = pj == 0 ? L.p[0].n_out : pj == 1 ? L.p[1].n_out : L.p[2].n_out;
    const int per = KIND == 0 && a.act != BRX_ACT_SILU_MLP ? kMxBlockN / 2 : kMxBlockN;
    if (nt * per >= N) return;
    if (MPX == 1 || rows <= 16) mx_tile<KIND, 1>(a, m, smem, e, m0, rows, ti.w, nt);
    else if (MPX == 2 || rows <= 32) mx_tile<KIND, 2>(a, m, smem, e, m0, rows, ti.w, nt);
    else mx_tile<KIND, 4>(a, m, smem, e, m0, rows, ti.w, nt);
}

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Pairs of the call's tallest M tile: what the mean expert's pairs fit in, while a tile's A rows, held
// whole, leave room in LDS.
int mx_tile_rows(int64_t pairs, int64_t experts, int K) {
    int r = pairs <= 8 * experts ? 16 : pairs <= 24 * experts ? 32 : 64;
    while (r > 16 && r * mx_row_lds(K) > 150 * 1024) r /= 2;
    return r;
}

struct MxWs {
    uint8_t *xq, *xs, *hq, *hs;
    int32_t *order, *offsets, *tile_start;
    int4* tinfo;
    uint16_t *y_routed, *y_shared;
    int mt_pad, tile, Imax;
    size_t bytes;
};

// The scratch of a call over P routed pairs (and T shared ones) of T token rows; `layer`: a whole layer
// (else an expert product, whose activations and rows are the caller's).
MxWs carve(const FwdArgs& a, bool layer, int proj, void* ws) {
    const int T_sh = a.auto_shared ? a.T : 0, P_ext = a.P + T_sh, E_ext = a.E + (a.shared ? 1 : 0);
    MxWs w{};
    w.Imax = a.shared && a.I_sh > a.I ? a.I_sh : a.I;
    const int Kmax = layer ? (a.H > w.Imax ? a.H : w.Imax) : proj == 2 ? w.Imax : a.H;
    w.tile = mx_tile_rows(P_ext, E_ext, Kmax);
    w.mt_pad = ((P_ext + w.tile - 1) / w.tile + E_ext + kXcd - 1) / kXcd * kXcd;
    char* b = reinterpret_cast<char*>(ws);
    size_t off = 0;
    auto take = [&](size_t n) { char* p = b + off; off = align256(off + n); return p; };
    w.order = (int32_t*)take(sizeof(int32_t) * P_ext);
    w.offsets = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
    w.tile_start = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
    w.tinfo = (int4*)take(sizeof(int4) * (P_ext / 16 + E_ext + kXcd));   // (any tile height's)
    if (layer) {
        w.xq = (uint8_t*)take((size_t)a.T * (a.H / 2));
        w.xs = (uint8_t*)take((size_t)a.T * (a.H / 32));
        w.hq = (uint8_t*)take((size_t)P_ext * (w.Imax / 2));
        w.hs = (uint8_t*)take((size_t)P_ext * (w.Imax / 32));
        w.y_routed = (uint16_t*)take(a.yun ? 0 : (size_t)a.P * a.H * 2);
        w.y_shared = (uint16_t*)take((size_t)T_sh * a.H * 2);
    }
    w.bytes = off;
    return w;
}

template <int KIND>
hipError_t launch_gemm(const FwdArgs& a, MxArgs m, const MxWs& w, int K, int N, hipStream_t s) {
    const int per = KIND == 0 && a.act != BRX_ACT_SILU_MLP ? kMxBlockN / 2 : kMxBlockN;
    m.ntn = (N + per - 1) / per;
    const dim3 grid(w.mt_pad * m.ntn);
    const int lds = w.tile * mx_row_lds(K);
    if (w.tile == 16) hipLaunchKernelGGL((k_mx_gemm<KIND, 1>), grid, dim3(kMxThreads), lds, s, a, m);
    else if (w.tile == 32) hipLaunchKernelGGL((k_mx_gemm<KIND, 2>), grid, dim3(kMxThreads), lds, s, a, m);
    else hipLaunchKernelGGL((k_mx_gemm<KIND, 4>), grid, dim3(kMxThreads), lds, s, a, m);
    return hipGetLastError();
}

MxArgs gemm_args(const FwdArgs& a, const MxWs& w) {
    MxArgs m{};
    m.order = w.order;
    m.tile_start = w.tile_start;
    m.tinfo = w.tinfo;
    m.E_ext = a.E + (a.shared ? 1 : 0);
    return m;
}

hipError_t bucket(const FwdArgs& a, const MxWs& w, hipStream_t s) {
    return launch_bucket(a.pexp, a.P, a.E, a.E + (a.shared ? 1 : 0), a.auto_shared ? a.T : 0, w.tile, a.g2s, a.capacity,
                         a.host != nullptr, a.err, w.order, w.offsets, w.tile_start, w.tinfo, s);
}

}  // namespace

size_t mx_workspace_bytes(const FwdArgs& a, bool layer, int proj) { return carve(a, layer, proj, nullptr).bytes; }

hipError_t launch_mx_layer(const FwdArgs& a, void* ws, hipStream_t s) {
    const MxWs w = carve(a, true, 0, ws);
    MxRows x{};
    x.x = const_cast<uint16_t*>(a.x);
    x.codes = w.xq;
    x.scales = w.xs;
    x.rows = a.T;
    x.cols = a.H;
    x.x_row = a.H;
    x.groups = (int64_t)a.T * (a.H / 32);
    hipError_t e = launch_mx_quantize(x, BRX_DT_BF16, s);
    if (e != hipSuccess) return e;
    if ((e = bucket(a, w, s)) != hipSuccess) return e;
    MxArgs m = gemm_args(a, w);
    m.xq = w.xq;
    m.xs = w.xs;
    m.hq = w.hq;
    m.hs = w.hs;
    m.hstride = w.Imax;
    m.y_routed = a.yun ? a.yun : w.y_routed;
    m.y_shared = w.y_shared;
    if ((e = launch_gemm<0>(a, m, w, a.H, w.Imax, s)) != hipSuccess) return e;
    if ((e = launch_gemm<1>(a, m, w, w.Imax, a.H, s)) != hipSuccess) return e;
    if (!a.out) return hipSuccess;
    return launch_combine(m.y_routed, a.auto_shared ? w.y_shared : nullptr, a.w, a.sgate, a.T, a.k, a.H, a.out, s);
}

hipError_t launch_mx_product(const FwdArgs& a, const uint8_t* codes, const uint8_t* scales, int proj, void* ws,
                             hipStream_t s) {
    const MxWs w = carve(a, false, proj, ws);
    hipError_t e = bucket(a, w, s);
    if (e != hipSuccess) return e;
    MxArgs m = gemm_args(a, w);
    m.xq = codes;
    m.xs = scales;
    m.y_routed = a.yun;
    m.proj = proj;
    return launch_gemm<2>(a, m, w, proj == 2 ? w.Imax : a.H, proj == 2 ? a.H : w.Imax, s);
}

}  // namespace brx
