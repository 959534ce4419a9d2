// Grouped GEMMs of MXFP4 activations with MXFP4 experts on the scaled matrix instructions, and the
// expert layer made of them (see mx_common.h for the format).
//
//   k_mx_gemm<0>  gate/up: A rows are the pairs' token rows, weight rows the gate and up rows of 32
//                 features a wave; the epilogue applies act() in fp32 and rounds h to MXFP4 in place
//                 (a wave holds whole groups), in bucketed order.
//   k_mx_gemm<1>  down: A = h rows; + bias, each pair's row at its (token, k) position in fp32 (for a sum), in
//                 bf16 (unreduced rows), or both.
//   k_mx_gemm<2>  one projection of the pairs' token rows (the expert product), in bf16.
//   k_mx_combine  the routing-weighted sums of the fp32 rows.
// The pairs are bucketed per expert and cut into M tiles by bucket.h: in k_mx_prepare, which rounds x beside it
// (a layer), or in k_bucket (a product).
//
// y[n][m] = sum over K groups g of 2^(es_w[m][g] + es_x[n][g] - 254) * sum_k w[m][k] x[n][k], exact
// products, fp32 sums in steps of 128 K in order. A row's bits do not depend on its tile.
//
// What bounds it. 512 tokens of the gpt-oss shape (16 pairs an expert, 1.70 GB of weights): the weight stream,
// 223 + 126 us, 4.9 TB/s, where a copy of 1 GiB reaches 4.8 to 5.1. 2048 tokens of the Qwen3 shape under a Zipf law
// (128 pairs an expert on average, 155 GFLOP): 88 + 78 us, 930 TFLOP/s, and 22 us for the sums (135 MB, 6.1
// TB/s); matrix instructions fill 15% of the time and vector ones half, and the rest is the wait for each chunk's
// weights: with 64 pairs a tile a wave has 64 + 64 registers of sums and weights, and a second set of weights
// does not fit.
#include <type_traits>

#include "bucket.h"
#include "mx_common.h"
#include "pf_common.h"

namespace brx {
namespace {
constexpr int kMxWaves = 4;
constexpr int kMxThreads = 64 * kMxWaves;
constexpr int kMxRows = 64;                      // weight rows of a wave: four fragments

// A rows pass through LDS in chunks of 512 K, two at a time: 256 bytes of codes a row (16-byte piece c
// in slot c ^ (row % 16), so that 16 rows read at one piece fall into different banks), and the 16
// scales two to a word (a 16-bit copy into LDS fills a word). The scales of a wave's weight rows are
// in LDS whole, as they lie in memory.
template <int MP>
constexpr int kMxA = 16 * MP * 256;
template <int MP>
constexpr int kMxBuf = kMxA<MP> + 16 * MP * 32;
__host__ __device__ constexpr int mx_table(int K) { return kMxWaves * kMxRows * (K / 32) + 16; }
// Copies of a chunk's scales a wave issues, 8 rows each (the last waves repeat the first ones' where rows run
// out); its codes are MP copies of 1 KB (4 rows) a wave.
template <int MP>
constexpr int kMxNS = (MP + 1) / 2;

// 16 or 2 bytes a lane from byte `off` of the buffer into LDS, lane after lane from `to` on (2 bytes fill
// a word).
__device__ __forceinline__ void copy16(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_PTR)to, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void copy2(__amdgpu_buffer_rsrc_t r, uint8_t* to, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_PTR)to, 2, off, 0, 0, 0);
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
    const int c0 = (nt * kMxWaves + wv) * (gated ? kMxRows / 2 : kMxRows);
    const int cr = min(c0, N - (gated ? kMxRows / 2 : kMxRows));
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(base, (uint32_t)L.bytes);
    // Codes: four neighbouring lanes read 64 bytes in a row, the cache's coalescing width (one row a
    // lane, 16 bytes each, costs it four times the lookups, and they bound the kernel): lane (g, m)
    // piece 4 g + m % 4 of row 4 (m / 4) + t in load t, and the four transpose (mx_transpose).
    const uint32_t vw = (uint32_t)P0.w + (uint32_t)(cr + 8 * (l16 >> 2)) * (uint32_t)(K / 2);
    const uint32_t dw = gated ? (uint32_t)(P1.w - P0.w) : 16u * (uint32_t)K;
    // A chunk comes in two halves of two fragments, each requested as soon as the one before it in its registers
    // is used (both at the end of a chunk: 512 tokens of the gpt-oss shape 355 us a layer, 349 so).
    struct Half {
        mx_u32x4 w[2][4];
    };
    // (pieces past the row's end read its last one: their A codes are zero; past the last chunk the request is
    // out of the buffer's range, wherever the scalar offset counts, and costs no memory access -- under a branch
    // the registers spilled)
    auto issue = [&](int ch, Half& q, uint32_t d) __attribute__((always_inline)) {
        const uint32_t v = 16 * ch < G ? vw + 16u * (uint32_t)min(16 * ch + 4 * g + (l16 & 3), G - 1) : 0x80000000u;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                q.w[f][t] = __builtin_amdgcn_raw_buffer_load_b128(rw, v, d + f * 2u * K + t * (uint32_t)(K / 2), 0);
        }
    };

    // ---- what this lane copies of the A rows: piece lc of tile row r at byte va of the codes, slot ls of
    // row r at byte vx of the scales; rows past the tile's pairs have pieces past every row's end
    constexpr int NC = MP, NS = kMxNS<MP>;
    constexpr int kNone = 1 << 28;
    const uint8_t* const srcc = KIND == 1 ? m.hq + (int64_t)m0 * (m.hstride / 2) : m.xq;
    const uint8_t* const srcs = KIND == 1 ? m.hs + (int64_t)m0 * (m.hstride / 32) : m.xs;
    const uint32_t sa = (uint32_t)(KIND == 1 ? m.hstride : K) / 2;
    const int64_t nrow = KIND == 1 ? rows : a.T;
    const __amdgpu_buffer_rsrc_t rc = make_rsrc(srcc, (uint32_t)(nrow * sa));
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(srcs, (uint32_t)(nrow * (sa / 16)));
    int pc[NC], px[NS], pd[MP];
    auto crow = [&](int i) { return 4 * (wv * NC + i) + (lane >> 4); };
    auto srow = [&](int i) { return 8 * ((wv * NS + i) % (2 * MP)) + (lane >> 3); };
    if constexpr (KIND != 1) {
#pragma unroll
        for (int i = 0; i < NC; ++i) pc[i] = m.order[m0 + min(crow(i), rows - 1)];
#pragma unroll
        for (int i = 0; i < NS; ++i) px[i] = m.order[m0 + min(srow(i), rows - 1)];
    }
    if constexpr (KIND != 0) {
#pragma unroll
        for (int p = 0; p < MP; ++p) pd[p] = m.order[m0 + min(16 * p + l16, rows - 1)];
    }
    // the outputs' biases, and the first steps' scales and codes under the pair list's round trip
    const bool biased = P0.bias >= 0;              // uniform
    u32x4_t bias[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bias[h] = u32x4_t{0u, 0u, 0u, 0u};
        if (biased)
            bias[h] = __builtin_amdgcn_raw_buffer_load_b128(
                rw, (uint32_t)P0.bias + 2u * (uint32_t)(cr + 8 * g), gated ? h * (P1.bias - P0.bias) : 64 * h, 0);
    }
    Half qa, qb;
    issue(0, qa, 0);
    issue(0, qb, dw);
    asm volatile("" ::: "memory");
    uint32_t va[NC], vx[NS];
    int lc[NC], ls[NS];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int r = crow(i);
        lc[i] = r < rows ? (lane & 15) ^ (r & 15) : kNone;
        va[i] = (uint32_t)(KIND == 1 ? min(r, rows - 1) : pair_token(a, pc[i])) * sa + 16u * (uint32_t)((lane & 15) ^ (r & 15));
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int r = srow(i);
        ls[i] = r < rows ? 2 * (lane & 7) : kNone;
        vx[i] = (uint32_t)(KIND == 1 ? min(r, rows - 1) : pair_token(a, px[i])) * (sa / 16) + 2u * (uint32_t)(lane & 7);
    }
    // pieces past a row's end are copied from past the buffer's end: the range check writes zeros
    auto issue_a = [&](int ch) __attribute__((always_inline)) {
        uint8_t* const buf = smem + (ch & 1) * kMxBuf<MP>;
#pragma unroll
        for (int i = 0; i < NC; ++i)
            copy16(rc, buf + (wv * NC + i) * 1024, lc[i] + 16 * ch < G ? va[i] + 256u * ch : 0xFFFFFF00u);
#pragma unroll
        for (int i = 0; i < NS; ++i)
            copy2(rs, buf + kMxA<MP> + (wv * NS + i) % (2 * MP) * 256,
                        ls[i] + 16 * ch < G ? vx[i] + 16u * ch : 0xFFFFFF00u);
    };
    issue_a(0);
    // the scales of the wave's rows: two runs of 32 rows, 16 bytes a lane
    uint8_t* const tbl = smem + 2 * kMxBuf<MP> + wv * kMxRows * G;
    const uint32_t ts = (uint32_t)P0.s + (uint32_t)(cr * G), ds = (gated ? (uint32_t)(P1.s - P0.s) : 32u * (uint32_t)G) - 32u * (uint32_t)G;
#pragma unroll 1
    for (int c = 0; c < 4 * G; c += 64)
        if (c + lane < 4 * G) copy16(rw, tbl + 16 * c, ts + 16u * (uint32_t)(c + lane) + (c + lane >= 2 * G ? ds : 0u));
    asm volatile("" ::: "memory");

    f32x4_t acc[MP][4];
#pragma unroll
    for (int p = 0; p < MP; ++p)
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[p][f] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    dma_wait_barrier<0>();
    const int nch = (G + 15) / 16;
    for (int ch = 0; ch < nch; ++ch) {
        if (ch + 1 < nch) issue_a(ch + 1);         // (every wave is done with the chunk that was there)
        asm volatile("" ::: "memory");
        const uint8_t* const buf = smem + (ch & 1) * kMxBuf<MP>;
        // groups past the row's end: zeros (another row's byte might be a NaN)
        const int left = G - (16 * ch + 4 * g);
        const uint32_t in = left >= 4 ? 0xFFFFFFFFu : left >= 2 ? 0xFFFFu : 0u;
        uint32_t xe[MP];       // the lane's four scales of its pairs' rows
#pragma unroll
        for (int p = 0; p < MP; ++p) {
            const u32x2_t v = *reinterpret_cast<const u32x2_t*>(buf + kMxA<MP> + p * 512 + l16 * 32 + 8 * g);
            xe[p] = v[0] | (v[1] << 16);
        }
        auto half = [&](Half& q, auto h_) __attribute__((always_inline)) {
            constexpr int h = decltype(h_)::value;
            uint32_t ws[2];
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                const uint16_t* const t =
                    reinterpret_cast<const uint16_t*>(tbl + (32 * h + 8 * (l16 >> 2) + 4 * f + (l16 & 3)) * G + 16 * ch + 4 * g);
                ws[f] = (t[0] | ((uint32_t)t[1] << 16)) & in;
                mx_transpose(q.w[f]);
            }
            auto step = [&](auto t_) __attribute__((always_inline)) {
                constexpr int t = decltype(t_)::value;
#pragma unroll
                for (int p = 0; p < MP; ++p) {
                    const mx_u32x4 xv = *reinterpret_cast<const mx_u32x4*>(buf + p * 4096 + l16 * 256 + 16 * ((4 * g + t) ^ l16));
#pragma unroll
                    for (int f = 0; f < 2; ++f) acc[p][2 * h + f] = mx_mfma<t>(q.w[f][t], ws[f], xv, xe[p], acc[p][2 * h + f]);
                }
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        };
        half(qa, std::integral_constant<int, 0>{});
        issue(ch + 1, qa, 0);
        __builtin_amdgcn_sched_barrier(0);
        half(qb, std::integral_constant<int, 1>{});
        if (ch + 1 == nch) break;
        issue(ch + 1, qb, dw);
        __builtin_amdgcn_sched_barrier(0);
        // the next chunk of A has landed (the weights were issued after its copies), and every wave is done
        // reading this one
        thin_wait_barrier<16>();
    }

    // ---- epilogue: lane (g, l16) has rows 8 g .. 8 g + 7 of each 32-row group for pair l16
    auto bias8 = [&](const u32x4_t& w, float (&b)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = bf2f((i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu);
    };
    if (c0 >= N) return;                           // (a wave past the last rows)
    const float nan = absent_nan();
    if constexpr (KIND == 0) {
        const bool clamped = a.act == BRX_ACT_SWIGLU_CLAMPED;
        const float alpha = clamped ? a.alpha : 1.0f;
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
                    hv[i] = mx_act(a, gated, clamped, alpha, acc[p][2 * h + (i >> 2)][i & 3] + b0[i],
                                   acc[p][2 + (i >> 2)][i & 3] + b1[i], absent);
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
        int row[MP];
#pragma unroll
        for (int p = 0; p < MP; ++p)
            row[p] = p * 16 + l16 >= rows ? -1 : KIND == 2 || pd[p] < a.P ? pair_row(a, pd[p]) : pd[p];
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
                if (row[p] < 0) continue;
                if (KIND == 1 && m.y32) {              // uniform
                    f32x4_t* const to = reinterpret_cast<f32x4_t*>(m.y32 + (int64_t)row[p] * N + col);
                    to[0] = f32x4_t{y[0], y[1], y[2], y[3]};
                    to[1] = f32x4_t{y[4], y[5], y[6], y[7]};
                }
                if ((KIND == 2 || m.y16) && row[p] < a.yrows)    // (no bf16 rows of the shared pairs)
                    *reinterpret_cast<u32x4_t*>(m.y16 + (int64_t)row[p] * N + col) =
                        u32x4_t{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3]), pk_bf16(y[4], y[5]), pk_bf16(y[6], y[7])};
            }
        }
    }
}

// MPX: the call's tallest tiles, in 16 pairs (a launch of low tiles takes fewer registers).
template <int KIND, int MPX>
__global__ __launch_bounds__(kMxThreads) __attribute__((amdgpu_waves_per_eu(MPX == 5 ? 2 : MPX == 2 ? 3 : 4)))
void k_mx_gemm(FwdArgs a, MxArgs m) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    prefetch_args(a);
    const int blk = blockIdx.x;
    const int loc = blk / kXcd;
    const int of = loc / (m.group * m.ntn), in = loc % (m.group * m.ntn);
    const int nt = in / m.group;
    const int mt = (of * kXcd + blk % kXcd) * m.group + in % m.group;
    const int total = m.tile_start[m.E_ext];
    const int4 ti = m.tinfo[mt];
    if (mt >= total) return;
    const int e = ti.x, m0 = ti.y, rows = ti.z;
    const Layout& L = e >= a.E ? a.lay_sh : a.lay;
    const int pj = KIND == 0 ? 0 : KIND == 1 ? 2 : m.proj;
    const int N = pj == 0 ? L.p[0].n_out : pj == 1 ? L.p[1].n_out : L.p[2].n_out;
    if (nt * kMxWaves * (KIND == 0 && a.act != BRX_ACT_SILU_MLP ? kMxRows / 2 : kMxRows) >= N) return;
    if (MPX == 1 || rows <= 16) mx_tile<KIND, 1>(a, m, smem, e, m0, rows, ti.w, nt);
    else if (MPX == 2 || rows <= 32) mx_tile<KIND, 2>(a, m, smem, e, m0, rows, ti.w, nt);
    else if (rows <= 64) mx_tile<KIND, 4>(a, m, smem, e, m0, rows, ti.w, nt);
    else mx_tile<KIND, 5>(a, m, smem, e, m0, rows, ti.w, nt);
}

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// Pairs of the call's tallest M tile: what the mean expert's pairs fit in (tiles of 128 pairs leave one wave a
// SIMD its registers: a 2048-token layer 195 us, 184 with 64).
int mx_tile_rows(int64_t pairs, int64_t experts) {
    return pairs <= 8 * experts ? 16 : pairs <= 24 * experts ? 32 : 64;
}
// Rows past a tile of 64 that join it (tiles of up to 80): the mean expert's pairs are near 64, 128, ..., and the
// few that pass it would read the expert's weights once more.
int mx_slack(int tile) { return tile == 64 ? 16 : 0; }
// Consecutive M tiles whose runs of columns an XCD takes in turn: an expert's tall tiles then read its weights
// from one L2 (a 2048-token layer 183 us one by one, 180 by two, 179 by four).
int mx_group(int tile) { return tile == 64 ? 4 : 1; }

struct MxWs {
    uint8_t *xq, *xs, *hq, *hs;
    int32_t *order, *offsets, *tile_start;
    int4* tinfo;
    float* y32;
    int mt_pad, tile, group, Imax;
    size_t bytes;
};

// The scratch of a call over P routed pairs (and T shared ones) of T token rows; `layer`: a whole layer
// (else an expert product, whose activations and rows are the caller's).
MxWs carve(const FwdArgs& a, bool layer, void* ws) {
    const int T_sh = a.auto_shared ? a.T : 0, P_ext = a.P + T_sh, E_ext = a.E + (a.shared ? 1 : 0);
    MxWs w{};
    w.Imax = a.shared && a.I_sh > a.I ? a.I_sh : a.I;
    w.tile = mx_tile_rows(P_ext, E_ext);
    w.group = mx_group(w.tile);
    const int step = kXcd * w.group;
    w.mt_pad = ((P_ext + w.tile - 1) / w.tile + (E_ext < P_ext ? E_ext : P_ext) + step - 1) / step * step;
    char* b = reinterpret_cast<char*>(ws);
    size_t off = 0;
    auto take = [&](size_t n) { char* p = b + off; off = align256(off + n); return p; };
    w.order = (int32_t*)take(sizeof(int32_t) * P_ext);
    w.offsets = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
    w.tile_start = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
    w.tinfo = (int4*)take(sizeof(int4) * (P_ext / 16 + E_ext + 4 * kXcd));   // (any tile height's)
    if (layer) {
        w.xq = (uint8_t*)take((size_t)a.T * (a.H / 2));
        w.xs = (uint8_t*)take((size_t)a.T * (a.H / 32));
        w.hq = (uint8_t*)take((size_t)P_ext * (w.Imax / 2));
        w.hs = (uint8_t*)take((size_t)P_ext * (w.Imax / 32));
        w.y32 = (float*)take(a.out ? (size_t)P_ext * a.H * 4 : 0);             // (rows alone go where the caller has them)
    }
    w.bytes = off;
    return w;
}

template <int KIND, int MPX>
hipError_t launch_tiles(const FwdArgs& a, MxArgs m, const MxWs& w, int K, int N, hipStream_t s) {
    const int per = kMxWaves * (KIND == 0 && a.act != BRX_ACT_SILU_MLP ? kMxRows / 2 : kMxRows);
    m.ntn = (N + per - 1) / per;
    hipLaunchKernelGGL((k_mx_gemm<KIND, MPX>), dim3(w.mt_pad * m.ntn), dim3(kMxThreads), 2 * kMxBuf<MPX> + mx_table(K), s, a, m);
    return hipGetLastError();
}

template <int KIND>
hipError_t launch_gemm(const FwdArgs& a, const MxArgs& m, const MxWs& w, int K, int N, hipStream_t s) {
    switch (w.tile) {
        case 16: return launch_tiles<KIND, 1>(a, m, w, K, N, s);
        case 32: return launch_tiles<KIND, 2>(a, m, w, K, N, s);
        default: return launch_tiles<KIND, 5>(a, m, w, K, N, s);
    }
}

MxArgs gemm_args(const FwdArgs& a, const MxWs& w) {
    MxArgs m{};
    m.order = w.order;
    m.tile_start = w.tile_start;
    m.group = w.group;
    m.tinfo = w.tinfo;
    m.E_ext = a.E + (a.shared ? 1 : 0);
    return m;
}

hipError_t bucket(const FwdArgs& a, const MxWs& w, hipStream_t s) {
    return launch_bucket(a.pexp, a.P, a.E, a.E + (a.shared ? 1 : 0), a.auto_shared ? a.T : 0, w.tile, a.g2s, a.capacity,
                         a.host != nullptr, a.err, w.order, w.offsets, w.tile_start, w.tinfo, s, mx_slack(w.tile));
}

// The first launch of a layer: blocks [0, E_ext) bucket the pairs, the others round x [n8 runs of 8 values] to
// MXFP4, a group per four neighbouring lanes. (Two launches: 3 us more a 64-token layer.)
template <int PER>
__global__ __launch_bounds__(kBucketThreads) void k_mx_prepare(const int32_t* __restrict__ pexp, int P, int E, int E_ext,
                                                               int T_sh, int lbm, int slack,
                                                               const int32_t* __restrict__ g2s,
                                                               int capacity, int host, int32_t* __restrict__ err,
                                                               int32_t* __restrict__ order,
                                                               int32_t* __restrict__ offsets,
                                                               int32_t* __restrict__ tile_start,
                                                               int4* __restrict__ tinfo, int lcap,
                                                               const uint16_t* __restrict__ x, int64_t n8,
                                                               uint8_t* __restrict__ xq, uint8_t* __restrict__ xs) {
    if ((int)blockIdx.x < E_ext) {
        bucket_block<PER>(blockIdx.x, pexp, P, E, E_ext, T_sh, lbm, slack, g2s, capacity, host, err, order, offsets,
                          tile_start, tinfo, lcap);
        return;
    }
    const int64_t i = (int64_t)(blockIdx.x - E_ext) * kBucketThreads + threadIdx.x;
    if (i >= n8) return;                           // (whole groups)
    const u32x4_t q = *reinterpret_cast<const u32x4_t*>(x + 8 * i);
    float v[8];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        v[k] = bf2f((k & 1) ? q[k >> 1] >> 16 : q[k >> 1] & 0xFFFFu);
        top = max(top, mx_mag(v[k]));
    }
    top = max(top, dpp_u<0xB1>(top));
    top = max(top, dpp_u<0x4E>(top));
    const uint32_t sb = mx_scale(top);
    reinterpret_cast<uint32_t*>(xq)[i] = mx_codes(v, sb);
    if ((i & 3) == 0) xs[i >> 2] = (uint8_t)sb;
}

// out[t] = sum_j w[t, j] y[t, j] (+ sg[t] y_shared[t]) over fp32 rows, j in order, four columns a thread.
__global__ __launch_bounds__(kMxThreads) void k_mx_combine(const float* __restrict__ y, const float* __restrict__ y_shared,
                                                           const float* __restrict__ w, const float* __restrict__ sg,
                                                           int k, int H, uint16_t* __restrict__ out) {
    const int t = blockIdx.y, n = (blockIdx.x * kMxThreads + threadIdx.x) * 4;
    if (n >= H) return;
    constexpr int U = 8;                           // rows in flight
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    f32x4_t sh{0.f, 0.f, 0.f, 0.f};
    if (y_shared) sh = *reinterpret_cast<const f32x4_t*>(y_shared + (int64_t)t * H + n);
    for (int j0 = 0; j0 < k; j0 += U) {
        f32x4_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const f32x4_t*>(y + ((int64_t)t * k + min(j0 + u, k - 1)) * H + n);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (j0 + u >= k) break;                // uniform
            const float wj = w[t * k + j0 + u];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(wj, v[u][i], o[i]);
        }
    }
    if (y_shared) {
        const float g = sg[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = fmaf(g, sh[i], o[i]);
    }
    *reinterpret_cast<u32x2_t*>(out + (int64_t)t * H + n) =
        u32x2_t{f2bf(o[0]) | (f2bf(o[1]) << 16), f2bf(o[2]) | (f2bf(o[3]) << 16)};
}

hipError_t prepare(const FwdArgs& a, const MxWs& w, hipStream_t s) {
    const int E_ext = a.E + (a.shared ? 1 : 0), T_sh = a.auto_shared ? a.T : 0;
    const int lcap = bucket_list(a.P + T_sh);
    const int64_t n8 = (int64_t)a.T * (a.H / 8);
    const dim3 grid((unsigned)(E_ext + (n8 + kBucketThreads - 1) / kBucketThreads));
#define BRX_PREPARE(PER) hipLaunchKernelGGL(k_mx_prepare<PER>, grid, dim3(kBucketThreads), sizeof(int32_t) * (E_ext + lcap), s, \
                                            a.pexp, a.P, a.E, E_ext, T_sh, __builtin_ctz(w.tile), mx_slack(w.tile), a.g2s, a.capacity, \
                                            a.host != nullptr ? 1 : 0, a.err, w.order, w.offsets, w.tile_start, w.tinfo, lcap, \
                                            a.x, n8, w.xq, w.xs)
    switch (bucket_per(a.P + T_sh)) {
        case 2: BRX_PREPARE(2); break;
        case 4: BRX_PREPARE(4); break;
        default: BRX_PREPARE(16);
    }
#undef BRX_PREPARE
    return hipGetLastError();
}

}  // namespace

// The few-pair kernels have a block for every run of an expert's rows: they win while launches and round trips
// set the time. The line past 8 tokens is the pairs times an expert's bytes (what the pairs could read), these
// kernels against the grouped GEMM, three layers in turn: 2048 x 768, top-8, 9 tokens (180 MB) 34.8 / 38.0 us, 12
// (241 MB) 38.8 / 41.8, 24 (477 MB) 44.0 / 44.0; 2048 x 512, 256 experts and a shared one, 12 tokens (160 MB) 31.9 /
// 33.3, 16 (214 MB) 40.4 / 40.2; 2048 x 1024, top-8, 9 tokens (241 MB) 47.3 / 47.2; a 1024 x 256 MLP, 33 tokens (19
// MB) 14.2 / 18.0. Up to 8 tokens they lose only past that: 2880 x 2880, top-4, 7 tokens (371 MB) 92.2 / 95.5, 8
// (424 MB) 103.3 / 99.8. Up to 128 pairs every block plans the step (bucketed first: the MLP 16.2, 12 tokens of 2048
// x 768 40.8).
MxPath mx_path(const FwdArgs& a) {
    if (a.T <= kMxFewTokens && a.P <= kMxFewPairs) return kMxFew;
    if (a.T > kMxMidTokens || a.P > kMxMidPairs || a.P * a.lay.bytes > 260 * 1000 * 1000) return kMxMany;
    return a.P <= kMxPlanPairs ? kMxFew : kMxMid;
}

size_t mx_workspace_bytes(const FwdArgs& a, bool layer, MxPath path) {
    if (!layer && a.P <= kMxFewPairs) return 0;
    return layer && path != kMxMany ? mx_few_workspace_bytes(a, path == kMxMid) : carve(a, layer, nullptr).bytes;
}

hipError_t launch_mx_combine(const float* y, const float* y_shared, const float* w, const float* sg, int T, int k, int H,
                             uint16_t* out, hipStream_t s) {
    hipLaunchKernelGGL(k_mx_combine, dim3((H / 4 + kMxThreads - 1) / kMxThreads, T), dim3(kMxThreads), 0, s, y, y_shared, w,
                       sg, k, H, out);
    return hipGetLastError();
}

hipError_t launch_mx_layer(const FwdArgs& a, MxPath path, float* rows32, void* ws, hipStream_t s) {
    if (path != kMxMany) return launch_mx_few_layer(a, path == kMxMid, rows32, ws, s);
    const MxWs w = carve(a, true, ws);
    hipError_t e = prepare(a, w, s);
    if (e != hipSuccess) return e;
    MxArgs m = gemm_args(a, w);
    m.xq = w.xq;
    m.xs = w.xs;
    m.hq = w.hq;
    m.hs = w.hs;
    m.hstride = w.Imax;
    m.y16 = a.yun;
    m.y32 = rows32 ? rows32 : a.out ? w.y32 : nullptr;
    if ((e = launch_gemm<0>(a, m, w, a.H, w.Imax, s)) != hipSuccess) return e;
    if ((e = launch_gemm<1>(a, m, w, w.Imax, a.H, s)) != hipSuccess) return e;
    if (!a.out) return hipSuccess;
    return launch_mx_combine(w.y32, a.auto_shared ? w.y32 + (int64_t)a.P * a.H : nullptr, a.w, a.sgate, a.T, a.k, a.H, a.out, s);
}

hipError_t launch_mx_product(const FwdArgs& a, const uint8_t* codes, const uint8_t* scales, int proj, void* ws,
                             hipStream_t s) {
    // Past 64 pairs the one launch wins while the pairs' projections are at most so many bytes (against the two):
    // 2048 x 768, 72 pairs (60 MB) 13.5 / 15.9 us, 96 (80 MB) 16.2 / 16.3, 128 (107 MB) 17.3 / 16.9; 2048 x 512, 72
    // pairs of 256 experts (40 MB) 10.0 / 15.3, 128 (71 MB) 14.5 / 16.4; 1024 x 256, 128 (18 MB) 5.7 / 10.2; 2880 x
    // 2880, 68 (300 MB) 62.4 / 59.1.
    if (a.P <= kMxFewPairs || (a.P <= kMxPlanPairs && (int64_t)a.P * a.I * a.H / 32 * 17 <= 75 * 1000 * 1000))
        return launch_mx_few_product(a, codes, scales, proj, s);
    const MxWs w = carve(a, false, ws);
    hipError_t e = bucket(a, w, s);
    if (e != hipSuccess) return e;
    MxArgs m = gemm_args(a, w);
    m.xq = codes;
    m.xs = scales;
    m.y16 = a.yun;
    m.proj = proj;
    return launch_gemm<2>(a, m, w, proj == 2 ? w.Imax : a.H, proj == 2 ? a.H : w.Imax, s);
}

}  // namespace brx
