// MXFP4 products of few (token, expert) pairs: a decode step's expert layer in two launches, a short
// list's expert product in one.
//
//   k_mx_few_up    grid (32 features, entry): the entry's token rows rounded to MXFP4 in LDS, the gate and up
//                  rows of its expert, act() and h in MXFP4; also writes the entry table.
//   k_mx_few_rows  <true>: 16 output columns of every entry's down rows and, in the epilogue, their weighted
//                  sum (grid H / 16). <false>: one projection's rows for a list of pairs (grid
//                  (n_out / 16, entries / 8)).
// An entry is an expert with up to 16 of the step's pairs, in order of its first pair; the shared
// expert's comes last. The arithmetic is k_mx_gemm's to the bit: the same 512-K chunks in the same order, the
// same roundings.
//
// What bounds it: the weights are read once, and a wave requests the whole of its 16 rows (up to 4 chunks,
// 16 KB; wider rows three chunks at a time) before it multiplies anything, so a call is a few dependent round
// trips -- the routing, the table, the weights (of rows wider than four chunks once more: the second three are
// requested behind the first three's products) -- and little else. One token of the gpt-oss shape (53 MB) takes
// 12.9 + 7.1 us (2.7 TB/s), 8 tokens of 256 experts and a shared one (59 MB) 14.4 + 9.2. The gate and up rows are
// split by entry, the down rows are not (a block has every entry's 16 columns), so that the sum over a token's
// experts is in one block's LDS and needs neither atomics nor a third launch.
#include <type_traits>

#include "mx_common.h"
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kUpWaves = 4;
constexpr int kRowWaves = 8;

// Pairs of an entry, and what the second launch reads of it.
struct MxEntry {
    int32_t slot, n;
    int32_t pair[16];
};
struct MxTable {
    int32_t n, pad[3];
    MxEntry ent[kMxMidPairs + kMxMidTokens];
};

// One entry as a wave holds it: its expert, slot code, pairs (column c's pair in lanes c, c + 16, ..; the last
// one again past the end), and the step's number of entries. Returns false past the last entry.
struct MxPlan {
    int e, slot, n, pair, entries;
};
constexpr int kIdBits = 10;                        // expert ids, the shared one's among them, are at most 512
constexpr int kSlotRegs = 8;                       // the slot table of up to 512 experts, 64 a register
template <int R>                                   // pairs a lane: up to 64 R in all
__device__ __forceinline__ bool mx_plan(const FwdArgs& a, int u, int32_t* s_pair, MxPlan& o) {
    const int lane = threadIdx.x & 63;
    const int P = a.P, emax = a.shared ? a.E : a.E - 1;
    // the slot table comes with the routing, not a round trip after it
    int e[R];
#pragma unroll
    for (int r = 0; r < R; ++r) e[r] = a.pexp[min(lane + 64 * r, P - 1)];
    int slots[kSlotRegs];
#pragma unroll
    for (int i = 0; i < kSlotRegs; ++i) slots[i] = 64 * i < a.E ? a.g2s[min(lane + 64 * i, a.E - 1)] : 0;
    // same[r][c]: the pairs of register c that have the expert of the lane's pair r, found an id bit at a time
    uint64_t same[R][R], live[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        e[r] = min(max(e[r], 0), emax);
        live[r] = __ballot(lane + 64 * r < P);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < R; ++c) same[r][c] = live[c];
#pragma unroll
    for (int i = 0; i < kIdBits; ++i) {
        uint64_t one[R];
#pragma unroll
        for (int c = 0; c < R; ++c) one[c] = __ballot((e[c] >> i) & 1);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < R; ++c) same[r][c] &= (e[r] >> i) & 1 ? one[c] : ~one[c];
    }
    // an expert's 1st, 17th, .. pair leads an entry
    const uint64_t below = (1ull << lane) - 1ull;
    int rank[R];
    uint64_t leads[R];
    int routed = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        rank[r] = __popcll(same[r][r] & below);
#pragma unroll
        for (int c = 0; c < r; ++c) rank[r] += __popcll(same[r][c]);
        leads[r] = __ballot(lane + 64 * r < P && (rank[r] & 15) == 0);
        routed += __popcll(leads[r]);
    }
    o.entries = routed + (a.auto_shared ? (a.T + 15) / 16 : 0);
    if (u >= o.entries) return false;
    if (u >= routed) {                             // 16 tokens of the shared expert
        const int t0 = 16 * (u - routed);
        o.e = a.E;
        o.slot = -1;
        o.n = min(16, a.T - t0);
        o.pair = P + t0 + min(lane & 15, o.n - 1);
        return true;
    }
    int r0 = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int n = __popcll(leads[r]);
        if (u >= 0 && u < n) {                     // uniform
            const int lead = __builtin_ctzll(__ballot(((leads[r] >> lane) & 1) && __popcll(leads[r] & below) == u));
            o.e = __builtin_amdgcn_readlane(e[r], lead);
            r0 = __builtin_amdgcn_readlane(rank[r], lead);
        }
        u -= n;
    }
    o.n = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool in = lane + 64 * r < P && e[r] == o.e && rank[r] >= r0 && rank[r] < r0 + 16;
        o.n += __popcll(__ballot(in));
        if (in) s_pair[rank[r] - r0] = lane + 64 * r;      // (the wave's own words)
    }
    __builtin_amdgcn_wave_barrier();
    o.pair = s_pair[min(lane & 15, o.n - 1)];
    int v = 0;
#pragma unroll
    for (int i = 0; i < kSlotRegs; ++i)
        if ((o.e >> 6) == i) v = __builtin_amdgcn_readlane(slots[i], o.e & 63);
    o.slot = o.e < a.E ? slot_code(a, o.e, v) : -1;
    if (o.slot == kAbsentCode && lane == 0) note_absent(a, o.e);
    return true;
}

// NB chunks of 16 weight rows as a wave loads them: the codes as k_mx_gemm, and each row's 16 scale bytes by
// four neighbouring lanes.
template <int NB>
struct FewW {
    mx_u32x4 w[NB][4];
    uint32_t s[NB];
};
// w0 and s0: byte offsets of the fragment's codes row and scales row 0; row m of the fragment is `step` rows
// apart in blocks of four (8: rows 8 (m / 4) + m % 4; 4: the rows in order).
template <int NB>
__device__ __forceinline__ void few_load(__amdgpu_buffer_rsrc_t r, uint32_t w0, uint32_t s0, int step, int K, int ch0,
                                         FewW<NB>& o) {
    const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15, G = K / 32;
    const uint32_t row = (uint32_t)(K / 2);
    const uint32_t vw = w0 + (uint32_t)(step * (l16 >> 2)) * row;
    const uint32_t vs = s0 + (uint32_t)(step * (lane >> 4) + ((lane >> 2) & 3)) * (uint32_t)G;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int ch = ch0 + j;
        o.s[j] = __builtin_amdgcn_raw_buffer_load_b32(r, vs + (uint32_t)min(16 * ch + 4 * (lane & 3), G - 4), 0, 0);
        const uint32_t v = vw + 16u * (uint32_t)min(16 * ch + 4 * g + (l16 & 3), G - 1);
#pragma unroll
        for (int t = 0; t < 4; ++t) o.w[j][t] = __builtin_amdgcn_raw_buffer_load_b128(r, v, t * row, 0);
    }
}
// acc += the fragment's chunk ch times X's (pieces xv of this lane's K groups, their scales xe).
__device__ __forceinline__ void few_mul(mx_u32x4 (&w)[4], uint32_t s, int ch, int K, const mx_u32x4 (&xv)[4], uint32_t xe,
                                        f32x4_t& acc) {
    const int lane = threadIdx.x & 63, g = lane >> 4, G = K / 32;
    // lane (g, m) takes word g of row m's scales from lane 4 m + g; its first group is byte `off` of the word,
    // and groups past the row's end are zeros
    s = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (4 * (lane & 15) + g), (int)s);
    const int first = 16 * ch + 4 * g, off = max(first - (G - 4), 0);
    const uint32_t ws = (s >> ((8 * off) & 31)) & (uint32_t)((first - G) >> 31);
    mx_transpose(w);
    acc = mx_mfma<0>(w[0], ws, xv[0], xe, acc);
    acc = mx_mfma<1>(w[1], ws, xv[1], xe, acc);
    acc = mx_mfma<2>(w[2], ws, xv[2], xe, acc);
    acc = mx_mfma<3>(w[3], ws, xv[3], xe, acc);
}

// LDS of a staged token row of nch chunks: an odd number of 16-byte pieces, an odd number of words of scales.
__host__ __device__ inline int few_code_pitch(int nch) { return nch * 256 + 16; }
__host__ __device__ inline int few_scale_pitch(int nch) { return nch * 16 + 4; }

// R = 0: the entries are the tiles of 16 pairs that k_bucket made; else every block plans the step itself, R pairs
// a lane.
template <int NB, int R>
__global__ __launch_bounds__(64 * kUpWaves) void k_mx_few_up(FwdArgs a, MxArgs m, MxTable* __restrict__ table) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    __shared__ __attribute__((aligned(16))) f32x4_t red[4][64];
    __shared__ int32_t s_pair[kUpWaves][16];
    prefetch_args(a);
    prefetch_args(m);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    MxPlan pl;
    if constexpr (R == 0) {
        const int u = blockIdx.y;
        pl.entries = m.tile_start[m.E_ext];
        const int4 ti = m.tinfo[u];                // (the list is at least as long as the grid)
        if (u >= pl.entries) return;
        pl.e = __builtin_amdgcn_readfirstlane(ti.x);
        pl.n = __builtin_amdgcn_readfirstlane(ti.z);
        pl.slot = pl.e >= a.E ? -1 : __builtin_amdgcn_readfirstlane(ti.w);
        pl.pair = m.order[ti.y + min(lane & 15, pl.n - 1)];
    } else if (!mx_plan<R>(a, blockIdx.y, s_pair[wv], pl)) {
        return;
    }
    const bool gated = a.act != BRX_ACT_SILU_MLP, sh = pl.e >= a.E;
    const Layout& L = sh ? a.lay_sh : a.lay;
    const int K = a.H, N = L.p[0].n_out, G = K / 32, nch = (G + 15) / 16;
    const int c0 = blockIdx.x * (gated ? 32 : 64);
    if (blockIdx.x == 0 && wv == 0) {
        MxEntry& en = table->ent[blockIdx.y];
        if (lane == 0) {
            en.slot = pl.slot;
            en.n = pl.n;
            if (blockIdx.y == 0) table->n = pl.entries;
        }
        if (lane < 16) en.pair[lane] = pl.pair;
    }
    if (c0 >= N) return;
    const uint8_t* base = sh ? a.shared : code_base(a, clamp_code(a, pl.slot));
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(base, (uint32_t)L.bytes);
    // wave f: fragment f (0, 1: the first 32 rows' blocks of four in turn; 2, 3: the up rows, or the next 32)
    const bool second = wv >= 2;
    const Proj& P = gated && second ? L.p[1] : L.p[0];
    const int r0 = c0 + (gated || !second ? 0 : 32) + 4 * (wv & 1);
    FewW<NB> q;
    // (x first: its rounding goes on while the weights come)
    const int token = pl.pair >= a.P ? pl.pair - a.P : pair_tok(a, pl.pair);
    if (lane < 16) s_pair[wv][lane] = token;
    __builtin_amdgcn_wave_barrier();
    const int pieces = pl.n * (K / 8);             // 8 values each
    const int PC = few_code_pitch(nch), PS = few_scale_pitch(nch);
    uint8_t* const sc = smem + pl.n * PC;
    constexpr int U = 4;
    u32x4_t xr[U];
    auto x_at = [&](int i) __attribute__((always_inline)) {
        const int r = min(i, pieces - 1) / (K / 8), c = min(i, pieces - 1) - r * (K / 8);
        return *reinterpret_cast<const u32x4_t*>(a.x + (int64_t)s_pair[wv][r] * K + 8 * c);
    };
    auto x_put = [&](int i, const u32x4_t& v4) __attribute__((always_inline)) {
        const int r = min(i, pieces - 1) / (K / 8), c = min(i, pieces - 1) - r * (K / 8);
        float v[8];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            v[k] = bf2f((k & 1) ? v4[k >> 1] >> 16 : v4[k >> 1] & 0xFFFFu);
            top = max(top, mx_mag(v[k]));
        }
        top = max(top, dpp_u<0xB1>(top));
        top = max(top, dpp_u<0x4E>(top));
        const uint32_t sb = mx_scale(top), o = mx_codes(v, sb);
        if (i < pieces) {
            *reinterpret_cast<uint32_t*>(smem + r * PC + 4 * c) = o;
            if ((c & 3) == 0) sc[r * PS + c / 4] = (uint8_t)sb;
        }
    };
#pragma unroll
    for (int k = 0; k < U; ++k) xr[k] = x_at(tid + k * 64 * kUpWaves);
    asm volatile("" ::: "memory");
    const uint32_t w0 = (uint32_t)P.w + (uint32_t)r0 * (uint32_t)(K / 2), s0 = (uint32_t)P.s + (uint32_t)r0 * (uint32_t)G;
    few_load<NB>(rw, w0, s0, 8, K, 0, q);
    // the biases of this block's outputs (used by the first wave)
    u32x4_t bias[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        bias[h] = u32x4_t{0u, 0u, 0u, 0u};
        const Proj& B = gated && h ? L.p[1] : L.p[0];
        if (B.bias >= 0)
            bias[h] = __builtin_amdgcn_raw_buffer_load_b128(rw, (uint32_t)(B.bias + 2 * (c0 + (gated || !h ? 0 : 32) + 8 * g)), 0, 0);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) x_put(tid + k * 64 * kUpWaves, xr[k]);
    for (int i0 = U * 64 * kUpWaves; i0 < pieces; i0 += U * 64 * kUpWaves) {
#pragma unroll
        for (int k = 0; k < U; ++k) xr[k] = x_at(i0 + tid + k * 64 * kUpWaves);
#pragma unroll
        for (int k = 0; k < U; ++k) x_put(i0 + tid + k * 64 * kUpWaves, xr[k]);
    }
    // zeros past the rows' ends, up to whole chunks
    const int padp = 16 * nch - G;
    for (int i = tid; i < pl.n * padp; i += 64 * kUpWaves) {
        const int r = i / padp, c = G + i % padp;
        *reinterpret_cast<u32x4_t*>(smem + r * PC + 16 * c) = u32x4_t{0u, 0u, 0u, 0u};
        sc[r * PS + c] = 0;
    }
    lds_barrier();
    f32x4_t acc{0.f, 0.f, 0.f, 0.f};
    const int xrow = min(l16, pl.n - 1);
    for (int ch0 = 0; ch0 < nch; ch0 += NB) {
        if (ch0) few_load<NB>(rw, w0, s0, 8, K, ch0, q);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            if (ch0 + j < nch) {                   // uniform
                mx_u32x4 xv[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    xv[t] = *reinterpret_cast<const mx_u32x4*>(smem + xrow * PC + (ch0 + j) * 256 + 16 * (4 * g + t));
                const uint32_t xe = *reinterpret_cast<const uint32_t*>(sc + xrow * PS + (ch0 + j) * 16 + 4 * g);
                few_mul(q.w[j], q.s[j], ch0 + j, K, xv, xe, acc);
            }
        }
    }
    red[wv][lane] = acc;
    lds_barrier();
    if (wv != 0) return;
    // lane (g, n): columns 8 g .. 8 g + 7 of each 32 for pair n, as in k_mx_gemm's epilogue
    const f32x4_t d[4] = {red[0][lane], red[1][lane], red[2][lane], red[3][lane]};
    const bool clamped = a.act == BRX_ACT_SWIGLU_CLAMPED;
    const float alpha = clamped ? a.alpha : 1.0f;
    float b[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) b[h][i] = bf2f((i & 1) ? bias[h][i >> 1] >> 16 : bias[h][i >> 1] & 0xFFFFu);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (gated && h == 1) break;
        float hv[8];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            hv[i] = mx_act(a, gated, clamped, alpha, d[2 * h + (i >> 2)][i & 3] + b[h][i], d[2 + (i >> 2)][i & 3] + b[1][i],
                           pl.slot == kAbsentCode);
            top = max(top, mx_mag(hv[i]));
        }
        top = max(top, lane_xor16(top));
        top = max(top, lane_xor32(top));
        const uint32_t sb = mx_scale(top);
        if (l16 < pl.n) {
            const int64_t row = pl.pair;
            const int col = c0 + 32 * h + 8 * g;
            *reinterpret_cast<uint32_t*>(m.hq + row * (m.hstride / 2) + col / 2) = mx_codes(hv, sb);
            if (g == 0) m.hs[row * (m.hstride / 32) + col / 32] = (uint8_t)sb;
        }
    }
}

// DOWN: the second launch of a layer, over the entry table, NE entries of NB chunks a wave at once; else one
// projection's rows of a list that every block plans, R pairs a lane.
template <bool DOWN, int NB, int NE, int R = 1>
__global__ __launch_bounds__(64 * kRowWaves) void k_mx_few_rows(FwdArgs a, MxArgs m, const MxTable* __restrict__ table) {
    __shared__ __attribute__((aligned(16))) float ys[DOWN ? kMxMidPairs + kMxMidTokens : 1][16];
    __shared__ int32_t s_pair[kRowWaves][16];
    prefetch_args(a);
    prefetch_args(m);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, l16 = lane & 15;
    const int c0 = blockIdx.x * 16;
    int entries = 1;
    MxPlan pl[NE];
    auto entry = [&](int u, MxPlan& o) __attribute__((always_inline)) {       // (u may be past the last: any)
        const MxEntry& en = table->ent[min(u, kMxMidPairs + kMxMidTokens - 1)];
        o.slot = en.slot;
        o.n = en.n;
        o.pair = en.pair[l16];
    };
    if constexpr (DOWN) {
        entries = table->n;
#pragma unroll
        for (int v = 0; v < NE; ++v) entry(wv + kRowWaves * v, pl[v]);
        entries = __builtin_amdgcn_readfirstlane(entries);
    } else {
        if (!mx_plan<R>(a, blockIdx.y * kRowWaves + wv, s_pair[wv], pl[0])) return;
    }
    for (int u0 = DOWN ? wv : 0; u0 < entries; u0 += kRowWaves * NE) {
        FewW<NB> q[NE];
        mx_u32x4 xv[NE][NB][4];
        uint32_t xe[NE][NB];
        u32x2_t bias[NE];
        f32x4_t acc[NE];
        int Ks[NE];
        bool absent[NE];
        auto load = [&](int v, int ch0) __attribute__((always_inline)) {
            const int slot = __builtin_amdgcn_readfirstlane(pl[v].slot);
            const bool sh = DOWN ? slot == -1 : pl[v].e >= a.E;
            const Layout& L = sh ? a.lay_sh : a.lay;
            const Proj P = DOWN ? L.p[2] : m.proj == 0 ? L.p[0] : m.proj == 1 ? L.p[1] : L.p[2];
            const uint8_t* base = sh ? a.shared : code_base(a, clamp_code(a, slot));
            const __amdgpu_buffer_rsrc_t rw = make_rsrc(base, (uint32_t)L.bytes);
            const int K = P.n_in, G = K / 32;
            Ks[v] = K;
            absent[v] = slot == kAbsentCode;
            few_load<NB>(rw, (uint32_t)P.w + (uint32_t)c0 * (uint32_t)(K / 2), (uint32_t)P.s + (uint32_t)c0 * (uint32_t)G, 4, K, ch0, q[v]);
            if (ch0 == 0) {
                bias[v] = u32x2_t{0u, 0u};
                if (P.bias >= 0) bias[v] = __builtin_amdgcn_raw_buffer_load_b64(rw, (uint32_t)(P.bias + 2 * (c0 + 4 * g)), 0, 0);
            }
            const int64_t xr = DOWN ? pl[v].pair : pair_tok(a, pl[v].pair);
            const int64_t stride = DOWN ? m.hstride : K;
            const uint8_t* const xc = (DOWN ? m.hq : m.xq) + xr * (stride / 2);
            const uint8_t* const xs = (DOWN ? m.hs : m.xs) + xr * (stride / 32);
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int first = 16 * (ch0 + j) + 4 * g;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    // (pieces past the row's end: any, and zeros below)
                    const u32x4_t x4 = *reinterpret_cast<const u32x4_t*>(xc + 16 * min(first + t, G - 1));
                    xv[v][j][t] = mx_u32x4{x4[0], x4[1], x4[2], x4[3]};
                }
                // two groups at a time: rows of scales are 2-byte aligned
                const uint32_t lo = *reinterpret_cast<const uint16_t*>(xs + min(first, G - 2));
                const uint32_t hi = *reinterpret_cast<const uint16_t*>(xs + min(first + 2, G - 2));
                xe[v][j] = lo | (hi << 16);
            }
        };
        auto mul = [&](int v, int ch0) __attribute__((always_inline)) {
            const int K = Ks[v], G = K / 32, nch = (G + 15) / 16;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if (ch0 + j < nch) {               // uniform
                    const int first = 16 * (ch0 + j) + 4 * g;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t in = (uint32_t)((first + t - G) >> 31);
#pragma unroll
                        for (int i = 0; i < 4; ++i) xv[v][j][t][i] &= in;
                    }
                    few_mul(q[v].w[j], q[v].s[j], ch0 + j, K, xv[v][j], xe[v][j], acc[v]);
                }
            }
        };
#pragma unroll
        for (int v = 0; v < NE; ++v) {
            acc[v] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            if (NE == 1 || u0 + kRowWaves * v < entries) load(v, 0);          // uniform
        }
#pragma unroll
        for (int v = 0; v < NE; ++v) {
            if (NE == 1 || u0 + kRowWaves * v < entries) {
                mul(v, 0);
                for (int ch0 = NB; 32 * 16 * ch0 < Ks[v]; ch0 += NB) {        // (wider than the launch's batch)
                    load(v, ch0);
                    mul(v, ch0);
                }
                // lane (g, n): columns 4 g .. 4 g + 3 of pair n
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b = bias[v][i >> 1];
                    y[i] = absent[v] ? absent_nan() : acc[v][i] + bf2f((i & 1) ? b >> 16 : b & 0xFFFFu);
                }
                if (l16 < pl[v].n) {
                    if constexpr (DOWN) {
                        *reinterpret_cast<f32x4_t*>(&ys[pl[v].pair][4 * g]) = f32x4_t{y[0], y[1], y[2], y[3]};
                    } else {
                        const int N = m.proj == 2 ? a.H : a.I;
                        *reinterpret_cast<u32x2_t*>(m.y16 + (int64_t)pair_row(a, pl[v].pair) * N + c0 + 4 * g) =
                            u32x2_t{pk_bf16(y[0], y[1]), pk_bf16(y[2], y[3])};
                    }
                }
            }
        }
        if constexpr (DOWN) {
#pragma unroll
            for (int v = 0; v < NE; ++v) entry(u0 + kRowWaves * (NE + v), pl[v]);
        }
    }
    if constexpr (DOWN) {
        lds_barrier();
        // two columns a thread
        const int c = 2 * (tid & 7);
        if (m.y32) {
            for (int q = tid >> 3; q < a.P; q += 8 * kRowWaves) {
                typedef float f32x2_t __attribute__((ext_vector_type(2)));
                *reinterpret_cast<f32x2_t*>(m.y32 + (int64_t)pair_row(a, q) * a.H + c0 + c) = f32x2_t{ys[q][c], ys[q][c + 1]};
            }
        }
        if (a.yun) {
            for (int q = tid >> 3; q < a.P; q += 8 * kRowWaves)
                *reinterpret_cast<uint32_t*>(a.yun + (int64_t)pair_row(a, q) * a.H + c0 + c) = pk_bf16(ys[q][c], ys[q][c + 1]);
        }
        if (a.out && tid < 8 * a.T) {
            const int t = tid >> 3;
            float o0 = 0.f, o1 = 0.f;
            auto add = [&](float w, int q) __attribute__((always_inline)) {
                o0 = fmaf(w, ys[q][c], o0);
                o1 = fmaf(w, ys[q][c + 1], o1);
            };
            for (int j = 0; j < a.k; ++j) add(a.w[t * a.k + j], t * a.k + j);
            if (a.auto_shared && a.sgate) add(a.sgate[t], a.P + t);
            *reinterpret_cast<uint32_t*>(a.out + (int64_t)t * a.H + c0 + c) = f2bf(o0) | (f2bf(o1) << 16);
        }
    }
}

inline size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

struct FewWs {
    MxTable* table;
    uint8_t *hq, *hs;
    int32_t *order, *offsets, *tile_start;         // tiles only
    int4* tinfo;
    int Imax, tiles;                               // at most so many tiles (entries)
    size_t bytes;
};
FewWs carve_few(const FwdArgs& a, bool tiles, void* ws) {
    FewWs w{};
    w.Imax = a.shared && a.I_sh > a.I ? a.I_sh : a.I;
    const int rows = a.P + (a.auto_shared ? a.T : 0), E_ext = a.E + (a.shared ? 1 : 0);
    w.tiles = rows / 16 + (E_ext < rows ? E_ext : rows);
    if (w.tiles > rows) w.tiles = rows;            // (an entry has a pair)
    uint8_t* b = reinterpret_cast<uint8_t*>(ws);
    size_t off = 0;
    auto take = [&](size_t n) { uint8_t* p = b + off; off = align256(off + n); return p; };
    w.table = (MxTable*)take(sizeof(MxTable));
    w.hq = take((size_t)rows * (w.Imax / 2));
    w.hs = take((size_t)rows * (w.Imax / 32));
    if (tiles) {
        w.order = (int32_t*)take(sizeof(int32_t) * rows);
        w.offsets = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
        w.tile_start = (int32_t*)take(sizeof(int32_t) * (E_ext + 1));
        w.tinfo = (int4*)take(sizeof(int4) * w.tiles);
    }
    w.bytes = off;
    return w;
}

// Chunks a wave loads at once: all of a row's up to four, of wider rows three and three (one token of the
// gpt-oss shape, 6 chunks a row: 22.8 us all at once, 19.2 by three, 19.8 by two).
inline int few_batch(int K) { const int nch = (K + 511) / 512; return nch <= 2 ? nch : nch <= 4 ? 4 : 3; }

}  // namespace

size_t mx_few_workspace_bytes(const FwdArgs& a, bool tiles) { return carve_few(a, tiles, nullptr).bytes; }

hipError_t launch_mx_few_layer(const FwdArgs& a, bool tiles, float* rows32, void* ws, hipStream_t s) {
    const FewWs w = carve_few(a, tiles, ws);
    MxArgs m{};
    m.hq = w.hq;
    m.hs = w.hs;
    m.hstride = w.Imax;
    m.y32 = rows32;
    m.E_ext = a.E + (a.shared ? 1 : 0);
    hipError_t e = hipSuccess;
    if (tiles) {
        m.order = w.order;
        m.tile_start = w.tile_start;
        m.tinfo = w.tinfo;
        e = launch_bucket(a.pexp, a.P, a.E, m.E_ext, a.auto_shared ? a.T : 0, 16, a.g2s, a.capacity, a.host != nullptr,
                          a.err, w.order, w.offsets, w.tile_start, w.tinfo, s);
        if (e != hipSuccess) return e;
    }
    const int per = a.act == BRX_ACT_SILU_MLP ? 64 : 32, nch = (a.H + 511) / 512;
    int most = a.P < 16 ? a.P : 16;                // pairs of an entry, at most
    if (a.auto_shared && a.T > most) most = a.T < 16 ? a.T : 16;
    // planned by the blocks: the entries of the routed pairs, and of the shared expert
    const int routed = a.P / 16 + a.E + (a.shared ? 1 : 0);
    const int planned = (routed < a.P ? routed : a.P) + (a.auto_shared ? (a.T + 15) / 16 : 0);
    const dim3 grid((w.Imax + per - 1) / per, tiles ? w.tiles : planned);
    const size_t lds = (size_t)most * (few_code_pitch(nch) + few_scale_pitch(nch));
#define BRX_UP(NB) \
    if (tiles) hipLaunchKernelGGL((k_mx_few_up<NB, 0>), grid, dim3(64 * kUpWaves), lds, s, a, m, w.table); \
    else if (a.P > 64) hipLaunchKernelGGL((k_mx_few_up<NB, 2>), grid, dim3(64 * kUpWaves), lds, s, a, m, w.table); \
    else hipLaunchKernelGGL((k_mx_few_up<NB, 1>), grid, dim3(64 * kUpWaves), lds, s, a, m, w.table)
    switch (few_batch(a.H)) {
        case 1: BRX_UP(1); break;
        case 2: BRX_UP(2); break;
        case 4: BRX_UP(4); break;
        default: BRX_UP(3);
    }
#undef BRX_UP
    if ((e = hipGetLastError()) != hipSuccess) return e;
#define BRX_DOWN(NB, NE) hipLaunchKernelGGL((k_mx_few_rows<true, NB, NE>), dim3(a.H / 16), dim3(64 * kRowWaves), 0, s, a, m, w.table)
    // a wave with several entries takes them two or four at once, as their rows allow
    const bool one = a.P + (a.auto_shared ? 1 : 0) <= kRowWaves;
    switch (few_batch(w.Imax)) {
        case 1: if (one) BRX_DOWN(1, 1); else BRX_DOWN(1, 4); break;
        case 2: if (one) BRX_DOWN(2, 1); else BRX_DOWN(2, 2); break;
        case 4: BRX_DOWN(4, 1); break;
        default: BRX_DOWN(3, 1);
    }
#undef BRX_DOWN
    return hipGetLastError();
}

hipError_t launch_mx_few_product(const FwdArgs& a, const uint8_t* codes, const uint8_t* scales, int proj, hipStream_t s) {
    MxArgs m{};
    m.xq = codes;
    m.xs = scales;
    m.y16 = a.yun;
    m.proj = proj;
    const int most = a.P / 16 + (a.E + 1 < a.P ? a.E + 1 : a.P), entries = most < a.P ? most : a.P;   // at most
    const dim3 grid((proj == 2 ? a.H : a.I) / 16, (entries + kRowWaves - 1) / kRowWaves);
#define BRX_ROWS(NB) \
    if (a.P > 64) hipLaunchKernelGGL((k_mx_few_rows<false, NB, 1, 2>), grid, dim3(64 * kRowWaves), 0, s, a, m, (const MxTable*)nullptr); \
    else hipLaunchKernelGGL((k_mx_few_rows<false, NB, 1, 1>), grid, dim3(64 * kRowWaves), 0, s, a, m, (const MxTable*)nullptr)
    switch (few_batch(proj == 2 ? a.I : a.H)) { case 1: BRX_ROWS(1); break; case 2: BRX_ROWS(2); break; case 4: BRX_ROWS(4); break; default: BRX_ROWS(3); }
#undef BRX_ROWS
    return hipGetLastError();
}

}  // namespace brx
