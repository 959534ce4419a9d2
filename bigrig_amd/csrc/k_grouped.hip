// Products of rows sorted by expert with each expert's matrix, and the gradients, bf16 or fp16 on the matrix
// instructions, fp32 sums rounded once. (Each step of a sum is rounded to nearest: the gradient of a run of 2^23 rows of one sign is off
// by 1e-5 of itself before its rounding.)
//
//   rows      out[r]  = W[e] a[r] (+ bias[e])         offsets[e] <= r < offsets[e + 1]; 0 behind the last run
//   rows^T    out[r]  = W[e]^T a[r]                   the gradient of the rows
//   weight    out[e]  = sum over e's run of a[r] b[r]^T   the gradient of the matrices (0 for an empty run)
//   bias      out[e]  = sum over e's run of a[r]
//
// One tile code for the three products. A block copies 64 steps of the reduction of both operands into LDS by the
// buffer unit, 16 bytes a lane, into a ring of stages; an operand whose reduction runs along its rows (X) lies there
// as rows of 128 bytes and is read 8 values a lane, one whose reduction runs across its rows (Y: W in rows^T, both in
// weight) lies as 64 rows of the tile's width and is read by the transposing LDS loads. Reductions end inside a stage:
// what lies past the end comes from past the buffer's end, as zeros, in both operands, so that a NaN next to them does
// not enter.
#include "block_ops.h"
#include "grouped_tiles.h"
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kG = 64;                // reduction steps of a stage
constexpr uint32_t kPast = 0x80000000u;   // a byte offset past every buffer
constexpr int kNonTemporal = 2;       // cache policy of a buffer store: not kept

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4_t* LDS_TR;

template <int DT>
__device__ __forceinline__ f32x16_t mfma(const s16x8_t& a, const s16x8_t& b, const f32x16_t& c) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    if constexpr (DT == BRX_DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Swizzle key of step k of a Y tile: half a wave's transposing load reads 64 bytes of each of 4 steps (k & 3), whose 16-byte
// slots are put into four different quarters of the banks (in the same quarter a load takes twice the cycles).
__device__ __forceinline__ int y_key(int k) { return 4 * (k & 3); }

// 16 bytes a lane from byte offset `at` of the buffer at p (`bytes` long; past them: zeros) into the 1 KB at `to`. In assembly:
// where the compiler knows of a copy into LDS in flight, it waits for all of them before each transposing load. It has
// no result register; whoever reads `to` waits for it (copies_left). m0, which holds the LDS address, is put back.
__device__ __forceinline__ void copy16(const void* p, uint32_t bytes, uint32_t at, const void* to) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const uint64_t base = (uint64_t)(uintptr_t)p;
    const u32x4 r = {(uint32_t)base, (uint32_t)(base >> 32) & 0xFFFFu, bytes, 0x00020000u};
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "s"((uint32_t)(uintptr_t)(LDS_PTR)to), "v"(at), "s"(r) : "memory");
}

// One operand of a tile: `M` values along the output, laid out X or Y, of which wave w of W copies its share.
template <bool Y, int M, int W>
struct Operand {
    static constexpr int kBytes = M * kG * 2;
    static constexpr int kCopies = kBytes / 1024;             // 1 KB copies a stage
    static constexpr int kMine = (kCopies + W - 1) / W;       // of a wave (past the last: repeated)
    static constexpr int kRow = M * 2;                        // bytes of a step (Y)
    static_assert(!Y || M >= 128, "a step of a Y tile has 16 slots or more");

    uint32_t at[kMine];       // the lane's byte offset in a stage at step 0
    int step[kMine];          // the reduction step of that offset in a stage: the first of 8 (X) or the only one (Y)

    __device__ __forceinline__ int copy(int wv, int i) const { return min(wv * kMine + i, kCopies - 1); }

    // X: row m of the tile lies `ld` values behind row m - 1. Y: step k lies `ld` values behind step k - 1. `m_all`: values
    // along the output that exist from the tile's start.
    __device__ __forceinline__ void init(int wv, int lane, int64_t ld, int m_all) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int c = copy(wv, i);
            if constexpr (!Y) {
                const int m = c * 8 + (lane >> 3), ch = (lane & 7) ^ a_key(m);
                step[i] = ch * 8;
                at[i] = m < m_all ? (uint32_t)(m * ld * 2) + ch * 16 : kPast;
            } else {
                constexpr int kLanes = kRow / 16;             // lanes a step
                const int k = c * (64 / kLanes) + lane / kLanes, ch = (lane % kLanes) ^ y_key(k);
                step[i] = k;
                at[i] = ch * 8 < m_all ? (uint32_t)(k * ld * 2) + ch * 16 : kPast;
            }
        }
    }
    // Stage `left` steps before the reduction's end of the buffer at p, into `lds`.
    __device__ __forceinline__ void issue(const void* p, uint32_t bytes, int left, uint8_t* lds, int wv) const {
#pragma unroll
        for (int i = 0; i < kMine; ++i) copy16(p, bytes, step[i] < left ? at[i] : kPast, lds + copy(wv, i) * 1024);
    }
};

// The lane's place in fragment f (32 values along the output) of an operand's stage, and the fragment of MFMA kk (16
// steps; the lane's half of the wave takes 8 of them).
template <bool Y, int M>
__device__ __forceinline__ uint32_t frag_at(int lane, int f) {
    if constexpr (!Y) {
        return (uint32_t)((f * 32 + (lane & 31)) * 128);
    } else {
        const int i = lane & 15, g = (lane >> 4) & 1, kh = lane >> 5;
        const int k = 8 * kh + (i >> 2), ch = f * 4 + 2 * g + ((i & 3) >> 1);
        return (uint32_t)(k * M * 2 + ((ch ^ y_key(k)) << 4) + (i & 1) * 8);
    }
}
template <bool Y, int M>
__device__ __forceinline__ s16x8_t frag(const uint8_t* stage, uint32_t at, int lane, int kk) {
    if constexpr (!Y) {
        const int kh = lane >> 5, l32 = lane & 31;
        return *reinterpret_cast<const s16x8_t*>(stage + at + (((2 * kk + kh) ^ a_key(l32)) << 4));
    } else {
        const uint8_t* p = stage + at + kk * (16 * M * 2);
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_TR)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_TR)(p + 4 * M * 2));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// Shape of a tile: fragments of a wave, waves, ring stages.
template <int TM_, int TN_, int WM_, int WN_, int NS_>
struct Shape {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, NS = NS_;
    static constexpr int W = WM * WN, kThreads = W * 64;
    static constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int kStage = (BM + BN) * kG * 2;
    static constexpr int kPitch = BN + 8;                     // values of a row of the output tile
    static constexpr int kTile = BM * kPitch * 2;
    static constexpr int kLds = NS * kStage > kTile ? NS * kStage : kTile;
};

// Tile of `rows` x `cols` values (of what exists) at `out` (rows `ld` values apart): the sum over `steps` of the
// operands at a and b. X operands advance along their rows, Y operands by whole steps.
template <int DT, bool AY, bool BY, class S>
__device__ __forceinline__ void tile(uint8_t* lds, const uint16_t* a, int64_t a_ld, int rows, const uint16_t* b, int64_t b_ld,
                                     int cols, int steps, const uint16_t* bias, uint16_t* out, int64_t ld) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wv / S::WN, wn = wv % S::WN;
    typedef Operand<AY, S::BM, S::W> A;
    typedef Operand<BY, S::BN, S::W> B;
    A oa;
    B ob;
    oa.init(wv, lane, a_ld, rows);
    ob.init(wv, lane, b_ld, cols);
    const int nst = (steps + kG - 1) / kG;
    // an X operand's stage covers the rows of the tile, a Y operand's the steps left of the stage
    auto copy = [&](auto& op, bool y, const uint16_t* p, int64_t op_ld, int m, int s, uint8_t* to) __attribute__((always_inline)) {
        const int left = steps - s * kG;
        const int n = y ? min(left, kG) : m, run = y ? m : left;
        const uint32_t bytes = left > 0 ? (uint32_t)(((int64_t)(n - 1) * op_ld + run) * 2) : 0u;
        op.issue(y ? p + (int64_t)s * kG * op_ld : p + s * kG, bytes, left, to, wv);
    };
    auto issue = [&](int s, int at) __attribute__((always_inline)) {
        uint8_t* st = lds + at * S::kStage;
        copy(oa, AY, a, a_ld, min(rows, S::BM), s, st);
        copy(ob, BY, b, b_ld, min(cols, S::BN), s, st + A::kBytes);
    };
    f32x16_t acc[S::TM][S::TN];
#pragma unroll
    for (int m = 0; m < S::TM; ++m)
#pragma unroll
        for (int n = 0; n < S::TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;
    uint32_t fa[S::TM], fb[S::TN];
#pragma unroll
    for (int m = 0; m < S::TM; ++m) fa[m] = frag_at<AY, S::BM>(lane, wm * S::TM + m);
#pragma unroll
    for (int n = 0; n < S::TN; ++n) fb[n] = A::kBytes + frag_at<BY, S::BN>(lane, wn * S::TN + n);

#pragma unroll
    for (int s = 0; s < S::NS - 1; ++s) issue(s, s);
    int at = 0, next = S::NS - 1;
    for (int s = 0; s < nst; ++s) {
        // stage s has landed for every wave, and every wave has read stage s - 1, whose slot is next
        thin_wait_barrier<(S::NS - 2) * (A::kMine + B::kMine)>();
        issue(s + S::NS - 1, next);
        const uint8_t* st = lds + at * S::kStage;
#pragma unroll
        for (int kk = 0; kk < kG / 16; ++kk) {
            s16x8_t af[S::TM], bf[S::TN];
#pragma unroll
            for (int n = 0; n < S::TN; ++n) bf[n] = frag<BY, S::BN>(st, fb[n], lane, kk);
#pragma unroll
            for (int m = 0; m < S::TM; ++m) af[m] = frag<AY, S::BM>(st, fa[m], lane, kk);
#pragma unroll
            for (int m = 0; m < S::TM; ++m)
#pragma unroll
                for (int n = 0; n < S::TN; ++n) acc[m][n] = mfma<DT>(af[m], bf[n], acc[m][n]);
        }
        at = at + 1 == S::NS ? 0 : at + 1;
        next = next + 1 == S::NS ? 0 : next + 1;
    }
    thin_wait_barrier<0>();

    // the tile through LDS, then 16-byte stores. Element i of a fragment is row 8 (i / 4) + 4 kh + i % 4, column l32.
    uint16_t* T = reinterpret_cast<uint16_t*>(lds);
    const int kh = lane >> 5, l32 = lane & 31;
#pragma unroll
    for (int n = 0; n < S::TN; ++n) {
        const int col = (wn * S::TN + n) * 32 + l32;
        const float add = bias ? to_f<DT>(bias[min(col, cols - 1)]) : 0.f;
#pragma unroll
        for (int m = 0; m < S::TM; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                T[((wm * S::TM + m) * 32 + 8 * (i >> 2) + 4 * kh + (i & 3)) * S::kPitch + col] = from_f<DT>(acc[m][n][i] + add);
    }
    lds_barrier();
    constexpr int CH = S::BN / 8;
#pragma unroll 1
    for (int c = tid; c < S::BM * CH; c += S::kThreads) {
        const int r = c / CH, cl = (c % CH) * 8;
        if (r >= rows || cl >= cols) continue;
        set16(out + (int64_t)r * ld + cl, *reinterpret_cast<const v4u_t*>(T + r * S::kPitch + cl));
    }
}

// Tile `mt` of the rows' runs, cut into tiles of BM rows expert by expert, the rows behind the last run as one more run
// (expert E): its expert, first row and rows; -1 past the last tile. Every wave finds it by itself. Runs that offsets
// out of order or out of range would make are clamped into the rows there are.
struct RowTile {
    int e, first, rows;
};
__device__ __forceinline__ RowTile find_tile(const int32_t* __restrict__ offsets, int E, int P, int BM, int mt) {
    constexpr int kChunks = kMaxExperts / kWave + 1;
    const int lane = threadIdx.x & 63;
    int at[kChunks + 1];              // offsets of this lane's experts; loaded all at once
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
        if (i * kWave <= E) at[i] = offsets[min(i * kWave + lane, E)];
    int run = 0;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        if (i * kWave > E) break;     // uniform
        const int e = i * kWave + lane;
        int lo = e == 0 ? 0 : at[i];
        // the next expert's start: the lane above's, or the first of the next 64
        const int up = (i + 1) * kWave <= E ? __builtin_amdgcn_readlane(at[i + 1 < kChunks ? i + 1 : i], 0) : P;
        int hi = __builtin_amdgcn_ds_bpermute(min(lane + 1, 63) * 4, at[i]);
        hi = e >= E ? P : lane == 63 ? up : hi;
        const RowRun own = run_between(lo, e <= E ? hi : lo, P);
        lo = own.first;
        hi = own.end;
        const int n = run_tiles(own, BM);
        const int incl = wave_incl_scan(n);
        const uint64_t past = __ballot(run + incl > mt);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int k = mt - run - __builtin_amdgcn_readlane(incl - n, l);
            const int first = __builtin_amdgcn_readlane(lo, l) + k * BM;
            return {i * kWave + l, first, min(BM, __builtin_amdgcn_readlane(hi, l) - first)};
        }
        run += __builtin_amdgcn_readlane(incl, 63);
    }
    return {-1, 0, 0};
}

// BY: W is read across its rows (rows^T).
template <int DT, bool BY, class S>
__global__ __launch_bounds__(S::kThreads) void k_grouped_rows(GroupedArgs g, int mtiles, int ntiles) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[S::kLds];
    // an XCD takes every column tile of a row tile before its next row tile
    const int loc = blockIdx.x / kXcd;
    const int nt = loc % ntiles, mt = loc / ntiles * kXcd + blockIdx.x % kXcd;
    if (mt >= mtiles) return;
    const RowTile t = find_tile(g.offsets, g.E, g.P, S::BM, mt);
    if (t.e < 0) return;
    const int n0 = nt * S::BN;
    const bool none = t.e >= g.E;
    const uint16_t* w = g.b + (none ? 0 : (int64_t)t.e * g.b_expert) + (BY ? n0 : (int64_t)n0 * g.b_row);
    tile<DT, false, BY, S>(lds, g.a + (int64_t)t.first * g.K, g.K, t.rows, w, g.b_row, g.N - n0, none ? 0 : g.K,
                           g.bias && !none ? g.bias + (int64_t)t.e * g.N + n0 : nullptr, g.out + (int64_t)t.first * g.N + n0, g.N);
}

// out [E, K, N] = sum over the run of a [P, K] (x) b [P, N].
template <int DT, class S>
__global__ __launch_bounds__(S::kThreads) void k_grouped_weight(GroupedArgs g, int mtiles, int ntiles) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[S::kLds];
    const int e = blockIdx.y, m0 = blockIdx.x / ntiles * S::BM, n0 = blockIdx.x % ntiles * S::BN;
    const RowRun run = run_between(e == 0 ? 0 : g.offsets[e], g.offsets[e + 1], g.P);
    const int64_t lo = run.first;
    tile<DT, true, true, S>(lds, g.a + lo * g.K + m0, g.K, g.K - m0, g.b + lo * g.N + n0, g.N, g.N - n0, run.end - run.first,
                            nullptr, g.out + ((int64_t)e * g.K + m0) * g.N + n0, g.N);
}

// out [E, K] = sum over the run of a [P, K]: 128 columns a block, 8 a lane; 64 lanes take every 64th row each and join in
// order.
constexpr int kColThreads = 1024, kColLanes = 16, kColRows = kColThreads / kColLanes;
template <int DT>
__global__ __launch_bounds__(kColThreads) void k_grouped_bias(GroupedArgs g) {
    __shared__ float s[kColRows][kColLanes * 8 + 4];
    const int e = blockIdx.y, lane = threadIdx.x % kColLanes, r0 = threadIdx.x / kColLanes;
    const RowRun run = run_between(e == 0 ? 0 : g.offsets[e], g.offsets[e + 1], g.P);
    const int c0 = blockIdx.x * kColLanes * 8, col = c0 + lane * 8;
    const uint16_t* p = g.a + min(col, g.K - 8);
    float v[8] = {};
#pragma unroll 4
    for (int r = run.first + r0; r < run.end; r += kColRows) {
        float x[8];
        unpack<DT>(get16(p + (int64_t)r * g.K), x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += x[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[r0][lane * 8 + i] = v[i];
    __syncthreads();
    const int c = threadIdx.x;
    if (c < kColLanes * 8 && c0 + c < g.K) {
        float t = 0.f;
        for (int r = 0; r < kColRows; ++r) t += s[r][c];
        g.out[(int64_t)e * g.K + c0 + c] = from_f<DT>(t);
    }
}

// ------------------------------------------------------------------ thin tiles
// Up to 16 rows of a run times 32 columns, for calls of few rows, where reading the matrices is all the time there is: no LDS
// on the way, a lane's loads (16 bytes of a matrix row, 64 a row and instruction) go straight to the operands of
// v_mfma_f32_16x16x32, many in flight. The reduction is dealt to the block's four waves in units of 64 steps (whole
// lines), whose sums are joined in the waves' order.
constexpr int kThinCols = 32, kThinThreads = 256, kThinWaves = 4;
constexpr int kThinAhead = 8;         // units a wave loads at a time

template <int DT>
__device__ __forceinline__ f32x4_t mfma16(const v4u_t& a, const v4u_t& b, const f32x4_t& c) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    if constexpr (DT == BRX_DT_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__global__ __launch_bounds__(kThinThreads) void k_grouped_thin(GroupedArgs g, int ntiles) {
    __shared__ f32x4_t sums[kThinWaves][2][kWave];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int nt = blockIdx.x % ntiles;
    const RowTile t = find_tile(g.offsets, g.E, g.P, kThinRows, blockIdx.x / ntiles);
    if (t.e < 0) return;
    const int n0 = nt * kThinCols;
    const bool none = t.e >= g.E;
    const int l16 = lane & 15, ch = lane >> 4;
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(g.a + (int64_t)t.first * g.K, (uint32_t)(t.rows * g.K * 2));
    const __amdgpu_buffer_rsrc_t rw = make_rsrc(g.b + (none ? 0 : (int64_t)t.e * g.b_expert) + (int64_t)n0 * g.b_row,
                                                (uint32_t)((min(kThinCols, g.N - n0) - 1) * g.b_row + g.K) * 2);
    // (rows past the tile's and columns past the matrix's: past the buffers, zeros)
    const uint32_t ax = (uint32_t)(l16 * g.K + ch * 8) * 2, aw = (uint32_t)(l16 * g.b_row + ch * 8) * 2, dw = (uint32_t)(16 * g.b_row * 2);
    f32x4_t acc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
    const int steps = none ? 0 : g.K;
    for (int k0 = wv * 64; k0 < steps; k0 += kThinWaves * 64 * kThinAhead) {
        v4u_t x[kThinAhead][2], w[kThinAhead][2][2];
#pragma unroll
        for (int u = 0; u < kThinAhead; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = k0 + u * kThinWaves * 64 + h * 32;
                const bool in = k + ch * 8 < steps;
                x[u][h] = __builtin_bit_cast(v4u_t, __builtin_amdgcn_raw_buffer_load_b128(rx, in ? ax + k * 2 : kPast, 0, 0));
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    w[u][h][n] = __builtin_bit_cast(v4u_t, __builtin_amdgcn_raw_buffer_load_b128(rw, in ? aw + n * dw + k * 2 : kPast, 0, 0));
            }
        __builtin_amdgcn_sched_barrier(0);     // (all requested before the first is waited for)
#pragma unroll
        for (int u = 0; u < kThinAhead; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n) acc[n] = mfma16<DT>(w[u][h][n], x[u][h], acc[n]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) sums[wv][n][lane] = acc[n];
    __syncthreads();
    if (wv >= 2) return;
    f32x4_t v = sums[0][wv][lane];
#pragma unroll
    for (int w = 1; w < kThinWaves; ++w) v += sums[w][wv][lane];
    // element i: row l16, column 4 ch + i
    const int c = n0 + 16 * wv + 4 * ch;
    if (l16 >= t.rows || c >= g.N) return;
    uint32_t o[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float p = v[2 * i], q = v[2 * i + 1];
        if (g.bias && !none) {
            p += to_f<DT>(g.bias[(int64_t)t.e * g.N + c + 2 * i]);
            q += to_f<DT>(g.bias[(int64_t)t.e * g.N + c + 2 * i + 1]);
        }
        o[i] = (uint32_t)from_f<DT>(p) | ((uint32_t)from_f<DT>(q) << 16);
    }
    *reinterpret_cast<u32x2_t*>(g.out + (int64_t)(t.first + l16) * g.N + c) = u32x2_t{o[0], o[1]};
}

// ------------------------------------------------------------------ tall tiles
// Tiles of 256 x 256 for calls of many tiles, one block of 8 waves a CU that goes from tile to tile. Wave
// (wm, wn) owns the fragments 2 j + wm of the rows (so a tile of fewer rows leaves out the last ones of both) and 64
// columns. A stage of 64 steps is taken in four parts -- steps 0-31 and 32-63 of the first 128 rows, then of the others --
// and what each part has read is free for copies two stages ahead: b (held in registers for the second half) and the
// first rows after two parts, so that a copy has a stage and a half to land. The block's two groups of waves, one wave of
// each on a SIMD, are half a part apart: one reads and copies while the other's products run. The copies go on into the
// next tile, whose first stages land while the last one's sums are stored, straight from registers.
//
// Bound: the copies. 32768 rows of 8 experts of 4096 x 4096 take 890 us (1.24 PFLOP/s; 730 without copies, 690 without
// products), of 128 experts of 1536 x 2048 (256 rows each) 290 (280 without products; the matrices alone, 805 MB, take 150).
// (Timed in turn on one part; on another 942 and 297.) One stage ahead instead of one and a half: 940 and 316. One tile a block, 128 x 128 with two blocks a CU: 1250 and 340.
#define BRX_FENCE() __builtin_amdgcn_sched_barrier(0)
__device__ __forceinline__ void meet() {
    BRX_FENCE();
    asm volatile("s_barrier" ::: "memory");
    BRX_FENCE();
}
__device__ __forceinline__ void lds_read_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_left() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0xF << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
}

constexpr int kTallThreads = 512, kTallWaves = 8;
constexpr int kHalf = 128;                   // rows of a tile's halves
constexpr int kUnitB = kTall * kG * 2, kUnitA = kHalf * kG * 2;
constexpr int kTallRing = 2 * kUnitB + 5 * kUnitA;      // b and the first rows twice, the other rows three times

// One operand's copies: `M` values along the output, rows or steps `ld` values apart.
template <bool Y, int M>
struct Copies {
    static constexpr int kMine = M * kG * 2 / 1024 / kTallWaves;
    static constexpr int kLanes = M / 8;     // lanes of a step (Y)
    uint32_t at[kMine];
    int step[kMine], col[kMine];             // the chunk's reduction step in a stage; its first value along the output (Y)
    __device__ __forceinline__ void init(int wv, int lane, int64_t ld) {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int c = wv * kMine + i;
            if constexpr (!Y) {
                const int m = c * 8 + (lane >> 3), ch = (lane & 7) ^ a_key(m);
                step[i] = ch * 8;
                col[i] = 0;
                at[i] = (uint32_t)(m * ld * 2) + ch * 16;
            } else {
                const int k = c * (64 / kLanes) + lane / kLanes, ch = (lane % kLanes) ^ y_key(k);
                step[i] = k;
                col[i] = ch * 8;
                at[i] = (uint32_t)(k * ld * 2) + ch * 16;
            }
        }
    }
    // The stage at p: `left` steps and `m` values along the output are left of what there is.
    __device__ __forceinline__ void issue(const uint16_t* p, int64_t ld, int m, int left, uint8_t* to, int wv) const {
        const int rows = Y ? min(left, kG) : min(m, M), run = Y ? min(m, M) : left;
        const bool any = rows > 0 && run > 0;
        const uint32_t bytes = any ? (uint32_t)(((int64_t)(rows - 1) * ld + run) * 2) : 0u;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const bool on = Y ? col[i] < m : step[i] < left;
            copy16(p, bytes, on ? at[i] : kPast, to + (wv * kMine + i) * 1024);
        }
    }
};

// A tile: operands at its start, the values that exist along its rows and columns, its reduction, its output.
struct TallTile {
    const uint16_t *a, *b, *bias;
    uint16_t* out;
    int rows, cols, steps;
};

enum { kRows, kRowsT, kWeight };

// What the tiles of a call are found by: of each expert its run's start and the row tiles before it (entry E: the rows
// behind the last run; entry E + 1: the ends).
struct TallTable {
    int32_t first[kMaxExperts + 2], tiles[kMaxExperts + 2];
    int32_t order[kMaxExperts];       // experts by their runs' length, the longest first (products over the runs)
    int32_t sums[kTallWaves];
};

__device__ __forceinline__ void tall_table(TallTable& t, const int32_t* offsets, int E, int P) {
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    int base = 0;
    for (int e0 = 0; e0 <= E; e0 += kTallThreads) {
        const int e = e0 + tid;
        int lo = e == 0 ? 0 : offsets[min(e, E)], hi = e < E ? offsets[min(e + 1, E)] : P;
        const RowRun own = run_between(lo, e <= E ? hi : lo, P);
        lo = own.first;
        hi = own.end;
        const int n = run_tiles(own, kTall);
        const int incl = wave_incl_scan(n);
        __syncthreads();
        if (lane == 63) t.sums[wv] = incl;
        __syncthreads();
        int before = base;
        for (int w = 0; w < kTallWaves; ++w) {
            const int v = t.sums[w];
            if (w < wv) before += v;
            base += v;
        }
        if (e <= E) {
            t.first[e] = lo;
            t.tiles[e] = before + incl - n;
        }
        if (e == E) t.first[E + 1] = hi;
    }
    if (tid == 0) t.tiles[E + 1] = base;
    __syncthreads();
}

// Long reductions first, so that the last tiles to run are short.
__device__ __forceinline__ void tall_order(TallTable& t, int E) {
    const int e = threadIdx.x;               // (a thread an expert)
    static_assert(kTallThreads >= kMaxExperts, "");
    if (e < E) {
        const int n = t.first[e + 1] - t.first[e];
        int rank = 0;
        for (int f = 0; f < E; ++f) {
            const int m = t.first[f + 1] - t.first[f];
            rank += m > n || (m == n && f < e);
        }
        t.order[rank] = e;
    }
    __syncthreads();
}

// The last entry of v[0 .. n) that is at most x (v[0] is 0 and v does not decrease): 64 lanes look at a time.
__device__ __forceinline__ int last_at_most(const int32_t* v, int n, int x) {
    const int lane = threadIdx.x & 63;
    int at = 0;
    for (int e0 = 0; e0 < n; e0 += kWave) {
        const uint64_t m = __ballot(e0 + lane < n && v[min(e0 + lane, n - 1)] <= x);
        if (!m) break;
        at = e0 + 63 - __builtin_clzll(m);
    }
    return __builtin_amdgcn_readfirstlane(at);
}

// The tiles of a call in one sequence, two row tiles by all columns (of the runs' products: one by all) after another. A round
// gives each block one, each XCD neighbours, which share operands. The last round's, where they are few, are cut into two or
// four by their rows. (XCDs with sequences of their own, nothing cut: 8192 rows of 8 x 2048 x 2048 110 us against 99, 32768 of 64 x 512 x 512
// 41.7 / 38.4, 24000 of 8 x 2048 x 2048 173 / 179.)
template <int KIND>
struct TallList {
    const GroupedArgs& g;
    const TallTable& t;
    int ntiles, mtiles;       // column tiles; row tiles (in all, or of an expert's matrix)
    int xcd, place, per;      // this block's XCD, its place there; blocks an XCD
    int round;
    Rounds rounds;

    __device__ __forceinline__ void init() {
        round = 0;
        rounds = rounds_of(mtiles * ntiles * (KIND == kWeight ? g.E : 1), per * kXcd);
    }

    // The next tile of this block; false behind the last.
    __device__ __forceinline__ bool next(TallTile& o) {
        const Dealt d = deal(rounds, round, xcd, place, per);
        if (!d.rows) return false;
        ++round;
        const int at = d.tile, part = d.part, rows = d.rows;
        if constexpr (KIND == kWeight) {
            const int u = at / ntiles, nt = at - u * ntiles;
            const int e = __builtin_amdgcn_readfirstlane(t.order[u / mtiles]), m0 = u % mtiles * kTall + part * rows, n0 = nt * kTall;
            const int lo = t.first[e], hi = t.first[e + 1];
            const int l = __builtin_amdgcn_readfirstlane(lo), h = __builtin_amdgcn_readfirstlane(max(hi, lo));
            o.a = g.a + (int64_t)l * g.K + m0;
            o.b = g.b + (int64_t)l * g.N + n0;
            o.bias = nullptr;
            o.out = g.out + ((int64_t)e * g.K + m0) * g.N + n0;
            o.rows = min(g.K - m0, rows);
            o.cols = g.N - n0;
            o.steps = h - l;
        } else {
            const RowColumn rc = row_column(at, mtiles, ntiles);
            const int mt = rc.mt, nt = rc.nt;
            const int e = last_at_most(t.tiles, g.E + 1, mt);
            const int lo = __builtin_amdgcn_readfirstlane(t.first[e]), hi = __builtin_amdgcn_readfirstlane(t.first[e + 1]);
            const int m0 = lo + (mt - __builtin_amdgcn_readfirstlane(t.tiles[e])) * kTall + part * rows, n0 = nt * kTall;
            const bool none = e >= g.E;
            o.a = g.a + (int64_t)m0 * g.K;
            o.b = g.b + (none ? 0 : (int64_t)e * g.b_expert) + (KIND == kRowsT ? n0 : (int64_t)n0 * g.b_row);
            o.bias = g.bias && !none ? g.bias + (int64_t)e * g.N + n0 : nullptr;
            o.out = g.out + (int64_t)m0 * g.N + n0;
            o.rows = min(max(hi, lo) - m0, rows);
            o.cols = g.N - n0;
            o.steps = none ? 0 : g.K;
        }
        return o.rows > 0;                   // (a part past the tile's rows: nothing is behind it)
    }
};

// What a block carries from tile to tile: the copies' side, two stages ahead, and the ring's places.
template <int KIND>
struct TallState {
    static constexpr bool AY = KIND == kWeight, BY = KIND != kRows;
    const GroupedArgs& g;
    TallList<KIND> ahead;
    Copies<AY, kHalf> ca;
    Copies<BY, kTall> cb;
    uint8_t *lds_b, *lds_0, *lds_1;
    TallTile src;
    uint32_t fa[2], fb[2];
    int64_t a_ld, b_ld, a_step, b_step, a_half;
    int left;                                // steps of src's tile that are not copied yet (a tile without any: one empty stage)
    bool more;
    int at, at1, to1;
    int lane, wv, wm, wn;
    int stores;                              // stores issued behind the last tile
    static constexpr int kStageCopies = 2 * Copies<AY, kHalf>::kMine + Copies<BY, kTall>::kMine;

    __device__ __forceinline__ void advance() {
        left -= kG;
        if (left > 0) {
            src.a += a_step;
            src.b += b_step;
        } else if (more) {
            more = ahead.next(src);
            left = more ? src.steps : 0;
        } else {
            left = 0;
        }
    }
    // Waits for what the next stage reads. Behind it are this stage's copies and, in a tile's first stage, the last tile's
    // stores, which need not have landed (stages of one tile each would wait for every tile's stores in turn).
    template <int N>
    __device__ __forceinline__ void landed(int s) const {
        if (s > 0 || stores < 4) copies_left<N>();
        else if (stores < 16) copies_left<N + 4>();
        else copies_left<N + 16>();
    }
    __device__ __forceinline__ void copy_b(int slot) { cb.issue(src.b, b_ld, src.cols, left, lds_b + slot * kUnitB, wv); }
    __device__ __forceinline__ void copy_a(int h, uint8_t* to) { ca.issue(src.a + h * a_half, a_ld, src.rows - h * kHalf, left, to, wv); }
};

// A tile whose rows fill NF fragments of a wave.
template <int DT, int KIND, int NF>
__device__ __forceinline__ void tall_tile(TallState<KIND>& c, const TallTile& dst) {
    constexpr bool AY = TallState<KIND>::AY, BY = TallState<KIND>::BY;
    constexpr int kLeft = TallState<KIND>::kStageCopies;
    const int lane = c.lane;
    const bool late = c.wm;                  // (the group that is half a part behind)
    f32x16_t acc[NF][2];
#pragma unroll
    for (int m = 0; m < NF; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;
    const int nst = max((dst.steps + kG - 1) / kG, 1);
    for (int s = 0; s < nst; ++s) {
        uint8_t* const sb = c.lds_b + c.at * kUnitB;
        uint8_t* const s0 = c.lds_0 + c.at * kUnitA;
        const uint8_t* const s1 = c.lds_1 + c.at1 * kUnitA;
        s16x8_t bf[4][2];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int k0 = 2 * (p & 1), m0 = (p >> 1) * 2;
            constexpr int kNone = 0;
            const int mf = NF - m0 < kNone ? kNone : NF - m0 > 2 ? 2 : NF - m0;   // fragments of this half
            if (NF <= 2 && p == 3) break;    // (its copies are part 2's)
            s16x8_t af[2][2];
            if (p < 2) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int n = 0; n < 2; ++n) bf[k0 + q][n] = frag<BY, kTall>(sb, c.fb[n], lane, k0 + q);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int m = 0; m < mf; ++m) af[q][m] = frag<AY, kHalf>(p < 2 ? s0 : s1, c.fa[m], lane, k0 + q);
            const bool last = p == (NF <= 2 ? 2 : 3);
            if (p == 0) c.copy_a(1, c.lds_1 + c.to1 * kUnitA);
            if (p == 2) c.copy_b(c.at);
            if (last) {
                c.copy_a(0, s0);
                c.advance();
            }
            lds_read_done();
            if (last && late) c.template landed<kLeft>(s);
            meet();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int m = 0; m < mf; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n) acc[m0 + m][n] = mfma<DT>(bf[k0 + q][n], af[q][m], acc[m0 + m][n]);
            __builtin_amdgcn_s_setprio(0);
            if (last && !late) c.template landed<kLeft>(s);
            meet();
        }
        c.at ^= 1;
        c.at1 = c.at1 == 2 ? 0 : c.at1 + 1;
        c.to1 = c.to1 == 2 ? 0 : c.to1 + 1;
    }
    // Element i of a fragment is column 8 (i / 4) + 4 kh + i % 4 of row l32: two groups of four columns, exchanged
    // between the halves of the wave, are 16 bytes of a row, and a row's four such pieces, exchanged among four lanes,
    // make a store eight rows of 128 bytes.
    const int kh = lane >> 5, l32 = lane & 31;
    const int col = c.wn * 64 + 16 * (l32 & 3) + 8 * kh;
    const bool in = col < dst.cols, odd = lane & 1, high = lane & 2;
    // (every store is issued, those of rows and columns that do not exist past the buffer's end: the next stage's wait counts them)
    const __amdgpu_buffer_rsrc_t ro = make_rsrc(dst.out, (uint32_t)((min(dst.rows, kTall) - 1) * c.g.N + min(dst.cols, kTall)) * 2);
    u32x2_t add[2][2][2];                    // four columns' values each
    if (dst.bias) {
        typedef u32x2_t __attribute__((aligned(2))) V;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    add[n][j][h] = *reinterpret_cast<const V*>(dst.bias + min(c.wn * 64 + 32 * n + 16 * j + 8 * h + 4 * kh, dst.cols - 4));
    }
#pragma unroll
    for (int m = 0; m < NF; ++m) {
        uint32_t q[4][4];                    // [piece of 16 columns][word]
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = acc[m][n][8 * j + i];
                    const uint32_t b = add[n][j][i >> 2][(i & 3) >> 1];
                    if (dst.bias) v[i] += to_f<DT>((uint16_t)(i & 1 ? b >> 16 : b & 0xFFFFu));
                }
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (uint32_t)from_f<DT>(v[2 * i]) | ((uint32_t)from_f<DT>(v[2 * i + 1]) << 16);
                const auto lo = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
                const auto hi = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
                q[2 * n + j][0] = lo[0];
                q[2 * n + j][1] = hi[0];
                q[2 * n + j][2] = lo[1];
                q[2 * n + j][3] = hi[1];
            }
        // piece b of lane i to lane b's place i, in lanes 4 a + b: neighbours first, then pairs
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int p = 0; p < 4; p += 2) {
                const uint32_t e = q[p][x], o = q[p + 1][x], ne = dpp_u<0xB1>(e), no = dpp_u<0xB1>(o);
                q[p][x] = odd ? no : e;
                q[p + 1][x] = odd ? o : ne;
            }
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const uint32_t e = q[p][x], o = q[p + 2][x], ne = dpp_u<0x4E>(e), no = dpp_u<0x4E>(o);
                q[p][x] = high ? no : e;
                q[p + 2][x] = high ? o : ne;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (2 * m + c.wm) * 32 + (l32 & 28) + i;
            const v4u_t v = {q[i][0], q[i][1], q[i][2], q[i][3]};
            const uint32_t to = in && row < dst.rows ? (uint32_t)(row * c.g.N + col) * 2 : kPast;
            if (KIND == kWeight && c.g.past_cache) __builtin_amdgcn_raw_buffer_store_b128(v, ro, to, 0, kNonTemporal);
            else __builtin_amdgcn_raw_buffer_store_b128(v, ro, to, 0, 0);
        }
    }
    c.stores = 4 * NF;
}

template <int DT, int KIND>
__global__ __launch_bounds__(kTallThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
void k_grouped_tall(GroupedArgs g, int ntiles, int mtiles) {
    constexpr bool AY = KIND == kWeight, BY = KIND != kRows;
    // (one array: given several, the compiler waits for all copies in flight before each read)
    __shared__ __attribute__((aligned(16))) uint8_t lds[kTallRing + sizeof(TallTable)];
    TallTable& table = *reinterpret_cast<TallTable*>(lds + kTallRing);
    const int tid = threadIdx.x;
    tall_table(table, g.offsets, g.E, g.P);
    if constexpr (KIND == kWeight) tall_order(table, g.E);
    else mtiles = __builtin_amdgcn_readfirstlane(table.tiles[g.E + 1]);
    TallList<KIND> list{g, table, ntiles, mtiles, (int)blockIdx.x % kXcd, (int)blockIdx.x / kXcd, (int)gridDim.x / kXcd};
    list.init();
    TallState<KIND> c{g, list};
    c.lane = tid & 63;
    c.wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    c.wm = c.wv >> 2;
    c.wn = c.wv & 3;
    c.a_ld = g.K;
    c.b_ld = KIND == kWeight ? g.N : g.b_row;
    c.a_step = AY ? kG * c.a_ld : kG;
    c.b_step = BY ? kG * c.b_ld : kG;
    c.a_half = AY ? kHalf : kHalf * c.a_ld;
    c.ca.init(c.wv, c.lane, c.a_ld);
    c.cb.init(c.wv, c.lane, c.b_ld);
    c.lds_b = lds;
    c.lds_0 = lds + 2 * kUnitB;
    c.lds_1 = c.lds_0 + 2 * kUnitA;
#pragma unroll
    for (int m = 0; m < 2; ++m) c.fa[m] = frag_at<AY, kHalf>(c.lane, 2 * m + c.wm);
#pragma unroll
    for (int n = 0; n < 2; ++n) c.fb[n] = frag_at<BY, kTall>(c.lane, c.wn * 2 + n);
    TallTile dst;
    if (!list.next(dst)) return;             // (uniform: a block without tiles)
    c.more = c.ahead.next(c.src);
    c.left = c.src.steps;
    // in the order of the loop: the other rows, b, the first rows
    c.copy_a(1, c.lds_1);
    c.copy_b(0);
    c.copy_a(0, c.lds_0);
    c.advance();
    c.copy_a(1, c.lds_1 + kUnitA);
    c.copy_b(1);
    c.copy_a(0, c.lds_0 + kUnitA);
    c.advance();
    copies_left<TallState<KIND>::kStageCopies>();
    meet();
    if (c.wm) meet();
    c.at = c.at1 = c.stores = 0;
    c.to1 = 2;
    do {
        const int nf = (min(dst.rows, kTall) + 63) / 64;
        if (nf == 4) tall_tile<DT, KIND, 4>(c, dst);
        else if (nf == 3) tall_tile<DT, KIND, 3>(c, dst);
        else if (nf == 2) tall_tile<DT, KIND, 2>(c, dst);
        else tall_tile<DT, KIND, 1>(c, dst);
    } while (list.next(dst));
    if (!c.wm) meet();
    copies_left<0>();                        // (none is in flight when the block's LDS goes to another)
}

// (named here: left to their first use, the compiler emits the launch code of one of them only)
#define BRX_TALL(DT)                                                              \
    template __global__ void k_grouped_tall<DT, kRows>(GroupedArgs, int, int);    \
    template __global__ void k_grouped_tall<DT, kRowsT>(GroupedArgs, int, int);   \
    template __global__ void k_grouped_tall<DT, kWeight>(GroupedArgs, int, int)
BRX_TALL(BRX_DT_BF16);
BRX_TALL(BRX_DT_F16);
#undef BRX_TALL

typedef Shape<2, 2, 2, 2, 2> Square;      // 128 x 128, four waves: two blocks a CU
typedef Shape<1, 1, 2, 4, 3> Half;        // 64 x 128, eight waves, one stage more ahead
typedef Shape<1, 1, 1, 4, 4> Low;         // 32 x 128, four waves, two stages more ahead
typedef Shape<1, 2, 4, 2, 2> Eight;       // 128 x 128, eight waves

// Which kernel. Products of rows, by what bounds them. Where runs are short, by the matrices' bytes: thin tiles for up to 8 rows,
// 32 x 128 up to 16 rows a run on average, 64 x 128 up to 48 (and where 128 x 128 could not give each CU one): lower tiles
// leave LDS for more of the matrices in flight. Where whole tiles of 256 x 256 give each CU one: the persistent kernel. Between:
// 128 x 128, two blocks a CU. bf16, us, thin / 32 / 64 / 128 / 256 (rows; rows^T in brackets):
//   128 experts of 2048 -> 1536   8 rows 14.6 / 16.6 / 20 / 25 / -        16 rows 20.4 / 19.3 / 20 / - / -
//                               512 rows 131 / 125 / 132 / 147 / - (- / 115 / 117 / 133)
//                              2048 rows - / 157 / 170 / 189 / - (- / 146 / 146 / 150)
//                              6144 rows - / 225 / 172 / 195 / 194 (- / 233 / 161 / 164 / 152)
//                              8192 rows - / 272 / 190 / 202 / 202 (- / 271 / 184 / 171 / 162)
//                             32768 rows - / - / - / 340 / 294 (- / - / - / 352 / 268)
//   64 experts, thin / 32: 8 rows 2048 -> 2048 16.5 / 16.5, 4096 -> 1024 21 / 25, 2880 -> 2880 27 / 24; 32 rows 41 / 39, 52 / 40, 88 / 84
//   256 experts of 2048 -> 4096 8192 rows - / 872 / 806 / 914 / 902 (- / 909 / 750 / 750 / 705: the persistent kernel before 64 x 128)
//   64 experts of 512 -> 512    4096 rows - / 19.4 / 14.1 / 13.0 / 20.1,  32768 rows - / - / - / 43.0 / 41.9
//   8 experts, 1000 rows   1024 -> 1024 - / 19.6 / 13.0 / 17.0 / 52,  1024 -> 2048 (256 tiles of 128) - / 29 / 21.4 / 19.3 / 54
// Products over the runs write every tile in any case: the persistent kernel where those are as many as the CUs (128 by four
// waves / 256: 64 x 512 x 512 of 4096 rows 18.0 / 18.2, 60 x 712 x 1000 of 2804 34.3 / 29.8, 128 x 1536 x 2048 of 1024 231 / 162,
// of 32768 478 / 343), else 128 x 128 by eight waves (by four / by eight / 256: 8 x 1024 x 1024 of 1000 rows 12.0 / 11.8 / 16.3,
// 8 x 1024 x 2048 of 4000 33.3 / 28.7 / 28.6).
static_assert(kChipCus == kCus && kChipXcds == kXcd, "");

// Gradients of the matrices that are larger than the chip's last cache, and whose rows are whole lines, are stored past the
// caches (128 x 1536 x 2048, 805 MB, of 32768 rows: 378 -> 323 us, a read of them right behind it included 700 -> 676; all three
// products of 16000 rows of 128 x 1024 x 2048 482 -> 440, of the former no difference: other kernels wait for less that is
// written back, and the clocks fall). Of what fits, the read finds less (24 x 1024 x 2048, 101 MB: 86 -> 80, with the read 115 ->
// 121), and parts of lines cost more (60 x 712 x 1000: 30 -> 46).
constexpr int64_t kCacheBytes = 256ll << 20;

template <int DT, bool BY, class S>
hipError_t launch_tiles(const GroupedArgs& g, hipStream_t s) {
    const int mt = (int)row_tiles(g.P, g.E, S::BM), nt = (g.N + S::BN - 1) / S::BN;
    hipLaunchKernelGGL((k_grouped_rows<DT, BY, S>), dim3((mt + kXcd - 1) / kXcd * kXcd * nt), dim3(S::kThreads), 0, s, g, mt, nt);
    return hipGetLastError();
}

template <int DT, bool BY>
hipError_t launch_rows(const GroupedArgs& g, hipStream_t s) {
    const RowForm form = row_form(g.P, g.E, g.N, BY);
    if constexpr (!BY) {
        if (form == kFormThin) {
            const int nt = (g.N + kThinCols - 1) / kThinCols;
            hipLaunchKernelGGL(k_grouped_thin<DT>, dim3((unsigned)(row_tiles(g.P, g.E, kThinRows) * nt)), dim3(kThinThreads), 0, s, g, nt);
            return hipGetLastError();
        }
    }
    if (form == kFormLow) return launch_tiles<DT, BY, Low>(g, s);
    if (form == kFormHalf) return launch_tiles<DT, BY, Half>(g, s);
    if (form == kFormSquare) return launch_tiles<DT, BY, Square>(g, s);
    constexpr int kind = BY ? kRowsT : kRows;
    hipLaunchKernelGGL((k_grouped_tall<DT, kind>), dim3(kCus), dim3(kTallThreads), 0, s, g, (g.N + kTall - 1) / kTall, 0);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_weight(const GroupedArgs& g, hipStream_t s) {
    const int tall_mt = (g.K + kTall - 1) / kTall, tall_nt = (g.N + kTall - 1) / kTall;
    if ((int64_t)g.E * tall_mt * tall_nt >= kCus) {
        GroupedArgs a = g;
        a.past_cache = (int64_t)g.E * g.K * g.N * 2 > kCacheBytes && g.N % 64 == 0;
        hipLaunchKernelGGL((k_grouped_tall<DT, kWeight>), dim3(kCus), dim3(kTallThreads), 0, s, a, tall_nt, tall_mt);
        return hipGetLastError();
    }
    typedef Eight S;
    const int mt = (g.K + S::BM - 1) / S::BM, nt = (g.N + S::BN - 1) / S::BN;
    hipLaunchKernelGGL((k_grouped_weight<DT, S>), dim3(mt * nt, g.E), dim3(S::kThreads), 0, s, g, mt, nt);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_grouped_rows(const GroupedArgs& g, bool transposed, int dtype, hipStream_t s) {
    if (dtype == BRX_DT_BF16) return transposed ? launch_rows<BRX_DT_BF16, true>(g, s) : launch_rows<BRX_DT_BF16, false>(g, s);
    return transposed ? launch_rows<BRX_DT_F16, true>(g, s) : launch_rows<BRX_DT_F16, false>(g, s);
}

hipError_t launch_grouped_weight(const GroupedArgs& g, int dtype, hipStream_t s) {
    return dtype == BRX_DT_BF16 ? launch_weight<BRX_DT_BF16>(g, s) : launch_weight<BRX_DT_F16>(g, s);
}

hipError_t launch_grouped_bias(const GroupedArgs& g, int dtype, hipStream_t s) {
    const dim3 grid((g.K + kColLanes * 8 - 1) / (kColLanes * 8), g.E);
    if (dtype == BRX_DT_BF16) hipLaunchKernelGGL(k_grouped_bias<BRX_DT_BF16>, grid, dim3(kColThreads), 0, s, g);
    else hipLaunchKernelGGL(k_grouped_bias<BRX_DT_F16>, grid, dim3(kColThreads), 0, s, g);
    return hipGetLastError();
}

}  // namespace brx
