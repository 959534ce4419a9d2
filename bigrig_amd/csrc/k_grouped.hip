// Products of rows sorted by expert with each expert's matrix, and the gradients, bf16 or fp16 on the matrix
// instructions, fp32 sums rounded once.
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
#include "pf_common.h"

namespace brx {
namespace {

constexpr int kG = 64;                // reduction steps of a stage
constexpr uint32_t kPast = 0x80000000u;   // a byte offset past every buffer

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

// Swizzle key of step k of a Y tile: a transposing load reads 32 bytes of 4 steps (k & 3) for each of two halves of the
// wave (8 steps apart), so the 16-byte slots of those 8 steps are put into 8 different 32-byte pieces of the banks.
__device__ __forceinline__ int y_key(int k) { return 2 * ((k & 3) | ((k >> 3) & 1) << 2); }

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
    // Stage `left` steps before the reduction's end, into `lds`.
    __device__ __forceinline__ void issue(const __amdgpu_buffer_rsrc_t& r, uint32_t soff, int left, uint8_t* lds, int wv) const {
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const uint32_t v = step[i] < left ? at[i] : kPast;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LDS_PTR)(lds + copy(wv, i) * 1024), 16, v, soff, 0, 0);
        }
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
    // a stage's descriptor: an X operand's covers the rows of the tile, a Y operand's the steps left of the stage
    auto desc = [&](bool y, const uint16_t* p, int64_t op_ld, int m_all, int s, int most) __attribute__((always_inline)) {
        const int left = min(steps - s * kG, kG);
        if (left <= 0) return make_rsrc(p, 0);
        if (!y) return make_rsrc(p + s * kG, (uint32_t)(((int64_t)(min(m_all, most) - 1) * op_ld + (steps - s * kG)) * 2));
        return make_rsrc(p + (int64_t)s * kG * op_ld, (uint32_t)(((int64_t)(left - 1) * op_ld + min(m_all, most)) * 2));
    };
    auto issue = [&](int s, int at) __attribute__((always_inline)) {
        uint8_t* st = lds + at * S::kStage;
        const int left = steps - s * kG;
        oa.issue(desc(AY, a, a_ld, rows, s, S::BM), 0, left, st, wv);
        ob.issue(desc(BY, b, b_ld, cols, s, S::BN), 0, left, st + A::kBytes, wv);
        asm volatile("" ::: "memory");
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
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int e0 = 0; e0 <= E; e0 += kWave) {
        const int e = e0 + lane;
        int lo = e == 0 ? 0 : offsets[min(e, E)], hi = e < E ? offsets[min(e + 1, E)] : P;
        lo = min(max(lo, 0), P);
        hi = e <= E ? min(max(hi, lo), P) : lo;
        const int n = (hi - lo + BM - 1) / BM;
        const int incl = wave_incl_scan(n);
        const uint64_t past = __ballot(run + incl > mt);
        if (past) {
            const int l = __builtin_ctzll(past);
            const int k = mt - run - __builtin_amdgcn_readlane(incl - n, l);
            const int first = __builtin_amdgcn_readlane(lo, l) + k * BM;
            return {e0 + l, first, min(BM, __builtin_amdgcn_readlane(hi, l) - first)};
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
    int lo = e == 0 ? 0 : g.offsets[e], hi = g.offsets[e + 1];
    lo = min(max(lo, 0), g.P);
    hi = min(max(hi, lo), g.P);
    tile<DT, true, true, S>(lds, g.a + (int64_t)lo * g.K + m0, g.K, g.K - m0, g.b + (int64_t)lo * g.N + n0, g.N, g.N - n0, hi - lo,
                            nullptr, g.out + ((int64_t)e * g.K + m0) * g.N + n0, g.N);
}

// out [E, K] = sum over the run of a [P, K]: 64 columns a block, its waves take every 16th row each and join in order.
constexpr int kColThreads = 1024;
template <int DT>
__global__ __launch_bounds__(kColThreads) void k_grouped_bias(GroupedArgs g) {
    constexpr int W = kColThreads / kWave;
    __shared__ float s[W][kWave];
    const int e = blockIdx.y, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    int lo = e == 0 ? 0 : g.offsets[e], hi = g.offsets[e + 1];
    lo = min(max(lo, 0), g.P);
    hi = min(max(hi, lo), g.P);
    const int col = blockIdx.x * kWave + lane;
    const uint16_t* p = g.a + min(col, g.K - 1);
    float v = 0.f;
#pragma unroll 4
    for (int r = lo + wv; r < hi; r += W) v += to_f<DT>(p[(int64_t)r * g.K]);
    s[wv][lane] = v;
    __syncthreads();
    if (wv == 0 && col < g.K) {
        for (int w = 1; w < W; ++w) v += s[w][lane];
        g.out[(int64_t)e * g.K + col] = from_f<DT>(v);
    }
}

// Row tiles of BM rows a call can have: the whole ones, and one of each run that is not empty.
inline int64_t row_tiles(const GroupedArgs& g, int BM) {
    const int64_t runs = g.E + 1;
    return g.P / BM + (runs < g.P ? runs : g.P);
}

template <int DT, bool BY, class S>
hipError_t rows_shape(const GroupedArgs& g, hipStream_t s) {
    const int mt = (int)row_tiles(g, S::BM), nt = (g.N + S::BN - 1) / S::BN;
    hipLaunchKernelGGL((k_grouped_rows<DT, BY, S>), dim3((mt + kXcd - 1) / kXcd * kXcd * nt), dim3(S::kThreads), 0, s, g, mt, nt);
    return hipGetLastError();
}

typedef Shape<2, 2, 2, 2, 2> Square;      // 128 x 128

template <int DT>
hipError_t weight_shape(const GroupedArgs& g, hipStream_t s) {
    typedef Square S;
    const int mt = (g.K + S::BM - 1) / S::BM, nt = (g.N + S::BN - 1) / S::BN;
    hipLaunchKernelGGL((k_grouped_weight<DT, S>), dim3(mt * nt, g.E), dim3(S::kThreads), 0, s, g, mt, nt);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_grouped_rows(const GroupedArgs& g, bool transposed, int dtype, hipStream_t s) {
    if (dtype == BRX_DT_BF16) {
        if (transposed) return rows_shape<BRX_DT_BF16, true, Square>(g, s);
        return rows_shape<BRX_DT_BF16, false, Square>(g, s);
    }
    if (transposed) return rows_shape<BRX_DT_F16, true, Square>(g, s);
    return rows_shape<BRX_DT_F16, false, Square>(g, s);
}

hipError_t launch_grouped_weight(const GroupedArgs& g, int dtype, hipStream_t s) {
    return dtype == BRX_DT_BF16 ? weight_shape<BRX_DT_BF16>(g, s) : weight_shape<BRX_DT_F16>(g, s);
}

hipError_t launch_grouped_bias(const GroupedArgs& g, int dtype, hipStream_t s) {
    const dim3 grid((g.K + kWave - 1) / kWave, g.E);
    if (dtype == BRX_DT_BF16) hipLaunchKernelGGL(k_grouped_bias<BRX_DT_BF16>, grid, dim3(kColThreads), 0, s, g);
    else hipLaunchKernelGGL(k_grouped_bias<BRX_DT_F16>, grid, dim3(kColThreads), 0, s, g);
    return hipGetLastError();
}

}  // namespace brx
