// (token, expert) pairs sorted by expert, tokens' rows into that order and back, and the gradients.
//
//   offsets[e]  = pairs of experts below e;  position[p] = offsets[e(p)] + pairs q < p of the same expert
//   order[position[p]] = p
//   dispatch    rows[position[t, j]] = x[t]
//   combine     out[t] = sum_j w[t, j] rows[position[t, j]]                    (fp32, j in order)
//   its gradient  drows[position[t, j]] = w[t, j] dout[t],  dw[t, j] = <dout[t], rows[position[t, j]]>
// Dispatch's gradient is a combine without weights, drows a dispatch with them.
//
// A pair whose expert is outside [0, E) is dropped: it takes one of the rows behind offsets[E], and its
// position is -1 - that row, so each row belongs to one pair and the rows behind the last one are cleared
// by whoever writes the rows, without a count read from memory. Sums run over a token's pairs, so there are
// no atomics and every result is the same bits on every run.
//
// A row whose width is no multiple of a 16-byte run ends in a run that overlaps the one before: both write the same
// values there. (Runs start at any address their type is aligned to.)
//
// Bound: memory. Token-centred, so that a token's row is read (or its sum written) once for its k pairs.
#include "block_ops.h"

namespace brx {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kCopies = 4;            // counters that all lanes add to come so often, 16 neighbouring pairs to one: a popular
                                      // expert is among each token's (Zipf, 16384 pairs of 128 experts: 11.0 -> 7.0 us)
// Pairs of a list whose blocks count all of it themselves, in one launch. Zipf, 128 experts, us as a graph's nodes, one launch /
// two: 4096 pairs 4.4 / 7.9, 16384 6.1 / 9.4, 24576 7.6 / 10.0, 32768 8.5 / 8.8 (60 experts 8.1 / 8.2, 512 8.6 / 10.1). The line is where
// brx.h has it, which says that up to there a plan needs no scratch; past it a call from the host has a second launch's 4 us to pay.
constexpr int kPlanSelf = 16384;

// Groups of 64 pairs a wave holds: few, so that a list is spread over CUs, more where there are so many blocks that adding up
// their counts costs more.
inline int plan_groups(int64_t n) { return n <= kPlanSelf ? 1 : n <= 64 * 4 * kPlanThreads ? 4 : 16; }
inline int plan_blocks(int64_t n) {
    const int64_t chunk = (int64_t)plan_groups(n) * kPlanThreads;
    return (int)((n + chunk - 1) / chunk);
}

// Lanes of the wave whose value is this lane's (values below 2^bits).
__device__ __forceinline__ uint64_t same_lanes(int v, int bits) {
    uint64_t m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const bool on = (v >> b) & 1;
        const uint64_t have = __ballot(on);
        m &= on ? have : ~have;
    }
    return m;
}

// Keeps a wave's LDS accesses in the order they are written (they execute in it).
__device__ __forceinline__ void wave_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

static_assert((kPlanWaves + 2 * kCopies) * (kMaxExperts + 1) * 4 <= 65536 - 1024, "the counters fit a block's LDS");

enum { kPlanAlone, kPlanCount, kPlanPlace };

// A stable counting sort. A block takes a contiguous chunk of the pairs, its waves (only as many as the chunk fills) contiguous
// parts of it, held in registers, so a pair's place is (pairs of lower experts) + (the same expert's pairs in earlier
// blocks, earlier waves, earlier groups of this wave, lower lanes). A wave's 64 pairs meet their equals by ballots of the
// id's bits, and one lane of each set of equals counts for all of it, so no order of atomics decides anything. Dropped
// pairs count as expert E. MODE: alone, each block counting all pairs (one launch), or the counts of each block and then the
// places.
template <int MODE, int G>
__global__ __launch_bounds__(kPlanThreads) void k_pairs_plan(PairsPlan p) {
    extern __shared__ int32_t hist[];                 // [waves, E1]
    const int E1 = p.E + 1;
    __shared__ int32_t wtot[kPlanWaves];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int n = p.n, base = blockIdx.x * (G * kPlanThreads), mine_n = min(n - base, G * kPlanThreads);
    const int waves = MODE == kPlanCount ? kCopies : (mine_n + G * kWave - 1) / (G * kWave);
    const int lo = base + wv * (G * kWave);
    const int bits = 32 - __builtin_clz(p.E);
    int e[G];
    if (lo < n) {                                     // (whole waves)
#pragma unroll
        for (int g = 0; g < G; ++g) e[g] = p.idx[min(lo + g * kWave + lane, n - 1)];
    }
    for (int i = tid; i < waves * E1; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    if constexpr (MODE == kPlanCount) {
        if (lo < n) {
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (lo + g * kWave + lane < n) atomicAdd(&hist[(lane >> 4) * E1 + ((unsigned)e[g] < (unsigned)p.E ? e[g] : p.E)], 1);
        }
        __syncthreads();
        if (tid < E1) {
            int v = 0;
#pragma unroll
            for (int c = 0; c < kCopies; ++c) v += hist[c * E1 + tid];
            p.counts[blockIdx.x * E1 + tid] = v;
        }
        return;
    }
    int32_t* const all = hist + kPlanWaves * E1;      // (alone, of several blocks) counts of earlier blocks' pairs, and of the rest
    int32_t* const earlier = all + kCopies * E1;
    const bool several = MODE == kPlanAlone && gridDim.x > 1;
    if (several) {                                    // uniform
        for (int i = tid; i < 2 * kCopies * E1; i += kPlanThreads) all[i] = 0;
        __syncthreads();
        int v[kPlanSelf / kPlanThreads];              // (all requested at once)
#pragma unroll
        for (int i = 0; i < kPlanSelf / kPlanThreads; ++i) v[i] = p.idx[min(i * kPlanThreads + tid, n - 1)];
#pragma unroll
        for (int i = 0; i < kPlanSelf / kPlanThreads; ++i) {
            const int q = i * kPlanThreads + tid, x = (unsigned)v[i] < (unsigned)p.E ? v[i] : p.E;
            if (q < n) atomicAdd((q < base ? earlier : all) + (lane >> 4) * E1 + x, 1);
        }
    }
    int32_t* mine = hist + wv * E1;
    uint64_t m[G];
    if (lo < n) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            e[g] = (unsigned)e[g] < (unsigned)p.E ? e[g] : p.E;
            const bool in = lo + g * kWave + lane < n;
            m[g] = same_lanes(e[g], bits) & __ballot(in);
            if (in && lane == __builtin_ctzll(m[g])) atomicAdd(&mine[e[g]], __popcll(m[g]));
        }
    }
    __syncthreads();
    // thread e: what of expert e the waves have, and earlier blocks
    int total = 0, before = 0;
    if (tid < E1) {
        if constexpr (MODE == kPlanPlace) {
#pragma unroll 8
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int v = p.counts[b * E1 + tid];
                before += b < (int)blockIdx.x ? v : 0;
                total += v;
            }
        } else if (several) {
#pragma unroll
            for (int c = 0; c < kCopies; ++c) {
                before += earlier[c * E1 + tid];
                total += all[c * E1 + tid];
            }
            total += before;
        } else {
#pragma unroll 4
            for (int w = 0; w < waves; ++w) total += hist[w * E1 + tid];
        }
    }
    const int incl = wave_incl_scan(total);
    if (lane == 63) wtot[wv] = incl;
    __syncthreads();
    int off = incl - total;
#pragma unroll
    for (int w = 0; w < kMaxExperts / kWave; ++w) off += w < wv ? wtot[w] : 0;
    if (tid < E1) {
        if (blockIdx.x == 0) p.offsets[tid] = off;    // (entry E: where the dropped ones start, the pairs kept)
        int at = off + before;
#pragma unroll 4
        for (int w = 0; w < waves; ++w) {
            const int v = hist[w * E1 + tid];
            hist[w * E1 + tid] = at;
            at += v;
        }
    }
    __syncthreads();
    if (lo >= n) return;
    int at[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const bool in = lo + g * kWave + lane < n;
        at[g] = mine[e[g]];
        wave_order();
        if (in && lane == __builtin_ctzll(m[g])) atomicAdd(&mine[e[g]], __popcll(m[g]));
        wave_order();
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
        const int q = lo + g * kWave + lane;
        if (q >= n) break;
        const int r = at[g] + __popcll(m[g] & ((1ull << lane) - 1ull));
        const bool kept = e[g] < p.E;
        p.position[q] = kept ? r : -1 - r;
        p.order[r] = kept ? q : -1;
    }
}

// ------------------------------------------------------------------ rows
constexpr int kThreads = 256;
constexpr int kAhead = 8;             // pairs of a token in flight

// The row of a position, and whether its pair is dropped.
__device__ __forceinline__ int row_of(int pos) { return pos < 0 ? -1 - pos : pos; }

// rows[position[t, j]] = (w[t, j]) x[t]; cleared where the pair is dropped. `lanes` threads a token (a power of
// two). WEIGHTED: times w, in fp32, rounded once.
template <int DT, bool WEIGHTED>
__global__ __launch_bounds__(kThreads) void k_pairs_dispatch(PairRows p, int lanes) {
    typedef typename Elem<DT>::T ET;
    constexpr int V = Elem<DT>::kVec;
    const int t = blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    if (t >= p.T) return;
    const int n = p.T * p.k;
    const int32_t* pos = p.position + (int64_t)t * p.k;
    const float* w = p.w + (WEIGHTED ? (int64_t)t * p.k : 0);
    const ET* x = (const ET*)p.x + (int64_t)t * p.x_row;
    ET* out = (ET*)p.out;
    for (int c0 = (threadIdx.x & (lanes - 1)) * V; c0 < p.H; c0 += lanes * V) {
        const int c = min(c0, p.H - V);
        if (p.H >= V) {
            const v4u_t q = get16(x + c);
            float f[V];
            if constexpr (WEIGHTED) unpack<DT>(q, f);
            for (int j = 0; j < p.k; ++j) {
                const int at = pos[j], r = row_of(at);
                v4u_t v = q;
                if constexpr (WEIGHTED) {
                    float g[V];
                    const float s = w[j];
#pragma unroll
                    for (int i = 0; i < V; ++i) g[i] = f[i] * s;
                    v = pack<DT>(g);
                }
                if (at < 0) v = v4u_t{0, 0, 0, 0};
                if (r < n) set16(out + (int64_t)r * p.H + c, v);
            }
        } else {
            for (int i = 0; i < p.H; ++i)
                for (int j = 0; j < p.k; ++j) {
                    const int at = pos[j], r = row_of(at);
                    ET v = x[i];
                    if constexpr (WEIGHTED) v = from_f<DT>(to_f<DT>(v) * w[j]);
                    if (r < n) out[(int64_t)r * p.H + i] = at < 0 ? ET(0) : v;
                }
        }
    }
}

// out[t] = sum_j (w[t, j]) rows[position[t, j]], fp32, j in order.
template <int DT, bool WEIGHTED>
__global__ __launch_bounds__(kThreads) void k_pairs_combine(PairRows p, int lanes) {
    typedef typename Elem<DT>::T ET;
    constexpr int V = Elem<DT>::kVec;
    const int t = blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
    if (t >= p.T) return;
    const int n = p.T * p.k;
    const int32_t* pos = p.position + (int64_t)t * p.k;
    const float* w = p.w + (WEIGHTED ? (int64_t)t * p.k : 0);
    const ET* rows = (const ET*)p.rows;
    ET* out = (ET*)p.out + (int64_t)t * p.H;
    for (int c0 = (threadIdx.x & (lanes - 1)) * V; c0 < p.H; c0 += lanes * V) {
        const int c = min(c0, p.H - V);
        if (p.H >= V) {
            float acc[V];
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = 0.f;
            for (int j0 = 0; j0 < p.k; j0 += kAhead) {
                // (unconditional loads, so that all are in flight; what is dropped or past k is left out by the select)
                v4u_t q[kAhead];
                bool on[kAhead];
                float s[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int j = min(j0 + u, p.k - 1), at = pos[j];
                    on[u] = j0 + u < p.k && (unsigned)at < (unsigned)n;
                    if constexpr (WEIGHTED) s[u] = w[j];
                    q[u] = get16(rows + (int64_t)(on[u] ? at : 0) * p.H + c);
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    float v[V];
                    unpack<DT>(q[u], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float a = WEIGHTED ? __builtin_fmaf(s[u], v[i], acc[i]) : acc[i] + v[i];
                        acc[i] = on[u] ? a : acc[i];
                    }
                }
            }
            set16(out + c, pack<DT>(acc));
        } else {
            for (int i = 0; i < p.H; ++i) {
                float acc = 0.f;
                for (int j = 0; j < p.k; ++j) {
                    const int at = pos[j];
                    if ((unsigned)at >= (unsigned)n) continue;
                    const float v = to_f<DT>(rows[(int64_t)at * p.H + i]);
                    acc = WEIGHTED ? __builtin_fmaf(w[j], v, acc) : acc + v;
                }
                out[i] = from_f<DT>(acc);
            }
        }
    }
}

// drows (out, or null) and dw of a combine, one wave a token: dout's chunk is read once for kAhead pairs. (drows alone are a
// dispatch with the weights.)
template <int DT>
__global__ __launch_bounds__(kThreads) void k_pairs_combine_backward(PairRows p) {
    typedef typename Elem<DT>::T ET;
    constexpr int V = Elem<DT>::kVec;
    const int lane = threadIdx.x & 63;
    const int t = blockIdx.x * (kThreads / kWave) + (threadIdx.x >> 6);
    if (t >= p.T) return;
    const int n = p.T * p.k;
    const int32_t* pos = p.position + (int64_t)t * p.k;
    const ET* d = (const ET*)p.x + (int64_t)t * p.x_row;
    const ET* rows = (const ET*)p.rows;
    ET* out = (ET*)p.out;
    for (int j0 = 0; j0 < p.k; j0 += kAhead) {
        int at[kAhead];
        float s[kAhead], dot[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = min(j0 + u, p.k - 1);
            at[u] = pos[j];
            s[u] = p.w ? p.w[(int64_t)t * p.k + j] : 1.0f;
            dot[u] = 0.f;
        }
        for (int c0 = lane * V; c0 < p.H; c0 += kWave * V) {
            const int c = min(c0, p.H - V), own = c0 - c;      // (elements below `own` are another lane's)
            if (p.H >= V) {
                v4u_t q[kAhead];
                const v4u_t dq = get16(d + c);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) q[u] = get16(rows + (int64_t)((unsigned)at[u] < (unsigned)n ? at[u] : 0) * p.H + c);
                float f[V];
                unpack<DT>(dq, f);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    float v[V];
                    unpack<DT>(q[u], v);
#pragma unroll
                    for (int i = 0; i < V; ++i) dot[u] = i >= own ? __builtin_fmaf(f[i], v[i], dot[u]) : dot[u];
                    const int r = row_of(at[u]);
                    if (out && j0 + u < p.k && r < n) {
                        float g[V];
#pragma unroll
                        for (int i = 0; i < V; ++i) g[i] = f[i] * s[u];
                        set16(out + (int64_t)r * p.H + c, at[u] < 0 ? v4u_t{0, 0, 0, 0} : pack<DT>(g));
                    }
                }
            } else {
                for (int i = 0; i < p.H; ++i) {
                    const float f = to_f<DT>(d[i]);
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int r = row_of(at[u]);
                        if (j0 + u >= p.k || r >= n) continue;
                        if (at[u] >= 0) dot[u] = __builtin_fmaf(f, to_f<DT>(rows[(int64_t)r * p.H + i]), dot[u]);
                        if (out) out[(int64_t)r * p.H + i] = at[u] < 0 ? ET(0) : from_f<DT>(f * s[u]);
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const float v = wave_sum(dot[u]);
            if (lane == 0 && j0 + u < p.k) p.dw[(int64_t)t * p.k + j0 + u] = (unsigned)at[u] < (unsigned)n ? v : 0.f;
        }
    }
}

// Threads a token's row of H values takes: one 16-byte run each, up to a block.
inline int row_lanes(int H, int vec) {
    const int runs = (H + vec - 1) / vec;
    int l = 8;
    while (l < runs && l < kThreads) l *= 2;
    return l;
}

}  // namespace

size_t pairs_plan_workspace(int64_t n, int E) {
    return n <= kPlanSelf ? 0 : (size_t)plan_blocks(n) * (E + 1) * sizeof(int32_t);
}

template <int MODE>
static hipError_t plan_launch(const PairsPlan& p, hipStream_t s) {
    const int groups = plan_groups(p.n), per = groups * kWave, blocks = p.n ? plan_blocks(p.n) : 1;
    // counters: of each wave (a list of one block has only as many as it fills), and the two of a list whose blocks count it all
    const int sets = MODE == kPlanCount ? kCopies
                     : blocks == 1 ? (p.n ? (p.n + per - 1) / per : 1) : kPlanWaves + (MODE == kPlanAlone ? 2 * kCopies : 0);
    const size_t lds = (size_t)sets * (p.E + 1) * sizeof(int32_t);
    if constexpr (MODE == kPlanAlone) hipLaunchKernelGGL((k_pairs_plan<MODE, 1>), dim3(blocks), dim3(kPlanThreads), lds, s, p);
    else if (groups == 4) hipLaunchKernelGGL((k_pairs_plan<MODE, 4>), dim3(blocks), dim3(kPlanThreads), lds, s, p);
    else hipLaunchKernelGGL((k_pairs_plan<MODE, 16>), dim3(blocks), dim3(kPlanThreads), lds, s, p);
    return hipGetLastError();
}

hipError_t launch_pairs_plan(const PairsPlan& p, hipStream_t s) {
    if (p.n <= kPlanSelf) return plan_launch<kPlanAlone>(p, s);
    const hipError_t e = plan_launch<kPlanCount>(p, s);
    return e != hipSuccess ? e : plan_launch<kPlanPlace>(p, s);
}

#define BRX_ROWS(KERNEL, DT)                                                                                           \
    do {                                                                                                               \
        const int lanes = row_lanes(p.H, Elem<DT>::kVec), per = kThreads / lanes;                                      \
        const dim3 grid((p.T + per - 1) / per);                                                                        \
        if (p.w) hipLaunchKernelGGL((KERNEL<DT, true>), grid, dim3(kThreads), 0, s, p, lanes);                         \
        else hipLaunchKernelGGL((KERNEL<DT, false>), grid, dim3(kThreads), 0, s, p, lanes);                            \
    } while (0)

hipError_t launch_pairs_dispatch(const PairRows& p, int dtype, hipStream_t s) {
    if (dtype == BRX_DT_F32) BRX_ROWS(k_pairs_dispatch, BRX_DT_F32);
    else if (dtype == BRX_DT_BF16) BRX_ROWS(k_pairs_dispatch, BRX_DT_BF16);
    else BRX_ROWS(k_pairs_dispatch, BRX_DT_F16);
    return hipGetLastError();
}

hipError_t launch_pairs_combine(const PairRows& p, int dtype, hipStream_t s) {
    if (dtype == BRX_DT_F32) BRX_ROWS(k_pairs_combine, BRX_DT_F32);
    else if (dtype == BRX_DT_BF16) BRX_ROWS(k_pairs_combine, BRX_DT_BF16);
    else BRX_ROWS(k_pairs_combine, BRX_DT_F16);
    return hipGetLastError();
}
#undef BRX_ROWS

hipError_t launch_pairs_combine_backward(const PairRows& p, int dtype, hipStream_t s) {
    const dim3 grid((p.T + 3) / 4), block(kThreads);
    if (dtype == BRX_DT_F32) hipLaunchKernelGGL(k_pairs_combine_backward<BRX_DT_F32>, grid, block, 0, s, p);
    else if (dtype == BRX_DT_BF16) hipLaunchKernelGGL(k_pairs_combine_backward<BRX_DT_BF16>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(k_pairs_combine_backward<BRX_DT_F16>, grid, block, 0, s, p);
    return hipGetLastError();
}

}  // namespace brx
