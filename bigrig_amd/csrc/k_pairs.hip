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
constexpr int kPlanOne = 16384;       // pairs one block sorts by itself
constexpr int kPlanBlocks = 64;       // blocks of a longer list, at most
constexpr int kGroup = 4;             // groups of 64 pairs a wave has in flight

// Pairs of one block: a multiple of the 64 kGroup a wave takes at a time, over all waves.
inline int plan_chunk(int64_t n) {
    const int64_t unit = (int64_t)kPlanThreads * kGroup;
    if (n <= kPlanOne) return (int)((n + kPlanThreads - 1) / kPlanThreads) * kPlanThreads;
    const int64_t per = (n + kPlanBlocks - 1) / kPlanBlocks;
    return (int)((per + unit - 1) / unit * unit);
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

enum { kPlanWhole, kPlanCount, kPlanPlace };

// A stable counting sort. A block takes a contiguous chunk of the pairs, wave w of it the w-th contiguous part,
// so a pair's place is (pairs of lower experts) + (the same expert's pairs in earlier blocks, earlier waves,
// earlier groups of this wave, lower lanes). A wave's 64 pairs meet their equals by ballots of the id's bits,
// and one lane of each set of equals counts for all of it, so the counters need no atomics across lanes.
// Dropped pairs count as expert E. MODE: a list of one block, or the counts of each block and then the places.
// 8192 / 16384 pairs of 128 experts ... us in one block, 65536 ... us in two launches.
template <int MODE>
__global__ __launch_bounds__(kPlanThreads) void k_pairs_plan(PairsPlan p, int chunk) {
    extern __shared__ int32_t lds[];
    const int E1 = p.E + 1;
    int32_t* hist = lds;                              // [waves, E1]
    __shared__ int32_t wtot[kPlanWaves];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int n = p.n, base = blockIdx.x * chunk, per = chunk / kPlanWaves, lo = base + wv * per;
    const int bits = 32 - __builtin_clz(p.E);
    for (int i = tid; i < kPlanWaves * E1; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    int32_t* mine = hist + wv * E1;
    auto load = [&](int g, int (&e)[kGroup]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kGroup; ++u) e[u] = p.idx[min(lo + (g + u) * kWave + lane, n - 1)];
#pragma unroll
        for (int u = 0; u < kGroup; ++u) e[u] = (unsigned)e[u] < (unsigned)p.E ? e[u] : p.E;
    };
    const int groups = per / kWave;
    for (int g = 0; g < groups; g += kGroup) {
        int e[kGroup];
        load(g, e);
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            const bool in = g + u < groups && lo + (g + u) * kWave + lane < n;
            const uint64_t m = same_lanes(e[u], bits) & __ballot(in);
            if (in && lane == __builtin_ctzll(m)) mine[e[u]] += __popcll(m);
            wave_order();
        }
    }
    __syncthreads();
    // thread e: the waves' counts of expert e into prefixes, their sum, what earlier blocks have of it
    int total = 0, before = 0;
    if (tid < E1) {
        for (int w = 0; w < kPlanWaves; ++w) {
            const int v = hist[w * E1 + tid];
            hist[w * E1 + tid] = total;
            total += v;
        }
        if constexpr (MODE == kPlanCount) p.counts[blockIdx.x * E1 + tid] = total;
        if constexpr (MODE == kPlanPlace) {
            total = 0;
            for (int b = 0; b < (int)gridDim.x; ++b) {
                const int v = p.counts[b * E1 + tid];
                before += b < (int)blockIdx.x ? v : 0;
                total += v;
            }
        }
    }
    if constexpr (MODE == kPlanCount) return;
    const int incl = wave_incl_scan(total);
    if (lane == 63) wtot[wv] = incl;
    __syncthreads();
    int off = incl - total;
    for (int w = 0; w < wv; ++w) off += wtot[w];
    if (tid < E1) {
        if (blockIdx.x == 0) p.offsets[tid] = off;     // (entry E: where the dropped ones start, the pairs kept)
        for (int w = 0; w < kPlanWaves; ++w) hist[w * E1 + tid] += off + before;
    }
    __syncthreads();
    for (int g = 0; g < groups; g += kGroup) {
        int e[kGroup];
        load(g, e);
#pragma unroll
        for (int u = 0; u < kGroup; ++u) {
            const int q = lo + (g + u) * kWave + lane;
            const bool in = g + u < groups && q < n;
            const uint64_t m = same_lanes(e[u], bits) & __ballot(in);
            const int at = mine[e[u]];
            wave_order();
            if (in) {
                const int r = at + __popcll(m & ((1ull << lane) - 1ull));
                const bool kept = e[u] < p.E;
                p.position[q] = kept ? r : -1 - r;
                p.order[r] = kept ? q : -1;
                if (lane == __builtin_ctzll(m)) mine[e[u]] = at + __popcll(m);
            }
            wave_order();
        }
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

// drows (out) and dw of a combine, one wave a token: dout's chunk is read once for kAhead pairs. Either output may
// be null.
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
                if (p.dw) {
#pragma unroll
                    for (int u = 0; u < kAhead; ++u)
                        q[u] = get16(rows + (int64_t)((unsigned)at[u] < (unsigned)n ? at[u] : 0) * p.H + c);
                }
                float f[V];
                unpack<DT>(dq, f);
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (p.dw) {
                        float v[V];
                        unpack<DT>(q[u], v);
#pragma unroll
                        for (int i = 0; i < V; ++i) dot[u] = i >= own ? __builtin_fmaf(f[i], v[i], dot[u]) : dot[u];
                    }
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
                        if (p.dw && at[u] >= 0) dot[u] = __builtin_fmaf(f, to_f<DT>(rows[(int64_t)r * p.H + i]), dot[u]);
                        if (out) out[(int64_t)r * p.H + i] = at[u] < 0 ? ET(0) : from_f<DT>(f * s[u]);
                    }
                }
            }
        }
        if (p.dw) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const float v = wave_sum(dot[u]);
                if (lane == 0 && j0 + u < p.k) p.dw[(int64_t)t * p.k + j0 + u] = (unsigned)at[u] < (unsigned)n ? v : 0.f;
            }
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
    if (n <= kPlanOne) return 0;
    const int chunk = plan_chunk(n);
    return (size_t)((n + chunk - 1) / chunk) * (E + 1) * sizeof(int32_t);
}

hipError_t launch_pairs_plan(const PairsPlan& p, hipStream_t s) {
    const int chunk = plan_chunk(p.n);
    const int blocks = (p.n + chunk - 1) / chunk;
    const size_t lds = (size_t)kPlanWaves * (p.E + 1) * sizeof(int32_t);
    if (p.n <= kPlanOne) {
        hipLaunchKernelGGL(k_pairs_plan<kPlanWhole>, dim3(1), dim3(kPlanThreads), lds, s, p, chunk);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_pairs_plan<kPlanCount>, dim3(blocks), dim3(kPlanThreads), lds, s, p, chunk);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_pairs_plan<kPlanPlace>, dim3(blocks), dim3(kPlanThreads), lds, s, p, chunk);
    return hipGetLastError();
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
