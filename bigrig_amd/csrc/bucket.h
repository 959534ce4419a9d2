// The bucketing of (token, expert) pairs, one block per expert: k_bucket (k_prefill.hip) and launches that
// do it beside other work.
#pragma once

#include <type_traits>

#include "brx_internal.h"

namespace brx {
namespace {

// Pairs are read coalesced: in each pass of 1024 PER pairs, wave w takes the 64 PER pairs
// [64 PER w, 64 PER (w + 1)) and its lane l the pairs l + 64 i (i < PER), so a load instruction
// reads 64 consecutive pairs, and the histogram's LDS atomics of one instruction (8 tokens x
// top-8, distinct experts within a token) hit one address at most 8 times. The stable compaction
// of a pass is PER ballots per wave and one scan of the 16 wave totals. PER is 16 for many pairs
// (one pass of 2048 top-8 tokens), and 2 or 4 for up to 2048 or 8192: there the launch is bound by
// its cold code and chain of barriers, not by the pairs (one kernel of 16 pairs a lane, 10 KB of
// code, took 7.8 us for 256 pairs and 13.5 for 2709 pairs of 257 experts; now 3.6 and 4.8).
constexpr int kBucketThreads = 1024;
constexpr int kBucketListMax = 8192;                          // pairs an LDS list may hold

// The experts of a lane's pairs pb + 64 i (i < PER; id E for the shared expert's pairs past the P
// routed ones). The loads are unconditional (index clamped into the routed pairs), so a lane's
// are in flight together rather than one round trip each.
template <int PER>
__device__ __forceinline__ void bucket_experts(const int32_t* __restrict__ pexp, int pb, int P, int E, int emax,
                                               int ex[PER]) {
    if (P > 0) {   // uniform
#pragma unroll
        for (int i = 0; i < PER; ++i) ex[i] = pexp[min(pb + i * kWave, P - 1)];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) ex[i] = pb + i * kWave < P ? min(max(ex[i], 0), emax) : E;
}

// Block e of the bucketing (kBucketThreads threads, (E_ext + lcap) words of dynamic LDS).
template <int PER>
__device__ __forceinline__ void bucket_block(int e, const int32_t* __restrict__ pexp, int P, int E, int E_ext, int T_sh,
                                             int lbm, int slack, const int32_t* __restrict__ g2s, int capacity, int host,
                                             int32_t* __restrict__ err, int32_t* __restrict__ order,
                                             int32_t* __restrict__ offsets, int32_t* __restrict__ tile_start,
                                             int4* __restrict__ tinfo, int lcap) {
    // E_ext = E + 1 when a shared expert exists (id E); T_sh shared pairs follow the P routed; the M
    // tile height is 1 << lbm, and an expert's last full tile takes up to `slack` rows more. LDS: the
    // histogram [E_ext], then a list of up to lcap of this expert's pairs.
    extern __shared__ int32_t hist[];
    int32_t* list = hist + E_ext;
    constexpr int kNw = kBucketThreads / kWave;
    constexpr int kPass = kBucketThreads * PER;
    __shared__ int32_t wsum[kNw];
    __shared__ int32_t base_s[3];
    const int BM = 1 << lbm;
    const int P_ext = P + T_sh;
    const int emax = E_ext - 1;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint64_t below = (1ull << lane) - 1ull;
    int slot = 0;   // the slot code: a slot, -2 - e for an expert read from host backing
    if (tinfo && e < E && g2s) {
        const int v = g2s[e];
        slot = v >= 0 ? min(v, capacity - 1) : (host ? -2 - e : kAbsentCode);
    }
    for (int i = tid; i < E_ext; i += kBucketThreads) hist[i] = 0;
    __syncthreads();
    // This expert's pairs of the pass at p0, in pair order (pass, wave, i, lane), handed to put(place,
    // pair) from place `run` on; returns the pass's count. COUNT also counts every pair's expert
    // into the histogram (each block needs all counts below its own expert).
    auto compact = [&](int p0, int run, auto count, auto put) __attribute__((always_inline)) {
        const int pb = p0 + wv * (kWave * PER) + lane;
        int ex[PER];
        bucket_experts<PER>(pexp, pb, P, E, emax, ex);
        uint64_t m[PER];
        int cnt = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool in = pb + i * kWave < P_ext;
            if (decltype(count)::value && in) atomicAdd(&hist[ex[i]], 1);
            m[i] = __ballot(in && ex[i] == e);
            cnt += __popcll(m[i]);
        }
        if (lane == 0) wsum[wv] = cnt;
        __syncthreads();
        // lane w < 16: the total of wave w; its prefix below this wave and the pass's total
        const int incl = wave_incl_scan(lane < kNw ? wsum[lane] : 0);
        const int before = __builtin_amdgcn_readlane(incl, max(wv - 1, 0));
        const int total = __builtin_amdgcn_readlane(incl, kNw - 1);
        int dst = run + (wv > 0 ? before : 0);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if ((m[i] >> lane) & 1ull) put(dst + __popcll(m[i] & below), pb + i * kWave);
            dst += __popcll(m[i]);
        }
        __syncthreads();
        return total;
    };
    // rows of the last tile of n pairs where it is not full; up to `slack` of them join the tile before
    auto last_rows = [&](int n) __attribute__((always_inline)) {
        const int r = n & (BM - 1);
        return r <= slack && n >= BM ? 0 : r;
    };
    int run = 0;
    for (int p0 = 0; p0 < P_ext; p0 += kPass)
        run += compact(p0, run, std::true_type{}, [&](int q, int p) { if (q < lcap) list[q] = p; });
    if (wv == 0) {
        // expert e's run offset (counts of the experts before it) and its tiles' places in the
        // tile list, which holds the tiles of more than BM / 2 rows of every expert first, then
        // the smaller ones (at most one per expert, its last), each class in expert order, so
        // the GEMMs take the long tiles first. The two counts of a class pair share a word (a
        // call has fewer than 2^16 small tiles, one an expert).
        int off = 0, below_e = 0, big_all = 0, small_all = 0, big = 0;
        for (int j = lane; j < E_ext; j += 64) {
            const int n = hist[j], r = last_rows(n);
            const int nb = (n >> lbm) + (r > BM / 2 ? 1 : 0), ns = (r > 0 && r <= BM / 2) ? 1 : 0;
            if (j < e) { off += n; big += nb; below_e += ns; }
            big_all += nb;
            small_all += ns;
        }
        off = wave_incl_scan(off);          // lane 63 holds the sums
        big = wave_incl_scan(big);
        big_all = wave_incl_scan(big_all);
        const int small2 = wave_incl_scan(below_e | (small_all << 16));
        if (lane == 63) {
            const int small = small2 & 0xFFFF, smalls = small2 >> 16;
            base_s[0] = off;
            base_s[1] = big;
            base_s[2] = big_all + small;
            offsets[e] = off;
            tile_start[e] = big;
            if (e == E_ext - 1) {
                offsets[E_ext] = P_ext;
                tile_start[E_ext] = big_all + smalls;   // tiles in all (what the GEMMs read)
            }
        }
    }
    __syncthreads();
    const int n = hist[e], off = base_s[0];
    if (tinfo) {
        const int big = base_s[1], small = base_s[2];
        if (slot == kAbsentCode && n > 0 && tid == 0 && err) {
            err[1] = e;
            err[0] = 1;
        }
        const int all = (n >> lbm) + (last_rows(n) > 0 ? 1 : 0);
        for (int j = tid; j < all; j += kBucketThreads) {
            const int rows = j == all - 1 ? n - j * BM : BM;
            tinfo[rows > BM / 2 ? big + j : small] = make_int4(e, off + j * BM, rows, slot);
        }
    }
    if (n <= lcap) {
        // the run, copied out in order (coalesced)
        for (int i = tid; i < n; i += kBucketThreads) order[off + i] = list[i];
        return;
    }
    // the expert's pairs did not fit the LDS list: a second pass compacts straight into the run
    if constexpr (PER > 4) {
        run = off;
        for (int p0 = 0; p0 < P_ext; p0 += kPass)
            run += compact(p0, run, std::false_type{}, [&](int q, int p) { order[q] = p; });
    }
}

// The widest PER loads (bucket_block's template argument) a call of so many pairs takes, and the pairs its LDS
// lists hold (an expert with more takes a second pass over the pairs).
inline int bucket_per(int P_ext) { return P_ext <= 2 * kBucketThreads ? 2 : P_ext <= kBucketListMax ? 4 : 16; }
inline int bucket_list(int P_ext) { return P_ext < kBucketListMax ? P_ext : kBucketListMax; }

}  // namespace
}  // namespace brx
