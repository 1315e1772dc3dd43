// Eviction from a KV cache by the attention weight that its keys have received.
//
// Per (batch, KV head), of n = lens[b] rows min(n, keep) stay: those whose position is among the newest `recent`
// (position > newest - recent), then those of the largest weight; of equal ones the lower row.  Rows that stay and lie below `keep`
// are not touched; the j-th of those behind goes to the j-th place that has become free.  (The rows of a cache need no order: they
// carry their positions in their rotation.  So at most n - keep rows move, and no row is read that another is written over, where
// closing the gaps in order would move nearly all and in sequence.)  K and V change in place; weights and positions are read from one
// pair of arrays and written whole to another, so that every CTA of a unit can decide for itself, from inputs that nobody changes:
//
// A CTA (p.ranks of them per unit) reads all of its unit's weights and positions, finds the keep-th largest by digits of 11, 11
// and 10 bits (histograms in shared memory), numbers the free places and the rows to move, and moves its share of them.
// What bounds it: the moved bytes where units are many and long; else the chain of reading, three histograms and three sweeps.
#pragma once

#include <limits.h>

#include "ptx.cuh"

namespace b200attn {

struct EvictParams {
    uint16_t *k, *v;          // [B, Hkv, L_cap, D]
    const float* w;           // [B, Hkv, L_cap]
    const int* pos;           // [B, Hkv, L_cap]
    float* w_out;
    int* pos_out;
    const int* lens;          // [B] or nullptr: L
    const int* status;
    int L, L_cap, Hkv, keep, recent;
    int ranks;                // CTAs per unit
};

constexpr int kEvictThreads = 512, kEvictWarps = kEvictThreads / 32, kEvictBins = 2048;
constexpr int kEvictWindow = 2048;          // moves that are listed at a time
constexpr int kEvictMaxKeys = 46 * 1024;    // rows whose keys fit shared memory
constexpr int kEvictFixedSmem = kEvictBins * 4 + 2 * kEvictWindow * 4;

// The order of the weights as unsigned numbers: -0 is 0, NaN is above all (as in a sort), protected rows above that.
__device__ __forceinline__ uint32_t evict_key(float w, bool recent) {
    if (recent) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// sum over the block of one value per thread, to all threads
__device__ __forceinline__ int evict_block_max(int v, int* s_red) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s_red[0];
    for (int i = 1; i < kEvictWarps; ++i) v = max(v, s_red[i]);
    return v;
}
// what the warps in front of this one have counted (each lane passes the warp's count), and the total
__device__ __forceinline__ int evict_warps_before(int count, int* s_red, int* total) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = count;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < kEvictWarps; ++i) {
        if (i < int(threadIdx.x >> 5)) before += s_red[i];
        all += s_red[i];
    }
    *total = all;
    return before;
}

// BIG: the keys do not fit shared memory and are made anew from weight and position at every sweep
template <int D, bool BIG>
__global__ void __launch_bounds__(kEvictThreads) kv_evict_kernel(const EvictParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    int* s_hist = reinterpret_cast<int*>(smem);        // [kEvictBins]
    int* s_hole = s_hist + kEvictBins;                 // [kEvictWindow] free places, in order
    int* s_move = s_hole + kEvictWindow;               // [kEvictWindow] rows that move, in order
    uint32_t* s_key = reinterpret_cast<uint32_t*>(s_move + kEvictWindow);  // [n]
    __shared__ int s_red[kEvictWarps], s_pick[2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned below = (1u << lane) - 1u;
    const int ranks = p.ranks, unit = int(blockIdx.x) / ranks, rank = int(blockIdx.x) - unit * ranks;
    const size_t base = size_t(unit) * p.L_cap;
    const float* const w = p.w + base;
    const int* const pos = p.pos + base;
    float* const w_out = p.w_out + base;
    int* const pos_out = p.pos_out + base;
    grid_dep_wait();
    if (*reinterpret_cast<const volatile int*>(p.status) != 0) return;
    const int n = p.lens ? max(0, min(__ldg(p.lens + unit / p.Hkv), p.L)) : p.L;
    const int left = min(n, p.keep);
    // this CTA's share of the rows whose weight and position it writes
    const int r0 = int((long long)p.L_cap * rank / ranks), r1 = int((long long)p.L_cap * (rank + 1) / ranks);
    for (int i = max(r0, left) + tid; i < r1; i += kEvictThreads) w_out[i] = 0.f, pos_out[i] = -1;
    if (n <= p.keep) {
        for (int i = r0 + tid; i < min(r1, n); i += kEvictThreads) w_out[i] = __ldg(w + i), pos_out[i] = __ldg(pos + i);
        return;
    }

    // ---- the newest position; rows beyond newest - recent are protected
    int newest = INT_MIN;
    for (int i = tid; i < n; i += kEvictThreads) {
        const int at = __ldg(pos + i);
        newest = max(newest, at);
        if (!BIG) s_key[i] = uint32_t(at);
    }
    newest = evict_block_max(newest, s_red);
    const long long first = (long long)newest - p.recent;
    if (!BIG)
        for (int i = tid; i < n; i += kEvictThreads) s_key[i] = evict_key(__ldg(w + i), int(s_key[i]) > first);
    auto key_of = [&](int i) { return BIG ? evict_key(__ldg(w + i), __ldg(pos + i) > first) : s_key[i]; };

    // ---- the left-th largest key, by its digits from the top: `want` of the rows that share the digits so far are needed
    uint32_t digits = 0, mask = 0;
    int want = left;
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
        for (int i = tid; i < kEvictBins; i += kEvictThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i = tid; i < n; i += kEvictThreads) {
            const uint32_t key = key_of(i);
            if ((key & mask) == digits) atomicAdd(&s_hist[(key >> shift) & ((1u << bits) - 1u)], 1);
        }
        __syncthreads();
        // thread t has the bins top - 4t .. top - 4t - 3, from the largest down
        int c[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) c[k] = s_hist[kEvictBins - 1 - 4 * tid - k], sum += c[k];
        int incl = sum;
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        int total, above = evict_warps_before(__shfl_sync(0xffffffffu, incl, 31), s_red, &total) + incl - sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (above < want && above + c[k] >= want) s_pick[0] = kEvictBins - 1 - 4 * tid - k, s_pick[1] = want - above;
            above += c[k];
        }
        __syncthreads();
        digits |= uint32_t(s_pick[0]) << shift;
        want = s_pick[1];
        mask |= ((1u << bits) - 1u) << shift;
    }
    // rows of a larger key stay, and the first `want` of those whose key is `digits`

    // ---- every warp has a run of rows; what lies in front of it: equal keys, free places, rows that move
    const int run = ((n + kEvictWarps - 1) / kEvictWarps + 31) & ~31, w0 = min(n, warp * run), w1 = min(n, w0 + run);
    int total, count = 0;
    for (int i0 = w0; i0 < w1; i0 += 32) count += __popc(__ballot_sync(0xffffffffu, i0 + lane < w1 && key_of(i0 + lane) == digits));
    const int equal0 = evict_warps_before(count, s_red, &total);
    // visit(row, stays) for the warp's rows, 32 at a time
    auto sweep = [&](auto visit) {
        int equal = equal0;
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t key = i < w1 ? key_of(i) : 0u;
            const unsigned same = __ballot_sync(0xffffffffu, i < w1 && key == digits);
            visit(i, i < w1 && (key > digits || (key == digits && equal + __popc(same & below) < want)));
            equal += __popc(same);
        }
    };
    int holes = 0, moves = 0;
    sweep([&](int i, bool stays) {
        holes += __popc(__ballot_sync(0xffffffffu, i < left && !stays));
        moves += __popc(__ballot_sync(0xffffffffu, i >= left && stays));
    });
    const int hole0 = evict_warps_before(holes, s_red, &total);
    const int move0 = evict_warps_before(moves, s_red, &total);  // as many moves as holes

    // ---- this CTA's share of the moves, a window at a time
    const int m0 = int((long long)total * rank / ranks), m1 = int((long long)total * (rank + 1) / ranks);
    bool first_window = true;
    for (int at = m0; at < m1 || first_window; at += kEvictWindow) {
        const int end = min(m1, at + kEvictWindow);
        int hole = hole0, move = move0;
        sweep([&](int i, bool stays) {
            const bool is_hole = i < left && !stays, is_move = i >= left && stays;
            const unsigned hb = __ballot_sync(0xffffffffu, is_hole), mb = __ballot_sync(0xffffffffu, is_move);
            const int h = hole + __popc(hb & below), m = move + __popc(mb & below);
            if (is_hole && h >= at && h < end) s_hole[h - at] = i;
            if (is_move && m >= at && m < end) s_move[m - at] = i;
            hole += __popc(hb), move += __popc(mb);
            if (first_window && i < left && stays && i >= r0 && i < r1) w_out[i] = __ldg(w + i), pos_out[i] = __ldg(pos + i);
        });
        first_window = false;
        __syncthreads();
        // 16 bytes a lane: the K row and the V row of 32 / (D / 4) moves per warp
        constexpr int LPM = D / 4;  // lanes per move
        constexpr int U = 4;
        const int sub = lane / LPM, li = lane % LPM;
        const bool is_v = li >= LPM / 2;
        uint16_t* const rows = (is_v ? p.v : p.k) + base * D + (li % (LPM / 2)) * 8;
        const int m = end - at, step = kEvictWarps * (32 / LPM);
        for (int e0 = warp * (32 / LPM) + sub; e0 < m; e0 += U * step) {
            uint4 x[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (e0 + k * step < m) x[k] = __ldcs(reinterpret_cast<const uint4*>(rows + size_t(s_move[e0 + k * step]) * D));
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (e0 + k * step < m) *reinterpret_cast<uint4*>(rows + size_t(s_hole[e0 + k * step]) * D) = x[k];
        }
        for (int e = tid; e < m; e += kEvictThreads) w_out[s_hole[e]] = __ldg(w + s_move[e]), pos_out[s_hole[e]] = __ldg(pos + s_move[e]);
        __syncthreads();
    }
}

}  // namespace b200attn
