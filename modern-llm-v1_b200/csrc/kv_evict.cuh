// Eviction from a KV cache by the attention weight that its keys have received.
//
// Per (batch, KV head), of n = lens[b] rows min(n, keep) stay: those whose position is among the newest `recent`
// (position > newest - recent), then those of the largest weight; of equal ones the lower row.  Rows that stay and lie below `keep`
// are not touched; the j-th of those behind goes to the j-th place that has become free.  (The rows of a cache need no order: they
// carry their positions in their rotation.  So at most n - keep rows move, and no row is read that another is written over, where
// closing the gaps in order would move nearly all and in sequence.)  K and V change in place; weights and positions are read from one
// pair of arrays and written whole to another, so that every CTA of a unit can decide for itself, from inputs that nobody changes.
//
// kv_evict_kernel: a CTA reads all of its unit's weights and positions, finds the keep-th largest by digits of 11, 11 and 10 bits
// (histograms in shared memory), numbers the free places and the rows to move, and
//   LIST = false  moves its share of them (p.ranks CTAs per unit, each of which selects for itself): few units
//   LIST = true   leaves them in the workspace for kv_move_kernel, whose CTAs take 128 moves each, whichever unit they are of
// What bounds it: the moved bytes where units are many and long (B=32 L<=6000 keep=2500 4 heads D=128: 30 to 32 us; cold and one at a time
// the selection's chain on one SM per unit takes 16 of them and 80 MB of moves 17.5; 45 us with one kernel whose CTAs had a unit each, 39 with
// four CTAs a unit), else that chain: status and length, the inputs, three histograms and two sweeps, about 1 us each (one sequence, L=2048
// 2 heads D=64: 8.1 us).
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
    int2* moves;              // LIST: [unit][most] (from, to)
    int* n_moves;             // LIST: [unit]
    int most, blocks;         // most moves of a unit, blocks of kv_move_kernel per unit
};

constexpr int kEvictThreads = 1024, kEvictWarps = kEvictThreads / 32, kEvictBins = 2048;
constexpr int kEvictWindow = 2048;          // moves that are listed at a time
constexpr int kEvictMaxKeys = 46 * 1024;    // rows whose keys fit shared memory
constexpr int kEvictFixedSmem = kEvictBins * 4 + kEvictWindow * 8;

// The order of the weights as unsigned numbers: -0 is 0, NaN is above all (as in a sort), protected rows above that.
__device__ __forceinline__ uint32_t evict_key(float w, bool recent) {
    if (recent) return 0xffffffffu;
    if (w != w) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// What the warps in front of this one have counted, of two counts at once (each lane passes its warp's), and the total of the first.
// s_red: [2][warps], a place that no earlier exchange may still be read from
__device__ __forceinline__ int2 evict_warps_before(int a, int b, int2* s_red, int* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s_red[warp] = make_int2(a, b);
    __syncthreads();
    const int2 own = s_red[lane];
    int2 incl = own;
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl.x, o), y = __shfl_up_sync(0xffffffffu, incl.y, o);
        if (lane >= o) incl.x += x, incl.y += y;
    }
    *total = __shfl_sync(0xffffffffu, incl.x, 31);
    return make_int2(__shfl_sync(0xffffffffu, incl.x - own.x, warp), __shfl_sync(0xffffffffu, incl.y - own.y, warp));
}
static_assert(kEvictWarps == 32, "a lane per warp");

// Moves `m` rows of K and V, from[e] to to[e]: 16 bytes a lane, a move's K and V row side by side
template <int D, int WARPS, int U, typename Pair>
__device__ __forceinline__ void evict_move(uint16_t* k, uint16_t* v, int m, int warp, int lane, Pair pair) {
    constexpr int LPM = D / 4;  // lanes per move; U: moves of a lane in flight
    const int sub = lane / LPM, li = lane % LPM;
    uint16_t* const rows = (li >= LPM / 2 ? v : k) + (li % (LPM / 2)) * 8;
    constexpr int STEP = WARPS * (32 / LPM);
    for (int e0 = warp * (32 / LPM) + sub; e0 < m; e0 += U * STEP) {
        uint4 x[U];
        int to[U];
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (e0 + i * STEP < m) {
                const int2 ft = pair(e0 + i * STEP);
                x[i] = __ldcs(reinterpret_cast<const uint4*>(rows + size_t(ft.x) * D));
                to[i] = ft.y;
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (e0 + i * STEP < m) *reinterpret_cast<uint4*>(rows + size_t(to[i]) * D) = x[i];
    }
}

// BIG: the keys do not fit shared memory and are made anew from weight and position at every sweep
template <int D, bool BIG, bool LIST>
__global__ void __launch_bounds__(kEvictThreads, 1) kv_evict_kernel(const EvictParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    int* s_hist = reinterpret_cast<int*>(smem);            // [kEvictBins]
    int* s_from = s_hist + kEvictBins;                     // [kEvictWindow] rows that move, in order
    int* s_to = s_from + kEvictWindow;                     // [kEvictWindow] free places, in order
    uint32_t* s_key = reinterpret_cast<uint32_t*>(s_to + kEvictWindow);  // [n]
    __shared__ int s_max[kEvictWarps], s_pick[3][3], s_status;
    __shared__ int2 s_red[5][kEvictWarps];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned below = (1u << lane) - 1u;
    const int ranks = LIST ? 1 : p.ranks, unit = int(blockIdx.x) / ranks, rank = int(blockIdx.x) - unit * ranks;
    const size_t base = size_t(unit) * p.L_cap;
    const float* const w = p.w + base;
    const int* const pos = p.pos + base;
    float* const w_out = p.w_out + base;
    int* const pos_out = p.pos_out + base;
    grid_dep_wait();
    if (LIST) grid_dep_launch();
    // The status word, which other streams and the host may change at any time: a CTA goes by what one thread has read once, since rows
    // are listed and moved by all threads together.  (Looked at where something is written: no round trip of its own.)
    const int status = *reinterpret_cast<const volatile int*>(p.status);
    const int n = p.lens ? max(0, min(__ldg(p.lens + unit / p.Hkv), p.L)) : p.L;
    const int left = min(n, p.keep);
    // this CTA's share of the rows whose weight and position it writes
    const int r0 = int((long long)p.L_cap * rank / ranks), r1 = int((long long)p.L_cap * (rank + 1) / ranks);
    if (n <= p.keep) {
        if (LIST && tid == 0) p.n_moves[unit] = 0;
        if (__syncthreads_or(status != 0)) return;
        for (int i = r0 + tid; i < r1; i += kEvictThreads) w_out[i] = i < n ? __ldg(w + i) : 0.f, pos_out[i] = i < n ? __ldg(pos + i) : -1;
        return;
    }

    // ---- the newest position; rows beyond newest - recent are protected.  (Weights come in the same round trip.)
    int newest = INT_MIN;
    for (int i0 = tid; i0 < n; i0 += 8 * kEvictThreads) {
        int at[8];
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k * kEvictThreads;
            at[k] = INT_MIN, x[k] = 0.f;
            if (i < n) {
                at[k] = __ldg(pos + i);
                if (!BIG) x[k] = __ldg(w + i);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int i = i0 + k * kEvictThreads;
            newest = max(newest, at[k]);
            if (!BIG && i < n) s_key[i] = __float_as_uint(x[k]);
        }
    }
    for (int o = 16; o > 0; o >>= 1) newest = max(newest, __shfl_xor_sync(0xffffffffu, newest, o));
    if (lane == 0) s_max[warp] = newest;
    if (tid == 0) s_status = status;
    for (int i = tid; i < kEvictBins; i += kEvictThreads) s_hist[i] = 0;
    __syncthreads();
    newest = s_max[lane];
    for (int o = 16; o > 0; o >>= 1) newest = max(newest, __shfl_xor_sync(0xffffffffu, newest, o));
    const long long first = (long long)newest - p.recent;
    auto key_of = [&](int i) { return BIG ? evict_key(__ldg(w + i), __ldg(pos + i) > first) : s_key[i]; };

    // ---- the left-th largest key, by its digits from the top: `want` of the rows that share the digits so far are needed
    uint32_t digits = 0, mask = 0;
    int want = left, equal = 0, total;
    for (int round = 0; round < 3; ++round) {
        const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
        if (round == 0) {
            for (int i = tid; i < n; i += kEvictThreads) {
                const uint32_t key = evict_key(BIG ? __ldg(w + i) : __uint_as_float(s_key[i]), __ldg(pos + i) > first);
                if (!BIG) s_key[i] = key;
                atomicAdd(&s_hist[key >> 21], 1);
            }
        } else {
            for (int i = tid; i < n; i += kEvictThreads) {
                const uint32_t key = key_of(i);
                if ((key & mask) == digits) atomicAdd(&s_hist[(key >> shift) & ((1u << bits) - 1u)], 1);
            }
        }
        __syncthreads();
        // thread t has the bins top - 2t and top - 2t - 1, from the largest down, and clears them for the next round
        int2* const mine = reinterpret_cast<int2*>(s_hist) + kEvictBins / 2 - 1 - tid;
        const int2 c = *mine;
        *mine = make_int2(0, 0);
        int incl = c.x + c.y;
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const int above = evict_warps_before(__shfl_sync(0xffffffffu, incl, 31), 0, s_red[round], &total).x + incl - c.x - c.y;
        if (above < want && above + c.y >= want) s_pick[round][0] = kEvictBins - 1 - 2 * tid, s_pick[round][1] = want - above, s_pick[round][2] = c.y;
        else if (above + c.y < want && above + c.y + c.x >= want)
            s_pick[round][0] = kEvictBins - 2 - 2 * tid, s_pick[round][1] = want - above - c.y, s_pick[round][2] = c.x;
        __syncthreads();
        digits |= uint32_t(s_pick[round][0]) << shift;
        want = s_pick[round][1];
        equal = s_pick[round][2];
        mask |= ((1u << bits) - 1u) << shift;
    }
    // Rows of a larger key stay, and the first `want` of the `equal` whose key is `digits`.

    // ---- every warp has a run of rows
    const int run = ((n + kEvictWarps - 1) / kEvictWarps + 31) & ~31, w0 = min(n, warp * run), w1 = min(n, w0 + run);
    int equal0 = 0;  // rows of that key in front of the warp's
    if (equal > want) {  // (else all of them stay)
        int count = 0;
        for (int i0 = w0; i0 < w1; i0 += 32) count += __popc(__ballot_sync(0xffffffffu, i0 + lane < w1 && key_of(i0 + lane) == digits));
        equal0 = evict_warps_before(count, 0, s_red[3], &total).x;
    }
    // visit(row, stays) for the warp's rows, 32 at a time
    auto sweep = [&](auto visit) {
        int before = equal0;
        for (int i0 = w0; i0 < w1; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t key = i < w1 ? key_of(i) : 0u;
            const unsigned same = __ballot_sync(0xffffffffu, i < w1 && key == digits);
            visit(i, i < w1 && (key > digits || (key == digits && (equal <= want || before + __popc(same & below) < want))));
            before += __popc(same);
        }
    };
    int holes = 0, moves = 0;
    sweep([&](int i, bool stays) {
        holes += __popc(__ballot_sync(0xffffffffu, i < left && !stays));
        moves += __popc(__ballot_sync(0xffffffffu, i >= left && stays));
    });
    const int2 at0 = evict_warps_before(holes, moves, s_red[4], &total);  // as many moves as free places

    if (s_status != 0) {
        if (LIST && tid == 0) p.n_moves[unit] = 0;
        return;
    }
    // ---- this CTA's share of the moves, a window at a time; with the first, the weights and positions that do not move
    const int m0 = int((long long)total * rank / ranks), m1 = int((long long)total * (rank + 1) / ranks);
    bool first_window = true;
    for (int at = m0; at < m1 || first_window; at += kEvictWindow) {
        const int end = min(m1, at + kEvictWindow), m = end - at;
        int hole = at0.x, move = at0.y;
        sweep([&](int i, bool stays) {
            const bool is_hole = i < left && !stays, is_move = i >= left && stays;
            const unsigned hb = __ballot_sync(0xffffffffu, is_hole), mb = __ballot_sync(0xffffffffu, is_move);
            const int h = hole + __popc(hb & below), e = move + __popc(mb & below);
            if (is_hole && h >= at && h < end) s_to[h - at] = i;
            if (is_move && e >= at && e < end) s_from[e - at] = i;
            hole += __popc(hb), move += __popc(mb);
            if (first_window && i < left && stays && i >= r0 && i < r1) w_out[i] = __ldg(w + i), pos_out[i] = __ldg(pos + i);
        });
        if (first_window)
            for (int i = max(r0, left) + tid; i < r1; i += kEvictThreads) w_out[i] = 0.f, pos_out[i] = -1;
        first_window = false;
        __syncthreads();
        if (LIST) {
            for (int e = tid; e < m; e += kEvictThreads) p.moves[size_t(unit) * p.most + at + e] = make_int2(s_from[e], s_to[e]);
        } else {
            evict_move<D, kEvictWarps, 4>(p.k + base * D, p.v + base * D, m, warp, lane, [&](int e) { return make_int2(s_from[e], s_to[e]); });
        }
        for (int e = tid; e < m; e += kEvictThreads) w_out[s_to[e]] = __ldg(w + s_from[e]), pos_out[s_to[e]] = __ldg(pos + s_from[e]);
        __syncthreads();
    }
    if (LIST && tid == 0) p.n_moves[unit] = total;
}

// (What it needs is bytes in flight: with 64 moves a CTA, four per lane in flight and the list read behind its length it took 22 us of B=32
// L<=6000 keep=2500 4 heads D=128, three round trips per CTA in six waves of CTAs.)
constexpr int kMoveThreads = 256, kMoveRows = 128;  // moves of a CTA
template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const EvictParams p) {
    __shared__ int2 s_move[kMoveRows];
    const int tid = threadIdx.x, unit = int(blockIdx.x) / p.blocks, e0 = (int(blockIdx.x) - unit * p.blocks) * kMoveRows;
    grid_dep_wait();
    // (Not a second look at the status word: what is listed is moved, as the weights and positions have been, and a unit that was not
    // selected has no moves.)
    const int m = min(kMoveRows, __ldcg(p.n_moves + unit) - e0);
    if (tid < kMoveRows && e0 + tid < p.most) s_move[tid] = __ldcg(p.moves + size_t(unit) * p.most + e0 + tid);  // (some may not be set)
    if (m <= 0) return;
    __syncthreads();
    const size_t base = size_t(unit) * p.L_cap * D;
    evict_move<D, kMoveThreads / 32, 8>(p.k + base, p.v + base, m, tid >> 5, tid & 31, [&](int e) { return s_move[e]; });
}

}  // namespace b200attn
