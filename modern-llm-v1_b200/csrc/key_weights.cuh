// The attention weight that each cached key has received, what an eviction (kv_evict.cuh) goes by:
//
//   w[b, hk, key] += sum over the heads h of the group and the query rows t that see the key of  p = exp(scale q[h, t] . k[key] - lse[h, t])
//
// with lse the rows' logsumexp over all keys they see, so p is the softmax's probability.
//
// One new token per sequence: the decode kernel leaves its scores (kDecodeScores) and decode_weights_kernel, behind it, has only to
// take the exponentials against the final lse: 4 G bytes a key written and read through L2 beside the 4 D of its K and V rows, instead
// of a second pass over K.  Measured on B200 against the decode alone, us: B=1 L=1500 16/4 D=128 8.6 and 6.0, B=32 L<=4096 16/4 D=64 22.2 to 24.3
// and 18.4: the second launch and the scores.
//
// A chunk of new tokens: key_weights_kernel computes S^T = K Q^T by tiles of 128 keys (lanes of tensor memory) and 128 query rows
// (columns), so that a key's sum runs inside a thread and needs no exchange.
#pragma once

#include <limits.h>

#include "attn_decode.cuh"
#include "ptx.cuh"

namespace b200attn {

constexpr float kLog2e = 1.4426950408889634f;

struct DecodeWeightsParams {
    const float* scores;  // [unit][L][G], raw score units
    const float* lse;     // [B, Hq]
    float* w;             // [B, Hkv, L_cap]
    const int* lens;      // [B] or nullptr
    const int* status;
    int L, L_cap, Hkv, G, n_chunks;
    int blocks;           // of keys per (batch, KV head)
    float scale_log2;
};
constexpr int kDecodeWeightsThreads = 256, kDecodeWeightsKeys = 4;  // keys per thread: their loads are all issued before the first is used

// a block: 1024 keys of one (batch, KV head)
__global__ void __launch_bounds__(kDecodeWeightsThreads) decode_weights_kernel(const DecodeWeightsParams p) {
    constexpr int K = kDecodeWeightsKeys, STEP = kDecodeWeightsThreads;
    __shared__ float s_lse[16];
    const int u = int(blockIdx.x) / p.blocks, key0 = (int(blockIdx.x) - u * p.blocks) * K * STEP, b = u / p.Hkv;
    const int group = p.G * p.n_chunks;
    grid_dep_launch();  // (the next step's first kernel waits for the end of this one, but not with its set-up)
    grid_dep_wait();
    // What the length and the status word say is looked at behind the loads, which go as far as L: one round trip
    const int status = *reinterpret_cast<const volatile int*>(p.status), len = p.lens ? max(1, min(__ldg(p.lens + b), p.L)) : p.L;
    float* const w = p.w + size_t(u) * p.L_cap + key0 + threadIdx.x;
    const int left = p.L - key0 - int(threadIdx.x), count = len - key0 - int(threadIdx.x);  // key k of this thread: k * STEP < left, < count
    float old[K], acc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) old[k] = k * STEP < left ? w[k * STEP] : 0.f, acc[k] = 0.f;
    for (int c = 0; c < p.n_chunks; ++c) {  // (a chunk: at most 16 heads)
        const float* const s = p.scores + ((size_t(u) * p.n_chunks + c) * p.L + key0 + threadIdx.x) * p.G;
        const float lse = int(threadIdx.x) < p.G ? __ldcg(p.lse + size_t(u) * group + c * p.G + threadIdx.x) * kLog2e : 0.f;
        if (c) __syncthreads();
        for (int g0 = 0; g0 < p.G; g0 += 4) {
            float v[K][4];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (k * STEP >= left) continue;
                if (!(p.G & 3)) {
                    const float4 x = __ldcg(reinterpret_cast<const float4*>(s + size_t(k * STEP) * p.G + g0));
                    v[k][0] = x.x, v[k][1] = x.y, v[k][2] = x.z, v[k][3] = x.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[k][e] = g0 + e < p.G ? __ldcg(s + size_t(k * STEP) * p.G + g0 + e) : 0.f;
                }
            }
            if (g0 == 0) {
                if (int(threadIdx.x) < p.G) s_lse[threadIdx.x] = lse;
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k * STEP < left && g0 + e < p.G) acc[k] += ex2_approx(fmaf(v[k][e], p.scale_log2, -s_lse[g0 + e]));
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k * STEP < count && status == 0) w[k * STEP] = old[k] + acc[k];
}

// ------------------------------------------------------------------------------------------------------------------------------
// A chunk of T new tokens behind pos0: row t sees the keys 0 .. pos0 + t.
//
// An item is 128 keys of a (batch, KV head); its units are the tiles of query rows that see any of them, each of one head and 128
// tokens or, for a chunk of fewer tokens, of several heads and all of them.  The units of all items are numbered through and the CTAs
// take ranges of them of the same length (to one): equal work whatever the diagonal does.  What a CTA's groups of warps have added up of an
// item they leave in the workspace, each for itself (joined within the CTA the groups waited for each other at every item's end), and
// key_weights_add_kernel adds these up in their order, so a call repeats bit for bit.
//
// Roles (608 threads): warps 0-15 exponentials and sums, four groups of four that take units in turn, thread = key; warp 16 loads (K
// of an item, a ring of Q tiles); warp 17 issues the products; warp 18 brings the columns' lse.  TMEM: four score buffers of 128 columns,
// one per group.
// What bounds it: 128 x 128 exponentials a unit at 16 a clock, 1024 clocks, where the products take 256 (D = 64) or 512.  A quarter of them
// goes to the FMA pipes; a unit then takes 1280 clocks, the special-function units at 52 % (D = 64) and 44 %, the issue slots at 58 and 53 %,
// what is left being the latency of four warps a scheduler.  Measured on B200, us per call: B=1 T=4000 16/4 D=64 68.7 with two groups of four
// warps that fetched the lse themselves and joined their sums at every item's end, 61 with four groups, 54 with the lse brought by a warp of
// its own, 51.5 with sums joined by the kernel behind, 52.6 with every column a query row (infinities); B=2, 500 tokens behind 3000, 16/4
// D=128 35.7 -> 27.5, some 9 of them the two launches, the first loads and the second kernel.
struct KeyWeightsParams {
    const float* lse;   // [B, Hq, T]
    const int* rows;    // [B] or nullptr: of the T query rows those that count (a padded batch)
    float* w;           // [B, Hkv, L_cap]
    float* part;        // [item + CTA][group of warps][128]
    int* status;
    int T, pos0, L, L_cap, Hq, Hkv, group;
    int tokens, heads;  // of a unit: tokens * heads <= 128
    int n_qt, n_hc;     // tiles of tokens, chunks of heads
    int n_kt, full_kt;  // tiles of keys; those up to this one are seen by every tile of tokens
    FastDiv div_hc, div_tokens;
    int total;          // units
    int n_ctas, per_cta, more;  // CTAs, units of each, the first `more` of which have one more
    float scale_log2;
};

constexpr int kKeyWeightsGroups = 4;
template <int D>
struct KeyWeightsCfg {
    static constexpr int kTileBytes = 128 * D * 2, kBoxBytes = 128 * 128, kBoxes = D / 64;
    static constexpr int kStages = 3;
    static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 2 * kKeyWeightsGroups * 512 + 512 + 256;
};
constexpr int kKeyWeightsThreads = (kKeyWeightsGroups * 4 + 3) * 32;

// Units of a (batch, KV head) in front of key tile kt: tile i is seen by n_qt - max(0, i - full_kt) tiles of tokens.  (All units are fewer
// than 2^31, so that kt n_qt, of which at most half is taken off, and m (m - 1) are below 2^32: unsigned.)
__host__ __device__ __forceinline__ int key_weights_before(const KeyWeightsParams& p, int kt) {
    const unsigned m = kt > p.full_kt ? kt - p.full_kt : 0;
    return int((unsigned(kt) * unsigned(p.n_qt) - m * (m - 1) / 2) * unsigned(p.n_hc));
}
struct KeyWeightsItem {
    int bh, kt;        // batch * Hkv + KV head, tile of keys
    int start, units;  // its first unit, and how many it has
};
// The item that unit u (< total) belongs to
__host__ __device__ __forceinline__ KeyWeightsItem key_weights_item(const KeyWeightsParams& p, int u) {
    const int per = key_weights_before(p, p.n_kt);
    KeyWeightsItem it;
    it.bh = u / per;
    const int r = u - it.bh * per;
    int lo = 0, hi = p.n_kt - 1;  // the last tile that begins at or before r
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (key_weights_before(p, mid) <= r) lo = mid;
        else hi = mid - 1;
    }
    it.kt = lo;
    it.start = it.bh * per + key_weights_before(p, lo);
    it.units = key_weights_before(p, lo + 1) - key_weights_before(p, lo);
    return it;
}
__host__ __device__ __forceinline__ void key_weights_next(const KeyWeightsParams& p, KeyWeightsItem& it) {
    it.start += it.units;
    if (++it.kt == p.n_kt) it.kt = 0, ++it.bh;
    it.units = key_weights_before(p, it.kt + 1) - key_weights_before(p, it.kt);
}
// First unit of CTA c's range, and the CTA whose range holds unit u
__host__ __device__ __forceinline__ int key_weights_range(const KeyWeightsParams& p, int c) { return c * p.per_cta + (c < p.more ? c : p.more); }
__host__ __device__ __forceinline__ int key_weights_cta(const KeyWeightsParams& p, int u) {
    const int longer = p.more * (p.per_cta + 1);
    return u < longer ? u / (p.per_cta + 1) : p.more + (u - longer) / p.per_cta;
}

template <int D>
__global__ void __launch_bounds__(kKeyWeightsThreads, 1)
key_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const KeyWeightsParams p) {
    using Cfg = KeyWeightsCfg<D>;
    constexpr int NST = Cfg::kStages, NG = kKeyWeightsGroups;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sK = smem;                              // [2]
    uint8_t* sQ = sK + 2 * Cfg::kTileBytes;          // [NST]
    float* sLse = reinterpret_cast<float*>(sQ + NST * Cfg::kTileBytes);  // [group of warps][2][128], negative
    int* sTok = reinterpret_cast<int*>(sLse + 2 * NG * 128);  // [128] token within the unit
    uint64_t* bars = reinterpret_cast<uint64_t*>(sTok + 128);
    uint64_t* bar_k_full = bars;           // [2] (phase: piece / 2)
    uint64_t* bar_k_free = bars + 2;       // [2]
    uint64_t* bar_q_full = bars + 4;       // [NST] (phase: unit / NST)
    uint64_t* bar_q_free = bars + 4 + NST; // [NST]
    uint64_t* bar_s_full = bars + 4 + 2 * NST;   // [NG] buffer unit % NG (phase: unit / NG)
    uint64_t* bar_s_free = bars + 4 + NG + 2 * NST;  // [NG]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 4 + 2 * NG + 2 * NST);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cols = p.tokens * p.heads;
    if (warp == 4 * NG && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&bar_k_full[i], 1);
            mbar_init(&bar_k_free[i], 1);
        }
        for (int i = 0; i < NST; ++i) {
            mbar_init(&bar_q_full[i], 1);
            mbar_init(&bar_q_free[i], 1);
        }
        for (int i = 0; i < NG; ++i) {
            mbar_init(&bar_s_full[i], 2);  // the products and the lse
            mbar_init(&bar_s_free[i], 128);
        }
        fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == 4 * NG + 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (cols < 128 && tid < NG * 128) {  // rows that no load writes: columns that count for nothing, but NaN times nothing is NaN
        for (int i = tid; i < NST * Cfg::kTileBytes / 16; i += NG * 128) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
    }
    if (tid < 128) sTok[tid] = tid < cols ? tid % p.tokens : INT_MAX / 2;  // (no token: behind all that count)
    grid_dep_wait();
    if (tid == 0) {
        const int failed = *reinterpret_cast<volatile int*>(p.status);
        if (failed != 0) *abort_flag = failed;
    }
    grid_dep_launch();  // (the kernel behind takes next to nothing of an SM)
    const int u0 = key_weights_range(p, int(blockIdx.x)), n = key_weights_range(p, int(blockIdx.x) + 1) - u0;
    KeyWeightsItem it = key_weights_item(p, u0);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // unit `u` of item `it`: its tile of tokens (the last ones are seen by most) and its chunk of heads
    auto unit_qt = [&](int in_item, int* hc) {
        const int q = int(fastdiv(in_item, p.div_hc));
        *hc = in_item - q * p.n_hc;
        return p.n_qt - 1 - q;
    };
    // A tile's first token.  The last tile ends with the last token, whatever it has in common with the tile in front (the lse of which counts
    // those tokens once): every column is a query row then, where rows of zeros would score NaN with a key that holds an infinity.
    const int last_tile = p.T - p.tokens;
    auto tile_token = [&](int qt) { return min(qt * p.tokens, last_tile); };

    if (*abort_flag != 0) {
        // an earlier kernel has failed
    } else if (warp == 4 * NG) {
        // ------------------------------------------------------------------ producer
        bool ok = true;
        for (int i = 0, piece = 0; ok && i < n; ++piece) {
            const int first = u0 + i - it.start, m = min(it.units - first, n - i);
            const int b = it.bh / p.Hkv, hk = it.bh - b * p.Hkv;
            if (piece >= 2) ok = mbar_wait_warp(&bar_k_free[piece & 1], uint32_t(piece / 2 - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE);
            if (!ok) break;
            if (elect_one()) {
                mbar_arrive_expect_tx(&bar_k_full[piece & 1], Cfg::kTileBytes);
#pragma unroll
                for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                    tma_load_4d(sK + (piece & 1) * Cfg::kTileBytes + bx * Cfg::kBoxBytes, &tmK, &bar_k_full[piece & 1], bx * 64, it.kt * 128, hk, b);
            }
            __syncwarp();
            for (int e = 0; e < m; ++e, ++i) {
                int hc;
                const int s = i % NST, qt = unit_qt(first + e, &hc);
                if (i >= NST) ok = mbar_wait_warp(&bar_q_free[s], uint32_t(i / NST - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE);
                if (!ok) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&bar_q_full[s], cols * D * 2);
#pragma unroll
                    for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                        tma_load_4d(sQ + s * Cfg::kTileBytes + bx * Cfg::kBoxBytes, &tmQ, &bar_q_full[s], bx * 64, tile_token(qt), hk * p.group + hc * p.heads, b);
                }
                __syncwarp();
            }
            key_weights_next(p, it);
        }
    } else if (warp == 4 * NG + 1) {
        // ------------------------------------------------------------------ products
        constexpr uint32_t idesc = make_idesc_bf16(128, 128, 0, 0);
        bool ok = true;
        for (int i = 0, piece = 0; ok && i < n; ++piece) {
            const int first = u0 + i - it.start, m = min(it.units - first, n - i);
            ok = mbar_wait_warp(&bar_k_full[piece & 1], uint32_t(piece / 2) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            const uint64_t k_desc = make_sdesc_sw128(smem_u32(sK + (piece & 1) * Cfg::kTileBytes), 16, 1024);
            for (int e = 0; ok && e < m; ++e, ++i) {
                const int s = i % NST, buf = i % NG;
                ok = mbar_wait_warp(&bar_q_full[s], uint32_t(i / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
                if (ok && i >= NG) ok = mbar_wait_warp(&bar_s_free[buf], uint32_t(i / NG - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
                if (!ok) break;
                tc_fence_after_sync();
                const uint64_t q_desc = make_sdesc_sw128(smem_u32(sQ + s * Cfg::kTileBytes), 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        umma_ss(tmem + buf * 128, k_desc + kmajor_step(ks, Cfg::kBoxBytes), q_desc + kmajor_step(ks, Cfg::kBoxBytes), idesc, ks > 0);
                    umma_commit(&bar_s_full[buf]);
                    umma_commit(&bar_q_free[s]);
                    if (e + 1 == m) umma_commit(&bar_k_free[piece & 1]);
                }
                __syncwarp();
            }
            key_weights_next(p, it);
        }
        // nothing may be in flight when tensor memory is freed: the last unit's products
        if (ok && n > 0) mbar_wait_warp(&bar_s_full[(n - 1) % NG], uint32_t((n - 1) / NG) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
    } else if (warp == 4 * NG + 2) {
        // ------------------------------------------------------------------ lse of the units' columns, negative and in powers of two
        // lane's columns: lane + 32 k
        int h_col[4], t_col[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) h_col[c] = int(fastdiv(lane + 32 * c, p.div_tokens)), t_col[c] = lane + 32 * c - h_col[c] * p.tokens;
        auto rows_of = [&](int bh) {
            const int b = bh / p.Hkv;
            return p.lse + (size_t(b) * p.Hq + (bh - b * p.Hkv) * p.group) * p.T;
        };
        auto count_of = [&](int bh) { return p.rows ? min(p.T, __ldg(p.rows + bh / p.Hkv)) : p.T; };
        const float* rows = rows_of(it.bh);
        int T = count_of(it.bh);
        int in_item = u0 - it.start;
        float v[2][4];
        auto load = [&](float (&v)[4]) {  // of the unit at `in_item` of `it`, and on to the next
            int hc;
            const int qt = unit_qt(in_item, &hc);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int t = tile_token(qt) + t_col[c];
                // 2^(x - inf) = 0
                v[c] = lane + 32 * c < cols && t >= qt * p.tokens && t < T ? __ldg(rows + size_t(hc * p.heads + h_col[c]) * p.T + t) * -kLog2e : -INFINITY;
            }
            if (++in_item == it.units) {
                const int bh = it.bh;
                key_weights_next(p, it);
                if (it.bh != bh && it.start < p.total) rows = rows_of(it.bh), T = count_of(it.bh);
                in_item = 0;
            }
        };
        bool ok = true;
        if (n > 0) load(v[0]);
        auto put = [&](int i, float (&now)[4], float (&then)[4]) {
            if (i + 1 < n) load(then);
            // (the group's scores of the unit before are in registers, so it is through with the lse of the one before that, whose buffer this is)
            if (i >= NG) ok = mbar_wait_warp(&bar_s_free[i % NG], uint32_t(i / NG - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
            if (!ok) return;
            float* lse = sLse + ((i % NG) * 2 + (i / NG & 1)) * 128 + lane;
#pragma unroll
            for (int c = 0; c < 4; ++c) lse[32 * c] = now[c];
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_s_full[i % NG]);
        };
        for (int i = 0; ok && i < n; i += 2) {
            put(i, v[0], v[1]);
            if (ok && i + 1 < n) put(i + 1, v[1], v[0]);
        }
    } else {
        // ------------------------------------------------------------------ exponentials and sums
        const int wg = warp >> 2, key = tid & 127;
        const uint32_t t_s = tmem + (uint32_t((warp & 3) * 32) << 16) + wg * 128;
        const int n_c = (cols + 15) / 16;
        const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
        bool ok = true;
        for (int i = 0; ok && i < n;) {
            const int first = u0 + i - it.start, m = min(it.units - first, n - i);
            float acc = 0.f;
            const int k_lim = it.kt * 128 + key - p.pos0;  // tokens below it do not see the key
            const int rows = p.rows ? __ldg(p.rows + it.bh / p.Hkv) : p.T;
            for (int e = (wg - i % NG + NG) % NG; e < m; e += NG) {
                int hc;
                const int k = i + e, t_first = tile_token(unit_qt(first + e, &hc)), lim = k_lim - t_first;
                // chunks that end behind it have columns that do not count: whatever their rows hold, and the key
                const int padding = t_first + p.tokens > rows ? 0 : cols;
                const bool diagonal = lim + 127 - key > 0;  // whether any key of the tile is unseen by the unit's first token
                const float* lse = sLse + (wg * 2 + (k / NG & 1)) * 128;
                ok = mbar_wait_warp(&bar_s_full[wg], uint32_t(k / NG) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after_sync();
                uint64_t sum2[2] = {0ull, 0ull};
                uint32_t v[2][16];
                auto chunk = [&](int c, uint32_t (&v)[16]) {
                    if (c * 16 + 16 > padding) {
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            if (t_first + sTok[c * 16 + x] >= rows) v[x] = 0u;
                    }
                    if (diagonal) {
                        if (p.heads == 1) {  // (column = token)
                            if (lim > c * 16) {
#pragma unroll
                                for (int x = 0; x < 16; ++x)
                                    if (c * 16 + x < lim) v[x] = 0xff800000u;  // -inf
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                if (sTok[c * 16 + x] < lim) v[x] = 0xff800000u;
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 16; x += 8) {
                        const float4 la = *reinterpret_cast<const float4*>(lse + c * 16 + x), lb = *reinterpret_cast<const float4*>(lse + c * 16 + x + 4);
                        const float l8[8] = {la.x, la.y, la.z, la.w, lb.x, lb.y, lb.z, lb.w};
#pragma unroll
                        for (int e2 = 0; e2 < 4; ++e2) {
                            const uint64_t a = fma_f32x2(pack_f32x2(__uint_as_float(v[x + 2 * e2]), __uint_as_float(v[x + 2 * e2 + 1])), scale2,
                                                         pack_f32x2(l8[2 * e2], l8[2 * e2 + 1]));
                            if (e2 == 3) {  // a quarter of them on the FMA pipes
                                sum2[1] = add_f32x2(sum2[1], exp2_fma_f32x2(a));
                            } else {
                                float a0, a1;
                                unpack_f32x2(a, a0, a1);
                                sum2[e2 & 1] = add_f32x2(sum2[e2 & 1], pack_f32x2(ex2_approx(a0), ex2_approx(a1)));
                            }
                        }
                    }
                };
                // The next 16 columns are on their way while 16 are worked on; the buffer goes back once all are in registers.  (Two chunks
                // of code, not eight: the instruction cache.)
                tmem_ld_x16(t_s, v[0]);
#pragma unroll 1
                for (int c = 0; c < n_c; c += 2) {
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        if (c + d >= n_c) break;
                        tmem_wait_ld();
                        if (c + d + 1 < n_c) {
                            tmem_ld_x16(t_s + (c + d + 1) * 16, v[d ^ 1]);
                        } else {
                            tc_fence_before_sync();
                            mbar_arrive(&bar_s_free[wg]);
                        }
                        chunk(c + d, v[d]);
                    }
                }
                float s0, s1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                acc += s0 + s1;
            }
            i += m;
            if (ok) p.part[((size_t(it.bh) * p.n_kt + it.kt + blockIdx.x) * NG + wg) * 128 + key] = acc;
            key_weights_next(p, it);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 4 * NG + 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// The items' pieces added up in their order.  grid: items; thread = key.
__global__ void __launch_bounds__(128) key_weights_add_kernel(const KeyWeightsParams p) {
    const int bh = int(blockIdx.x) / p.n_kt, kt = int(blockIdx.x) - bh * p.n_kt, key = kt * 128 + threadIdx.x;
    const int per = key_weights_before(p, p.n_kt), start = bh * per + key_weights_before(p, kt), end = bh * per + key_weights_before(p, kt + 1);
    const int first = key_weights_cta(p, start), last = key_weights_cta(p, end - 1);
    constexpr int NG = kKeyWeightsGroups;
    grid_dep_wait();
    if (key >= p.L || *reinterpret_cast<volatile int*>(p.status) != 0) return;
    float* const w = p.w + size_t(bh) * p.L_cap + key;
    const float old = *w;
    float acc = 0.f;
    for (int c = first; c <= last; ++c) {
        const float* const part = p.part + (size_t(blockIdx.x) + c) * NG * 128 + threadIdx.x;
        float v[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) v[g] = __ldcg(part + g * 128);
#pragma unroll
        for (int g = 0; g < NG; ++g) acc += v[g];
    }
    *w = old + acc;
}

}  // namespace b200attn
