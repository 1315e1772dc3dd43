// The attention weight that each cached key has received, what an eviction (kv_evict.cuh) goes by:
//
//   w[b, hk, key] += sum over the heads h of the group and the query rows t that see the key of  p = exp(scale q[h, t] . k[key] - lse[h, t])
//
// with lse the rows' logsumexp over all keys they see, so p is the softmax's probability.
//
// One new token per sequence: the decode kernel leaves its scores (kDecodeScores) and decode_weights_kernel, behind it, has only to
// take the exponentials against the final lse: 4 G bytes a key written and read through L2 beside the 4 D of its K and V rows, instead
// of a second pass over K.
//
// A chunk of new tokens: key_weights_kernel computes S^T = K Q^T by tiles of 128 keys (lanes of tensor memory) and 128 query rows
// (columns), so that a key's sum runs inside a thread and needs no exchange.
#pragma once

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
constexpr int kDecodeWeightsThreads = 256;

// a block: keys of one (batch, KV head); thread = key
__global__ void __launch_bounds__(kDecodeWeightsThreads) decode_weights_kernel(const DecodeWeightsParams p) {
    __shared__ float s_lse[128];
    const int u = int(blockIdx.x) / p.blocks, key0 = (int(blockIdx.x) - u * p.blocks) * kDecodeWeightsThreads, b = u / p.Hkv, key = key0 + int(threadIdx.x);
    const int group = p.G * p.n_chunks;
    grid_dep_wait();
    const int len = p.lens ? max(1, min(__ldg(p.lens + b), p.L)) : p.L;
    if (key0 >= len || *reinterpret_cast<const volatile int*>(p.status) != 0) return;
    float acc = 0.f;
    float* const w = p.w + size_t(u) * p.L_cap + key;
    const float old = key < len ? *w : 0.f;
    for (int g0 = 0; g0 < group; g0 += 128) {  // (a group of more than 128 heads goes by parts)
        if (g0) __syncthreads();
        for (int g = threadIdx.x; g < min(128, group - g0); g += kDecodeWeightsThreads)
            s_lse[g] = __ldcg(p.lse + size_t(u) * group + g0 + g) * kLog2e;
        __syncthreads();
        if (key >= len) continue;
        for (int g = g0; g < min(group, g0 + 128); ++g) {
            const int chunk = g / p.G;
            const float s = __ldcg(p.scores + ((size_t(u) * p.n_chunks + chunk) * p.L + key) * p.G + g - chunk * p.G);
            acc += ex2_approx(fmaf(s, p.scale_log2, -s_lse[g - g0]));
        }
    }
    if (key < len) *w = old + acc;
}

// ------------------------------------------------------------------------------------------------------------------------------
// A chunk of T new tokens behind pos0: row t sees the keys 0 .. pos0 + t.
//
// An item is 128 keys of a (batch, KV head); its units are the tiles of query rows that see any of them, each of one head and 128
// tokens or, for a chunk of fewer tokens, of several heads and all of them.  The units of all items are numbered through and CTA c of n
// takes the units [c total / n, (c + 1) total / n): equal work whatever the diagonal does.  A piece that is not a whole item is left
// in the workspace and key_weights_add_kernel adds the pieces up in their order, so a call repeats bit for bit.
//
// Roles (320 threads): warps 0-7 exponentials and sums, two groups of four that take units in turn, thread = key; warp 8 loads (K of
// an item, a ring of Q tiles); warp 9 issues the products.  TMEM: four score buffers of 128 columns, two per group.
// What bounds it: 128 x 128 exponentials a unit at 16 a clock, 1024 clocks, where the product takes 256 (D = 128).
struct KeyWeightsParams {
    const float* lse;   // [B, Hq, T]
    float* w;           // [B, Hkv, L_cap]
    float* part;        // [item + CTA][128]
    int* status;
    int T, pos0, L, L_cap, Hq, Hkv, group;
    int tokens, heads;  // of a unit: tokens * heads <= 128
    int n_qt, n_hc;     // tiles of tokens, chunks of heads
    int n_kt, full_kt;  // tiles of keys; those up to this one are seen by every tile of tokens
    long long total;    // units
    float scale_log2;
};

template <int D>
struct KeyWeightsCfg {
    static constexpr int kTileBytes = 128 * D * 2, kBoxBytes = 128 * 128, kBoxes = D / 64;
    static constexpr int kStages = 3;
    static constexpr int kSmemBytes = (2 + kStages) * kTileBytes + 4 * 512 + 2 * 1024 + 512 + 256;
};
constexpr int kKeyWeightsThreads = 320;

// Units of a (batch, KV head) in front of key tile kt, per chunk of heads: tile i is seen by n_qt - max(0, i - full_kt) tiles of tokens
__host__ __device__ __forceinline__ long long key_weights_before(const KeyWeightsParams& p, int kt) {
    const long long m = kt > p.full_kt ? kt - p.full_kt : 0;
    return ((long long)kt * p.n_qt - m * (m - 1) / 2) * p.n_hc;
}
struct KeyWeightsItem {
    int bh, kt;         // batch * Hkv + KV head, tile of keys
    long long start;    // its first unit, and how many it has
    int units;
};
// The item that unit u (< total) belongs to
__host__ __device__ __forceinline__ KeyWeightsItem key_weights_item(const KeyWeightsParams& p, long long u) {
    const long long per = key_weights_before(p, p.n_kt);
    KeyWeightsItem it;
    it.bh = int(u / per);
    const long long r = u - it.bh * per;
    int lo = 0, hi = p.n_kt - 1;  // the last tile that begins at or before r
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (key_weights_before(p, mid) <= r) lo = mid;
        else hi = mid - 1;
    }
    it.kt = lo;
    it.start = it.bh * per + key_weights_before(p, lo);
    it.units = int(key_weights_before(p, lo + 1) - key_weights_before(p, lo));
    return it;
}
__host__ __device__ __forceinline__ void key_weights_next(const KeyWeightsParams& p, KeyWeightsItem& it) {
    it.start += it.units;
    if (++it.kt == p.n_kt) it.kt = 0, ++it.bh;
    it.units = int(key_weights_before(p, it.kt + 1) - key_weights_before(p, it.kt));
}
__host__ __device__ __forceinline__ long long key_weights_range(const KeyWeightsParams& p, int c, int n) { return p.total / n * c + p.total % n * c / n; }

template <int D>
__global__ void __launch_bounds__(kKeyWeightsThreads, 1)
key_weights_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const KeyWeightsParams p) {
    using Cfg = KeyWeightsCfg<D>;
    constexpr int NST = Cfg::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sK = smem;                              // [2]
    uint8_t* sQ = sK + 2 * Cfg::kTileBytes;          // [NST]
    float* sLse = reinterpret_cast<float*>(sQ + NST * Cfg::kTileBytes);  // [group of warps][2][128]
    float* sW = sLse + 4 * 128;                      // [2][2][128]
    int* sTok = reinterpret_cast<int*>(sW + 4 * 128);  // [128] token within the unit
    uint64_t* bars = reinterpret_cast<uint64_t*>(sTok + 128);
    uint64_t* bar_k_full = bars;           // [2] (phase: piece / 2)
    uint64_t* bar_k_free = bars + 2;       // [2]
    uint64_t* bar_q_full = bars + 4;       // [NST] (phase: unit / NST)
    uint64_t* bar_q_free = bars + 4 + NST; // [NST]
    uint64_t* bar_s_full = bars + 4 + 2 * NST;   // [4] buffer unit % 4 (phase: unit / 4)
    uint64_t* bar_s_free = bars + 8 + 2 * NST;   // [4]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 12 + 2 * NST);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int cols = p.tokens * p.heads;
    if (warp == 8 && lane == 0) {
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
        for (int i = 0; i < 4; ++i) {
            mbar_init(&bar_s_full[i], 1);
            mbar_init(&bar_s_free[i], 128);
        }
        fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    if (cols < 128 && tid < 256) {  // rows that no load writes: columns that count for nothing, but NaN times nothing is NaN
        for (int i = tid; i < NST * Cfg::kTileBytes / 16; i += 256) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
    }
    if (tid < 128) sTok[tid] = tid % p.tokens;
    grid_dep_wait();
    if (tid == 0) {
        const int failed = *reinterpret_cast<volatile int*>(p.status);
        if (failed != 0) *abort_flag = failed;
    }
    const long long u0 = key_weights_range(p, int(blockIdx.x), int(gridDim.x)), u1 = key_weights_range(p, int(blockIdx.x) + 1, int(gridDim.x));
    const int n = int(u1 - u0);
    KeyWeightsItem it = key_weights_item(p, u0);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    // unit `u` of item `it`: its tile of tokens (the last ones are seen by most) and its chunk of heads
    auto unit_qt = [&](const KeyWeightsItem& it, int in_item) { return p.n_qt - 1 - in_item / p.n_hc; };

    if (*abort_flag != 0) {
        // an earlier kernel has failed
    } else if (warp == 8) {
        // ------------------------------------------------------------------ producer
        bool ok = true;
        for (int i = 0, piece = 0; ok && i < n; ++piece) {
            const int first = int(u0 + i - it.start), m = min(it.units - first, n - i);
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
                const int s = i % NST, qt = unit_qt(it, first + e), hc = (first + e) % p.n_hc;
                if (i >= NST) ok = mbar_wait_warp(&bar_q_free[s], uint32_t(i / NST - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE);
                if (!ok) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&bar_q_full[s], cols * D * 2);
#pragma unroll
                    for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                        tma_load_4d(sQ + s * Cfg::kTileBytes + bx * Cfg::kBoxBytes, &tmQ, &bar_q_full[s], bx * 64, qt * p.tokens, hk * p.group + hc * p.heads, b);
                }
                __syncwarp();
            }
            key_weights_next(p, it);
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ products
        constexpr uint32_t idesc = make_idesc_bf16(128, 128, 0, 0);
        bool ok = true;
        for (int i = 0, piece = 0; ok && i < n; ++piece) {
            const int first = int(u0 + i - it.start), m = min(it.units - first, n - i);
            ok = mbar_wait_warp(&bar_k_full[piece & 1], uint32_t(piece / 2) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            const uint64_t k_desc = make_sdesc_sw128(smem_u32(sK + (piece & 1) * Cfg::kTileBytes), 16, 1024);
            for (int e = 0; ok && e < m; ++e, ++i) {
                const int s = i % NST, buf = i & 3;
                ok = mbar_wait_warp(&bar_q_full[s], uint32_t(i / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
                if (ok && i >= 4) ok = mbar_wait_warp(&bar_s_free[buf], uint32_t(i / 4 - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
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
        if (ok && n > 0) mbar_wait_warp(&bar_s_full[(n - 1) & 3], uint32_t((n - 1) / 4) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
    } else {
        // ------------------------------------------------------------------ exponentials and sums
        const int wg = warp >> 2, key = tid & 127;
        const uint32_t t_lane = tmem + (uint32_t((warp & 3) * 32) << 16);
        // The lse of this thread's column in the unit that lies `i` units into the CTA's range
        auto load_lse = [&](const KeyWeightsItem& it, int in_item) -> float {
            const int qt = unit_qt(it, in_item), hc = in_item % p.n_hc;
            const int t = qt * p.tokens + sTok[key], h = hc * p.heads + key / p.tokens;
            const int b = it.bh / p.Hkv, hk = it.bh - b * p.Hkv;
            if (key >= cols || t >= p.T || h >= p.group) return INFINITY;  // 2^(x - inf) = 0
            return __ldg(p.lse + (size_t(b) * p.Hq + hk * p.group + h) * p.T + t) * kLog2e;
        };
        bool ok = true;
        float next = 0.f;
        KeyWeightsItem ahead = it;  // the item of this group's next unit
        auto fetch = [&](int i) {
            if (i >= n) return;
            while (u0 + i >= ahead.start + ahead.units) key_weights_next(p, ahead);
            next = load_lse(ahead, int(u0 + i - ahead.start));
        };
        fetch(wg);
        for (int i = 0, piece = 0; i < n; ++piece) {
            const int first = int(u0 + i - it.start), m = min(it.units - first, n - i);
            float acc = 0.f;
            for (int e = (i & 1) == wg ? 0 : 1; e < m; e += 2) {
                const int k = i + e, buf = k & 3, qt = unit_qt(it, first + e);
                float* lse = sLse + (wg * 2 + ((k >> 1) & 1)) * 128;
                lse[key] = next;
                fetch(k + 2);
                named_bar_sync(1 + wg, 128);  // (the buffer's last readers were two units of this group ago: one such barrier between)
                if (ok) ok = mbar_wait_warp(&bar_s_full[buf], uint32_t(k / 4) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
                if (!ok) continue;  // (a warp that has given up still meets the others at the named barriers)
                tc_fence_after_sync();
                const int k_pos = it.kt * 128 + key, t_first = qt * p.tokens;  // this thread's key, the unit's first token
                const bool diagonal = it.kt * 128 + 127 > p.pos0 + t_first;
                const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2);
                uint64_t sum2[2] = {0ull, 0ull};
                const uint32_t t_s = t_lane + buf * 128;
                const int n_c = (cols + 31) / 32;
                for (int c = 0; c < n_c; ++c) {
                    uint32_t v[32];
                    tmem_ld_x32(t_s + c * 32, v);
                    tmem_wait_ld();
                    if (diagonal) {
#pragma unroll
                        for (int x = 0; x < 32; ++x)
                            if (k_pos > p.pos0 + t_first + sTok[c * 32 + x]) v[x] = 0xff800000u;  // -inf
                    }
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        const float4 ls = *reinterpret_cast<const float4*>(lse + c * 32 + x);
                        float a0, a1, a2, a3;
                        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[x]), __uint_as_float(v[x + 1])), scale2, pack_f32x2(-ls.x, -ls.y)), a0, a1);
                        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[x + 2]), __uint_as_float(v[x + 3])), scale2, pack_f32x2(-ls.z, -ls.w)), a2, a3);
                        sum2[0] = add_f32x2(sum2[0], pack_f32x2(ex2_approx(a0), ex2_approx(a1)));
                        sum2[1] = add_f32x2(sum2[1], pack_f32x2(ex2_approx(a2), ex2_approx(a3)));
                    }
                }
                tc_fence_before_sync();
                mbar_arrive(&bar_s_free[buf]);
                float s0, s1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                acc += s0 + s1;
            }
            i += m;
            // the two groups' sums of the piece
            float* w2 = sW + (piece & 1) * 256;
            if (wg == 1) w2[key] = acc;
            named_bar_sync(3, 256);
            if (wg == 0 && ok && *abort_flag == 0) {
                acc += w2[key];
                if (m == it.units) {
                    if (it.kt * 128 + key < p.L) p.w[size_t(it.bh) * p.L_cap + it.kt * 128 + key] += acc;
                } else {
                    p.part[(size_t(it.bh) * p.n_kt + it.kt + blockIdx.x) * 128 + key] = acc;
                }
            }
            key_weights_next(p, it);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// Items that several CTAs share: their pieces added up in their order.  grid: items; thread = key.
__global__ void __launch_bounds__(128) key_weights_add_kernel(const KeyWeightsParams p, const int n_ctas) {
    const int bh = blockIdx.x / p.n_kt, kt = blockIdx.x - bh * p.n_kt, key = kt * 128 + threadIdx.x;
    const long long per = key_weights_before(p, p.n_kt), start = bh * per + key_weights_before(p, kt), end = bh * per + key_weights_before(p, kt + 1);
    // the CTA whose range holds unit u: the last one that begins at or before it
    auto cta_of = [&](long long u) {
        int lo = 0, hi = n_ctas - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (key_weights_range(p, mid, n_ctas) <= u) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    const int first = cta_of(start), last = cta_of(end - 1);
    grid_dep_wait();
    if (first == last || key >= p.L || *reinterpret_cast<volatile int*>(p.status) != 0) return;
    float* const w = p.w + size_t(bh) * p.L_cap + key;
    float acc = 0.f;
    for (int c = first; c <= last; ++c) acc += __ldcg(p.part + (size_t(blockIdx.x) + c) * 128 + threadIdx.x);
    *w += acc;
}

}  // namespace b200attn
