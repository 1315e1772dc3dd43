// Attention of one query token per sequence over a prompt that several sequences share, the prompt's part of it: each K and V byte
// of the prompt is read once for all of its sequences and all the heads of a group, instead of once per sequence.
//
//   rows  (sequence s of the prompt's n, head j of the chunk's): x = q[s, j] . K^T in raw score units, keys 0 .. P - 1
//   left  m, l = sum 2^((x - m) scale_log2), O = sum 2^((x - m) scale_log2) V, per row and split of the keys, un-normalised
//
// The decode kernel behind (attn_decode.cuh, kDecodeShared) goes on with the sequences' own rows and joins the two: the softmax of a
// union is the partial results' sum with weights 2^((m_i - max m) scale_log2).
//
// A CTA takes a tile of 128 rows (a row = a lane of tensor memory: S = Q K^T with Q's rows as M) and a share of the prompt's key tiles;
// rows that the tile does not have cost their part of the products, which are not what bounds it: 128 rows x 64 keys x 128 are 256
// clocks of the tensor pipe, the tile's 32 KB take 1400 at an SM's share of HBM, the exponentials of 128 rows 512.  Up to 128 rows the
// kernel is bound by HBM (latency when the prompt is short); further tiles of rows read the prompt through L2.
//
// Roles (192 threads): warps 0-3 softmax, thread = row, as in attn_fwd.cuh (scores into registers in one go, S handed back at once,
// rescaling only where the maximum grew by 2^8); warps that have no row are not waited for and leave.  Warp 4 loads: a ring of 16 KB
// places in the order in which the products read them (K of a tile ahead of V of the one before).  Warp 5 issues the products.
// TMEM (256 columns): D = 64 S 128, O 64, P 64; D = 128 S 64, P 32, O 128.
#pragma once

#include "ptx.cuh"

namespace b200attn {

struct PrefixParams {
    int P;                  // keys of the longest prompt
    int n;                  // sequences per prompt
    int heads, seqs;        // of a tile of rows: heads x seqs <= 128
    int group, n_chunks, Hkv;
    int splits, tiles;      // shares of the keys, tiles of rows per chunk
    FastDiv div_splits, div_tiles, div_chunks, div_hkv;
    const int* lens;        // [prompts] or nullptr: P
    float scale_log2;
    float* o;               // [slot][D / 4][128][4]
    float2* ml;             // [slot][128]
    int* status;
};

template <int D>
struct PrefixCfg {
    static constexpr int kKeys = D == 64 ? 128 : 64;
    static constexpr int kTileBytes = kKeys * D * 2;   // 16 KB
    static constexpr int kBoxBytes = kKeys * 128;      // [kKeys][64] BF16
    static constexpr int kBoxes = D / 64;
    static constexpr int kStages = D == 64 ? 6 : 5;    // with Q's tile two CTAs fit an SM, of this kernel or one beside a decode CTA
    static constexpr int kQBoxBytes = 128 * 128;
    static constexpr int kSmemBytes = kBoxes * kQBoxBytes + kStages * kTileBytes + 256;
    static_assert(2 * (kSmemBytes + 1024) <= 228 * 1024, "two CTAs per SM");
    static constexpr int kTmemCols = 256, kColS = 0, kColO = 128, kColP = D == 64 ? 192 : 64;
};
constexpr int kPrefixThreads = 192;
constexpr float kPrefixRescaleLog2 = 8.0f;  // P <= 2^8: its rounding to BF16 (the second product's operand) is relative

// Place in the order of loads: K of tile 0, then K of tile j + 1 and V of tile j in turn
__host__ __device__ __forceinline__ int prefix_k_at(int j) { return j == 0 ? 0 : 2 * j - 1; }
__host__ __device__ __forceinline__ int prefix_v_at(int j, int n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; }
// The i-th load: whether it is a K tile, and of which tile
__host__ __device__ __forceinline__ bool prefix_load_at(int i, int n, int* j) {
    const bool is_k = i == 0 || ((i & 1) && i + 1 < 2 * n);
    *j = i == 0 ? 0 : is_k ? (i + 1) / 2 : (i & 1) ? n - 1 : i / 2 - 1;
    return is_k;
}

template <int D>
__global__ void __launch_bounds__(kPrefixThreads, 2)
attn_prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PrefixParams p) {
    using Cfg = PrefixCfg<D>;
    constexpr int KEYS = Cfg::kKeys, NST = Cfg::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sRing = sQ + Cfg::kBoxes * Cfg::kQBoxBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(sRing + NST * Cfg::kTileBytes);
    uint64_t* bar_full = bars;              // [NST]                                  (phase: load / NST)
    uint64_t* bar_free = bars + NST;        // [NST] the products that read it are done
    uint64_t* bar_q = bars + 2 * NST;
    uint64_t* bar_s_full = bar_q + 1;       //                                         (phase: tile)
    uint64_t* bar_s_loaded = bar_q + 2;     // S is in registers                       (phase: tile)
    uint64_t* bar_p_full = bar_q + 3;       // P written, O rescaled                   (phase: tile)
    uint64_t* bar_pv = bar_q + 4;           // P V of a tile is complete               (phase: tile)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_q + 5);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // blockIdx.x -> (prompt, KV head, chunk of heads, tile of rows, split)
    int id = int(blockIdx.x);
    const int unit = int(fastdiv(id, p.div_splits)), split = id - unit * p.splits;
    const int uc = int(fastdiv(unit, p.div_tiles)), qt = unit - uc * p.tiles;
    const int uh = int(fastdiv(uc, p.div_chunks)), chunk = uc - uh * p.n_chunks;
    const int prompt = int(fastdiv(uh, p.div_hkv)), hk = uh - prompt * p.Hkv;
    const int n_rows = min(p.seqs, p.n - qt * p.seqs) * p.heads;
    const int n_warps = (n_rows + 31) / 32;  // softmax warps that have rows

    if (warp == 4 && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < NST; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_free[s], 1);
        }
        mbar_init(bar_q, 1);
        mbar_init(bar_s_full, 1);
        mbar_init(bar_s_loaded, 32 * n_warps);
        mbar_init(bar_p_full, 32 * n_warps);
        mbar_init(bar_pv, 1);
        fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == 5) {
        tmem_alloc(tmem_slot, Cfg::kTmemCols);
        tmem_relinquish();
    }
    grid_dep_wait();
    // Everything older than this kernel is complete.  The decode behind, which reads all but this kernel's results, may start.
    grid_dep_launch();
    if (tid == 0) {
        const int failed = *reinterpret_cast<volatile int*>(p.status);
        if (failed != 0) *abort_flag = failed;
    }
    const int len = p.lens ? max(0, min(__ldg(p.lens + prompt), p.P)) : p.P;
    const int all = (len + KEYS - 1) / KEYS;
    const int j0 = int(fastdiv(all * split, p.div_splits)), n_tiles = int(fastdiv(all * (split + 1), p.div_splits)) - j0;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    if (*abort_flag != 0) {
        // an earlier kernel has failed: nothing is loaded, nothing is written
    } else if (warp == 4) {
        // ------------------------------------------------------------------ producer
        auto load = [&](const CUtensorMap* map, int at, int j) {  // one thread
            uint8_t* dst = sRing + (at % NST) * Cfg::kTileBytes;
            mbar_arrive_expect_tx(&bar_full[at % NST], Cfg::kTileBytes);
#pragma unroll
            for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                tma_load_4d(dst + bx * Cfg::kBoxBytes, map, &bar_full[at % NST], bx * 64, (j0 + j) * KEYS, hk, prompt);
        };
        for (int i = 0; i < 2 * n_tiles; ++i) {
            int j;
            const bool is_k = prefix_load_at(i, n_tiles, &j);
            if (i >= NST && !mbar_wait_warp(&bar_free[i % NST], uint32_t(i / NST - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE)) break;
            if (elect_one()) {
                load(is_k ? &tmK : &tmV, i, j);
                if (i == 0) {
                    mbar_arrive_expect_tx(bar_q, Cfg::kBoxes * p.heads * p.seqs * 128);
#pragma unroll
                    for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                        tma_load_4d(sQ + bx * Cfg::kQBoxBytes, &tmQ, bar_q, bx * 64, hk * p.group + chunk * p.heads, prompt * p.n + qt * p.seqs, 0);
                }
            }
            __syncwarp();
        }
    } else if (warp == 5) {
        // ------------------------------------------------------------------ products
        constexpr uint32_t idesc_s = make_idesc_bf16(128, KEYS, 0, 0), idesc_o = make_idesc_bf16(128, D, 0, 1);
        const uint32_t ring = smem_u32(sRing);
        const uint64_t q_desc = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
        bool ok = n_tiles > 0 && mbar_wait_warp(bar_q, 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
        auto issue_s = [&](int j) {  // S = Q K^T of tile j, once S of the tile before is in registers
            const int at = prefix_k_at(j);
            ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (ok && j > 0) ok = mbar_wait_warp(bar_s_loaded, uint32_t(j - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
            if (!ok) return;
            tc_fence_after_sync();
            const uint64_t k_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, 16, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(tmem + Cfg::kColS, q_desc + kmajor_step(ks, Cfg::kQBoxBytes), k_desc + kmajor_step(ks, Cfg::kBoxBytes), idesc_s, ks > 0);
                umma_commit(bar_s_full);
                umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
        };
        if (ok) issue_s(0);
        for (int j = 0; ok && j < n_tiles; ++j) {
            if (j + 1 < n_tiles) issue_s(j + 1);
            const int at = prefix_v_at(j, n_tiles);
            if (ok) ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (ok) ok = mbar_wait_warp(bar_p_full, uint32_t(j) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t v_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, Cfg::kBoxBytes, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < KEYS / 16; ++ks)
                    umma_ts(tmem + Cfg::kColO, tmem + Cfg::kColP + ks * 8, v_desc + uint64_t(ks * 128), idesc_o, (j > 0) || (ks > 0));
                umma_commit(bar_pv);
                umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
        }
        // nothing may be in flight when tensor memory is freed
        if (ok && n_tiles > 0) mbar_wait_warp(bar_pv, uint32_t(n_tiles - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
    } else if (warp < n_warps) {
        // ------------------------------------------------------------------ softmax, thread = row
        const uint32_t lanes = uint32_t(warp * 32) << 16;
        const uint32_t t_s = tmem + lanes + Cfg::kColS, t_p = tmem + lanes + Cfg::kColP, t_o = tmem + lanes + Cfg::kColO;
        bool ok = true;
        float m_ref = -INFINITY, l = 0.f;
        for (int j = 0; j < n_tiles; ++j) {
            ok = mbar_wait_warp(bar_s_full, uint32_t(j) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after_sync();
            uint32_t sr[KEYS];
#pragma unroll
            for (int c = 0; c < KEYS; c += 32) tmem_ld_x32(t_s + c, &sr[c]);
            tmem_wait_ld();
            tc_fence_before_sync();
            mbar_arrive(bar_s_loaded);
            const int left = len - (j0 + j) * KEYS;  // keys of this tile
            if (left < KEYS) {
#pragma unroll
                for (int c = 0; c < KEYS; ++c)
                    if (c >= left) sr[c] = 0xff800000u;  // -inf
                if (p.lens) {
                    // rows of the prompt's buffer beyond its length may hold anything: 0 * NaN would be NaN
                    const int at = prefix_v_at(j, n_tiles);
                    ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
                    if (!ok) break;
                    uint8_t* v = sRing + (at % NST) * Cfg::kTileBytes;
                    for (int i = left * 8 * Cfg::kBoxes + tid; i < KEYS * 8 * Cfg::kBoxes; i += 32 * n_warps) {
                        const int r = i / (8 * Cfg::kBoxes), part = i % (8 * Cfg::kBoxes);
                        *reinterpret_cast<uint4*>(v + (part / 8) * Cfg::kBoxBytes + r * 128 + (part % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();  // (in front of the arrival on bar_p_full, upon which the product reads them)
                }
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < KEYS; c += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mx[k] = fmaxf(mx[k], fmaxf(__uint_as_float(sr[c + 2 * k]), __uint_as_float(sr[c + 2 * k + 1])));
            const float m_new = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m_ref);
            float alpha = 1.f;
            if ((m_new - m_ref) * p.scale_log2 > kPrefixRescaleLog2) {  // also true for m_ref == -inf
                alpha = ex2_approx((m_ref - m_new) * p.scale_log2);
                m_ref = m_new;
            }
            const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref * p.scale_log2;  // (all scores -inf so far: exponentials 0, not NaN)
            const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), neg2 = pack_f32x2(neg_m, neg_m);
            uint64_t sum2[2] = {0ull, 0ull};
            // P V of the tile before reads the columns that P goes to and adds to O
            if (j > 0) ok = mbar_wait_warp(bar_pv, uint32_t(j - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll
            for (int c = 0; c < KEYS / 32; ++c) {
                uint32_t pk[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float a0, a1;
                    unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sr[c * 32 + 2 * i]), __uint_as_float(sr[c * 32 + 2 * i + 1])), scale2, neg2), a0, a1);
                    a0 = ex2_approx(a0);
                    a1 = ex2_approx(a1);
                    sum2[i & 1] = add_f32x2(sum2[i & 1], pack_f32x2(a0, a1));
                    pk[i] = pack_bf16x2(a0, a1);
                }
                tmem_st_x16(t_p + c * 16, pk);
            }
            float s0, s1;
            unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
            l = l * alpha + (s0 + s1);
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t orr[32];
                    tmem_ld_x32(t_o + c * 32, orr);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
                    tmem_st_x32(t_o + c * 32, orr);
                }
            }
            tmem_wait_st();
            tc_fence_before_sync();
            mbar_arrive(bar_p_full);
        }
        if (ok && n_tiles > 0) ok = mbar_wait_warp(bar_pv, uint32_t(n_tiles - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
        if (ok) {
            const size_t slot = blockIdx.x;
            if (n_tiles > 0) {
                tc_fence_after_sync();
                float4* out = reinterpret_cast<float4*>(p.o) + slot * (D / 4) * 128 + tid;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld_x32(t_o + c * 32, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (tid < n_rows)
                            out[(c * 8 + i) * 128] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]),
                                                                 __uint_as_float(v[4 * i + 3]));
                }
            }
            if (tid < n_rows) p.ml[slot * 128 + tid] = make_float2(m_ref, l);
        }
        tc_fence_before_sync();
    }
    // teardown: every role comes here, also after a wait that gave up
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 5) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
}

}  // namespace b200attn
