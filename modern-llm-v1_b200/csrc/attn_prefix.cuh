// Attention of one query token per sequence over a prompt that several sequences share, the prompt's part of it: each K and V byte
// of the prompt is read once for all of its sequences and all the heads of a group, instead of once per sequence.
//
//   rows  (sequence s of the prompt's n, head j of the chunk's): x = q[s, j] . K^T in raw score units, keys 0 .. P - 1
//   left  m, l = sum 2^((x - m) scale_log2), O = sum 2^((x - m) scale_log2) V, per row and split of the keys, un-normalised
//
// The decode kernel behind (attn_decode.cuh, kDecodeShared) goes on with the sequences' own rows and joins the two: the softmax of a
// union is the partial results' sum with weights 2^((m_i - max m) scale_log2).
//
// A CTA takes a tile of 128 rows (a row = a lane of tensor memory: S = Q K^T with Q's rows as M) and a share of the prompt's key tiles
// (128 keys); rows that the tile does not have cost their part of the products, which are not what bounds it, and further tiles of rows
// read the prompt through L2.  What a single online softmax cannot do is keep up: product, scores out of tensor memory, maximum,
// exponentials, P back and the next product are a chain of 3300 clocks, in which an SM's share of HBM brings 64 KB, a tile at D = 128.  So
// a CTA runs two of them, taking its tiles in turn, each with S and O of its own; the two results are joined through shared memory at
// the end, and a tile takes 1440 clocks at D = 64 and 2180 at D = 128.  Up to 64 rows the second softmax has them in lanes 64 .. 127, so that each has two of the SM's four schedulers for itself.
// P goes over S's columns, which leaves room for 128 keys and two softmaxes at both head dimensions.
//
// Roles (576 threads): warps 0-7 the one softmax, 8-15 the other; thread = row and half of the tile's keys (two warps share a row's maximum
// through shared memory), rescaling only where the maximum grew by 2^8 as in attn_fwd.cuh; warps that have no row are not waited for
// and leave.  Warp 16 loads, a ring of K and V tiles in the order in which the products read them; warp 17 issues the products.  TMEM
// (512 columns), per softmax: S 128 with P over each half's scores, O D.
//
// Measured on B200, us per call, this kernel and the decode behind (G prompts, n sequences each, 16/4 heads):
//   G=8 n=16 P<=2000 L<=300 D=64: one softmax 28.3, two, thread = row 27.0, thread = row and half 25.3; with the decode's units in turn 21.7, two splits 16.6 to 17.5
//   G=1 n=64 P=16384 L=256 D=128: one softmax 31.5, two, thread = row and half 27.4, as it is 26.1 (67 MB: 2.6 TB/s)
//   G=1 n=8 P=500 L=12 6/2 D=64: 6.9, 7.0 and 7.0 to 7.5 (the two launches' latency)
// Measured and dropped: tiles of 64 keys with P beside S (Q K^T takes 64 clocks a step for half the keys); two tiles of rows in a CTA, every K and
// V tile used twice, 31.5 where two CTAs that each read them take 27.4 (the partial results of 256 rows are as many bytes as 256 keys, and
// twice as many shares have to be joined); its results added up over a cluster through distributed shared memory (35: clusters of four
// crowd into a few GPCs, whose bandwidth they then share); a second warp for the products (38: the two interleave on the tensor pipe).
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

constexpr int kPrefixKeys = 128;  // per tile
constexpr int kPrefixThreads = 576;
template <int D>
struct PrefixCfg {
    static constexpr int kTileBytes = kPrefixKeys * D * 2;
    static constexpr int kBoxBytes = kPrefixKeys * 128;  // [keys][64] BF16
    static constexpr int kBoxes = D / 64;
    static constexpr int kStages = D == 64 ? 8 : 4;      // 128 KB
    static constexpr int kQBoxBytes = 128 * 128;
    static constexpr int kQBytes = 2 * kBoxes * kQBoxBytes;  // once, and once more 64 rows further down
    static constexpr int kSmemBytes = kQBytes + kStages * kTileBytes + 6144 + 256;
    static_assert(kStages * kTileBytes >= 128 * D * 4, "one softmax's O goes to the other through the ring");
    static constexpr int kColS = 0, kColO = 128;         // + 256 for the second softmax
};
constexpr float kPrefixRescaleLog2 = 8.0f;  // P <= 2^8: its rounding to BF16 (the second product's operand) is relative

// Place of a load: K of tiles 0 and 1, then V of tile j and K of tile j + 2 in turn, the last two V tiles at the end
__host__ __device__ __forceinline__ int prefix_k_at(int j) { return j < 2 ? j : 2 * j - 1; }
__host__ __device__ __forceinline__ int prefix_v_at(int j, int n) { return j + 2 < n ? 2 * j + 2 : n + j; }
// The i-th load of 2 n: whether it is a K tile, and of which tile
__host__ __device__ __forceinline__ bool prefix_load_at(int i, int n, int* j) {
    if (i < 2 && i < n) return *j = i, true;
    if (i >= 2 && i < 2 * n - 2) return (i & 1) ? (*j = (i + 1) / 2, true) : (*j = i / 2 - 1, false);
    return *j = i - n, false;
}

template <int D>
__global__ void __launch_bounds__(kPrefixThreads, 1)
attn_prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PrefixParams p) {
    using Cfg = PrefixCfg<D>;
    constexpr int KEYS = kPrefixKeys, NST = Cfg::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sRing = sQ + Cfg::kQBytes;
    float* sMax = reinterpret_cast<float*>(sRing + NST * Cfg::kTileBytes);  // [softmax][tile & 1][half][128] maxima of the rows' halves
    float* sL = sMax + 1024;                                                // [softmax][128] at the end, l of the second halves
    float2* sMl = reinterpret_cast<float2*>(sL + 256);                      // [128] at the end, the second softmax's (m, l)
    uint64_t* bars = reinterpret_cast<uint64_t*>(sMl + 128);
    uint64_t* bar_full = bars;              // [NST]                                          (phase: load / NST)
    uint64_t* bar_free = bars + NST;        // [NST] the products that read it are done
    uint64_t* bar_q = bars + 2 * NST;
    uint64_t* bar_s_full = bar_q + 1;       // [2] per softmax                                (phase: its tile)
    uint64_t* bar_p_full = bar_q + 3;       // [2] P written, O rescaled
    uint64_t* bar_o = bar_q + 5;            // [2] O is complete                              (once)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_q + 7);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // blockIdx.x -> (prompt, KV head, chunk of heads, tile of rows, split)
    const int id = int(blockIdx.x);
    const int unit = int(fastdiv(id, p.div_splits)), split = id - unit * p.splits;
    const int uc = int(fastdiv(unit, p.div_tiles)), qt = unit - uc * p.tiles;
    const int uh = int(fastdiv(uc, p.div_chunks)), chunk = uc - uh * p.n_chunks;
    const int prompt = int(fastdiv(uh, p.div_hkv)), hk = uh - prompt * p.Hkv;
    const int rows = min(p.seqs, p.n - qt * p.seqs) * p.heads, n_warps = (rows + 31) / 32;  // warps of 32 rows
    const int lane1 = p.heads * p.seqs <= 64 ? 64 : 0;  // tensor memory lane of the second softmax's first row (Q's box has that many rows)

    if (warp == 16 && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < NST; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_free[s], 1);
        }
        mbar_init(bar_q, 1);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bar_s_full[x], 1);
            mbar_init(&bar_p_full[x], 64 * n_warps);
            mbar_init(&bar_o[x], 1);
        }
        fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == 17) {
        tmem_alloc(tmem_slot, 512);
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
    } else if (warp == 16) {
        // ------------------------------------------------------------------ producer
        for (int i = 0; i < 2 * n_tiles; ++i) {
            int j;
            const bool is_k = prefix_load_at(i, n_tiles, &j);
            if (i >= NST && !mbar_wait_warp(&bar_free[i % NST], uint32_t(i / NST - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE)) break;
            if (elect_one()) {
                if (i == 0) {
                    const int boxes = (lane1 ? 2 : 1) * Cfg::kBoxes;
                    mbar_arrive_expect_tx(bar_q, boxes * p.heads * p.seqs * 128);
                    for (int e = 0; e < boxes; ++e)
                        tma_load_4d(sQ + e * Cfg::kQBoxBytes + (e >= Cfg::kBoxes ? lane1 * 128 : 0), &tmQ, bar_q, (e % Cfg::kBoxes) * 64,
                                    hk * p.group + chunk * p.heads, prompt * p.n + qt * p.seqs, 0);
                }
                uint8_t* dst = sRing + (i % NST) * Cfg::kTileBytes;
                mbar_arrive_expect_tx(&bar_full[i % NST], Cfg::kTileBytes);
#pragma unroll
                for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                    tma_load_4d(dst + bx * Cfg::kBoxBytes, is_k ? &tmK : &tmV, &bar_full[i % NST], bx * 64, (j0 + j) * KEYS, hk, prompt);
            }
            __syncwarp();
        }
    } else if (warp == 17) {
        // ------------------------------------------------------------------ products
        constexpr uint32_t idesc_s = make_idesc_bf16(128, KEYS, 0, 0), idesc_o = make_idesc_bf16(128, D, 0, 1);
        const uint32_t ring = smem_u32(sRing);
        bool ok = n_tiles > 0 && mbar_wait_warp(bar_q, 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
        auto issue_s = [&](int j) {  // S = Q K^T of tile j; P of the softmax's tile before, over S, has been read by the products in front
            const int x = j & 1, at = prefix_k_at(j);
            ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (!ok) return;
            tc_fence_after_sync();
            const uint64_t q_desc = make_sdesc_sw128(smem_u32(sQ + (lane1 ? x : 0) * Cfg::kBoxes * Cfg::kQBoxBytes), 16, 1024);
            const uint64_t k_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, 16, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(tmem + x * 256 + Cfg::kColS, q_desc + kmajor_step(ks, Cfg::kQBoxBytes), k_desc + kmajor_step(ks, Cfg::kBoxBytes), idesc_s, ks > 0);
                umma_commit(&bar_s_full[x]);
                umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
        };
        for (int j = 0; ok && j < min(2, n_tiles); ++j) issue_s(j);
        for (int j = 0; ok && j < n_tiles; ++j) {
            const int x = j & 1, at = prefix_v_at(j, n_tiles);
            ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (ok) ok = mbar_wait_warp(&bar_p_full[x], uint32_t(j / 2) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t v_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, Cfg::kBoxBytes, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < KEYS / 16; ++ks)  // P of keys 0-63 in columns 0-31, of keys 64-127 in columns 64-95
                    umma_ts(tmem + x * 256 + Cfg::kColO, tmem + x * 256 + Cfg::kColS + (ks % 4) * 8 + (ks / 4) * 64, v_desc + uint64_t(ks * 128), idesc_o,
                            (j > 1) || (ks > 0));
                if (j + 2 >= n_tiles) umma_commit(&bar_o[x]);
                umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
            if (j + 2 < n_tiles) issue_s(j + 2);
        }
        // nothing may be in flight when tensor memory is freed
        for (int x = 0; ok && x < min(2, n_tiles); ++x) ok = mbar_wait_warp(&bar_o[x], 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
    } else {
        // ------------------------------------------------------------------ softmax, thread = row and half of the keys
        const int x = warp >> 3, half = (warp >> 2) & 1, row = (tid & 127) - (x ? lane1 : 0);
        if (row >= 0 && row < 32 * n_warps) {
            constexpr int COLS = KEYS / 2, CH = 16;
            const uint32_t lanes = (uint32_t((warp & 3) * 32) << 16) + x * 256;
            const uint32_t t_s = tmem + lanes + Cfg::kColS + half * COLS, t_p = t_s,  // (each half's P over its own scores)
                           t_o = tmem + lanes + Cfg::kColO + half * (D / 2);
            const int mine = (n_tiles - x + 1) / 2;   // tiles of this softmax
            const int pair = 1 + x * 4 + (warp & 3);  // named barrier of the two warps that share rows
            bool ok = true;
            float m_ref = -INFINITY, l = 0.f;
            for (int e = 0; e < mine; ++e) {
                const int j = 2 * e + x;
                if (ok) ok = mbar_wait_warp(&bar_s_full[x], uint32_t(e) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
                tc_fence_after_sync();
                const int left = len - (j0 + j) * KEYS - half * COLS;  // keys of this half tile
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                // visit(16 columns, the first of which is c) for the thread's scores, the next of which are on their way meanwhile
                uint32_t v[2][CH];
                auto columns = [&](auto visit) {
                    tmem_ld_x16(t_s, v[0]);
#pragma unroll
                    for (int c = 0; c < COLS; c += CH) {
                        tmem_wait_ld();
                        if (c + CH < COLS) tmem_ld_x16(t_s + c + CH, v[(c / CH + 1) & 1]);
                        uint32_t(&now)[CH] = v[(c / CH) & 1];
                        if (left < COLS) {
#pragma unroll
                            for (int k = 0; k < CH; ++k)
                                if (c + k >= left) now[k] = 0xff800000u;  // -inf
                        }
                        visit(c, now);
                    }
                };
                if (ok)
                    columns([&](int, uint32_t (&sr)[CH]) {
#pragma unroll
                        for (int k = 0; k < CH; k += 4)
#pragma unroll
                            for (int q = 0; q < 2; ++q)
                                mx[(k / 4 % 2) * 2 + q] = fmaxf(mx[(k / 4 % 2) * 2 + q], fmaxf(__uint_as_float(sr[k + 2 * q]), __uint_as_float(sr[k + 2 * q + 1])));
                    });
                // The other half's maximum.  (The place was last read two tiles ago, in front of the barrier of the tile between.)
                const float m_half = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                float* const s_max = sMax + (x * 2 + (e & 1)) * 256 + (tid & 127);
                s_max[half * 128] = m_half;
                named_bar_sync(pair, 64);
                if (!ok) continue;  // (a warp that has given up still meets the other at the barriers)
                if (p.lens && len - (j0 + j) * KEYS < KEYS) {
                    // rows of the prompt's buffer beyond its length may hold anything: 0 * NaN would be NaN
                    const int at = prefix_v_at(j, n_tiles), first = len - (j0 + j) * KEYS;
                    ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
                    if (!ok) continue;
                    uint8_t* v = sRing + (at % NST) * Cfg::kTileBytes;
                    for (int i = first * 8 * Cfg::kBoxes + row * 2 + half; i < KEYS * 8 * Cfg::kBoxes; i += 64 * n_warps) {
                        const int r = i / (8 * Cfg::kBoxes), part = i % (8 * Cfg::kBoxes);
                        *reinterpret_cast<uint4*>(v + (part / 8) * Cfg::kBoxBytes + r * 128 + (part % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_proxy_async_smem();  // (in front of the arrival on bar_p_full, upon which the product reads them)
                }
                const float m_new = fmaxf(fmaxf(m_half, s_max[128 - half * 128]), m_ref);
                float alpha = 1.f;
                if ((m_new - m_ref) * p.scale_log2 > kPrefixRescaleLog2) {  // also true for m_ref == -inf
                    alpha = ex2_approx((m_ref - m_new) * p.scale_log2);
                    m_ref = m_new;
                }
                const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref * p.scale_log2;  // (all scores -inf so far: exponentials 0, not NaN)
                const uint64_t scale2 = pack_f32x2(p.scale_log2, p.scale_log2), neg2 = pack_f32x2(neg_m, neg_m);
                uint64_t sum2[2] = {0ull, 0ull};
                // (P V of the tile before, which adds to O, is complete: it lies in front of this S in the pipe)
                columns([&](int c, uint32_t (&sr)[CH]) {
                    uint32_t pk[CH / 2];
#pragma unroll
                    for (int i = 0; i < CH / 2; ++i) {
                        const uint64_t a = fma_f32x2(pack_f32x2(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), scale2, neg2);
                        float a0, a1;
                        if (i % 4 == 3) {  // a quarter of them on the FMA pipes
                            const uint64_t e2 = exp2_fma_f32x2(a);
                            sum2[i & 1] = add_f32x2(sum2[i & 1], e2);
                            unpack_f32x2(e2, a0, a1);
                        } else {
                            unpack_f32x2(a, a0, a1);
                            a0 = ex2_approx(a0);
                            a1 = ex2_approx(a1);
                            sum2[i & 1] = add_f32x2(sum2[i & 1], pack_f32x2(a0, a1));
                        }
                        pk[i] = pack_bf16x2(a0, a1);
                    }
                    tmem_st_x8(t_p + c / 2, pk);
                });
                float s0, s1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                l = l * alpha + (s0 + s1);
                if (e > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 64; ++c) {
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
                mbar_arrive(&bar_p_full[x]);
            }
            if (ok && mine > 0) ok = mbar_wait_warp(&bar_o[x], 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
            tc_fence_after_sync();
            // ---- O, m, l out: the halves' sums first.  Columns 4 c .. 4 c + 3 of all rows lie together: a warp's stores are whole lines.
            float* const s_l = sL + x * 128 + (tid & 127);
            if (half == 1) *s_l = l;
            named_bar_sync(pair, 64);
            if (half == 0) l += *s_l;
            const size_t slot = (size_t(uc) * p.tiles + qt) * p.splits + split;
            const int c0 = half * (D / 8);  // first 16-byte column
            float4* const out = reinterpret_cast<float4*>(p.o) + (slot * (D / 4) + c0) * 128 + row;
            float4* const other = reinterpret_cast<float4*>(sRing) + c0 * 128 + row;  // the second softmax's O, [D / 4][128]
            const bool join = n_tiles > 1;
            const int all_threads = 128 * n_warps;
            if (join && x == 1) {
                named_bar_sync(9, all_threads);  // both softmaxes' last products are done: nothing reads the ring; the maxima are read
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {
                    uint32_t v[32];
                    tmem_ld_x32(t_o + c * 32, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        other[(c * 8 + i) * 128] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]),
                                                               __uint_as_float(v[4 * i + 3]));
                }
                if (half == 0) sMl[row] = make_float2(m_ref, l);
                named_bar_sync(9, all_threads);
            } else if (x == 0) {
                float f0 = 1.f, f1 = 0.f;
                if (join) {
                    named_bar_sync(9, all_threads);
                    named_bar_sync(9, all_threads);  // the other's results are there
                    const float2 b = sMl[row];
                    const float m = fmaxf(m_ref, b.x);
                    f0 = m_ref == -INFINITY ? 1.f : ex2_approx((m_ref - m) * p.scale_log2);  // (-inf: l and O are 0, or NaN)
                    f1 = b.x == -INFINITY ? 1.f : ex2_approx((b.x - m) * p.scale_log2);
                    l = l * f0 + b.y * f1;
                    m_ref = m;
                }
                ok = ok && *abort_flag == 0;
                if (mine > 0) {
#pragma unroll 1
                    for (int c = 0; c < D / 64; ++c) {
                        uint32_t v[32];
                        tmem_ld_x32(t_o + c * 32, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float4 r = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                            if (join) {
                                const float4 b = other[(c * 8 + i) * 128];
                                r.x = r.x * f0 + b.x * f1, r.y = r.y * f0 + b.y * f1, r.z = r.z * f0 + b.z * f1, r.w = r.w * f0 + b.w * f1;
                            }
                            if (ok && row < rows) out[(c * 8 + i) * 128] = r;
                        }
                    }
                }
                if (ok && half == 0 && row < rows) p.ml[slot * 128 + row] = make_float2(m_ref, l);
            }
            tc_fence_before_sync();
        }
    }
    // teardown: every role comes here, also after a wait that gave up
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace b200attn
