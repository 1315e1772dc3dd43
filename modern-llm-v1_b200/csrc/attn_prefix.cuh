// Attention of one query token per sequence over a prompt that several sequences share, the prompt's part of it: each K and V byte
// of the prompt is read once for all of its sequences and all the heads of a group, instead of once per sequence.
//
//   rows  (sequence s of the prompt's n, head j of the chunk's): x = q[s, j] . K^T in raw score units, keys 0 .. P - 1
//   left  m, l = sum 2^((x - m) scale_log2), O = sum 2^((x - m) scale_log2) V, per row and split of the keys, un-normalised
//
// The decode kernel behind (attn_decode.cuh, kDecodeShared) goes on with the sequences' own rows and joins the two: the softmax of a
// union is the partial results' sum with weights 2^((m_i - max m) scale_log2).
//
// A CTA takes a share of the prompt's key tiles (128 keys) and one or two tiles of 128 rows (a row = a lane of tensor memory:
// S = Q K^T with Q's rows as M); rows that a tile does not have cost their part of the products, which are not what bounds it.  What a
// single online softmax cannot do is keep up: product, scores out of tensor memory, maximum, exponentials, P back and the next product
// are a chain of some 2800 clocks (D = 128), in which an SM's share of HBM brings 64 KB, the tile.  So a CTA runs two of them, each with S
// and O of its own, and one's chain passes under the other's exponentials (1024 clocks a tile and 128 rows):
//   ROWS2 = false  one tile of rows, key tiles in turn (the two results are joined through shared memory at the end)
//   ROWS2 = true   two tiles of rows, every K and V tile used twice (more than 128 rows; further ones read the prompt through L2)
// P goes over S's columns once S is in registers, which leaves room for 128 keys and two softmaxes at both head dimensions: with tiles of
// 64 keys a step of Q K^T, both operands in shared memory, takes the same 64 clocks for half the keys (B=64 P=16384 16/4 D=128, this
// kernel: 21.5 -> XX us).
//
// Roles (320 threads): warps 0-3 and 4-7 softmax, thread = row, as in attn_fwd.cuh (rescaling only where the maximum grew by 2^8); warps
// that have no row are not waited for and leave.  Warp 8 loads: a ring of K and V tiles in the order in which the products read them.
// Warp 9 issues the products.  TMEM (512 columns), per softmax: S 128 with P over its first 64, O D.
#pragma once

#include "ptx.cuh"

namespace b200attn {

struct PrefixParams {
    int P;                  // keys of the longest prompt
    int n;                  // sequences per prompt
    int heads, seqs;        // of a tile of rows: heads x seqs <= 128
    int group, n_chunks, Hkv;
    int splits, tiles;      // shares of the keys, tiles of rows per chunk
    FastDiv div_splits, div_blocks, div_chunks, div_hkv;  // blocks: of tiles, ceil(tiles / 2) or tiles
    const int* lens;        // [prompts] or nullptr: P
    float scale_log2;
    float* o;               // [slot][D / 4][128][4]
    float2* ml;             // [slot][128]
    int* status;
};

constexpr int kPrefixKeys = 128;  // per tile
template <int D, bool ROWS2>
struct PrefixCfg {
    static constexpr int kTileBytes = kPrefixKeys * D * 2;
    static constexpr int kBoxBytes = kPrefixKeys * 128;  // [keys][64] BF16
    static constexpr int kBoxes = D / 64;
    static constexpr int kStages = D == 64 ? 8 : 4;      // 128 KB
    static constexpr int kQBoxBytes = 128 * 128, kQTiles = ROWS2 ? 2 : 1;
    static constexpr int kAhead = ROWS2 ? 1 : 2;       // K tiles loaded ahead of V of tile 0
    static constexpr int kSmemBytes = kQTiles * kBoxes * kQBoxBytes + kStages * kTileBytes + 1024 + 256;
    static_assert(kStages * kTileBytes >= 128 * D * 4, "one softmax's O goes to the other through the ring");
    static constexpr int kColS = 0, kColO = 128;       // + 256 for the second softmax
};
constexpr int kPrefixThreads = 320;
constexpr float kPrefixRescaleLog2 = 8.0f;  // P <= 2^8: its rounding to BF16 (the second product's operand) is relative

// Place of a load: first `ahead` K tiles, then V of tile j and K of tile j + ahead in turn, the last V tiles at the end
__host__ __device__ __forceinline__ int prefix_k_at(int j, int ahead) { return j < ahead ? j : 2 * j - ahead + 1; }
__host__ __device__ __forceinline__ int prefix_v_at(int j, int n, int ahead) { return j + ahead < n ? 2 * j + ahead : n + j; }
// The i-th load of 2 n: whether it is a K tile, and of which tile
__host__ __device__ __forceinline__ bool prefix_load_at(int i, int n, int ahead, int* j) {
    const int pairs = n - ahead;  // loads [ahead, ahead + 2 pairs) come in pairs
    if (i < ahead && i < n) return *j = i, true;
    if (pairs > 0 && i < ahead + 2 * pairs) {
        const int e = i - ahead;
        return (e & 1) ? (*j = ahead + e / 2, true) : (*j = e / 2, false);
    }
    return *j = i - n, false;
}

template <int D, bool ROWS2>
__global__ void __launch_bounds__(kPrefixThreads, 1)
attn_prefix_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const PrefixParams p) {
    using Cfg = PrefixCfg<D, ROWS2>;
    constexpr int KEYS = kPrefixKeys, NST = Cfg::kStages, A = Cfg::kAhead;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sQ = smem;
    uint8_t* sRing = sQ + Cfg::kQTiles * Cfg::kBoxes * Cfg::kQBoxBytes;
    float2* sMl = reinterpret_cast<float2*>(sRing + NST * Cfg::kTileBytes);  // [128]
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
    // blockIdx.x -> (prompt, KV head, chunk of heads, tiles of rows, split)
    const int id = int(blockIdx.x);
    const int unit = int(fastdiv(id, p.div_splits)), split = id - unit * p.splits;
    const int uc = int(fastdiv(unit, p.div_blocks)), block = unit - uc * int(p.div_blocks.d);
    const int uh = int(fastdiv(uc, p.div_chunks)), chunk = uc - uh * p.n_chunks;
    const int prompt = int(fastdiv(uh, p.div_hkv)), hk = uh - prompt * p.Hkv;
    auto rows_of = [&](int qt) { return max(0, min(p.seqs, p.n - qt * p.seqs)) * p.heads; };
    const int qt0 = ROWS2 ? 2 * block : block;
    const int rows0 = rows_of(qt0), rows1 = ROWS2 ? rows_of(qt0 + 1) : rows0;  // of the two softmaxes
    const bool two = rows1 > 0;

    if (warp == 8 && lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < NST; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_free[s], 1);
        }
        mbar_init(bar_q, 1);
        for (int x = 0; x < 2; ++x) {
            const int n = max(32, ((x ? rows1 : rows0) + 31) / 32 * 32);
            mbar_init(&bar_s_full[x], 1);
            mbar_init(&bar_p_full[x], n);
            mbar_init(&bar_o[x], 1);
        }
        fence_mbar_init();
        *abort_flag = 0;
    }
    if (warp == 9) {
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
    // A unit is a tile's turn in one of the softmaxes: unit i is softmax i & 1's, of tile i / 2 (ROWS2) or i.
    const int n_units = ROWS2 ? 2 * n_tiles : n_tiles;

    if (*abort_flag != 0) {
        // an earlier kernel has failed: nothing is loaded, nothing is written
    } else if (warp == 8) {
        // ------------------------------------------------------------------ producer
        for (int i = 0; i < 2 * n_tiles; ++i) {
            int j;
            const bool is_k = prefix_load_at(i, n_tiles, A, &j);
            if (i >= NST && !mbar_wait_warp(&bar_free[i % NST], uint32_t(i / NST - 1) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_FREE)) break;
            if (elect_one()) {
                if (i == 0) {
                    mbar_arrive_expect_tx(bar_q, Cfg::kQTiles * Cfg::kBoxes * p.heads * p.seqs * 128);
#pragma unroll
                    for (int e = 0; e < Cfg::kQTiles * Cfg::kBoxes; ++e)
                        tma_load_4d(sQ + e * Cfg::kQBoxBytes, &tmQ, bar_q, (e % Cfg::kBoxes) * 64, hk * p.group + chunk * p.heads,
                                    prompt * p.n + (qt0 + e / Cfg::kBoxes) * p.seqs, 0);
                }
                uint8_t* dst = sRing + (i % NST) * Cfg::kTileBytes;
                mbar_arrive_expect_tx(&bar_full[i % NST], Cfg::kTileBytes);
#pragma unroll
                for (int bx = 0; bx < Cfg::kBoxes; ++bx)
                    tma_load_4d(dst + bx * Cfg::kBoxBytes, is_k ? &tmK : &tmV, &bar_full[i % NST], bx * 64, (j0 + j) * KEYS, hk, prompt);
            }
            __syncwarp();
        }
    } else if (warp == 9) {
        // ------------------------------------------------------------------ products
        constexpr uint32_t idesc_s = make_idesc_bf16(128, KEYS, 0, 0), idesc_o = make_idesc_bf16(128, D, 0, 1);
        const uint32_t ring = smem_u32(sRing);
        bool ok = n_tiles > 0 && mbar_wait_warp(bar_q, 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
        // the tile's place is free behind its last unit
        auto last_use = [&](int i) { return !ROWS2 || (i & 1) || !two; };
        auto issue_s = [&](int i) {  // S = Q K^T of unit i; P of the softmax's unit before, over S, has been read by the products in front
            const int x = i & 1, j = ROWS2 ? i >> 1 : i, at = prefix_k_at(j, A);
            if (ROWS2 && x && !two) return;
            ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (!ok) return;
            tc_fence_after_sync();
            const uint64_t q_desc = make_sdesc_sw128(smem_u32(sQ + (ROWS2 ? x : 0) * Cfg::kBoxes * Cfg::kQBoxBytes), 16, 1024);
            const uint64_t k_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, 16, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    umma_ss(tmem + x * 256 + Cfg::kColS, q_desc + kmajor_step(ks, Cfg::kQBoxBytes), k_desc + kmajor_step(ks, Cfg::kBoxBytes), idesc_s, ks > 0);
                umma_commit(&bar_s_full[x]);
                if (last_use(i)) umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
        };
        for (int i = 0; ok && i < min(2, n_units); ++i) issue_s(i);
        for (int i = 0; ok && i < n_units; ++i) {
            const int x = i & 1, j = ROWS2 ? i >> 1 : i, at = prefix_v_at(j, n_tiles, A);
            if (ROWS2 && x && !two) continue;
            ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
            if (ok) ok = mbar_wait_warp(&bar_p_full[x], uint32_t(i / 2) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_SOFTMAX);
            if (!ok) break;
            tc_fence_after_sync();
            const uint64_t v_desc = make_sdesc_sw128(ring + (at % NST) * Cfg::kTileBytes, Cfg::kBoxBytes, 1024);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < KEYS / 16; ++ks)
                    umma_ts(tmem + x * 256 + Cfg::kColO, tmem + x * 256 + Cfg::kColS + ks * 8, v_desc + uint64_t(ks * 128), idesc_o, (i > 1) || (ks > 0));
                if (i + 2 >= n_units) umma_commit(&bar_o[x]);
                if (last_use(i)) umma_commit(&bar_free[at % NST]);
            }
            __syncwarp();
            if (i + 2 < n_units) issue_s(i + 2);
        }
        // nothing may be in flight when tensor memory is freed
        for (int x = 0; ok && x < 2; ++x)
            if (n_units > x && (two || x == 0)) ok = mbar_wait_warp(&bar_o[x], 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
    } else {
        // ------------------------------------------------------------------ softmax, thread = row
        const int x = warp >> 2, row = tid & 127, rows = x ? rows1 : rows0, n_warps = (rows + 31) / 32;
        if ((warp & 3) < n_warps) {
            const uint32_t lanes = (uint32_t((warp & 3) * 32) << 16) + x * 256;
            const uint32_t t_s = tmem + lanes + Cfg::kColS, t_p = t_s, t_o = tmem + lanes + Cfg::kColO;
            const int mine = (n_units - x + 1) / 2;  // units of this softmax
            bool ok = true;
            float m_ref = -INFINITY, l = 0.f;
            for (int e = 0; e < mine; ++e) {
                const int j = ROWS2 ? e : 2 * e + x;
                ok = mbar_wait_warp(&bar_s_full[x], uint32_t(e) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
                if (!ok) break;
                tc_fence_after_sync();
                uint32_t sr[KEYS];
#pragma unroll
                for (int c = 0; c < KEYS; c += 32) tmem_ld_x32(t_s + c, &sr[c]);
                tmem_wait_ld();
                const int left = len - (j0 + j) * KEYS;  // keys of this tile
                if (left < KEYS) {
#pragma unroll
                    for (int c = 0; c < KEYS; ++c)
                        if (c >= left) sr[c] = 0xff800000u;  // -inf
                    if (p.lens) {
                        // Rows of the prompt's buffer beyond its length may hold anything: 0 * NaN would be NaN.  (With two tiles of rows
                        // both softmaxes clear them, each in front of its own product.)
                        const int at = prefix_v_at(j, n_tiles, A);
                        ok = mbar_wait_warp(&bar_full[at % NST], uint32_t(at / NST) & 1, abort_flag, p.status, DEV_WAIT_TIMEOUT_LOAD);
                        if (!ok) break;
                        uint8_t* v = sRing + (at % NST) * Cfg::kTileBytes;
                        for (int i = left * 8 * Cfg::kBoxes + row; i < KEYS * 8 * Cfg::kBoxes; i += 32 * n_warps) {
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
                // (P V of the tile before, which adds to O, is complete: it lies in front of this S in the pipe)
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
                if (e > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
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
                mbar_arrive(&bar_p_full[x]);
            }
            if (ok && mine > 0) ok = mbar_wait_warp(&bar_o[x], 0, abort_flag, p.status, DEV_WAIT_TIMEOUT_MMA);
            tc_fence_after_sync();
            // ---- O, m, l out.  Columns 4 c .. 4 c + 3 of all rows lie together: a warp's stores are whole lines.
            const int qt = qt0 + (ROWS2 ? x : 0);
            const size_t slot = (size_t(uc) * p.tiles + qt) * p.splits + split;
            float4* const out = reinterpret_cast<float4*>(p.o) + slot * (D / 4) * 128 + row;
            float4* const other = reinterpret_cast<float4*>(sRing) + row;  // the second softmax's O, [D / 4][128]
            const bool join = !ROWS2 && n_tiles > 1;
            if (join && x == 1) {
                // (the ring's last tiles have been read: the last P V of both softmaxes is waited for below in front of the reads, here
                // of this one's, and of the other's by the barrier)
                named_bar_sync(1, 64 * n_warps);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld_x32(t_o + c * 32, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        other[(c * 8 + i) * 128] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]),
                                                               __uint_as_float(v[4 * i + 3]));
                }
                sMl[row] = make_float2(m_ref, l);
                named_bar_sync(1, 64 * n_warps);
            } else if (ROWS2 || x == 0) {
                float f0 = 1.f, f1 = 0.f;
                if (join) {
                    named_bar_sync(1, 64 * n_warps);  // both softmaxes' last products are done
                    named_bar_sync(1, 64 * n_warps);  // the other's results are there
                    const float2 b = sMl[row];
                    const float m = fmaxf(m_ref, b.x);
                    f0 = m_ref == -INFINITY ? 1.f : ex2_approx((m_ref - m) * p.scale_log2);  // (-inf: l and O are 0, or NaN)
                    f1 = b.x == -INFINITY ? 1.f : ex2_approx((b.x - m) * p.scale_log2);
                    l = l * f0 + b.y * f1;
                    m_ref = m;
                }
                ok = ok && *abort_flag == 0;
                if (mine > 0) {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
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
                if (ok && row < rows) p.ml[slot * 128 + row] = make_float2(m_ref, l);
            }
            tc_fence_before_sync();
        }
    }
    // teardown: every role comes here, also after a wait that gave up
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace b200attn
