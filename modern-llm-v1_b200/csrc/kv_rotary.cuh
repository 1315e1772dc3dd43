// KV-cache append for caches whose rows and positions part ways: behind a prompt that several sequences share a token's position
// is the prompt's length plus its own row, and an eviction takes rows away, not positions.  kv_append_kernel (kv_cache.cuh) has
// one number for both, the reference's rotation and the norm always; here are all forms of rotary.cuh, and every k row's position
// is noted where the cache keeps positions.
//
//   q rows [B, n_new, Hq, D]  -> rotated at pos + t (norm) -> BF16 q_out [B, Hq, n_new, D]
//   k rows [B, n_new, Hkv, D] -> rotated at pos + t (norm) -> BF16 kcache[b, h, row + t, :],  positions[b, h, row + t] = pos + t,
//                                                             weights[b, h, row + t] = 0: whatever token the row held before
//   v rows                    -> BF16 vcache[b, h, row + t, :]
//
// The same deal of rows to lanes as kv_append_kernel: latency at one token (1.5 us as one of a graph's launches, 64 sequences 16/4 D=64 1.9);
// a prompt is bound by the latency of one row a lane in flight (B=2 T=4000 16/4, us and TB/s: D=64 BF16 20.1, 2.4, FP32 18.0, 4.1; D=128
// BF16 without the norm 34.9, 2.8, interleaved with it 39.3, 2.5).  The row arithmetic is rotary.cuh's, so a cache filled token by token has the
// bits of one filled from rotary_forward.
#pragma once

#include "kv_cache.cuh"
#include "rotary.cuh"

namespace b200attn {

struct KvRotaryParams : KvAppendParams {
    const int* rows;  // [B] first cache row per sequence, or nullptr: row0
    int* positions;   // [B, Hkv, L_cap] or nullptr
    float* weights;   // the same
    int row0, n_pos, R;
};

template <int D, bool F32, bool HALF, bool NORM>
__global__ void __launch_bounds__(kKvAppendThreads)
kv_rotary_kernel(const __grid_constant__ KvRotaryParams p) {
    constexpr int LPR = D / 8, RPS = 32 / LPR;
    const int lane = threadIdx.x & 31, sub = lane / LPR, li = lane % LPR;
    const unsigned warp0 = (blockIdx.x * kKvAppendThreads + threadIdx.x) >> 5, n_warps = (gridDim.x * kKvAppendThreads) >> 5;
    const unsigned n_rows = p.rows_q + 2u * p.rows_kv;
    RotaryLane<D, HALF> rl(p.R, li);
    if (p.n_new == 1) grid_dep_launch();  // (as in kv_append_kernel)
    grid_dep_wait();

    for (unsigned long long r0 = static_cast<unsigned long long>(warp0) * RPS; r0 < n_rows; r0 += static_cast<unsigned long long>(n_warps) * RPS) {
        const bool live = r0 + sub < n_rows;
        unsigned r = unsigned(r0 + sub);
        int which = 0;  // 0 q, 1 k, 2 v
        if (live && r >= p.rows_q) {
            r -= p.rows_q;
            which = 1;
            if (r >= p.rows_kv) r -= p.rows_kv, which = 2;
        }
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, rot[8], gm[8];
        int b = 0, t = 0, h = 0;
        long long pos = 0, row = 0;
        int bad = 0;
        if (live) {
            const int H = which == 0 ? p.Hq : p.Hkv;
            const unsigned bt = fastdiv(r, which == 0 ? p.div_hq : p.div_hkv);
            h = int(r - bt * unsigned(H));
            b = int(fastdiv(bt, p.div_n));
            t = int(bt - unsigned(b) * unsigned(p.n_new));
            pos = p.pos ? __ldg(p.pos + b) : p.pos0;
            row = p.rows ? __ldg(p.rows + b) : p.row0;
            // (all of a sequence's new tokens or none)
            if (row < 0 || row + p.n_new > p.L_cap) bad = DEV_KV_CACHE_OVERFLOW;
            else if (pos < 0 || pos + p.n_new > p.n_pos) bad = DEV_ROTARY_POSITION;
            if (bad) pos = row = 0;
            pos += t, row += t;
            RotaryRaw<F32, HALF> raw;
            raw.load(which == 0 ? p.xq : which == 1 ? p.xk : p.xv, static_cast<long long>(r) * D, rl.at, rl.more);
            raw.r.get(v);
            if (NORM && which != 2) {
                // (16-byte aligned, as b200attn_kv_append_rotary asks: this is loaded with every row)
                const float* const gamma = (which == 0 ? p.gamma_q : p.gamma_k) + rl.at;
                const float4 ga = *reinterpret_cast<const float4*>(gamma), gb = *reinterpret_cast<const float4*>(gamma + rl.more);
                gm[0] = ga.x, gm[1] = ga.y, gm[2] = ga.z, gm[3] = ga.w, gm[4] = gb.x, gm[5] = gb.y, gm[6] = gb.z, gm[7] = gb.w;
            }
        }
        // (a position that the tables do not have reads their first rows: t < n_new <= n_pos was checked by the host)
        rl.load(p.cos_t, p.sin_t, p.R, li, pos);
        rl.template rotate<false>(v, rot);
        float ss = 0.f;
        if constexpr (NORM) {
#pragma unroll
            for (int e = 0; e < 8; e += 2) ss += rot[e] * rot[e] + rot[e + 1] * rot[e + 1];
            ss = rn_row_sum<LPR>(ss);  // every lane takes part in the shuffles
        }
        if (!live) continue;
        if (bad) {
            if (li == 0) atomicCAS(p.status, 0, bad);
            continue;
        }
        const long long at = (static_cast<long long>(b) * p.Hkv + h) * p.L_cap + row;  // of k and v rows
        if (which == 2) {
            rotary_store8<false, HALF>(p.vcache, at * D, rl.at, rl.more, v);
            continue;
        }
        if constexpr (NORM) {
            const float rstd = rn_rstd<D>(ss, p.eps);
            float out[8];
            rn_scale8(rot, rstd, gm, out);
#pragma unroll
            for (int e = 0; e < 8; ++e) rot[e] = out[e];
        }
        if (which == 0) {
            rotary_store8<false, HALF>(p.q_out, ((static_cast<long long>(b) * p.Hq + h) * p.n_new + t) * D, rl.at, rl.more, rot);
        } else {
            rotary_store8<false, HALF>(p.kcache, at * D, rl.at, rl.more, rot);
            if (p.positions && li == 0) p.positions[at] = int(pos);
            if (p.weights && li == 0) p.weights[at] = 0.f;
        }
    }
}

}  // namespace b200attn
