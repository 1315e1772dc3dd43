// Rotary positions in other layouts than the reference's, on the way into the attention kernels and back: pairs of neighbours or of the
// two halves, the first R of a head's D elements, a position per token, with the QK-norm behind the rotation (where the reference has it)
// or without.  A norm in front of the rotation is not among them: with a gamma that differs within a pair the two do not commute.
// (rope_norm.cuh is the reference's one form of it: all of the head, neighbours, the norm always, llm/src/model/rope.cu:25-65.)
//
//   the pair i < R / 2 of a row at position p is  (a, b) = (x[2i], x[2i+1])  or  (x[i], x[i + R/2])
//   r: (a cos - b sin, a sin + b cos) with cos, sin = tables[p][i];  elements >= R stay
//   y = r, or with the norm  rstd = rsqrt(mean r^2 + eps), y = r rstd gamma
//   back, with the norm:  g = dy gamma, s = sum g r, dr = rstd g - rstd^3 / D s r, d_gamma += sum over rows of dy r rstd;
//   without it dr = dy (x is not read);  dx: (da cos + db sin, -da sin + db cos)
//
// Bound by HBM like rope_norm.cuh, whose deal of the work this is: a lane owns 8 elements of a row, a warp 256 / D tokens and a chunk of
// heads, so that a token's cosines and sines stay in registers.  Where the halves are paired a lane's 8 elements are four pairs, two
// pieces of four R / 2 apart (R is a multiple of 16); behind R they are two pieces side by side.  (Eight elements in a row, with the
// partners by shuffle, took twice the registers for the tables and 8 to 16 shuffles a row: backward with the norm, BF16 B=4 T=8192 16/4
// D=128, 122.8 us instead of 106.)  Measured, q and k together: that backward 4.8 TB/s (interleaved 100 us); FP32 forward with the norm,
// B=16 T=1024 16/4 D=64 R=32, 23.4 us, 5.4 TB/s; without the norm B=4 T=8192 16/4 D=128 BF16 58.0 us forward and 58.3 back (5.8 TB/s), FP32
// R=64 82.5 and 86.9 (6.1, 5.8); one token 4 us, a launch.  More rows in flight (3 or 4 instead of 2), 2 or 4 CTAs per SM
// instead of 3: all slower (102.6 -> 105 to 130).
#pragma once

#include "rope_norm.cuh"

namespace b200attn {

struct RotaryParams : RopeNormParams {
    const int* pos;  // [B, T] positions, or nullptr: token t has position t
    int n_pos;       // rows of the tables [n_pos, R / 2]
    int R;
    int* status;     // set to DEV_ROTARY_POSITION when a position is not a row of the tables (the token's rows are skipped)
};

// A lane's 8 elements of a row and its share of one row of the tables: four pairs either way, (v[2i], v[2i+1]) of neighbours, (v[i], v[i+4])
// of halves.
template <int D, bool HALF>
struct RotaryLane {
    float c[4], s[4];
    bool turns;    // the lane's elements are rotated
    int at, more;  // the lane's first four elements, and how much further the other four are (4 but for pairs of halves)
    // li: the lane within its row's D / 8
    __device__ __forceinline__ RotaryLane(int R, int li) {
        turns = li * 8 < R;
        at = HALF && turns ? li * 4 : li * 8;
        more = HALF && turns ? R / 2 : 4;
    }
    __device__ __forceinline__ void load(const float* cos_t, const float* sin_t, int R, int li, long long pos) {
        if (!turns) {
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = 1.f, s[e] = 0.f;
            return;
        }
        const long long at_t = pos * (R / 2) + li * 4;
        const float4 cv = *reinterpret_cast<const float4*>(cos_t + at_t), sv = *reinterpret_cast<const float4*>(sin_t + at_t);
        c[0] = cv.x, c[1] = cv.y, c[2] = cv.z, c[3] = cv.w;
        s[0] = sv.x, s[1] = sv.y, s[2] = sv.z, s[3] = sv.w;
    }
    // BACK: by the opposite angle
    template <bool BACK>
    __device__ __forceinline__ void rotate(const float (&v)[8], float (&out)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = HALF ? i : 2 * i, y = HALF ? i + 4 : 2 * i + 1;
            const float a = v[x], b = v[y];
            // (elements that do not turn are copied: times one plus zero times another would make NaN of infinities)
            out[x] = !turns ? a : BACK ? a * c[i] + b * s[i] : a * c[i] - b * s[i];
            out[y] = !turns ? b : BACK ? b * c[i] - a * s[i] : a * s[i] + b * c[i];
        }
    }
};
// The lane's 8 elements of the row that begins at element offset `row`, as they lie in memory
template <bool F32, bool HALF>
struct RotaryRaw {
    RnRaw<F32> r;
    __device__ __forceinline__ void load(const void* base, long long row, int at, int more) {
        if constexpr (!HALF) {
            r.load(base, row + at);
        } else if constexpr (F32) {
            const float* const ptr = static_cast<const float*>(base) + row + at;
            r.w[0] = __ldcs(reinterpret_cast<const uint4*>(ptr)), r.w[1] = __ldcs(reinterpret_cast<const uint4*>(ptr + more));
        } else {
            const uint16_t* const ptr = static_cast<const uint16_t*>(base) + row + at;
            const uint2 a = __ldcs(reinterpret_cast<const uint2*>(ptr)), b = __ldcs(reinterpret_cast<const uint2*>(ptr + more));
            r.w[0] = make_uint4(a.x, a.y, b.x, b.y);
        }
    }
};
template <bool F32, bool HALF>
__device__ __forceinline__ void rotary_store8(void* base, long long row, int at, int more, const float (&v)[8]) {
    if constexpr (!HALF) {
        rn_store8<F32>(base, row + at, v);
    } else if constexpr (F32) {
        float* const ptr = static_cast<float*>(base) + row + at;
        *reinterpret_cast<float4*>(ptr) = make_float4(v[0], v[1], v[2], v[3]), *reinterpret_cast<float4*>(ptr + more) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint16_t* const ptr = static_cast<uint16_t*>(base) + row + at;
        *reinterpret_cast<uint2*>(ptr) = make_uint2(rn_pack_bf16x2(v[0], v[1]), rn_pack_bf16x2(v[2], v[3]));
        *reinterpret_cast<uint2*>(ptr + more) = make_uint2(rn_pack_bf16x2(v[4], v[5]), rn_pack_bf16x2(v[6], v[7]));
    }
}
// gamma of the lane's elements, one by one: it may begin at any float of a buffer that holds all of a model's parameters.  (Once per
// warp, in front of its rows; against 16-byte loads only the backward of FP32 half pairs takes longer, by a spill: B=4 T=4096 16/4 D=128
// 72.2 us instead of 71.5.)
__device__ __forceinline__ void rotary_gamma(const float* gamma, int at, int more, float (&g)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = gamma[at + e], g[e + 4] = gamma[at + more + e];
}

// The position of a lane's token; a token whose position the tables do not have is dropped (live = false).
template <int D>
__device__ __forceinline__ int rotary_position(const RotaryParams& p, RnItem<D>& it) {
    if (!p.pos || !it.live) return it.live ? it.t : 0;
    const int pos = __ldg(p.pos + static_cast<long long>(it.b) * p.T + it.t);
    if (pos >= 0 && pos < p.n_pos) return pos;
    it.live = false;
    atomicCAS(p.status, 0, int(DEV_ROTARY_POSITION));
    return 0;
}

template <int D, bool F32, bool HALF, bool NORM>
__device__ __forceinline__ unsigned rotary_fwd_tensor(const RotaryParams& p, unsigned item, unsigned n_warps) {
    constexpr int LPR = D / 8;
    constexpr int kUnroll = 4;
    const int lane = threadIdx.x & 31;
    const int sub = lane / LPR, li = lane % LPR;
    RotaryLane<D, HALF> rl(p.R, li);
    float gm[8];
    if constexpr (NORM) {
        rotary_gamma(p.gamma, rl.at, rl.more, gm);
    }
    for (; item < p.n_items; item += n_warps) {
        RnItem<D> it(p, item, sub);
        rl.load(p.cos_t, p.sin_t, p.R, li, rotary_position<D>(p, it));
        const long long x_off = it.b * p.x_sb + it.t * p.x_st, y_off = it.b * p.y_sb + it.t * p.y_st;
        float* rstd_t = NORM ? p.rstd + static_cast<long long>(it.b) * p.H * p.T + it.t : nullptr;
        for (int h = it.h0; h < it.h1; h += kUnroll) {
            RotaryRaw<F32, HALF> raw[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                raw[k].r.clear();
                if (it.live && h + k < it.h1) raw[k].load(p.x, x_off + (h + k) * p.x_sh, rl.at, rl.more);
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                if (h + k >= it.h1) break;
                float v[8], rot[8];
                raw[k].r.get(v);
                rl.template rotate<false>(v, rot);
                if constexpr (NORM) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) ss += rot[e] * rot[e] + rot[e + 1] * rot[e + 1];
                    const float rstd = rn_rstd<D>(rn_row_sum<LPR>(ss), p.eps);
                    float out[8];
                    rn_scale8(rot, rstd, gm, out);
                    if (it.live) {
                        rotary_store8<false, HALF>(p.y, y_off + (h + k) * p.y_sh, rl.at, rl.more, out);
                        if (li == 0) rstd_t[static_cast<long long>(h + k) * p.T] = rstd;
                    }
                } else if (it.live) {
                    rotary_store8<false, HALF>(p.y, y_off + (h + k) * p.y_sh, rl.at, rl.more, rot);
                }
            }
        }
    }
    return item - p.n_items;
}

template <int D, bool F32, bool HALF, bool NORM>
__global__ void __launch_bounds__(kRopeNormThreads, kRopeNormFwdBlocks)
rotary_fwd_kernel(const __grid_constant__ RotaryParams p0, const __grid_constant__ RotaryParams p1) {
    const unsigned warp = (blockIdx.x * kRopeNormThreads + threadIdx.x) >> 5, n_warps = (gridDim.x * kRopeNormThreads) >> 5;
    grid_dep_wait();
    const unsigned next = rotary_fwd_tensor<D, F32, HALF, NORM>(p0, warp, n_warps);
    rotary_fwd_tensor<D, F32, HALF, NORM>(p1, next, n_warps);
}

// One tensor's backward; with the norm it leaves this CTA's d_gamma sums in p.partial, which rope_norm_dgamma_kernel adds up.
template <int D, bool F32, bool HALF, bool NORM>
__device__ __forceinline__ unsigned rotary_bwd_tensor(const RotaryParams& p, unsigned item, unsigned n_warps, float (*s_part)[D]) {
    constexpr int LPR = D / 8;
    constexpr int kUnroll = NORM ? 2 : 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int sub = lane / LPR, li = lane % LPR;
    RotaryLane<D, HALF> rl(p.R, li);
    float gm[8], dg[8];
    if constexpr (NORM) {
        rotary_gamma(p.gamma, rl.at, rl.more, gm);
#pragma unroll
        for (int e = 0; e < 8; ++e) dg[e] = 0.f;
    }
    for (; item < p.n_items; item += n_warps) {
        RnItem<D> it(p, item, sub);
        rl.load(p.cos_t, p.sin_t, p.R, li, rotary_position<D>(p, it));
        const long long x_off = it.b * p.x_sb + it.t * p.x_st, y_off = it.b * p.y_sb + it.t * p.y_st;
        const float* rstd_t = NORM ? p.rstd + static_cast<long long>(it.b) * p.H * p.T + it.t : nullptr;
        for (int h = it.h0; h < it.h1; h += kUnroll) {
            RotaryRaw<F32, HALF> raw_x[NORM ? kUnroll : 1];
            RotaryRaw<false, HALF> raw_dy[kUnroll];
            float rstd[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                if constexpr (NORM) raw_x[k].r.clear();
                raw_dy[k].r.clear();
                rstd[k] = 0.f;
                if (it.live && h + k < it.h1) {
                    raw_dy[k].load(p.dy, y_off + (h + k) * p.y_sh, rl.at, rl.more);
                    if constexpr (NORM) {
                        raw_x[k].load(p.x, x_off + (h + k) * p.x_sh, rl.at, rl.more);
                        rstd[k] = rstd_t[static_cast<long long>(h + k) * p.T];
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                if (h + k >= it.h1) break;
                float d[8], dx[8];
                raw_dy[k].r.get(d);
                if constexpr (NORM) {
                    float v[8], rot[8];
                    raw_x[k].r.get(v);
                    rl.template rotate<false>(v, rot);
                    const float rs = rstd[k];
                    float s = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float g = d[e] * gm[e];
                        s += g * rot[e];
                        dg[e] += d[e] * rot[e] * rs;
                        d[e] = g;
                    }
                    s = rn_row_sum<LPR>(s);
                    const float coeff = rs * rs * rs * (1.f / float(D)) * s;
#pragma unroll
                    for (int e = 0; e < 8; ++e) d[e] = rs * d[e] - coeff * rot[e];
                }
                rl.template rotate<true>(d, dx);
                if (it.live) rotary_store8<F32, HALF>(p.y, x_off + (h + k) * p.x_sh, rl.at, rl.more, dx);
            }
        }
    }
    if constexpr (NORM) {  // as in rope_norm_bwd_tensor: the lanes with the same columns, then the CTA's warps, in a fixed order
#pragma unroll
        for (int e = 0; e < 8; ++e) {
#pragma unroll
            for (int o = LPR; o < 32; o <<= 1) dg[e] += __shfl_xor_sync(0xffffffffu, dg[e], o);
        }
        if (sub == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s_part[warp][rl.at + (e < 4 ? e : rl.more + e - 4)] = dg[e];
        }
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kRopeNormThreads) {
            float acc = 0.f;
#pragma unroll
            for (int w = 0; w < kRopeNormThreads / 32; ++w) acc += s_part[w][d];
            p.partial[static_cast<long long>(blockIdx.x) * D + d] = acc;
        }
    }
    return item - p.n_items;
}

template <int D, bool F32, bool HALF, bool NORM>
__global__ void __launch_bounds__(kRopeNormThreads, kRopeNormBwdBlocks)
rotary_bwd_kernel(const __grid_constant__ RotaryParams p0, const __grid_constant__ RotaryParams p1) {
    __shared__ float s_part[2][NORM ? kRopeNormThreads / 32 : 1][D];
    const unsigned warp = (blockIdx.x * kRopeNormThreads + threadIdx.x) >> 5, n_warps = (gridDim.x * kRopeNormThreads) >> 5;
    grid_dep_wait();
    const unsigned next = rotary_bwd_tensor<D, F32, HALF, NORM>(p0, warp, n_warps, s_part[0]);
    rotary_bwd_tensor<D, F32, HALF, NORM>(p1, next, n_warps, s_part[1]);
}

// The tables: angle = position * frequency of the pair, in 64 bits (in 32 a position of 30000 turns the fastest pair by up to
// 2^-9 too far), rounded once as cosine and sine.  The frequencies come from base^(-2i/R), see b200attn_rotary_table for `scaling`.
struct RotaryTableParams {
    int T, half;
    double base, divide;                       // frequency base^(-i / half) / divide
    double trained, factor, fast, slow;        // by parts (trained > 0): frequencies that turn less often lie below
    float *cos_t, *sin_t;
};
__global__ void __launch_bounds__(256) rotary_table_kernel(const RotaryTableParams p) {
    const long long n = static_cast<long long>(p.T) * p.half;
    grid_dep_wait();
    for (long long k = blockIdx.x * 256ll + threadIdx.x; k < n; k += gridDim.x * 256ll) {
        const int t = int(k / p.half), i = int(k - static_cast<long long>(t) * p.half);
        double freq = pow(p.base, -double(i) / double(p.half)) / p.divide;
        if (p.trained > 0.0) {
            const double turns = p.trained * freq * 0.15915494309189535;  // within the trained length
            const double keep = fmin(fmax((turns - p.slow) / (p.fast - p.slow), 0.0), 1.0);
            freq = freq * keep + freq / p.factor * (1.0 - keep);
        }
        double sn, cs;
        sincos(double(t) * freq, &sn, &cs);
        p.cos_t[k] = float(cs);
        p.sin_t[k] = float(sn);
    }
}

}  // namespace b200attn
