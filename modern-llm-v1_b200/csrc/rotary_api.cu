// C ABI of the rotary positions (rotary.cuh, kv_rotary.cuh; contract in include/b200attn.h).
#include "kv_rotary.cuh"
#include "rope_norm_host.h"
#include "rotary.cuh"

#include <math.h>

#include <type_traits>

using namespace b200attn;

namespace {

struct RotaryTensor {  // what differs between q and k
    const void* x;
    void* y;         // forward: y; backward: d_x
    const void* dy;  // backward only
    float* rstd;
    const float* gamma;
    float* d_gamma;
    int H;
};

int rotary_check_pairs(int D, int R, int pairs) {
    if (D != 64 && D != 128) return B200ATTN_ERR_UNSUPPORTED;
    if (R <= 0 || R > D || R % 16 != 0) return B200ATTN_ERR_INVALID_ARG;
    if (pairs != B200ATTN_PAIRS_INTERLEAVED && pairs != B200ATTN_PAIRS_HALF) return B200ATTN_ERR_INVALID_ARG;
    return B200ATTN_OK;
}

template <int D, bool F32, bool HALF, bool NORM>
int rotary_launch(bool backward, RotaryParams* p, float* ws, cudaStream_t st) {
    const int blocks = backward ? kRopeNormBwdBlocks : kRopeNormFwdBlocks;
    rope_norm_plan(p, 2, D, (unsigned)(blocks * (kRopeNormThreads / 32) * sm_count()));
    const unsigned grid = rope_norm_grid(p, 2, blocks);
    if (!backward) {
        launch_pdl(rotary_fwd_kernel<D, F32, HALF, NORM>, dim3(grid), kRopeNormThreads, 0, st, p[0], p[1]);
    } else {
        if (NORM) {
            p[0].partial = ws;
            p[1].partial = ws + (size_t)kRopeNormMaxCtasPerSm * sm_count() * D;
        }
        launch_pdl(rotary_bwd_kernel<D, F32, HALF, NORM>, dim3(grid), kRopeNormThreads, 0, st, p[0], p[1]);
        if (NORM) {
            const float *part0 = p[0].partial, *part1 = p[1].partial;
            launch_pdl(rope_norm_dgamma_kernel<D>, dim3(2 * (D / 8)), kDgammaThreads, 0, st, part0, p[0].d_gamma, part1, p[1].d_gamma, (int)grid);
        }
    }
    return cudaGetLastError() == cudaSuccess ? B200ATTN_OK : B200ATTN_ERR_CUDA;
}

int rotary_run(bool backward, const RotaryTensor (&t)[2], int x_dtype, int x_layout, int y_layout, const float* cos_t, const float* sin_t,
               const int* pos, int n_pos, int R, int pairs, int B, int T, int D, float eps, void* workspace, size_t workspace_bytes,
               void* stream) {
    int rc = rotary_check_pairs(D, R, pairs);
    if (rc) return rc;
    const bool norm = t[0].gamma != nullptr;
    RotaryParams p[2] = {};
    for (int i = 0; i < 2; ++i) {
        rc = rope_norm_check(B, T, t[i].H, D, x_dtype, x_layout, y_layout);
        if (rc) return rc;
        if (!t[i].y || (t[i].gamma != nullptr) != norm || (norm && !t[i].rstd)) return B200ATTN_ERR_INVALID_ARG;
        if ((!backward || norm) && !t[i].x) return B200ATTN_ERR_INVALID_ARG;
        if (backward && (!t[i].dy || (norm && !t[i].d_gamma))) return B200ATTN_ERR_INVALID_ARG;
        if (!aligned16(t[i].x) || !aligned16(t[i].y) || !aligned16(t[i].dy)) return B200ATTN_ERR_ALIGNMENT;
        rope_norm_fill(p[i], B, T, t[i].H, D, x_layout, y_layout);
        p[i].x = t[i].x;
        p[i].y = t[i].y;
        p[i].dy = static_cast<const uint16_t*>(t[i].dy);
        p[i].rstd = t[i].rstd;
        p[i].gamma = t[i].gamma;
        p[i].d_gamma = t[i].d_gamma;
        p[i].cos_t = cos_t;
        p[i].sin_t = sin_t;
        p[i].eps = eps;
        p[i].pos = pos;
        p[i].n_pos = n_pos;
        p[i].R = R;
    }
    if (!cos_t || !sin_t || n_pos <= 0 || (!pos && n_pos < T)) return B200ATTN_ERR_INVALID_ARG;
    if (!aligned16(cos_t) || !aligned16(sin_t)) return B200ATTN_ERR_ALIGNMENT;
    if (backward && norm && (!workspace || workspace_bytes < b200attn_rope_norm_bwd_workspace_bytes(D) ||
                             (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))
        return B200ATTN_ERR_WORKSPACE;
    p[0].status = p[1].status = status_ptr(&rc);
    if (!p[0].status) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    const bool f32 = x_dtype == B200ATTN_DTYPE_F32, half = pairs == B200ATTN_PAIRS_HALF;
    auto go = [&](auto d, auto f, auto h, auto n) { return rotary_launch<d.value, f.value, h.value, n.value>(backward, p, ws, st); };
    using std::integral_constant;
    const integral_constant<bool, true> yes;
    const integral_constant<bool, false> no;
    auto by_norm = [&](auto d, auto f, auto h) { return norm ? go(d, f, h, yes) : go(d, f, h, no); };
    auto by_half = [&](auto d, auto f) { return half ? by_norm(d, f, yes) : by_norm(d, f, no); };
    auto by_type = [&](auto d) { return f32 ? by_half(d, yes) : by_half(d, no); };
    return D == 64 ? by_type(integral_constant<int, 64>()) : by_type(integral_constant<int, 128>());
}

template <int D, bool F32, bool HALF, bool NORM>
int launch_kv_rotary(const KvRotaryParams& p, cudaStream_t st) {
    const long long rows = (long long)p.rows_q + 2LL * p.rows_kv, rows_per_cta = (kKvAppendThreads / 32) * (256 / D);
    const long long grid = std::min((rows + rows_per_cta - 1) / rows_per_cta, 8LL * sm_count());
    if (launch_pdl(kv_rotary_kernel<D, F32, HALF, NORM>, dim3((unsigned)grid), kKvAppendThreads, 0, st, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}

int kv_append_rotary_run(const void* xq, const void* xk, const void* xv, int x_dtype, void* q_out, void* kcache, void* vcache, int* positions,
                         float* weights, const float* gamma_q, const float* gamma_k, const float* cos_t, const float* sin_t, int n_pos, int R,
                         int pairs, const int* pos, int pos0, const int* rows, int row0, int B, int n_new, int L_cap, int Hq, int Hkv, int D,
                         float eps, void* stream) {
    if (B <= 0 || n_new <= 0 || pos0 < 0 || row0 < 0 || L_cap <= 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || n_pos <= 0) return B200ATTN_ERR_INVALID_ARG;
    if (Hq % Hkv != 0 || (long long)(rows ? 0 : row0) + n_new > L_cap || (long long)(pos ? 0 : pos0) + n_new > n_pos) return B200ATTN_ERR_INVALID_ARG;
    if (x_dtype != B200ATTN_DTYPE_BF16 && x_dtype != B200ATTN_DTYPE_F32) return B200ATTN_ERR_INVALID_ARG;
    int rc = rotary_check_pairs(D, R, pairs);
    if (rc) return rc;
    if (!xq || !xk || !xv || !q_out || !kcache || !vcache || !cos_t || !sin_t || (gamma_q != nullptr) != (gamma_k != nullptr))
        return B200ATTN_ERR_INVALID_ARG;
    for (const void* a : {xq, xk, xv, (const void*)q_out, (const void*)kcache, (const void*)vcache, (const void*)gamma_q, (const void*)gamma_k,
                          (const void*)cos_t, (const void*)sin_t})
        if (!aligned16(a)) return B200ATTN_ERR_ALIGNMENT;
    const long long rows_q = (long long)B * n_new * Hq, rows_kv = (long long)B * n_new * Hkv;
    if (rows_q + 2 * rows_kv >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;
    KvRotaryParams p = {};
    p.status = status_ptr(&rc);
    if (!p.status) return rc;
    p.pos = pos, p.pos0 = pos0, p.rows = rows, p.row0 = row0, p.positions = positions, p.weights = weights, p.n_pos = n_pos, p.R = R;
    p.xq = xq, p.xk = xk, p.xv = xv;
    p.q_out = static_cast<uint16_t*>(q_out);
    p.kcache = static_cast<uint16_t*>(kcache);
    p.vcache = static_cast<uint16_t*>(vcache);
    p.gamma_q = gamma_q, p.gamma_k = gamma_k, p.cos_t = cos_t, p.sin_t = sin_t;
    p.B = B, p.n_new = n_new, p.L_cap = L_cap, p.Hq = Hq, p.Hkv = Hkv;
    p.rows_q = (unsigned)rows_q, p.rows_kv = (unsigned)rows_kv;
    p.div_hq = fastdiv_make((unsigned)Hq), p.div_hkv = fastdiv_make((unsigned)Hkv), p.div_n = fastdiv_make((unsigned)n_new);
    p.eps = eps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f32 = x_dtype == B200ATTN_DTYPE_F32, half = pairs == B200ATTN_PAIRS_HALF, norm = gamma_q != nullptr;
    using std::integral_constant;
    const integral_constant<bool, true> yes;
    const integral_constant<bool, false> no;
    auto go = [&](auto d, auto f, auto h, auto n) { return launch_kv_rotary<d.value, f.value, h.value, n.value>(p, st); };
    auto by_norm = [&](auto d, auto f, auto h) { return norm ? go(d, f, h, yes) : go(d, f, h, no); };
    auto by_half = [&](auto d, auto f) { return half ? by_norm(d, f, yes) : by_norm(d, f, no); };
    auto by_type = [&](auto d) { return f32 ? by_half(d, yes) : by_half(d, no); };
    return D == 64 ? by_type(integral_constant<int, 64>()) : by_type(integral_constant<int, 128>());
}

}  // namespace

extern "C" int b200attn_rotary_table(int T, int R, double base, int scaling, double factor, double trained, double turns_fast,
                                     double turns_slow, float* cos_t, float* sin_t, void* stream) {
    if (T <= 0 || R <= 0 || (R & 1) || !cos_t || !sin_t || !(base > 0.0) || !isfinite(base)) return B200ATTN_ERR_INVALID_ARG;
    if (scaling < B200ATTN_SCALING_NONE || scaling > B200ATTN_SCALING_PARTS) return B200ATTN_ERR_INVALID_ARG;
    if (scaling != B200ATTN_SCALING_NONE && (!(factor > 0.0) || !isfinite(factor))) return B200ATTN_ERR_INVALID_ARG;
    RotaryTableParams p = {};
    p.T = T, p.half = R / 2, p.base = base, p.divide = 1.0, p.factor = 1.0, p.cos_t = cos_t, p.sin_t = sin_t;
    if (scaling == B200ATTN_SCALING_LINEAR) p.divide = factor;
    if (scaling == B200ATTN_SCALING_BASE) {
        if (R <= 2) return B200ATTN_ERR_INVALID_ARG;
        p.base = base * pow(factor, double(R) / double(R - 2));  // the slowest pair, base^(-(R-2)/R), is slowed by the factor
        if (!isfinite(p.base)) return B200ATTN_ERR_INVALID_ARG;
    }
    if (scaling == B200ATTN_SCALING_PARTS) {
        if (!(trained > 0.0) || !isfinite(trained) || !(turns_slow >= 0.0) || !(turns_fast > turns_slow) || !isfinite(turns_fast))
            return B200ATTN_ERR_INVALID_ARG;
        p.trained = trained, p.factor = factor, p.fast = turns_fast, p.slow = turns_slow;
    }
    const long long n = (long long)T * p.half;
    if (launch_pdl(rotary_table_kernel, dim3((unsigned)std::min((n + 255) / 256, 8LL * sm_count())), 256, 0, static_cast<cudaStream_t>(stream), p) !=
        cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}

extern "C" int b200attn_rotary_fwd(const void* xq, const void* xk, int x_dtype, int x_layout, void* yq, void* yk, int y_layout, float* rstd_q,
                                   float* rstd_k, const float* gamma_q, const float* gamma_k, const float* cos_t, const float* sin_t,
                                   const int* pos, int n_pos, int R, int pairs, int B, int T, int Hq, int Hkv, int D, float eps, void* stream) {
    const RotaryTensor t[2] = {{xq, yq, nullptr, rstd_q, gamma_q, nullptr, Hq}, {xk, yk, nullptr, rstd_k, gamma_k, nullptr, Hkv}};
    return rotary_run(false, t, x_dtype, x_layout, y_layout, cos_t, sin_t, pos, n_pos, R, pairs, B, T, D, eps, nullptr, 0, stream);
}

extern "C" int b200attn_rotary_bwd(const void* dyq, const void* dyk, int y_layout, const void* xq, const void* xk, int x_dtype, int x_layout,
                                   const float* rstd_q, const float* rstd_k, const float* gamma_q, const float* gamma_k, const float* cos_t,
                                   const float* sin_t, const int* pos, int n_pos, int R, int pairs, void* dxq, void* dxk, float* d_gamma_q,
                                   float* d_gamma_k, int B, int T, int Hq, int Hkv, int D, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    const RotaryTensor t[2] = {{xq, dxq, dyq, const_cast<float*>(rstd_q), gamma_q, d_gamma_q, Hq},
                               {xk, dxk, dyk, const_cast<float*>(rstd_k), gamma_k, d_gamma_k, Hkv}};
    return rotary_run(true, t, x_dtype, x_layout, y_layout, cos_t, sin_t, pos, n_pos, R, pairs, B, T, D, 0.f, workspace, workspace_bytes, stream);
}

extern "C" int b200attn_kv_append_rotary(const void* xq, const void* xk, const void* xv, int x_dtype, void* q_out, void* kcache, void* vcache,
                                         int* positions, const float* gamma_q, const float* gamma_k, const float* cos_t, const float* sin_t,
                                         int n_pos, int R, int pairs, const int* pos, int pos0, const int* rows, int row0, int B, int n_new,
                                         int L_cap, int Hq, int Hkv, int D, float eps, void* stream) {
    return kv_append_rotary_run(xq, xk, xv, x_dtype, q_out, kcache, vcache, positions, nullptr, gamma_q, gamma_k, cos_t, sin_t, n_pos, R, pairs,
                                pos, pos0, rows, row0, B, n_new, L_cap, Hq, Hkv, D, eps, stream);
}

extern "C" int b200attn_kv_append_weights(const void* xq, const void* xk, const void* xv, int x_dtype, void* q_out, void* kcache, void* vcache,
                                          int* positions, float* weights, const float* gamma_q, const float* gamma_k, const float* cos_t,
                                          const float* sin_t, int n_pos, int R, int pairs, const int* pos, int pos0, const int* rows, int row0,
                                          int B, int n_new, int L_cap, int Hq, int Hkv, int D, float eps, void* stream) {
    if (!weights) return B200ATTN_ERR_INVALID_ARG;
    return kv_append_rotary_run(xq, xk, xv, x_dtype, q_out, kcache, vcache, positions, weights, gamma_q, gamma_k, cos_t, sin_t, n_pos, R, pairs,
                                pos, pos0, rows, row0, B, n_new, L_cap, Hq, Hkv, D, eps, stream);
}
