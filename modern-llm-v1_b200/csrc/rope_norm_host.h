// How the RoPE kernels' work is dealt out on the host (rope_norm.cuh, rotary.cuh).
#pragma once

#include <algorithm>

#include "host_common.h"
#include "rope_norm.cuh"

namespace b200attn {

constexpr int kRopeNormMaxCtasPerSm = 8;  // of the backward, as far as its workspace goes
static_assert(kRopeNormBwdBlocks <= kRopeNormMaxCtasPerSm, "a partial sum per CTA");

inline int rope_norm_check(int B, int T, int H, int D, int x_dtype, int x_layout, int y_layout) {
    if (B <= 0 || T <= 0 || H <= 0 || D <= 0) return B200ATTN_ERR_INVALID_ARG;
    if (x_dtype != B200ATTN_DTYPE_BF16 && x_dtype != B200ATTN_DTYPE_F32) return B200ATTN_ERR_INVALID_ARG;
    for (int l : {x_layout, y_layout})
        if (l != B200ATTN_LAYOUT_BHTD && l != B200ATTN_LAYOUT_BTHD) return B200ATTN_ERR_INVALID_ARG;
    if (D != 64 && D != 128) return B200ATTN_ERR_UNSUPPORTED;
    if ((long long)B * T * H >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;  // rows are counted in 32 bits
    return B200ATTN_OK;
}

// Heads per item: eight of them share a token's cosines and sines and addresses, fewer when that leaves less than four items
// for a resident warp (one eighth of a wave is then the most that the last round can waste).
template <typename Params>
void rope_norm_plan(Params* p, int n_tensors, int D, unsigned warps) {
    int chunk = 8;
    auto items = [&](const RopeNormParams& q) { return (long long)((q.n_tokens + 256u / D - 1) / (256u / D)) * ((q.H + chunk - 1) / chunk); };
    auto all = [&] { return items(p[0]) + (n_tensors > 1 ? items(p[1]) : 0); };
    while (chunk > 1 && all() < (chunk > 4 ? 4LL : 1LL) * warps) chunk /= 2;
    for (int i = 0; i < n_tensors; ++i) {
        p[i].chunk = chunk;
        p[i].n_items = (unsigned)items(p[i]);
        p[i].div_chunks = fastdiv_make((unsigned)((p[i].H + chunk - 1) / chunk));
    }
}

// CTAs that the device keeps resident at once, never more than the items need
template <typename Params>
unsigned rope_norm_grid(const Params* p, int n_tensors, int blocks) {
    const long long items = (long long)p[0].n_items + (n_tensors > 1 ? p[1].n_items : 0);
    const long long need = (items + kRopeNormThreads / 32 - 1) / (kRopeNormThreads / 32);
    return (unsigned)std::min<long long>(need, (long long)blocks * sm_count());
}

inline void rope_norm_fill(RopeNormParams& p, int B, int T, int H, int D, int x_layout, int y_layout) {
    const Strides sx = strides_for(x_layout, H, T, D), sy = strides_for(y_layout, H, T, D);
    p.B = B;
    p.T = T;
    p.H = H;
    p.n_tokens = (unsigned)B * (unsigned)T;
    p.x_st = sx.t, p.x_sh = sx.h, p.x_sb = sx.b;
    p.y_st = sy.t, p.y_sh = sy.h, p.y_sb = sy.b;
    p.div_t = fastdiv_make((unsigned)T);
}

}  // namespace b200attn
