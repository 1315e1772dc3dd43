// C ABI of the operators for long-context sampling: decode behind a shared prompt, attention weights of cached keys, eviction
// (attn_prefix.cuh, key_weights.cuh, kv_evict.cuh; contract in include/b200attn.h).
#include "context_plan.h"
#include "kv_evict.cuh"
#include "tmap.h"

#include <algorithm>
#include <math.h>

using namespace b200attn;

namespace {

inline float scale_of(float softmax_scale, int D) { return softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D); }
inline bool workspace_ok(const void* ws, size_t have, size_t need) { return ws && have >= need && (reinterpret_cast<uintptr_t>(ws) & 255u) == 0; }

template <int D>
int launch_prefix(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PrefixParams& p, unsigned grid, cudaStream_t st) {
    constexpr int smem = PrefixCfg<D>::kSmemBytes;
    static bool set[kMaxDevices] = {false};
    const int rc = set_smem_once(attn_prefix_kernel<D>, smem, set);
    if (rc) return rc;
    if (launch_pdl(attn_prefix_kernel<D>, dim3(grid), kPrefixThreads, smem, st, tq, tk, tv, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}
template <int D>
int launch_key_weights(const CUtensorMap& tq, const CUtensorMap& tk, const KeyWeightsParams& p, unsigned items, cudaStream_t st) {
    static bool set[kMaxDevices] = {false};
    const int rc = set_smem_once(key_weights_kernel<D>, KeyWeightsCfg<D>::kSmemBytes, set);
    if (rc) return rc;
    if (launch_pdl(key_weights_kernel<D>, dim3(p.n_ctas), kKeyWeightsThreads, KeyWeightsCfg<D>::kSmemBytes, st, tq, tk, p) != cudaSuccess ||
        launch_pdl(key_weights_add_kernel, dim3(items), 128, 0, st, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}

// Eviction by one kernel, whose CTAs select for themselves, or by two: with more units than this an SM would have to select more often than
// its share of the moves is worth.
constexpr int kEvictListUnits = 74;

template <int D, bool BIG, bool LIST>
int launch_evict_kernel(const EvictParams& p, unsigned grid, cudaStream_t st) {
    static bool set[kMaxDevices] = {false};
    const int rc = set_smem_once(kv_evict_kernel<D, BIG, LIST>, kEvictFixedSmem + (BIG ? 0 : kEvictMaxKeys * 4), set);
    if (rc) return rc;
    if (launch_pdl(kv_evict_kernel<D, BIG, LIST>, dim3(grid), kEvictThreads, kEvictFixedSmem + (BIG ? 0 : (size_t)p.L * 4), st, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}
template <int D>
int launch_evict(const EvictParams& p, long long units, cudaStream_t st) {
    const bool big = p.L > kEvictMaxKeys;
    if (!p.moves) {
        const unsigned grid = (unsigned)(units * p.ranks);
        return big ? launch_evict_kernel<D, true, false>(p, grid, st) : launch_evict_kernel<D, false, false>(p, grid, st);
    }
    const int rc = big ? launch_evict_kernel<D, true, true>(p, (unsigned)units, st) : launch_evict_kernel<D, false, true>(p, (unsigned)units, st);
    if (rc) return rc;
    if (launch_pdl(kv_move_kernel<D>, dim3((unsigned)(units * p.blocks)), kMoveThreads, 0, st, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}
// Most moves of a unit, and whether they are listed for a kernel of their own (see kv_evict.cuh)
inline int evict_most(int L, int keep) { return std::max(0, std::min(keep, L - keep)); }
inline bool evict_lists(long long units, int L, int keep) { return units > kEvictListUnits && evict_most(L, keep) > 0; }

}  // namespace

extern "C" size_t b200attn_decode_shared_workspace_bytes(int B, int G, int P, int L, int Hq, int Hkv, int D) {
    if (!shared_sizes_ok(B, G, P, L, Hq, Hkv, D)) return 0;
    return std::max(prefix_plan(B, G, P, L, Hq, Hkv, D, false).bytes, prefix_plan(B, G, P, L, Hq, Hkv, D, true).bytes);
}

extern "C" int b200attn_decode_shared(const void* q, const void* kprefix, const void* vprefix, const void* kcache, const void* vcache, void* o,
                                      float* lse, const int* prefix_lens, const int* lens, int B, int G, int P, int P_cap, int L, int L_cap,
                                      int Hq, int Hkv, int D, float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_common(B, L, Hq, Hkv, D, B200ATTN_LAYOUT_BHTD);
    if (rc) return rc;
    if (!shared_sizes_ok(B, G, P, L, Hq, Hkv, D) || P_cap < P || L_cap < L) return B200ATTN_ERR_INVALID_ARG;
    if (!q || !kprefix || !vprefix || !kcache || !vcache || !o) return B200ATTN_ERR_INVALID_ARG;
    for (const void* a : {q, kprefix, vprefix, kcache, vcache, (const void*)o})
        if (!aligned16(a)) return B200ATTN_ERR_ALIGNMENT;
    const PrefixPlan x = prefix_plan(B, G, P, L, Hq, Hkv, D, lens != nullptr);
    if (x.units * x.splits >= (1LL << 31) || x.grid >= (1LL << 31) || (long long)B * Hq * D >= (1LL << 37)) return B200ATTN_ERR_TOO_LARGE;
    if (!workspace_ok(workspace, workspace_bytes, b200attn_decode_shared_workspace_bytes(B, G, P, L, Hq, Hkv, D))) return B200ATTN_ERR_WORKSPACE;
    int* status = status_ptr(&rc);
    if (!status) return rc;
    const Strides sp = strides_for(B200ATTN_LAYOUT_BHTD, Hkv, P_cap, D);
    CUtensorMap tq, tkp, tvp, tk, tv;
    // rows of q as (head, sequence): "tokens" of the map are heads, its "heads" are sequences
    if (!make_tmap_bf16_4d(&tq, q, D, Hq, B, 1, D, (long long)Hq * D, (long long)B * Hq * D, x.heads, x.seqs) ||
        !make_tmap_bf16_4d(&tkp, kprefix, D, P, Hkv, G, sp.t, sp.h, sp.b, kPrefixKeys) || !make_tmap_bf16_4d(&tvp, vprefix, D, P, Hkv, G, sp.t, sp.h, sp.b, kPrefixKeys))
        return B200ATTN_ERR_TENSOR_MAP;
    const DecodePlan& d = x.decode;
    DecodeParams dp;
    rc = decode_fill(d, dp, tk, tv, q, kcache, vcache, o, lse, lens, B, L, L_cap, Hq, Hkv, D, softmax_scale, workspace, status);
    if (rc) return rc;
    PrefixParams p = {};
    p.P = P, p.n = B / G, p.heads = x.heads, p.seqs = x.seqs, p.group = Hq / Hkv, p.n_chunks = x.n_chunks, p.Hkv = Hkv;
    p.splits = x.splits, p.tiles = x.tiles;
    p.div_splits = fastdiv_make((unsigned)x.splits), p.div_tiles = fastdiv_make((unsigned)x.tiles);
    p.div_chunks = fastdiv_make((unsigned)x.n_chunks), p.div_hkv = fastdiv_make((unsigned)Hkv);
    p.lens = prefix_lens;
    p.scale_log2 = dp.scale_log2;
    p.o = reinterpret_cast<float*>(static_cast<char*>(workspace) + x.decode_bytes);
    p.ml = reinterpret_cast<float2*>(p.o + x.slots * 128 * D);
    p.status = status;
    DecodePrefix& e = dp.prefix;
    e.o = p.o, e.ml = p.ml, e.splits = x.splits, e.tiles = x.tiles, e.n_chunks = x.n_chunks, e.Hkv = Hkv;
    e.div_n = fastdiv_make((unsigned)p.n), e.div_heads = fastdiv_make((unsigned)x.heads), e.div_seqs = fastdiv_make((unsigned)x.seqs);
    if (d.shares == 0) {
        e.own_o = reinterpret_cast<float*>(p.ml + x.slots * 128);
        e.own_ml = reinterpret_cast<float2*>(e.own_o + (size_t)B * Hq * D);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)x.grid;
    rc = D == 64 ? launch_prefix<64>(tq, tkp, tvp, p, grid, st) : launch_prefix<128>(tq, tkp, tvp, p, grid, st);
    if (!rc) rc = d.in_turn ? launch_decode<kDecodeSharedTurn>(D, tk, tv, dp, d.n_ctas, st) : launch_decode<kDecodeShared>(D, tk, tv, dp, d.n_ctas, st);
    return rc;
}

extern "C" size_t b200attn_decode_weights_workspace_bytes(int B, int L, int Hq, int Hkv, int D) {
    if (B <= 0 || L <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || (D != 64 && D != 128)) return 0;
    return round256(b200attn_decode_workspace_bytes(B, L, Hq, Hkv, D, 0)) + (size_t)B * Hq * ((size_t)L + 1) * sizeof(float);
}

extern "C" int b200attn_decode_weights(const void* q, const void* kcache, const void* vcache, void* o, float* lse, float* weights,
                                       const int* lens, int B, int L, int L_cap, int Hq, int Hkv, int D, float softmax_scale,
                                       void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_common(B, L, Hq, Hkv, D, B200ATTN_LAYOUT_BHTD);
    if (rc) return rc;
    if (L_cap < L || !q || !kcache || !vcache || !o || !weights) return B200ATTN_ERR_INVALID_ARG;
    for (const void* a : {q, kcache, vcache, (const void*)o})
        if (!aligned16(a)) return B200ATTN_ERR_ALIGNMENT;
    if (!workspace_ok(workspace, workspace_bytes, b200attn_decode_weights_workspace_bytes(B, L, Hq, Hkv, D))) return B200ATTN_ERR_WORKSPACE;
    const int blocks = (L + kDecodeWeightsThreads * kDecodeWeightsKeys - 1) / (kDecodeWeightsThreads * kDecodeWeightsKeys);
    if ((long long)B * Hkv * blocks >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;
    int* status = status_ptr(&rc);
    if (!status) return rc;
    float* own = reinterpret_cast<float*>(static_cast<char*>(workspace) + round256(b200attn_decode_workspace_bytes(B, L, Hq, Hkv, D, 0)));
    if (!lse) lse = own + (size_t)B * Hq * L;
    const DecodePlan d = decode_plan(B, L, Hq, Hkv, D, 0, lens != nullptr);
    CUtensorMap tk, tv;
    DecodeParams p;
    rc = decode_fill(d, p, tk, tv, q, kcache, vcache, o, lse, lens, B, L, L_cap, Hq, Hkv, D, softmax_scale, workspace, status);
    if (rc) return rc;
    p.scores = own;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = launch_decode<kDecodeScores>(D, tk, tv, p, d.n_ctas, st);
    if (rc) return rc;
    DecodeWeightsParams w = {own, lse, weights, lens, status, L, L_cap, Hkv, d.G, d.n_chunks, blocks, p.scale_log2};
    if (launch_pdl(decode_weights_kernel, dim3((unsigned)(B * Hkv * blocks)), kDecodeWeightsThreads, 0, st, w) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}

extern "C" size_t b200attn_key_weights_workspace_bytes(int B, int T, int pos0, int Hkv) {
    if (B <= 0 || T <= 0 || pos0 < 0 || Hkv <= 0 || (long long)pos0 + T > INT_MAX) return 0;
    return key_weights_bytes(B, T, pos0, Hkv);
}

extern "C" int b200attn_key_weights(const void* q, int q_layout, const void* kcache, const float* lse, float* weights, const int* new_lens, int B,
                                    int T, int pos0, int L_cap, int Hq, int Hkv, int D, float softmax_scale, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    int rc = check_common(B, T, Hq, Hkv, D, q_layout);
    if (rc) return rc;
    if (pos0 < 0 || (long long)pos0 + T > L_cap || !q || !kcache || !lse || !weights) return B200ATTN_ERR_INVALID_ARG;
    if (!aligned16(q) || !aligned16(kcache)) return B200ATTN_ERR_ALIGNMENT;
    if (!workspace_ok(workspace, workspace_bytes, b200attn_key_weights_workspace_bytes(B, T, pos0, Hkv))) return B200ATTN_ERR_WORKSPACE;
    KeyWeightsParams p = {};
    key_weights_plan(p, B, T, pos0, Hq, Hkv);
    const long long items = (long long)B * Hkv * p.n_kt;
    const long long total = key_weights_total(p, B);
    if (items >= (1LL << 31) || total >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;
    key_weights_deal(p, (int)total);
    p.status = status_ptr(&rc);
    if (!p.status) return rc;
    p.lse = lse, p.rows = new_lens, p.w = weights, p.part = static_cast<float*>(workspace), p.L_cap = L_cap;
    p.scale_log2 = scale_of(softmax_scale, D) * kLog2e;
    const Strides sq = strides_for(q_layout, Hq, T, D), sk = strides_for(B200ATTN_LAYOUT_BHTD, Hkv, L_cap, D);
    CUtensorMap tq, tk;
    // (the map of k ends at the newest token: zeros beyond it, whatever the cache holds there)
    if (!make_tmap_bf16_4d(&tq, q, D, T, Hq, B, sq.t, sq.h, sq.b, p.tokens, p.heads) ||
        !make_tmap_bf16_4d(&tk, kcache, D, p.L, Hkv, B, sk.t, sk.h, sk.b, 128))
        return B200ATTN_ERR_TENSOR_MAP;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return D == 64 ? launch_key_weights<64>(tq, tk, p, (unsigned)items, st) : launch_key_weights<128>(tq, tk, p, (unsigned)items, st);
}

extern "C" size_t b200attn_kv_evict_workspace_bytes(int B, int L, int Hkv, int keep) {
    if (B <= 0 || L <= 0 || Hkv <= 0 || keep <= 0) return 0;
    const long long units = (long long)B * Hkv;
    return evict_lists(units, L, keep) ? (size_t)units * (evict_most(L, keep) * sizeof(int2) + sizeof(int)) : 0;
}

extern "C" int b200attn_kv_evict(void* kcache, void* vcache, const float* weights, const int* positions, float* weights_out, int* positions_out,
                                 const int* lens, int B, int L, int L_cap, int Hkv, int D, int keep, int recent, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    if (B <= 0 || L <= 0 || Hkv <= 0 || L_cap < L || keep <= 0 || recent < 0 || recent > keep) return B200ATTN_ERR_INVALID_ARG;
    if (D != 64 && D != 128) return B200ATTN_ERR_UNSUPPORTED;
    if (!kcache || !vcache || !weights || !positions || !weights_out || !positions_out) return B200ATTN_ERR_INVALID_ARG;
    if (!aligned16(kcache) || !aligned16(vcache)) return B200ATTN_ERR_ALIGNMENT;
    const long long units = (long long)B * Hkv;
    if (units >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;
    // every CTA reads all of the inputs: no output may lie over them
    const size_t rows = (size_t)units * L_cap;
    auto apart = [&](const void* a, const void* b) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
        return x + rows * 4 <= y || y + rows * 4 <= x;
    };
    if (!apart(weights, weights_out) || !apart(positions, positions_out) || !apart(weights, positions_out) || !apart(positions, weights_out) ||
        !apart(weights_out, positions_out))
        return B200ATTN_ERR_INVALID_ARG;
    const bool lists = evict_lists(units, L, keep);
    if (lists && !workspace_ok(workspace, workspace_bytes, b200attn_kv_evict_workspace_bytes(B, L, Hkv, keep))) return B200ATTN_ERR_WORKSPACE;
    int rc = B200ATTN_OK;
    EvictParams p = {};
    p.status = status_ptr(&rc);
    if (!p.status) return rc;
    p.k = static_cast<uint16_t*>(kcache), p.v = static_cast<uint16_t*>(vcache);
    p.w = weights, p.pos = positions, p.w_out = weights_out, p.pos_out = positions_out, p.lens = lens;
    p.L = L, p.L_cap = L_cap, p.Hkv = Hkv, p.keep = keep, p.recent = recent;
    p.ranks = (int)std::max<long long>(1, std::min<long long>(std::min<long long>(8, (L + 255) / 256), sm_count() / units));
    if (lists) {
        p.most = evict_most(L, keep);
        p.blocks = (p.most + kMoveRows - 1) / kMoveRows;
        p.moves = static_cast<int2*>(workspace);
        p.n_moves = reinterpret_cast<int*>(p.moves + (size_t)units * p.most);
    }
    if (units * std::max(p.ranks, p.blocks) >= (1LL << 31)) return B200ATTN_ERR_TOO_LARGE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return D == 64 ? launch_evict<64>(p, units, st) : launch_evict<128>(p, units, st);
}
