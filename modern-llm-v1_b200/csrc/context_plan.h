// How the operators for long contexts deal out their work: decode behind shared prompts (attn_prefix.cuh, attn_decode.cuh) and the keys'
// weights of a chunk (key_weights.cuh).  Host arithmetic only.
#pragma once

#include "attn_prefix.cuh"
#include "decode_plan.h"
#include "host_common.h"
#include "key_weights.cuh"

#include <algorithm>

namespace b200attn {

inline size_t round256(size_t n) { return (n + 255) & ~size_t(255); }
// the largest divisor of n that is at most `most`
inline int divisor(int n, int most) {
    int g = std::min(n, most);
    while (n % g) --g;
    return g;
}

// How the prompts' rows and keys are dealt (attn_prefix.cuh), and the decode behind
struct PrefixPlan {
    int heads, n_chunks, seqs, tiles, splits;
    long long units;  // tiles of rows of all prompts, KV heads and chunks
    long long grid;
    DecodePlan decode;
    size_t decode_bytes, bytes;  // of the workspace: the decode's own, all
    size_t slots;
};
// The two kernels run side by side, the prompts' one CTA per SM and the decode two on each of the others.  SMs are shared out so that the
// longer of the two, and the join behind it, is shortest; of a decode in shares of units only the join is counted, as if it were always done
// when the prompts are.  What a CTA takes, in us, from timing calls with every number of splits:
constexpr double kPrefixStart = 4.0, kUnitStart = 2.0, kDecodeTile = 0.95;  // a prompt's CTA without its tiles, a decode's unit without its tiles, one of those (32 KB)
constexpr double prefix_tile(int D) { return D == 64 ? 0.95 : 1.1; }
constexpr double kJoinRound = 0.7;
// (us with so many splits; G prompts x n samples, P, L, heads, D, lengths up to L.  8 x 16 2000 300 16/4 64: 1 22.0, 2 18.4, 3 21.7, 4 22.1;
// the same with L=1: 20.8, 15.7, 19.4, 19.8; 2 x 57 2432 6 16/4 64: 2 16.7, 4 14.5, 6 17.9, 8 18.2; 1 x 128 8000 100 16/4 64: 3 25.6, 5 20.7, 6 22.5,
// 8 25.9; 4 x 16 8000 200 16/4 128: 3 30.1, 5 25.2, 6 25.9, 8 32.9.  By the keys to be gone through alone, as before, it took 1, 1, 3, 5 and 5; as it is
// 2, 2, 4, 5 and 7.)
inline PrefixPlan prefix_plan(int B, int G, int P, int L, int Hq, int Hkv, int D, bool ragged) {
    PrefixPlan d;
    const int group = Hq / Hkv, n = B / G, sms = sm_count();
    d.heads = divisor(group, 128);
    d.n_chunks = group / d.heads;
    d.seqs = std::min(n, 128 / d.heads);
    d.tiles = (n + d.seqs - 1) / d.seqs;
    d.units = (long long)G * Hkv * d.n_chunks * d.tiles;
    const int all = (P + kPrefixKeys - 1) / kPrefixKeys;
    const long long decode_units = (long long)B * Hkv * (group / decode_heads_per_cta(group));
    const int keys = decode_tile_keys(D);
    const double unit = kUnitStart + kDecodeTile * (ragged ? 0.5 + 0.5 * L / keys : (double)((L + keys - 1) / keys));
    // `splits` of the keys, and what that takes
    const auto deal = [&](int splits) {
        d.splits = splits;
        d.grid = d.units * splits;
        const int left = d.grid < sms ? sms - (int)d.grid : sms, cap = std::min(2 * left, kDecodeMaxCtas);
        d.decode = decode_plan(B, L, Hq, Hkv, D, 0, ragged, cap, true, splits);
        if (d.grid >= sms) d.decode.turn = d.decode.n_ctas;  // all of them start as the prompts' CTAs end
        const double prompts = kPrefixStart + prefix_tile(D) * ((all + splits - 1) / splits);
        if (d.decode.shares > 0) return prompts + kJoinRound * decode_join_rounds(d.decode.G, D, d.decode.cluster, splits);
        const long long units = (decode_units + cap - 1) / cap;
        return std::max(prompts, unit * (double)decode_units / cap) + kJoinRound * (double)((units * d.decode.G * (D / 4) + 255) / 256) * ((splits + 3) / 4);
    };
    int per = (int)std::max<long long>(1, std::min<long long>(all, (all * d.units + sms - 1) / sms)), best = (all + per - 1) / per;  // tiles of keys a split
    if (best * d.units >= sms && per < all) best = (all + per) / (per + 1), ++per;
    double least = deal(best);
    for (per += 1 + per / 8; per < all + 1 + all / 8 && kPrefixStart + prefix_tile(D) * std::min(per, all) < least * 1.03; per += 1 + per / 8) {
        const int splits = (all + per - 1) / per;
        const double t = deal(splits);
        if (t <= least * 1.03) best = splits;  // (of about equal ones the one that leaves the decode more SMs)
        least = std::min(least, t);
    }
    deal(best);
    d.slots = (size_t)d.units * d.splits;
    d.decode_bytes = round256((size_t)B * Hq * d.decode.splits * (size_t)(D + 2) * sizeof(float));
    d.bytes = d.decode_bytes + (d.slots * 128 + (size_t)B * Hq) * (D + 2) * sizeof(float);
    return d;
}

inline bool shared_sizes_ok(int B, int G, int P, int L, int Hq, int Hkv, int D) {
    return B > 0 && G > 0 && B % G == 0 && P > 0 && L > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && (D == 64 || D == 128);
}

// How a chunk's units are made (key_weights.cuh)
inline void key_weights_plan(KeyWeightsParams& p, int B, int T, int pos0, int Hq, int Hkv) {
    p.T = T, p.pos0 = pos0, p.L = pos0 + T, p.Hq = Hq, p.Hkv = Hkv, p.group = Hq / Hkv;
    p.tokens = std::min(T, 128);
    p.heads = divisor(p.group, 128 / p.tokens);
    p.n_qt = (T + p.tokens - 1) / p.tokens;
    p.n_hc = p.group / p.heads;
    p.div_hc = fastdiv_make((unsigned)p.n_hc), p.div_tokens = fastdiv_make((unsigned)p.tokens);
    p.n_kt = (p.L + 127) / 128;
    // tiles of keys up to full_kt are seen by all tiles of tokens (a chunk of at most 128 tokens is one tile)
    p.full_kt = p.n_qt == 1 ? p.n_kt : (pos0 + 127) / 128;
}
// units of all items, beyond 32 bits too
inline long long key_weights_total(const KeyWeightsParams& p, int B) {
    const long long m = std::max(0, p.n_kt - p.full_kt);
    return (long long)B * p.Hkv * (((long long)p.n_kt * p.n_qt - m * (m - 1) / 2) * p.n_hc);
}
// What each CTA takes of them
inline void key_weights_deal(KeyWeightsParams& p, int total) {
    p.total = total;
    p.n_ctas = std::min(sm_count(), total);
    p.per_cta = total / p.n_ctas, p.more = total % p.n_ctas;
}
inline size_t key_weights_bytes(int B, int T, int pos0, int Hkv) {
    return ((size_t)B * Hkv * ((pos0 + (size_t)T + 127) / 128) + sm_count()) * kKeyWeightsGroups * 128 * sizeof(float);
}

}  // namespace b200attn
