// How a decode launch deals its units' tiles (attn_decode.cuh).
#pragma once

#include <algorithm>

#include "attn_decode.cuh"
#include "host_common.h"

namespace b200attn {

// Query heads served per decode CTA: the largest divisor of the group size that is <= 16
// (the row count of the kernel's MMA shape).
inline int decode_heads_per_cta(int group) {
    for (int g = 16; g >= 1; --g)
        if (group % g == 0) return g;
    return 1;
}

inline int decode_tile_keys(int D) { return D == 64 ? DecodeCfg<64>::kKeys : DecodeCfg<128>::kKeys; }
inline int decode_max_ctas() { return std::min(2 * sm_count(), kDecodeMaxCtas); }  // two fit an SM: all are resident at once

struct DecodePlan {
    int G, n_chunks;
    int slots;    // workspace slots per unit for partial results
    int splits;   // and with the room for the counters behind them
    int shares;   // CTAs per unit, or 0: ranges of tiles
    int cluster;  // CTAs per cluster
    bool whole;   // ranges of whole units
    int n_ctas, slot_mode;
};

// The deal (see attn_decode.cuh).
//
// Ranges cost about 3 us at the end (partial results through memory, a counter, the last CTA's additions), clusters
// about 1 us, whole units nothing.  So units stay whole or in clusters unless that leaves the memory system idle for longer
// than that: some 60 SMs saturate HBM, so what counts is how many CTAs the last round has (all, where the units are fewer
// than the SMs) and how long a unit is, and, for sequences of different lengths, how much memory there is to read at all.
// kRangesBytes is what HBM delivers in those 3 us.
//
// A cluster is the smallest that leaves a CTA at most two tiles, as far as that is one CTA per SM: more of them saturate
// HBM by themselves.
//
// n_splits > 0 asks for that many shares per unit (at most 64, none empty): a cluster where it can have that size.
constexpr long long kRangesBytes = 16ll << 20;
constexpr int kSaturatingCtas = 60;

inline DecodePlan decode_plan(int B, int L, int Hq, int Hkv, int D, int n_splits, bool ragged) {
    DecodePlan d;
    const int group = Hq / Hkv, cap = decode_max_ctas();
    d.G = decode_heads_per_cta(group);
    d.n_chunks = group / d.G;
    const long long units = (long long)B * Hkv * d.n_chunks;
    const int keys = decode_tile_keys(D), n_all = (L + keys - 1) / keys, n_128 = (L + 127) / 128;
    const long long unit_bytes = 4ll * L * D, tiles = units * n_all;
    d.shares = d.cluster = 1;
    d.whole = false;
    d.slot_mode = kDecodeSlotTile;
    long long counters = 0;
    if (n_splits > 0) {
        const int want = std::min(std::min(n_splits, n_128), 64), per = (n_128 + want - 1) / want;
        d.slots = d.shares = (n_128 + per - 1) / per;
        if (d.shares <= kDecodeMaxCluster && (d.shares & (d.shares - 1)) == 0) {
            d.cluster = d.shares;
        } else {
            d.slot_mode = kDecodeSlotCta;
            counters = units * d.shares;
        }
    } else {
        d.slots = (int)std::min<long long>(n_all, (2 * cap + units - 1) / units);
        if (n_all > 1) counters = std::min<long long>(tiles, cap);  // (a single tile is never shared)
        while (d.cluster < kDecodeMaxCluster && units * d.cluster * 2 <= sm_count() && n_all > 2 * d.cluster) d.cluster *= 2;
        d.shares = d.cluster;
        const long long ctas = units * d.cluster, last = ctas % cap ? ctas % cap : cap;
        const long long idle = last < kSaturatingCtas ? unit_bytes / d.cluster * (kSaturatingCtas - last) : 0;
        if (tiles > d.cluster * units && (idle > kRangesBytes || (ragged && units * unit_bytes > kRangesBytes))) {
            d.shares = 0;
            d.cluster = 1;
            d.slot_mode = d.slots == n_all ? kDecodeSlotTile : kDecodeSlotTwo;
        }
    }
    // the counters behind the slots, in units of a slot of every (batch, query head)
    const long long slot_bytes = (long long)B * Hq * (D + 2) * 4;
    d.splits = d.slots + (int)((8 * counters + slot_bytes - 1) / slot_bytes);
    if (d.shares == 0) {
        d.n_ctas = (int)std::min<long long>(tiles, cap);
        return d;
    }
    d.n_ctas = (int)std::min<long long>(units * d.shares, 1ll << 30);
    if (d.shares == 1 && units > cap && !ragged) {  // the ring of a CTA then runs on from unit to unit
        d.shares = 0;
        d.whole = true;
        d.n_ctas = cap;
    }
    return d;
}

}  // namespace b200attn
