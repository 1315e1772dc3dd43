// How a decode launch deals its units' tiles (attn_decode.cuh).
#pragma once

#include <algorithm>
#include <math.h>

#include "attn_decode.cuh"
#include "host_common.h"
#include "tmap.h"

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
    bool in_turn; // kDecodeSharedTurn
    int turn;     // and DecodeParams::turn
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
constexpr long long kTurnBytes = 3ll << 18;

// Rounds of loads in which the CTAs of a unit's cluster join it with the prompt's results (decode_add_prefix): about 0.7 us each, so a
// cluster that saves two of them is worth its own 1 us (1 prompt x 12 samples, P=3220 L=3 8/1 D=128, 26 splits: 18.6 -> 11.3 us).
inline int decode_join_rounds(int G, int D, int cluster, int prompt_splits) { return (G * (D / 2) / cluster + 127) / 128 * ((prompt_splits + 7) / 8); }

// cap: CTAs that may run at once, or 0: as many as fit the device.
//
// Behind shared prompts (`shared`, cap: CTAs on the SMs that the prompts' kernel leaves) the CTAs wait for the prompts' kernel at their ends.
// More units than those CTAs, of at most kTurnBytes: each takes a whole unit, then the next that nobody has taken, and so do the CTAs that
// start on the SMs which the prompts' kernel frees.  Longer units are dealt in ranges among cap CTAs, which come out more even.  (us, units of
// different lengths up to L, ranges / in turn, as both were at first; G prompts x n samples, P, L, heads, D: 8 x 16 2000 300 16/4 64 25.7 / 21.7;
// 16 x 16 500 300 8/4 64 45.0 / 28.3; 2 x 128 3000 250 32/8 128 97.0 / 61.1; 16 x 4 4000 256 16/8 64 75.1 / 41.6; 8 x 8 1000 100 16/16 64 114.7 / 31.3;
// units of 512 KB 4 x 40 1000 2000 16/4 64 54.1 / 50.5; of 1 MB 2 x 20 2000 2000 32/8 128 57.9 / 58.7, 1 x 300 1000 4000 8/1 64 52.9 / 57.2; equal
// lengths, whole units dealt beforehand / in turn: 4 x 64 8192 256 16/4 128 57.3 / 51.6.)
inline DecodePlan decode_plan(int B, int L, int Hq, int Hkv, int D, int n_splits, bool ragged, int cap = 0, bool shared = false, int prompt_splits = 0) {
    DecodePlan d;
    const int group = Hq / Hkv;
    if (cap <= 0) cap = decode_max_ctas();
    d.G = decode_heads_per_cta(group);
    d.n_chunks = group / d.G;
    const long long units = (long long)B * Hkv * d.n_chunks;
    const int keys = decode_tile_keys(D), n_all = (L + keys - 1) / keys, n_128 = (L + 127) / 128;
    const long long unit_bytes = 4ll * L * D, tiles = units * n_all;
    d.shares = d.cluster = 1;
    d.whole = false;
    d.slot_mode = kDecodeSlotTile;
    d.in_turn = shared && units > cap && units < kDecodeTurnUnits && unit_bytes <= kTurnBytes;
    d.turn = 0;
    long long counters = 0;
    if (d.in_turn) {
        d.shares = 0;
        d.slots = 0, d.splits = 1;  // no partial results: room for the counter
        d.turn = cap;
        d.n_ctas = (int)std::min<long long>(units, decode_max_ctas());
        return d;
    }
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
        while (d.cluster < kDecodeMaxCluster && units * d.cluster * 2 <= (shared ? cap / 2 : sm_count()) &&
               (n_all > 2 * d.cluster || decode_join_rounds(d.G, D, d.cluster, prompt_splits) > decode_join_rounds(d.G, D, d.cluster * 2, prompt_splits) + 1))
            d.cluster *= 2;
        d.shares = d.cluster;
        const long long ctas = units * d.cluster, last = ctas % cap ? ctas % cap : cap;
        const long long idle = last < kSaturatingCtas ? unit_bytes / d.cluster * (kSaturatingCtas - last) : 0;
        if ((tiles > d.cluster * units && (idle > kRangesBytes || (ragged && units * unit_bytes > kRangesBytes))) || (shared && ragged && units > cap)) {
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

// A launch's parameters and tensor maps from checked arguments
inline int decode_fill(const DecodePlan& d, DecodeParams& p, CUtensorMap& tk, CUtensorMap& tv, const void* q, const void* kcache,
                       const void* vcache, void* o, float* lse, const int* lens, int B, int L, int L_cap, int Hq, int Hkv, int D,
                       float softmax_scale, void* workspace, int* status) {
    // the maps end at row L of every (batch, head): rows of the cache beyond it are never read (TMA fills zeros)
    const Strides sk = strides_for(B200ATTN_LAYOUT_BHTD, Hkv, L_cap, D);
    if (!make_tmap_bf16_4d(&tk, kcache, D, L, Hkv, B, sk.t, sk.h, sk.b, decode_tile_keys(D)) ||
        !make_tmap_bf16_4d(&tv, vcache, D, L, Hkv, B, sk.t, sk.h, sk.b, decode_tile_keys(D)))
        return B200ATTN_ERR_TENSOR_MAP;
    p = {};
    p.B = B;
    p.L = L;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.group = Hq / Hkv;
    p.G = d.G;
    p.n_chunks = d.n_chunks;
    p.units_per_seq = Hkv * d.n_chunks;
    p.div_units = fastdiv_make((unsigned)p.units_per_seq);
    p.div_chunks = fastdiv_make((unsigned)d.n_chunks);
    p.div_shares = fastdiv_make((unsigned)std::max(d.shares, 1));
    p.div_tiles = fastdiv_make((unsigned)((L + decode_tile_keys(D) - 1) / decode_tile_keys(D)));
    p.div_slice = fastdiv_make((unsigned)(d.G * (D / 2) / d.cluster));
    p.shares = d.shares;
    p.cluster = d.cluster;
    p.whole = d.whole;
    p.slot_mode = d.slot_mode;
    p.turn = d.turn;
    p.units = B * p.units_per_seq;
    p.scale = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
    p.scale_log2 = p.scale * 1.4426950408889634f;
    p.lens = lens;
    p.q = static_cast<const uint16_t*>(q);
    p.o = static_cast<uint16_t*>(o);
    p.lse = lse;
    const size_t rows = (size_t)B * Hq * d.slots;  // slots x heads per slot
    p.part_o = static_cast<float*>(workspace);
    p.part_m = p.part_o + rows * D;
    p.part_l = p.part_m + rows;
    p.counters = reinterpret_cast<unsigned long long*>(p.part_l + rows);  // (D + 2 is even: 8-byte aligned)
    p.tag = next_decode_tag();
    p.status = status;
    return B200ATTN_OK;
}

template <int D, int NH, int PF, int MODE>
int launch_decode_pf(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p, int n_ctas, cudaStream_t st) {
    using Cfg = DecodeCfg<D>;
    static bool set[kMaxDevices] = {false};
    int rc = set_smem_once(attn_decode_kernel<D, NH, PF, MODE>, Cfg::kSmemBytes, set);
    if (rc) return rc;
    if (launch_cluster(attn_decode_kernel<D, NH, PF, MODE>, dim3(n_ctas), kDecodeThreads, Cfg::kSmemBytes, st, p.cluster, tk, tv, p) != cudaSuccess) {
        cudaGetLastError();
        return B200ATTN_ERR_CUDA;
    }
    return B200ATTN_OK;
}

// Where the CTAs fill most of the device the launch is bound by HBM, and the first two tiles of each come into L2 while the kernel
// in front ends, provided that it lets this one start early, as the append of one token and the decode itself do (us per call over
// caches larger than L2 in turn, without / with: append + decode B=48 L<=6000 16/4 D=64 35.6 / 34.3, B=64 L<=4096 33.5 / 31.8, B=20 L<=1500
// D=128 19.3 / 18.0; decode behind decode B=64 L=4096 16/4 D=64 41.9 / 41.3, B=300 L=200 8/8 24.0 / 22.8, B=64 L=1000 6/2 9.0 / 8.5, B=8
// L=2000 8/8 D=128, 128 CTAs, 14.3 / 14.1).  With a matrix product in front of each append + decode, the product included: 40.6 / 39.9,
// 38.3 / 37.5, 23.4 / 23.0.  Behind a kernel that does not release this one early the tiles are asked for twice: product and decode
// 46.1 / 46.0, 29.8 / 29.5, 13.3 / 13.4, 19.1 / 19.3; a first pass on new buffers on an idle device gains nothing (host's time of a call,
// B=300 41.8 / 42.1, append + decode B=48 67.3 / 67.0).  With three tiles the gain is smaller, with six it is gone.
// Fewer CTAs are bound by latency, of which this hides nothing: B=6 L<=3000 8/1 D=128 8.5 -> 8.6, B=1 L=1500 16/4 5.26 -> 5.30.
constexpr int kPrefetchCtas = 128;
// (Behind a shared prompt's kernel the loads themselves begin that early.)
template <int MODE, int D, int NH>
int launch_decode_heads(const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p, int n_ctas, cudaStream_t st) {
    constexpr bool behind_prompts = MODE == kDecodeShared || MODE == kDecodeSharedTurn;
    if (!behind_prompts && n_ctas >= kPrefetchCtas) return launch_decode_pf<D, NH, behind_prompts ? 0 : 2, MODE>(tk, tv, p, n_ctas, st);
    return launch_decode_pf<D, NH, 0, MODE>(tk, tv, p, n_ctas, st);
}
template <int MODE>
int launch_decode(int D, const CUtensorMap& tk, const CUtensorMap& tv, const DecodeParams& p, int n_ctas, cudaStream_t st) {
    if (D == 64) return p.G <= 8 ? launch_decode_heads<MODE, 64, 1>(tk, tv, p, n_ctas, st) : launch_decode_heads<MODE, 64, 2>(tk, tv, p, n_ctas, st);
    return p.G <= 8 ? launch_decode_heads<MODE, 128, 1>(tk, tv, p, n_ctas, st) : launch_decode_heads<MODE, 128, 2>(tk, tv, p, n_ctas, st);
}

}  // namespace b200attn
