"""The plans that the long-context calls are launched by, run on the host over shapes of every kind: each unit of work has one owner, each
result a place of its own inside the workspace that the library asks for, units in turn are handed out once and the count of them ends
where it began."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "modern-llm-v1_b200", "csrc")

DRIVER = r"""
#include <cstdio>
#include <random>
#include <set>
#include <vector>
#include "context_plan.h"
static int g_sms = 148;
int b200attn::sm_count() { return g_sms; }
using namespace b200attn;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)
struct Rng {
    std::mt19937 r;
    int operator()(int lo, int hi) { return lo + int(r() % unsigned(hi - lo + 1)); }
    int log(int lo, int hi) {  // spread over the logarithm
        const double x = std::uniform_real_distribution<double>(0, 1)(r);
        return std::min(hi, std::max(lo, int(lo * std::pow(double(hi) / lo, x) + 0.5)));
    }
};

static int key_weights(Rng& rng) {
    KeyWeightsParams p = {};
    const int B = rng(1, 3), Hkv = rng(1, 3), group = rng(1, 24), T = rng(0, 1) ? rng(1, 130) : rng.log(1, 3000), pos0 = rng(0, 2) ? rng.log(1, 4000) : 0;
    key_weights_plan(p, B, T, pos0, group * Hkv, Hkv);
    CHECK(p.heads >= 1 && p.tokens * p.heads <= 128 && p.heads * p.n_hc == group && p.n_qt * p.tokens >= T && p.n_kt * 128 >= p.L && p.L == pos0 + T);
    const long long total = key_weights_total(p, B);
    CHECK(total == (long long)B * Hkv * key_weights_before(p, p.n_kt) && total < (1ll << 31));
    g_sms = rng(1, 160);
    key_weights_deal(p, int(total));
    // a tile of keys is seen by the last tiles of tokens, from the last one down
    for (int kt = 0; kt < p.n_kt; ++kt) {
        const int units = key_weights_before(p, kt + 1) - key_weights_before(p, kt);
        CHECK(units > 0 && units % p.n_hc == 0);
        for (int qt = 0; qt < p.n_qt; ++qt) {
            const int last = std::min((qt + 1) * p.tokens, T) - 1;
            CHECK((kt * 128 <= pos0 + last) == (qt >= p.n_qt - units / p.n_hc));
        }
    }
    const size_t slots = key_weights_bytes(B, T, pos0, Hkv) / (kKeyWeightsGroups * 128 * sizeof(float));
    std::vector<char> taken(total);
    std::set<size_t> used;
    for (int c = 0; c < p.n_ctas; ++c) {
        const int u0 = key_weights_range(p, c), u1 = key_weights_range(p, c + 1);
        CHECK(u1 > u0 && u1 - u0 <= total / p.n_ctas + 1);
        KeyWeightsItem it = key_weights_item(p, u0);
        for (int u = u0; u < u1;) {
            CHECK(it.start <= u && u < it.start + it.units && it.bh < B * Hkv && it.kt < p.n_kt);
            const size_t slot = size_t(it.bh) * p.n_kt + it.kt + c;  // of the sums that the CTA leaves
            CHECK(slot < slots && used.insert(slot).second);
            for (const int end = std::min(u1, it.start + it.units); u < end; ++u) {
                CHECK(key_weights_cta(p, u) == c && !taken[u]);
                taken[u] = 1;
            }
            key_weights_next(p, it);
        }
    }
    for (char t : taken) CHECK(t);
    return 0;
}

static int in_turn_seen = 0, ranges_seen = 0, clusters_seen = 0;
static int shared(Rng& rng) {
    static const int heads[][2] = {{6, 2}, {16, 4}, {8, 8}, {12, 4}, {8, 1}, {4, 2}, {24, 1}, {34, 2}, {130, 1}, {300, 2}, {5, 1}};
    g_sms = rng(0, 3) ? 148 : rng(1, 160);
    const int h = rng(0, 10), Hq = heads[h][0], Hkv = heads[h][1], D = rng(0, 1) ? 64 : 128, group = Hq / Hkv;
    const int G = rng.log(1, 40), n = rng.log(1, 300), B = G * n, P = rng.log(1, 20000), L = rng.log(1, 4000);
    CHECK(shared_sizes_ok(B, G, P, L, Hq, Hkv, D));
    const size_t bytes = std::max(prefix_plan(B, G, P, L, Hq, Hkv, D, false).bytes, prefix_plan(B, G, P, L, Hq, Hkv, D, true).bytes);
    for (bool ragged : {false, true}) {
        const PrefixPlan x = prefix_plan(B, G, P, L, Hq, Hkv, D, ragged);
        const int all = (P + kPrefixKeys - 1) / kPrefixKeys;
        CHECK(x.heads * x.seqs <= 128 && x.heads * x.n_chunks == group && x.tiles * x.seqs >= n && (x.tiles - 1) * x.seqs < n);
        CHECK(x.units == (long long)G * Hkv * x.n_chunks * x.tiles && x.splits >= 1 && x.splits <= all && x.grid == x.units * x.splits);
        CHECK(x.slots == size_t(x.grid) && x.bytes <= bytes && x.decode_bytes % 256 == 0);
        // every split of every length begins where the one before ends
        const FastDiv div = fastdiv_make((unsigned)x.splits);
        for (int tiles : {0, 1, all / 2, all - 1, all}) {
            CHECK(fastdiv(0, div) == 0u);
            for (int s = 0; s <= x.splits; ++s) CHECK(fastdiv(unsigned(tiles * s), div) == unsigned((long long)tiles * s / x.splits));
        }
        // the rows of the prompts' partial results: no two (sequence, head) share one, all in their slots
        DecodePrefix e = {};
        e.splits = x.splits, e.tiles = x.tiles, e.n_chunks = x.n_chunks, e.Hkv = Hkv;
        e.div_n = fastdiv_make((unsigned)n), e.div_heads = fastdiv_make((unsigned)x.heads), e.div_seqs = fastdiv_make((unsigned)x.seqs);
        if (!ragged) {
            std::vector<char> used(x.units * 128);
            for (int b = 0; b < B; ++b)
                for (int hk = 0; hk < Hkv; ++hk)
                    for (int j = 0; j < group; ++j) {
                        int row;
                        const size_t slot = decode_prefix_row(e, b, hk, j, &row);
                        CHECK(row >= 0 && row < x.heads * x.seqs && slot % x.splits == 0 && slot + x.splits <= x.slots);
                        char& u = used[slot / x.splits * 128 + row];
                        CHECK(!u);
                        u = 1;
                        // and the row that the prompts' kernel gives it
                        const long long unit = slot / x.splits, uc = unit / x.tiles, uh = uc / x.n_chunks;
                        CHECK(uh / Hkv == b / n && uh % Hkv == hk && uc % x.n_chunks == j / x.heads);
                        CHECK(row == (b % n - int(unit % x.tiles) * x.seqs) * x.heads + j % x.heads);
                    }
        }
        // the workspace: the decode's partial results and counters, the prompts' results, the finished units' own
        const DecodePlan& d = x.decode;
        const long long units = (long long)B * Hkv * d.n_chunks;
        const int n_all = (L + decode_tile_keys(D) - 1) / decode_tile_keys(D);
        const size_t rows = (size_t)B * Hq * d.slots;
        CHECK(d.G <= 16 && d.G * d.n_chunks == group);
        size_t counters = 0;
        if (d.in_turn) counters = 1;
        else if (d.shares == 0 && !d.whole && n_all > 1) counters = d.n_ctas;
        CHECK(rows * (D + 2) * 4 + 8 * counters <= x.decode_bytes);
        const size_t own = d.shares == 0 ? (size_t)B * Hq * (D + 2) * 4 : 0;
        CHECK(x.decode_bytes + x.slots * 128 * (D + 2) * 4 + own <= bytes);
        if (d.shares == 0 && !d.in_turn && !d.whole && n_all > 1) {
            if (d.slot_mode == kDecodeSlotTile) {
                CHECK(d.slots == n_all);
            } else {
                CHECK(d.slot_mode == kDecodeSlotTwo && units * d.slots >= 2ll * d.n_ctas);
            }
        }
        if (d.shares > 0) {
            CHECK(d.shares == d.cluster && d.n_ctas == units * d.cluster && d.cluster <= kDecodeMaxCluster);
            ++clusters_seen;
        } else if (!d.in_turn) {
            ++ranges_seen;
        }
        CHECK(d.n_ctas >= 1 && (d.shares > 0 || d.n_ctas <= kDecodeMaxCtas));
        if (!d.in_turn) continue;
        // units in turn: every CTA begins with the unit of its number or asks, and then asks until it is told that there are no more
        ++in_turn_seen;
        DecodeParams p = {};
        p.turn = d.turn, p.units = int(units);
        std::vector<char> taken(units);
        std::vector<int> alive(d.n_ctas), asked(d.n_ctas);
        for (int c = 0; c < d.n_ctas; ++c) {
            alive[c] = c;
            if (c >= p.turn) continue;
            CHECK(c < p.units);
            taken[c] = 1;
        }
        int asks = 0;
        bool last = false;
        while (!alive.empty()) {
            const int i = rng(0, int(alive.size()) - 1), nr = asks++;
            CHECK(!last);
            last = decode_last_ask(p, nr, d.n_ctas);
            const int unit = decode_asked_unit(p, nr);
            if (unit < 0) {
                alive[i] = alive.back(), alive.pop_back();
                continue;
            }
            CHECK(unit < p.units && !taken[unit]);
            taken[unit] = 1;
        }
        CHECK(last && asks < (1 << kDecodeTurnBits));
        for (char t : taken) CHECK(t);
    }
    return 0;
}

// chunks whose units are counted up to the last of 31 bits: the numbers on the way to a count are larger
static int longest(Rng& rng) {
    g_sms = 148;
    int most = 0;
    for (int i = 0; i < 200; ++i) {
        KeyWeightsParams p = {};
        const int pos0 = rng(0, 1) ? 0 : rng.log(1, 60000000), T = i < 4 ? 8388480 - i * 1000000 : rng.log(100000, 8388480), group = rng(0, 3) ? 1 : rng(1, 8);
        key_weights_plan(p, 1, T, pos0, group, 1);
        const long long total = key_weights_total(p, 1);
        if (total >= (1ll << 31)) continue;
        key_weights_deal(p, int(total));
        auto before = [&](int kt) {
            const long long m = std::max(0, kt - p.full_kt);
            return ((long long)kt * p.n_qt - m * (m - 1) / 2) * p.n_hc;
        };
        for (int e = 0; e < 2000; ++e) {
            const int kt = e < 8 ? p.n_kt - e : rng(0, p.n_kt);
            CHECK(kt < 0 || key_weights_before(p, kt) == before(kt));
        }
        for (int c : {0, 1, p.n_ctas / 2, p.n_ctas - 2, p.n_ctas - 1})
            for (int u : {key_weights_range(p, c), key_weights_range(p, c + 1) - 1}) {
                const KeyWeightsItem it = key_weights_item(p, u);
                CHECK(it.bh == 0 && it.kt >= 0 && it.kt < p.n_kt && it.start == before(it.kt) && it.units == before(it.kt + 1) - before(it.kt));
                CHECK(it.start <= u && u < it.start + it.units && key_weights_cta(p, u) == c);
            }
        most = std::max(most, p.total);
    }
    CHECK(most > (1 << 30));
    return 0;
}

int main(int argc, char**) {
    Rng rng{std::mt19937(3)};
    if (argc > 1) return longest(rng);
    for (int i = 0; i < 1000; ++i)
        if (key_weights(rng)) return 1;
    for (int i = 0; i < 1000; ++i)
        if (shared(rng)) return 1;
    std::printf("%d %d %d\n", in_turn_seen, ranges_seen, clusters_seen);
}
"""


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("context_plan")
    (d / "driver.cu").write_text(DRIVER)
    subprocess.check_call([os.environ.get("NVCC", "nvcc"), "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-o",
                           str(d / "driver"), str(d / "driver.cu")])
    return str(d / "driver")


def test_the_plans_that_ship(driver):
    out = subprocess.run([driver], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stdout
    assert all(int(n) > 100 for n in out.stdout.split()), out.stdout  # deals of every kind were among them


def test_the_longest_chunks(driver):
    out = subprocess.run([driver, "longest"], capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stdout
