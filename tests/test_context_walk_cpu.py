"""How the long-context kernels deal out their work, run on the host: every unit once, every piece in a slot of its own, loads in the
order in which the products read them."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "modern-llm-v1_b200", "csrc")

DRIVER = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>
#include "attn_prefix.cuh"
#include "key_weights.cuh"
using namespace b200attn;
#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

static int key_weights(std::mt19937& rng) {
    auto upto = [&](int lo, int hi) { return lo + int(rng() % unsigned(hi - lo + 1)); };
    KeyWeightsParams p = {};
    const int B = upto(1, 3), T = upto(1, 3) == 1 ? upto(1, 130) : upto(1, 1500), pos0 = upto(0, 2) ? upto(0, 2000) : 0;
    p.Hkv = upto(1, 3), p.group = upto(1, 6), p.T = T, p.pos0 = pos0, p.L = pos0 + T;
    p.tokens = T < 128 ? T : 128;
    p.heads = 1;
    while (p.heads * 2 * p.tokens <= 128 && p.group % (p.heads * 2) == 0) p.heads *= 2;
    p.n_qt = (T + p.tokens - 1) / p.tokens, p.n_hc = p.group / p.heads, p.n_kt = (p.L + 127) / 128;
    p.full_kt = p.n_qt == 1 ? p.n_kt : (pos0 + 127) / 128;
    p.total = B * p.Hkv * key_weights_before(p, p.n_kt);
    // the units of a key tile are the tiles of tokens that see any of its keys
    for (int kt = 0; kt < p.n_kt; ++kt) {
        int seen = 0;
        for (int qt = 0; qt < p.n_qt; ++qt) {
            const int last = (qt + 1) * p.tokens < T ? (qt + 1) * p.tokens - 1 : T - 1;
            const bool sees = kt * 128 <= pos0 + last;
            seen += sees;
            // taken from the last tile down
            const int units = int(key_weights_before(p, kt + 1) - key_weights_before(p, kt)) / p.n_hc;
            CHECK(sees == (qt >= p.n_qt - units));
        }
        CHECK(seen * p.n_hc == key_weights_before(p, kt + 1) - key_weights_before(p, kt));
    }
    const int n = p.n_ctas = std::min(upto(1, 148), p.total);
    p.per_cta = p.total / n, p.more = p.total % n;
    std::vector<int> taken(p.total);
    std::set<long long> slots;
    for (int c = 0; c < n; ++c) {
        const int u0 = key_weights_range(p, c), u1 = key_weights_range(p, c + 1);
        CHECK(u1 > u0 && u1 - u0 <= p.total / n + 1);
        KeyWeightsItem it = key_weights_item(p, u0);
        for (int u = u0; u < u1;) {
            CHECK(it.start <= u && u < it.start + it.units && it.bh < B * p.Hkv && it.kt < p.n_kt);
            const int end = std::min(u1, it.start + it.units);
            const long long slot = (long long)it.bh * p.n_kt + it.kt + c;
            CHECK(slot < (long long)B * p.Hkv * p.n_kt + n && slots.insert(slot).second);
            for (; u < end; ++u) {
                CHECK(key_weights_cta(p, u) == c);
                ++taken[u];
            }
            key_weights_next(p, it);
        }
    }
    for (int t : taken) CHECK(t == 1);
    return 0;
}

static int prefix() {
    for (int n = 1; n < 40; ++n) {
        int i = 0;  // the products: S of the first two tiles, then P V of tile j and S of tile j + 2
        auto next = [&](bool k, int j) {
            int lj;
            const bool lk = prefix_load_at(i, n, &lj);
            return lk == k && lj == j && i++ == (k ? prefix_k_at(j) : prefix_v_at(j, n));
        };
        for (int j = 0; j < 2 && j < n; ++j) CHECK(next(true, j));
        for (int j = 0; j < n; ++j) {
            CHECK(next(false, j));
            if (j + 2 < n) CHECK(next(true, j + 2));
        }
        CHECK(i == 2 * n);
    }
    return 0;
}

int main() {
    std::mt19937 rng(1);
    for (int i = 0; i < 400; ++i)
        if (key_weights(rng)) return 1;
    return prefix();
}
"""


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    d = tmp_path_factory.mktemp("context_walk")
    (d / "driver.cu").write_text(DRIVER)
    subprocess.check_call([os.environ.get("NVCC", "nvcc"), "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, "-o",
                           str(d / "driver"), str(d / "driver.cu")])
    return str(d / "driver")


def test_the_deal(driver):
    out = subprocess.run([driver], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
