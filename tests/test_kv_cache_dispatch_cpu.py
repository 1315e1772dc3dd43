"""Which native calls a cache makes: one with the reference's rotation and nothing else goes straight to its two, without a GPU."""
import copy

import pytest
import torch

import modern_llm_v1_b200 as m
from modern_llm_v1_b200 import _lib


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, len(a)))


@pytest.mark.parametrize("copied", [False, True])
def test_the_calls_of_each_kind_of_cache(monkeypatch, copied):
    new = lambda **kw: m.KVCache(1, 2, 4, 2, 64, 8, device="cpu", **kw)  # noqa: E731
    prompts = new()
    prompts.advance(3)
    caches = [(new(), ["kv_append", "kv_attend"]), (new(T_max=32), ["append_rotary", "kv_attend"]), (new(track_weights=True), ["append_rotary", "decode_weights"]),
              (new(prefix=prompts), ["append_rotary", "decode_shared"])]
    host = Recorder()
    monkeypatch.setattr(_lib, "_host", host)
    x, q = torch.zeros(2, 1, 2, 64), torch.zeros(2, 4, 1, 64)
    for cache, names in caches:
        if copied:
            cache = copy.deepcopy(cache)
        host.calls.clear()
        cache.append(0, x, x, x, None, None, q)
        cache.attend(0, q, q, None)
        cache.attend(0, q, q, None, softmax_scale=0.5)
        assert [n for n, _ in host.calls] == names + names[1:]
    host.calls.clear()
    caches[2][0].attend(0, q, q, q, n_new=2, new_lens=torch.ones(2, dtype=torch.int32))
    assert [n for n, _ in host.calls] == ["kv_attend", "key_weights"]


def test_the_flags_are_the_instances_alone():
    for name in ("_plain", "_alone", "_pos", "_changes", "prefix", "track_weights"):
        assert name not in vars(m.KVCache) and hasattr(m.KVCache.__new__(m.KVCache), name)
