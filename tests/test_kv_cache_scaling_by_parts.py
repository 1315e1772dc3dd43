"""A cache whose frequencies are scaled by parts between other numbers of turns than the usual ones."""
import pytest
import torch

import modern_llm_v1_b200 as m


def test_the_tables_are_made_with_the_turns_given(monkeypatch):
    from modern_llm_v1_b200 import kv_cache

    asked = []

    def tables(T, R, base, scaling, factor, trained, turns_fast, turns_slow, device):
        asked.append((T, R, base, scaling, factor, trained, turns_fast, turns_slow))
        return torch.zeros(T, R // 2), torch.zeros(T, R // 2)

    monkeypatch.setattr(kv_cache, "make_rotary_cache", tables)
    kw = dict(scaling="parts", factor=8.0, trained=16.0, device="cpu")
    prompts = m.KVCache(1, 2, 4, 2, 64, 8, turns_fast=4.0, turns_slow=1.5, **kw)
    m.KVCache(1, 4, 4, 2, 64, 8, prefix=prompts, device="cpu")
    m.KVCache(1, 2, 4, 2, 64, 8, **kw)
    assert asked == [(8, 64, 10000.0, "parts", 8.0, 16.0, 4.0, 1.5), (16, 64, 10000.0, "parts", 8.0, 16.0, 4.0, 1.5), (8, 64, 10000.0, "parts", 8.0, 16.0, 32.0, 1.0)]
    for kw in (dict(turns_fast=8.0), dict(turns_slow=1.0)):
        with pytest.raises(ValueError, match="as theirs does"):
            m.KVCache(1, 4, 4, 2, 64, 8, prefix=prompts, device="cpu", **kw)
    m.KVCache(1, 4, 4, 2, 64, 8, prefix=prompts, device="cpu", turns_fast=4.0, turns_slow=1.5)


@pytest.mark.gpu
def test_the_cache_has_the_values_of_the_tables():
    cache = m.KVCache(1, 2, 4, 2, 64, 100, scaling="parts", factor=8.0, trained=16.0, turns_fast=4.0, turns_slow=1.0)
    cos, sin = m.make_rotary_cache(100, 64, 10000.0, "parts", 8.0, 16.0, 4.0, 1.0)
    other, _ = m.make_rotary_cache(100, 64, 10000.0, "parts", 8.0, 16.0)
    assert torch.equal(cache.cos, cos) and torch.equal(cache.sin, sin) and not torch.equal(cos, other)
