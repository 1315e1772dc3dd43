"""A cache that continues shared prompts takes the prompts' rotation and norm, or refuses; without a GPU."""
import pytest

import modern_llm_v1_b200 as m


def new(L_cap=8, **kw):
    return m.KVCache(1, 2, 4, 2, 64, L_cap, device="cpu", **kw)


def test_the_norm_is_that_of_the_prompts():
    assert new(prefix=new(eps=1e-6)).eps == 1e-6
    assert new(prefix=new(eps=1e-6), eps=1e-6).eps == 1e-6
    assert new(prefix=new()).eps == new().eps == 1e-5
    with pytest.raises(ValueError, match="as theirs does"):
        new(prefix=new(eps=1e-6), eps=1e-5)


def test_a_rotation_of_its_own_is_refused():
    prompts = new(rope_base=5000.0)
    for kw in (dict(rope_base=10000.0), dict(factor=4.0), dict(trained=128.0)):
        with pytest.raises(ValueError, match="as theirs does"):
            new(prefix=prompts, **kw)
    for kw in ({}, dict(rope_base=5000.0)):
        own = new(prefix=prompts, **kw)
        assert own.cos.shape == (16, 32) and (own.cos[:8] == prompts.cos).all() and (own.sin[:8] == prompts.sin).all()
    assert (new().cos == new(rope_base=10000.0).cos).all()


@pytest.mark.parametrize("how", ["refilled", "same lengths again", "longer and back"])
def test_prompts_that_have_changed_are_noticed(how):
    """also where they have the same length as before"""
    prompts = new()
    prompts.advance(5)
    samples = new(prefix=prompts)
    assert samples.next_position == 5
    samples.advance()
    assert samples.next_position == 6
    if how == "refilled":
        prompts.reset()
        prompts.advance(5)
    elif how == "same lengths again":
        prompts.set_lengths([5, 5])
    else:
        prompts.advance(1)
        prompts.reset()
        prompts.advance(5)
    with pytest.raises(ValueError, match="prompts have changed"):
        samples.next_position
    samples.reset()
    at = samples.next_position
    assert at == 5 if how != "same lengths again" else at.tolist() == [5, 5]


def test_positions_that_were_asked_for_stay_what_they_were():
    """also after the next token: the cache counts on in a tensor of its own"""
    prompts = new()
    prompts.advance(5)
    prompts.set_lengths([5, 3])
    samples = new(prefix=prompts)
    at = samples.next_position
    samples.advance()
    assert at.tolist() == [5, 3]
    at.zero_()
    assert samples.next_position.tolist() == [6, 4]
