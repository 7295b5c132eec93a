"""What flex_attention keeps of a score_mod: as long as the callable lives, and no longer."""

import gc

import torch

from chia_proj_b200 import flex

H = 4


def make(i):
    if i % 2:
        return lambda sc, b, h, qi, kj: sc * (0.5 + i + 0 * h)
    return lambda sc, b, h, qi, kj: sc + (1.0 + i) * (kj - qi)


def test_a_callable_at_another_ones_address():
    seen, again = set(), 0
    for i in range(200):
        f = make(i)
        again += id(f) in seen
        seen.add(id(f))
        sm = flex._score_of(f, H, "cpu")
        want = (("temp", 0.5 + i) if i % 2 else ("alibi", 1.0 + i))
        assert sm.mod == want[0] and torch.allclose(sm.head_param, torch.full((H,), want[1]))
        assert flex._score_of(f, H, "cpu") is sm  # kept while it lives
        del f, sm
    assert again > 0  # addresses did come again
    gc.collect()
    assert len(flex._score_cache) == 0


class Unhashable:
    __hash__ = None
    __slots__ = ()

    def __call__(self, sc, b, h, qi, kj):
        return sc * 3.0


def test_callables_that_cannot_be_kept():
    f = Unhashable()
    assert flex._score_of(f, H, "cpu").mod == "temp" and flex._score_of(None, H, "cpu").mod == "none"
