"""What flex_attention keeps of a score_mod: as long as the callable lives, and no longer."""

import gc

import pytest
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


# ---- what a callable depends on may change while it lives
T2 = torch.tensor([1.0, 2.0, 3.0, 4.0])
CAP = 20.0


def kinds(f, h=H):
    sm = flex._score_of(f, h, "cpu")
    return sm.mod, sm.softcap if sm.mod == "softcap" else None if sm.head_param is None else sm.head_param.tolist()


def softcap(sc, cap):
    return cap * torch.tanh(sc / cap)


def test_a_captured_tensor_changes_in_place():
    t = torch.tensor([1.0, 2.0, 3.0, 4.0])
    f = lambda sc, b, h, qi, kj: sc * t[h]
    assert kinds(f) == ("temp", [1, 2, 3, 4])
    t.mul_(2)
    assert kinds(f) == ("temp", [2, 4, 6, 8])
    t.data.add_(1)  # (no version tells of this)
    assert kinds(f) == ("temp", [3, 5, 7, 9])
    t.fill_(1)
    assert kinds(f) == ("none", None)
    t.numpy()[:] = 5
    assert kinds(f) == ("temp", [5, 5, 5, 5])
    slopes = torch.nn.Parameter(torch.zeros(H))
    g = lambda sc, b, h, qi, kj: sc + slopes[h] * (kj - qi)
    assert kinds(g)[0] == "none"
    with torch.no_grad():
        slopes.copy_(torch.arange(1.0, H + 1))
    assert kinds(g) == ("alibi", [1, 2, 3, 4])


def test_other_names_change():
    global CAP
    cap = 30.0
    f = lambda sc, b, h, qi, kj: softcap(sc, cap)
    assert kinds(f)[0] == "softcap" and abs(kinds(f)[1] - 30) < 1e-3
    cap = 10.0
    assert abs(kinds(f)[1] - 10) < 1e-3
    g = lambda sc, b, h, qi, kj: softcap(sc, CAP)  # a global, of another function's too
    nested = lambda sc, b, h, qi, kj: g(sc, b, h, qi, kj)
    assert abs(kinds(nested)[1] - 20) < 1e-3
    CAP = 5.0
    assert abs(kinds(g)[1] - 5) < 1e-3 and abs(kinds(nested)[1] - 5) < 1e-3
    CAP = 20.0
    table = {"t": 2.0, "l": [3.0]}
    t = lambda sc, b, h, qi, kj: sc * (table["t"] * table["l"][0] + 0 * h)
    assert kinds(t)[1][0] == 6
    table["l"][0] = 4.0
    assert kinds(t)[1][0] == 8

    def d(sc, b, h, qi, kj, by=2.0):
        return sc * by
    assert kinds(d)[1][0] == 2
    d.__defaults__ = (7.0,)
    assert kinds(d)[1][0] == 7
    from functools import partial
    p = partial(lambda w, sc, b, h, qi, kj: sc * w["x"], table)
    table["x"] = 2.0
    assert kinds(p)[1][0] == 2
    table["x"] = 9.0
    assert kinds(p)[1][0] == 9


class Cap:
    scale = 1.0

    def __init__(self, cap):
        self.cap = cap

    def __call__(self, sc, b, h, qi, kj):
        return softcap(sc, self.cap * self.scale)

    def other(self, sc, b, h, qi, kj):
        return sc * (self.cap * self.scale)


class Layer(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.t = torch.nn.Parameter(torch.full((H,), 2.0))

    def score(self, sc, b, h, qi, kj):
        return sc * self.t[h]


def test_attributes_and_bound_methods():
    f = Cap(30.0)
    assert abs(kinds(f)[1] - 30) < 1e-3
    f.cap = 10.0
    assert abs(kinds(f)[1] - 10) < 1e-3
    assert kinds(f.other)[1][0] == 10 and abs(kinds(f)[1] - 10) < 1e-3  # two of one object
    Cap.scale = 2.0
    try:
        assert abs(kinds(f)[1] - 20) < 1e-3 and kinds(f.other)[1][0] == 20
    finally:
        Cap.scale = 1.0
    # a bound method is another object each time; what was found stays with its own object
    assert flex._score_of(f.other, H, "cpu") is flex._score_of(f.other, H, "cpu")
    m = Layer()
    assert flex._score_of(m.score, H, "cpu") is flex._score_of(m.score, H, "cpu")
    with torch.no_grad():
        m.t.mul_(3)
    assert kinds(m.score) == ("temp", [6.0] * H)
    m.load_state_dict({"t": torch.full((H,), 4.0)})
    assert kinds(m.score) == ("temp", [4.0] * H)
    m.t = torch.nn.Parameter(torch.full((H,), 5.0))
    assert kinds(m.score) == ("temp", [5.0] * H)
    m.t.register_hook(lambda g: m and g)  # (a parameter that leads back to its object)
    assert kinds(m.score) == ("temp", [5.0] * H)
    del f, m
    gc.collect()
    assert len(flex._score_cache) == 0


def test_callables_without_tensors_are_evaluated_once():
    calls = []
    cap = 30.0

    def f(sc, b, h, qi, kj):
        calls.append(1)  # (the list grows: what it holds is a dependency too)
        return softcap(sc, cap)
    kinds(f), kinds(f)
    assert len(calls) == 2

    seen = []
    orig = flex._evaluate
    flex._evaluate = lambda *a: seen.append(1) or orig(*a)
    try:
        for g in (lambda sc, b, h, qi, kj: softcap(sc, 30.0), Cap(20.0), Cap(20.0).other,
                  lambda sc, b, h, qi, kj: sc + 0.5 * (kj - qi)):
            seen.clear()
            kinds(g), kinds(g), kinds(g)
            assert len(seen) == 1
            kinds(g, H + 1)
            assert len(seen) == 2
        t = torch.ones(H)
        g = lambda sc, b, h, qi, kj: sc * t[h]
        seen.clear()
        kinds(g), kinds(g)
        assert len(seen) == 2  # tensors may change unseen
    finally:
        flex._evaluate = orig


def test_what_cannot_be_listed_is_evaluated_again():
    import numpy as np
    box = np.ones(1)
    f = lambda sc, b, h, qi, kj: sc * float(box[0])
    assert kinds(f)[0] == "none"
    box[0] = 2
    assert kinds(f)[1][0] == 2

    class Hidden:
        def __getattr__(self, name):
            return state[0]
    state, hid = [2.0], Hidden()
    g = lambda sc, b, h, qi, kj: sc * hid.anything
    assert kinds(g)[1][0] == 2
    state[0] = 3.0
    assert kinds(g)[1][0] == 3

    def late(sc, b, h, qi, kj):
        import math
        return sc * math.tau_of_this_test
    import math
    math.tau_of_this_test = 2.0
    try:
        assert kinds(late)[1][0] == 2
        math.tau_of_this_test = 4.0
        assert kinds(late)[1][0] == 4
    finally:
        del math.tau_of_this_test


@pytest.mark.gpu
def test_in_a_graph(cuda):
    """What the last call before the capture found is captured; what is known to have changed is refused."""
    import chia_proj_b200 as cp
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, H, 200, 64, generator=g).to(torch.bfloat16).cuda() for _ in range(3))
    cap = torch.tensor(30.0, device="cuda")

    class Hidden:
        def __getattr__(self, name):
            return 30.0
    hid = Hidden()
    want = cp.attention(q, k, v, mod="softcap", softcap=30.0, mask=cp.FULL)
    for f in (lambda sc, b, h, qi, kj: softcap(sc, cap), lambda sc, b, h, qi, kj: softcap(sc, hid.x),
              lambda sc, b, h, qi, kj: softcap(sc, 30.0), Cap(30.0)):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            eager = flex.flex_attention(q, k, v, score_mod=f)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = flex.flex_attention(q, k, v, score_mod=f)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(eager, want)
    f = lambda sc, b, h, qi, kj: softcap(sc, cap)
    flex.flex_attention(q, k, v, score_mod=f)
    cap.mul_(0.5)
    new = lambda sc, b, h, qi, kj: softcap(sc, 10.0)
    for bad in (f, new):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="before the capture"):
                flex.flex_attention(q, k, v, score_mod=bad)
            q + 1
    out = flex.flex_attention(q, k, v, score_mod=f)
    assert torch.equal(out, cp.attention(q, k, v, mod="softcap", softcap=15.0, mask=cp.FULL))
