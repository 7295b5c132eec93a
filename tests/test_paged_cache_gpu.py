"""The write into the paged 8-bit K/V cache and its tables where calls are ragged: many runs of tokens in the rows that
one CTA looks at, skipped tokens, pages out of range. Contents are compared exactly with ``paged_oracle.py``."""

import pytest
import torch

import chia_proj_b200 as cp
import paged_oracle as po
from test_paged_gpu import BF16, E4M3, F16, I8, check_append, ints, make_cache  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


@pytest.mark.parametrize("page,hkv,D,ct,dtype,T", [(16, 8, 64, E4M3, BF16, 2500), (64, 16, 64, I8, F16, 4000),
                                                   (128, 16, 64, E4M3, F16, 9000), (32, 8, 128, I8, BF16, 3200)])
@pytest.mark.parametrize("seed", range(4))
def test_runs_between_skipped_tokens(cuda, page, hkv, D, ct, dtype, T, seed):
    """So many tokens that a CTA looks at a whole page's worth of them: runs that begin in the rows of one CTA and end
    in the next one's, skipped tokens of every number behind them, pages that are not in the cache, short runs."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    slots, pages, bad = [], 0, False
    while len(slots) < T:
        off = rnd(page) if rnd(3) else 0
        n = 1 + rnd(page - off) if rnd(3) else page - off
        if rnd(8) == 0:
            p, bad = 100000 + pages, True
        else:
            p, pages = pages, pages + 1
        slots += [p * page + off + i for i in range(n)]
        slots += [-1] * (rnd(6) if rnd(2) else 0)
    kinds = 2 * hkv
    assert len(slots) // page * kinds >= 8 * 148  # the rule by which a CTA looks at a page's worth
    cache = make_cache(pages, hkv, page, D, ct, g)
    x = torch.randn(len(slots), kinds, D, generator=g).to(dtype).cuda()
    check_append(x[:, :hkv], x[:, hkv:], slots, cache)
    if bad:
        with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
            cp.check_device_status(0)


def compact(slots, x):
    """The tokens that are not skipped: what one page gets in one call is written together."""
    keep = [t for t, s in enumerate(slots) if s >= 0]
    return [slots[t] for t in keep], x[keep]


def check_contents(x, slots, before, cache, hkv):
    """The cache after the call, against the oracle's write of these tokens into what was there before."""
    for i in range(2):
        w, s = (before[i].double(), cache[i].dtype), before[2 + i].double()
        po.append(x[:, i * hkv:(i + 1) * hkv], slots, w, s)
        assert torch.equal(cache[2 + i].double().cpu(), s)
        assert torch.equal(cache[i].double().cpu(), w[0])


@pytest.mark.parametrize("page,hkv,D,ct,T", [(16, 8, 64, E4M3, 2500), (64, 16, 64, I8, 4000), (128, 16, 64, E4M3, 9000),
                                             (16, 2, 128, I8, 300), (128, 1, 128, E4M3, 400)])
@pytest.mark.parametrize("seed", range(3))
def test_skipped_tokens_within_a_page(cuda, page, hkv, D, ct, T, seed):
    """Tokens of runs of every kind skipped at random, also a page's first and all but its last: as if the others alone
    were there, with one scale for them all."""
    g = torch.Generator().manual_seed(100 + seed)
    rnd = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    slots, pages = [], 0
    while len(slots) < T:
        off = rnd(page) if rnd(3) else 0
        n = 1 + rnd(page - off) if rnd(3) else page - off
        run = [pages * page + off + i for i in range(n)]
        pages += 1
        often = rnd(4)
        slots += [-1 if rnd(4) < often else s for s in run]
    cache = make_cache(pages, hkv, page, D, ct, g)
    before = [c.clone().cpu() for c in cache]
    x = (torch.randn(len(slots), 2 * hkv, D, generator=g) * 30).to(BF16)
    dev = x.cuda()
    cp.cache_append(dev[:, :hkv], dev[:, hkv:], ints(slots), *cache)
    kept, xs = compact(slots, x)
    check_contents(xs, kept, before, cache, hkv)


@pytest.mark.parametrize("page,hkv,lead", [(16, 2, 0), (32, 1, 0), (64, 2, 0), (128, 2, 0), (16, 8, 75), (64, 16, 40), (128, 16, 40)])
def test_a_page_that_comes_again_is_reported(cuda, page, hkv, lead):
    """Two requests' tokens by turns, a page behind another one, more rows than a page has: what came first is written.
    Alone, where a CTA looks at one token, and behind so many pages (lead) that it looks at a page's worth."""
    D = 64
    g = torch.Generator().manual_seed(page)
    a, b, c = ([(lead + p) * page + i for i in range(page)] for p in (2, 0, 3))
    ahead = [p * page + i for p in range(lead) for i in range(page)][:lead * page - 5]
    n = len(ahead)
    assert not lead or n // page * 2 * hkv >= 8 * 148
    for slots, first in (([a[1], b[1], a[2], b[2]], [0, 1]), (a[3:6] + b[:2] + a[6:8] + c[1:2], [0, 1, 2, 3, 4, 7]),
                         (a + [a[0]], range(page)), (a + a[:3] + b[4:6], [*range(page), page + 3, page + 4]),
                         (a + [-1, -1, a[5]] + b[4:6], [*range(page), page + 3, page + 4])):
        cache = make_cache(lead + 4, hkv, page, D, E4M3, g)
        before = [t.clone().cpu() for t in cache]
        slots = ahead + slots
        x = torch.randn(len(slots), 2 * hkv, D, generator=g).to(BF16)
        dev = x.cuda()
        cp.cache_append(dev[:, :hkv], dev[:, hkv:], ints(slots), *cache)
        with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
            cp.check_device_status(0)
        kept = [*range(n), *(n + t for t in first)]
        check_contents(x[kept], [slots[t] for t in kept], before, cache, hkv)


@pytest.mark.parametrize("B", [3, 1024, 2300])
def test_release_of_bad_lengths(cuda, B):
    """Lengths that no row holds, near 2^31 and below zero, give nothing back; the others' pages come back in order."""
    page, width = 16, 5
    bad = {0: 2 ** 31 - 1, 1: -1, B // 2: 2 ** 31 - 9, B - 1: width * page + 1, 2 * B // 3: -2 ** 31}
    lens = [bad.get(b, (7 * b) % (width * page + 1)) for b in range(B)]
    table = [[width * b + p for p in range(width)] for b in range(B)]
    back = [p for b in range(B) if b not in bad for p in table[b][:po.pages_for(lens[b], page)]]
    ring = ints([-5] * (B * width))
    lens2, state = cp.release_pages(ints([1] * B), ints(lens), ints(table), ring, ints([4, 2]), page_size=page)
    assert state.tolist() == [4, 2 + len(back)]
    got = ring.tolist()
    at = [(6 + i) % (B * width) for i in range(len(back))]
    assert [got[i] for i in at] == back
    assert all(got[i] == -5 for i in set(range(B * width)) - set(at))
    assert lens2.tolist() == [max(bad[b], 0) if b in bad else 0 for b in range(B)]
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)


@pytest.mark.parametrize("state", [[-1, 2], [5, 0], [2 ** 31 - 1, 1], [0, 6], [0, -1], [3, 2 ** 31 - 1]])
def test_release_into_a_bad_ring(cuda, state):
    """Nobody is released, and the ring that is returned hands out nothing."""
    ring = ints([9, 8, 7, 6, 5])
    table = ints([[1, 2], [3, 4]])
    lens, got = cp.release_pages(ints([1, 0]), ints([20, 30]), table, ring, ints(state), page_size=16)
    assert lens.tolist() == [20, 30] and got.tolist() == [0, 0] and ring.tolist() == [9, 8, 7, 6, 5]
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)
    step = cp.page_tables(lens, ints([1, 3]), table, ring, got, page_size=16, max_tokens=4)
    assert step.slots.tolist() == [36, -1, -1, -1] and step.seq_lens.tolist() == [21, 30]
    with pytest.raises(cp.ChiaError, match="NO_PAGES"):
        cp.check_device_status(0)


@pytest.mark.parametrize("most", [0, 1, 40, 1500, 2999])
def test_no_page_is_lost_past_max_tokens(cuda, most):
    """A step with more tokens than max_tokens is reported; the pages that it took stand in the table all the same, so that
    they can be given back."""
    page, width = 16, 80
    lens, new = [5, 0, 33], [1000, 1200, 800]
    table = torch.full((3, width), -9, dtype=torch.int32)
    table[0, 0], table[2, :3] = 500, torch.tensor([501, 502, 503])
    ring = list(range(300))
    want = po.tables(lens, new, table.tolist(), ring, [290, 250], page, 3000)
    dev, dring = table.cuda(), ints(ring)
    got = cp.page_tables(ints(lens), ints(new), dev, dring, ints([290, 250]), page_size=page, max_tokens=most)
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)
    assert got.slots.tolist() == want[0][:most] and got.positions.tolist() == want[1][:most]
    assert got.cu_q.tolist() == want[2] and got.seq_lens.tolist() == want[3] and got.free_state.tolist() == want[4]
    assert dev.tolist() == want[5]
    _, state = cp.release_pages(ints([1, 1, 1]), got.seq_lens, dev, dring, got.free_state, page_size=page)
    assert state.tolist()[1] == 250 + 4


@pytest.mark.parametrize("B,page", [(1, 16), (7, 32), (1500, 16)])
def test_rejected_tokens_give_their_pages_back(cuda, B, page):
    """Steps of drafted tokens of which some are rejected: every page is in one request or in the ring, in the order of
    the requests, and the tables go on as the oracle's do."""
    g = torch.Generator().manual_seed(B)
    rnd = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    width = 12
    total = B * width + 3
    ring, state = torch.randperm(total, generator=g).tolist(), [total - 2, total]
    lens, table = [0] * B, [[0] * width for _ in range(B)]
    dev = [ints(lens), ints(table), ints(ring), ints(state)]
    for step in range(12):
        new = [rnd(page + 9) if (step + b) % 3 else 0 for b in range(B)]
        new = [n if lens[b] + n <= width * page else 0 for b, n in enumerate(new)]
        T = sum(new)
        want = po.tables(lens, new, table, ring, state, page, T)
        got = cp.page_tables(dev[0], ints(new), dev[1], dev[2], dev[3], page_size=page, max_tokens=T)
        assert got.slots.tolist() == want[0] and got.seq_lens.tolist() == want[3] and got.free_state.tolist() == want[4]
        lens, state, table = want[3], want[4], want[5]
        keep = [n - rnd(m + 1) if b % 5 else n - m for b, (n, m) in enumerate(zip(lens, new))]
        for b in range(B):
            for p in range(po.pages_for(keep[b], page), po.pages_for(lens[b], page)):
                ring[(state[0] + state[1]) % total] = table[b][p]
                state = [state[0], state[1] + 1]
        lens2, state2 = cp.release_pages(None, got.seq_lens, dev[1], dev[2], got.free_state, page_size=page, keep_lens=ints(keep))
        assert lens2.tolist() == keep and state2.tolist() == state and dev[2].tolist() == ring
        dev[0], dev[3], lens = lens2, state2, keep
    held = [table[b][p] for b in range(B) for p in range(po.pages_for(lens[b], page))]
    assert sorted(held + [ring[(state[0] + i) % total] for i in range(state[1])]) == list(range(total))


def test_kept_lengths_out_of_range(cuda):
    table, ring = ints([[1, 2], [3, 4], [5, 6]]), ints([0] * 9)
    lens, state = cp.release_pages(None, ints([20, 30, 17]), table, ring, ints([8, 0]), page_size=16, keep_lens=ints([21, -1, 16]))
    assert lens.tolist() == [20, 30, 16] and state.tolist() == [8, 1] and ring.tolist() == [0] * 8 + [6]
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)
    args = (ints([20, 30, 17]), table, ring, ints([8, 0]))
    for done, kw in ((None, {}), (ints([1, 0, 0]), dict(keep_lens=ints([0, 0, 0]))), (None, dict(keep_lens=ints([0])))):
        with pytest.raises(ValueError):
            cp.release_pages(done, *args, page_size=16, **kw)


def test_attention_after_a_rollback(cuda):
    """Drafted tokens are written, rejected and written over: the answer is that of a cache that never saw them. (The
    scales of the pages they shared may stay larger: within the rounding that this leaves, 2^-3 of a value at most here.)"""
    g = torch.Generator().manual_seed(3)
    page, hkv, H, D, n = 16, 2, 8, 64, 70
    x = torch.randn(n + 40, 2 * hkv, D, generator=g).to(BF16).cuda()
    q = torch.randn(1, H, D, generator=g).to(BF16).cuda()

    def play(steps):
        cache = cp.new_cache(9, hkv, D, page_size=page)
        lens, table = ints([0]), torch.zeros(1, 8, dtype=torch.int32, device="cuda")
        ring, state = ints(list(range(9))), ints([0, 9])
        for rows, keep in steps:
            t = cp.page_tables(lens, ints([len(rows)]), table, ring, state, page_size=page, max_tokens=len(rows))
            cp.cache_append(x[rows][:, :hkv], x[rows][:, hkv:], t.slots, *cache)
            lens, state = t.seq_lens, t.free_state
            if keep < int(lens):
                lens, state = cp.release_pages(None, lens, table, ring, state, page_size=page, keep_lens=ints([keep]))
        assert int(lens) == n and int(state[1]) == 9 - 5
        return cp.paged_attention(q, *cache, table, lens).float()

    plain = play([(list(range(n)), n)])
    drafts = play([(list(range(60)), 60), (list(range(80, 109)), 63), (list(range(70, 73)), 60), (list(range(60, n)), n)])
    assert (plain - drafts).norm() / plain.norm() < 0.06  # e4m3: 2.6% rms in K and in V, either way


def test_writes_are_known_to_autograd(cuda):
    """What is written in place has a new version, so that a graph that saved it refuses its backward pass; inference
    tensors have none. A forward-mode tangent, which would be dropped, is refused."""
    def play():
        cache = cp.new_cache(4, 2, 64, page_size=16)
        x = torch.randn(3, 2, 64, dtype=BF16, device="cuda")
        table, ring, out = ints([[0, 0]]), ints([2, 1, 0]), torch.zeros_like(x)
        kept = [*cache, table, ring, out]
        before = None if x.is_inference() else [t._version for t in kept]
        step = cp.page_tables(ints([0]), ints([3]), table, ring, ints([0, 3]), page_size=16, max_tokens=3)
        cp.cache_append(x, x, step.slots, *cache)
        cp.paged_attention(x, *cache, table, step.seq_lens, step.cu_q, out=out)
        cp.release_pages(ints([1]), step.seq_lens, table, ring, step.free_state, page_size=16)
        return kept, before, x
    kept, before, x = play()
    assert all(t._version > v for t, v in zip(kept, before))
    with torch.inference_mode():
        play()
    w = torch.ones(4, 2, device="cuda", requires_grad=True)
    loss = (w * kept[2]).sum()  # saves k_scale
    cp.cache_append(x, x, ints([5, 6, 7]), *kept[:4])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for k, v in ((dual, x), (x, dual)):
            with pytest.raises(ValueError, match="tangent"):
                cp.cache_append(k, v, ints([5, 6, 7]), *kept[:4])
        with pytest.raises(ValueError, match="tangent"):
            cp.paged_attention(dual, *kept[:4], kept[4], ints([3]))
