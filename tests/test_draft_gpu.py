"""Tables, verification and compaction of drafted tokens (include/chia_draft.h) on the GPU against plain 64-bit
restatements (``draft_oracle.py``), exactly."""

import math

import pytest
import torch

import chia_proj_b200 as cp
import draft_oracle as do
import paged_oracle as po

pytestmark = pytest.mark.gpu
E4M3, I8 = torch.float8_e4m3fn, torch.int8


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def reported():
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)


# ---------------------------------------------------------------------- tables
@pytest.mark.parametrize("sizes", [[1], [2], [64], [0, 1, 0, 64, 33, 32, 31, 0], [65, 3, 300, 64], [5] * 700,
                                   [13, 0, 7, 64, 1] * 9])
@pytest.mark.parametrize("shape", ["tree", "chain", "wide"])
def test_tree_tables(cuda, sizes, shape):
    lens = [n + (37 * i) % 1000 for i, n in enumerate(sizes)]
    lens[0] = sizes[0] + 2 ** 30  # far positions
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    parents = [p for i, n in enumerate(sizes) for p in do.tree(n, i, shape == "chain", shape == "wide")]
    rows = cu[-1] + 11  # rows behind the last request
    got = cp.tree_tables(ints(parents + [99] * 11), ints(cu), ints(lens))
    pos, words = do.tables(parents, cu, lens, rows)
    assert got.positions.dtype == torch.int32 and got.ancestors.dtype == torch.int64
    assert got.positions.tolist() == pos and got.ancestors.tolist() == words


def test_tree_tables_bad_values_are_reported(cuda):
    t = cp.tree_tables(ints([-1, 1, -2, 0, 7, 1]), ints([0, 6]), ints([10]))  # parents that do not come before: roots
    assert t.positions.tolist() == [4, 4, 4, 5, 4, 5] and t.ancestors.tolist() == [1, 2, 4, 9, 16, 34]
    reported()
    t = cp.tree_tables(ints([-1, 0, -1, 0, -1, 0]), ints([0, 2, 1, 4]), ints([5, 5, 5]))  # offsets that fall
    assert t.positions.tolist() == [3, 4, 0, 0, 0, 0] and t.ancestors.tolist() == [1, 3, 0, 0, 0, 0]
    reported()
    t = cp.tree_tables(ints([-1, 0]), ints([0, 9]), ints([5]))
    assert t.positions.tolist() == [0, 0]
    reported()
    t = cp.tree_tables(ints([3, -1, 0, 3]), ints([1, 3]), ints([2]))  # rows before the first request
    assert t.positions.tolist() == [0, 0, 1, 0] and t.ancestors.tolist() == [0, 1, 3, 0]
    cp.check_device_status(0)
    assert cp.tree_tables(ints([]), ints([0, 0]), ints([3])).positions.shape == (0,)


# ---------------------------------------------------------------- verification
def rows(n, V, g, dtype, sharp=3.0):
    return torch.softmax(sharp * torch.randn(n, V, generator=g), 1).to(dtype)


def drawn(parents, q, g):
    """Children's tokens, drawn one after another without replacement from their parents' rows."""
    tokens, left = [0] * len(parents), {}
    for i, p in enumerate(parents):
        if p >= 0:
            row = left.setdefault(p, q[p].double().clone())
            if not row.sum() > 0:
                row += 1.0
            tokens[i] = int(torch.multinomial(row, 1, generator=g))
            row[tokens[i]] = 0.0
    return tokens


def check_verify(p, tokens, parents, cu, u, q, most, device_rows=None):
    dev_p, dev_q = device_rows if device_rows else (p.cuda(), None if q is None else q.cuda())
    got = cp.verify_drafts(dev_p, ints(tokens), ints(parents), ints(cu), u.cuda(), draft_probs=dev_q, max_tokens=most)
    counts, toks, path = do.verify(p, tokens, parents, cu, u, q, most)
    assert got.counts.tolist() == counts
    assert got.path.tolist() == path
    assert got.tokens.tolist() == toks
    return counts


@pytest.mark.parametrize("V", [1, 2, 100, 511, 512, 513, 4097, 12345])
@pytest.mark.parametrize("drafts", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_verify(cuda, V, drafts, dtype):
    g = torch.Generator().manual_seed(V + drafts)
    sizes = [7, 0, 1, 20, 3, 64, 2]
    parents = [x for i, n in enumerate(sizes) for x in do.tree(n, i, chain=i % 3 == 0)]
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    n, seen = cu[-1], 0
    p = rows(n, V, g, dtype)
    q = torch.softmax(p.float().log() + 0.7 * torch.randn(n, V, generator=g), 1).to(dtype)
    tokens = [t for b in range(len(sizes)) for t in drawn(parents[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], g)]
    for most in (1, 2, 5, 70):
        u = torch.rand(n, generator=g)
        seen += sum(check_verify(p, tokens, parents, cu, u, q if drafts else None, most))
    # some drafts were accepted (without draft rows a token's chance is its own probability, near 1 / V: perhaps none)
    assert V < 100 or not drafts or seen > 4 * 6


def test_verify_many_rejections(cuda):
    """All children of a root, most of them rejected: a pass for each; masses that come near nothing."""
    g = torch.Generator().manual_seed(5)
    V, n = 3000, 64
    parents, cu = [-1] + [0] * (n - 1), [0, n]
    p, q = rows(n, V, g, torch.float32, 1.0), rows(n, V, g, torch.float32, 4.0)
    tokens = drawn(parents, q, g)
    for lo in (0.0, 0.9, 0.9999):
        u = lo + (1 - lo) * torch.rand(n, generator=g)
        u = u.clamp(max=1 - 2.0 ** -24)
        check_verify(p, tokens, parents, cu, u, q, 4)
        check_verify(p, tokens, parents, cu, u, None, 4)


def test_verify_rows_at_the_border(cuda):
    V, n = 700, 3
    u = torch.tensor([0.5, 0.5, 0.5])
    one = torch.zeros(n, V)
    one[0, 3], one[1, 699], one[2, 0] = 1.0, 1.0, 1.0
    chain, cu = [-1, 0, 1], [0, 3]
    for q in (None, one):  # drafts of the only token there is, right and wrong
        assert check_verify(one, [9, 3, 699], chain, cu, u, q, 5) == [3]
        check_verify(one, [9, 4, 699], chain, cu, u, q, 5)
        check_verify(one, [9, 3, 698], chain, cu, u, q, 5)
    check_verify(one, [9, 3, 699], chain, cu, torch.zeros(n), None, 5)  # u = 0
    check_verify(one, [9, 3, 699], chain, cu, torch.full((n,), 1 - 2.0 ** -24), one, 5)
    empty = torch.zeros(n, V)
    assert check_verify(empty, [9, 3, 3], chain, cu, u, None, 5) == [1]  # nothing to draw: -1
    check_verify(empty, [9, 3, 3], chain, cu, u, one, 5)
    # the target equal to the draft: never rejected
    g = torch.Generator().manual_seed(1)
    p = rows(n, V, g, torch.float32)
    assert check_verify(p, [0] + drawn(chain, p, g)[1:], chain, cu, torch.full((n,), 1 - 2.0 ** -24), p, 5) == [3]
    # entries that are no probabilities count as nothing; the same token twice among siblings
    p[0, 5], p[1, 6], p[2, 7], p[2, 8] = float("nan"), float("inf"), -1.0, -float("inf")
    for tokens in ([0, 5, 6], [0, 10, 10], [0, 7, 8]):
        for q in (None, p.flip(0).contiguous()):
            check_verify(p, tokens, [-1, 0, 0], cu, u, q, 5)
            check_verify(p, tokens, chain, cu, torch.tensor([0.99, 0.0, 0.01]), q, 5)


def test_verify_strides_and_types(cuda):
    g = torch.Generator().manual_seed(7)
    n, V, parents, cu = 5, 1000, [-1, 0, 0, 1, 2], [0, 5]
    p, q = rows(n, V, g, torch.bfloat16), rows(n, V, g, torch.bfloat16)
    tokens, u = drawn(parents, q, g), torch.rand(n, generator=g)
    wide = torch.full((n, V + 13), 0.5, dtype=torch.bfloat16, device="cuda")  # odd strides and bases
    wide[:, 5:5 + V] = p.cuda()
    turned = torch.empty(V, n, dtype=torch.bfloat16, device="cuda").t().copy_(q)  # copied
    check_verify(p, tokens, parents, cu, u, q, 4, (wide[:, 5:5 + V], turned))
    same = p[:1].expand(n, V)  # one row for all nodes
    check_verify(same.contiguous(), tokens, parents, cu, u, None, 4, (same.cuda(), None))


def test_verify_a_large_vocabulary(cuda):
    g = torch.Generator().manual_seed(11)
    n, V = 2, 1 << 22
    p = torch.rand(n, V, generator=g) / V * 2
    for x in (0.0, 1e-7, 0.25, 0.999999):
        u = torch.tensor([x, 0.999])
        got = cp.verify_drafts(p.cuda(), ints([0, 5]), ints([-1, 0]), ints([0, 2]), u.cuda(), max_tokens=2)
        r = p[0].double().clone()
        r[5] = 0.0
        sums = r.cumsum(0)
        want = int((sums <= float(u[0]) * float(sums[-1])).sum())
        assert got.counts.tolist() == [1] and got.tokens.tolist() == [[want, -1]]


def test_verify_bad_values_are_reported(cuda):
    g = torch.Generator().manual_seed(2)
    p, u = rows(6, 50, g, torch.float32).cuda(), torch.zeros(6, device="cuda")
    ok = cp.verify_drafts(p, ints([0] * 6), ints([-1, 0, 1, -1, 0, 1]), ints([0, 3, 6]), u, max_tokens=4)
    assert ok.counts.tolist() == [3, 3]
    cp.check_device_status(0)
    # tokens and parents out of range are never accepted
    for tokens, parents in (([0, 50, 0, 0, -1, 0], [-1, 0, 1, -1, 0, 1]), ([0] * 6, [-1, 1, 1, -1, 5, 1]),
                            ([0] * 6, [-1, -2, 1, -1, 2 ** 30, 1])):
        got = cp.verify_drafts(p, ints(tokens), ints(parents), ints([0, 3, 6]), u, max_tokens=4)
        assert got.counts.tolist() == [1, 1] and got.path[:, 0].tolist() == [0, 0]
        reported()
    # offsets out of range; a request of more than 64 tokens
    got = cp.verify_drafts(p, ints([0] * 6), ints([-1] + [0] * 5), ints([0, 3, 9]), u, max_tokens=4)
    assert got.counts.tolist() == [2, 0] and got.tokens[1].tolist() == [-1] * 4 and got.path[1].tolist() == [-1] * 4
    reported()
    big = cp.verify_drafts(p[:1].expand(70, 50), ints([0] * 70), ints([-1] + [0] * 69), ints([0, 70]),
                           torch.zeros(70, device="cuda"), max_tokens=4)
    assert big.counts.tolist() == [0]
    reported()


# ------------------------------------------------------------------ compaction
def cache_of(pages, hkv, page, D, ct, g, spread=6):
    k, v = (torch.randn(pages, hkv, page, D, generator=g) * 100 for _ in range(2))
    k, v = (x.clamp(-448, 448).to(ct) if ct == E4M3 else x.round().clamp(-127, 127).to(ct) for x in (k, v))
    ks, vs = (2.0 ** torch.randint(-6, -6 + spread, (pages, hkv), generator=g).float() for _ in range(2))
    return [k, v, ks, vs]


def check_compact(sizes, bases, paths, page, hkv, D, ct, seed=0, most=None, stride=0):
    g = torch.Generator().manual_seed(seed)
    lens = [b + n for b, n in zip(bases, sizes)]
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    need = [po.pages_for(n, page) for n in lens]
    perm = torch.randperm(sum(need) + 2, generator=g).tolist()
    width = max(max(need), 1)
    table = [perm[sum(need[:i]):sum(need[:i + 1])] + [10 ** 6] * (width - need[i]) for i in range(len(need))]
    k, v, ks, vs = cache_of(len(perm), hkv, page, D, ct, g)
    dev = [t.cuda() for t in (k, v, ks, vs)]
    most = most or max(map(len, paths))
    path = [p + [-5] * (most - len(p)) for p in paths]
    wide = torch.full((len(table), width + stride), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, :width] = ints(table)
    keep = cp.cache_compact(ints(path), ints([len(p) for p in paths]), ints(cu), ints(lens), wide[:, :width], *dev)
    kd, vd, ksd, vsd = (t.double() for t in (k, v, ks, vs))
    want = do.compact(paths, [len(p) for p in paths], cu, lens, table, kd, ksd, ct)
    do.compact(paths, [len(p) for p in paths], cu, lens, table, vd, vsd, ct)
    assert keep.tolist() == want
    for a, b in zip(dev, (kd, vd, ksd, vsd)):
        assert torch.equal(a.double().cpu(), b)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("ct", [E4M3, I8])
@pytest.mark.parametrize("hkv,D", [(1, 64), (3, 128)])
def test_compact(cuda, page, ct, hkv, D):
    check_compact([13], [page - 3], [[0, 4, 5, 9, 12]], page, hkv, D, ct)
    check_compact([64, 1, 0, 25, 64, 2, 30, 64],
                  [5, 0, 7, 2 * page - 1, 0, page - 1, 3, page - 8],
                  [[0, 1, 2, 10, 40, 63], [0], [], [0, 24], list(range(64)), [1], [0, 1, 2], [x for x in range(64) if x % 3 != 1]],
                  page, hkv, D, ct, seed=page, stride=3)


@pytest.mark.parametrize("seed", range(4))
def test_compact_drawn(cuda, seed):
    g = torch.Generator().manual_seed(100 + seed)
    B = 40
    sizes = torch.randint(0, 65, (B,), generator=g).tolist()
    bases = torch.randint(0, 100, (B,), generator=g).tolist()
    paths = [sorted(torch.randperm(n, generator=g)[:int(torch.randint(0, n + 1, (1,), generator=g))].tolist()) for n in sizes]
    check_compact(sizes, bases, paths, 16, 2, 64, I8 if seed % 2 else E4M3, seed=seed, most=64)


def test_compact_special_values(cuda):
    """A page without a scale, NaN bytes."""
    table, cu, lens = ints([[1, 0]]), ints([0, 20]), ints([20])
    k, v, ks, vs = (t.cuda() for t in cache_of(2, 1, 16, 64, E4M3, torch.Generator().manual_seed(1)))
    k.view(torch.uint8)[0, 0, 3, 7] = 0x7f
    ks.zero_()
    vs[1], vs[0] = 0.0, 0.25
    before = k.clone()
    keep = cp.cache_compact(ints([[0, 19]]), ints([2]), cu, lens, table, k, v, ks, vs)
    assert keep.tolist() == [2] and not ks.any()
    assert torch.equal(k.view(torch.uint8)[1, 0, 1], before.view(torch.uint8)[0, 0, 3])  # as it is, NaN and all
    assert vs.flatten().tolist() == [0.25, 0.25] and torch.equal(v[1, 0, 1].float(), v[0, 0, 3].float())
    assert not v[1, 0, 0].float().any()  # what a page without a scale held stands for nothing


def test_compact_bad_values_are_reported(cuda):
    cache = [t.cuda() for t in cache_of(4, 1, 16, 64, I8, torch.Generator().manual_seed(1))]
    before = [t.clone() for t in cache]
    table = [[0, 1], [2, 3]]

    def run(path=((0, 2), (0, 1)), counts=(2, 2), cu=(0, 5, 10), lens=(20, 12), tab=table):
        return cp.cache_compact(ints(path), ints(counts), ints(cu), ints(lens), ints(tab), *cache).tolist()

    for kw, want in ((dict(path=((1, 1), (0, 1))), [20, 9]), (dict(path=((0, 5), (0, 1))), [20, 9]),
                     (dict(path=((-1, 2), (0, 1))), [20, 9]), (dict(counts=(3, 2)), [20, 9]), (dict(counts=(-1, 2)), [20, 9]),
                     (dict(lens=(33, 12)), [33, 9]), (dict(lens=(4, 12)), [4, 9]), (dict(lens=(-4, 12)), [-4, 9]),
                     (dict(tab=[[0, 4], [2, 3]]), [20, 9]), (dict(tab=[[0, -1], [2, 3]]), [20, 9]),
                     (dict(cu=(-1, 5, 10)), [20, 9]), (dict(cu=(7, 5, 10)), [20, 9])):
        assert run(**kw) == want, kw
        reported()
        for a, b in zip(cache, before):
            assert torch.equal(a, b)
    # a chunk of a prompt beside a tree is left as it is
    big = [t.cuda() for t in cache_of(12, 1, 16, 64, I8, torch.Generator().manual_seed(2))]
    was = [t.clone() for t in big]
    keep = cp.cache_compact(ints([[0, 9], [0, 1]]), ints([2, 2]), ints([0, 70, 75]), ints([100, 5]),
                            ints([[0, 1, 2, 3, 4, 5, 6], [7, 0, 0, 0, 0, 0, 0]]), *big)
    assert keep.tolist() == [100, 2] and all(torch.equal(a, b) for a, b in zip(big, was))


# ------------------------------------------------------------ streams and graphs
def test_streams_and_graphs(cuda):
    """Two streams at once; captured calls replayed on new values."""
    g = torch.Generator().manual_seed(21)
    sizes = [9, 30, 1, 64]
    cu = [sum(sizes[:i]) for i in range(5)]
    parents = [p for i, n in enumerate(sizes) for p in do.tree(n, i)]
    n, V = cu[-1], 5000
    p, q, u = rows(n, V, g, torch.float32), rows(n, V, g, torch.float32), torch.rand(n, generator=g)
    tokens = [t for b in range(4) for t in drawn(parents[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], g)]
    dp, dq, du, dt, dpar, dcu = p.cuda(), q.cuda(), u.cuda(), ints(tokens), ints(parents), ints(cu)
    lens, table = ints([s + 20 for s in sizes]), ints([[6 * b + i for i in range(6)] for b in range(4)])
    cache = [t.cuda() for t in cache_of(24, 2, 16, 64, E4M3, g)]

    def step(cache):
        done = cp.verify_drafts(dp, dt, dpar, dcu, du, draft_probs=dq, max_tokens=8)
        return [*done, cp.cache_compact(done.path, done.counts, dcu, lens, table, *cache), *cp.tree_tables(dpar, dcu, lens)]

    first = [t.clone() for t in cache]
    want = step(first)
    assert want[0].tolist() == do.verify(p, tokens, parents, cu, u, q, 8)[0]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([(c, step(c)) for c in [[t.clone() for t in cache] for _ in range(3)]])
    torch.cuda.synchronize()
    for runs in got:
        for c, r in runs:
            assert all(torch.equal(a, b) for a, b in zip(r, want))
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c, first))
    mine = [t.clone() for t in cache]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(mine)
    u2 = torch.rand(n, generator=g)
    du.copy_(u2)
    for a, b in zip(mine, cache):
        a.copy_(b)
    graph.replay()
    other = [t.clone() for t in cache]
    again = step(other)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(mine, other))
    assert out[0].tolist() == do.verify(p, tokens, parents, cu, u2, q, 8)[0]


def test_autograd_sees_what_is_written(cuda):
    """The cache's tensors have new versions; probabilities that learn are taken without a graph."""
    cache = [t.cuda() for t in cache_of(4, 1, 16, 64, E4M3, torch.Generator().manual_seed(1))]
    was = [t._version for t in cache]
    cp.cache_compact(ints([[0, 3]]), ints([2]), ints([0, 5]), ints([9]), ints([[0, 1]]), *cache)
    assert all(t._version > v for t, v in zip(cache, was))
    p = torch.rand(3, 40, device="cuda", requires_grad=True)
    r = cp.verify_drafts(p, ints([0, 1, 2]), ints([-1, 0, 1]), ints([0, 3]), torch.rand(3, device="cuda"), max_tokens=3)
    assert not any(t.requires_grad for t in r)


# -------------------------------------------------------------------- refusals
def test_refusals(cuda):
    p, u, i = torch.rand(4, 9, device="cuda"), torch.rand(4, device="cuda"), ints([0, 0, 0, 0])
    good = dict(target_probs=p, tokens=i, parents=ints([-1, 0, 1, 2]), cu_q=ints([0, 4]), uniforms=u, max_tokens=3)
    cp.verify_drafts(**good)
    for bad in (dict(target_probs=p.double()), dict(target_probs=p[:, :0]), dict(tokens=i[:3]), dict(tokens=i.long()),
                dict(parents=i[:2]), dict(cu_q=ints([0])), dict(uniforms=u.double()), dict(uniforms=u[:3]),
                dict(uniforms=torch.rand(8, device="cuda")[::2]), dict(max_tokens=0), dict(draft_probs=p.half()),
                dict(draft_probs=p[:, :8]), dict(target_probs=p[0])):
        with pytest.raises(ValueError):
            cp.verify_drafts(**{**good, **bad})
    for bad in ((i.long(), ints([0, 4]), ints([4])), (i, ints([0]), ints([])), (i, ints([0, 4]), ints([4, 4])),
                (ints([0] * 8)[::2], ints([0, 4]), ints([4]))):
        with pytest.raises(ValueError):
            cp.tree_tables(*bad)
    cache = cp.new_cache(2, 1, 64, page_size=16)
    good = dict(path=ints([[0, 1]]), counts=ints([1]), cu_q=ints([0, 2]), seq_lens=ints([2]), block_table=ints([[0]]),
                k_cache=cache[0], v_cache=cache[1], k_scale=cache[2], v_scale=cache[3])
    assert cp.cache_compact(**good).tolist() == [1]
    for bad in (dict(path=ints([0, 1])), dict(path=ints([[0], [1]])), dict(path=ints([[0, 1], [1, 2]]).t()[:1]), dict(counts=ints([1, 1])),
                dict(cu_q=ints([0])), dict(seq_lens=ints([2]).long()), dict(block_table=ints([[0], [1]])),
                dict(k_cache=cache[0].view(torch.int8)), dict(v_scale=cache[3][:1])):
        with pytest.raises(ValueError):
            cp.cache_compact(**{**good, **bad})


@pytest.mark.parametrize("ct,page", [(E4M3, 16), (I8, 64)])
def test_a_step_that_was_not_served_can_be_run_again(cuda, ct, page):
    """The second of three requests finds no page. Its cache and its length stay as they were, the others go on as alone;
    with pages the same step serves it."""
    g = torch.Generator().manual_seed(page)
    B, hkv, D, n = 3, 2, 64, 12
    start = [page - 3, 2 * page - 2, 5]  # the first and the second need a page for 12 more (the third, in small pages)
    cache = cp.new_cache(12, hkv, D, page_size=page, dtype=ct)
    table, ring = ints([[0] * 4] * B), torch.arange(12, dtype=torch.int32, device="cuda")
    first = cp.page_tables(ints([0] * B), ints(start), table, ring, ints([0, 12]), page_size=page, max_tokens=sum(start))
    kv = torch.randn(sum(start), 2, hkv, D, generator=g).to(torch.bfloat16).cuda()
    cp.cache_append(kv[:, 0], kv[:, 1], first.slots, *cache)
    parents = [-1, 0, 0, 1, 1, 2, 2, 5, 6, 7, 8, 9]
    kv = torch.randn(B * n, 2, hkv, D, generator=g).to(torch.bfloat16).cuda()
    path, counts = ints([[0, 2, 6, 8]] * B), ints([4] * B)

    def step(cache, table, free):
        st = cp.page_tables(first.seq_lens, ints([n] * B), table, ring, free, page_size=page, max_tokens=B * n)
        cp.tree_tables(ints(parents * B), st.cu_q, st.seq_lens)
        cp.cache_append(kv[:, 0], kv[:, 1], st.slots, *cache)
        return st, cp.cache_compact(path, counts, st.cu_q, st.seq_lens, table, *cache, st.slots)

    copy = lambda: ([t.clone() for t in cache], table.clone())
    (few, few_table), (all_, all_table) = copy(), copy()
    head = int(first.free_state[0])
    st, keep = step(few, few_table, ints([head, 1]))  # a page for the first alone
    with pytest.raises(cp.ChiaError, match="NO_PAGES"):
        cp.check_device_status(0)
    served = [bool((st.slots[b * n:(b + 1) * n] >= 0).all()) for b in range(B)]
    assert served[0] and not served[1]
    assert keep.tolist() == [s + 4 if ok else s for s, ok in zip(start, served)]
    st2, keep2 = step(all_, all_table, ints([head, 12 - head]))
    assert keep2.tolist() == [s + 4 for s in start]
    used = lambda tab, b, m: tab[b, :po.pages_for(m, page)].long()
    for b in range(B):
        for a, c, was in zip(*([t.view(torch.uint8) for t in ts] for ts in (few, all_, cache))):
            if served[b]:  # as with pages enough (a page of another number may hold it)
                x, y = a[used(few_table, b, start[b] + n)], c[used(all_table, b, start[b] + n)]
            else:
                x, y = a[used(few_table, b, start[b])], was[used(table, b, start[b])]
            assert torch.equal(x, y)
    # without the slots the last tokens of the request would be moved
    lost = [t.clone() for t in cache]
    bad = cp.cache_compact(path[1:2], counts[1:2], ints([0, n]), st.seq_lens[1:2], few_table[1:2], *lost)
    assert bad.tolist() == [start[1] - n + 4]


def test_compact_refuses_other_slots(cuda):
    cache = [t.cuda() for t in cache_of(2, 1, 16, 64, E4M3, torch.Generator().manual_seed(1))]
    args = (ints([[0, 1]]), ints([2]), ints([0, 2]), ints([2]), ints([[0]]), *cache)
    assert cp.cache_compact(*args, ints([0, 1])).tolist() == [2]
    assert cp.cache_compact(*args, ints([0])).tolist() == [2] and cp.cache_compact(*args, ints([0, -1])).tolist() == [2]
    assert cp.cache_compact(*args, torch.empty(0, dtype=torch.int32, device="cuda")).tolist() == [2]
    for bad in (torch.tensor([0, 1], device="cuda"), ints([[0, 1]]), ints([0, 9, 1, 9])[::2]):
        with pytest.raises(ValueError):
            cp.cache_compact(*args, bad)
    with pytest.raises(RuntimeError):
        cp.cache_compact(*args, torch.zeros(2, dtype=torch.int32))
