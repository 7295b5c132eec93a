"""paged_attention(tree=...) (chia_tree_attn of include/chia_draft.h) on the GPU against the plain 64-bit restatement
(``draft_oracle.py``), and a whole step of speculative decoding.

Tolerances, element by element, as of the attention without trees: the output is rounded once (2^-8 relative for bf16,
2^-11 for fp16); P may be rounded to 11 significant bits before P V (2^-12 of each term, the sum of whose sizes is the
oracle's ``mass``); exponentials, hyperbolic tangents, reciprocals and sums in fp32 stay under 2^-14 of a term for the
scores used here (|s| < 64). 2^-8 |o| (2^-11) + 2^-10 mass + 2^-24 is allowed; a log-sum-exp is off by 2^-11 at most.
"""

import math

import pytest
import torch

import chia_proj_b200 as cp
import draft_oracle as do
import paged_oracle as po

pytestmark = pytest.mark.gpu
E4M3, I8 = torch.float8_e4m3fn, torch.int8
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(sizes, bases, *, H=8, hkv=2, D=128, page=64, ct=E4M3, dtype=BF16, seed=0, shape="tree", q_size=1.0):
    """Requests of sizes[b] nodes behind bases[b] keys (negative: fewer keys than nodes)."""
    g = torch.Generator().manual_seed(seed)
    lens = [b + n for b, n in zip(bases, sizes)]
    cu = [sum(sizes[:i]) for i in range(len(sizes) + 1)]
    parents = [p for i, n in enumerate(sizes) for p in do.tree(n, seed + i, shape == "chain", shape == "wide")]
    need = [po.pages_for(n, page) for n in lens]
    pages = sum(need) + 2
    perm = torch.randperm(pages, generator=g).tolist()
    width = max(max(need), 1) + 1
    table = [perm[sum(need[:i]):sum(need[:i + 1])] + [-7] * (width - need[i]) for i in range(len(need))]

    def cache():
        x = torch.randn(pages, hkv, page, D, generator=g) * (150 if ct == E4M3 else 40)
        x = x.clamp(-448, 448).to(ct) if ct == E4M3 else x.round().clamp(-127, 127).to(ct)
        return x, 2.0 ** torch.randint(-9, -6, (pages, hkv), generator=g).float()

    (k, ks), (v, vs) = cache(), cache()
    q = (torch.randn(cu[-1], H, D, generator=g) * q_size).to(dtype)
    return dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, lens=lens, cu=cu, parents=parents)


def run(c, tree=None, **kw):
    d = [c[n].cuda() for n in ("k", "v", "ks", "vs")]
    lens, cu = ints(c["lens"]), ints(c["cu"])
    if tree is None:
        tree = cp.tree_tables(ints(c["parents"]), cu, lens)
    return cp.paged_attention(c["q"].cuda(), *d, ints(c["table"]), lens, cu, tree=tree, **kw)


def check(c, got, lse=None, rows=None, **kw):
    mask = kw.pop("mask", cp.CAUSAL)
    out, want_lse, mass = do.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], c["cu"], c["parents"],
                                       mask=mask, **kw)
    rel = 2.0 ** -8 if c["q"].dtype == BF16 else 2.0 ** -11
    ok = (got.double().cpu() - out).abs() <= rel * out.abs() + 2.0 ** -10 * mass + 2.0 ** -24
    assert ok[rows].all() if rows is not None else ok.all()
    if lse is not None:
        l = lse.double().cpu()
        assert torch.equal(l == -math.inf, want_lse == -math.inf)
        assert ((l - want_lse).abs()[want_lse > -math.inf] <= 2.0 ** -11).all()


SIZES = [13, 1, 0, 5, 30, 2]
BASES = [100, 0, 0, 31, 257, 64]
KINDS = [dict(), dict(mod="softcap", softcap=20.0), dict(mod="alibi"), dict(mod="temp"), dict(norm="sigmoid", sig_bias=-2.0),
         dict(norm="relu", out_scale=0.01)]
MASKS = [cp.CAUSAL, cp.Mask(left=6, right=0), cp.Mask(left=70, right=0), cp.Mask(right=0, block=24),
         cp.Mask(right=0, dilation=3), cp.Mask(left=10, right=0, prefix=20), cp.FULL]


def with_params(kw, H):
    if kw.get("mod") in ("alibi", "temp"):
        return {**kw, "head_param": [0.25 + 0.1 * h for h in range(H)]}
    return kw


# Trees of more than 64 rows (nodes x heads of a group) in the mean take the kernel of many queries: with 16 heads to each
# K/V head and a max_q that allows it. Both kernels serve any tree.
def heads(max_q, hkv=2):
    return hkv * (4 if max_q == 1 else 16)


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("kind", range(len(KINDS)))
@pytest.mark.parametrize("ct,dtype,D,page", [(E4M3, BF16, 128, 64), (I8, F16, 64, 16), (E4M3, F16, 64, 32), (I8, BF16, 128, 128)])
def test_kinds(cuda, max_q, kind, ct, dtype, D, page):
    H = heads(max_q)
    kw = with_params(KINDS[kind], H)
    c = make(SIZES, BASES, H=H, D=D, page=page, ct=ct, dtype=dtype, seed=kind)
    check(c, run(c, max_q=max_q, **kw), **kw)


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("kind", [0, 2])
@pytest.mark.parametrize("page", [16, 64])
def test_masks(cuda, max_q, mask, kind, page):
    H = heads(max_q)
    kw = with_params(KINDS[kind], H)
    c = make([13, 64, 3, 40], [50, 20, 5, 130], H=H, page=page, seed=mask)
    if kind == 0:
        got, lse = run(c, max_q=max_q, mask=MASKS[mask], return_lse=True, **kw)
    else:
        got, lse = run(c, max_q=max_q, mask=MASKS[mask], **kw), None
    check(c, got, lse, mask=MASKS[mask], **kw)


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("shape", ["tree", "chain", "wide"])
@pytest.mark.parametrize("H,hkv", [(4, 4), (8, 1), (14, 2), (6, 2)])
def test_shapes(cuda, max_q, shape, H, hkv):
    c = make([64, 33, 1, 32, 63], [0, 31, 700, 33, 15], H=H, hkv=hkv, page=32, shape=shape, seed=H)
    got = run(c, max_q=max_q)
    check(c, got)
    if shape == "chain":  # in a row they are what drafted tokens are without a tree
        d = [c[n].cuda() for n in ("k", "v", "ks", "vs")]
        plain = cp.paged_attention(c["q"].cuda(), *d, ints(c["table"]), ints(c["lens"]), ints(c["cu"]), max_q=max_q)
        check(c, plain)


@pytest.mark.parametrize("max_q", [1, 64])
def test_long_contexts_are_split(cuda, max_q):
    """Units that several CTAs share, trees at the end of the last one's piece, and in pages that end inside a tile."""
    c = make([64, 7, 25], [9000, 4099, 1], H=heads(max_q), hkv=2, page=16, seed=3)
    got, lse = run(c, max_q=max_q, return_lse=True)
    check(c, got, lse)


@pytest.mark.parametrize("max_q", [1, 64])
def test_chunks_beside_trees(cuda, max_q):
    """A request of more than 64 queries is a chunk of a prompt."""
    c = make([5, 65, 20, 130], [40, 10, 0, 77], H=heads(max_q), seed=9)
    check(c, run(c, max_q=max_q, mask=cp.Mask(left=50, right=0)), mask=cp.Mask(left=50, right=0))
    check(c, run(c, max_q=max_q))


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("mask", [cp.Mask(right=0, prefix=38), cp.Mask(left=12, right=0, prefix=38, dilation=3),
                                  cp.Mask(left=10, right=0, prefix=60), cp.Mask(left=5, right=9), cp.FULL])
@pytest.mark.parametrize("sizes,bases", [([90, 5], [1, 40]), ([5, 65, 20, 130], [40, 10, 0, 0])])
def test_chunks_beside_trees_see_what_follows(cuda, max_q, mask, sizes, bases):
    """A chunk that begins inside the prefix sees all of it, with a mask that shows later keys also those: what the call
    without trees gives it."""
    c = make(sizes, bases, H=heads(max_q), page=32, seed=5)
    got, lse = run(c, max_q=max_q, mask=mask, return_lse=True)
    check(c, got, lse, mask=mask)


@pytest.mark.parametrize("max_q", [1, 64])
def test_more_nodes_than_keys(cuda, max_q):
    """Lengths that do not hold the tree: the first nodes have no place in the cache, and none for a first node's row."""
    c = make([10, 6, 3], [-4, -6, 20], H=heads(max_q), seed=2, shape="chain")
    got, lse = run(c, max_q=max_q, return_lse=True)
    check(c, got, lse)
    assert not got[10:16].float().any()


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("B", [513, 1100])
def test_many_requests(cuda, max_q, B):
    H = 2 if max_q == 1 else 32
    c = make([1 + i % 4 for i in range(B)], [(7 * i) % 40 for i in range(B)], H=H, hkv=1, D=64, page=16, seed=B)
    check(c, run(c, max_q=max_q))


@pytest.mark.parametrize("max_q", [1, 64])
@pytest.mark.parametrize("kind", [0, 4])
def test_nan_of_nodes_that_are_not_seen(cuda, max_q, kind):
    """NaN values (e4m3) in a node's place reach those that see it, and nobody else; scales of places that no row sees
    may be anything."""
    kw = KINDS[kind]
    H = heads(max_q)
    c = make([20, 9], [45, 3], H=H, page=16, seed=6)
    base, page = 45, 16
    seen = do.paths(c["parents"][:20])
    node = 11
    p, o = c["table"][0][(base + node) // page], (base + node) % page
    clean = run(c, max_q=max_q, **kw)
    c["v"].view(torch.uint8)[p, 0, o, 3] = 0x7f
    got = run(c, max_q=max_q, **kw)
    hit = torch.tensor([node in s for s in seen] + [False] * 9)
    assert hit.any() and not hit.all()
    assert got.cpu()[hit][:, :H // 2, 3].isnan().all()
    keep = torch.ones_like(got, dtype=torch.bool).cpu()
    keep[hit.nonzero().flatten(), :H // 2, 3] = False
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])


@pytest.mark.parametrize("max_q", [1, 64])
def test_bad_pages_and_offsets(cuda, max_q):
    H = heads(max_q)
    c = make([13, 4], [50, 30], H=H, page=16, seed=4)
    clean = run(c, max_q=max_q)
    c["table"][1][1] = 10 ** 6  # keys 16 .. 31 of the second request are left out
    got = run(c, max_q=max_q)
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)
    assert torch.equal(got[:13], clean[:13]) and got.isfinite().all()
    c["table"][1][1] = 0
    tree = cp.tree_tables(ints(c["parents"]), ints(c["cu"]), ints(c["lens"]))
    c["cu"] = [0, 13, 12]
    out = torch.full((17, H, 128), 5.0, dtype=BF16, device="cuda")
    got = run(c, tree=tree, max_q=max_q, out=out)
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)
    check(dict(c, cu=[0, 13, 17]), got, rows=slice(0, 13))  # (fewer requests are cut into other pieces: not bit by bit)
    assert (got[13:] == 5).all()  # rows that nobody owns stay


@pytest.mark.parametrize("max_q", [1, 64])
def test_words_of_any_kind(cuda, max_q):
    """Positions out of range and words with any bits: the result may be anything, but memory is not left, and what the
    bits beyond the tree say is not looked at."""
    c = make([9, 64], [20, 100], H=heads(max_q), seed=12)
    tree = cp.tree_tables(ints(c["parents"]), ints(c["cu"]), ints(c["lens"]))
    want = run(c, tree=tree, max_q=max_q)
    more = tree._replace(ancestors=tree.ancestors.clone())
    more.ancestors[:9] |= -1 << 9
    assert torch.equal(run(c, tree=more, max_q=max_q), want)
    wild = tree._replace(positions=torch.where(tree.positions % 2 == 0, -2 ** 31, 2 ** 31 - 1).int(),
                         ancestors=torch.full_like(tree.ancestors, -1))
    for kw in (dict(), dict(mod="alibi", head_param=[0.5] * c["q"].shape[1]), dict(mask=cp.Mask(left=3, right=0, dilation=2))):
        assert run(c, tree=wild, max_q=max_q, **kw).shape == want.shape
    only = torch.arange(9).tolist() + torch.arange(64).tolist()  # nodes that see themselves and the context alone
    alone = tree._replace(ancestors=torch.tensor([1 << i if i < 63 else -2 ** 63 for i in only], device="cuda"),
                          positions=ints([20] * 9 + [100] * 64))
    check(dict(c, parents=[-1] * 73), run(c, tree=alone, max_q=max_q))


@pytest.mark.parametrize("max_q", [1, 64])
def test_trees_of_one_size_without_offsets(cuda, max_q):
    c = make([12] * 5, [7, 0, 300, 64, 31], H=heads(max_q), seed=15)
    d = [c[n].cuda() for n in ("k", "v", "ks", "vs")]
    tree = cp.tree_tables(ints(c["parents"]), ints(c["cu"]), ints(c["lens"]))
    q = c["q"].cuda().repeat_interleave(2, 0)[::2]  # (rows with a stride)
    out = torch.zeros(60, 2 * q.shape[1], 128, dtype=BF16, device="cuda")[:, ::2]
    got = cp.paged_attention(q, *d, ints(c["table"]), ints(c["lens"]), tree=tree, out=out, max_q=max(max_q, 12))
    assert got.data_ptr() == out.data_ptr()
    check(c, got)


def test_refusals(cuda):
    c = make([4, 3], [10, 20], seed=1)
    tree = cp.tree_tables(ints(c["parents"]), ints(c["cu"]), ints(c["lens"]))
    for bad in (tree.positions, (tree.positions,), tree._replace(positions=tree.positions[:5]),
                tree._replace(positions=tree.ancestors), tree._replace(ancestors=tree.positions),
                tree._replace(ancestors=tree.ancestors[:-1]), tree._replace(ancestors=tree.ancestors.repeat(2)[::2]),
                tree._replace(ancestors=tree.ancestors.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            run(c, tree=bad)


def test_streams_and_graphs(cuda):
    """Two streams at once, and a captured step that is replayed on new trees."""
    c = make([13, 40, 2], [300, 20, 0], H=32, seed=8)
    d = [c[n].cuda() for n in ("k", "v", "ks", "vs")]
    q, table, lens, cu, parents = c["q"].cuda(), ints(c["table"]), ints(c["lens"]), ints(c["cu"]), ints(c["parents"])

    def step():
        tree = cp.tree_tables(parents, cu, lens)
        return [cp.paged_attention(q, *d, table, lens, cu, max_q=m, tree=tree) for m in (1, 64)]

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([step() for _ in range(3)])
    torch.cuda.synchronize()
    for runs in got:
        for r in runs:
            assert torch.equal(r[0], want[0]) and torch.equal(r[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = [p for i, n in enumerate([13, 40, 2]) for p in do.tree(n, 77 + i)]
    parents.copy_(ints(other))
    lens.copy_(ints([250, 60, 2]))
    graph.replay()
    again = step()
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
    check(dict(c, parents=other, lens=[250, 60, 2]), out[0])


@pytest.mark.parametrize("ct,page,dtype", [(E4M3, 16, BF16), (I8, 64, F16)])
def test_steps_of_speculative_decoding(cuda, ct, page, dtype):
    """Three steps of all operators together. After each, the pages that requests hold and the free ones are all there
    is; the cache holds what appending the accepted tokens alone would have left, to the cache's precision."""
    H, hkv, D, V, B, pages = 16, 2, 64, 300, 5, 60  # (the kernel of few queries in the second step)
    g = torch.Generator().manual_seed(page)
    cache = cp.new_cache(pages, hkv, D, page_size=page, dtype=ct)
    table, ring = ints([[0] * 12] * B), torch.arange(pages, dtype=torch.int32, device="cuda")
    state, lens = ints([0, pages]), ints([0] * B)
    freqs = cp.rope_frequencies(D)
    qw, kw = (torch.ones(D, dtype=dtype, device="cuda") for _ in range(2))
    known = [[] for _ in range(B)]  # K and V of each request's tokens, normed and turned, in 16 bits
    for it, sizes in enumerate([[64, 1, 20, 0, 33], [13, 25, 7, 9, 1], [30, 30, 30, 30, 30]]):
        T = sum(sizes)
        cu = [sum(sizes[:i]) for i in range(B + 1)]
        parents = [p for i, n in enumerate(sizes) for p in do.tree(n, 10 * it + i)]
        qkv = torch.randn(T, H + 2 * hkv, D, generator=g).to(dtype).cuda()
        q, k, v = qkv.split([H, hkv, hkv], 1)
        st = cp.page_tables(lens, ints(sizes), table, ring, state, page_size=page, max_tokens=T)
        tree = cp.tree_tables(ints(parents), st.cu_q, st.seq_lens)
        q, k = cp.qk_norm_rope(q, k, qw, kw, freqs, tree.positions)
        cp.cache_append(k, v, st.slots, *cache)
        got = cp.paged_attention(q, *cache, table, st.seq_lens, st.cu_q, max_q=max(sizes), tree=tree)
        c = dict(q=q.cpu(), k=cache[0].cpu(), v=cache[1].cpu(), ks=cache[2].cpu(), vs=cache[3].cpu(), table=table.tolist(),
                 lens=st.seq_lens.tolist(), cu=cu, parents=parents)
        assert st.cu_q.tolist() == cu
        check(c, got)
        p = torch.softmax(2 * torch.randn(T, V, generator=g), 1)
        d = torch.softmax(p.log() + 0.3 * torch.randn(T, V, generator=g), 1)
        tokens, u = [0] * T, torch.rand(T, generator=g)
        for b in range(B):
            left = {}
            for i in range(sizes[b]):
                up = parents[cu[b] + i]
                if up >= 0:
                    row = left.setdefault(up, d[cu[b] + up].clone())
                    tokens[cu[b] + i] = int(torch.multinomial(row, 1, generator=g))
                    row[tokens[cu[b] + i]] = 0
        done = cp.verify_drafts(p.cuda(), ints(tokens), ints(parents), st.cu_q, u.cuda(), draft_probs=d.cuda(), max_tokens=9)
        counts, toks, path = do.verify(p, tokens, parents, cu, u, d, 9)
        assert done.counts.tolist() == counts and done.tokens.tolist() == toks and done.path.tolist() == path
        keep = cp.cache_compact(done.path, done.counts, st.cu_q, st.seq_lens, table, *cache)
        before = lens.tolist()
        assert keep.tolist() == [n + m for n, m in zip(before, counts)]
        lens, state = cp.release_pages(None, st.seq_lens, table, ring, st.free_state, page_size=page, keep_lens=keep)
        assert lens.tolist() == keep.tolist()
        held = [x for b in range(B) for x in table[b, :po.pages_for(int(lens[b]), page)].tolist()]
        first, count = state.tolist()
        free = [int(ring[(first + i) % pages]) for i in range(count)]
        assert sorted(held + free) == list(range(pages))
        for b in range(B):
            rows = [cu[b] + x for x in path[b][:counts[b]]]
            known[b] += [(k[r].double().cpu(), v[r].double().cpu()) for r in rows]
            if not known[b]:
                continue
            at = torch.arange(len(known[b]))
            pg = table[b].cpu()[at // page].long()
            for x, (codes, scale) in enumerate(((cache[0], cache[2]), (cache[1], cache[3]))):
                s = scale.double().cpu()[pg][:, :, None]  # [n, heads, 1]
                have = codes.double().cpu()[pg, :, at % page] * s
                want = torch.stack([kv[x] for kv in known[b]])
                # each of up to four roundings (appended, expressed in a larger scale, moved, expressed again) is off by
                # half a step: int8 0.5 of the scale; e4m3 2^-4 of the value, or 2^-10 of the scale where it is subnormal
                step = 0.5 * s if ct == I8 else torch.maximum(want.abs() * 2.0 ** -4, s * 2.0 ** -10)
                assert ((have - want).abs() <= 4.6 * step).all()


def test_wide_tables(cuda):
    """Tables of a million tokens for 4096 requests, whose line of key tiles fits 32 bits in units of 256 rows only. The
    lengths are short, so the answer is that with the tables' first columns, from the other kernel; both within the
    tolerance above, that is within twice of it of one another (mass: at most the largest value, since the weights' sum is
    1)."""
    g = torch.Generator().manual_seed(5)
    B, n, H, hkv, D, page = 4096, 8, 64, 8, 64, 64
    sizes = [(64 if b % 97 == 0 else 1 + b % 8) for b in range(B)]
    cu = [0]
    for m in sizes:
        cu.append(cu[-1] + m)
    T = max(cu[-1], B * n)  # (rows behind the last request)
    lens = [m + b % 50 for b, m in enumerate(sizes)]
    parents = [i - 1 if i < 2 else i - 2 for m in sizes for i in range(m)]
    table = torch.full((B, 16384), -1, dtype=torch.int32, device="cuda")
    table[:, :2] = torch.randint(0, 40, (B, 2), generator=g).to(torch.int32).cuda()
    q = torch.randn(T, H, D, generator=g).to(BF16).cuda()
    cache = [torch.randn(40, hkv, page, D, generator=g).mul(100).clamp(-448, 448).to(E4M3).cuda() for _ in range(2)]
    scale = torch.full((40, hkv), 2.0 ** -7, device="cuda")
    lens, cu = ints(lens), ints(cu)
    tree = cp.tree_tables(torch.nn.functional.pad(ints(parents), (0, T - len(parents))), cu, lens)
    with torch.no_grad():
        wide = cp.paged_attention(q, *cache, scale, scale, table, lens, cu, max_q=64, tree=tree)
        near = cp.paged_attention(q, *cache, scale, scale, table[:, :2].contiguous(), lens, cu, max_q=64, tree=tree)
    rows = int(cu[-1])
    top = 448 * 2.0 ** -7
    err = (wide[:rows].float() - near[:rows].float()).abs()
    assert (err <= 2.0 ** -7 * near[:rows].float().abs() + 2.0 ** -9 * top).all()


def test_a_step_with_chunks_and_trees(cuda):
    """Trees first, chunks of prompts behind them: one call for all where they are alike, and the trees' part of the tables
    for the verification and the compaction."""
    g = torch.Generator().manual_seed(11)
    H, hkv, D, V, page, pages = 8, 2, 64, 200, 16, 60
    sizes, drafted = [13, 5, 40, 90], 2  # two trees; chunks of 40 and of 90 tokens
    B, T, n = len(sizes), sum(sizes), sum(sizes[:2])
    cache = cp.new_cache(pages, hkv, D, page_size=page)
    table, ring = ints([[0] * 12] * B), torch.arange(pages, dtype=torch.int32, device="cuda")
    lens, state = ints([0] * B), ints([0, pages])
    for it in range(2):
        cu = [sum(sizes[:i]) for i in range(B + 1)]
        parents = [p for i in range(drafted) for p in do.tree(sizes[i], 10 * it + i)]
        parents += [i - 1 for m in sizes[drafted:] for i in range(m)]  # (a chunk of up to 64 tokens is a row)
        q, k, v = torch.randn(T, H + 2 * hkv, D, generator=g).to(BF16).cuda().split([H, hkv, hkv], 1)
        before = lens.tolist()
        st = cp.page_tables(lens, ints(sizes), table, ring, state, page_size=page, max_tokens=T)
        tree = cp.tree_tables(ints(parents), st.cu_q, st.seq_lens)
        cp.cache_append(k, v, st.slots, *cache)
        got = cp.paged_attention(q, *cache, table, st.seq_lens, st.cu_q, max_q=max(sizes), tree=tree)
        c = dict(q=q.cpu(), k=cache[0].cpu(), v=cache[1].cpu(), ks=cache[2].cpu(), vs=cache[3].cpu(), table=table.tolist(),
                 lens=st.seq_lens.tolist(), cu=cu, parents=parents)
        check(c, got)
        p = torch.softmax(torch.randn(n, V, generator=g), 1)
        tokens, u = torch.randint(0, V, (n,), generator=g).tolist(), torch.rand(n, generator=g)
        part = st.cu_q[:drafted + 1]
        done = cp.verify_drafts(p.cuda(), ints(tokens), ints(parents[:n]), part, u.cuda(), max_tokens=9)
        counts, toks, path = do.verify(p, tokens, parents[:n], cu[:drafted + 1], u, None, 9)
        assert done.counts.tolist() == counts and done.tokens.tolist() == toks and done.path.tolist() == path
        keep = cp.cache_compact(done.path, done.counts, part, st.seq_lens[:drafted], table[:drafted], *cache, st.slots)
        keep = torch.cat([keep, st.seq_lens[drafted:]])
        lens, state = cp.release_pages(None, st.seq_lens, table, ring, st.free_state, page_size=page, keep_lens=keep)
        assert lens.tolist() == [b + (counts[i] if i < drafted else sizes[i]) for i, b in enumerate(before)]
