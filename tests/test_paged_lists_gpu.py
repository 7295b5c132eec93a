"""paged_attention where the lists that only the GPU sees are wrong: offsets that fall, pages that are not there. Nothing
outside the tensors is touched, the status word tells, and what is still defined is right."""

import pytest
import torch

import chia_proj_b200 as cp
import paged_oracle as po
from test_paged_gpu import BF16, E4M3, F16, I8, ints, kind_args, make_cache, setup  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def reported():
    with pytest.raises(cp.ChiaError, match="BAD_INDEX"):
        cp.check_device_status(0)


@pytest.mark.parametrize("counts", [[1, 2, 1, 3, 1], [90, 70, 1, 130, 2]])
def test_requests_behind_a_falling_offset(cuda, counts):
    """The requests before it are served, those behind it are not: their rows are not written."""
    lens = [200, 333, 70, 250, 90]
    q, k, v, ks, vs, table, cu = setup(lens, counts, 8, 2, 128, 32, E4M3, BF16)
    run = lambda c, out: cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(c), out=out)  # noqa: E731
    good = cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu)).double()
    for b, bad in ((3, 0), (3, -1), (1, 2 ** 31 - 1), (5, cu[5] + 1), (0, -2 ** 31)):
        c = list(cu)
        c[b] = bad
        first = min(i for i in range(5) if not 0 <= c[i] <= c[i + 1] <= cu[5])
        out = torch.full_like(q, 7.0)
        run(c, out)
        reported()
        a, w = out[:cu[first]].double(), good[:cu[first]]  # (another schedule: near, not equal)
        assert first == 0 or ((a - w).abs() <= 2.0 ** -7 * w.abs() + 2.0 ** -9 * w.abs().amax()).all()
        assert (out[cu[first]:] == 7).all()


def test_offsets_that_overlap_do_not_outgrow_the_line(cuda):
    """256 requests that all claim all rows, over 4 million keys each: their tiles would not be counted in 32 bits, though
    the rows and the table allow for the call. The first is served, as it is alone."""
    B, T, hkv, D, page, W = 512, 64, 8, 64, 128, 32800
    tiles = W * page // 32
    assert 256 * 8 * hkv * (tiles + 4) > 2 ** 31 > hkv * (T // 8 + B + 1) * (tiles + 6)
    g = torch.Generator().manual_seed(3)
    k, v, ks, vs = make_cache(300, hkv, page, D, E4M3, g)
    q = torch.randn(T, hkv, D, generator=g).to(BF16).cuda()
    table = torch.randint(0, 300, (1, W), generator=g, dtype=torch.int32).cuda()
    lens = ints([W * page] * B)
    out = torch.full_like(q, 7.0)
    cp.paged_attention(q, k, v, ks, vs, table.repeat(B, 1), lens, ints([0, T] * (B // 2) + [0]), max_q=1, out=out)
    reported()
    assert torch.equal(out, cp.paged_attention(q, k, v, ks, vs, table, lens[:1], ints([0, T]), max_q=1))


def attention_without(q, k, v, ks, vs, table, lens, cu, gone, mask, norm="softmax", mod="none", head_param=None, softcap=30.0,
                      sig_bias=0.0, out_scale=1.0):
    """64-bit (out, lse, mass) over the keys that are in pages of the cache; gone(page)."""
    T, H, D = q.shape
    hkv, page = k.shape[1:3]
    out, mass = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -float("inf"), dtype=torch.float64)
    for b, n in enumerate(lens):
        pages = torch.tensor(table[b][:po.pages_for(n, page)])
        there = torch.tensor([not gone(int(p)) for p in pages])
        pg = torch.where(there, pages, 0)
        kk, vv = ((x[pg].double() * s[pg].double()[:, :, None, None]).transpose(0, 1).reshape(hkv, -1, D)[:, :n]
                  for x, s in ((k, ks), (v, vs)))
        i, j = torch.arange(n - (cu[b + 1] - cu[b]), n)[:, None], torch.arange(n)[None]
        see = torch.ones(i.shape[0], n, dtype=torch.bool)
        see &= (i - j <= mask.left) if mask.left >= 0 else True
        see &= (j - i <= mask.right) if mask.right >= 0 else True
        see &= (i - j) % mask.dilation == 0
        see |= j < mask.prefix
        see &= there.repeat_interleave(page)[None, :n]
        for h in range(H):
            x = q[cu[b]:cu[b + 1], h].double() @ kk[h * hkv // H].T / D ** 0.5
            if mod == "softcap":
                x = softcap * torch.tanh(x / softcap)
            if mod == "alibi":
                x = x + float(head_param[h]) * (j - i)
            if mod == "temp":
                x = x * float(head_param[h])
            if norm == "softmax":
                x = x.masked_fill(~see, -float("inf"))
                lse[cu[b]:cu[b + 1], h] = torch.logsumexp(x, 1)
                p = torch.nan_to_num(torch.softmax(x, 1))
            else:
                p = torch.where(see, torch.sigmoid(x + sig_bias) if norm == "sigmoid" else x.clamp(min=0) * out_scale, 0.0)
            val = torch.nan_to_num(vv[h * hkv // H])
            out[cu[b]:cu[b + 1], h], mass[cu[b]:cu[b + 1], h] = p @ val, p.abs() @ val.abs()
    return out, lse, mass


@pytest.mark.parametrize("kind", ["plain", "softcap", "alibi", "temp", "sigmoid", "relu"])
@pytest.mark.parametrize("D,dtype,ct,page", [(128, BF16, E4M3, 16), (64, F16, I8, 64), (64, BF16, E4M3, 32),
                                             (128, F16, E4M3, 128), (128, BF16, I8, 16)])
def test_pages_out_of_range_are_skipped(cuda, kind, D, dtype, ct, page):
    """A page that is not there is as if its keys were masked, whatever an earlier call left in shared memory (here:
    NaN, or the largest bytes). All pages of a request; pages in the middle, at both ends and at the diagonal."""
    H, hkv = 8, 2
    kw = kind_args(kind, H)
    for lens, counts, bad in (([700, 33, 300], [1, 2, 1], {0: (0, 3, 4), 1: (0,), 2: (1,)}),
                              ([700, 90, 400], [150, 70, 3], {0: (0, 2, 3), 1: range(9), 2: (1, 2)})):
        q, k, v, ks, vs, table, cu = setup(lens, counts, H, hkv, D, page, ct, dtype, 5)
        dirty = [torch.full_like(x.view(torch.uint8), 0x7f).view(ct) for x in (k, v)]
        tables = [list(r) for r in table]
        for b, at in bad.items():
            for p in at:
                if p < po.pages_for(lens[b], page):
                    tables[b][p] = (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31)[p % 4]
        for b, n in enumerate(lens):
            if page >= 64 and b == 0:
                tables[b][po.pages_for(n, page) - 1] = -7  # beside the newest tokens
        args = (ints(lens), ints(cu))
        for mask in (cp.CAUSAL, cp.Mask(left=210, right=0, prefix=40), cp.Mask(left=-1, right=0, dilation=3)):
            cp.paged_attention(q, *dirty, ks.clamp(-1, 1), vs.clamp(-1, 1), ints(table), *args, mask=cp.FULL)
            got = cp.paged_attention(q, k, v, ks, vs, ints(tables), *args, mask=mask, return_lse=kind not in ("relu", "sigmoid"), **kw)
            reported()
            got, lse = got if isinstance(got, tuple) else (got, None)
            out, want_lse, mass = attention_without(q.cpu(), k.cpu(), v.cpu(), ks.cpu(), vs.cpu(), tables, lens, cu,
                                                    lambda p: not 0 <= p < k.shape[0], mask, **kw)
            err = (got.double().cpu() - out).abs()
            assert torch.isfinite(got).all()
            # (the tolerance is derived in test_paged_gpu.py)
            assert (err <= 2.0 ** (-8 if dtype == BF16 else -11) * out.abs() + 2.0 ** -10 * mass + 2.0 ** -23).all()
            if lse is not None:
                none = torch.isinf(want_lse)
                assert torch.equal(torch.isinf(lse.cpu()), none)
                assert ((lse.double().cpu() - want_lse).abs()[~none] <= 2.0 ** -12).all()


@pytest.mark.parametrize("counts", [[1, 1], [100, 90]])
def test_nan_beside_a_page_out_of_range(cuda, counts):
    """A NaN that rows see, in a tile that all rows would see as a whole if its first page were there."""
    lens = [400, 300]
    q, k, v, ks, vs, table, cu = setup(lens, counts, 4, 2, 128, 16, E4M3, BF16, 6)
    table[0][4] = -1  # keys 64 to 79
    run = lambda: cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu))  # noqa: E731
    raw = v.view(torch.uint8)
    raw[table[0][5], 1, 3, 77] = 0
    want = run().clone()
    raw[table[0][5], 1, 3, 77] = 0xff
    got = run()
    reported()
    want[:cu[1], 2:, 77] = float("nan")
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("counts", [[1, 3], [120, 100]])
def test_pages_that_no_query_sees_may_be_anything(cuda, counts, page):
    """A window has moved on and its old pages are given back: their entries are no pages any more. Nothing is reported,
    and no bit changes."""
    lens, mask = [1037, 796], cp.Mask(left=37, right=0, prefix=1)  # first keys of the windows amid a tile
    q, k, v, ks, vs, table, cu = setup(lens, counts, 8, 2, 64, page, E4M3, BF16, 7)
    run = lambda: cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu), mask=mask)  # noqa: E731
    want = run()
    for b, n in enumerate(lens):
        for p in range(1, (n - counts[b] - 37) // page):
            table[b][p] = (-1, 2 ** 31 - 1, k.shape[0])[p % 3]
    assert torch.equal(run(), want)
