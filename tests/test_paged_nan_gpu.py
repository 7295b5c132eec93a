"""NaN in a value (e4m3) that some rows see and others do not, in both attention kernels of the paged 8-bit K/V cache.

Expected, from the definition: NaN in that channel of every row that sees the key, whatever its weight, and nothing else
changes. The kernels take NaN out of the tiles that are not visible as a whole, so that the rows that do not see it have
the very bits that they have with a zero in its place; those are compared with the 64-bit oracle beside it, within
the tolerance derived in ``test_paged_gpu.py``."""

import pytest
import torch

import chia_proj_b200 as cp
import paged_oracle as po
from test_paged_gpu import BF16, E4M3, F16, ints, kind_args, setup

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def sees(i, j, mask):
    return j < mask.prefix or ((mask.left < 0 or i - j <= mask.left) and (mask.right < 0 or j - i <= mask.right)
                               and (not mask.block or i // mask.block == j // mask.block) and (i - j) % mask.dilation == 0)


def check(lens, counts, H, hkv, D, page, dtype, spots, kind="plain", mask=cp.CAUSAL, max_q=None, exact=True):
    """spots: (request, key, K/V head, channel) whose value is NaN."""
    q, k, v, ks, vs, table, cu = setup(lens, counts, H, hkv, D, page, E4M3, dtype, 11)
    kw = kind_args(kind, H)
    raw = v.view(torch.uint8)

    def run(byte):
        for b, j, h, c in spots:
            raw[table[b][j // page], h, j % page, c] = byte
        return cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu), max_q=max_q, mask=mask, **kw)

    zero = run(0)
    got = run(0x7f)
    want = zero.clone()
    g, some = H // hkv, 0
    for b, j, h, c in spots:
        for t in range(cu[b], cu[b + 1]):
            if sees(lens[b] - counts[b] + t - cu[b], j, mask):
                want[t, h * g:(h + 1) * g, c] = float("nan")
                some += 1
    assert some > 0
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    run(0)
    if exact:
        out, _, mass = po.attention(q.cpu(), k.cpu(), v.cpu(), ks.cpu(), vs.cpu(), table, lens, cu, mask=mask, **kw)
        err = (zero.double().cpu() - out).abs()
        assert (err <= 2.0 ** (-8 if dtype == BF16 else -11) * out.abs() + 2.0 ** -10 * mass + 2.0 ** -23).all()


MASKS = {"causal": cp.CAUSAL, "window": cp.Mask(left=60, right=0), "dilated": cp.Mask(left=-1, right=0, dilation=3),
         "all": cp.Mask(left=200, right=1, block=192, prefix=20, dilation=2)}


@pytest.mark.parametrize("name", list(MASKS))
@pytest.mark.parametrize("kind", ["plain", "alibi", "relu", "sigmoid"])
@pytest.mark.parametrize("counts", [[1, 4], [7, 20], [90, 130]])
def test_a_visible_nan(cuda, counts, kind, name):
    """Few rows and many; the NaN beside the diagonal, at a tile's ends, in the prefix, at the last key."""
    lens = [333, 400]
    spots = [(0, 333 - counts[0], 0, 5), (0, 330, 1, 127), (1, 0, 0, 64), (1, 399 - counts[1] // 2, 1, 31), (1, 383, 0, 32),
             (0, 332, 0, 0)]
    check(lens, counts, 8, 2, 128, 32, BF16, spots, kind, MASKS[name])
    check(lens, counts, 4, 2, 64, 16, F16, [(b, j, h, c % 64) for b, j, h, c in spots], kind, MASKS[name])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_nan_in_front_of_short_units(cuda, dtype):
    """Runs of 300 rows a K/V head: units of 256 rows, whose second half is slow where it looks for a NaN, and units of 44
    rows and dozens of tiles behind them, in which that half has no rows."""
    B = 40
    lens = [1100 + 37 * b for b in range(B)]
    spots = [(b, lens[b] - 180, b % 4, (7 * b) % 128) for b in range(0, B, 3)]
    check(lens, [300] * B, 4, 4, 128, 64, dtype, spots, max_q=300)
    check(lens, [300] * B, 4, 4, 64, 128, dtype, [(b, j, h, c % 64) for b, j, h, c in spots], "relu", max_q=300, exact=False)


def test_units_of_few_rows_behind_full_ones(cuda):
    """Without NaN: two query tiles, then one, over and over, against the kernel for few rows."""
    B, H, D, page = 64, 2, 128, 64
    lens = [700 + 61 * b for b in range(B)]
    counts = [256 + 1 + 2 * b for b in range(B)]
    q, k, v, ks, vs, table, cu = setup(lens, counts, H, H, D, page, E4M3, BF16, 12)
    a, b = (cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu), max_q=m).double() for m in (400, 1))
    assert ((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -9 * b.abs().amax(-1, keepdim=True)).all()
