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
