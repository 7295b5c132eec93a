"""Masks of paged_attention at positions beyond 2^30, where sums of a position and a mask's width leave 32 bits.

A table of eight million entries names three pages over and over: one whose keys score 0, one whose keys score so low that
a billion of them weigh nothing, and one for the newest tokens. The log-sum-exp is then the logarithm of a small count of
visible keys, which the mask's definition gives."""

import math

import pytest
import torch

import chia_proj_b200 as cp
from test_paged_gpu import BF16, E4M3, ints

pytestmark = pytest.mark.gpu
PAGE, D = 128, 64
LEN = 2 ** 30 + 200  # the last query is at 2^30 + 199


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


MASKS = {
    "left": cp.Mask(left=2 ** 30 + 120, right=0), "left past all": cp.Mask(left=2 ** 31 + 5, right=0),
    "right": cp.Mask(left=60, right=2 ** 30), "right past all": cp.Mask(left=3, right=2 ** 40),
    "block": cp.Mask(left=-1, right=0, block=2 ** 30 + 64), "block past all": cp.Mask(left=100, right=0, block=2 ** 33),
    "dilation": cp.Mask(left=-1, right=0, dilation=2 ** 30 + 190), "prefix": cp.Mask(left=0, right=0, prefix=2 ** 35),
}


@pytest.mark.parametrize("count", [1, 90])
@pytest.mark.parametrize("name", list(MASKS))
def test_masks_beyond_30_bits(cuda, name, count):
    m = MASKS[name]
    k = torch.zeros(3, 1, PAGE, D, dtype=torch.uint8, device="cuda").view(E4M3)
    v = torch.ones(3, 1, PAGE, D, device="cuda").to(E4M3)
    k[1] = torch.tensor(-448.0).to(E4M3)
    scales = torch.ones(3, 1, device="cuda")
    W = LEN // PAGE + 1
    table = torch.ones(1, W, dtype=torch.int32, device="cuda")
    table[0, 0], table[0, -2:] = 0, 2  # keys 0 to 127, and those from 2^30 on
    q = torch.full((count, 1, D), 1.0 / 8, dtype=BF16, device="cuda")  # low ones score -448
    out, lse = cp.paged_attention(q, k, v, scales, scales, table, ints([LEN]), ints([0, count]), max_q=count, mask=m,
                                  return_lse=True)
    near = [*range(128), *range(2 ** 30, LEN)]
    for t in range(count):
        i = LEN - count + t
        n = sum(j < m.prefix or ((m.left < 0 or i - j <= m.left) and (m.right < 0 or j - i <= m.right)
                                 and (not m.block or i // m.block == j // m.block) and (i - j) % m.dilation == 0) for j in near)
        assert n > 0 and abs(float(lse[t, 0]) - math.log(n)) < 2.0 ** -12, (t, n, float(lse[t, 0]))
    assert (out == 1).all()
