"""Attention under masks whose numbers lie beyond any position: as if they were at the last one.

A row that sees its own key alone has P = 1 (to 2^-12 in the kernels' halves), so its output is its value to the rounding of
the output (2^-8 relative in bf16, 2^-11 in fp16) and of P; 2^-7 and 2^-10 |v| are allowed. Its gradients are dv = dout
likewise, and dq = dk = 0: what is left of (dP - delta) is two fp32 sums of D products (2^-17 of some 100) and the output's
rounding in one of them (2^-9 of some 100), times keys of up to 5 and the scale 2^-3: 2^-2 is allowed where values are of
the order of one, and nothing that a second visible key gave (a term of dP itself, 10 or more) fits in it."""

import pytest
import torch

import chia_proj_b200 as cp
import paged_oracle as po
import test_tree_attn_gpu as ta

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
FAR = [2 ** 30, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 3 * 2 ** 31, 2 ** 63 - 1]


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def draw(S, D, dtype, seed, B=1, H=2, Sq=None):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(B, H, n, D, generator=g).to(dtype).cuda() for n in (Sq or S, S, S)]


@pytest.mark.parametrize("dilation", FAR)
@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (128, F16)])
def test_dilations(cuda, D, dtype, dilation):
    q, k, v = draw(300, D, dtype, 1)
    rel = 2.0 ** -7 if dtype == BF16 else 2.0 ** -10
    for mask in (cp.Mask(left=-1, right=0, dilation=dilation), cp.Mask(dilation=dilation), cp.Mask(left=7, right=7, dilation=dilation)):
        out = cp.attention(q, k, v, mask=mask)
        assert ((out - v).abs().float() <= rel * v.abs().float()).all()
    # behind a prefix that all rows see, and with few queries: as a dilation that is too large for these lengths already
    for a, kw in ((q, {}), (q[:, :, 100:110], {}), (q[:, :, 100:110], dict(split_kv=False))):
        far, near = (cp.attention(a, k, v, mask=cp.Mask(left=-1, right=0, prefix=9, dilation=d), **kw) for d in (dilation, 301))
        assert torch.equal(far, near)


@pytest.mark.parametrize("dilation", FAR)
@pytest.mark.parametrize("D", [64, 128])
def test_dilations_backward(cuda, D, dilation):
    q, k, v = (t.requires_grad_() for t in draw(300, D, BF16, 2))
    dout = torch.randn(v.shape, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    out = cp.attention(q, k, v, mask=cp.Mask(left=-1, right=0, dilation=dilation))
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    assert ((dv - dout).abs().float() <= 2.0 ** -7 * dout.abs().float()).all()
    assert dq.abs().max() <= 0.25 and dk.abs().max() <= 0.25


@pytest.mark.parametrize("far", [2 ** 30, 2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1])
def test_windows_and_blocks(cuda, far):
    q, k, v = draw(300, 128, BF16, 4)
    few = q[:, :, 40:44]
    for a, mask, want in ((q, cp.Mask(left=far, right=far), cp.FULL), (q, cp.Mask(left=far, right=0), cp.CAUSAL),
                          (q, cp.Mask(left=-1, right=0, block=far), cp.CAUSAL),
                          (few, cp.Mask(left=far, right=far, block=far), cp.FULL)):
        x, y = (cp.attention(a, k, v, mask=m).float() for m in (mask, want))
        assert ((x - y).abs() <= 2.0 ** -6 * y.abs() + 2.0 ** -9).all()
    assert cp.visible_pairs(cp.Mask(left=far, right=far, block=far), 300) == 300 * 300


@pytest.mark.parametrize("max_q", [1, 128])  # the kernel for few rows, and that for many
@pytest.mark.parametrize("dilation", [33, 2 ** 31 - 31, 2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("prefix", [0, 21])
def test_dilations_over_the_paged_cache(cuda, max_q, dilation, prefix):
    """With trees and without; tolerances as in ``test_tree_attn_gpu.py``."""
    mask = cp.Mask(left=-1, right=0, prefix=prefix, dilation=dilation)
    c = ta.make([13, 64, 90, 1], [50, 20, 5, 130], H=ta.heads(max_q), seed=6)  # (90: a chunk)
    got, lse = ta.run(c, max_q=max_q, mask=mask, return_lse=True)
    ta.check(c, got, lse, mask=mask)
    d = [c[n].cuda() for n in ("k", "v", "ks", "vs")]
    table, lens, cu = (ta.ints(c[n]) for n in ("table", "lens", "cu"))
    got = cp.paged_attention(c["q"].cuda(), *d, table, lens, cu, max_q=max_q, mask=mask)
    out, _, mass = po.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["lens"], c["cu"], mask=mask)
    assert ((got.double().cpu() - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -10 * mass + 2.0 ** -24).all()
