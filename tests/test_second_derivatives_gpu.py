"""Second derivatives of attention are refused by whatever way they are asked for, not left out."""

import pytest
import torch

import chia_proj_b200 as cp

pytestmark = pytest.mark.gpu
NO_SECOND = dict(match="second derivative")
CALLS = [dict(), dict(mod="softcap"), dict(norm="sigmoid"), dict(return_lse=True)]


@pytest.mark.parametrize("kw", CALLS)
@pytest.mark.parametrize("which", range(3))
def test_attention(cuda, which, kw):
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(1, 2, 150, 64, generator=g).to(torch.bfloat16).cuda().requires_grad_() for _ in range(3)]

    def loss():
        out = cp.attention(*x, **kw)
        return (out[0] if isinstance(out, tuple) else out).float().square().sum()
    y = loss()
    (d,) = torch.autograd.grad(y, x[which], create_graph=True)
    both = y + d.float().square().sum()
    for of, to in ((both, x[which]), (both, x[(which + 1) % 3]), (d.sum(), x[which])):
        with pytest.raises(RuntimeError, **NO_SECOND):
            torch.autograd.grad(of, to, retain_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):
        both.backward(inputs=[x[which]], retain_graph=True)
    first = torch.autograd.grad(y + d.detach().float().sum(), x, retain_graph=True)
    again = torch.autograd.grad(loss(), x)
    assert all(torch.equal(s, t) for s, t in zip(first[1:], again[1:]))
    # dq is summed in fp32 in an order that varies, then rounded once: a step of bf16, and of the largest one's 2^-9
    top = again[0].abs().max().float()
    assert ((first[0] - again[0]).abs().float() <= 2.0 ** -7 * again[0].abs().float() + 2.0 ** -9 * top).all()
    c = torch.randn(x[0].shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    out = cp.attention(*x, **kw)
    (d,) = torch.autograd.grad(out[0] if isinstance(out, tuple) else out, x[which], c, create_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):
        torch.autograd.grad(d.sum(), c)
