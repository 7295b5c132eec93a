"""The graph's node of qk_norm_rope among PyTorch's other tools: second derivatives are refused by whatever way they are asked
for, tensors that are saved elsewhere come back, a checkpoint computes again, transforms are refused."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import chia_proj_b200 as cp
from test_rope_gpu import BF16, F32, make

pytestmark = pytest.mark.gpu
NO_SECOND = dict(match="second derivative")


def leaves(seed=13, dtype=F32):
    q, k, qw, kw = make(1, 9, 2, 1, 64, dtype, dtype, seed=seed, fused=False)
    return [t.requires_grad_() for t in (q, k, qw, kw)]


@pytest.mark.parametrize("which", range(4))
def test_second_derivatives_beside_first_ones(cuda, which):
    """A loss of the outputs and of a gradient: the gradient's part is refused, not left out."""
    x, freqs = leaves(), cp.rope_frequencies(64)

    def both():
        a, b = cp.qk_norm_rope(*x, freqs)
        y = a.square().sum() + b.square().sum()
        (g,) = torch.autograd.grad(y, x[which], create_graph=True)
        return y + g.square().sum(), y, g
    loss, y, g = both()
    with pytest.raises(RuntimeError, **NO_SECOND):
        torch.autograd.grad(loss, x[which], retain_graph=True)
    for t in x:
        t.grad = None
    with pytest.raises(RuntimeError, **NO_SECOND):
        loss.backward(inputs=[x[which]], retain_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):
        torch.autograd.grad(g.sum(), x[which], retain_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):  # of another input
        torch.autograd.grad(g.sum(), x[(which + 1) % 4], retain_graph=True)
    # the first derivatives of the same graph, and a gradient taken as a number
    first = torch.autograd.grad(y + g.detach().square().sum(), x, retain_graph=True)
    again = torch.autograd.grad(both()[1], x)
    assert all(torch.equal(s, t) for s, t in zip(first, again))


def test_second_derivatives_of_what_comes_before_and_behind(cuda):
    """Inputs that are computed, and the gradient of the outputs."""
    x, freqs = leaves(), cp.rope_frequencies(64)
    s = torch.ones((), device="cuda", requires_grad=True)
    a, _ = cp.qk_norm_rope(x[0] * s, x[1], x[2], x[3], freqs)
    (g,) = torch.autograd.grad(a.square().sum(), x[1], create_graph=True, allow_unused=True)
    y = a.square().sum()
    (g,) = torch.autograd.grad(y, x[0], create_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):
        torch.autograd.grad(y + g.sum(), s, retain_graph=True)
    c = torch.randn(a.shape, device="cuda", requires_grad=True)
    a, _ = cp.qk_norm_rope(*x, freqs)
    (g,) = torch.autograd.grad(a, x[0], c, create_graph=True)
    with pytest.raises(RuntimeError, **NO_SECOND):
        torch.autograd.grad(g.sum(), c)
    x[0].grad = None
    a, _ = cp.qk_norm_rope(*x, freqs)
    a.square().sum().backward(create_graph=True)  # (gradients with a graph that nobody asks)
    want = torch.autograd.grad(cp.qk_norm_rope(*x, freqs)[0].square().sum(), x[0])[0]
    assert torch.equal(x[0].grad.detach(), want)
    for t in x:
        t.grad = None


def test_saved_elsewhere(cuda):
    """Saved-tensor hooks: on the host meanwhile, and packed by a function."""
    x, freqs = leaves(dtype=BF16), cp.rope_frequencies(64)
    pos = torch.randint(0, 900, (9,), generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()

    def grads():
        a, b = cp.qk_norm_rope(*x, freqs, pos)
        return a.float().square().sum() + b.float().sum()
    want = torch.autograd.grad(grads(), x)
    with torch.autograd.graph.save_on_cpu():
        y = grads()
    got = torch.autograd.grad(y, x)
    assert all(torch.equal(s, t) for s, t in zip(got, want))
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.clone(), lambda t: t):
        y = grads()
    got = torch.autograd.grad(y, x)
    assert all(torch.equal(s, t) for s, t in zip(got, want)) and len(packed) >= 6
    odd = torch.zeros(1, 9, 2, 131, dtype=BF16, device="cuda")[..., 1:65].copy_(x[0].detach().transpose(1, 2)).transpose(1, 2)
    odd.requires_grad_()  # (rows that are copied)
    with torch.autograd.graph.save_on_cpu():
        a, _ = cp.qk_norm_rope(odd, *x[1:], freqs, pos)
    assert torch.equal(torch.autograd.grad(a.float().square().sum(), odd)[0], want[0])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(cuda, reentrant):
    x, freqs = leaves(seed=15), cp.rope_frequencies(64)

    def part(q, k):
        a, b = cp.qk_norm_rope(q, k, x[2], x[3], freqs)
        return a * 2, b * 3
    want = part(x[0], x[1])
    want = torch.autograd.grad(want[0].sum() + want[1].square().sum(), x)
    a, b = checkpoint(part, x[0], x[1], use_reentrant=reentrant)
    if reentrant:
        (a.sum() + b.square().sum()).backward()
        got = [t.grad for t in x]
    else:
        got = torch.autograd.grad(a.sum() + b.square().sum(), x)
    assert all(torch.equal(s, t) for s, t in zip(got, want))


def test_errors_of_hooks_come_through(cuda):
    class Stop(Exception):
        pass

    def refuse(t):
        raise Stop("no room")
    x, freqs = leaves(), cp.rope_frequencies(64)
    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t):
        with pytest.raises(Stop, match="no room"):
            cp.qk_norm_rope(*x, freqs)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
        a, _ = cp.qk_norm_rope(*x, freqs)
    with pytest.raises(Stop, match="no room"):
        a.sum().backward()
    torch.autograd.grad(cp.qk_norm_rope(*x, freqs)[0].sum(), x)


@pytest.mark.parametrize("learns", [False, True])
def test_errors_of_the_library(cuda, learns):
    """The same error with gradients and without."""
    q, k = torch.zeros(1, 20000, 64, device="cuda", requires_grad=learns), torch.zeros(1, 1, 64, device="cuda")
    with pytest.raises(cp.ChiaError, match="INVALID_ARGUMENT"):
        cp.qk_norm_rope(q, k, None, None, cp.rope_frequencies(64))
    with pytest.raises(ValueError):
        cp.qk_norm_rope(q[:, :0], k, None, None, cp.rope_frequencies(64))


def test_transforms_are_refused(cuda):
    q, k, qw, kw = (t.detach() for t in leaves())
    freqs = cp.rope_frequencies(64)
    f = lambda x: cp.qk_norm_rope(x, k, qw, kw, freqs)[0].sum()
    for transformed in (lambda: torch.func.grad(f)(q), lambda: torch.func.vmap(f)(torch.stack([q, q])),
                        lambda: torch.func.jvp(f, (q,), (q,)), lambda: torch.func.vjp(f, q)):
        with pytest.raises((RuntimeError, ValueError)):
            transformed()
    with pytest.raises((RuntimeError, ValueError)):
        with torch.autograd.forward_ad.dual_level():
            f(torch.autograd.forward_ad.make_dual(q, q))
    assert torch.equal(f(q), f(q.clone()))
