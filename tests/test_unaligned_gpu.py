"""Dense inputs that begin at an address no 16-byte load can use, and single rows with odd strides: copied, as any other
input whose rows do not fit."""

import pytest
import torch

import chia_proj_b200 as cp

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


def odd(t):
    """The same values, dense, from the second element of a buffer on."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape).copy_(t)
    assert out.is_contiguous() and out.data_ptr() % 16 != 0
    return out


def one_row(t):
    """[1, ...] with an odd stride of the first dimension, which no step ever takes."""
    out = t.as_strided(t.shape, (t.numel() + 3, *t.stride()[1:]))
    assert out.shape[0] == 1 and out.stride(0) % 8 != 0
    return out


def draw(*shape, seed=0, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)


@pytest.mark.parametrize("change", [odd, one_row])
def test_norm_and_rotation(cuda, change):
    T = 1 if change is one_row else 5
    q, k, w = draw(T, 4, 64, seed=1), draw(T, 2, 64, seed=2), draw(64, seed=3)
    freqs = cp.rope_frequencies(64)
    assert same(cp.qk_norm_rope(change(q), change(k), w, odd(w), freqs), cp.qk_norm_rope(q, k, w, w, freqs))
    dq, dk = draw(T, 4, 64, seed=4), draw(T, 2, 64, seed=5)
    assert same(cp.qk_norm_rope_backward(change(dq), change(dk), change(q), change(k), w, odd(w), freqs),
                cp.qk_norm_rope_backward(dq, dk, q, k, w, w, freqs))
    x, y = change(q).requires_grad_(), q.clone().requires_grad_()
    assert same(torch.autograd.grad(cp.qk_norm_rope(x, k, w, w, freqs)[0], x, change(dq)),
                torch.autograd.grad(cp.qk_norm_rope(y, k, w, w, freqs)[0], y, dq))


@pytest.mark.parametrize("change", [odd, one_row])
def test_paged(cuda, change):
    T = 1 if change is one_row else 5
    q, k, v = draw(T, 4, 64, seed=1), draw(T, 2, 64, seed=2), draw(T, 2, 64, seed=3)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    a, b = cp.new_cache(2, 2, 64), cp.new_cache(2, 2, 64)
    cp.cache_append(k, v, ints(list(range(T))), *a)
    cp.cache_append(change(k), change(v), ints(list(range(T))), *b)
    assert same([t.view(torch.uint8) for t in a], [t.view(torch.uint8) for t in b])
    args = (*a, ints([[0]]), ints([T]), ints([0, T]))
    assert torch.equal(cp.paged_attention(q, *args), cp.paged_attention(change(q), *args))


@pytest.mark.parametrize("change", [odd, one_row])
@pytest.mark.parametrize("S", [4, 130])
def test_attention(cuda, change, S):
    q, k, v, d = (draw(1, 2, S, 64, seed=i) for i in range(4))
    assert torch.equal(cp.attention(q, k, v), cp.attention(change(q), change(k), change(v)))
    x, y = ([f(t).detach().requires_grad_() for t in (q, k, v)] for f in (change, torch.clone))
    assert same(torch.autograd.grad(cp.attention(*x), x, change(d)), torch.autograd.grad(cp.attention(*y), y, d))
