"""Rows and pages whose elements lie beyond 2^31 (and bytes beyond 2^32): each call on a large tensor gives for its last rows
what it gives for those alone."""

import pytest
import torch

import chia_proj_b200 as cp

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def clean(cuda):
    yield
    cp.check_device_status(0)
    torch.cuda.empty_cache()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_norm_and_rotation(cuda):
    T, H, Hk, D, last = 530000, 32, 1, 128, 300  # 2.17e9 elements
    q = torch.empty(T, H, D, dtype=BF16, device="cuda").zero_()
    k = torch.zeros(T, Hk, D, dtype=BF16, device="cuda")
    assert q.numel() > 2 ** 31
    for x in (q, k):
        x[-last:].copy_(torch.randn(x[-last:].shape, device="cuda"))
    w, freqs = torch.randn(D, device="cuda"), cp.rope_frequencies(D)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    a, b = cp.qk_norm_rope(q, k, w, w, freqs, pos)
    want = cp.qk_norm_rope(q[-last:], k[-last:], w, w, freqs, pos[-last:])
    assert torch.equal(a[-last:], want[0]) and torch.equal(b[-last:], want[1]) and not a[:1000].any()
    del a, b
    dq, dk, dqw, _ = cp.qk_norm_rope_backward(q, k, q, k, w, w, freqs, pos)
    want = cp.qk_norm_rope_backward(q[-last:], k[-last:], q[-last:], k[-last:], w, w, freqs, pos[-last:])
    assert torch.equal(dq[-last:], want[0]) and torch.equal(dk[-last:], want[1])
    # the other rows are zero and give the weights nothing; sums in another order: 2^-15 of the terms' sizes (300 x 32
    # of the order of |q| |xhat| <= 25)
    assert ((dqw - want[2]).abs() <= 2.0 ** -15 * last * H * 25).all()


def test_verification(cuda):
    V, T = 131072, 16450  # 2.16e9 elements
    p = torch.zeros(T, V, dtype=BF16, device="cuda")
    q = torch.zeros(T, V, dtype=BF16, device="cuda")
    assert p.numel() > 2 ** 31
    n = 20
    g = torch.Generator().manual_seed(1)
    for x in (p, q):
        x[-n:].copy_(torch.softmax(torch.randn(n, V, generator=g), 1))
    parents = [-1] + [(i - 1) // 2 for i in range(1, n)]
    tokens, u = torch.randint(0, V, (T,), generator=g).to(torch.int32).cuda(), torch.rand(T, generator=g).cuda()
    par = torch.zeros(T, dtype=torch.int32, device="cuda")
    par[-n:] = ints(parents)
    got = cp.verify_drafts(p, tokens, par, ints([T - n, T]), u, draft_probs=q, max_tokens=6)
    want = cp.verify_drafts(p[-n:].clone(), tokens[-n:].clone(), ints(parents), ints([0, n]), u[-n:].clone(),
                            draft_probs=q[-n:].clone(), max_tokens=6)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got.counts.item() >= 1 and got.tokens[0, 0].item() >= 0


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
def test_compaction(cuda, dtype):
    page, hkv, D, pages = 128, 8, 128, 33000  # 4.3e9 bytes each
    raw = [torch.zeros(pages, hkv, page, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    assert raw[0].numel() > 2 ** 32
    for x in raw:
        x[-2:].copy_(torch.randint(1, 100, x[-2:].shape, device="cuda"))
    scale = [torch.ones(pages, hkv, device="cuda") for _ in range(2)]
    scale[0][-1] = 4.0
    small = [x[-2:].clone() for x in raw + scale]
    args = (ints([[0, 30, 33, 63]]), ints([4]), ints([0, 64]), ints([page + 50]))
    keep = cp.cache_compact(*args, ints([[pages - 2, pages - 1]]), *(x.view(dtype) for x in raw), *scale)
    want = cp.cache_compact(*args, ints([[0, 1]]), *(x.view(dtype) for x in small[:2]), *small[2:])
    assert keep.tolist() == want.tolist() == [page + 50 - 64 + 4]
    assert all(torch.equal(a[-2:], b) for a, b in zip(raw + scale, small))
    assert not raw[0][:pages - 2].any() and not torch.equal(small[0][0], small[0][1])
