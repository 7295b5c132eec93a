"""qk_norm_rope (include/chia_rope.h) on the GPU against the plain 64-bit restatement (``draft_oracle.py``).

Tolerances, element by element. The output is rounded once to its type: half a step, ``eps / 2`` of the value, and of
fp16's subnormal numbers 2^-25. In fp32, the sum of squares (2^-20 of it with 128 terms, half of that in its root), the
reciprocal root and three products stay under 2^-20 of a value; a sine's or cosine's error is under 2^-22 (2^-23 of its own,
the angle's rounding pi 2^-25), and it multiplies both channels of a pair. 2^-19 of the pair's sizes is allowed. Gradients:
the same in fp32 for each of the two terms of dx, 2^-18 of their sizes; a weight's gradient is a sum of up to N products in
chains of at most 200 additions, 2^-16 of the sum of their sizes, and 2^-19 for the products: 2^-15.
"""

import pytest
import torch

import chia_proj_b200 as cp
import draft_oracle as do

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6


def half_step(t):
    return torch.finfo(t).eps / 2


def inv_freq(rot, base):
    return [base ** (-2.0 * i / rot) for i in range(rot // 2)]


def make(B, T, H, Hk, D, dtype, wdtype, seed, fused=True):
    """q, k as [B, H, T, D] views of one projection's output, weights."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, H + 2 * Hk, D, generator=g) * torch.exp(torch.randn(B, T, H + 2 * Hk, 1, generator=g))
    x = x.to(dtype).cuda()
    q, k, _ = x.split([H, Hk, Hk], 2)
    if not fused:
        q, k = q.contiguous(), k.contiguous()
    w = [None if wdtype is None else (1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).cuda() for _ in range(2)]
    return q.transpose(1, 2), k.transpose(1, 2), w[0], w[1]


def size_of_pairs(n, rot, interleaved):
    """|a| + |b| of each channel's pair (channels that do not turn: their own size)."""
    s = n.abs().clone()
    if rot:
        if interleaved:
            s[..., :rot] = (s[..., 0:rot:2] + s[..., 1:rot:2]).repeat_interleave(2, -1)
        else:
            h = rot // 2
            s[..., :rot] = (s[..., :h] + s[..., h:rot]).repeat(*([1] * (s.dim() - 1)), 2)
    return s


def check_forward(out, x, w, pos, freq, interleaved, offset):
    xd = x.detach().double().cpu()
    wd = None if w is None else w.detach().double().cpu()
    want = do.norm_rope(xd, wd, pos, freq, EPS, interleaved, offset)
    plain = do.norm_rope(xd, wd, pos, [], EPS, interleaved, offset)
    tol = half_step(x.dtype) * want.abs() + 2.0 ** -19 * size_of_pairs(plain, 2 * len(freq), interleaved) + 2.0 ** -25
    assert out.dtype == x.dtype and out.shape == x.shape
    assert ((out.detach().double().cpu() - want).abs() <= tol).all()


CASES = [  # B, T, H, Hk, D, rot, interleaved, dtype, weights, offset
    (1, 1, 32, 8, 128, 128, False, BF16, BF16, 0.0),
    (1, 7, 4, 1, 64, 64, False, F16, F32, 0.0),
    (2, 33, 5, 3, 128, 64, False, BF16, F32, 1.0),
    (1, 100, 8, 8, 64, 16, True, F16, F16, 1.0),
    (3, 50, 7, 1, 128, 128, True, F32, F32, 0.0),
    (1, 19, 2, 2, 64, 8, False, F32, BF16, 0.0),
    (1, 6000, 3, 1, 128, 96, False, BF16, None, 0.0),
    (2, 5, 1, 1, 64, 0, False, BF16, BF16, 0.0),
    (1, 3, 65, 13, 128, 8, True, BF16, BF16, 0.5),
]


@pytest.mark.parametrize("B,T,H,Hk,D,rot,inter,dtype,wdtype,offset", CASES)
def test_forward(cuda, B, T, H, Hk, D, rot, inter, dtype, wdtype, offset):
    q, k, qw, kw = make(B, T, H, Hk, D, dtype, wdtype, seed=T)
    base = 500000.0
    freqs, freq = cp.rope_frequencies(rot, base=base), inv_freq(rot, base) if rot else []
    pos = torch.randint(0, 100000, (B, T), generator=torch.Generator().manual_seed(1))
    pos[0, 0] = 2000003
    dev = pos.to(torch.int32).cuda()
    a, b = cp.qk_norm_rope(q, k, qw, kw, freqs, dev, interleaved=inter, weight_offset=offset)
    check_forward(a, q, qw, pos, freq, inter, offset)
    check_forward(b, k, kw, pos, freq, inter, offset)
    if B == 1:  # the same rows as [T, H, D]
        c, d = cp.qk_norm_rope(q[0].transpose(0, 1), k[0].transpose(0, 1), qw, kw, freqs, dev[0], interleaved=inter,
                               weight_offset=offset)
        assert torch.equal(c, a[0].transpose(0, 1)) and torch.equal(d, b[0].transpose(0, 1))
    else:  # positions that all entries share, and none
        a, b = cp.qk_norm_rope(q, k, qw, kw, freqs, dev[1], interleaved=inter, weight_offset=offset)
        check_forward(a, q, qw, pos[1:2].expand(B, T), freq, inter, offset)
        a, b = cp.qk_norm_rope(q, k, qw, kw, freqs, interleaved=inter, weight_offset=offset)
        check_forward(b, k, kw, torch.arange(T).expand(B, T), freq, inter, offset)


def test_far_and_negative_positions(cuda):
    """The angle is exact for any int32 position: 2^31 times a frequency's error in 64 bits (2^-53 of up to a radian) is
    2^-22, which the tolerance's 2^-19 of the pair holds."""
    q, k, qw, kw = make(1, 6, 2, 1, 128, F32, F32, seed=5)
    pos = torch.tensor([[2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 12345, -77777777, 0]])
    a, b = cp.qk_norm_rope(q, k, qw, kw, cp.rope_frequencies(128, base=10000.0), pos.to(torch.int32).cuda())
    check_forward(a, q, qw, pos, inv_freq(128, 10000.0), False, 0.0)
    check_forward(b, k, kw, pos, inv_freq(128, 10000.0), False, 0.0)


def reference_grads(x, w, pos, freq, inter, offset, dy):
    """dx and dw from the formula in 64 bits, and the sizes of what they sum."""
    xd, g = x.detach().double().cpu(), dy.double().cpu()
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.detach().double().cpu() + offset
    back = do.norm_rope(g * 0 + 1, None, pos, [], 0.0, inter, 0.0)  # ones; the rotation alone is turned back below
    assert torch.equal(back, torch.ones_like(back))
    half, gn, gs = len(freq), g.clone(), g.abs().clone()
    if half:
        angle = pos[:, None, :, None].double() * torch.tensor(freq, dtype=torch.float64)
        c, s = angle.cos(), angle.sin()
        one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if inter else (slice(0, half), slice(half, 2 * half))
        gn[..., one], gn[..., two] = g[..., one] * c + g[..., two] * s, g[..., two] * c - g[..., one] * s
        gs = size_of_pairs(g, 2 * half, inter)
    rstd = 1 / torch.sqrt((xd * xd).mean(-1, keepdim=True) + EPS)
    xhat = xd * rstd
    dx = rstd * (gn * wd - xhat * (gn * wd * xhat).mean(-1, keepdim=True))
    sx = rstd * (gs * wd.abs() + xhat.abs() * (gs * wd.abs() * xhat.abs()).mean(-1, keepdim=True))
    return dx, sx, (gn * xhat).flatten(0, -2).sum(0), (gs * xhat.abs()).flatten(0, -2).sum(0)


@pytest.mark.parametrize("B,T,H,Hk,D,rot,inter,dtype,wdtype,offset", CASES)
def test_backward(cuda, B, T, H, Hk, D, rot, inter, dtype, wdtype, offset):
    q, k, qw, kw = make(B, T, H, Hk, D, dtype, wdtype, seed=T + 1)
    freqs, freq = cp.rope_frequencies(rot), inv_freq(rot, 10000.0) if rot else []
    g = torch.Generator().manual_seed(9)
    pos = torch.randint(0, 5000, (B, T), generator=g)
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    for t in leaves:
        t.requires_grad_()
    out = cp.qk_norm_rope(q, k, qw, kw, freqs, pos.to(torch.int32).cuda(), interleaved=inter, weight_offset=offset)
    got = torch.autograd.grad(out, leaves, [dq, dk])
    again = cp.qk_norm_rope_backward(dq, dk, q, k, qw, kw, freqs, pos.to(torch.int32).cuda(), interleaved=inter,
                                     weight_offset=offset)
    for a, b in zip(got, [t for t in again if t is not None]):
        assert torch.equal(a, b)  # sums in an order that does not change
    for x, w, dy, i in ((q, qw, dq, 0), (k, kw, dk, 1)):
        dx, sx, dw, sw = reference_grads(x, w, pos, freq, inter, offset, dy)
        err = (got[i].double().cpu() - dx).abs()
        assert (err <= half_step(dtype) * dx.abs() + 2.0 ** -18 * sx + 2.0 ** -25).all()
        if w is not None:
            assert got[2 + i].dtype == w.dtype
            err = (got[2 + i].double().cpu() - dw).abs()
            assert (err <= half_step(w.dtype) * dw.abs() + 2.0 ** -15 * sw + 2.0 ** -25).all()


def test_backward_against_differences(cuda):
    """Along a direction, L = sum(out c) has the derivative <grad, d>. Differences over h = 2^-5 and 2 h, combined so that
    what is left of the cubic terms is of the order h^4 = 2^-20 of the fifth derivative (under 2^6 here: rows of norm 8
    moved by h). An output's error in fp32 is under 2^-17 (values of up to 4), 3 outputs to the unit of c, 192 outputs:
    2^-17 * 192 * 2 / h is 0.1 at the worst, against derivatives of about sqrt(192) = 14."""
    q, k, qw, kw = make(1, 1, 2, 1, 64, F32, F32, seed=2)
    q, k = (x.detach().contiguous() / x.detach().pow(2).mean(-1, keepdim=True).sqrt() for x in (q, k))
    freqs, pos = cp.rope_frequencies(32), torch.tensor([[123]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    c = [torch.randn(x.shape, generator=g).cuda() for x in (q, k)]
    d = [torch.randn(x.shape, generator=g).sign().cuda() for x in (q, k, qw, kw)]

    def loss(h):
        a, b = cp.qk_norm_rope(*(x + h * y for x, y in zip((q, k, qw, kw), d)), freqs, pos)
        return float((a.double() * c[0].double()).sum() + (b.double() * c[1].double()).sum())

    grads = cp.qk_norm_rope_backward(c[0], c[1], q, k, qw, kw, freqs, pos)
    want = sum(float((x.double() * y.double()).sum()) for x, y in zip(grads, d))
    h = 2.0 ** -5
    one, two = (loss(h) - loss(-h)) / (2 * h), (loss(2 * h) - loss(-2 * h)) / (4 * h)
    assert abs((4 * one - two) / 3 - want) <= 0.1


def test_only_what_is_wanted(cuda):
    """Gradients of the inputs or of one weight alone; a weight that is not there."""
    q, k, qw, kw = make(1, 9, 2, 1, 64, BF16, BF16, seed=3)
    freqs = cp.rope_frequencies(64)
    full = cp.qk_norm_rope_backward(q, k, q, k, qw, kw, freqs)
    kw.requires_grad_()
    out = cp.qk_norm_rope(q, k, qw, kw, freqs)
    assert torch.equal(torch.autograd.grad(out, kw, [q, k])[0], full[3])
    some = cp.qk_norm_rope_backward(q, k, q, k, qw, kw, freqs, weight_grads=(True, False))
    assert some[3] is None and torch.equal(some[2], full[2]) and torch.equal(some[0], full[0])
    qw.requires_grad_()
    only_k = torch.autograd.grad(cp.qk_norm_rope(q, k, None, kw, freqs), kw, [q, k])[0]  # no weight before it
    assert torch.equal(only_k, full[3])
    assert torch.equal(torch.autograd.grad(cp.qk_norm_rope(q, k, qw, None, freqs), qw, [q, k])[0], full[2])
    none = cp.qk_norm_rope_backward(q, k, q, k, qw, None, freqs)
    assert none[3] is None and torch.equal(none[0], full[0])
    assert not cp.qk_norm_rope(q, k, qw.detach(), kw.detach(), freqs)[0].requires_grad


def test_one_output_and_second_derivatives(cuda):
    q, k, qw, kw = make(1, 9, 2, 1, 64, F32, F32, seed=13, fused=False)
    freqs = cp.rope_frequencies(64)
    leaves = [t.requires_grad_() for t in (q, k, qw, kw)]
    a, b = cp.qk_norm_rope(*leaves, freqs)
    c = torch.randn(a.shape, device="cuda")
    got = torch.autograd.grad((a * c).sum(), leaves, retain_graph=True)
    want = cp.qk_norm_rope_backward(c, torch.zeros_like(k), q, k, qw, kw, freqs)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and not got[1].any() and not got[3].any()
    both = torch.autograd.grad((a, b), leaves, [c, torch.ones_like(k)])  # the same graph again
    assert torch.equal(both[0], want[0]) and both[1].any()
    a, _ = cp.qk_norm_rope(*leaves, freqs)
    (g,) = torch.autograd.grad(a.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):  # (not a part of the graph)
        torch.autograd.grad(g.sum(), q, retain_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()
    a, _ = cp.qk_norm_rope(*leaves, freqs)
    with torch.no_grad():
        q.add_(1.0)  # what is kept must not change
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        a.sum().backward()
    import threading
    seen = []
    x = q.detach().requires_grad_()
    th = threading.Thread(target=lambda: seen.append(torch.autograd.grad(cp.qk_norm_rope(x, k, qw, kw, freqs)[0].sum(), x)[0]))
    th.start(), th.join()
    assert torch.equal(seen[0], torch.autograd.grad(cp.qk_norm_rope(x, k, qw, kw, freqs)[0].sum(), x)[0])


def test_views_streams_and_empty_inputs(cuda):
    q, k, qw, kw = make(1, 40, 4, 2, 128, BF16, BF16, seed=8, fused=False)
    q, k, freqs = q[0].transpose(0, 1), k[0].transpose(0, 1), cp.rope_frequencies(128)
    want = cp.qk_norm_rope(q, k, qw, kw, freqs)
    # strides that no 16-byte load can use, and a last dimension that is not dense, are copied
    odd = torch.zeros(40, 4, 131, dtype=BF16, device="cuda")[..., 1:129].copy_(q)
    turned = torch.empty(40, 128, 2, dtype=BF16, device="cuda").transpose(1, 2).copy_(k)
    got = cp.qk_norm_rope(odd, turned, qw, kw, freqs)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    every = cp.qk_norm_rope(q.repeat_interleave(2, 0)[::2], k, qw.repeat_interleave(2)[::2], kw, freqs)
    assert torch.equal(every[0], want[0])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cp.qk_norm_rope(q, k, qw, kw, freqs)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0])
    a, b = cp.qk_norm_rope(q[:0], k[:0], qw, kw, freqs)
    assert a.shape == (0, 4, 128) and b.shape == (0, 2, 128)
    dq, dk, dqw, dkw = cp.qk_norm_rope_backward(q[:0], k[:0], q[:0], k[:0], qw, kw, freqs)
    assert dq.shape == (0, 4, 128) and not dqw.any() and not dkw.any()


def test_values_that_are_not_finite(cuda):
    """They stay in their row."""
    q, k, qw, kw = make(1, 8, 4, 2, 64, F32, F32, seed=10, fused=False)
    freqs = cp.rope_frequencies(32)
    want, _ = cp.qk_norm_rope(q, k, qw, kw, freqs)
    q2 = q.clone()
    q2[0, 1, 2, 5], q2[0, 3, 4, 6], q2[0, 0, 0] = float("nan"), float("inf"), 0.0
    got, _ = cp.qk_norm_rope(q2, k, qw, kw, freqs)
    keep = torch.ones(1, 4, 8, dtype=torch.bool)
    keep[0, 1, 2] = keep[0, 3, 4] = keep[0, 0, 0] = False
    assert torch.equal(got[keep], want[keep])
    assert got[0, 1, 2].isnan().all() and not got[0, 0, 0].any()


def capture(step):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    return graph, got


def test_in_a_graph(cuda):
    """Forward and backward captured and replayed on new values. While an eager graph of the same leaves lives, PyTorch
    itself refuses to capture their gradients (a leaf's node belongs to the stream that it was made on, for any operator);
    the explicit backward call has no such node."""
    q, k, qw, kw = make(1, 300, 4, 2, 128, BF16, F32, seed=11, fused=False)
    q, k = q.contiguous().requires_grad_(), k.contiguous().requires_grad_()
    qw.requires_grad_(), kw.requires_grad_()
    freqs, dy = cp.rope_frequencies(128), [torch.randn_like(x) for x in (q, k)]

    def step():
        out = cp.qk_norm_rope(q, k, qw, kw, freqs)
        return list(out) + list(torch.autograd.grad(out, (q, k, qw, kw), dy))

    def explicit():
        with torch.no_grad():
            return list(cp.qk_norm_rope(q, k, qw, kw, freqs)) + list(cp.qk_norm_rope_backward(*dy, q, k, qw, kw, freqs))

    graph, got = capture(step)
    alive = cp.qk_norm_rope(q, k, qw, kw, freqs)
    graph2, got2 = capture(explicit)
    with torch.no_grad():
        q.copy_(torch.randn_like(q))
        kw.mul_(0.5)
    graph.replay(), graph2.replay()
    for a, b, c in zip(got, got2, explicit()):
        assert torch.equal(a, c) and torch.equal(b, c)
    del alive


@pytest.mark.parametrize("dtype,code", [(BF16, 0), (F32, 2)])
def test_in_place_through_the_c_abi(lib, cuda, dtype, code):
    import ctypes

    from chia_proj_b200 import _native as N
    q, k, qw, kw = make(2, 37, 6, 2, 128, dtype, dtype, seed=17, fused=False)
    freqs = cp.rope_frequencies(64)
    want = cp.qk_norm_rope(q, k, qw, kw, freqs)
    p = N.RopeParams(abi_version=N.ROPE_ABI_VERSION, dtype=code, weight_dtype=code, head_dim=128, heads=6, heads_kv=2,
                     rot=64, batch=2, seqlen=37, q=q.data_ptr(), k=k.data_ptr(), q_out=q.data_ptr(), k_out=k.data_ptr(),
                     q_weight=qw.data_ptr(), k_weight=kw.data_ptr(), freqs=freqs.data_ptr(), eps=EPS)
    for f, t in (("q_stride", q), ("q_out_stride", q), ("k_stride", k), ("k_out_stride", k)):
        getattr(p, f)[:] = t.stride()[:3]
    stream = ctypes.c_void_p(torch.cuda.current_stream(cuda).cuda_stream)
    assert lib.chia_qk_norm_rope(bytes(p), stream) == 0
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_refusals(cuda):
    q, k, qw, kw = make(1, 4, 4, 2, 64, BF16, BF16, seed=1, fused=False)
    f, pos = cp.rope_frequencies(64), torch.arange(4, dtype=torch.int32, device="cuda")
    good = dict(q=q, k=k, q_weight=qw, k_weight=kw, freqs=f, positions=pos)
    cp.qk_norm_rope(**good)
    for bad in (dict(k=k[:, :, :3]), dict(k=k.half()), dict(k=k[0]), dict(q=q[..., :32], k=k[..., :32]), dict(q=q.double(), k=k.double()),
                dict(q=q[:, :0]), dict(q_weight=qw[:32]), dict(q_weight=qw.float()), dict(freqs=f.int()),
                dict(freqs=cp.rope_frequencies(72)), dict(freqs=f[:30]), dict(positions=pos.long()), dict(positions=pos[:3]),
                dict(positions=pos[None].expand(2, 4)), dict(eps=-1.0), dict(eps=float("nan")),
                dict(weight_offset=float("inf")), dict(q=q[0, 0], k=k[0, 0])):
        with pytest.raises(ValueError):
            cp.qk_norm_rope(**{**good, **bad})
    with pytest.raises(ValueError):
        cp.qk_norm_rope_backward(q.half(), k, **good)
    with pytest.raises(ValueError):
        cp.qk_norm_rope_backward(q, k[:, :, :3], **good)
    with pytest.raises(RuntimeError):
        cp.qk_norm_rope(**{**good, "freqs": f.cpu()})


@pytest.mark.parametrize("dtype,T,H,Hk,D,one_sign", [(BF16, 60001, 8, 1, 64, False), (BF16, 60001, 8, 1, 64, True),
                                                     (F32, 4 * 4096, 16, 16, 128, True)])
def test_long_sums_of_the_weights_gradients(cuda, dtype, T, H, Hk, D, one_sign):
    """Sums over up to half a million rows, also of products that all have one sign, where roundings add up. A thread adds
    the rows of its group, T H over the groups of all CTAs (4 an SM, of 16 or 8 groups; twice as many are allowed for, since
    groups differ by a token), then up to 16, 19 and 32 parts. A sum of n additions in a row is off by n 2^-24 of the
    terms' sizes, and 2^-19 of them for the products."""
    g = torch.Generator().manual_seed(T + one_sign)
    q, k = (torch.randn(T, h, D, generator=g).to(dtype).cuda() for h in (H, Hk))
    w = torch.ones(D, device="cuda")
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    if one_sign:
        dq, dk = dq.abs() * q.sign(), dk.abs() * k.sign()
    freqs = cp.rope_frequencies(0)
    got = cp.qk_norm_rope_backward(dq, dk, q, k, w, w, freqs)[2:]
    for x, dy, dw, h in ((q, dq, got[0], H), (k, dk, got[1], Hk)):
        xd, gd = x.double(), dy.double()
        xhat = xd / torch.sqrt((xd * xd).mean(-1, keepdim=True) + EPS)
        want, size = (gd * xhat).flatten(0, 1).sum(0), (gd * xhat).abs().flatten(0, 1).sum(0)
        chain = 2 * T * h / (4 * 132 * (128 // (D // 8))) + 100
        assert ((dw.double() - want).abs() <= (chain * 2.0 ** -24 + 2.0 ** -19) * size + 2.0 ** -24 * want.abs()).all()
