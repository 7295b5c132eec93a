"""The operators of a serving step together: replayed as a CUDA graph while the requests grow, and the two attention
kernels beside one another and beside the 64-bit oracle."""

import pytest
import torch

import chia_proj_b200 as cp
from test_paged_gpu import BF16, E4M3, I8, check_attention, ints, kind_args, near, setup

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status(cuda):
    yield
    cp.check_device_status(0)


@pytest.mark.parametrize("kind", ["alibi", "temp"])
@pytest.mark.parametrize("ct,D,page", [(E4M3, 128, 64), (I8, 64, 16)])
def test_head_parameters_with_many_rows(cuda, kind, ct, D, page):
    """bf16 outputs of the kernel for many rows (56 and more a K/V head)."""
    check_attention([300, 75, 513], [60, 75, 130], 8, 2, D, page, ct, BF16, **kind_args(kind, 8))
    check_attention([300, 975], [260, 1], 3, 1, D, page, ct, BF16, mask=cp.Mask(left=100, right=0, prefix=7), **kind_args(kind, 3))


@pytest.mark.parametrize("kind", ["plain", "softcap", "alibi", "temp", "sigmoid", "relu"])
def test_the_hint_chooses_the_kernel_not_the_result(cuda, kind):
    lens, counts = [900, 64, 2500, 3], [90, 64, 1, 3]
    q, k, v, ks, vs, table, cu = setup(lens, counts, 8, 2, 128, 32, E4M3, BF16, 21)
    kw = kind_args(kind, 8)
    a, b = (cp.paged_attention(q, k, v, ks, vs, ints(table), ints(lens), ints(cu), max_q=m, **kw) for m in (1, 90))
    assert not torch.equal(a, b)  # two schedules
    assert near(a, b, BF16)


@pytest.mark.parametrize("ct,window", [(E4M3, -1), (I8, 40)])
def test_a_graph_of_a_step_while_requests_grow(cuda, ct, window):
    """Tables, write and attention captured once and replayed: lengths, pages and inputs change from replay to replay
    and the outputs are those of the same calls made one by one, bit by bit."""
    B, hkv, H, D, page, W, steps = 5, 2, 8, 128, 16, 12, 90
    g = torch.Generator().manual_seed(8)
    qkv = torch.randn(steps, B, H + 2 * hkv, D, generator=g).to(BF16).cuda()
    mask = cp.Mask(left=window, right=0)
    start = [0, 3, 16, 31, 90]

    def fresh():
        cache = cp.new_cache(B * W, hkv, D, page_size=page, dtype=ct)
        lens, table = ints([0] * B), torch.zeros(B, W, dtype=torch.int32, device="cuda")
        ring, state = ints(list(range(B * W))), ints([7, B * W])
        x = torch.randn(sum(start), 2 * hkv, D, generator=torch.Generator().manual_seed(9)).to(BF16).cuda()
        t = cp.page_tables(lens, ints(start), table, ring, state, page_size=page, max_tokens=sum(start))
        cp.cache_append(x[:, :hkv], x[:, hkv:], t.slots, *cache)
        return cache, t.seq_lens.clone(), table, ring, t.free_state.clone()

    def step(x, cache, lens, table, ring, state, new):
        t = cp.page_tables(lens, new, table, ring, state, page_size=page, max_tokens=B)
        q, k, v = x.split([H, hkv, hkv], 1)
        cp.cache_append(k, v, t.slots, *cache)
        out = cp.paged_attention(q, *cache, table, t.seq_lens, t.cu_q, max_q=1, mask=mask)
        lens.copy_(t.seq_lens)
        state.copy_(t.free_state)
        return out

    one = ints([1] * B)
    eager = fresh()
    want = [step(x, *eager, one).clone() for x in qkv]
    again = fresh()
    x = qkv[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, *again, one)
    for i in range(steps):
        x.copy_(qkv[i])
        graph.replay()
        assert torch.equal(out, want[i]), i
    assert again[1].tolist() == [n + steps for n in start]
    for a, b in zip((*eager[0], *eager[1:]), (*again[0], *again[1:])):
        assert torch.equal(a.view(torch.uint8) if a.element_size() == 1 else a, b.view(torch.uint8) if b.element_size() == 1 else b)


def test_out_that_overlaps_itself_is_refused(cuda):
    """Rows that share memory would be written by many CTAs at a time. What does not overlap is taken in any order."""
    q, k, v, ks, vs, table, cu = setup([70, 33], [2, 1], 4, 2, 64, 16, E4M3, BF16)
    args = (q, k, v, ks, vs, ints(table), ints([70, 33]), ints(cu))
    want = cp.paged_attention(*args)
    buf = torch.zeros(4096, dtype=BF16, device="cuda")
    for strides in ((0, 64, 1), (256, 0, 1), (64, 64, 1), (248, 64, 1), (64, 128, 1), (256, 56, 1), (0, 0, 1)):
        with pytest.raises(ValueError, match="overlap"):
            cp.paged_attention(*args, out=buf.as_strided((3, 4, 64), strides))
    for strides in ((256, 64, 1), (64, 192, 1), (264, 64, 1), (1024, 72, 1), (72, 256, 1)):
        out = buf.as_strided((3, 4, 64), strides)
        assert torch.equal(cp.paged_attention(*args, out=out), want)
    one = buf.as_strided((1, 4, 64), (0, 64, 1))
    assert torch.equal(cp.paged_attention(q[2:], k, v, ks, vs, ints(table[1:]), ints([33]), out=one), want[2:])
