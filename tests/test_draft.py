"""The C ABI of drafted tokens (include/chia_draft.h) and of the norm and rotation of queries and keys (include/chia_rope.h)
and their Python entry points, without a GPU: exports, struct layouts, refusals before anything is launched."""

import ctypes
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

import chia_proj_b200 as cp
import draft_oracle as do
import paged_oracle as po
from chia_proj_b200 import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"chia_tree_params_t": N.TreeParams, "chia_verify_params_t": N.VerifyParams,
           "chia_compact_params_t": N.CompactParams, "chia_rope_params_t": N.RopeParams,
           "chia_rope_grads_t": N.RopeGrads}


@pytest.mark.parametrize("header,names", [("chia_draft.h", N.DRAFT_SYMBOLS), ("chia_rope.h", N.ROPE_SYMBOLS)])
def test_exports(lib, header, names):
    src = open(os.path.join(ROOT, "include", header)).read()
    declared = set(re.findall(r"CHIA_API\s+[\w\s\*]*?\b(chia_\w+)\s*\(", src))
    assert declared == set(names)
    for name in declared:
        assert hasattr(lib, name)
    assert f"#define CHIA_TREE_NODES {N.TREE_NODES}" in open(os.path.join(ROOT, "include", "chia_draft.h")).read()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
@pytest.mark.parametrize("name", list(STRUCTS))
def test_struct_layout_matches_header(tmp_path, name):
    fields = [f[0] for f in STRUCTS[name]._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", '#include "chia_draft.h"', "int main(void){",
            f'printf("%zu\\n", sizeof({name}));']
    prog += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]
    c, exe = tmp_path / "l.c", tmp_path / "l"
    c.write_text("\n".join(prog))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    vals = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(STRUCTS[name])
    assert vals[1:] == [getattr(STRUCTS[name], f).offset for f in fields]


A = 0x10000  # never dereferenced: each call is refused first


def packed(struct, **kw):
    s = struct()
    for f, v in kw.items():
        if isinstance(v, tuple):
            getattr(s, f)[:] = v
        else:
            setattr(s, f, v)
    return bytes(s)


TREE = dict(abi_version=1, batch=4, tokens=8, parents=A, cu_q=A, seq_lens=A, positions=A, ancestors=A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=2), 1), (dict(batch=0), 1), (dict(tokens=-1), 1), (dict(parents=None), 1), (dict(cu_q=None), 1),
    (dict(ancestors=None), 1), (dict(ancestors=A + 4), 3), (dict(positions=A + 1), 3),
])
def test_tree_tables_refusals(lib, change, code):
    assert lib.chia_tree_tables(packed(N.TreeParams, **{**TREE, **change}), None) == code
    assert lib.chia_tree_tables(None, None) == 1


PAGED = dict(abi_version=1, dtype=0, cache_dtype=0, head_dim=128, norm=0, mod=0, heads=8, heads_kv=2, page_size=64,
             max_q=1, batch=4, tokens=4, num_pages=10, table_width=5, table_stride=5, q=A, o=A, q_stride=(1024, 128),
             o_stride=(1024, 128), k_cache=A, v_cache=A, k_scale=A, v_scale=A, block_table=A, seq_lens=A, scale=0.1,
             softcap=30.0, out_scale=1.0, win_left=-1, dilation=1, workspace=A, workspace_bytes=1 << 40)


def test_tree_attn_refusals(lib):
    for change, code in [(dict(head_dim=96), 2), (dict(heads=9), 1), (dict(q=A + 2), 3), (dict(workspace_bytes=8), 1)]:
        assert lib.chia_tree_attn(packed(N.PagedParams, **{**PAGED, **change}), A, A, None) == code
    good = packed(N.PagedParams, **PAGED)
    assert lib.chia_tree_attn(good, None, A, None) == 1 and lib.chia_tree_attn(good, A, None, None) == 1
    assert lib.chia_tree_attn(good, A + 2, A, None) == 3 and lib.chia_tree_attn(good, A, A + 4, None) == 3
    assert lib.chia_tree_attn(None, A, A, None) == 1


VERIFY = dict(abi_version=1, dtype=2, batch=4, tokens=8, vocab=100, max_tokens=5, target_probs=A, draft_probs=A,
              target_stride=100, draft_stride=100, node_tokens=A, parents=A, cu_q=A, uniforms=A, counts=A, out_tokens=A,
              path=A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=0), 1), (dict(dtype=3), 2), (dict(batch=0), 1), (dict(vocab=0), 1), (dict(max_tokens=0), 1),
    (dict(vocab=2 ** 22 + 1, target_stride=2 ** 23, draft_stride=2 ** 23), 2), (dict(target_stride=99), 1),
    (dict(draft_stride=99), 1), (dict(target_probs=None), 1), (dict(uniforms=None), 1), (dict(counts=None), 1),
    (dict(target_probs=A + 2), 3), (dict(dtype=0, target_probs=A + 1), 3), (dict(path=A + 2), 3), (dict(tokens=-1), 1),
])
def test_verify_refusals(lib, change, code):
    assert lib.chia_verify_drafts(packed(N.VerifyParams, **{**VERIFY, **change}), None) == code
    assert lib.chia_verify_drafts(None, None) == 1


COMPACT = dict(abi_version=1, cache_dtype=0, head_dim=128, heads_kv=2, page_size=64, batch=4, max_tokens=5, num_pages=10,
               table_width=5, table_stride=5, path=A, counts=A, cu_q=A, seq_lens=A, block_table=A, k_cache=A, v_cache=A,
               k_scale=A, v_scale=A, keep_lens=2 * A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=0), 1), (dict(cache_dtype=2), 2), (dict(head_dim=96), 2), (dict(page_size=48), 2),
    (dict(heads_kv=0), 1), (dict(max_tokens=0), 1), (dict(num_pages=2 ** 30), 1), (dict(table_stride=4), 1),
    (dict(path=None), 1), (dict(keep_lens=A), 1), (dict(k_cache=A + 8), 3), (dict(counts=A + 1), 3),
    (dict(batch=2 ** 24, heads_kv=65535), 2),
])
def test_compact_refusals(lib, change, code):
    assert lib.chia_cache_compact(packed(N.CompactParams, **{**COMPACT, **change}), None) == code
    assert lib.chia_cache_compact(None, None) == 1


ROPE = dict(abi_version=1, dtype=0, weight_dtype=0, head_dim=128, heads=8, heads_kv=2, rot=128, batch=1, seqlen=4, q=A,
            k=A, q_out=A, k_out=A, q_stride=(0, 128, 1024), k_stride=(0, 128, 256), q_out_stride=(0, 128, 1024),
            k_out_stride=(0, 128, 256), q_weight=A, k_weight=A, freqs=A, eps=1e-6)
GRADS = dict(dq_out=A, dk_out=A, dq_out_stride=(0, 128, 1024), dk_out_stride=(0, 128, 256), dq=A, dk=A, dq_weight=A,
             dk_weight=A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=0), 1), (dict(dtype=3), 2), (dict(weight_dtype=4), 2), (dict(head_dim=96), 2), (dict(heads=0), 1),
    (dict(heads_kv=20000), 1), (dict(rot=132), 1), (dict(rot=12), 1), (dict(batch=0), 1), (dict(seqlen=-1), 1),
    (dict(batch=2 ** 20, seqlen=2 ** 20), 2), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(freqs=None), 1),
    (dict(q=None), 1), (dict(q=A + 8), 3), (dict(q_stride=(0, 100, 1024)), 3), (dict(k_out_stride=(-8, 128, 256)), 1),
    (dict(position_stride=-1), 1), (dict(weight_offset=float("inf")), 1), (dict(q_weight=A + 1), 3),
])
def test_rope_refusals(lib, change, code):
    p = packed(N.RopeParams, **{**ROPE, **change})
    assert lib.chia_qk_norm_rope(p, None) == code
    assert lib.chia_qk_norm_rope_bwd(p, packed(N.RopeGrads, **GRADS), A, 1 << 40, None) == code
    assert lib.chia_qk_norm_rope_bwd_workspace_bytes(p) == -1
    assert lib.chia_qk_norm_rope(None, None) == 1


@pytest.mark.parametrize("change,code", [
    (dict(dq_out=None), 1), (dict(dk=None), 1), (dict(dq=A + 4), 3), (dict(dk_out_stride=(0, 128, 100)), 3),
])
def test_rope_gradient_refusals(lib, change, code):
    p = packed(N.RopeParams, **ROPE)
    assert lib.chia_qk_norm_rope_bwd(p, packed(N.RopeGrads, **{**GRADS, **change}), A, 1 << 40, None) == code
    assert lib.chia_qk_norm_rope_bwd(p, None, A, 1 << 40, None) == 1
    assert lib.chia_qk_norm_rope_bwd(p, packed(N.RopeGrads, **GRADS), None, 1 << 40, None) == 1
    # a gradient of a weight that is not there
    p = packed(N.RopeParams, **{**ROPE, "q_weight": None})
    assert lib.chia_qk_norm_rope_bwd(p, packed(N.RopeGrads, **GRADS), A, 1 << 40, None) == 1
    assert lib.chia_qk_norm_rope_bwd_workspace_bytes(packed(N.RopeParams, **ROPE)) > 0


def test_no_cpu_fallback(lib):
    i = torch.zeros(2, dtype=torch.int32)
    x, p = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.zeros(2, 10)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.tree_tables(i, i, i[:1])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.verify_drafts(p, i, i, i, torch.zeros(2), max_tokens=3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.cache_compact(i[None], i[:1], i, i[:1], i[None], *cp.new_cache(2, 1, 64, page_size=16, device="cpu"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.qk_norm_rope(x, x, None, None, cp.rope_frequencies(64, device="cpu"))


def test_rope_frequencies(lib):
    f = cp.rope_frequencies(64, base=10000.0, device="cpu")
    assert f.dtype == torch.int64 and f.shape == (32,)
    # turns in units of 2^-64: rounded to a whole one (2^-65), the division by 2 pi in 64 bits (2^-52 of the value)
    for i, t in enumerate(f.tolist()):
        want = 10000.0 ** (-2 * i / 64) / (2 * math.pi)
        assert abs(t % 2 ** 64 / 2 ** 64 - want) <= 2.0 ** -52 * want + 2.0 ** -65
    assert torch.equal(f, cp.rope_frequencies(64, inv_freq=[10000.0 ** (-2 * i / 64) for i in range(32)], device="cpu"))
    # frequencies beyond a turn, and negative ones
    g = cp.rope_frequencies(16, inv_freq=[2 * math.pi * x for x in (0.25, 1.25, -0.25, 0.5, 0, 2, 3.5, -1)], device="cpu")
    assert [x % 2 ** 64 / 2 ** 64 for x in g.tolist()] == [0.25, 0.25, 0.75, 0.5, 0, 0, 0.5, 0]
    assert cp.rope_frequencies(0, device="cpu").shape == (0,)
    for bad in (dict(rot_dim=12), dict(rot_dim=-8), dict(rot_dim=16, base=0.0), dict(rot_dim=16, inv_freq=[1.0]),
                dict(rot_dim=8, inv_freq=[1.0, 2.0, 3.0, float("inf")])):
        with pytest.raises(ValueError):
            cp.rope_frequencies(device="cpu", **bad)


def test_verification_draws_from_the_target():
    """The rule itself, on a vocabulary of four: drafts drawn from q, verified against p, come out distributed as p. 20,000
    runs: a frequency is off by at most four standard deviations (0.0142) with a probability of 6e-5 a token."""
    g = torch.Generator().manual_seed(3)
    p = torch.tensor([[0.1, 0.2, 0.3, 0.4], [0.25, 0.25, 0.25, 0.25], [0.7, 0.1, 0.1, 0.1]], dtype=torch.float64)
    q = torch.tensor([[0.4, 0.3, 0.2, 0.1], [0.1, 0.2, 0.3, 0.4], [0.25] * 4], dtype=torch.float64)
    n, first = 20000, [0] * 4
    draws = torch.multinomial(q[0].expand(n, 4), 2, generator=g).tolist()  # two children, without replacement
    u = torch.rand(n, 3, generator=g)
    for i in range(n):
        _, out, _ = do.verify(p, [0] + draws[i], [-1, 0, 0], [0, 3], u[i], q, 2)
        first[out[0][0]] += 1
    for x in range(4):
        assert abs(first[x] / n - float(p[0, x])) < 0.0142


@pytest.mark.parametrize("mask", [cp.CAUSAL, cp.FULL, cp.Mask(right=0, prefix=38), cp.Mask(left=5, right=9),
                                  cp.Mask(left=10, right=0, prefix=60, dilation=2), cp.Mask(right=0, block=24)])
@pytest.mark.parametrize("base", [0, 1, 40, -5])
def test_chunks_attend_as_without_trees(mask, base):
    """The restatement's own: more than 64 queries are no tree, whatever the mask and the parents."""
    g, n, H, hkv, D, page = torch.Generator().manual_seed(3), 70, 4, 2, 8, 16
    length = n + base
    pages = po.pages_for(length, page)
    q = torch.randn(n, H, D, generator=g)
    k, v = torch.randn(pages, hkv, page, D, generator=g), torch.randn(pages, hkv, page, D, generator=g)
    ks, vs = torch.ones(pages, hkv), torch.ones(pages, hkv)
    a = (q, k, v, ks, vs, [list(range(pages))], [length], [0, n])
    want, got = po.attention(*a, mask=mask), do.attention(*a, [-1] * n, mask=mask)
    for x, y in zip(got, want):
        fin = torch.isfinite(y)
        assert torch.equal(fin, torch.isfinite(x))
        assert (x - y)[fin].abs().max() < 1e-12


# 4096 requests of 8 queries each, 64 query and 8 K/V heads, tables of a million tokens: in units of 16 rows the line of
# key tiles does not fit 32 bits, in units of 256 it does.
WIDE = dict(PAGED, head_dim=128, heads=64, heads_kv=8, max_q=64, batch=4096, tokens=4096 * 8, num_pages=16384,
            table_width=16384, table_stride=16384, cu_q=A, q_stride=(8192, 128), o_stride=(8192, 128))


@pytest.mark.parametrize("change,served", [
    (dict(), True),  # (both: in units of 256)
    (dict(table_width=1000), True),
    (dict(tokens=4096 * 64), True),
    (dict(max_q=6), True),  # without trees refused; with them served
    (dict(table_width=1 << 24, table_stride=1 << 24, num_pages=1 << 24), False),
    (dict(max_q=6, table_width=1 << 24, table_stride=1 << 24, num_pages=1 << 24), False)])
def test_workspace_of_wide_tables(lib, change, served):
    """A size for each call that chia_paged_attn or chia_tree_attn serves."""
    n = lib.chia_paged_attn_workspace_bytes(packed(N.PagedParams, **{**WIDE, **change}))
    assert n > 0 if served else n == -1


@pytest.mark.parametrize("change,code", [(dict(abi_version=3), 1), (dict(abi_version=2, slots=A + 2), 3),
                                         (dict(abi_version=2, slots=A, tokens=-1), 1), (dict(abi_version=1, slots=A + 2), 6),
                                         (dict(abi_version=2), 6), (dict(abi_version=2, slots=A, tokens=8), 6)])
def test_compact_refusals_with_slots(lib, change, code):
    """(6: no GPU here, the arguments were taken. Version 1 has no slots.)"""
    if code == 6 and torch.cuda.is_available():
        pytest.skip("would launch")
    assert lib.chia_cache_compact(packed(N.CompactParams, **{**COMPACT, **change}), None) == code
