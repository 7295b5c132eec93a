"""The C ABI of the paged 8-bit K/V cache (include/chia_paged.h) and its Python entry points, without a GPU:
exports, struct layouts, refusals before anything is launched."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import chia_proj_b200 as cp
from chia_proj_b200 import _native as N

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "chia_paged.h")
STRUCTS = {"chia_tables_params_t": N.TablesParams, "chia_append_params_t": N.AppendParams,
           "chia_paged_params_t": N.PagedParams}


def test_exports(lib):
    declared = set(re.findall(r"CHIA_API\s+[\w\s\*]*?\b(chia_\w+)\s*\(", open(HEADER).read()))
    assert declared == set(N.PAGED_SYMBOLS)
    for name in declared:
        assert hasattr(lib, name)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
@pytest.mark.parametrize("name", list(STRUCTS))
def test_struct_layout_matches_header(tmp_path, name):
    fields = [f[0] for f in STRUCTS[name]._fields_]
    prog = ["#include <stdio.h>", "#include <stddef.h>", '#include "chia_paged.h"', "int main(void){",
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


TABLES = dict(abi_version=1, page_size=64, batch=4, table_width=8, table_stride=8, ring_size=32, max_tokens=4,
              seq_lens=A, new_lens=A, block_table=A, free_pages=A, free_state=A, slots=A, positions=A, cu_q=A,
              new_seq_lens=2 * A, new_free_state=2 * A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=9), 1), (dict(page_size=48), 2), (dict(batch=0), 1), (dict(table_stride=7), 1),
    (dict(ring_size=0), 1), (dict(max_tokens=-1), 1), (dict(seq_lens=None), 1), (dict(slots=None), 1),
    (dict(cu_q=None), 1), (dict(new_seq_lens=A), 1), (dict(new_free_state=A), 1), (dict(block_table=A + 2), 3),
])
def test_tables_refusals(lib, change, code):
    assert lib.chia_page_tables(packed(N.TablesParams, **{**TABLES, **change}), None) == code
    if not set(change) & {"slots", "cu_q"}:
        assert lib.chia_release_pages(packed(N.TablesParams, **{**TABLES, **change}), None) == code
    assert lib.chia_page_tables(None, None) == 1


APPEND = dict(abi_version=1, dtype=0, cache_dtype=0, head_dim=128, heads_kv=4, page_size=64, tokens=8, num_pages=10,
              k=A, v=A, k_stride=(512, 128), v_stride=(512, 128), slots=A, k_cache=A, v_cache=A, k_scale=A, v_scale=A)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=0), 1), (dict(dtype=2), 2), (dict(cache_dtype=2), 2), (dict(head_dim=96), 2),
    (dict(page_size=8), 2), (dict(heads_kv=0), 1), (dict(tokens=-1), 1), (dict(num_pages=0), 1),
    (dict(num_pages=2 ** 26), 1), (dict(k=None), 1), (dict(slots=None), 1), (dict(v_cache=None), 1),
    (dict(k=A + 8), 3), (dict(k_stride=(511, 128)), 3), (dict(v_stride=(-512, 128)), 1), (dict(k_scale=A + 1), 3),
])
def test_append_refusals(lib, change, code):
    assert lib.chia_cache_append(packed(N.AppendParams, **{**APPEND, **change}), None) == code
    assert lib.chia_cache_append(None, None) == 1


PAGED = dict(abi_version=1, dtype=0, cache_dtype=0, head_dim=128, norm=0, mod=0, heads=8, heads_kv=2, page_size=64,
             max_q=1, batch=4, tokens=4, num_pages=10, table_width=5, table_stride=5, q=A, o=A, q_stride=(1024, 128),
             o_stride=(1024, 128), k_cache=A, v_cache=A, k_scale=A, v_scale=A, block_table=A, seq_lens=A, scale=0.1,
             softcap=30.0, out_scale=1.0, win_left=-1, dilation=1, workspace=A, workspace_bytes=1 << 40)


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=0), 1), (dict(dtype=2), 2), (dict(cache_dtype=-1), 2), (dict(head_dim=256), 2),
    (dict(norm=3), 1), (dict(mod=4), 1), (dict(norm=1, mod=1), 2), (dict(heads=9), 1), (dict(max_q=0), 1),
    (dict(page_size=24), 2), (dict(batch=0), 1), (dict(tokens=5), 1), (dict(num_pages=2 ** 40), 1),
    (dict(table_stride=4), 1), (dict(q=None), 1), (dict(k_scale=None), 1), (dict(block_table=None), 1),
    (dict(mod=2), 1), (dict(mod=1, softcap=0.0), 1), (dict(scale=float("nan")), 1), (dict(dilation=0), 1),
    (dict(win_left=-2), 1), (dict(q=A + 2), 3), (dict(o_stride=(1024, 100)), 3), (dict(workspace=None), 1),
    (dict(workspace_bytes=8), 1), (dict(workspace=A + 16), 3), (dict(lse=A + 2), 3),
])
def test_paged_refusals(lib, change, code):
    assert lib.chia_paged_attn(packed(N.PagedParams, **{**PAGED, **change}), None) == code
    assert lib.chia_paged_attn(None, None) == 1
    if not set(change) & {"workspace", "workspace_bytes"}:
        assert lib.chia_paged_attn_workspace_bytes(packed(N.PagedParams, **{**PAGED, **change})) == -1
    assert lib.chia_paged_attn_workspace_bytes(packed(N.PagedParams, **PAGED)) > 0


def test_no_cpu_fallback(lib):
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.page_tables(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i, page_size=16, max_tokens=2)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.release_pages(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i, page_size=16)
    cache = cp.new_cache(2, 1, 64, page_size=16, device="cpu")
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.cache_append(x, x, i, *cache)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.paged_attention(x, *cache, torch.zeros(2, 4, dtype=torch.int32), i)


def test_new_cache_refusals():
    for kw in (dict(page_size=20), dict(dtype=torch.float16), dict(head_dim=80)):
        with pytest.raises(ValueError):
            cp.new_cache(**{**dict(num_pages=2, heads_kv=1, head_dim=64, device="cpu"), **kw})
    k, v, ks, vs = cp.new_cache(3, 2, 64, page_size=32, dtype=torch.int8, device="cpu")
    assert k.shape == v.shape == (3, 2, 32, 64) and k.dtype == torch.int8 and ks.shape == vs.shape == (3, 2)


@pytest.mark.gpu
def test_python_refusals(cuda):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    cache = cp.new_cache(4, 2, 128, page_size=16)
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16, device="cuda")
    k = q[:, :2]
    table, lens = i32(2, 3), i32(2)
    bad_q = [q.float(), q[0], q[..., :64], q[:, :3], torch.zeros(3, 4, 128, dtype=torch.bfloat16, device="cuda"),
             q.clone().requires_grad_()]
    for x in bad_q:
        with pytest.raises(ValueError):
            cp.paged_attention(x, *cache, table, lens)
    for kw in (dict(norm="x"), dict(mod="x"), dict(norm="relu", mod="temp"), dict(norm="relu", return_lse=True),
               dict(max_q=0), dict(out=q[:1]), dict(mask=cp.Mask(dilation=0)), dict(cu_q=lens), dict(wait_limit_ns=-1),
               dict(mod="alibi", head_param=[1.0])):
        with pytest.raises(ValueError):
            cp.paged_attention(q, *cache, table, lens, **kw)
    with pytest.raises(ValueError):
        cp.paged_attention(q, *cache, table.long(), lens)
    with pytest.raises(ValueError):
        cp.paged_attention(q, *cache, table, i32(3))
    with pytest.raises(ValueError):
        cp.paged_attention(q, cache[0], cache[1].view(torch.int8), *cache[2:], table, lens)
    with pytest.raises(ValueError):
        cp.paged_attention(q, *cache[:2], cache[2][:, :1], cache[3], table, lens)
    for args in ((k.float(), k), (k, k.half()), (k[:1], k), (q, q)):
        with pytest.raises(ValueError):
            cp.cache_append(*args, lens, *cache)
    with pytest.raises(ValueError):
        cp.cache_append(k, k, i32(3), *cache)
    ring, state = i32(5), i32(2)
    for kw in (dict(page_size=8), dict(max_tokens=-1)):
        with pytest.raises(ValueError):
            cp.page_tables(lens, lens, table, ring, state, **{**dict(page_size=16, max_tokens=2), **kw})
    for args in ((lens, lens[:1], table, ring, state), (lens, lens, table.t(), ring, state),
                 (lens, lens, table, ring, ring), (lens.long(), lens, table, ring, state)):
        with pytest.raises(ValueError):
            cp.page_tables(*args, page_size=16, max_tokens=2)
    cp.check_device_status(0)
