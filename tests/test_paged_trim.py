"""chia_trim_pages (include/chia_paged.h) and its Python form without a GPU: refusals before anything is launched."""

import pytest
import torch

import chia_proj_b200 as cp
from chia_proj_b200 import _native as N
from test_paged import A, TABLES, packed


@pytest.mark.parametrize("change,code", [
    (dict(abi_version=9), 1), (dict(page_size=48), 2), (dict(batch=0), 1), (dict(table_stride=7), 1), (dict(ring_size=0), 1),
    (dict(seq_lens=None), 1), (dict(new_lens=None), 1), (dict(free_pages=None), 1), (dict(new_seq_lens=A), 1),
    (dict(new_free_state=A), 1), (dict(block_table=A + 2), 3),
])
def test_refusals(lib, change, code):
    assert lib.chia_trim_pages(packed(N.TablesParams, **{**TABLES, **change}), None) == code
    assert lib.chia_trim_pages(None, None) == 1


def test_python_form(lib):
    i = torch.zeros(2, dtype=torch.int32)
    args = (i, torch.zeros(2, 4, dtype=torch.int32), i, i)
    for done, keep in ((None, None), (i, i)):
        with pytest.raises(ValueError, match="either done or keep_lens"):
            cp.release_pages(done, *args, page_size=16, keep_lens=keep)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        cp.release_pages(None, *args, page_size=16, keep_lens=i)
