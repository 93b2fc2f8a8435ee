"""Refusals of the paged corpus that need no GPU, beside those of test_paged_cpu.py."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch


def test_topk_docs_refusals():
    from tilemaxsim_b200 import _lib as L
    lib, nul = L.load(), ctypes.c_void_p(0)
    p = ctypes.c_void_p(1 << 20)  # never read: every call below is refused or empty
    odd = ctypes.c_void_p((1 << 20) + 8)

    def call(s=p, rows=2, n=10, ld=10, k=3, ids=nul, lengths=p, docs=10, v=p, o=p, ws=p, wsb=1 << 20):
        return lib.tms_topk_docs(s, rows, n, ld, k, ids, lengths, docs, v, o, ws, wsb, nul)

    assert call(rows=-1) == call(ld=9) == call(k=11) == call(docs=-1) == L.TMS_ERR_INVALID
    assert call(s=nul) == call(lengths=nul) == call(v=nul) == call(o=nul) == call(ws=odd) == L.TMS_ERR_INVALID
    assert call(n=5000, ld=5000, k=2049) == L.TMS_ERR_UNSUPPORTED
    assert call(ws=nul) == call(wsb=79) == L.TMS_ERR_WORKSPACE
    assert call(rows=0) == call(k=0) == L.TMS_OK
    assert lib.tms_topk_docs_workspace_size(2, 10, 3) == 80
    assert lib.tms_topk_docs_workspace_size(2, 0, 3) == 0
    assert lib.tms_topk_docs_workspace_size(1, 100000, 10) > 800000


def _tables(n=2, cap=4):
    from tilemaxsim_b200 import PageTables
    return PageTables(torch.zeros(n + 1, dtype=torch.int64), torch.zeros(cap, dtype=torch.int32),
                      torch.zeros(cap, dtype=torch.int32), torch.zeros(n + 1, dtype=torch.int64), None)


@pytest.mark.parametrize("eps", [1e-50, 7e-46, 5e-324, 3.5e38, 1e39, 1e308])
@pytest.mark.parametrize("norm", ["l2", "rms", "none"])
def test_eps_outside_fp32(eps, norm):
    """The kernel takes eps in fp32: one that becomes nothing or infinite there is refused."""
    from tilemaxsim_b200 import page_write
    codes, scales = torch.zeros(4, 32, 128, dtype=torch.float8_e4m3fn), torch.zeros(4)
    with pytest.raises(ValueError, match="eps"):
        page_write(torch.zeros(8, 128).half(), _tables(), codes, scales, norm=norm, eps=eps)


@pytest.mark.parametrize("eps", [0.0, 1.5e-45, 1e-12, 3.4e38])
def test_eps_inside_fp32(eps):
    from tilemaxsim_b200 import page_write
    codes, scales = torch.zeros(4, 32, 128, dtype=torch.float8_e4m3fn), torch.zeros(4)
    with pytest.raises(ValueError, match="CUDA"):  # the next check
        page_write(torch.zeros(8, 128).half(), _tables(), codes, scales, eps=eps)


def test_c_abi_refuses_an_infinite_eps():
    from tilemaxsim_b200 import _lib as L
    lib, nul, p = L.load(), ctypes.c_void_p(0), ctypes.c_void_p(1 << 20)
    for norm in (0, 1, 2):
        for eps in (float("inf"), float("nan"), -1.0, -float("inf")):
            # no documents: refused before there is anything to do, or to read
            assert lib.tms_page_write(p, 0, 8, 0, 128, 0, nul, nul, norm, ctypes.c_float(eps), 128, 32, p, p, p, p, 0,
                                      4, p, p, 4, nul) == L.TMS_ERR_INVALID


@pytest.mark.parametrize("lengths", [
    [(1 << 63) - 1, (1 << 63) - 1, 2], [(1 << 62)] * 4, [(1 << 63) - 8, 8, 1 << 63], [1 << 40], np.array([(1 << 64) - 3, 3], np.uint64),
    torch.tensor([(1 << 63) - 1, (1 << 63) - 1, 2]), [(1 << 63) - 1] * 2 + [2] + [0] * 5])
def test_add_refuses_lengths_whose_sum_wraps(lengths):
    """Their sum, or the pages they round up to, leaves 64 bits: refused on the host, the corpus as it was."""
    from tilemaxsim_b200 import PagedCorpus
    c = PagedCorpus.__new__(PagedCorpus)
    c.page_size, c.d, c.n_pages, c.max_docs, c.n_docs, c.n_free, c.device = 16, 32, 10, 10, 0, 10, torch.device("cpu")
    with pytest.raises(ValueError, match="pages are needed|negative|sum to|integers"):
        c.add(torch.zeros(0, 32).half(), lengths)
    assert c.n_docs == 0 and c.n_free == 10
