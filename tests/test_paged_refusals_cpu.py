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
