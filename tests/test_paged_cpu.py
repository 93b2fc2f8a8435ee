"""The paged 8-bit corpus without a GPU: refusals of the Python layer and of the C ABI, and the plain
restatement that the GPU tests compare with."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import paged_ref as R


def _tables(n=2, cap=4):
    from tilemaxsim_b200 import PageTables
    return PageTables(torch.zeros(n + 1, dtype=torch.int64), torch.zeros(cap, dtype=torch.int32),
                      torch.zeros(cap, dtype=torch.int32), torch.zeros(n + 1, dtype=torch.int64), None)


def _pool(n=4, page=32, d=128):
    return torch.zeros(n, page, d, dtype=torch.float8_e4m3fn), torch.zeros(n)


def test_cpu_tensors_are_rejected():
    from tilemaxsim_b200 import PagedCorpus, page_read, page_tables, page_write, paged_maxsim, select_page_tables
    codes, scales = _pool()
    n = torch.tensor([3, 5])
    with pytest.raises(ValueError, match="CUDA"):
        page_tables(n, 32, torch.arange(4, dtype=torch.int32), 8)
    with pytest.raises(ValueError, match="CUDA"):
        select_page_tables(n, 32, torch.tensor([0, 1, 2]), torch.arange(2, dtype=torch.int32), torch.tensor([0]), 8)
    with pytest.raises(ValueError, match="CUDA"):
        page_write(torch.zeros(8, 128).half(), _tables(), codes, scales)
    with pytest.raises(ValueError, match="CUDA"):
        page_read(codes, scales, torch.tensor([0]))
    with pytest.raises(ValueError, match="CUDA"):
        paged_maxsim(torch.zeros(1, 32, 128).half(), codes, scales, _tables())
    with pytest.raises(ValueError, match="CUDA"):
        PagedCorpus(128, 10, 10, device="cpu")


@pytest.mark.parametrize("page", [0, 8, 24, 256])
def test_page_sizes(page):
    from tilemaxsim_b200 import PagedCorpus, page_tables
    with pytest.raises(ValueError, match="page_size"):
        page_tables(torch.tensor([3]), page, torch.arange(4, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="page_size"):
        PagedCorpus(128, 10, 10, page_size=page)


@pytest.mark.parametrize("d", [0, 8, 100, 272])
def test_token_widths(d):
    from tilemaxsim_b200 import PagedCorpus, page_read
    with pytest.raises(ValueError, match="multiple of 16"):
        PagedCorpus(d, 10, 10)
    with pytest.raises(ValueError, match="multiple of 16"):
        page_read(*_pool(d=d), torch.tensor([0]))


def test_argument_refusals():
    from tilemaxsim_b200 import PagedCorpus, page_read, page_tables, page_write, paged_maxsim
    codes, scales = _pool()
    t = _tables()
    x = torch.zeros(8, 128).half()
    for bad in (torch.tensor([1.5]), torch.tensor([[1]]), torch.tensor([True])):
        with pytest.raises(ValueError, match="integer"):
            page_tables(bad, 32, torch.arange(4, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="n_tokens"):
        page_tables(torch.tensor([1]), 32, torch.arange(4, dtype=torch.int32), -1)
    with pytest.raises(ValueError, match="norm"):
        page_write(x, t, codes, scales, norm="max")
    with pytest.raises(ValueError, match="weight"):
        page_write(x, t, codes, scales, weight=torch.ones(128).half())
    with pytest.raises(ValueError, match="eps"):
        page_write(x, t, codes, scales, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        page_write(x, t, codes, scales, eps=float("nan"))
    with pytest.raises(ValueError, match="float8"):
        page_read(codes.view(torch.uint8), scales, torch.tensor([0]))
    with pytest.raises(ValueError, match="scales"):
        page_read(codes, scales.double(), torch.tensor([0]))
    with pytest.raises(ValueError, match="scales"):
        paged_maxsim(torch.zeros(32, 128).half(), codes, scales[:3], t)
    with pytest.raises(ValueError, match="contiguous"):
        page_read(codes[:, :, :64], scales, torch.tensor([0]))
    with pytest.raises(ValueError, match="int32"):
        paged_maxsim(torch.zeros(32, 128).half(), codes, scales, t._replace(page_ids=t.page_ids.long()))
    with pytest.raises(ValueError, match="same length"):
        paged_maxsim(torch.zeros(32, 128).half(), codes, scales, t._replace(page_ids=t.page_ids[:2]))
    with pytest.raises(ValueError, match="n_docs"):
        paged_maxsim(torch.zeros(32, 128).half(), codes, scales, t._replace(token_offsets=t.token_offsets[:2]))
    with pytest.raises(ValueError, match="2\\^31"):
        PagedCorpus(128, 1 << 27, 10)


def test_c_abi_refusals_without_gpu():
    from tilemaxsim_b200 import _lib as L
    lib, nul = L.load(), ctypes.c_void_p(0)
    p = ctypes.c_void_p(1 << 20)  # an aligned address that is never read: every call below is refused or empty
    odd = ctypes.c_void_p((1 << 20) + 8)

    def tables(lengths=p, n=5000, page=32, po=p, ids=p, cap=4, ws=p, wsb=1 << 20):
        return lib.tms_page_tables(lengths, n, nul, 5000, nul, p, 4, page, po, p, ids, p, cap, nul, 0, ws, wsb, nul)

    assert tables(page=24) == L.TMS_ERR_UNSUPPORTED
    assert tables(n=1) == L.TMS_ERR_INVALID  # fewer lengths than documents
    assert tables(lengths=nul) == tables(po=nul) == tables(ids=nul) == tables(cap=-1) == L.TMS_ERR_INVALID
    assert tables(ws=nul) == tables(wsb=0) == L.TMS_ERR_WORKSPACE
    assert tables(cap=1 << 31) == L.TMS_ERR_UNSUPPORTED

    def write(x=p, dt=0, rows=8, st=128, w=nul, norm=1, eps=0.0, d=128, page=32, n=2, cap=4, codes=p):
        return lib.tms_page_write(x, dt, rows, 0, st, 0, nul, w, norm, ctypes.c_float(eps), d, page, p, p, p, p, n,
                                  cap, codes, p, 4, nul)

    assert write(dt=9) == write(norm=3) == write(w=p) == write(eps=-1.0) == write(x=nul) == L.TMS_ERR_INVALID
    assert write(x=odd) == write(codes=odd) == write(st=100) == L.TMS_ERR_INVALID
    assert write(d=100) == write(d=272) == write(page=33) == L.TMS_ERR_UNSUPPORTED
    assert write(n=0) == write(cap=0) == L.TMS_OK

    def read(codes=p, d=128, page=32, n=4, out=p, dt=0):
        return lib.tms_page_read(codes, p, 4, page, d, p, n, out, dt, nul)

    assert read(dt=5) == read(n=-1) == read(out=nul) == read(codes=odd) == read(out=odd) == L.TMS_ERR_INVALID
    assert read(d=24) == read(page=8) == L.TMS_ERR_UNSUPPORTED
    assert read(n=0) == L.TMS_OK

    def score(Q=p, dt=0, nb=1, nq=32, d=128, codes=p, pages=4, page=32, n=2, cap=4, out=p, ws=p, wsb=1 << 30):
        return lib.tms_paged_maxsim(Q, dt, nb, nq, d, codes, p, pages, page, p, p, p, n, cap, out, ws, wsb, nul)

    assert score(dt=L.TMS_F32) == score(nb=-1) == score(nq=0) == score(Q=nul) == score(out=nul) == L.TMS_ERR_INVALID
    assert score(Q=odd) == score(codes=odd) == L.TMS_ERR_INVALID
    assert score(d=40) == score(d=512) == score(page=48) == score(pages=1 << 27) == L.TMS_ERR_UNSUPPORTED
    assert score(nb=0) == score(n=0) == L.TMS_OK
    need = lib.tms_paged_workspace_size(1, 64, 128, 2, 32, 4)
    if need:
        assert score(nq=64, ws=nul) == score(nq=64, wsb=need - 1) == L.TMS_ERR_WORKSPACE


def test_reference_tables():
    po, ids, docs, to, slots = R.tables([3, 0, 17, 16], 16, [7, 4, 9, 2], 36)
    assert po.tolist() == [0, 1, 1, 3, 4] and to.tolist() == [0, 3, 3, 20, 36]
    assert ids.tolist() == [7, 4, 9, 2, -1, -1] and docs.tolist() == [0, 2, 2, 3, -1, -1]
    assert slots[:4].tolist() == [112, 113, 114, 64] and slots[19] == 144 and slots[20] == 32
    _, ids, docs, to, slots = R.tables([3, 0, 17, 16], 16, [7, 4, 9, 2], 40, doc_ids=[2, 9, 2], src_offsets=po)
    assert ids[:4].tolist() == [4, 9, 4, 9] and docs[:4].tolist() == [0, 0, 2, 2] and to.tolist() == [0, 17, 17, 34]
    assert (slots[34:] == -1).all() and (slots[:17] == slots[17:34]).all()


def test_reference_rounding_is_torchs():
    """half_step and torch's own conversion agree: every value is within half a step of its code."""
    t = np.random.default_rng(1).normal(size=20000) * np.exp(np.random.default_rng(2).uniform(-9, 6, 20000))
    t = np.clip(t, -448, 448).astype(np.float32)
    code = torch.from_numpy(t).to(torch.float8_e4m3fn).double().numpy()
    assert (np.abs(code - t) <= R.half_step(t.astype(np.float64))).all()
