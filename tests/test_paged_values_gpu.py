"""Values at which the paged corpus operators could go wrong: page ids past 32 bits, exact ties, wide queries."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _pool(n_pages, page, d):
    return (torch.zeros(n_pages, page, d, device="cuda").to(torch.float8_e4m3fn), torch.zeros(n_pages, device="cuda"))


@pytest.mark.parametrize("bad", [1 << 32, (1 << 32) + 2, (1 << 33) + 1, -(1 << 32) + 3, (1 << 40), -(1 << 63), (1 << 63) - 1])
def test_page_ids_of_64_bits_do_not_wrap(bad, cuda_device):
    """An id outside the pool is left out, also one whose low 32 bits name a page of it."""
    from tilemaxsim_b200 import page_tables, page_write, select_page_tables
    ids = torch.tensor([3, bad, 1], device=cuda_device)
    t = page_tables(torch.tensor([16, 16, 16], device=cuda_device), 16, ids, 48)
    got = t.page_ids.tolist()
    assert got[0] == 3 and got[2] == 1 and not 0 <= got[1] < 1 << 27
    codes, scales = _pool(4, 16, 32)
    page_write(torch.ones(48, 32, device=cuda_device).half(), t, codes, scales)
    assert (scales > 0).tolist() == [False, True, False, True]
    lengths, offsets = torch.tensor([16, 16, 16], device=cuda_device), torch.arange(4, device=cuda_device)
    s = select_page_tables(lengths, 16, offsets, ids, torch.tensor([1, 2], device=cuda_device), 32)
    assert not 0 <= s.page_ids[0].item() < 1 << 27 and s.page_ids[1].item() == 1
