"""PagedCorpus.search on the GPU: which documents it returns and in what order."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _queries(bq, nq, d, seed, dtype=torch.float16):
    return torch.nn.functional.normalize(torch.randn(bq, nq, d, generator=_rng(seed)), dim=-1).to(dtype).cuda()


def _corpus(lengths, d, seed, kinds=None, max_docs=None):
    """A corpus of the given lengths; `kinds`: so many different documents, given out in turn."""
    from tilemaxsim_b200 import PagedCorpus
    g = _rng(seed)
    n = len(lengths)
    pool = [torch.randn(max(lengths), d, generator=g).half() for _ in range(kinds or n)]
    c = PagedCorpus(d, n_pages=sum(-(-m // 16) for m in lengths) + 1, max_docs=max_docs or n, page_size=16)
    c.add(torch.cat([pool[i % len(pool)][:m] for i, m in enumerate(lengths)]).cuda(), lengths)
    return c


def _best(scores, ids, k):
    """By score descending, NaN last, then by id: one row's k best (score, id) pairs."""
    order = sorted(range(len(ids)), key=lambda i: (np.isnan(scores[i]), -scores[i] if scores[i] == scores[i] else 0, ids[i]))
    return [scores[i] for i in order[:k]], [ids[i] for i in order[:k]]


@pytest.mark.parametrize("n_cand", [100, 16384, 16385, 30000])
@pytest.mark.parametrize("bq", [1, 3])
def test_candidates_of_any_number_and_order(bq, n_cand, cuda_device):
    """Unsorted candidate lists, some ids more than once, many documents of equal scores."""
    c = _corpus([1, 2, 3] * 6000, 16, 1, kinds=96)
    ids = torch.cat([torch.randperm(c.n_docs, generator=_rng(2)), torch.randint(0, c.n_docs, (12000,), generator=_rng(3))])
    ids = ids[torch.randperm(30000, generator=_rng(4))][:n_cand]
    Q = _queries(bq, 8, 16, 5)
    k = 100
    vals, got = c.search(Q, k, ids.cuda())
    assert vals.shape == got.shape == (bq, k) and got.dtype == torch.int64
    full = c.score_queries(Q).cpu().numpy()
    for q in range(bq):
        want_v, want_i = _best(full[q][ids.numpy()], ids.tolist(), k)
        assert got[q].tolist() == want_i
        np.testing.assert_array_equal(vals[q].cpu().numpy(), want_v)
    one_v, one_i = c.search(Q[0], k, ids.to(torch.int32).cuda())
    assert torch.equal(one_v, vals[0]) and torch.equal(one_i, got[0])
