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


# ------------------------------------------------------------------------------------------ documents without tokens

def _with_gaps(cuda_device, n=40, nan_doc=37):
    """Documents of which one has a NaN, one was added empty, and several were removed."""
    from tilemaxsim_b200 import PagedCorpus
    lengths = [3] * n
    lengths[11] = 0
    x = torch.randn(sum(lengths), 16, generator=_rng(1)).half()
    x[sum(lengths[:nan_doc])] = float("nan")
    c = PagedCorpus(16, n_pages=n, max_docs=n + 5, page_size=16)
    c.add(x.cuda(), lengths)
    gone = [0, 1, 5, 20, 38, 39]
    c.remove(gone)
    return c, [i for i in range(n) if i not in gone and i != 11]


@pytest.mark.parametrize("single", [False, True])
def test_search_of_all_returns_documents_with_tokens_only(single, cuda_device):
    """k above the number of documents with tokens: they come first, one with a NaN after the others,
    then (-inf, -1)."""
    c, live = _with_gaps(cuda_device)
    Q = _queries(1 if single else 3, 5, 16, 2)
    full = c.score_queries(Q).cpu().numpy()
    for k in (1, len(live) - 1, len(live), len(live) + 2, 40):
        vals, ids = c.search(Q[0] if single else Q, k)
        vals, ids = (vals[None], ids[None]) if single else (vals, ids)
        assert vals.shape == ids.shape == (len(Q), k)
        for q in range(len(Q)):
            want_v, want_i = _best(full[q][live], live, k)
            more = k - len(want_i)
            assert ids[q].tolist() == want_i + [-1] * more
            np.testing.assert_array_equal(vals[q].cpu().numpy(), want_v + [-np.inf] * more)
    c.remove(live)
    vals, ids = c.search(Q, 7)
    assert (ids == -1).all() and (vals == float("-inf")).all()


@pytest.mark.parametrize("repeat", [1, 700])
def test_search_of_candidates_puts_those_without_tokens_last(repeat, cuda_device):
    """After the documents with tokens, one with a NaN among them: removed and empty candidates by
    their ids, then ids outside the corpus, as -1."""
    c, live = _with_gaps(cuda_device)
    Q = _queries(3, 5, 16, 2)
    full = c.score_queries(Q).cpu().numpy()
    cand = [37, 0, 4, 45, 11, -1, 39, 2, 30, -(1 << 40), 1 << 50, 3, 44, 5, 40] * repeat
    cand += [8, 9] * (20000 - len(cand)) if repeat > 1 else [8, 9]
    here = [i for i in cand if i in live]
    empty = sorted(i for i in cand if 0 <= i < 40 and i not in live)
    outside = len(cand) - len(here) - len(empty)
    ids_in = torch.tensor(cand)[torch.randperm(len(cand), generator=_rng(3))].cuda()
    for k in (1, len(here) - 1, len(here) + 1, len(here) + len(empty) + 2, len(cand)):
        if k > 2048:
            continue
        vals, ids = c.search(Q, k, ids_in)
        for q in range(3):
            want_v, want_i = _best(full[q][here], here, k)
            want_i = (want_i + empty + [-1] * outside)[:k]
            want_v += [-np.inf] * (k - len(want_v))
            assert ids[q].tolist() == want_i
            np.testing.assert_array_equal(vals[q].cpu().numpy(), want_v)
    if repeat > 1:  # mostly candidates without tokens
        few = ids_in.clone()
        few[torch.isin(few, torch.tensor([8, 9, 2, 3, 4, 30]).cuda())] = -7
        here = [i for i in few.tolist() if i == 37]
        vals, ids = c.search(Q, 2000, few)
        assert (ids[:, :700] == 37).all() and torch.isnan(vals[:, :700]).all()
        assert len(here) == 700 and (ids[:, 700:] == torch.tensor(empty[:1300]).cuda()).all()
        assert (vals[:, 700:] == float("-inf")).all()


def test_search_of_candidates_in_an_empty_corpus(cuda_device):
    from tilemaxsim_b200 import PagedCorpus
    c = PagedCorpus(16, 4, 4, page_size=16)
    vals, ids = c.search(_queries(2, 5, 16, 2), 2, torch.tensor([0, 3, -1, 9], device=cuda_device))
    assert (ids == -1).all() and (vals == float("-inf")).all()


@pytest.mark.parametrize("n", [40, 20000])
def test_captured_search_pads_what_is_removed_later(n, cuda_device):
    from tilemaxsim_b200 import GraphedStep
    c = _corpus([1] * n, 16, 1)
    Q = _queries(2, 5, 16, 2)
    cand = torch.tensor([7, 3, 5, 1], device=cuda_device)
    step = GraphedStep(lambda q: c.search(q, 4), Q)
    some = GraphedStep(lambda q, i: c.search(q, 4, i), Q, cand)
    want = c.search(Q, 4)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(step(Q), want))
    keep = [2, 5]
    c.remove([i for i in range(n) if i not in keep])
    vals, ids = step(Q)
    full = c.score_queries(Q).cpu()
    assert (ids[:, 2:] == -1).all() and (vals[:, 2:] == float("-inf")).all()
    for q in range(2):
        want_v, want_i = _best(full[q, keep].tolist(), keep, 2)
        assert ids[q, :2].tolist() == want_i and vals[q, :2].tolist() == want_v
    vals, ids = some(Q, cand)
    assert ids.tolist() == [[5, 1, 3, 7]] * 2 and torch.equal(vals[:, 0], full[:, 5]) and torch.isinf(vals[:, 1:]).all()


def test_lowest_scores_keep_their_order(cuda_device):
    """Scores that overflow to -inf belong to documents with tokens: after them a NaN, then the padding."""
    from tilemaxsim_b200 import PagedCorpus
    c = PagedCorpus(16, n_pages=8, max_docs=8, page_size=16)
    x = torch.full((5, 16), 1e30)
    x[1] *= -1
    x[3] = float("nan")
    c.add(x.cuda(), [1] * 5, norm="none")
    c.remove([0])
    vals, ids = c.search(torch.full((1, 4, 16), 1e30, dtype=torch.bfloat16, device=cuda_device), 5)
    assert ids.tolist() == [[2, 4, 1, 3, -1]]
    assert vals[0, :3].tolist() == [float("inf")] * 2 + [float("-inf")] and vals[0, 3].isnan() and vals[0, 4] == float("-inf")
    vals, ids = c.search(torch.full((1, 4, 16), 1e30, dtype=torch.bfloat16, device=cuda_device), 5,
                         torch.tensor([0, 1, 2, 3, 4], device=cuda_device))
    assert ids.tolist() == [[2, 4, 1, 3, 0]] and vals[0, 3].isnan()


def test_ivf_returns_documents_that_score_minus_infinity(cuda_device):
    """Only documents without tokens are padding, not those whose scores overflow."""
    from tilemaxsim_b200 import IVFIndex, PagedCorpus
    c = PagedCorpus(16, n_pages=8, max_docs=8, page_size=16)
    x = torch.full((5, 16), 1e30)
    x[1:4] *= -1
    c.add(x.cuda(), [1] * 5, norm="none")
    index = IVFIndex(torch.ones(1, 16, device=cuda_device), torch.zeros(5, dtype=torch.int64, device=cuda_device),
                     torch.arange(6, device=cuda_device))
    Q = torch.full((2, 4, 16), 1e30, dtype=torch.bfloat16, device=cuda_device)
    c.remove([2, 4])
    for k in (3, 5):
        vals, ids = index.search(Q, c, k, nprobe=1)
        assert ids.tolist() == [[0, 1, 3, -1, -1][:k]] * 2
        assert vals[:, 0].tolist() == [float("inf")] * 2 and (vals[:, 1:] == float("-inf")).all()
