"""PagedCorpus on the GPU over a long life: more documents than it has rows, captured selections."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _queries(bq, nq, d, seed, dtype=torch.float16):
    return torch.nn.functional.normalize(torch.randn(bq, nq, d, generator=_rng(seed)), dim=-1).to(dtype).cuda()


def test_more_documents_than_rows(cuda_device):
    """Documents come and go, many times max_docs in all; compact keeps every document's tokens and scores."""
    from tilemaxsim_b200 import PagedCorpus
    d, page = 32, 16
    c = PagedCorpus(d, n_pages=64, max_docs=20, page_size=page)
    Q = _queries(2, 7, d, 1)
    g = _rng(2)
    kept: dict[int, torch.Tensor] = {}  # id -> the tokens it was given
    added = 0
    for step in range(25):
        lengths = torch.randint(0, 40, (int(torch.randint(1, 9, (1,), generator=g)),), generator=g).tolist()
        if c.n_docs + len(lengths) > c.max_docs:
            with pytest.raises(ValueError, match="compact"):
                c.add(torch.zeros(sum(lengths), d).half().cuda(), lengths)
            before = {i: (c.tokens([i], torch.float32)[0], c.score_queries(Q, torch.tensor([i]).cuda())) for i in kept}
            n = c.n_docs
            new = c.compact()
            assert new.shape == (n,) and new.dtype == torch.int64 and c.n_docs == len(kept)
            ids = new.tolist()
            assert [i for i in range(n) if ids[i] >= 0] == sorted(kept)
            assert [j for j in ids if j >= 0] == list(range(len(kept)))
            for i, (tok, score) in before.items():
                j = ids[i]
                assert torch.equal(c.tokens([j], torch.float32)[0], tok)
                assert torch.equal(c.score_queries(Q, torch.tensor([j]).cuda()), score)
            kept = {ids[i]: x for i, x in kept.items()}
        x = torch.randn(sum(lengths), d, generator=g).half()
        ids = c.add(x.cuda(), lengths).tolist()
        added += len(lengths)
        kept |= {i: v for i, v in zip(ids, x.split(lengths)) if len(v)}
        assert c.n_free == c.n_pages - sum(-(-len(v) // page) for v in kept.values())
        full = c.score_queries(Q)
        assert torch.isfinite(full[0]).nonzero().flatten().tolist() == sorted(kept)
        for i, v in kept.items():
            tok = c.tokens([i], torch.float32)[0].cpu()
            want = torch.nn.functional.normalize(v.float(), dim=-1)
            assert tok.shape == want.shape and (tok - want).abs().max() <= want.abs().max() * 2.0 ** -4 * 1.01
        gone = [i for i in kept if torch.rand(1, generator=g) < 0.4 or sum(map(len, kept.values())) > 400]
        c.remove(gone)
        kept = {i: v for i, v in kept.items() if i not in gone}
    assert added > 3 * c.max_docs
    c.remove(list(kept))
    c.compact()
    assert c.n_docs == 0 and c.n_free == c.n_pages and sorted(c._free.tolist()) == list(range(c.n_pages))
    assert c.compact().numel() == 0
    assert c.score_queries(Q).shape == (2, 0)


def test_tables_hold_the_entries_in_use(cuda_device):
    """Whether documents are cut over several ranges goes by their mean length, for which a table's capacity
    stands: the empty part of a large pool does not make short documents long."""
    from tilemaxsim_b200 import GraphedStep, PagedCorpus, _lib, paged_maxsim
    c = PagedCorpus(64, n_pages=20000, max_docs=500)
    Q = _queries(2, 32, 64, 1)
    assert c.tables.page_ids.numel() == 0 and c.score_queries(Q).shape == (2, 0)
    c.add(torch.randn(100 * 40, 64, generator=_rng(2)).half().cuda(), [40] * 100)
    t = c.tables
    assert t.page_ids.numel() == t.page_docs.numel() == 200 == int(t.page_offsets[-1])
    size = _lib.load().tms_paged_workspace_size
    assert size(2, 32, 64, 100, 32, 200) == 0 < size(2, 32, 64, 100, 32, 20000)
    want = paged_maxsim(Q, c.codes, c.scales, t._replace(page_ids=c._page_ids, page_docs=c._page_docs))
    assert torch.equal(c.score_queries(Q), want)
    # a captured call's tables serve what is left of its documents, whatever comes after them
    step = GraphedStep(c.score_queries, Q)
    assert torch.equal(step(Q), want.cpu())
    c.remove(list(range(0, 100, 3)))
    c.add(torch.randn(300 * 90, 64, generator=_rng(3)).half().cuda(), [90] * 300)
    got = step(Q)
    want[:, ::3] = -float("inf")
    assert torch.equal(got, want.cpu()) and torch.equal(got, c.score_queries(Q)[:, :100].cpu())
    c.remove(list(range(400)))
    assert c.tables.page_ids.numel() == 0 and torch.isinf(step(Q)).all() and torch.isinf(c.score_queries(Q)).all()


def test_captured_search_of_candidates_beside_a_long_document(cuda_device):
    """Candidates times the longest document is far more than the corpus holds: outside a capture the host
    looks at their own sum, within one it cannot wait and takes the bound."""
    from tilemaxsim_b200 import GraphedStep, PagedCorpus
    c = PagedCorpus(16, n_pages=3000, max_docs=2100, page_size=16)
    lengths = [1] * 1000 + [20000] + [3] * 700
    c.add(torch.randn(sum(lengths), 16, generator=_rng(1)).half().cuda(), lengths)
    Q = _queries(2, 4, 16, 5)
    pick = [torch.randint(0, 1701, (5000,), generator=_rng(s)).cuda() for s in (2, 3)]
    step = GraphedStep(lambda q, i: c.search(q, 10, i), Q, pick[0])
    for ids in (*pick, torch.full((5000,), 1000).cuda()):  # at last the long document, again and again
        want = c.search(Q, 10, ids)
        assert all(torch.equal(a, b.cpu()) for a, b in zip(step(Q, ids), want))


@pytest.mark.parametrize("bq,nq,d,page", [(1, 32, 128, 32), (2, 32, 64, 16), (4, 20, 128, 64), (20, 32, 128, 32), (3, 77, 256, 16)])
def test_alone_and_among_others(bq, nq, d, page, cuda_device):
    """A query by itself and in a batch, a document by itself, among candidates and in a corpus of many
    steps: every score is within the bound of 64 bits' over the tokens that the pages hold."""
    import paged_ref as R
    from tilemaxsim_b200 import PagedCorpus
    lengths = torch.randint(0, 130, (8000,), generator=_rng(d)).tolist()
    c = PagedCorpus(d, n_pages=sum(-(-n // page) for n in lengths), max_docs=8000, page_size=page)
    c.add(torch.randn(sum(lengths), d, generator=_rng(1)).half().cuda(), lengths)
    Q = _queries(bq, nq, d, 2, torch.bfloat16)
    pick = [i for i in torch.randperm(8000, generator=_rng(3))[:60].tolist() if lengths[i]][:40]
    tok, off = c.tokens(pick, torch.float32)
    docs = [v.cpu().double().numpy() for v in tok.split((off[1:] - off[:-1]).tolist())]
    q = Q.cpu().double().numpy()
    want, bound = R.scores(q, docs), R.score_bound(q, docs)
    ids = torch.tensor(pick, device=cuda_device)

    def check(got, w, b):
        assert (abs(got.cpu().double().numpy() - w) <= b).all()

    check(c.score_queries(Q)[:, ids], want, bound)
    check(c.score_queries(Q, ids), want, bound)
    for i in range(0, bq, 3):
        check(c.score_queries(Q[i])[ids], want[i], bound[i])
        check(c.score_queries(Q[i:i + 1], ids), want[i:i + 1], bound[i:i + 1])
    for j in range(0, len(pick), 4):
        check(c.score_queries(Q, ids[j:j + 1]), want[:, j:j + 1], bound[:, j:j + 1])
        check(c.score_queries(Q[-1], ids[j:j + 1]), want[-1, j:j + 1], bound[-1, j:j + 1])
