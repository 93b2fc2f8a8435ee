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
