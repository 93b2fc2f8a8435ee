"""Plain restatements, in NumPy and 64 bits, of the paged 8-bit corpus operators: test infrastructure."""
from __future__ import annotations

import numpy as np

E4M3_MAX = 448.0


def tables(lengths, page_size, pages, n_tokens, doc_ids=None, src_offsets=None):
    """-> page_offsets, page_ids, page_docs, token_offsets, slots, one document and page after the other."""
    lengths = [int(x) for x in lengths]
    if doc_ids is None:
        docs = [(i, n) for i, n in enumerate(lengths)]
    else:
        docs = [(int(i), lengths[int(i)] if 0 <= int(i) < len(lengths) else 0) for i in doc_ids]
    n = len(docs)
    cap = (n_tokens + n * (page_size - 1)) // page_size
    po, to = [0], [0]
    ids, owners, slots = [], [], []
    for row, (doc, length) in enumerate(docs):
        length = max(length, 0)
        for k in range(-(-length // page_size)):
            at = len(ids) if src_offsets is None else int(src_offsets[doc]) + k
            pid = int(pages[at]) if 0 <= at < len(pages) else -1
            ids.append(pid)
            owners.append(row)
            for j in range(min(page_size, length - k * page_size)):
                slots.append(pid * page_size + j if pid >= 0 else -1)
        po.append(len(ids))
        to.append(to[-1] + length)
    pad = lambda v, m: np.array((v + [-1] * m)[:m], dtype=np.int64)  # noqa: E731
    return np.array(po), pad(ids, cap), pad(owners, cap), np.array(to), pad(slots, n_tokens)


def normalise(x, residual=None, weight=None, norm="l2", eps=None):
    """Float64 tokens of (..., d) float64 inputs."""
    h = x if residual is None else x + residual
    if norm == "l2":
        return h / np.maximum(np.sqrt((h * h).sum(-1, keepdims=True)), 1e-12 if eps is None else eps)
    if norm == "rms":
        y = h / np.sqrt((h * h).mean(-1, keepdims=True) + (1e-6 if eps is None else eps))
        return y if weight is None else y * weight
    return h


def half_step(t):
    """Half the distance of e4m3 values around |t| <= 448: steps of 2^-3 of the leading power of two, 2^-9 below 2^-6."""
    _, e = np.frexp(t)
    return np.ldexp(0.5, np.maximum(e - 1, -6) - 3)


def scores(Q, docs):
    """Q (B_q, Nq, d) and a list of (n, d) token matrices, float64 -> (B_q, n_docs); no token: -inf."""
    out = np.full((Q.shape[0], len(docs)), -np.inf)
    for i, D in enumerate(docs):
        if len(D):
            out[:, i] = np.einsum("qid,nd->qin", Q, D).max(-1).sum(-1)
    return out


def score_bound(Q, docs):
    """How far a kernel's fp32 scores may be from scores() on the same queries and stored tokens.

    A query element is held to at least 2^-10 of a unit in which its row's largest magnitude is 128
    or more: off by at most 2^-17 of that magnitude. The products are exact; d of them added in fp32
    in any order, by an adder taken at 4 ulps an addition, are off by at most d * 2^-22 of sum |q v|
    <= |q| |v|. The page scale, and the sum of Nq maxima, add a rounding each: (Nq + 2) * 2^-24 of
    sum |q| |v|."""
    d, nq = Q.shape[2], Q.shape[1]
    big, norm = np.abs(Q).max(-1), np.sqrt((Q * Q).sum(-1))
    out = np.zeros((Q.shape[0], len(docs)))
    for i, D in enumerate(docs):
        if len(D):
            v1, v2 = np.abs(D).sum(-1).max(), np.sqrt((D * D).sum(-1)).max()
            out[:, i] = (big.sum(-1) * 2.0 ** -17 * v1
                         + norm.sum(-1) * v2 * (d * 2.0 ** -22 + (nq + 2) * 2.0 ** -24) * 1.01)
    return out
