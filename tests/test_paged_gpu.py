"""The paged 8-bit corpus operators on the GPU against their plain restatement in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.cpu().numpy()


def _same_tables(got, want):
    for name, g, w in zip(("page_offsets", "page_ids", "page_docs", "token_offsets", "slots"), got, want):
        np.testing.assert_array_equal(_np(g), w, err_msg=name)


# ------------------------------------------------------------------------------------------ tables

@pytest.mark.parametrize("lengths,page", [
    ([1], 16), ([0], 32), ([0, 0, 5, 0], 16), ([31, 32, 33, 0, 1, 64, 65], 32), ([700, 1, 128, 127, 129, 0], 128),
    ([1] * 70 + [0] * 40 + [65] * 3, 64)])
def test_tables_small(lengths, page, cuda_device):
    from tilemaxsim_b200 import page_tables
    total = sum(lengths)
    need = sum(-(-n // page) for n in lengths)
    pages = torch.randperm(need + 3, generator=_rng(need)).to(torch.int32)
    for bound in (total, total + 77):
        t = page_tables(torch.tensor(lengths).to(cuda_device), page, pages.to(cuda_device), bound)
        _same_tables(t, R.tables(lengths, page, pages.tolist(), bound))
    t = page_tables(torch.tensor(lengths, dtype=torch.int32).to(cuda_device), page, pages.to(cuda_device), total, slots=False)
    assert t.slots is None
    # a free list that runs out: the entries it has no page for are -1
    short = pages[:need // 2]
    t = page_tables(torch.tensor(lengths).to(cuda_device), page, short.to(cuda_device), total)
    _same_tables(t, R.tables(lengths, page, short.tolist(), total))


@pytest.mark.parametrize("n,page,hi", [(1023, 32, 300), (1024, 16, 40), (1025, 64, 5), (4097, 32, 70), (20011, 16, 33)])
def test_tables_many_documents(n, page, hi, cuda_device):
    from tilemaxsim_b200 import page_tables, select_page_tables
    g = _rng(n)
    lengths = torch.randint(0, hi, (n,), generator=g)
    lengths[n // 3: n // 3 + 50] = 0
    total, need = int(lengths.sum()), int(((lengths + page - 1) // page).sum())
    pages = torch.randperm(need, generator=g).to(torch.int32)
    t = page_tables(lengths.to(cuda_device), page, pages.to(cuda_device), total)
    want = R.tables(lengths, page, pages.tolist(), total)
    _same_tables(t, want)
    ids = torch.randint(-3, n + 3, (1500,), generator=g)
    bound = 1500 * hi
    s = select_page_tables(lengths.to(cuda_device), page, t.page_offsets, t.page_ids, ids.to(cuda_device), bound)
    _same_tables(s, R.tables(lengths, page, want[1].tolist(), bound, ids, want[0]))


def test_tables_nothing(cuda_device):
    from tilemaxsim_b200 import page_tables, select_page_tables
    none = torch.zeros(0, dtype=torch.int64, device=cuda_device)
    pages = torch.arange(3, dtype=torch.int32, device=cuda_device)
    t = page_tables(none, 32, pages, 5)
    _same_tables(t, R.tables([], 32, [0, 1, 2], 5))
    t = select_page_tables(none, 32, torch.zeros(1, dtype=torch.int64, device=cuda_device), pages[:0],
                           torch.tensor([0, 4], device=cuda_device), 0)
    assert _np(t.page_offsets).tolist() == [0, 0, 0]


def test_tables_one_long_document_and_negative_lengths(cuda_device):
    from tilemaxsim_b200 import page_tables
    lengths = [5, -7, 100001, 3]
    pages = list(range(4000))[::-1]
    t = page_tables(torch.tensor(lengths).to(cuda_device), 32, torch.tensor(pages, dtype=torch.int32).to(cuda_device), 100009)
    _same_tables(t, R.tables(lengths, 32, pages, 100009))


def test_tables_bound_too_small(cuda_device):
    """A bound below the token count cuts the outputs off; nothing is written past them."""
    from tilemaxsim_b200 import page_tables
    lengths = [40, 50, 60]
    t = page_tables(torch.tensor(lengths).to(cuda_device), 16, torch.arange(20, dtype=torch.int32).to(cuda_device), 30)
    want = R.tables(lengths, 16, list(range(20)), 30)
    _same_tables(t, want)


# ------------------------------------------------------------------------------------------ write and read

def _layout(lengths, page, seed, spare=2):
    from tilemaxsim_b200 import page_tables
    need = sum(-(-n // page) for n in lengths)
    pages = torch.randperm(need + spare, generator=_rng(seed)).to(torch.int32).cuda()
    return page_tables(torch.tensor(lengths).cuda(), page, pages, sum(lengths)), need + spare


def _check_written(codes, scales, tables, lengths, tokens, page):
    """tokens: float64 normalised tokens of all documents, in order."""
    c, s = codes.cpu().double().numpy(), scales.cpu().double().numpy()
    ids, po = _np(tables.page_ids), _np(tables.page_offsets)
    at = 0
    for i, n in enumerate(lengths):
        for k in range(-(-n // page)):
            rows = tokens[at + k * page: at + min(n, (k + 1) * page)]
            pid = ids[po[i] + k]
            scale = np.abs(rows).max() / R.E4M3_MAX
            # one rounding to fp32 (to nothing below half its least value)
            assert abs(s[pid] - scale) <= max(scale * 2.0 ** -24 * 1.0001, 2.0 ** -150), (i, k)
            if s[pid] == 0:
                assert not c[pid].any()
                continue
            t = np.clip(rows / s[pid], -R.E4M3_MAX, R.E4M3_MAX)
            off = np.abs(c[pid][:len(rows)] - t)
            assert (off <= R.half_step(t) * (1 + 1e-9)).all(), (i, k, off.max())
            assert (c[pid][len(rows):] == c[pid][len(rows) - 1]).all(), (i, k)
        at += n
    return c, s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,residual,weight", [("l2", False, False), ("l2", True, False), ("rms", True, True),
                                                   ("rms", False, False), ("none", False, False), ("none", True, False)])
@pytest.mark.parametrize("page,d,lengths", [
    (16, 16, [1, 15, 16, 17, 0, 40]), (32, 128, [1, 0, 31, 32, 33, 100]), (64, 96, [64, 130, 5]), (128, 256, [1, 200, 128]),
    (32, 48, [7, 33])])
def test_write(page, d, lengths, norm, residual, weight, dtype, cuda_device):
    from tilemaxsim_b200 import page_read, page_write
    g = _rng(page + d)
    x = torch.randn(sum(lengths), d, generator=g).to(dtype)
    x[0] = 0  # a row of zeros has no direction
    r = torch.randn(sum(lengths), d, generator=g).to(dtype) if residual else None
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(dtype) if weight else None
    t, n_pages = _layout(lengths, page, 5)
    codes = torch.full((n_pages, page, d), 1.5, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.full((n_pages,), 7.0, device=cuda_device)
    out = page_write(x.cuda(), t, codes, scales, residual=r.cuda() if residual else None,
                     weight=w.cuda() if weight else None, norm=norm)
    assert out[0] is codes and out[1] is scales
    f = lambda v: None if v is None else v.double().numpy()  # noqa: E731
    c, s = _check_written(codes, scales, t, lengths, R.normalise(f(x), f(r), f(w), norm), page)
    free = sorted(set(range(n_pages)) - set(_np(t.page_ids)[:_np(t.page_offsets)[-1]].tolist()))
    assert len(free) == 2 and (s[free] == 7.0).all() and (c[free] == 1.5).all()  # left as they were
    # read back: the fp32 product rounded once to each type
    slots = _np(t.slots)
    want = c.reshape(-1, d)[slots] * s[slots // page][:, None]
    for dt in DTYPES:
        got = page_read(codes, scales, t.slots, dt).cpu().double().numpy()
        step = torch.finfo(dt).eps / 2 + 2.0 ** -24
        assert (np.abs(got - want) <= np.abs(want) * step + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,residual,weight", [("l2", False, False), ("rms", True, True), ("rms", False, True), ("none", False, False)])
@pytest.mark.parametrize("page,d", [(16, 128), (64, 128), (128, 128), (16, 64), (128, 16), (16, 256), (32, 256)])
def test_write_by_the_bytes_of_a_page(page, d, norm, residual, weight, dtype, cuda_device):
    """A page's input decides how many warps take it, and whether it is staged: 512 bytes to 128 KB."""
    lengths = [page * 3 + 1, 0, 1, page, page - 1] + torch.randint(0, 3 * page, (40,), generator=_rng(d)).tolist()
    test_write(page, d, lengths, norm, residual, weight, dtype, cuda_device)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_padded_batch_and_strides(dtype, cuda_device):
    """A padded batch with garbage (NaN) behind each document, and views with other strides, write the
    same pages as the ragged tokens."""
    from tilemaxsim_b200 import page_write
    lengths, L, d, page = [9, 0, 33, 50, 1], 50, 64, 32
    g = _rng(3)
    x = torch.randn(5, L, d, generator=g).to(dtype).cuda()
    r = torch.randn(5, L, d, generator=g).to(dtype).cuda()
    keep = torch.arange(L)[None] < torch.tensor(lengths)[:, None]
    xp, rp = x.clone(), r.clone()
    xp[~keep], rp[~keep] = float("nan"), float("inf")
    t, n_pages = _layout(lengths, page, 1)

    def write(x, r):
        codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
        scales = torch.zeros(n_pages, device=cuda_device)
        page_write(x, t, codes, scales, residual=r)
        return _np(codes.view(torch.uint8)), _np(scales)

    want = write(x[keep.cuda()], r[keep.cuda()])
    big = torch.full((5, L + 3, 2 * d + 16), float("nan"), dtype=dtype, device=cuda_device)
    big[:, 1:L + 1, 16:d + 16] = xp
    odd = torch.full((5, L, d + 1), float("nan"), dtype=dtype, device=cuda_device)
    odd[:, :, 1:] = xp
    for xv, rv in ((xp, rp), (big[:, 1:L + 1, 16:d + 16], rp), (odd[:, :, 1:], rp),
                   (xp.transpose(0, 1).contiguous().transpose(0, 1), rp)):
        got = write(xv, rv)
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])


def test_write_one_row_of_any_stride(cuda_device):
    """A dimension of one element may have any stride: a column seen as a row, a broadcast document."""
    from tilemaxsim_b200 import page_write
    d, page = 32, 16
    x = torch.randn(d, generator=_rng(3)).half().cuda()
    t, n_pages = _layout([1], page, 1)

    def write(v):
        codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
        scales = torch.zeros(n_pages, device=cuda_device)
        page_write(v, t, codes, scales)
        return torch.cat([codes.float().flatten(), scales])

    want = write(x[None])
    for v in (x[:, None].t(), x[:, None].t()[None], x.as_strided((1, 1, d), (3, 5, 1)), x.as_strided((1, d), (7, 1))):
        assert v.shape[-1] == d and torch.equal(write(v), want)
    # one token for every row of a padded batch
    t, n_pages = _layout([3, 2], page, 1)
    codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(x.expand(2, 3, d), t, codes, scales)
    rows = codes[t.page_ids[:2].long()].float()
    assert rows.any() and torch.equal(rows, rows[0, 0].expand_as(rows))


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("norm", ["l2", "rms", "none"])
def test_write_non_finite_poisons_its_page_only(value, norm, cuda_device):
    from tilemaxsim_b200 import page_read, page_write, paged_maxsim
    lengths, d, page = [20, 40, 10], 32, 16
    x = torch.randn(70, d, generator=_rng(8)).half()
    x[20 + 17, 3] = value  # document 1, page 1
    t, n_pages = _layout(lengths, page, 2, spare=0)
    codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(x.cuda(), t, codes, scales, norm=norm)
    got = page_read(codes, scales, t.slots, torch.float32)
    bad = torch.zeros(70, dtype=torch.bool)
    bad[36:52] = True
    assert torch.isnan(got.cpu()).all(1).tolist() == bad.tolist()
    s = _np(paged_maxsim(torch.randn(2, 5, d, generator=_rng(9)).half().cuda(), codes, scales, t))
    assert np.isnan(s[:, 1]).all() and np.isfinite(s[:, [0, 2]]).all()


def test_write_extreme_magnitudes(cuda_device):
    """Values near the ends of fp32, and pages whose scale rounds to nothing."""
    from tilemaxsim_b200 import page_write
    d, page, lengths = 16, 16, [4, 4, 4, 4]
    x = torch.randn(16, d, generator=_rng(1))
    x[:4] *= 1e38 / x[:4].abs().max()
    x[4:8] *= 1e-30
    x[8:12] *= 1e-43 / x[8:12].abs().max()
    x[12:] = 1e-45
    t, n_pages = _layout(lengths, page, 2)
    codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(x.cuda(), t, codes, scales, norm="none")
    _check_written(codes, scales, t, lengths, x.double().numpy(), page)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("amax", [224, 7, 112, 251, 13])
def test_write_ties_go_to_even(amax, dtype, cuda_device):
    """Whole numbers as they are: many lie exactly between two codes where the scale is a power of two,
    and a rounding of the scale away from it where it is not. The codes are those of x / scale in 64 bits."""
    from tilemaxsim_b200 import page_write
    d, page, n = 128, 32, 320
    x = torch.randint(-amax, amax + 1, (n, d), generator=_rng(amax)).to(dtype)
    x[:, 0] = amax
    t, n_pages = _layout([n], page, 2)
    codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(x.cuda(), t, codes, scales, norm="none")
    scale = float(np.float32(amax / 448))
    ids = t.page_ids[:n // page].long()
    assert (scales[ids] == scale).all()
    v = x.double().numpy() / scale
    step = 2 * R.half_step(v)
    want = np.clip(np.round(v / step) * step, -448, 448)  # np.round: ties to even
    np.testing.assert_array_equal(codes[ids].cpu().double().numpy().reshape(n, d), want)


@pytest.mark.parametrize("amax", [448.0, 1.0, 0.7310585, 3.3333333e-9, 2.9e20])
def test_write_values_beside_midpoints(amax, cuda_device):
    """fp32 values at, and up to three steps beside, every midpoint between two codes, the scale's
    rounding included: one rounding of x / scale, none before it."""
    from tilemaxsim_b200 import page_write
    scale = np.float32(np.float64(np.float32(amax)) / 448)
    codes = np.arange(0x7f, dtype=np.uint8)
    values = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    middles = (values[1:] + values[:-1]) / 2
    near = (middles * np.float64(scale)).astype(np.float32)
    rows = [near]
    up, down = near, near
    for _ in range(3):
        up, down = np.nextafter(up, np.float32(np.inf)), np.nextafter(down, np.float32(0))
        rows += [up, down]
    rows = np.stack(rows + [-r for r in rows])
    x = np.zeros((16, 128), np.float32)
    x[:len(rows), :near.size] = rows
    x[:, 127] = np.float32(amax)
    t, n_pages = _layout([16], 16, 2)
    pool = torch.zeros(n_pages, 16, 128, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(torch.from_numpy(x).cuda(), t, pool, scales, norm="none")
    ids = t.page_ids[:1].long()
    assert scales[ids].item() == scale
    v = x.astype(np.float64) / np.float64(scale)  # 2^-53 off: no fp32 quotient is that near a midpoint unless on it
    step = 2 * R.half_step(v)
    want = np.clip(np.round(v / step) * step, -448, 448)
    np.testing.assert_array_equal(pool[ids].cpu().double().numpy().reshape(16, 128), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_eps_and_weights(dtype, cuda_device):
    """Rows below and above eps, no eps at all, zero and tiny weights."""
    from tilemaxsim_b200 import page_write
    d, page, lengths = 32, 16, [5, 16, 3]
    x = torch.randn(24, d, generator=_rng(1)).to(dtype)
    x[3] *= 1e-3
    t, n_pages = _layout(lengths, page, 2)
    w = torch.ones(d).to(dtype)
    w[::3] = 0
    w[1] = 1e-7
    for norm, eps, weight in (("l2", 3.0, None), ("l2", 0.0, None), ("rms", 0.0, None), ("rms", 0.5, w),
                              ("rms", 1e-6, torch.zeros(d).to(dtype)), ("rms", 1e-6, w * 1e-30 if dtype != torch.float16 else w)):
        codes = torch.zeros(n_pages, page, d, device=cuda_device).to(torch.float8_e4m3fn)
        scales = torch.zeros(n_pages, device=cuda_device)
        page_write(x.cuda(), t, codes, scales, norm=norm, eps=eps, weight=None if weight is None else weight.cuda())
        y = R.normalise(x.double().numpy(), None, None if weight is None else weight.double().numpy(), norm, eps)
        _check_written(codes, scales, t, lengths, y, page)
    # a zero row has no direction without an eps: its page is not a number
    x[7] = 0
    for norm in ("l2", "rms"):
        page_write(x.cuda(), t, codes, scales, norm=norm, eps=0.0)
        assert torch.isnan(scales[t.page_ids[:3].long()]).tolist() == [False, True, False]  # one page a document


def test_write_malformed_tables_stay_inside(cuda_device):
    """Entries that name no page of the pool, no document, or rows that x does not have."""
    from tilemaxsim_b200 import PageTables, page_write
    d, page = 32, 16
    i64 = lambda *v: torch.tensor(v, dtype=torch.int64, device=cuda_device)  # noqa: E731
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)  # noqa: E731
    codes = torch.ones(4, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.ones(4, device=cuda_device)
    x = torch.randn(20, d, generator=_rng(4)).half().cuda()
    t = PageTables(i64(0, 2, 4, 6), i32(-1, 9, 1, 2, 3, 2147483647), i32(0, 0, 7, -1, 2, 2), i64(0, 20, 60, 90), None)
    page_write(x, t, codes, scales)  # entry 4: document 2 starts at row 60 of 20
    t = t._replace(token_offsets=i64(-5, 10, 1 << 40, -(1 << 50)))
    page_write(x, t, codes, scales)
    t = t._replace(page_offsets=i64(-(1 << 60), 1 << 60, 3, 6), page_docs=i32(0, 0, 1, 1, 2, 2))
    page_write(x, t, codes, scales)
    assert (scales[:3] == 1).all()


def test_read_slots_outside_the_pool(cuda_device):
    from tilemaxsim_b200 import page_read
    codes = torch.randn(3, 16, 48, generator=_rng(1)).cuda().to(torch.float8_e4m3fn)
    scales = torch.tensor([1.0, 2.0, 0.5], device=cuda_device)
    slots = torch.tensor([0, -1, 47, 48, 1 << 40, -(1 << 50), 16], device=cuda_device)
    got = page_read(codes, scales, slots, torch.float32).cpu()
    flat = codes.float().cpu().view(48, 48) * scales.cpu().repeat_interleave(16)[:, None]
    want = torch.zeros(7, 48)
    want[0], want[2], want[6] = flat[0], flat[47], flat[16]
    assert torch.equal(got, want)
    assert page_read(codes, scales, slots[:0]).shape == (0, 48)


# ------------------------------------------------------------------------------------------ scores

def _corpus(lengths, page, d, seed, dtype=torch.bfloat16):
    """A written pool and each document's stored tokens in float64."""
    from tilemaxsim_b200 import page_write
    x = torch.randn(sum(lengths), d, generator=_rng(seed)).to(dtype).cuda()
    t, n_pages = _layout(lengths, page, seed)
    codes = torch.full((n_pages, page, d), float("nan"), device="cuda").to(torch.float8_e4m3fn)
    scales = torch.full((n_pages,), float("nan"), device="cuda")
    page_write(x, t, codes, scales)
    slots = t.slots.cpu()
    flat = codes.float().cpu().view(-1, d)[slots].double() * scales.cpu().double()[slots // page][:, None]
    return t, codes, scales, [v.numpy() for v in flat.split(lengths)]


def _queries(bq, nq, d, seed, dtype):
    return torch.nn.functional.normalize(torch.randn(bq, nq, d, generator=_rng(seed)), dim=-1).to(dtype).cuda()


def _check_scores(got, Q, docs):
    q = Q.cpu().double().numpy()
    want, bound = R.scores(q, docs), R.score_bound(q, docs)
    got = _np(got).astype(np.float64)
    empty = np.isinf(want)
    np.testing.assert_array_equal(got[empty], want[empty])
    off = np.abs(np.where(empty, 0, got) - np.where(empty, 0, want))
    assert (off <= bound).all(), (off - bound).max()


RAGGED = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 0, 0, 127, 128, 129, 300, 2, 1, 1, 0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("bq,nq,d", [(1, 1, 128), (1, 32, 128), (2, 32, 64), (3, 20, 96), (1, 33, 128), (5, 32, 16),
                                      (1, 128, 128), (2, 77, 256), (17, 32, 128)])
def test_scores(bq, nq, d, page, dtype, cuda_device):
    from tilemaxsim_b200 import paged_maxsim
    t, codes, scales, docs = _corpus(RAGGED, page, d, bq * 100 + d)
    Q = _queries(bq, nq, d, 7, dtype)
    got = paged_maxsim(Q, codes, scales, t)
    assert got.shape == (bq, len(RAGGED)) and got.dtype == torch.float32
    _check_scores(got, Q, docs)
    assert torch.equal(got, paged_maxsim(Q, codes, scales, t))
    if bq == 1:
        assert torch.equal(got[0], paged_maxsim(Q[0], codes, scales, t))


@pytest.mark.parametrize("bq,nq,d,page,n,hi,dtype", [
    (1, 32, 128, 32, 3001, 300, torch.bfloat16), (1, 32, 128, 16, 2003, 40, torch.float16),
    (2, 32, 128, 32, 1501, 300, torch.float16), (4, 32, 64, 64, 1500, 200, torch.bfloat16),
    (64, 32, 128, 32, 700, 200, torch.bfloat16), (33, 40, 128, 16, 400, 100, torch.float16),
    (20, 8, 256, 128, 300, 300, torch.float16), (1, 32, 128, 32, 9000, 2, torch.bfloat16)])
def test_scores_larger(bq, nq, d, page, n, hi, dtype, cuda_device):
    from tilemaxsim_b200 import paged_maxsim
    lengths = torch.randint(0, hi + 1, (n,), generator=_rng(n)).tolist()
    t, codes, scales, docs = _corpus(lengths, page, d, n)
    Q = _queries(bq, nq, d, 3, dtype)
    _check_scores(paged_maxsim(Q, codes, scales, t), Q, docs)


def test_scores_long_documents(cuda_device):
    from tilemaxsim_b200 import paged_maxsim
    lengths = [20000, 1, 7001, 0, 30000]
    t, codes, scales, docs = _corpus(lengths, 32, 128, 1)
    Q = _queries(3, 32, 128, 3, torch.bfloat16)
    _check_scores(paged_maxsim(Q, codes, scales, t), Q, docs)


@pytest.mark.parametrize("lengths", [[5000], [100000], [1500, 1], [3000, 2000, 0, 9000, 1], list(range(1000, 3000, 37)),
                                     [4000] * 3 + [0] * 5 + [17] * 2])
@pytest.mark.parametrize("bq,nq,d,page,dtype", [(1, 32, 128, 32, torch.bfloat16), (2, 20, 64, 16, torch.float16),
                                                 (1, 70, 128, 128, torch.float16), (9, 32, 256, 64, torch.bfloat16),
                                                 (21, 32, 128, 32, torch.bfloat16)])
def test_scores_documents_over_several_ranges(bq, nq, d, page, dtype, lengths, cuda_device):
    """Few long documents are cut over the whole GPU and joined again."""
    from tilemaxsim_b200 import paged_maxsim
    if d * sum(lengths) > 13_000_000:
        lengths = [n // 2 for n in lengths]
    t, codes, scales, docs = _corpus(lengths, page, d, 1)
    Q = _queries(bq, nq, d, 3, dtype)
    got = paged_maxsim(Q, codes, scales, t)
    _check_scores(got, Q, docs)
    assert torch.equal(got, paged_maxsim(Q, codes, scales, t))


@pytest.mark.parametrize("d", [16, 32, 48, 80, 112, 144, 176, 240])
@pytest.mark.parametrize("bq,page,dtype", [(1, 16, torch.float16), (2, 32, torch.bfloat16), (3, 16, torch.bfloat16),
                                            (19, 32, torch.float16), (40, 16, torch.bfloat16)])
def test_scores_token_widths(bq, page, dtype, d, cuda_device):
    """Every kind of width, through enough documents that every stage is used several times."""
    from tilemaxsim_b200 import paged_maxsim
    lengths = torch.randint(0, 150, (1200,), generator=_rng(d)).tolist()
    t, codes, scales, docs = _corpus(lengths, page, d, 1)
    Q = _queries(bq, 32, d, 3, dtype)
    got = paged_maxsim(Q, codes, scales, t)
    pick = torch.randperm(1200, generator=_rng(2))[:200].tolist()
    _check_scores(got[:, pick], Q, [docs[i] for i in pick])
    for i in range(0, bq, 7):  # alone or in a batch: within the bound of the kernel's own arithmetic
        _check_scores(paged_maxsim(Q[i:i + 1], codes, scales, t)[:, pick], Q[i:i + 1], [docs[j] for j in pick])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bq,nq", [(1, 32), (1, 5), (2, 32), (1, 64), (3, 32)])
@pytest.mark.parametrize("page,n,hi", [(16, 700, 90), (32, 700, 90), (64, 300, 400), (128, 300, 400), (16, 5, 3000), (32, 5, 3000)])
def test_scores_two_tokens_a_row(page, n, hi, bq, nq, dtype, cuda_device):
    """d = 64: two tokens share 128 bytes. Streams of many tiles, documents cut by streams and ranges."""
    from tilemaxsim_b200 import paged_maxsim
    lengths = torch.randint(0, hi, (n,), generator=_rng(page + n)).tolist()
    t, codes, scales, docs = _corpus(lengths, page, 64, bq + nq)
    Q = _queries(bq, nq, 64, 7, dtype)
    got = paged_maxsim(Q, codes, scales, t)
    _check_scores(got, Q, docs)
    assert torch.equal(got, paged_maxsim(Q, codes, scales, t))


@pytest.mark.parametrize("bq", [1, 2])
def test_scores_two_tokens_a_row_which_is_which(bq, cuda_device):
    """Every token of a document in its turn the only one that a query finds, a NaN page beside it."""
    from tilemaxsim_b200 import page_write, paged_maxsim
    page, n = 16, 64
    t, n_pages = _layout([n, 16, n], page, 3)
    x = torch.zeros(n + 16 + n, 64)
    x[:n] = torch.eye(64)
    x[n:n + 16] = float("nan")
    x[n + 16:] = torch.eye(64).flip(0) * 0.5
    codes = torch.zeros(n_pages, page, 64, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    page_write(x.half().cuda(), t, codes, scales, norm="none")
    Q = torch.eye(64).view(64 // (32 * bq), bq, 32, 64).half().cuda()
    for q in Q:
        got = paged_maxsim(q, codes, scales, t).cpu()
        assert torch.equal(got[:, 0], torch.full((bq,), 32.0)) and got[:, 1].isnan().all()
        assert torch.equal(got[:, 2], torch.full((bq,), 16.0))


@pytest.mark.parametrize("bq,page", [(1, 32), (2, 16), (4, 64), (20, 32)])
def test_scores_long_streams(bq, page, cuda_device):
    """Enough documents that every part of the corpus takes many steps, and parts end at different ones:
    a query of a batch, and a document of a corpus, score what they score alone."""
    from tilemaxsim_b200 import paged_maxsim
    lengths = torch.randint(0, 201, (20000,), generator=_rng(1)).tolist()
    t, codes, scales, docs = _corpus(lengths, page, 128, 3)
    Q = _queries(bq, 32, 128, 3, torch.bfloat16)
    got = paged_maxsim(Q, codes, scales, t)
    pick = torch.randperm(20000, generator=_rng(2))[:400].tolist()
    _check_scores(got[:, pick], Q, [docs[i] for i in pick])
    best = torch.full((20000, bq * 32), float("-inf"), device=cuda_device)
    used = t.page_ids >= 0
    ids = t.page_ids[used].long()
    for a in range(0, ids.numel(), 20000):  # float32 over the whole corpus: every document, coarsely
        i = ids[a:a + 20000]
        tok = codes.view(torch.uint8)[i].view(torch.float8_e4m3fn).float() * scales[i][:, None, None]
        s = (tok.view(-1, 128) @ Q.float().view(-1, 128).T).view(i.numel(), page, -1).amax(1)
        best.scatter_reduce_(0, t.page_docs[used][a:a + 20000].long()[:, None].expand_as(s), s, "amax")
    torch.testing.assert_close(got, best.view(20000, bq, 32).sum(-1).T, rtol=1e-5, atol=1e-4)


@pytest.mark.parametrize("lengths", [[0], [0, 0, 0], [1], [3]])
def test_scores_hardly_anything(lengths, cuda_device):
    from tilemaxsim_b200 import paged_maxsim
    t, codes, scales, docs = _corpus(lengths, 32, 128, 1)
    Q = _queries(2, 40, 128, 3, torch.float16)
    _check_scores(paged_maxsim(Q, codes, scales, t), Q, docs)
    assert paged_maxsim(Q[:0], codes, scales, t).shape == (0, len(lengths))


def test_scores_query_values(cuda_device):
    """Zero rows, rows far apart in magnitude, outliers and subnormal values in one query; fp32 queries
    are rounded to fp16."""
    from tilemaxsim_b200 import paged_maxsim
    t, codes, scales, docs = _corpus(RAGGED, 32, 128, 4)
    for dtype, tiny, big in ((torch.float16, 6e-8, 6e4), (torch.bfloat16, 1e-38, 1e30)):
        Q = _queries(1, 40, 128, 5, torch.float32)
        Q[0, 1] = 0
        Q[0, 2] *= big / 2
        Q[0, 3] *= tiny * 20
        Q[0, 4, 7] = 100.0
        Q[0, 5] = 0
        Q[0, 5, 9] = 1.0
        Q = Q.to(dtype)
        for i in range(40):  # one row at a time: the bound is each row's own
            _check_scores(paged_maxsim(Q[:, i:i + 1], codes, scales, t), Q[:, i:i + 1], docs)
        _check_scores(paged_maxsim(Q, codes, scales, t), Q, docs)
    Q = _queries(2, 32, 128, 5, torch.float32)
    assert torch.equal(paged_maxsim(Q, codes, scales, t), paged_maxsim(Q.half(), codes, scales, t))


def test_scores_skip_entries_outside_the_pool(cuda_device):
    """A page id outside the pool is left out; a document all of whose pages are is empty."""
    from tilemaxsim_b200 import paged_maxsim
    t, codes, scales, docs = _corpus([40, 20, 33, 64], 32, 64, 4)
    ids = t.page_ids.clone()
    ids[1], ids[2], ids[3] = -1, 1 << 30, codes.shape[0]  # document 0's second page, 1's only one, 2's first
    Q = _queries(3, 32, 64, 5, torch.bfloat16)
    got = paged_maxsim(Q, codes, scales, t._replace(page_ids=ids))
    _check_scores(got, Q, [docs[0][:32], docs[1][:0], docs[2][32:], docs[3]])


def test_scores_malformed_offsets_stay_inside(cuda_device):
    from tilemaxsim_b200 import paged_maxsim
    t, codes, scales, _ = _corpus([40, 20, 33, 64], 32, 64, 4)
    Q = _queries(3, 32, 64, 5, torch.bfloat16)
    good = paged_maxsim(Q, codes, scales, t)
    for off in ([-5, 9, 2, 1 << 40, 3], [7, 7, 7, 7, 7], [1 << 62] * 5, [0, 0, 0, 0, -1], [6, 5, 4, 3, 2]):
        bad = t._replace(page_offsets=torch.tensor(off, dtype=torch.int64, device=cuda_device))
        assert paged_maxsim(Q, codes, scales, bad).shape == (3, 4)
    docs = t.page_docs.clone()
    docs[:] = torch.tensor([5, -1, 1 << 30, 0, 3, 2, 1, 0][:docs.numel()], dtype=torch.int32)
    assert paged_maxsim(Q, codes, scales, t._replace(page_docs=docs)).shape == (3, 4)
    assert torch.equal(paged_maxsim(Q, codes, scales, t), good)


def test_scores_other_stream_and_graph(cuda_device):
    from tilemaxsim_b200 import GraphedStep, paged_maxsim
    t, codes, scales, docs = _corpus(RAGGED, 32, 128, 4)
    Q = _queries(2, 40, 128, 5, torch.bfloat16)
    want = paged_maxsim(Q, codes, scales, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_maxsim(Q, codes, scales, t)
    side.synchronize()
    assert torch.equal(got, want)
    a = GraphedStep(lambda q: paged_maxsim(q, codes, scales, t), Q)
    b = GraphedStep(lambda q: paged_maxsim(q, codes, scales, t), Q)
    Q2 = _queries(2, 40, 128, 6, torch.bfloat16)
    assert torch.equal(a(Q), want.cpu())
    assert torch.equal(b(Q2), paged_maxsim(Q2, codes, scales, t).cpu())
    assert torch.equal(a(Q), want.cpu())


@pytest.mark.parametrize("n_docs", [30, 2500])
def test_chain_captured_and_replayed(n_docs, cuda_device):
    """Tables, writes, scores and reads in one graph: replays follow the lengths and tokens they find."""
    from tilemaxsim_b200 import GraphedStep, page_read, page_tables, page_write, paged_maxsim
    d, page, rows = 64, 16, 6
    bound = n_docs * rows
    pages = torch.randperm(n_docs, generator=_rng(3)).to(torch.int32).to(cuda_device)
    codes = torch.zeros(n_docs, page, d, device=cuda_device).to(torch.float8_e4m3fn)
    scales = torch.zeros(n_docs, device=cuda_device)
    Q = _queries(3, 32, d, 4, torch.float16)

    def chain(lengths, x):
        t = page_tables(lengths, page, pages, bound)
        page_write(x, t, codes, scales)
        return paged_maxsim(Q, codes, scales, t), page_read(codes, scales, t.slots, torch.float32)

    def example(seed):
        lengths = torch.randint(0, rows + 1, (n_docs,), generator=_rng(seed))
        return lengths, torch.randn(n_docs, rows, d, generator=_rng(seed + 1)).half()

    step = GraphedStep(chain, *(v.to(cuda_device) for v in example(1)))
    for seed in (10, 20, 1):
        lengths, x = (v.to(cuda_device) for v in example(seed))
        scores, tokens = step(lengths, x)
        want_scores, want_tokens = chain(lengths, x)
        assert torch.equal(scores, want_scores.cpu()) and torch.equal(tokens, want_tokens.cpu())
        docs = [v.double().numpy() for v in tokens[:int(lengths.sum())].split(lengths.tolist())]
        _check_scores(want_scores, Q, docs)
        assert not tokens[int(lengths.sum()):].any()


def test_two_streams_at_once(cuda_device):
    """Calls that overlap on the device share nothing: each kind on one stream against another on the other."""
    from tilemaxsim_b200 import page_read, paged_maxsim, select_page_tables
    lengths = torch.randint(0, 300, (400,), generator=_rng(8)).tolist()
    t, codes, scales, _ = _corpus(lengths, 32, 128, 4)
    dev_lengths = torch.tensor(lengths, device=cuda_device)
    pick = torch.randint(0, 400, (300,), generator=_rng(9)).to(cuda_device)

    def rerank(Q):
        sel = select_page_tables(dev_lengths, 32, t.page_offsets, t.page_ids, pick, 300 * 300)
        return paged_maxsim(Q, codes, scales, sel), page_read(codes, scales, sel.slots)

    Qs = [_queries(1, 32, 128, 5, torch.bfloat16), _queries(20, 40, 128, 6, torch.float16)]
    want = [rerank(Q) for Q in Qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in Qs]
    got = [[], []]
    for _ in range(20):
        for s, Q, out in zip(streams, Qs, got):
            with torch.cuda.stream(s):
                out.append(rerank(Q))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, w))


@pytest.mark.parametrize("page,d", [(128, 256), (16, 128)])
def test_pool_of_more_than_4_gib(page, d, cuda_device):
    """Pages whose bytes lie beyond 32-bit offsets, and those that 32 bits would take them for."""
    from tilemaxsim_b200 import page_read, page_tables, page_write, paged_maxsim
    wrap = 2 ** 32 // (page * d)
    n_pages = wrap + 100
    codes = torch.zeros(n_pages, page, d, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
    scales = torch.zeros(n_pages, device=cuda_device)
    lengths = [200, 1, 130, 64]
    need = sum(-(-n // page) for n in lengths)
    high = wrap + torch.randperm(100, generator=_rng(1))[:need]
    x = torch.randn(sum(lengths), d, generator=_rng(2)).half().to(cuda_device)
    t = page_tables(torch.tensor(lengths).to(cuda_device), page, high.to(torch.int32).to(cuda_device), sum(lengths))
    page_write(x, t, codes, scales)
    assert not codes[:100].view(torch.uint8).any() and not scales[:100].any()
    tokens = page_read(codes, scales, t.slots, torch.float32).cpu().double()
    y = torch.nn.functional.normalize(x.double().cpu(), dim=-1)
    most = y.abs().amax()
    assert ((tokens - y).abs() <= y.abs() * 2.0 ** -4 * 1.001 + most * 2.0 ** -10 / 448 * 1.001).all()
    Q = _queries(2, 32, d, 3, torch.float16)
    _check_scores(paged_maxsim(Q, codes, scales, t), Q, [v.numpy() for v in tokens.split(lengths)])


@pytest.mark.parametrize("bq", [1, 2, 9])
def test_scores_bounded_wait_reports_timeout(bq, cuda_device):
    """The loads stay out: every wait runs out after the (short) limit, the kernel returns, the host
    reads the status, and the next call is right."""
    from tilemaxsim_b200 import _lib, paged_maxsim
    lib = _lib.load()
    t, codes, scales, docs = _corpus(RAGGED, 32, 128, 4)
    Q = _queries(bq, 32, 128, 5, torch.bfloat16)
    paged_maxsim(Q, codes, scales, t)
    assert _lib.last_device_error(cuda_device)[0] == _lib.TMS_OK
    lib.tms_set_debug(50_000_000, 1)
    try:
        paged_maxsim(Q, codes, scales, t)
        rc, word = _lib.last_device_error(cuda_device)
    finally:
        lib.tms_set_debug(2_000_000_000, 0)
    assert rc == _lib.TMS_ERR_TIMEOUT and word & 0x80000000
    _check_scores(paged_maxsim(Q, codes, scales, t), Q, docs)
    assert _lib.last_device_error(cuda_device)[0] == _lib.TMS_OK


# ------------------------------------------------------------------------------------------ the corpus

def test_corpus_life(cuda_device):
    """Documents are added (ragged, padded), scored, selected, read, removed and added again."""
    from tilemaxsim_b200 import PagedCorpus, maxsim_batched
    d, page = 64, 16
    c = PagedCorpus(d, n_pages=60, max_docs=40, page_size=page)
    kept: dict[int, torch.Tensor] = {}

    def add(lengths, padded, seed):
        n = len(lengths)
        x = torch.randn(n, max(max(lengths), 1), d, generator=_rng(seed)).half().cuda()
        rows = [x[i, :m] for i, m in enumerate(lengths)]
        ids = c.add(x if padded else torch.cat(rows), torch.tensor(lengths) if padded else lengths)
        for i, r in zip(ids.tolist(), rows):
            kept[i] = torch.nn.functional.normalize(r.float(), dim=-1).cpu()
        return ids.tolist()

    Q = _queries(3, 32, d, 5, torch.float16)

    def check():
        n = c.n_docs
        tok, off = c.tokens(list(range(n)), torch.float32)
        tok, off = tok.cpu(), off.tolist()
        docs = [tok[off[i]:off[i + 1]] for i in range(n)]
        for i in range(n):
            assert docs[i].shape == kept[i].shape
            if len(docs[i]):  # e4m3 with a scale of the page's largest value: half a step of 2^-3, or of 2^-9 / 448 of it
                most = kept[i].abs().max()
                assert ((docs[i] - kept[i]).abs() <= kept[i].abs() * 2.0 ** -4 * 1.001 + most * 2.0 ** -10 / 448 * 1.001).all()
        _check_scores(c.score_queries(Q), Q, [v.double().numpy() for v in docs])
        pick = torch.tensor([n - 1, 0, n // 2, 0, n + 5, -1])
        sel = c.score_queries(Q, pick.cuda())
        assert torch.equal(sel[:, :4], c.score_queries(Q)[:, pick[:4].cuda()]) and torch.isinf(sel[:, 4:]).all()
        v, i = c.search(Q, 5)
        vs, is_ = c.search(Q, 3, pick[:3].cuda())
        assert torch.equal(v[:, 0], c.score_queries(Q).amax(1)) and set(is_.flatten().tolist()) <= set(pick[:3].tolist())
        # the same tokens through the dense kernel: fp16 rounding of the tokens, its 1e-3 tolerance
        t16, o16 = c.tokens(list(range(n)))
        dense = maxsim_batched(Q, t16, o16)
        fin = torch.isfinite(dense)
        assert torch.equal(torch.isfinite(c.score_queries(Q)), fin)
        torch.testing.assert_close(c.score_queries(Q)[fin], dense[fin], rtol=1e-3, atol=1e-3)

    assert add([5, 16, 17, 0, 40], False, 1) == [0, 1, 2, 3, 4]
    check()
    add([33, 1, 100], True, 2)
    check()
    free = c.n_free
    c.remove(torch.tensor([2, 7, 2, 3]))
    c.remove([2])
    for i in (2, 7):
        kept[i] = kept[i][:0]
    assert c.n_free == free + 2 + 7
    check()
    assert add([100, 90, 17], False, 3) == [8, 9, 10]
    check()
    before = [t.clone() for t in c.tables[:4]]
    with pytest.raises(ValueError, match="pages are needed"):
        c.add(torch.zeros(1000, d).half().cuda(), [1000])
    with pytest.raises(ValueError, match="no room"):
        c.add(torch.zeros(0, d).half().cuda(), [0] * 30)
    with pytest.raises(ValueError, match="sum"):
        c.add(torch.zeros(5, d).half().cuda(), [4])
    with pytest.raises(ValueError, match="fit"):
        c.add(torch.zeros(1, 5, d).half().cuda(), [6])
    with pytest.raises(ValueError, match="negative"):
        c.add(torch.zeros(5, d).half().cuda(), [6, -1])
    with pytest.raises(TypeError):
        c.add(torch.zeros(5, d).double().cuda(), [5])
    with pytest.raises(IndexError):
        c.remove([11])
    with pytest.raises(ValueError, match="integers"):
        c.remove([1.0])
    with pytest.raises(ValueError, match="integers"):
        c.add(torch.zeros(5, d).half().cuda(), [5.0])
    with pytest.raises(ValueError, match="weight"):
        c.add(torch.zeros(5, d).half().cuda(), [5], norm="rms", weight=torch.ones(d).cuda())
    c.remove([])
    assert c.n_docs == 11 and all(torch.equal(a, b) for a, b in zip(before, c.tables[:4]))
    c.remove(list(range(11)))
    assert c.n_free == 60 and sorted(c._free.tolist()) == list(range(60))
    assert torch.isinf(c.score_queries(Q)).all()
    for i in list(kept):
        kept[i] = kept[i][:0]
    add([60 * 16], False, 9)
    assert c.n_free == 0
    check()


def test_corpus_selection_of_many_short_documents_and_a_long_one(cuda_device):
    """The longest document's length for each candidate would be far more than the corpus holds."""
    from tilemaxsim_b200 import PagedCorpus
    c = PagedCorpus(16, n_pages=3000, max_docs=2100, page_size=16)
    lengths = [1] * 1000 + [20000] + [3] * 700
    x = torch.randn(sum(lengths), 16, generator=_rng(1)).half().cuda()
    c.add(x, torch.tensor(lengths).cuda())
    ids = torch.randint(-5, 1710, (5000,), generator=_rng(2))
    ids[ids == 1000] = 7  # the long one is no candidate
    t = c.select(ids.cuda(), slots=True)
    assert t.slots.numel() == sum(lengths[i] if 0 <= i < 1701 else 0 for i in ids.tolist())
    Q = _queries(2, 4, 16, 5, torch.float16)
    full, got = c.score_queries(Q), c.score_queries(Q, ids.cuda())
    real = (ids >= 0) & (ids < 1701)
    assert torch.equal(got[:, real.cuda()], full[:, ids[real].cuda()]) and torch.isinf(got[:, ~real.cuda()]).all()


def test_corpus_captured_search_sees_removals(cuda_device):
    from tilemaxsim_b200 import GraphedStep, PagedCorpus
    c = PagedCorpus(128, n_pages=100, max_docs=50)
    g = _rng(2)
    c.add(torch.randn(600, 128, generator=g).half().cuda(), [100, 200, 50, 250])
    Q = _queries(2, 32, 128, 5, torch.float16)
    step = GraphedStep(lambda q: c.search(q, 2), Q)
    v, i = step(Q)
    want_v, want_i = c.search(Q, 2)
    assert torch.equal(v, want_v.cpu()) and torch.equal(i, want_i.cpu())
    c.remove([int(want_i[0, 0])])
    c.add(torch.randn(64, 128, generator=g).half().cuda(), [64])
    v, i = step(Q)
    want = c.score_queries(Q)[:, :4].topk(2)
    assert torch.equal(v, want.values.cpu()) and torch.equal(i, want.indices.cpu())


def test_ivf_candidates_reranked_in_place(cuda_device):
    """IVFIndex takes a PagedCorpus as the tokens it reranks: the scores are the corpus's own."""
    from tilemaxsim_b200 import IVFIndex, PagedCorpus
    g = _rng(6)
    lengths = torch.randint(1, 60, (200,), generator=g)
    off = torch.zeros(201, dtype=torch.int64)
    off[1:] = torch.cumsum(lengths, 0)
    x = torch.nn.functional.normalize(torch.randn(int(off[-1]), 64, generator=g), dim=-1).half().cuda()
    cent = torch.nn.functional.normalize(torch.randn(50, 64, generator=g), dim=-1).half().cuda()
    index = IVFIndex(cent, (x @ cent.T).argmax(1), off.cuda())
    corpus = PagedCorpus(64, n_pages=700, max_docs=200, page_size=16)
    corpus.add(x, lengths)
    Q = _queries(4, 32, 64, 5, torch.float16)
    vals, ids = index.search(Q, corpus, 7, nprobe=2)
    bitmaps, cand = index.candidates(Q, 2)
    full = corpus.score_queries(Q)
    for q in range(4):
        mine = [d for d in cand.tolist() if int(bitmaps[q, d >> 5]) >> (d & 31) & 1]
        best = sorted(mine, key=lambda d: (-float(full[q, d]), d))[:7]
        assert ids[q, :len(best)].tolist() == best
        assert torch.equal(vals[q, :len(best)], full[q, best])
    gone = [int(ids[0, 0]), int(ids[1, 0])]
    corpus.remove(gone)
    vals2, ids2 = index.search(Q, corpus, 7, nprobe=2)
    assert not set(gone) & set(ids2.flatten().tolist()) and torch.equal(vals2[0, :6], vals[0, 1:])
    assert PagedCorpus(64, 4, 4).n_docs == 0
    with pytest.raises(ValueError, match="documents"):
        index.search(Q, PagedCorpus(64, 4, 4), 7, nprobe=2)
