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


def _four_squares(n):
    """Four whole numbers whose squares sum to n."""
    for a in range(int(n ** 0.5), -1, -1):
        for b in range(int(max(n - a * a, 0) ** 0.5), -1, -1):
            rest = n - a * a - b * b
            for c in range(int(rest ** 0.5), int((rest / 2) ** 0.5) - 1, -1):
                d = round((rest - c * c) ** 0.5)
                if c * c + d * d == rest:
                    return [a, b, c, d]
    raise AssertionError(n)


def _row_of_ties(d, rng, norm):
    """Whole numbers whose squares sum to norm^2 = (3 * 2^k)^2, the largest 7 norm / 16, and sixteen of those
    that lie exactly between two codes once divided by the norm and by the scale that the largest gives (2^-10)."""
    top = 7 * norm // 16
    ties = [3 * m * norm // 768 for m in list(range(17, 32, 2)) + list(range(34, 64, 4)) + list(range(68, 84, 8))]
    row = [top] + rng.choice(ties, 16).tolist()
    while (rest := norm * norm - sum(v * v for v in row)) > 4 * top * top:
        row.append(top)
    if rest < 0 or len(row) > d - 4:
        return None
    row += _four_squares(rest)
    row += [0] * (d - len(row))
    return None if max(row) > top else [v * s for v, s in zip(row, rng.choice([-1, 1], d))]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("norm,residual,weight", [("l2", False, None), ("l2", True, None), ("rms", False, None), ("rms", True, 3.0),
                                                   ("rms", False, 0.5)])
@pytest.mark.parametrize("page,d", [(16, 64), (32, 128), (128, 64), (64, 256)])
def test_write_exact_ties_of_normalised_values(page, d, norm, residual, weight, dtype, cuda_device):
    """Norms and scales that are exact: what lies between two codes goes to the even one, decided by the
    norm's quotient itself, not by a factor that comes near it."""
    from tilemaxsim_b200 import page_tables, page_write
    rng = np.random.default_rng(page + d)
    rows = []
    while len(rows) < page:
        r = _row_of_ties(d, rng, 768)
        rows += [r] if r else []
    h = np.array(rows, dtype=np.float64)
    assert ((h * h).sum(1) == 768.0 ** 2).all()
    res = rng.integers(-64, 65, h.shape) if residual else None
    x = torch.from_numpy(h if res is None else h - res).to(dtype)
    assert (x.double().numpy() + (0 if res is None else res) == h).all()
    w = None if weight is None else torch.full((d,), weight).to(dtype)
    codes, scales = _pool(1, page, d)
    t = page_tables(torch.tensor([page], device=cuda_device), page, torch.zeros(1, dtype=torch.int32, device=cuda_device), page)
    page_write(x.cuda(), t, codes, scales, residual=None if res is None else torch.from_numpy(res).to(dtype).cuda(),
               weight=None if w is None else w.cuda(), norm=norm, eps=0.0)
    n = 768.0 if norm == "l2" else np.sqrt(768.0 ** 2 / d)
    y = h / n * (weight or 1.0)
    scale = float(np.float32(np.abs(y).max() / 448))
    assert scales.item() == scale
    v = h * (weight or 1.0) / (n * scale)
    if scale == np.abs(y).max() / 448:  # where the scale is not rounded there are ties
        step = 2 * R.half_step(v)
        assert (np.abs(v / step % 1 - 0.5) == 0).mean() >= 16 / d
    step = 2 * R.half_step(v)
    want = np.clip(np.round(v / step) * step, -448, 448)  # np.round: ties to even
    np.testing.assert_array_equal(codes[0].cpu().double().numpy(), want)


@pytest.mark.parametrize("small,weight,eps", [(1e-26, 1e-24, e) for e in (0.0, 1e-38, 1e-30, 1e-20, 1e-7)]
                         + [(1e-24, 1e-22, e) for e in (1e-42, 1e-40, 1e-38, 1e-37, 1e-30)])
@pytest.mark.parametrize("d,page", [(16, 16), (128, 32)])
def test_write_products_with_weights_below_fp32(d, page, small, weight, eps, cuda_device):
    """h * weight and h^2 vanish in fp32 where their quotient by the root does not: fp64 decides. Beside
    them rows of zeros, in a page of their own and in one with others."""
    from tilemaxsim_b200 import page_tables, page_write
    g = _rng(d)
    x = torch.randn(2 * page + 3, d, generator=g) * small
    x[1] = 0
    x[page:2 * page] = 0
    w = (1 + 0.1 * torch.randn(d, generator=g)) * weight
    lengths = [page, page, 3]
    t = page_tables(torch.tensor(lengths, device=cuda_device), page, torch.arange(3, dtype=torch.int32, device=cuda_device), len(x))
    codes, scales = _pool(3, page, d)
    page_write(x.cuda(), t, codes, scales, norm="rms", weight=w.cuda(), eps=eps)
    # without an eps a row of zeros is not a number
    with np.errstate(invalid="ignore"):
        y = R.normalise(x.double().numpy(), None, w.double().numpy(), "rms", float(np.float32(eps)))
    for i, rows in enumerate(np.split(y, [page, 2 * page])):
        s = scales[i].item()
        if np.isnan(rows).any():
            assert np.isnan(s)
            continue
        want = np.abs(rows).max() / 448
        assert abs(s - want) <= max(want * 2.0 ** -24 * 1.0001, 2.0 ** -150)
        if s > 0:
            v = rows / s
            assert (np.abs(codes[i, :len(rows)].cpu().double().numpy() - np.clip(v, -448, 448)) <= R.half_step(np.clip(v, -448, 448)) * (1 + 1e-9)).all()


def _wide_rows(n, d, seed):
    """Rows whose elements lie far apart: one outlier beside a normal distribution, magnitudes over many powers of
    two, one element alone, and ordinary ones."""
    g = _rng(seed)
    q = torch.randn(n, d, generator=g)
    q[0::4, d // 3] = 64.0
    wide = torch.exp2(-20 * torch.rand(n, d, generator=g)) * q.sign()
    q[1::4] = wide[1::4]
    q[2::4] *= 0.01
    q[2::4, d - 1] = -3.0
    return q


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bq,nq", [(1, 1), (1, 32), (2, 5), (1, 64), (3, 20), (20, 32), (5, 1)])
@pytest.mark.parametrize("page,d", [(16, 64), (32, 64), (32, 128), (16, 128), (32, 96), (64, 256), (16, 144)])
def test_scores_find_every_element_of_a_query(page, d, bq, nq, dtype, cuda_device):
    """A document for each dimension, whose token is nothing elsewhere: its score is that element of the
    query's rows. The row's largest magnitude being 128 or more of a unit, an element is held to 2^-14 of
    that unit, 2^-21 of the largest magnitude, and its terms' products and the row's sums are fp32."""
    from tilemaxsim_b200 import page_tables, page_write, paged_maxsim
    codes, scales = _pool(d, page, d)
    t = page_tables(torch.ones(d, dtype=torch.int64, device=cuda_device), page,
                    torch.randperm(d, generator=_rng(1)).to(torch.int32).to(cuda_device), d)
    page_write((448 * torch.eye(d)).half().cuda(), t, codes, scales, norm="none")
    assert (scales == 1).all()
    Q = _wide_rows(bq * nq, d, d + bq).view(bq, nq, d).to(dtype)
    got = paged_maxsim(Q.cuda(), codes, scales, t).cpu().double() / 448
    q = Q.double()
    big = q.abs().amax(-1, keepdim=True)
    bound = (big * 2.0 ** -21 + q.abs() * (nq + 4) * 2.0 ** -23).sum(1)
    off = (got - q.sum(1)).abs()
    assert (off <= bound).all(), (off / bound).max()


def _row_beside_a_scale_midpoint(rng, d, rms, above):
    """An fp32 row whose largest |y| over 448 lies within 2^-44 of the middle between two fp32 numbers, on the
    side asked for: one small element is chosen to bring the norm there. None where it does not come near.
    Nearer than 2^-49 is left out: in 64 bits a sum of squares takes at most 13 roundings of 2^-53 one after the
    other (8 fmas, 5 exchanges), of which the root keeps half, and the root, the mean, the quotient and 1 / 448
    one or two each: under 11 * 2^-53 = 2^-49.5."""
    L = np.longdouble
    x = np.clip(rng.normal(size=d), -3.5, 3.5).astype(np.float32)
    top = np.float32(4 + rng.random())
    x[0], x[1] = top, 0
    rest = (x.astype(L) ** 2).sum()
    mean = L(d) if rms else L(1)
    s = L(top) / np.sqrt(rest / mean) / 448
    low = np.nextafter(np.float32(s), np.float32(0))
    low = np.nextafter(low, np.float32(0))
    middle = (L(low) + L(np.nextafter(low, np.float32(1)))) / 2
    need = (L(top) / (448 * middle)) ** 2 * mean - rest
    x[1] = np.float32(np.sqrt(need))
    for _ in range(4):
        s = L(top) / np.sqrt((x.astype(L) ** 2).sum() / mean) / 448
        off = (s - middle) / middle
        if 2.0 ** -49 < abs(off) < 2.0 ** -44 and (off > 0) == above:
            return x, np.float32(low) if off < 0 else np.nextafter(low, np.float32(1))
        x[1] = np.nextafter(x[1], np.float32(0 if off < 0 else 1))
    return None


@pytest.mark.parametrize("above", [False, True])
@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("d,page", [(16, 16), (64, 32), (128, 32), (256, 128)])
def test_write_scales_beside_a_midpoint(d, page, rms, above, cuda_device):
    """The scale is rounded once, from what 64 bits give, also where that is next to the middle of two fp32
    numbers: rows of one-token documents, checked in 80 bits."""
    from tilemaxsim_b200 import page_tables, page_write
    rng = np.random.default_rng(d)
    rows, want = [], []
    for _ in range(20000):
        if (r := _row_beside_a_scale_midpoint(rng, d, rms, above)) is not None:
            rows.append(r[0])
            want.append(r[1])
        if len(rows) == 64:
            break
    n = len(rows)
    assert n == 64
    t = page_tables(torch.ones(n, dtype=torch.int64, device=cuda_device), page, torch.arange(n, dtype=torch.int32, device=cuda_device), n)
    codes, scales = _pool(n, page, d)
    page_write(torch.from_numpy(np.stack(rows)).cuda(), t, codes, scales, norm="rms" if rms else "l2", eps=0.0)
    np.testing.assert_array_equal(scales.cpu().numpy(), np.array(want))
