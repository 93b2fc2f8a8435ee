"""An 8-bit corpus in pages: documents can join and leave it, and are scored where they lie.

A pool of pages holds the tokens: each page has ``page_size`` rows of d e4m3 values and one fp32
scale, so a token costs one byte a dimension. A document owns as many pages as its length needs,
anywhere in the pool; its page table lists them. Four operators work on that layout, each one a
stream-ordered call of the C ABI:

    page_tables / select_page_tables   lengths -> page tables and the slot of every token
    page_write                         tokens (+ residual) -> normalised, e4m3 with a scale a page
    paged_maxsim                       queries x documents -> MaxSim scores
    page_read                          slots -> tokens

``PagedCorpus`` keeps a pool, its free pages and the tables of its documents, and builds on them.
The reference has no such corpus: its corpora are fixed tensors (src/flash_maxsim_kernel.py:248-273).
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from . import _lib

PAGE_SIZES = (16, 32, 64, 128)
_NORMS = {"none": _lib.TMS_NORM_NONE, "l2": _lib.TMS_NORM_L2, "rms": _lib.TMS_NORM_RMS}
_EPS = {"none": 0.0, "l2": 1e-12, "rms": 1e-6}
_FP32_MAX = torch.finfo(torch.float32).max


class PageTables(NamedTuple):
    """Where n documents live. page_offsets (n + 1,) int64: document i owns table entries
    [page_offsets[i], page_offsets[i + 1]); page_ids, page_docs (capacity,) int32: each entry's page
    and document, -1 past the last; token_offsets (n + 1,) int64: running token counts; slots
    (tokens,) int64: page id * page_size + row of every token, -1 past the last (or None)."""
    page_offsets: torch.Tensor
    page_ids: torch.Tensor
    page_docs: torch.Tensor
    token_offsets: torch.Tensor
    slots: torch.Tensor | None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _device(*tensors: torch.Tensor) -> torch.device:
    """The tensors' common CUDA device (as _lib.require_cuda, which says what is wrong where it is not)."""
    index = tensors[0].get_device()
    if index < 0 or any([t.get_device() != index for t in tensors]):
        return _lib.require_cuda(*tensors)
    return tensors[0].device


def _workspace(nbytes: int, dev: torch.device) -> tuple[torch.Tensor | None, int | None]:
    return _lib.workspace(nbytes, dev, align=256) if nbytes else (None, None)


def _page_size(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    return int(page_size)


def _ints(t: torch.Tensor, dtype: torch.dtype, name: str) -> torch.Tensor:
    if t.dim() != 1 or (t.dtype != dtype and (t.is_floating_point() or t.is_complex() or t.dtype == torch.bool)):
        raise ValueError(f"{name} must be a 1-D integer tensor, got {t.dtype} {tuple(t.shape)}")
    if t.dtype != dtype:
        if dtype == torch.int32 and t.element_size() >= 4:  # an id that 32 bits do not hold stays one that no pool has
            t = t.to(torch.int64).clamp(-1, (1 << 31) - 1)
        t = t.to(dtype)
    return t.contiguous()


def _tables_call(lengths, doc_ids, src_offsets, pages, page_size, n_tokens, with_slots) -> PageTables:
    lib = _lib.load()
    given = [t for t in (lengths, doc_ids, src_offsets, pages) if t is not None]
    dev = _device(*given)
    n_docs = lengths.numel() if doc_ids is None else doc_ids.numel()
    capacity = (n_tokens + n_docs * (page_size - 1)) // page_size
    with _lib.on_device(dev):
        def empty(n, dtype):
            return torch.empty(n, dtype=dtype, device=dev)
        out = PageTables(empty(n_docs + 1, torch.int64), empty(capacity, torch.int32), empty(capacity, torch.int32),
                         empty(n_docs + 1, torch.int64), empty(n_tokens, torch.int64) if with_slots else None)
        ws_bytes = lib.tms_page_tables_workspace_size(n_docs, capacity)
        ws, ws_ptr = _workspace(ws_bytes, dev)
        rc = lib.tms_page_tables(
            _ptr(lengths), lengths.numel(), _ptr(doc_ids), n_docs, _ptr(src_offsets), _ptr(pages), pages.numel(),
            page_size, _ptr(out.page_offsets), _ptr(out.token_offsets), _ptr(out.page_ids), _ptr(out.page_docs),
            capacity, _ptr(out.slots), n_tokens, ws_ptr, ws_bytes,
            _lib.stream_handle(dev))
        _lib.check(rc, "tms_page_tables")
        del ws
    return out


def page_tables(lengths: torch.Tensor, page_size: int, free_pages: torch.Tensor, n_tokens: int,
                slots: bool = True) -> PageTables:
    """The tables of new documents of the given lengths (n,), whose pages are the first ones of
    ``free_pages`` (1-D page ids), in order. n_tokens: the sum of the lengths, or a bound on it (it
    sizes the outputs, without a host synchronisation). Where the free list runs out, page ids and
    slots are -1: compare page_offsets[-1] with free_pages.numel() to see it."""
    page_size = _page_size(page_size)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    lengths = _ints(lengths, torch.int64, "lengths")
    free_pages = _ints(free_pages, torch.int32, "free_pages")
    return _tables_call(lengths, None, None, free_pages, page_size, int(n_tokens), slots)


def select_page_tables(lengths: torch.Tensor, page_size: int, page_offsets: torch.Tensor, page_ids: torch.Tensor,
                       doc_ids: torch.Tensor, n_tokens: int, slots: bool = True) -> PageTables:
    """The tables of documents ``doc_ids`` (n,) of a store with the given lengths (N,), page_offsets
    (N + 1,) and page_ids: candidates are scored or read where they lie. The same id may come more
    than once; an id outside the store is an empty document. n_tokens bounds their tokens."""
    page_size = _page_size(page_size)
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    lengths = _ints(lengths, torch.int64, "lengths")
    page_offsets = _ints(page_offsets, torch.int64, "page_offsets")
    if page_offsets.numel() < lengths.numel():
        raise ValueError(f"{lengths.numel()} lengths need as many page_offsets, got {page_offsets.numel()}")
    return _tables_call(lengths, _ints(doc_ids, torch.int64, "doc_ids"), page_offsets,
                        _ints(page_ids, torch.int32, "page_ids"), page_size, int(n_tokens), slots)


def _check_pool(codes: torch.Tensor, scales: torch.Tensor) -> tuple[int, int, int]:
    if codes.dim() != 3 or codes.dtype != torch.float8_e4m3fn or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous (n_pages, page_size, d) float8_e4m3fn tensor, got "
                         f"{codes.dtype} {tuple(codes.shape)}")
    n_pages, page_size, d = codes.shape
    _page_size(page_size)
    if d % 16 or not 0 < d <= _lib.TMS_PAGED_MAX_D:
        raise ValueError(f"d must be a multiple of 16, at most {_lib.TMS_PAGED_MAX_D}, got {d}")
    if scales.shape != (n_pages,) or scales.dtype != torch.float32 or not scales.is_contiguous():
        raise ValueError(f"scales must be a contiguous ({n_pages},) float32 tensor, got {scales.dtype} "
                         f"{tuple(scales.shape)}")
    if codes.data_ptr() % 16:
        raise ValueError("codes must be 16-byte aligned")
    return n_pages, page_size, d


def _check_tables(t: PageTables) -> int:
    offsets, ids, docs, tokens = t.page_offsets, t.page_ids, t.page_docs, t.token_offsets
    i64, i32 = torch.int64, torch.int32
    if not (offsets.dtype is i64 and tokens.dtype is i64 and offsets.dim() == 1 and tokens.dim() == 1
            and offsets.is_contiguous() and tokens.is_contiguous()):
        raise ValueError("page_offsets and token_offsets must be contiguous 1-D int64 tensors")
    if not (ids.dtype is i32 and docs.dtype is i32 and ids.dim() == 1 and docs.dim() == 1
            and ids.is_contiguous() and docs.is_contiguous()):
        raise ValueError("page_ids and page_docs must be contiguous 1-D int32 tensors")
    if ids.numel() != docs.numel():
        raise ValueError("page_ids and page_docs must have the same length")
    n = offsets.numel() - 1
    if n < 0 or tokens.numel() != n + 1:
        raise ValueError("page_offsets and token_offsets must have n_docs + 1 entries each")
    return n


def _fits(t: torch.Tensor) -> bool:
    """Whether rows of t can be read 16 bytes at a time as they lie."""
    if t.data_ptr() % 16:
        return False
    each = 16 // t.element_size()  # elements of 16 bytes; a contiguous row has a multiple of them
    return t.is_contiguous() or (t.stride(-1) == 1 and all(s % each == 0 and s >= 0 for s in t.stride()[:-1]))


def page_write(x: torch.Tensor, tables: PageTables, codes: torch.Tensor, scales: torch.Tensor, *,
               residual: torch.Tensor | None = None, weight: torch.Tensor | None = None, norm: str = "l2",
               eps: float | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Writes documents into their pages: h = x + residual; y = h / max(|h|, eps) for norm "l2", h /
    sqrt(mean(h^2) + eps) * weight for "rms", h for "none"; each page's scale is its largest |y|
    over 448, its codes are e4m3(y / scale).

    x: the tokens of all documents (T, d), document i's at token_offsets[i].., or a padded batch
    (n_docs, L, d) whose document i has its tokens in the first rows (lengths must not exceed L);
    fp16, bf16 or fp32; residual: same shape and dtype; weight: (d,) of x's dtype. codes and scales
    are updated in place and returned; pages that the tables do not name keep their content. A page
    belongs to one document: of one that the tables name twice the content is undefined."""
    lib = _lib.load()
    if norm not in _NORMS:
        raise ValueError(f"norm must be one of {sorted(_NORMS)}, got {norm!r}")
    if weight is not None and norm != "rms":
        raise ValueError("weight goes with norm='rms' only")
    eps = _EPS[norm] if eps is None else float(eps)
    if not 0.0 <= eps <= _FP32_MAX or (eps > 0.0 and np.float32(eps) == 0):  # the kernel takes it in fp32
        raise ValueError(f"eps must be finite and not negative, in fp32 too, got {eps}")
    n_pages, page_size, d = _check_pool(codes, scales)
    n_docs = _check_tables(tables)
    dev = _device(x, codes, scales, tables.page_offsets, tables.page_ids, tables.page_docs, tables.token_offsets,
                  *(t for t in (residual, weight) if t is not None))
    if x.dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {x.dtype}; use float16, bfloat16 or float32")
    if x.dim() not in (2, 3) or x.shape[-1] != d:
        raise ValueError(f"expected x (T, {d}) or (n_docs, L, {d}), got {tuple(x.shape)}")
    padded = x.dim() == 3
    if padded and x.shape[0] != n_docs:
        raise ValueError(f"a padded x has a document for each of the tables' {n_docs}, got {x.shape[0]}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("residual must have the shape and dtype of x")
    if weight is not None and (weight.shape != (d,) or weight.dtype != x.dtype):
        raise ValueError(f"weight must be ({d},) {x.dtype}, got {tuple(weight.shape)} {weight.dtype}")
    with _lib.on_device(dev):
        if not _fits(x) or (residual is not None and (not _fits(residual) or residual.stride() != x.stride())):
            x = x.clone(memory_format=torch.contiguous_format)
            residual = None if residual is None else residual.clone(memory_format=torch.contiguous_format)
        if weight is not None:
            weight = weight.contiguous()
            weight = weight if weight.data_ptr() % 16 == 0 else weight.clone()
        rc = lib.tms_page_write(
            _ptr(x), _lib.DTYPE_CODE[x.dtype], x.shape[-2], x.stride(0) if padded and n_docs > 1 else 0,
            x.stride(-2) if x.shape[-2] > 1 else d, int(padded),  # a dimension of one may have any stride
            _ptr(residual), _ptr(weight), _NORMS[norm], eps, d, page_size, _ptr(tables.page_offsets),
            _ptr(tables.token_offsets), _ptr(tables.page_ids), _ptr(tables.page_docs), n_docs,
            tables.page_ids.numel(), _ptr(codes), _ptr(scales), n_pages, _lib.stream_handle(dev))
        _lib.check(rc, "tms_page_write")
    return codes, scales


def page_read(codes: torch.Tensor, scales: torch.Tensor, slots: torch.Tensor,
              dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The tokens in the given slots (n,) as (n, d) fp16, bf16 or fp32 values scale * code; a slot
    outside the pool (-1 among them) gives a row of zeros."""
    lib = _lib.load()
    n_pages, page_size, d = _check_pool(codes, scales)
    if dtype not in _lib.DTYPE_CODE:
        raise TypeError(f"unsupported dtype {dtype}; use float16, bfloat16 or float32")
    slots = _ints(slots, torch.int64, "slots")
    dev = _device(codes, scales, slots)
    with _lib.on_device(dev):
        out = torch.empty((slots.numel(), d), dtype=dtype, device=dev)
        rc = lib.tms_page_read(_ptr(codes), _ptr(scales), n_pages, page_size, d, _ptr(slots), slots.numel(),
                               _ptr(out), _lib.DTYPE_CODE[dtype], _lib.stream_handle(dev))
        _lib.check(rc, "tms_page_read")
    return out


def paged_maxsim(Qb: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, tables: PageTables) -> torch.Tensor:
    """MaxSim of every query against every document of the tables, straight from the pages.

    Qb: (B_q, Nq, d) or (Nq, d), fp16 or bf16 (fp32 is rounded to fp16, where magnitudes of 65,520 and
    more are infinite and make the query's scores NaN: give such queries in bf16). Returns fp32 (B_q, n_docs),
    or (n_docs,) for a single 2-D query. A document without pages scores -inf, one with a NaN among
    its pages NaN."""
    lib = _lib.load()
    n_pages, page_size, d = _check_pool(codes, scales)
    n_docs = _check_tables(tables)
    single = Qb.dim() == 2
    if single:
        Qb = Qb.unsqueeze(0)
    dev = _device(Qb, codes, scales, tables.page_offsets, tables.page_ids, tables.page_docs)
    if Qb.dim() != 3 or Qb.shape[2] != d:
        raise ValueError(f"expected Q (B_q, Nq, {d}) or (Nq, {d}), got {tuple(Qb.shape)}")
    if Qb.dtype == torch.float32:
        Qb = Qb.to(torch.float16)
    if Qb.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {Qb.dtype}; use float16, bfloat16 or float32")
    Bq, Nq, _ = Qb.shape
    if Nq == 0:
        raise ValueError("a query needs at least one token")
    with _lib.on_device(dev):
        Qb = Qb.contiguous()
        Qb = Qb if Qb.data_ptr() % 16 == 0 else Qb.clone()
        out = torch.empty((Bq, n_docs), dtype=torch.float32, device=dev)
        if Bq > 0 and n_docs > 0:
            ws_bytes = lib.tms_paged_workspace_size(Bq, Nq, d, n_docs, page_size, tables.page_ids.numel())
            ws, ws_ptr = _workspace(ws_bytes, dev)
            rc = lib.tms_paged_maxsim(
                _ptr(Qb), _lib.DTYPE_CODE[Qb.dtype], Bq, Nq, d, _ptr(codes), _ptr(scales), n_pages, page_size,
                _ptr(tables.page_offsets), _ptr(tables.page_ids), _ptr(tables.page_docs), n_docs,
                tables.page_ids.numel(), _ptr(out), ws_ptr, ws_bytes,
                _lib.stream_handle(dev))
            _lib.check(rc, "tms_paged_maxsim")
            del ws
    return out[0] if single else out


class PagedCorpus:
    """A pool of pages with room for n_pages * page_size tokens and max_docs documents.

    Documents get ascending ids in the order they are added; a removed document's id is not given
    out again and scores -inf, and its row of the tables counts towards max_docs until ``compact``
    drops it and numbers the others anew. All device buffers are allocated here and updated in place, so a
    captured search (``GraphedStep``) sees later additions to the documents it was captured for
    being removed, and never reads memory that was freed; documents added after the capture are not
    in its output (after a ``compact``, capture it again). ``add`` and ``remove`` synchronise with the host; order them against searches on
    other streams as with any tensor that one stream writes and another reads."""

    def __init__(self, d: int, n_pages: int, max_docs: int, page_size: int = 32,
                 device: torch.device | str = "cuda"):
        self.page_size = _page_size(page_size)
        if d % 16 or not 0 < d <= _lib.TMS_PAGED_MAX_D:
            raise ValueError(f"d must be a multiple of 16, at most {_lib.TMS_PAGED_MAX_D}, got {d}")
        if n_pages < 1 or max_docs < 1 or n_pages * page_size >= 1 << 31 or max_docs >= 1 << 31:
            raise ValueError("n_pages and max_docs must be positive, n_pages * page_size and max_docs below 2^31, got "
                             f"{n_pages} pages of {page_size} and {max_docs}")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"tilemaxsim_b200 scores CUDA tensors only (no CPU fallback); got {device}")
        self.d, self.n_pages, self.max_docs = d, n_pages, max_docs
        self.codes = torch.zeros(n_pages, self.page_size, d, dtype=torch.float8_e4m3fn, device=device)
        self.scales = torch.zeros(n_pages, dtype=torch.float32, device=device)
        self.device = self.codes.device
        self._lengths = torch.zeros(max_docs, dtype=torch.int64, device=device)
        self._page_offsets = torch.zeros(max_docs + 1, dtype=torch.int64, device=device)
        self._token_offsets = torch.zeros(max_docs + 1, dtype=torch.int64, device=device)
        self._page_ids = torch.full((n_pages,), -1, dtype=torch.int32, device=device)
        self._page_docs = torch.full((n_pages,), -1, dtype=torch.int32, device=device)
        # free pages, the next ones to give out at the end
        self._free = torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device)
        self._host_lengths = np.zeros(max_docs, dtype=np.int64)
        self._longest = self._n_tokens = 0  # a bound on the lengths, and their sum
        self.n_docs = 0  # documents added so far, removed ones included
        self.n_free = n_pages

    @property
    def tables(self) -> PageTables:
        """The tables of all documents (views of the corpus's own buffers, without slots). Their capacity
        is the entries in use: later removals leave fewer, and documents added later are not theirs."""
        n, used = self.n_docs, self.n_pages - self.n_free
        return PageTables(self._page_offsets[:n + 1], self._page_ids[:used], self._page_docs[:used],
                          self._token_offsets[:n + 1], None)

    def _capturing(self) -> bool:
        with _lib.on_device(self.device):
            return torch.cuda.is_current_stream_capturing()

    def _pages_of(self, lengths: np.ndarray) -> int:
        return int(((lengths + self.page_size - 1) // self.page_size).sum())

    def add(self, x: torch.Tensor, lengths: torch.Tensor | list[int], *, residual: torch.Tensor | None = None,
            weight: torch.Tensor | None = None, norm: str = "l2", eps: float | None = None) -> torch.Tensor:
        """Adds documents of the given lengths, their tokens in x as page_write takes them (ragged
        (T, d) or padded (n, L, d)). Returns their ids (n,) int64. Raises ValueError, with the corpus
        as it was, when the pool or the document table has no room."""
        host = np.asarray(lengths.tolist() if isinstance(lengths, torch.Tensor) else lengths)
        if host.ndim != 1 or (host.size and host.dtype.kind not in "iu"):
            raise ValueError(f"lengths must be a 1-D list or tensor of integers, got {host.dtype} {host.shape}")
        host = host.astype(np.int64)
        n, n_tok, first = host.size, int(host.sum()), self.n_docs
        if n and host.min() < 0:
            raise ValueError("lengths must not be negative")
        if n and host.max() > self.n_pages * self.page_size:  # before sums and pages of such lengths can wrap
            raise ValueError(f"{-(-int(host.max()) // self.page_size)} pages are needed, {self.n_free} are free")
        if x.dim() == 2 and x.shape[0] != n_tok:
            raise ValueError(f"x has {x.shape[0]} tokens, the lengths sum to {n_tok}")
        if x.dim() == 3 and (x.shape[0] != n or host.max(initial=0) > x.shape[1]):
            raise ValueError(f"lengths do not fit a padded batch of shape {tuple(x.shape)}")
        need = self._pages_of(host)
        if need > self.n_free:
            raise ValueError(f"{need} pages are needed, {self.n_free} are free")
        if first + n > self.max_docs:
            raise ValueError(f"no room for {n} documents: {first} of {self.max_docs} rows are taken, {self._gone()} of "
                             "them by documents without tokens, which compact() drops")
        ids = torch.arange(first, first + n, device=self.device)
        if n == 0:
            return ids
        with torch.cuda.device(self.device):
            dev_lengths = torch.from_numpy(host).to(self.device)
            free = self._free[self.n_free - need:self.n_free].flip(0)
            t = page_tables(dev_lengths, self.page_size, free, n_tok, slots=False)
            page_write(x, t, self.codes, self.scales, residual=residual, weight=weight, norm=norm, eps=eps)
            used = self.n_pages - self.n_free
            self._page_ids[used:used + need] = t.page_ids[:need]
            self._page_docs[used:used + need] = t.page_docs[:need] + first
            self._page_offsets[first + 1:first + 1 + n] = t.page_offsets[1:] + used
            self._page_offsets[first + 1 + n:] = used + need
            self._token_offsets[first + 1:first + 1 + n] = t.token_offsets[1:] + self._token_offsets[first]
            self._token_offsets[first + 1 + n:] = self._token_offsets[first + n].clone()
            self._lengths[first:first + n] = dev_lengths
        self._host_lengths[first:first + n] = host
        self._longest = max(self._longest, int(host.max()))
        self._n_tokens += n_tok
        self.n_docs += n
        self.n_free -= need
        return ids

    def _host_ids(self, doc_ids: torch.Tensor | list[int]) -> np.ndarray:
        ids = np.asarray(doc_ids.tolist() if isinstance(doc_ids, torch.Tensor) else doc_ids)
        if ids.ndim != 1 or (ids.size and ids.dtype.kind not in "iu"):
            raise ValueError(f"document ids must be a 1-D list or tensor of integers, got {ids.dtype} {ids.shape}")
        if ids.size and (ids.min() < 0 or ids.max() >= self.n_docs):
            raise IndexError(f"document ids must be in [0, {self.n_docs})")
        return ids.astype(np.int64)

    def remove(self, doc_ids: torch.Tensor | list[int]) -> None:
        """Removes documents and frees their pages. An id may come twice; a document that is removed
        already, or empty, is left as it is."""
        ids = np.unique(self._host_ids(doc_ids))
        ids = ids[self._host_lengths[ids] > 0]
        if not ids.size:
            return
        freed = self._pages_of(self._host_lengths[ids])
        used = self.n_pages - self.n_free
        with torch.cuda.device(self.device):
            gone = torch.zeros(self.max_docs, dtype=torch.bool, device=self.device)
            gone[torch.from_numpy(ids).to(self.device)] = True
            out = gone[self._page_docs[:used].long()]
            pages, docs = self._page_ids[:used].clone(), self._page_docs[:used].clone()
            self._free[self.n_free:self.n_free + freed] = pages[out]
            self._page_ids[:used - freed] = pages[~out]
            self._page_docs[:used - freed] = docs[~out]
            self._page_ids[used - freed:used] = -1
            self._page_docs[used - freed:used] = -1
            self._lengths[gone] = 0
            self._count_offsets()
        self._n_tokens -= int(self._host_lengths[ids].sum())
        self._host_lengths[ids] = 0
        self.n_free += freed

    def _without_tokens(self, doc_ids: torch.Tensor) -> torch.Tensor:
        """Which of the documents doc_ids (n,), ids of the corpus on its device, are removed or empty: (n,) bool."""
        return self._lengths[doc_ids] == 0

    def _count_offsets(self) -> None:
        self._page_offsets[1:] = torch.cumsum((self._lengths + self.page_size - 1) // self.page_size, 0)
        self._token_offsets[1:] = torch.cumsum(self._lengths, 0)

    def _gone(self) -> int:
        return self.n_docs - int(np.count_nonzero(self._host_lengths[:self.n_docs]))

    def compact(self) -> torch.Tensor:
        """Drops the rows of documents without tokens (removed, or added empty) and numbers the others
        anew, in their order: document i becomes the returned (n_docs,) int64 ids' entry i, -1 if it
        is dropped. No token moves. Ids held elsewhere (an ``IVFIndex``, a captured search) are the old ones."""
        n, used = self.n_docs, self.n_pages - self.n_free
        old = np.flatnonzero(self._host_lengths[:n])
        new = np.full(n, -1, dtype=np.int64)
        new[old] = np.arange(old.size)
        with torch.cuda.device(self.device):
            ids = torch.from_numpy(new).to(self.device)
            self._page_docs[:used] = ids[self._page_docs[:used].long()].to(torch.int32)
            kept = self._lengths[torch.from_numpy(old).to(self.device)]
            self._lengths[:n] = 0
            self._lengths[:old.size] = kept
            self._count_offsets()
        self._host_lengths[:old.size] = self._host_lengths[old]
        self._host_lengths[old.size:n] = 0
        self._longest = int(self._host_lengths.max())
        self.n_docs = old.size
        return ids

    def select(self, doc_ids: torch.Tensor, n_tokens: int | None = None, slots: bool = False) -> PageTables:
        """The tables of the given documents (an id outside the corpus is an empty document).
        n_tokens bounds their tokens. By default it is the longest document's length for each, and
        where that is far more than the corpus holds, their own sum, for which the host waits (but
        not in a capture, whose replays bring other documents: the bound stays)."""
        doc_ids = _ints(doc_ids, torch.int64, "doc_ids")
        if n_tokens is None:
            n_tokens = doc_ids.numel() * self._longest
            if n_tokens > max(4 * self._n_tokens, 1 << 24) and not self._capturing():
                inside = (doc_ids >= 0) & (doc_ids < self.n_docs)
                n_tokens = int(self._lengths[doc_ids.clamp(0, self.max_docs - 1)][inside].sum())
        n = self.n_docs
        return select_page_tables(self._lengths[:n], self.page_size, self._page_offsets[:n + 1], self._page_ids, doc_ids,
                                  n_tokens, slots=slots)

    def score_queries(self, Qb: torch.Tensor, doc_ids: torch.Tensor | None = None) -> torch.Tensor:
        """Qb (B_q, Nq, d) or (Nq, d) -> fp32 scores (B_q, n) or (n,) of all documents, or of doc_ids
        (n,) in their order."""
        tables = self.tables if doc_ids is None else self.select(doc_ids)
        return paged_maxsim(Qb, self.codes, self.scales, tables)

    def search(self, Qb: torch.Tensor, k: int, doc_ids: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The k best documents of each query, of all or of the candidates doc_ids (n,): scores
        (B_q, k) fp32 and ids (B_q, k) int64, by score descending (NaN last) and id ascending. An id
        that comes twice among the candidates is ranked twice. Documents without tokens (removed, or
        added empty) come after all others with -inf: as id -1 in a search of all documents, by their
        own ids among candidates, where ids outside the corpus end the list as -1."""
        if doc_ids is not None:
            doc_ids = _ints(doc_ids, torch.int64, "doc_ids")
            if doc_ids.numel() > _lib.TMS_TOPK_MAX_IDS:  # ties go by column there
                outside = (doc_ids < 0) | (doc_ids >= self.n_docs)
                doc_ids = doc_ids.masked_fill(outside, torch.iinfo(torch.int64).max).sort().values
        return self._topk(self.score_queries(Qb, doc_ids), k, doc_ids)

    def _topk(self, scores: torch.Tensor, k: int, doc_ids: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
        lib = _lib.load()
        single = scores.dim() == 1
        rows, n = scores.shape if not single else (1, scores.numel())
        if not 0 < k <= n:
            raise ValueError(f"k={k} must be in [1, n={n}]")
        with _lib.on_device(self.device):
            vals = torch.empty((rows, k), dtype=torch.float32, device=self.device)
            ids = torch.empty((rows, k), dtype=torch.int64, device=self.device)
            ws_bytes = lib.tms_topk_docs_workspace_size(rows, n, k)
            ws, ws_ptr = _workspace(ws_bytes, self.device)
            rc = lib.tms_topk_docs(_ptr(scores), rows, n, n, k, _ptr(doc_ids), _ptr(self._lengths), self.n_docs,
                                   _ptr(vals), _ptr(ids), ws_ptr, ws_bytes, _lib.stream_handle(self.device))
            _lib.check(rc, "tms_topk_docs")
            del ws
        return (vals[0], ids[0]) if single else (vals, ids)

    def tokens(self, doc_ids: torch.Tensor | list[int], dtype: torch.dtype = torch.float16
               ) -> tuple[torch.Tensor, torch.Tensor]:
        """The stored tokens of the given documents: (T, d) values and (n + 1,) int64 offsets, the
        layout maxsim_batched and save_shard take."""
        ids = self._host_ids(doc_ids)
        t = self.select(torch.from_numpy(ids).to(self.device), int(self._host_lengths[ids].sum()), slots=True)
        return page_read(self.codes, self.scales, t.slots, dtype), t.token_offsets
