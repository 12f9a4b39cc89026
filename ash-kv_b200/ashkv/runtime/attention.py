"""Attention over tiered pages while a sequence is being generated.

The reference only moves pages: its engine promotes a compressed page before
it attends it (ashkv/runtime/migrate.py:35-191).  Here a decode step reads
every page where its tier keeps it, so a demoted page costs its compressed
bytes, and the step also produces what decides about pages:

* :func:`decode_attention`: one new query per sequence over its page list
  (pool rows, INT8 / FP8 / INT4 / dithered slots alike), split over the length
  and joined; with ``page_mass`` it keeps a decayed sum of the attention
  weight that each page drew;
* :class:`PageBounds` and :func:`select_pages`: int8 bounds of each page's
  keys, and the pages that a query scores highest by them; their positions go
  to ``decode_attention(selected=...)``;
* :func:`evict_pages`: the pages of least accumulated mass leave a sequence
  that is over its budget.

Pages are rows of a :class:`~ashkv.runtime.batch.DevicePageTable`; a sequence
is a row of ``page_ids`` [n_seqs, max_pages] int32 (page-table rows in order;
entries past the sequence's last page are not read) and its ``lengths`` entry
(int32 tokens).  All calls run on the current stream of the tensors' device,
allocate their outputs and workspace from torch's allocator (each call its
own), never wait for the device, and can be captured in a CUDA graph.  A page
that does not exist is left out and sets ``_native.FLAG_INDEX_RANGE`` in
``status`` (int32 [1], if given).
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from typing import Mapping, NamedTuple, Optional

import torch

from .. import _native
from .batch import NUM_TIERS, DevicePageTable, KVLayers, TierStore


def _on(device: torch.device):
    """Make ``device`` current for a call, if it is not already."""
    return _SAME if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


_SAME = nullcontext()


def _refuse(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    """Says what keeps ``t`` from being a tensor of ``dtype`` and ``shape`` on ``device``."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")


def _require_dense(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> None:
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device.index:  # (-1 on the host)
        _refuse(t, name, dtype, shape, device)
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _require_rows(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: torch.device) -> torch.Tensor:
    """[rows, width], dense in its width, with any row stride that keeps rows apart (returned with a
    stride of at least the width: a single row may carry any)."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device.index:  # (-1 on the host)
        _refuse(t, name, dtype, shape, device)
    if t.is_contiguous():
        return t if shape[0] != 1 or t.stride(0) >= shape[1] else t.view(-1).view(shape)
    if shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must be dense in its last dimension")
    if t.stride(0) < shape[1]:
        if shape[0] > 1:
            raise ValueError(f"{name} rows overlap")
        return t.as_strided(shape, (shape[1], 1))
    return t


def _require_query(q: torch.Tensor) -> None:
    if q.dim() != 3:
        raise ValueError("q must be [n_seqs, heads_q, head_dim]")
    if not q.is_cuda or q.dtype != torch.bfloat16:
        _refuse(q, "q", torch.bfloat16, q.shape, q.device)
    if q.shape[2] not in (64, 128):
        raise ValueError("head_dim must be 64 or 128")
    if q.stride(2) != 1:
        raise ValueError("q must be dense in its last dimension")
    if q.shape[1] == 0:
        raise ValueError("q has no heads")


_MOST = 2 ** 31 - 1  # the library takes sizes as int32


def _require_window(window: Optional[int], sinks: int) -> None:
    if window is not None and not 0 < window <= _MOST:
        raise ValueError("window must be at least 1 and fit an int32")
    if not 0 <= sinks <= _MOST:
        raise ValueError("sinks must not be negative and fit an int32")
    if window is None and sinks:
        raise ValueError("sinks need a window")


def _require_tokens_per_page(n: int) -> None:
    if not 0 < n <= _MOST:
        raise ValueError("tokens_per_page must be positive and fit an int32")


def _require_lists(page_ids: torch.Tensor, lengths: torch.Tensor, n_seqs: int, device: torch.device) -> torch.Tensor:
    if page_ids.dim() != 2:
        raise ValueError("page_ids must be [n_seqs, max_pages]")
    if page_ids.shape[1] > _MOST or n_seqs > _MOST:
        raise ValueError("page_ids is too large")
    _require_dense(lengths, "lengths", torch.int32, (n_seqs,), device)
    return _require_rows(page_ids, "page_ids", torch.int32, (n_seqs, page_ids.shape[1]), device)


def _require_starts(starts: torch.Tensor, n_seqs: int, device: torch.device) -> None:
    _require_dense(starts, "starts", torch.int32, (n_seqs + 1,), device)


_StoreDescs = _native.TierStoreDesc * NUM_TIERS
_NO_STORES = bytes(_StoreDescs(*(_native.TierStoreDesc(
    None, 0, 0, _native.PAGE_NONE if t else _native.PAGE_BF16, None, None) for t in range(NUM_TIERS))))


def _pages_desc(table: DevicePageTable, kv: KVLayers, stores: Optional[Mapping[int, TierStore]], head_dim: int,
                tokens_per_page: int, device: torch.device):
    """The ashkv_paged_kv_t of a table, its pool and its stores, and the store array it points to."""
    if kv.row_len % head_dim:
        raise ValueError(f"the pool's rows of {kv.row_len} values are no whole number of heads of {head_dim}")
    pool = kv.k[0].shape
    if len(pool) > 2 and pool[-1] != head_dim:
        raise ValueError(f"the pool's heads have {pool[-1]} channels, not {head_dim}")
    n = table.tier.numel()
    _require_dense(table.tier, "table.tier", torch.int8, (n,), device)
    _require_dense(table.layer, "table.layer", torch.int32, (n,), device)
    _require_dense(table.token_start, "table.token_start", torch.int32, (n,), device)
    _require_dense(table.slot, "table.slot", torch.int32, (n,), device)
    if kv.k[0].device != device:
        raise ValueError(f"the KV pool is on {kv.k[0].device}, expected {device}")
    _require_tokens_per_page(tokens_per_page)
    descs = _StoreDescs.from_buffer_copy(_NO_STORES)
    cap = 0
    for t, s in (stores or {}).items():
        if not 0 < int(t) < NUM_TIERS:
            raise ValueError(f"tier {t} cannot have a store")
        if s.data.device != device:
            raise ValueError(f"the store of tier {t} is on {s.data.device}, expected {device}")
        if s.tokens_per_page != tokens_per_page or s.row_len != kv.row_len:
            raise _native.KernelError("tier store", _native.BAD_ARGUMENT,
                                      f"the store of tier {t} was laid out for pages of {s.tokens_per_page} x {s.row_len}, "
                                      f"not {tokens_per_page} x {kv.row_len}")
        if s.data.numel() * s.data.element_size() < s.n_slots * s.slot_bytes:
            raise ValueError(f"the store of tier {t} holds fewer than its {s.n_slots} slots")
        descs[int(t)] = s.desc()
        if s.format in (_native.PAGE_NBIT4, _native.PAGE_NBIT2):
            if cap and cap != s.outlier_cap:
                raise ValueError("dithered stores must share one outlier capacity")
            cap = s.outlier_cap
    desc = _native.PagedKVDesc(
        table.tier.data_ptr(), table.layer.data_ptr(), table.token_start.data_ptr(), table.slot.data_ptr(), n,
        kv.k_ptrs.data_ptr(), kv.v_ptrs.data_ptr(), kv.k[0].shape[0], kv.row_len, kv.n_layers, tokens_per_page,
        kv.row_len // head_dim, head_dim, cap, _native.ctypes.addressof(descs))
    return desc, descs


def decode_attention(q: torch.Tensor, table: DevicePageTable, kv: KVLayers,
                     stores: Optional[Mapping[int, TierStore]], page_ids: torch.Tensor, lengths: torch.Tensor, *,
                     tokens_per_page: int = 16, scale: Optional[float] = None,
                     selected: Optional[torch.Tensor] = None, selected_count: Optional[torch.Tensor] = None,
                     page_mass: Optional[torch.Tensor] = None, decay: float = 1.0,
                     window: Optional[int] = None, sinks: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False,
                     status: Optional[torch.Tensor] = None):
    """Attention of one new token per sequence over its pages, whatever tier holds them.

    ``q`` is bf16 [n_seqs, heads_q, head_dim] (any strides with a dense last dimension), head_dim
    64 or 128; query head h reads key head h / (heads_q / heads_kv).  ``stores`` maps each
    compressed tier to its store, as for :class:`~ashkv.runtime.batch.BatchMigrator`.  ``scale``
    defaults to 1/sqrt(head_dim).  Returns the bf16 result [n_seqs, heads_q, head_dim]
    (``out``, if given), with ``return_lse`` also the fp32 log of the sum of exponentials
    [n_seqs, heads_q].  A sequence of length 0 gives zeros and -inf.  The lists hold up to
    2^31 - 1 - 2^16 entries together.  A store must have been made for pages of
    ``tokens_per_page`` tokens of the pool's rows.

    Compressed codes count as the numbers they stand for (a decode's rounding to bf16 is left
    out; dithered pages count as the bf16 values of their decoder).

    ``selected`` [n_seqs, heads_kv, width] int32 with ``selected_count`` [n_seqs, heads_kv]
    restricts each key head to those page positions (see :func:`select_pages`).  ``page_mass``
    fp32 [n_seqs, max_pages] is updated in place: for each position j that holds tokens,
    ``page_mass[b, j] = decay * page_mass[b, j] +`` the attention weight of page j summed over
    heads and tokens; it cannot be combined with ``selected``.

    With ``window`` only the newest ``window`` tokens and the first ``sinks`` are attended, and
    only their pages are looked up and read (the list's other entries may be anything);
    ``selected`` has first and last pages of its own and takes no window."""
    _require_query(q)
    _require_window(window, sinks)
    n_seqs, heads_q, d = q.shape
    dev = q.device
    page_ids = _require_lists(page_ids, lengths, n_seqs, dev)
    desc, keep = _pages_desc(table, kv, stores, d, tokens_per_page, dev)
    if heads_q % desc.heads_kv:
        raise ValueError(f"{heads_q} query heads are no multiple of {desc.heads_kv} key heads")
    width = page_ids.shape[1]
    if (selected is None) != (selected_count is None):
        raise ValueError("selected and selected_count go together")
    if selected is not None:
        if page_mass is not None:
            raise ValueError("page_mass cannot be combined with selected")
        if window is not None:
            raise ValueError("a window cannot be combined with selected")
        if selected.dim() != 3 or selected.shape[2] == 0:
            raise ValueError("selected must be [n_seqs, heads_kv, width] with a width of at least 1")
        width = selected.shape[2]
        _require_dense(selected, "selected", torch.int32, (n_seqs, desc.heads_kv, width), dev)
        _require_dense(selected_count, "selected_count", torch.int32, (n_seqs, desc.heads_kv), dev)
    if page_mass is not None:
        page_mass = _require_rows(page_mass, "page_mass", torch.float32, page_ids.shape, dev)
    if status is not None:
        _require_dense(status, "status", torch.int32, (1,), dev)
    if out is None:
        out = q.new_empty(n_seqs, heads_q, d)
    else:
        _require_dense(out, "out", torch.bfloat16, (n_seqs, heads_q, d), dev)
    lse = torch.empty(n_seqs, heads_q, dtype=torch.float32, device=dev) if return_lse else None
    if n_seqs:
        with _on(dev):
            scratch = torch.empty(_native.decode_scratch_floats(n_seqs, heads_q, desc.heads_kv, d, width,
                                                                page_mass is not None),
                                  dtype=torch.float32, device=dev)
            scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
            if window is None:
                _native.decode_attention(desc, q, page_ids, lengths, selected, selected_count, scale, page_mass,
                                         float(decay), out, lse, scratch, status)
            else:
                _native.decode_attention_window(desc, q, page_ids, lengths, window, sinks, scale, page_mass,
                                                float(decay), out, lse, scratch, status)
    return (out, lse) if return_lse else out


def prompt_attention(q: torch.Tensor, table: DevicePageTable, kv: KVLayers,
                     stores: Optional[Mapping[int, TierStore]], page_ids: torch.Tensor, lengths: torch.Tensor,
                     starts: torch.Tensor, *, tokens_per_page: int = 16, scale: Optional[float] = None,
                     window: Optional[int] = None, sinks: int = 0, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False, status: Optional[torch.Tensor] = None):
    """Causal attention of the new tokens of each sequence (a prompt, a chunk of one, drafted tokens).

    ``q`` is bf16 [n_rows, heads_q, head_dim] (any strides with a dense last dimension); rows
    ``starts[b] .. starts[b + 1] - 1`` (int32 [n_seqs + 1], ascending) are the newest tokens of sequence
    b, whose ``lengths`` count them and whose pages hold their keys and values already (see
    :func:`~ashkv.runtime.cache.write_kv`).  The query at position p attends the tokens up to p; with
    ``window`` only the newest ``window`` of them and the first ``sinks``, and pages that no query of a
    sequence sees are not looked up.  Pages of any tier are read where they lie; compressed ones count
    as the bf16 values that they decode to (what :func:`~ashkv.runtime.cache.read_kv` gives).  Returns
    the bf16 result [n_rows, heads_q, head_dim] (``out``, if given: contiguous, 16-byte aligned, not
    ``q``), with ``return_lse`` also the fp32 log of the sum of exponentials [n_rows, heads_q].  A query
    without tokens gives zeros and -inf.  Rows of no sequence are left as they were."""
    _require_query(q)
    _require_window(window, sinks)
    n_rows, heads_q, d = q.shape
    dev = q.device
    n_seqs = lengths.numel()
    page_ids = _require_lists(page_ids, lengths, n_seqs, dev)
    _require_starts(starts, n_seqs, dev)
    desc, keep = _pages_desc(table, kv, stores, d, tokens_per_page, dev)
    if heads_q % desc.heads_kv:
        raise ValueError(f"{heads_q} query heads are no multiple of {desc.heads_kv} key heads")
    if status is not None:
        _require_dense(status, "status", torch.int32, (1,), dev)
    if out is None:
        out = q.new_empty(n_rows, heads_q, d)
    else:
        _require_dense(out, "out", torch.bfloat16, (n_rows, heads_q, d), dev)
        if out.data_ptr() % 16:
            raise ValueError("out must be 16-byte aligned")
        if out.data_ptr() == q.data_ptr() and n_rows:
            raise ValueError("out must not be q")
    lse = torch.empty(n_rows, heads_q, dtype=torch.float32, device=dev) if return_lse else None
    if n_seqs and n_rows:
        with _on(dev):
            scratch = torch.empty(_native.prompt_scratch_floats(n_rows, n_seqs, heads_q, desc.heads_kv, d, kv.n_layers),
                                  dtype=torch.float32, device=dev)
            _native.prompt_attention(desc, q, page_ids, lengths, starts, window or 0, sinks,
                                     1.0 / math.sqrt(d) if scale is None else float(scale), out, lse, scratch, status)
    return (out, lse) if return_lse else out


class PageBounds:
    """Int8 bounds of the keys of each page of a table, per key head.

    ``codes`` int8 [n_pages, heads_kv, 2, head_dim] holds a lower and an upper bound per channel
    in units of 2^``exponents`` (int8 [n_pages, heads_kv]), rounded outwards.  A page's bounds
    are taken while it is in the BF16 tier (:meth:`update`) and stay valid, to the codec's
    error, wherever it is moved."""

    def __init__(self, codes: torch.Tensor, exponents: torch.Tensor):
        if codes.dim() != 4 or codes.shape[2] != 2 or codes.shape[3] not in (64, 128):
            raise ValueError("codes must be [n_pages, heads_kv, 2, head_dim] with a head_dim of 64 or 128")
        _require_dense(codes, "codes", torch.int8, tuple(codes.shape), codes.device)
        _require_dense(exponents, "exponents", torch.int8, tuple(codes.shape[:2]), codes.device)
        if codes.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        self.codes, self.exponents = codes, exponents

    @staticmethod
    def empty(n_pages: int, heads_kv: int, head_dim: int, device: torch.device) -> "PageBounds":
        return PageBounds(torch.zeros(n_pages, heads_kv, 2, head_dim, dtype=torch.int8, device=device),
                          torch.zeros(n_pages, heads_kv, dtype=torch.int8, device=device))

    def update(self, table: DevicePageTable, kv: KVLayers, pages: torch.Tensor, *,
               count: Optional[torch.Tensor] = None, valid: Optional[torch.Tensor] = None,
               tokens_per_page: int = 16, status: Optional[torch.Tensor] = None) -> None:
        """Bounds of the listed BF16 pages (int32 page-table rows; the first ``*count`` of them, if
        given): ``valid[i]`` tokens of page ``pages[i]``, all of them without ``valid``.  Other rows
        are left as they were.  A page listed twice must have one ``valid``."""
        dev = self.codes.device
        if pages.numel() > _MOST:
            raise ValueError("pages is too long")
        desc, keep = _pages_desc(table, kv, None, self.codes.shape[3], tokens_per_page, dev)
        if desc.heads_kv != self.codes.shape[1] or desc.n_pages != self.codes.shape[0]:
            raise ValueError("the bounds were made for another page table or another number of key heads")
        _require_dense(pages, "pages", torch.int32, (pages.numel(),), dev)
        if count is not None:
            _require_dense(count, "count", torch.int32, (1,), dev)
        if valid is not None:
            _require_dense(valid, "valid", torch.int32, (pages.numel(),), dev)
        if status is not None:
            _require_dense(status, "status", torch.int32, (1,), dev)
        with _on(dev):
            _native.page_bounds(desc, pages, count, valid, self.codes, self.exponents, status)


def select_pages(q: torch.Tensor, bounds: PageBounds, page_ids: torch.Tensor, lengths: torch.Tensor, budget: int, *,
                 sink: int = 1, recent: int = 1, tokens_per_page: int = 16, status: Optional[torch.Tensor] = None):
    """For each sequence and key head the positions of up to ``budget`` pages to attend, ascending.

    Always the first ``sink`` and the last ``recent`` pages; the others by the largest score of
    the key head's queries against the page's bounds (an upper bound of q . k with q rounded to
    int8; whole-number arithmetic, so the choice is exact; of equal scores the lower position).
    Returns ``selected`` int32 [n_seqs, heads_kv, budget], padded with -1, and the number of
    positions int32 [n_seqs, heads_kv]."""
    _require_query(q)
    n_seqs, heads_q, d = q.shape
    dev = q.device
    page_ids = _require_lists(page_ids, lengths, n_seqs, dev)
    heads_kv = bounds.codes.shape[1]
    if bounds.codes.device != dev:
        raise ValueError(f"the bounds are on {bounds.codes.device}, expected {dev}")
    if bounds.codes.shape[3] != d or heads_kv == 0 or heads_q % heads_kv:
        raise ValueError("q and the bounds differ in head_dim, or the query heads are no multiple of the key heads")
    if budget < 1 or sink < 0 or recent < 0 or sink + recent > budget or budget > _MOST:
        raise ValueError("budget must be at least 1, at least sink + recent (neither negative) and fit an int32")
    _require_tokens_per_page(tokens_per_page)
    if status is not None:
        _require_dense(status, "status", torch.int32, (1,), dev)
    selected, count = page_ids.new_empty(n_seqs, heads_kv, budget), page_ids.new_empty(n_seqs, heads_kv)
    if n_seqs:
        with _on(dev):
            scratch = torch.empty(_native.select_scratch_floats(n_seqs, heads_kv, page_ids.shape[1]),
                                  dtype=torch.float32, device=dev)
            _native.select_pages(q, bounds.codes, bounds.exponents, page_ids, lengths, tokens_per_page,
                                 budget, sink, recent, selected, count, scratch, status)
    return selected, count


class Eviction(NamedTuple):
    """What :func:`evict_pages` returns."""
    page_ids: torch.Tensor    # int32 [n_seqs, max_pages], the kept pages in order, then -1
    page_mass: torch.Tensor   # fp32 [n_seqs, max_pages], their mass, then 0
    lengths: torch.Tensor     # int32 [n_seqs], the tokens left
    evicted: torch.Tensor     # int32 [n_seqs, max_pages], the pages that left, then -1
    n_evicted: torch.Tensor   # int32 [n_seqs]


def evict_pages(page_mass: torch.Tensor, page_ids: torch.Tensor, lengths: torch.Tensor, budget: int, *,
                sink: int = 1, recent: int = 1, tokens_per_page: int = 16) -> Eviction:
    """Drop the pages of least accumulated attention from sequences of more than ``budget`` pages.

    ``page_mass`` is what :func:`decode_attention` keeps.  The first ``sink`` and the last
    ``recent`` (at least the page being filled) pages stay, and of the others those of greatest
    mass (of equal mass the lower position, NaN counts as the least).  A length beyond
    ``max_pages`` pages is cut there; a negative one is none.  The inputs are not changed; the pages that leave are listed, their slots and pool rows stay the caller's to
    give back (another sequence may share them)."""
    if page_ids.dim() != 2:
        raise ValueError("page_ids must be [n_seqs, max_pages]")
    n_seqs, width = page_ids.shape
    dev = page_ids.device
    page_ids = _require_lists(page_ids, lengths, n_seqs, dev)
    page_mass = _require_rows(page_mass, "page_mass", torch.float32, (n_seqs, width), dev)
    if recent < 1 or sink < 0 or sink + recent > budget or budget > _MOST:
        raise ValueError("recent must be at least 1, sink not negative, budget at least sink + recent and fit an int32")
    _require_tokens_per_page(tokens_per_page)
    ids = page_ids.new_empty  # (sizes as plain arguments: a tuple takes 0.4 us longer to parse)
    got = Eviction(ids(n_seqs, width), page_mass.new_empty(n_seqs, width), ids(n_seqs), ids(n_seqs, width), ids(n_seqs))
    if n_seqs:
        with _on(dev):
            _native.evict_pages(page_mass, page_ids, lengths, tokens_per_page, budget, sink,
                                recent, got.page_ids, got.page_mass, got.lengths, got.evicted, got.n_evicted)
    return got


__all__ = ["decode_attention", "prompt_attention", "PageBounds", "select_pages", "Eviction", "evict_pages"]
