"""The paged serving operators without a GPU: refused arguments at the C boundary, scratch sizes,
host tensors, and the oracle's own consistency."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import attention as O

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime.batch import DevicePageTable

X = ctypes.c_void_p(256)  # an aligned address that no refused call may touch


def desc(tiers=None, **change):
    store = (N.TierStoreDesc * 6)(*tiers) if tiers else A._StoreDescs.from_buffer_copy(A._NO_STORES)
    fields = dict(d_tier=256, d_layer_id=256, d_token_start=256, d_page_slot=256, n_pages=4, d_layer_k=256,
                  d_layer_v=256, pool_tokens=64, row_stride=256, n_layers=1, tokens_per_page=16, heads_kv=2,
                  head_dim=128, outlier_cap=0, stores=ctypes.addressof(store))
    d = N.PagedKVDesc(**{**fields, **change})
    d.keep = store
    return d


def decode(d, **change):
    a = dict(q=X, qs=1024, qh=128, n=1, hq=8, ids=X, ids_stride=4, pages=4, lengths=X, sel=None, cnt=None, width=0,
             scale=1.0, mass=None, mass_stride=0, decay=1.0, out=X, lse=None, scratch=X, status=None, stream=None)
    a.update(change)
    return N.lib().ashkv_decode_attention(None if d is None else ctypes.addressof(d), *a.values())


def test_decode_refusals():
    assert decode(None) == N.BAD_ARGUMENT
    for bad in (dict(head_dim=96), dict(heads_kv=0), dict(tokens_per_page=0), dict(n_layers=0), dict(n_pages=-1),
                dict(pool_tokens=-1), dict(row_stride=255), dict(row_stride=260), dict(d_tier=None),
                dict(d_layer_v=None), dict(outlier_cap=-1), dict(stores=None), dict(tokens_per_page=65536, row_stride=1 << 20)):
        assert decode(desc(**bad)) == N.BAD_ARGUMENT, bad
        assert b"ashkv_decode_attention" in N.lib().ashkv_last_error()
    for bad in (dict(n=-1), dict(pages=-1), dict(hq=7), dict(hq=0), dict(n=1 << 22, hq=8), dict(ids_stride=3),
                dict(q=None), dict(lengths=None), dict(out=None), dict(scratch=None), dict(scratch=ctypes.c_void_p(24)),
                dict(ids=None), dict(sel=X, width=4), dict(sel=X, cnt=X, width=4, mass=X, mass_stride=4),
                dict(mass=X, mass_stride=3), dict(n=1 << 16, pages=1 << 16, ids_stride=1 << 16)):
        assert decode(desc(), **bad) == N.BAD_ARGUMENT, bad
    assert decode(desc(), n=0, q=None, out=None) == N.OK


def test_decode_store_refusals():
    def store(fmt, slot_bytes, data=256, n=4):
        return N.TierStoreDesc(data, slot_bytes, n, fmt, 256, 256)

    none, pool = store(N.PAGE_NONE, 0), store(N.PAGE_BF16, 0)
    need = N.page_slot_bytes(N.PAGE_INT8, 16, 256)
    for s in (store(N.PAGE_INT8, need - 256), store(N.PAGE_INT8, need, data=264), store(N.PAGE_INT8, need + 8),
              store(N.PAGE_INT8, need, n=1 << 24), store(9, need)):
        assert decode(desc([pool, s, none, none, none, none])) == N.BAD_ARGUMENT
    assert decode(desc([none] * 6)) == N.BAD_ARGUMENT  # store 0 must be the pool
    good = store(N.PAGE_INT8, 1 << 20)
    # a page of 2 * 16 * 192 values, of 65536 * 2, and rows that are no power of two
    assert decode(desc([pool, good, none, none, none, none], head_dim=64, heads_kv=3, row_stride=192)) == N.BAD_ARGUMENT
    assert decode(desc([pool, good, none, none, none, none], tokens_per_page=256)) == N.BAD_ARGUMENT
    assert decode(desc([pool, good, none, none, none, none], n_pages=0), n=0) == N.OK


def test_bounds_select_evict_refusals():
    lib, d = N.lib(), desc()
    P = ctypes.addressof(d)
    assert lib.ashkv_page_bounds(None, X, None, 1, None, X, X, None, None) == N.BAD_ARGUMENT
    assert lib.ashkv_page_bounds(P, X, None, -1, None, X, X, None, None) == N.BAD_ARGUMENT
    assert lib.ashkv_page_bounds(P, None, None, 1, None, X, X, None, None) == N.BAD_ARGUMENT
    assert lib.ashkv_page_bounds(P, X, None, 1, None, ctypes.c_void_p(8), X, None, None) == N.BAD_ARGUMENT
    assert lib.ashkv_page_bounds(P, None, None, 0, None, None, None, None, None) == N.OK

    def select(**change):
        a = dict(q=X, qs=1024, qh=128, n=1, hq=8, hkv=2, dim=128, codes=X, exps=X, n_pages=4, ids=X, ids_stride=4,
                 pages=4, lengths=X, T=16, budget=3, sink=1, recent=1, sel=X, cnt=X, scratch=X, status=None, stream=None)
        a.update(change)
        return lib.ashkv_select_pages(*a.values())

    for bad in (dict(dim=32), dict(n=-1), dict(n=65536), dict(hq=7), dict(hkv=0), dict(T=0), dict(budget=0),
                dict(sink=2, recent=2), dict(sink=-1), dict(recent=-1), dict(q=None), dict(ids_stride=3), dict(codes=None),
                dict(codes=ctypes.c_void_p(8)), dict(scratch=None), dict(hq=2 * 129), dict(pages=-1)):
        assert select(**bad) == N.BAD_ARGUMENT, bad
    assert select(n=0, q=None) == N.OK

    def evict(**change):
        a = dict(mass=X, mass_stride=4, ids=X, ids_stride=4, lengths=X, n=1, pages=4, T=16, budget=3, sink=1, recent=1,
                 oi=X, om=X, ol=X, ev=X, ec=X, stream=None)
        a.update(change)
        return lib.ashkv_evict_pages(*a.values())

    for bad in (dict(n=-1), dict(pages=-1), dict(T=0), dict(recent=0), dict(sink=-1), dict(budget=1), dict(mass=None),
                dict(ol=None), dict(ids_stride=3), dict(mass_stride=3)):
        assert evict(**bad) == N.BAD_ARGUMENT, bad
    assert evict(n=0, lengths=None) == N.OK


def test_scratch_sizes():
    f = N.decode_scratch_floats
    assert f(1, 7, 2, 128, 4, False) == -1 and f(-1, 8, 2, 128, 4, False) == -1
    # a partial row per (range, sequence), its log-sum, first and last range per list
    few = f(2, 8, 2, 128, 3, False)  # at most one range per entry: 6
    assert few == (6 + 2) * 8 * 129 + 2 * 2 * 2
    assert f(2, 8, 2, 128, 3, True) == few + 2 * 3 * 8
    assert f(1, 8, 2, 128, 1 << 20, False) < 20_000_000  # bounded by what fills the GPU
    assert N.select_scratch_floats(3, 2, 10) == 60 and N.select_scratch_floats(-1, 2, 10) == -1


def test_host_tensors_are_refused():
    z = torch.zeros(4)
    i = torch.zeros(4, dtype=torch.int32)
    table = DevicePageTable(z, z, z, z, i.to(torch.int8), i, i, i, i)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        A.decode_attention(q, table, None, None, i.view(1, 4), i[:1])
    with pytest.raises(ValueError, match="CUDA"):
        A.PageBounds.empty(4, 1, 64, torch.device("cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        A.evict_pages(z.view(1, 4), i.view(1, 4), i[:1], 2)
    with pytest.raises(ValueError, match="CUDA"):
        A.select_pages(q, None, i.view(1, 4), i[:1], 2)


def test_oracle_bounds_hold_and_scores_are_upper_bounds():
    g = np.random.default_rng(0)
    K = g.standard_normal((16, 2, 64)) * np.exp2(g.integers(-20, 20, (1, 2, 1)).astype(np.float64))
    codes, exps = O.page_bounds(K, 16)
    unit = np.exp2(exps.astype(np.float64))[:, None]
    assert (codes[:, 0] * unit <= K.min(0)).all() and (codes[:, 1] * unit >= K.max(0)).all()
    assert np.abs(codes.astype(int)).max() <= 127 and (np.abs(codes.astype(int)).max(axis=(1, 2)) >= 63).all()
    q = np.rint(g.standard_normal((3, 64)) * 40)  # whole numbers: rounding the query changes nothing
    for h in range(2):
        score = O.page_scores(q, codes[None, h], exps[None, h])[0]
        assert score >= (K[:, h] @ q.T).max()


def test_oracle_keeps_by_score_then_position():
    s = np.array([5.0, 1.0, 3.0, 3.0, np.nan, 3.0, 0.0])
    assert O.keep_highest(s, 7, 0, 1) == list(range(7))
    assert O.keep_highest(s, 3, 0, 1) == [0, 2, 6]
    assert O.keep_highest(s, 5, 1, 1) == [0, 2, 3, 5, 6]
    assert O.keep_highest(s, 6, 1, 1) == [0, 1, 2, 3, 5, 6]
    assert O.keep_highest(s, 1, 0, 1) == [6]


def test_overlapped_kernels_promise_nothing_of_what_they_read():
    """A kernel launched by launch_overlapped is resident while its predecessor still writes: no
    pointer of its file is __restrict__ and no load takes the path of data that never changes."""
    csrc = Path(__file__).resolve().parent.parent / "ash-kv_b200" / "csrc"
    seen = 0
    for f in sorted(csrc.glob("*.cu")):
        code = re.sub(r"//[^\n]*", "", f.read_text())
        if "launch_overlapped(" not in code:
            continue
        seen += 1
        for word in ("__restrict__", "ld_nc", "__ldg", "ld.global.nc"):
            assert word not in code, f"{f.name}: {word}"
    assert seen == 2


def test_decode_refuses_lists_whose_positions_leave_an_int():
    most = 2 ** 31 - 1 - 2 ** 16
    for n, pages in ((1, 2 ** 31 - 1), (1, most + 1), (16, most // 16 + 1)):
        assert decode(desc(), n=n, pages=pages, ids_stride=pages) == N.BAD_ARGUMENT
        assert b"too many list entries" in N.lib().ashkv_last_error()
        assert decode(desc(), n=n, sel=X, cnt=X, width=pages) == N.BAD_ARGUMENT
        assert b"too many list entries" in N.lib().ashkv_last_error()


def test_layers_of_two_devices_are_refused():
    """The kernels follow every layer's address on the device of the first."""
    class Layer:
        dtype, shape, is_cuda = torch.bfloat16, torch.Size([32, 2, 64]), True

        def __init__(self, device):
            self.device = torch.device(device)

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 256

    from ashkv.runtime.batch import KVLayers
    for k, v in ((["cuda:0", "cuda:1"], ["cuda:0"] * 2), (["cuda:0"] * 2, ["cuda:0", "cuda:1"]), (["cuda:0"], ["cuda:1"])):
        with pytest.raises(ValueError, match="one device"):
            KVLayers([Layer(d) for d in k], [Layer(d) for d in v])
