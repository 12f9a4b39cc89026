"""Writing, reading and attending tiered pages, without a GPU: refused arguments at the C boundary,
and the sources' promises."""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

from test_paged_attention import X, desc

from ashkv import _native as N


def write(d, **change):
    a = dict(k=X, ks=256, kh=128, v=X, vs=256, vh=128, n=3, ids=X, ids_stride=4, pages=4, lengths=X, starts=X, seqs=1,
             status=None, stream=None)
    a.update(change)
    return N.lib().ashkv_write_kv(None if d is None else ctypes.addressof(d), *a.values())


def read(d, **change):
    a = dict(ids=X, ids_stride=4, pages=4, lengths=X, starts=X, seqs=1, n=3, k=X, v=X, status=None, stream=None)
    a.update(change)
    return N.lib().ashkv_read_kv(None if d is None else ctypes.addressof(d), *a.values())


def test_refusals():
    for call, name in ((write, b"ashkv_write_kv"), (read, b"ashkv_read_kv")):
        assert call(None) == N.BAD_ARGUMENT
        for bad in (dict(head_dim=12), dict(head_dim=0), dict(heads_kv=0), dict(tokens_per_page=0), dict(n_layers=0),
                    dict(n_pages=-1), dict(pool_tokens=-1), dict(row_stride=248), dict(d_tier=None), dict(d_layer_k=None),
                    dict(stores=None)):
            assert call(desc(**bad)) == N.BAD_ARGUMENT, bad
            assert name in N.lib().ashkv_last_error()
        for bad in (dict(n=-1), dict(n=2 ** 31), dict(seqs=-1), dict(pages=-1), dict(ids_stride=3), dict(ids=None),
                    dict(lengths=None), dict(starts=None), dict(k=None), dict(v=None),
                    dict(seqs=1 << 16, pages=1 << 16, ids_stride=1 << 16)):
            assert call(desc(), **bad) == N.BAD_ARGUMENT, bad
        assert call(desc(), n=0, k=None) == N.OK and call(desc(), seqs=0, lengths=None, starts=None) == N.OK
    assert write(desc(), k=ctypes.c_void_p(257)) == N.BAD_ARGUMENT
    assert read(desc(), v=ctypes.c_void_p(264)) == N.BAD_ARGUMENT


def test_store_refusals():
    def store(fmt, slot_bytes):
        return N.TierStoreDesc(256, slot_bytes, 4, fmt, 256, 256)

    none, pool = store(N.PAGE_NONE, 0), store(N.PAGE_BF16, 0)
    need = N.page_slot_bytes(N.PAGE_INT8, 16, 256)
    small, good = store(N.PAGE_INT8, need - 256), store(N.PAGE_INT8, 1 << 20)
    for call in (write, read):
        assert call(desc([pool, small, none, none, none, none])) == N.BAD_ARGUMENT
        assert call(desc([pool, good, none, none, none, none], head_dim=64, heads_kv=3, row_stride=192)) == N.BAD_ARGUMENT
        assert call(desc([pool, good, none, none, none, none]), n=0) == N.OK


def test_window_refusals():
    def decode(**change):
        a = dict(q=X, qs=1024, qh=128, n=1, hq=8, ids=X, ids_stride=4, pages=4, lengths=X, window=4, sinks=0, scale=1.0,
                 mass=None, mass_stride=0, decay=1.0, out=X, lse=None, scratch=X, status=None, stream=None)
        a.update(change)
        d = desc()
        return N.lib().ashkv_decode_attention_window(ctypes.addressof(d), *a.values())

    for bad in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(n=-1), dict(hq=7), dict(q=None), dict(mass=X, mass_stride=3)):
        assert decode(**bad) == N.BAD_ARGUMENT, bad
        assert b"ashkv_decode_attention_window" in N.lib().ashkv_last_error()
    assert decode(n=0, q=None) == N.OK


def test_prompt_refusals():
    def prompt(**change):
        a = dict(q=X, qs=1024, qh=128, n=3, hq=8, ids=X, ids_stride=4, pages=4, lengths=X, starts=X, seqs=1, window=0, sinks=0,
                 scale=1.0, out=X, lse=None, scratch=X, status=None, stream=None)
        kv = change.pop("kv", desc())
        a.update(change)
        return N.lib().ashkv_prompt_attention(None if kv is None else ctypes.addressof(kv), *a.values())

    assert prompt(kv=None) == N.BAD_ARGUMENT
    for bad in (dict(head_dim=32), dict(head_dim=96), dict(heads_kv=0), dict(tokens_per_page=0), dict(row_stride=248), dict(d_tier=None)):
        assert prompt(kv=desc(**bad)) == N.BAD_ARGUMENT, bad
    for bad in (dict(hq=0), dict(hq=7), dict(hq=16384), dict(n=-1), dict(n=2 ** 28), dict(seqs=-1), dict(pages=-1), dict(ids_stride=3),
                dict(window=-1), dict(sinks=-1, window=1), dict(sinks=1), dict(q=None), dict(out=None), dict(scratch=None),
                dict(q=ctypes.c_void_p(257)), dict(out=ctypes.c_void_p(264)), dict(scratch=ctypes.c_void_p(260)),
                dict(lengths=None), dict(starts=None), dict(ids=None)):
        assert prompt(**bad) == N.BAD_ARGUMENT, bad
        assert b"ashkv_prompt_attention" in N.lib().ashkv_last_error()
    assert prompt(n=0, q=None, out=None, scratch=None) == N.OK and prompt(seqs=0, lengths=None, starts=None) == N.OK


def test_prompt_scratch():
    size = N.lib().ashkv_prompt_scratch_floats
    for bad in ((-1, 1, 8, 2, 128, 1), (1, -1, 8, 2, 128, 1), (1, 1, 0, 2, 128, 1), (1, 1, 8, 0, 128, 1), (1, 1, 7, 2, 128, 1),
                (1, 1, 8, 2, 0, 1), (1, 1, 8, 2, 128, 0)):
        assert size(*bad) == -1, bad
    # a row of results in fp32 and its sum for each place that a cut item can have, of at most 256 rows
    assert 0 < size(1, 1, 8, 2, 128, 1) < 2 ** 20
    assert size(8192, 1, 32, 8, 128, 1) < 2 ** 25
    assert size(300, 1, 8, 2, 128, 1) < 2 ** 27
    for n in (1, 40, 8192, 1 << 20):  # more of anything needs no less within a rule of cutting
        assert size(n, 2, 8, 2, 128, 1) <= size(n, 2, 8, 2, 128, 9)


def test_kernels_over_page_lists_promise_nothing_of_what_they_read():
    """launch_paged overlaps a kernel with the one before it, as launch_overlapped does: the same rules."""
    csrc = Path(__file__).resolve().parent.parent / "ash-kv_b200" / "csrc"
    seen = []
    for f in sorted(csrc.glob("*.cu")) + [csrc / "paged_kv.cuh", csrc / "page_codec.cuh"]:
        code = re.sub(r"//[^\n]*", "", f.read_text())
        if f.suffix == ".cu" and "launch_paged(" not in code:
            continue
        seen.append(f.name)
        for word in ("__restrict__", "ld_nc", "__ldg", "ld.global.nc"):
            assert word not in code, f"{f.name}: {word}"
    assert {"cache.cu", "prompt.cu"} <= set(seen)
