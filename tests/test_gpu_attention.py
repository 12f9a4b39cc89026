"""GPU tests of the paged serving operators against float64.

Tolerances, from the arithmetic and not from runs.  With u = 2^-24:
  a score is an fp32 sum of dim exact products, scaled by a few factors:
      |ds| <= (dim + 16) * u * size,  size = max_t scale * sum_d |q_d k_d|, plus
      4 u |s| for the scale and 2^-22 of a weight for exp2; over INT8 and INT4 pages the
      queries are whole numbers off by at most 2^-22 of their largest value, 4 u * wide,
      wide = max_t scale * max|q| sum_d |k_d|;
  a weight is then off by a factor of at most 1 + dp, dp = 2 max|ds| + 2^-20;
  weights are rounded once before the product with V: 2^-11 (fp16) or, in two
      bf16 parts, 2^-16; the product accumulates in fp32 over the tokens;
  an fp16 weight below 2^-14 is a multiple of 2^-24, off by 2^-25; weights are
      scaled so that (largest row scale) * c >= 2^6 and codes are at most 2^7 - 1
      or 7 times their row scale's divisor, so that is at most 2^-31 of the largest
      |v| per token, against a sum of weights of at least 1;
  the result is rounded to bf16: 2^-8 of its value.
So |out - exact| <= 2^-8 |exact| + (2^-11 + 2 dp + n u) * sum_t P |v| + n 2^-31 max |v|.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from oracle import attention as O

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime.batch import DevicePageTable, KVLayers, TierStore

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CAP = 512
TIER = {N.PAGE_BF16: 0, N.PAGE_INT8: 1, N.PAGE_FP8: 1, N.PAGE_INT4: 2, N.PAGE_NBIT4: 2, N.PAGE_NBIT2: 3}


def bits(t: torch.Tensor) -> np.ndarray:
    return t.cpu().contiguous().view(torch.int16).numpy().view(np.uint16)


class Cache:
    """A page table over ``layers`` pool layers with each page in a random place of its format's tier."""

    def __init__(self, dev, formats, T, heads, dim, seed=0, layers=2, std=1.0, pool_bits=None):
        g = np.random.default_rng(seed)
        self.T, self.heads, self.dim, self.formats = T, heads, dim, list(formats)
        n, row = len(self.formats), heads * dim
        fill = torch.Generator().manual_seed(seed)
        pages = (torch.randn(n, 2 * T * row, generator=fill) * std)
        pages[:, ::701] *= 6.0
        self.bits = bits(pages.to(torch.bfloat16)) if pool_bits is None else pool_bits
        spots = g.permutation(layers * n)[:n]
        layer, start = spots % layers, spots // layers * T
        pool = np.zeros((2, layers, n * T, row), np.uint16)
        pool[:] = 0x7FC0  # NaN wherever no page of the BF16 tier lives
        tier, slot = np.zeros(n, np.int8), np.full(n, -1, np.int32)
        self.values, stores = [], {}
        for fmt in sorted(set(self.formats) - {N.PAGE_BF16}):
            stores[TIER[fmt]] = TierStore(fmt, n, dev, T, row, CAP if fmt in (N.PAGE_NBIT4, N.PAGE_NBIT2) else 0)
        slots = {t: np.full((n, s.slot_bytes), 0xFF, np.uint8) for t, s in stores.items()}
        free = {t: list(g.permutation(n)) for t in stores}
        for i, fmt in enumerate(self.formats):
            x = self.bits[i]
            if fmt == N.PAGE_BF16:
                pool[0, layer[i], start[i]:start[i] + T] = x[:T * row].reshape(T, row)
                pool[1, layer[i], start[i]:start[i] + T] = x[T * row:].reshape(T, row)
                self.values.append(O.page_values(fmt, x, T, heads, dim))
                continue
            data, _, n_out = oracle.page_encode(fmt, x, T, row, page_id=i, outlier_cap=CAP)
            assert n_out <= CAP
            tier[i], slot[i] = TIER[fmt], free[TIER[fmt]].pop()
            slots[TIER[fmt]][slot[i], :len(data)] = data
            self.values.append(O.page_values(fmt, data, T, heads, dim, CAP))
        for t, s in stores.items():
            s.data[:n * s.slot_bytes].copy_(torch.from_numpy(slots[t].reshape(-1)))
        up = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
        z = torch.zeros(n, device=dev)
        self.table = DevicePageTable(z, z, z, z, up(tier), up(np.zeros(n, np.int32)), up(layer.astype(np.int32)),
                                     up(start.astype(np.int32)), up(slot))
        tens = [[up(pool[i, l].view(np.int16)).view(torch.bfloat16).view(n * T, heads, dim) for l in range(layers)]
                for i in range(2)]
        self.kv = KVLayers(tens[0], tens[1])
        self.stores = stores

    def lists(self, page_ids, lengths):
        T = self.T
        return [[[(j, self.values[page_ids[b][j]]) for j in range(-(-int(lengths[b]) // T))]] * self.heads
                for b in range(len(lengths))]


def queries(n, hq, dim, seed, std=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(n, hq, dim, generator=g) * std).to(torch.bfloat16)


def check(got, lse, want, dim, n_tokens, mass=None, acc=None, decay=1.0):
    out = got.double().cpu().numpy()
    ds = (dim + 20) * U * want["size"] + 4 * U * want["wide"]
    dp = 2 * ds + 2.0 ** -20
    tol = 2.0 ** -8 * np.abs(want["out"]) + (2.0 ** -11 + 2 * dp + n_tokens * U)[..., None] * want["reach"]
    tol = tol + n_tokens * 2.0 ** -31 * want["largest"][..., None] + 1e-37
    assert np.isfinite(out).all()
    worst = np.max(np.abs(out - want["out"]) / tol) if out.size else 0.0
    assert worst <= 1.0, f"result off by {worst} of its tolerance"
    l = lse.double().cpu().numpy()
    none = np.isneginf(want["lse"])
    assert (np.isneginf(l) == none).all()
    t = (ds + 2.0 ** -19 + 8 * U * np.abs(want["lse"], where=~none, out=np.zeros_like(l)))[~none]
    assert (np.abs(l[~none] - want["lse"][~none]) <= t).all()
    if mass is not None:
        m = mass.double().cpu().numpy()
        drawn = want["mass"] - np.where(want["mass"] != acc, decay * acc, want["mass"])
        tm = (2 * dp.max() + 2.0 ** -19 + n_tokens * U) * np.abs(drawn) + 8 * U * (np.abs(acc) + np.abs(want["mass"]))
        assert (np.abs(m - want["mass"]) <= tm).all(), np.max(np.abs(m - want["mass"]) / (tm + 1e-300))


FORMATS = {"bf16": [N.PAGE_BF16], "int8": [N.PAGE_INT8], "fp8": [N.PAGE_FP8], "int4": [N.PAGE_INT4],
           "nbit4": [N.PAGE_NBIT4], "nbit2": [N.PAGE_NBIT2],
           "mixed": [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT2],
           "mixed8": [N.PAGE_FP8, N.PAGE_NBIT4, N.PAGE_BF16, N.PAGE_NBIT2]}


def run_case(dev, tiers, T, heads_q, heads, dim, lengths, seed, with_mass=True, decay=0.75, std=1.0):
    P = max(1, max(-(-x // T) for x in lengths))
    n = len(lengths) * P
    g = np.random.default_rng(seed)
    kinds = FORMATS[tiers]
    c = Cache(dev, [kinds[i] for i in g.integers(0, len(kinds), n)], T, heads, dim, seed, std=std)
    ids = g.permutation(n).astype(np.int32).reshape(len(lengths), P)
    q = queries(len(lengths), heads_q, dim, seed, 2.0)
    acc = g.random((len(lengths), P), dtype=np.float32)
    mass = torch.from_numpy(acc.copy()).to(dev) if with_mass else None
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    L = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = A.decode_attention(q.to(dev), c.table, c.kv, c.stores, torch.from_numpy(ids).to(dev), L,
                                  tokens_per_page=T, page_mass=mass, decay=decay, return_lse=True, status=status)
    want = O.decode_attention(q.double().numpy(), c.lists(ids, lengths), lengths, T, dim ** -0.5, acc, decay)
    assert int(status) == 0
    check(out, lse, want, dim, max(lengths) + 1, mass, acc, decay)
    return c, ids, q, out, lse, mass


@pytest.mark.parametrize("tiers", list(FORMATS))
@pytest.mark.parametrize("heads_q,heads,dim", [(8, 2, 128), (3, 1, 128), (4, 4, 64), (16, 2, 64)])
def test_decode_formats(cuda, tiers, heads_q, heads, dim):
    run_case(cuda, tiers, 16, heads_q, heads, dim, [70, 0, 1, 16, 33, 257], 1)


@pytest.mark.parametrize("tiers", ["bf16", "mixed", "int4"])
@pytest.mark.parametrize("heads_q,heads", [(8, 8), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 2)])
def test_decode_head_layouts(cuda, tiers, heads_q, heads):
    run_case(cuda, tiers, 16, heads_q, heads, 128, [50, 131], 2)


@pytest.mark.parametrize("T,tiers", [(1, "bf16"), (5, "bf16"), (7, "bf16"), (24, "bf16"), (8, "mixed"), (12, "int8"),
                                     (20, "int4"), (32, "mixed8"), (40, "mixed"), (64, "int8")])
def test_decode_page_sizes(cuda, T, tiers):
    run_case(cuda, tiers, T, 4, 2, 128, [1, T, T + 1, 3 * T - 1, 150], 3)


@pytest.mark.parametrize("tiers", ["bf16", "int8", "int4"])
def test_decode_many_sequences_and_one_long(cuda, tiers):
    run_case(cuda, tiers, 16, 4, 2, 64, [(37 * i) % 90 for i in range(150)], 4)
    run_case(cuda, tiers, 16, 4, 2, 64, [4001], 5)


@pytest.mark.parametrize("T,lengths", [(1000, [2001, 999, 1]), (65536, [65541])])
def test_decode_very_large_pages(cuda, T, lengths):
    run_case(cuda, "bf16", T, 2, 1, 64, lengths, 84)


def test_decode_one_long_sequence_among_short_ones(cuda):
    """One row of many partial results beside rows of one or two."""
    T, heads, dim, n = 16, 8, 64, 41
    c = Cache(cuda, [N.PAGE_BF16] * 375, T, heads, dim, 83)
    lengths = [(7 * i) % 40 for i in range(n)]
    lengths[13] = 375 * T - 3
    ids = np.stack([np.random.default_rng(b).permutation(375) for b in range(n)]).astype(np.int32)
    q, acc = queries(n, 16, dim, 83), np.zeros((n, 375))
    mass = torch.zeros(n, 375, device=cuda)
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, None, torch.from_numpy(ids).to(cuda),
                                  torch.tensor(lengths, dtype=torch.int32, device=cuda), page_mass=mass, return_lse=True)
    want = O.decode_attention(q.double().numpy(), c.lists(ids, lengths), lengths, T, dim ** -0.5, acc, 1.0)
    check(out, lse, want, dim, max(lengths), mass, acc, 1.0)


@pytest.mark.parametrize("tiers", ["bf16", "int8", "mixed"])
@pytest.mark.parametrize("std", [1e-3, 30.0])
def test_decode_value_ranges(cuda, tiers, std):
    """Small values, and scores in the hundreds (one token takes the whole row)."""
    run_case(cuda, tiers, 16, 4, 2, 128, [100, 17], 6, std=std)


@pytest.mark.parametrize("tiers", list(FORMATS))
def test_decode_query_extremes(cuda, tiers):
    """Largest significands (1.1111111b), negative ones, powers of two, a lone large channel, zeros."""
    T, heads, dim = 16, 1, 128
    c = Cache(cuda, [FORMATS[tiers][i % len(FORMATS[tiers])] for i in range(8)], T, heads, dim, 21)
    ids = np.arange(8, dtype=np.int32).reshape(1, 8)
    q = queries(1, 8, dim, 21)
    q[0, 0, :7] = 255 / 128
    q[0, 1, :7] = -255 / 128
    q[0, 2, 5] = 255 / 128 * 4
    q[0, 3, 9] = 255 / 128 * 64
    q[0, 4, 9] = -512.0
    q[0, 5] = 0.0
    q[0, 6] = torch.where(torch.arange(dim) % 2 == 0, 255 / 128, -255 / 128)
    q[0, 7] *= 2.0 ** -120
    L = torch.tensor([120], dtype=torch.int32, device=cuda)
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda), L, scale=0.05,
                                  return_lse=True)
    want = O.decode_attention(q.double().numpy(), c.lists(ids, [120]), [120], T, 0.05)
    check(out, lse, want, dim, 120)


@pytest.mark.parametrize("kinds,sizes", [
    ([N.PAGE_INT4, N.PAGE_BF16, N.PAGE_INT4], [1e-7, 1e15, 1.0]), ([N.PAGE_BF16, N.PAGE_INT4, N.PAGE_BF16], [1.0, 1e-7, 1e12]),
    ([N.PAGE_INT4] * 3, [3e35, 1e-7, 1e35]), ([N.PAGE_INT4, N.PAGE_FP8, N.PAGE_FP8], [1e-7, 1e2, 1.0]),
    ([N.PAGE_INT8, N.PAGE_NBIT4], [1e-7, 1e15])])
def test_decode_values_of_far_apart_sizes(cuda, kinds, sizes):
    """Rows whose scales differ by many powers of two, the smallest first: no sum overflows."""
    T, heads, dim = 16, 2, 128
    g = torch.Generator().manual_seed(81)
    pages = torch.randn(len(kinds), 2, T * heads * dim, generator=g)
    pages[:, 1] *= torch.tensor(sizes)[:, None]
    c = Cache(cuda, kinds, T, heads, dim, 81, pool_bits=bits(pages.reshape(len(kinds), -1).to(torch.bfloat16)))
    ids, lengths = np.arange(len(kinds), dtype=np.int32)[None], [len(kinds) * T - 3]
    q = queries(1, 8, dim, 81)
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda),
                                  torch.tensor(lengths, dtype=torch.int32, device=cuda), return_lse=True)
    want = O.decode_attention(q.double().numpy(), c.lists(ids, lengths), lengths, T, dim ** -0.5)
    check(out, lse, want, dim, lengths[0])


def test_decode_no_tokens_and_no_sequences(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 4, 16, 2, 64)
    ids = torch.arange(4, dtype=torch.int32, device=cuda).view(2, 2)
    q = queries(2, 4, 64, 0).to(cuda)
    zero = torch.zeros(2, dtype=torch.int32, device=cuda)
    mass = torch.ones(2, 2, device=cuda)
    out, lse = A.decode_attention(q, c.table, c.kv, None, ids, zero, page_mass=mass, decay=0.5, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all() and (mass == 1).all()
    out, lse = A.decode_attention(q, c.table, c.kv, None, ids[:, :0], zero, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    assert A.decode_attention(q[:0], c.table, c.kv, None, ids[:0], zero[:0]).shape == (0, 4, 64)


@pytest.mark.parametrize("fmt", [N.PAGE_BF16, N.PAGE_FP8, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT2])
def test_tokens_past_the_length_do_not_count(cuda, fmt):
    """A page that ends inside its last tile may hold anything behind its last token."""
    T, heads, dim, length = 16, 2, 128, 21
    a = Cache(cuda, [fmt, fmt], T, heads, dim, 7)
    page = np.concatenate([a.bits[1].reshape(2, T, -1)], 0).copy()
    ids = torch.arange(2, dtype=torch.int32, device=cuda).view(1, 2)
    L = torch.tensor([length], dtype=torch.int32, device=cuda)
    q = queries(1, 8, dim, 7).to(cuda)
    ref = A.decode_attention(q, a.table, a.kv, a.stores, ids, L)
    if fmt == N.PAGE_BF16:
        l, s = int(a.table.layer[1]), int(a.table.token_start[1])
        for t, junk in enumerate((float("nan"), float("inf"), -float("inf"), 3e38)):
            for x in (a.kv.k[l], a.kv.v[l]):
                x[s + length - T + t::T][:1] = junk
                x[s + length - T + 4:s + T] = float("nan")
    else:
        st = a.stores[TIER[fmt]]
        slot = st.slot_view()[int(a.table.slot[1])]
        row = heads * dim
        if fmt == N.PAGE_INT8:  # scales and codes of the unused rows
            for r in list(range(5, T)) + list(range(T + 5, 2 * T)):
                slot[2 * r:2 * r + 2] = torch.tensor([0xFF, 0x7F], dtype=torch.uint8)
        elif fmt == N.PAGE_FP8:
            for r in list(range(5, T)) + list(range(T + 5, 2 * T)):
                slot[r * row:(r + 1) * row] = 0x7F
        elif fmt == N.PAGE_INT4:
            for r in list(range(5, T)) + list(range(T + 5, 2 * T)):
                slot[r * row // 32:(r + 1) * row // 32] = 0xFF
        else:
            for r in list(range(5, T)) + list(range(T + 5, 2 * T)):
                slot[16 + r * row // 16:16 + (r + 1) * row // 16] = 0xFF
    got = A.decode_attention(q, a.table, a.kv, a.stores, ids, L)
    assert torch.isfinite(got).all() and torch.equal(got, ref)
    assert page.size


def test_decode_nan_and_inf_in_use_come_through(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 2, 16, 1, 64, 8)
    ids = torch.arange(2, dtype=torch.int32, device=cuda).view(1, 2)
    L = torch.tensor([32], dtype=torch.int32, device=cuda)
    q = queries(1, 2, 64, 8).to(cuda)
    l, s = int(c.table.layer[0]), int(c.table.token_start[0])
    c.kv.v[l][s + 3, 0, 5] = float("nan")
    out = A.decode_attention(q, c.table, c.kv, None, ids, L)
    assert torch.isnan(out[..., 5]).all() and torch.isfinite(out[..., :5]).all()
    c.kv.k[l][s + 3, 0, 5] = float("nan")
    out, lse = A.decode_attention(q, c.table, c.kv, None, ids, L, return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()


def test_all_scores_minus_infinity(cuda):
    c = Cache(cuda, [N.PAGE_BF16], 16, 1, 64, 9)
    l, s = int(c.table.layer[0]), int(c.table.token_start[0])
    c.kv.k[l][s:s + 16] = -float("inf")
    out, lse = A.decode_attention(torch.ones(1, 1, 64, dtype=torch.bfloat16, device=cuda), c.table, c.kv, None,
                                  torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                                  torch.tensor([16], dtype=torch.int32, device=cuda), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_decode_strides_shared_pages_and_out(cuda):
    """A query cut out of a fused projection, a block table with spare columns, one page in two rows."""
    T, heads, dim = 16, 2, 128
    c = Cache(cuda, [N.PAGE_INT8, N.PAGE_BF16, N.PAGE_INT8, N.PAGE_BF16], T, heads, dim, 10)
    ids = torch.full((3, 9), 77, dtype=torch.int32, device=cuda)
    ids[:, :3] = torch.tensor([[0, 1, 2], [0, 1, 3], [0, 0, 1]], dtype=torch.int32)
    L = torch.tensor([40, 48, 33], dtype=torch.int32, device=cuda)
    fused = torch.randn(3, 12 * dim + 6, device=cuda).bfloat16()
    q = fused[:, 3:3 + 8 * dim].unflatten(1, (8, dim))
    mass = torch.zeros(3, 11, device=cuda)
    out = torch.full((3, 8, dim), 7.0, dtype=torch.bfloat16, device=cuda)
    back, lse = A.decode_attention(q, c.table, c.kv, c.stores, ids[:, :3], L, page_mass=mass[:, 4:7], out=out,
                                   return_lse=True)
    assert back is out and (mass[:, :4] == 0).all() and (mass[:, 7:] == 0).all()
    want = O.decode_attention(q.double().cpu().numpy(), c.lists(ids.cpu().numpy(), L.cpu().numpy()), L.cpu().numpy(),
                              T, dim ** -0.5, np.zeros((3, 3)), 1.0)
    check(out, lse, want, dim, 49, mass[:, 4:7].contiguous(), np.zeros((3, 3)))
    over = q.contiguous()  # the result in place of the query
    assert torch.equal(A.decode_attention(over, c.table, c.kv, c.stores, ids[:, :3], L, out=over), out)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    assert torch.equal(A.decode_attention(swapped, c.table, c.kv, c.stores, ids[:, :3], L), out)


def test_decode_bad_pages_are_left_out_and_flagged(cuda):
    T, heads, dim = 16, 2, 64
    fmts = [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_BF16, N.PAGE_INT8, N.PAGE_BF16, N.PAGE_BF16]
    c = Cache(cuda, fmts, T, heads, dim, 11)
    q = queries(1, 4, dim, 11).to(cuda)
    full = torch.tensor([6 * T], dtype=torch.int32, device=cuda)
    ids = torch.arange(6, dtype=torch.int32, device=cuda).view(1, 6)
    good = {name: getattr(c.table, name).clone() for name in ("tier", "slot", "layer", "token_start")}

    def status_of(ids_, L):
        st = torch.zeros(1, dtype=torch.int32, device=cuda)
        out, lse = A.decode_attention(q, c.table, c.kv, c.stores, ids_, L, return_lse=True, status=st)
        return out, lse, int(st)

    without = O.decode_attention(q.double().cpu().numpy(), [[[(j, c.values[j]) for j in (0, 2, 3, 4, 5)]] * heads],
                                 [6 * T], T, dim ** -0.5)
    for name, value in (("tier", 3), ("tier", -1), ("tier", 6), ("slot", -1), ("slot", 6)):
        getattr(c.table, name)[1] = value
        out, lse, st = status_of(ids, full)
        assert st == N.FLAG_INDEX_RANGE, name
        check(out, lse, without, dim, 6 * T)
        getattr(c.table, name).copy_(good[name])
    without = O.decode_attention(q.double().cpu().numpy(), [[[(j, c.values[j]) for j in (0, 1, 3, 4, 5)]] * heads],
                                 [6 * T], T, dim ** -0.5)
    for name, value in (("layer", -1), ("layer", 2), ("token_start", -1), ("token_start", 6 * T - T + 1)):
        getattr(c.table, name)[2] = value
        out, lse, st = status_of(ids, full)
        assert st == N.FLAG_INDEX_RANGE, name
        check(out, lse, without, dim, 6 * T)
        getattr(c.table, name).copy_(good[name])
    for bad in (-1, 6, 2 ** 31 - 1):
        ids2 = ids.clone()
        ids2[0, 2] = bad
        out, lse, st = status_of(ids2, full)
        assert st == N.FLAG_INDEX_RANGE
        check(out, lse, without, dim, 6 * T)
    # a length beyond the list is cut there, a negative one is none
    ref = status_of(ids, full)
    out, lse, st = status_of(ids, full + 5)
    assert st == N.FLAG_INDEX_RANGE and torch.equal(out, ref[0]) and torch.equal(lse, ref[1])
    out, lse, st = status_of(ids, torch.full_like(full, -3))
    assert st == N.FLAG_INDEX_RANGE and (out == 0).all()


def test_decode_offsets_beyond_32_bits(cuda):
    """Pool rows and slots that lie more than 2^32 bytes from their base."""
    T, heads, dim = 16, 8, 128
    tokens = (1 << 32) // (heads * dim * 2) + 4 * T
    k = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=cuda)
    v = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=cuda)
    far = tokens - T
    g = torch.Generator().manual_seed(12)
    kp, vp = (torch.randn(T, heads, dim, generator=g).bfloat16() for _ in range(2))
    k[far:], v[far:] = kp.to(cuda), vp.to(cuda)
    row = heads * dim
    n_slots = (1 << 32) // N.page_slot_bytes(N.PAGE_INT8, T, row) + 3
    store = TierStore(N.PAGE_INT8, n_slots, cuda, T, row)
    page = bits((torch.randn(2 * T * row, generator=g)).bfloat16())
    data = oracle.page_encode(N.PAGE_INT8, page, T, row)[0]
    store.slot_view()[n_slots - 1, :len(data)] = torch.from_numpy(data).to(cuda)
    z, i32 = torch.zeros(2, device=cuda), lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    table = DevicePageTable(z, z, z, z, torch.tensor([0, 1], dtype=torch.int8, device=cuda), i32(0, 0), i32(0, 0),
                            i32(far, 0), i32(-1, n_slots - 1))
    q = queries(1, 16, dim, 12)
    out, lse = A.decode_attention(q.to(cuda), table, KVLayers([k], [v]), {1: store}, i32(0, 1).view(1, 2), i32(30),
                                  return_lse=True)
    vals = [(kp.double().numpy(), vp.double().numpy()), O.page_values(N.PAGE_INT8, data, T, heads, dim)]
    want = O.decode_attention(q.double().numpy(), [[list(enumerate(vals))] * heads], [30], T, dim ** -0.5)
    check(out, lse, want, dim, 30)
    bounds = A.PageBounds.empty(2, heads, dim, cuda)
    bounds.update(table, KVLayers([k], [v]), i32(0))
    codes, exps = O.page_bounds(vals[0][0], T)
    assert np.array_equal(bounds.codes[0].cpu().numpy(), codes) and np.array_equal(bounds.exponents[0].cpu().numpy(), exps)


def test_decode_streams_and_graphs(cuda):
    """The same call on two side streams at once, and two captured graphs replayed together."""
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT2] * 8, 16, 2, 128, 13)
    ids = torch.randperm(32, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 16).to(cuda)
    L = torch.tensor([250, 101], dtype=torch.int32, device=cuda)
    qs = [queries(2, 8, 128, 20 + i).to(cuda) for i in range(2)]
    want = [A.decode_attention(q, c.table, c.kv, c.stores, ids, L) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = []
    for q, s in zip(qs, streams):
        with torch.cuda.stream(s):
            got.append(A.decode_attention(q, c.table, c.kv, c.stores, ids, L))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs, ins, masses = [], [], [], []
    for q in qs:
        ins.append(q.clone())
        masses.append(torch.zeros(2, 16, device=cuda))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(A.decode_attention(ins[-1], c.table, c.kv, c.stores, ids, L, page_mass=masses[-1], decay=0.5))
        graphs.append(g)
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # three replays of decay 0.5: 1 + 1/2 + 1/4 of a step's mass
    once = torch.zeros(2, 16, device=cuda)
    A.decode_attention(qs[0], c.table, c.kv, c.stores, ids, L, page_mass=once, decay=0.5)
    assert torch.allclose(masses[0], 1.75 * once, rtol=8 * 2.0 ** -23)
    ins[0].copy_(qs[1])  # a graph reads its inputs anew
    L.fill_(60)
    graphs[0].replay()
    assert torch.equal(outs[0], A.decode_attention(qs[1], c.table, c.kv, c.stores, ids, L))


def test_captured_fork_of_the_operators(cuda):
    """Bounds on one stream of a capture and attention with its eviction on another, then a selection after both."""
    T, heads, dim, P = 16, 2, 128, 12
    c = Cache(cuda, [N.PAGE_BF16] * (2 * P), T, heads, dim, 82)
    ids = torch.randperm(2 * P, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(2, P).to(cuda)
    L = torch.tensor([P * T, 100], dtype=torch.int32, device=cuda)
    q = queries(2, 8, dim, 82).to(cuda)
    mass, bounds = torch.zeros(2, P, device=cuda), A.PageBounds.empty(2 * P, heads, dim, cuda)
    pages = ids.view(-1)

    def step(side):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            bounds.update(c.table, c.kv, pages)
        out = A.decode_attention(q, c.table, c.kv, None, ids, L, page_mass=mass)
        kept = A.evict_pages(mass, ids, L, 6)
        main.wait_stream(side)
        sel, cnt = A.select_pages(q, bounds, ids, L, 4)
        part = A.decode_attention(q, c.table, c.kv, None, ids, L, selected=sel, selected_count=cnt)
        return [out, *kept, sel, cnt, part]

    side = torch.cuda.Stream()
    want = [t.clone() for t in step(side)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(side)
    for _ in range(3):
        mass.zero_()
        bounds.codes.zero_(), bounds.exponents.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ----------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("heads,dim,T", [(2, 128, 16), (8, 64, 16), (1, 128, 5), (3, 64, 40)])
def test_page_bounds(cuda, heads, dim, T):
    n = 12
    c = Cache(cuda, [N.PAGE_BF16] * n, T, heads, dim, 30, layers=2)
    special = [0.0, -0.0, float("inf"), -float("inf"), float("nan"), 1e-38, -1e-38, 3e38, 127.0, 127.5, 2.0 ** -130]
    g = np.random.default_rng(3)
    for i in range(n // 2):  # half of the pages get special values
        l, s = int(c.table.layer[i]), int(c.table.token_start[i])
        for x in special:
            c.kv.k[l][s + int(g.integers(T)), int(g.integers(heads)), int(g.integers(dim))] = x
    l, s = int(c.table.layer[0]), int(c.table.token_start[0])
    c.kv.k[l][s:s + T, 0] = 0.0
    c.kv.k[l][s:s + T, 0, 3] = float("nan")
    b = A.PageBounds.empty(n, heads, dim, cuda)
    b.codes.fill_(55), b.exponents.fill_(9)
    pages = torch.tensor([0, 1, 2, 3, 7, 8, 9], dtype=torch.int32, device=cuda)
    valid = [T, T - 1, 1, 0, T, max(1, T // 2), T + 9]
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    b.update(c.table, c.kv, pages, valid=torch.tensor(valid, dtype=torch.int32, device=cuda), tokens_per_page=T,
             status=status)
    assert int(status) == 0
    listed = dict(zip(pages.tolist(), valid))
    for p in range(n):
        if p not in listed:
            assert (b.codes[p] == 55).all() and (b.exponents[p] == 9).all()
            continue
        l, s = int(c.table.layer[p]), int(c.table.token_start[p])
        codes, exps = O.page_bounds(c.kv.k[l][s:s + T].double().cpu().numpy(), min(listed[p], T))
        assert np.array_equal(b.exponents[p].cpu().numpy(), exps), p
        assert np.array_equal(b.codes[p].cpu().numpy(), codes), p


def test_page_bounds_count_and_bad_pages(cuda):
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_BF16, N.PAGE_BF16], 16, 2, 64, 31)
    b = A.PageBounds.empty(4, 2, 64, cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    pages = torch.tensor([0, 2, 3], dtype=torch.int32, device=cuda)
    b.update(c.table, c.kv, pages, count=torch.tensor([2], dtype=torch.int32, device=cuda), status=status)
    assert int(status) == 0 and (b.codes[3] == 0).all() and (b.codes[2] != 0).any()
    was = b.codes.clone()
    for bad in (1, -1, 4):  # a compressed page, ids outside the table
        status.zero_()
        b.update(c.table, c.kv, torch.tensor([bad], dtype=torch.int32, device=cuda), status=status)
        assert int(status) == N.FLAG_INDEX_RANGE and torch.equal(b.codes, was)
    c.table.token_start[3] = 4 * 16 - 15
    status.zero_()
    b.update(c.table, c.kv, pages, status=status)
    assert int(status) == N.FLAG_INDEX_RANGE and torch.equal(b.codes, was)
    b.update(c.table, c.kv, pages[:0])


# ----------------------------------------------------------------------------- selection
def select_want(q, b, ids, lengths, T, budget, sink, recent):
    codes, exps = b.codes.cpu().numpy(), b.exponents.cpu().numpy()
    group = q.shape[1] // codes.shape[1]
    want = []
    for i in range(len(lengths)):
        row = []
        for h in range(codes.shape[1]):
            pages = ids[i][:max(0, -(-int(lengths[i]) // T))]
            score = O.page_scores(q[i, h * group:(h + 1) * group].double().numpy(), codes[pages, h], exps[pages, h])
            row.append(O.keep_highest(score, budget, sink, recent))
        want.append(row)
    return want


def check_selected(sel, cnt, want):
    sel, cnt = sel.cpu().numpy(), cnt.cpu().numpy()
    for i, row in enumerate(want):
        for h, keep in enumerate(row):
            assert cnt[i, h] == len(keep)
            assert sel[i, h, :len(keep)].tolist() == keep, (i, h)
            assert (sel[i, h, len(keep):] == -1).all()


@pytest.mark.parametrize("heads_q,heads,dim", [(8, 2, 128), (4, 4, 64), (6, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 0), (3, 1, 2), (10, 0, 1), (40, 4, 4), (500, 1, 1)])
def test_select_pages(cuda, heads_q, heads, dim, budget, sink, recent):
    T, lengths = 16, [0, 1, 16, 900, 2000, 305]
    P = 130
    g = torch.Generator().manual_seed(40)
    n = P * 3
    b = A.PageBounds.empty(n, heads, dim, cuda)
    lo = torch.randint(-127, 60, (n, heads, dim), generator=g)
    hi = (lo + torch.randint(0, 60, (n, heads, dim), generator=g)).clamp_max(127)
    b.codes.copy_(torch.stack((lo, hi), 2).to(torch.int8))
    b.exponents.copy_(torch.randint(-3, 3, (n, heads), generator=g).to(torch.int8))
    ids = torch.randint(0, n, (len(lengths), P + 5), generator=g).to(torch.int32)  # pages repeat: ties
    q = queries(len(lengths), heads_q, dim, 41)
    q[3, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e-38])
    q[4] = 0.0  # every score alike
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    sel, cnt = A.select_pages(q.to(cuda), b, ids.to(cuda)[:, :P], torch.tensor(lengths, dtype=torch.int32, device=cuda),
                              budget, sink=sink, recent=recent, tokens_per_page=T, status=status)
    assert int(status) == 0
    check_selected(sel, cnt, select_want(q, b, ids[:, :P].numpy(), lengths, T, budget, sink, recent))


def test_select_long_row_and_bad_ids(cuda):
    T, n = 16, 5000
    g = torch.Generator().manual_seed(42)
    b = A.PageBounds.empty(n, 1, 64, cuda)
    b.codes.copy_(torch.randint(-127, 128, b.codes.shape, generator=g).sort(2).values.to(torch.int8))  # lo <= hi
    ids = torch.randperm(n, generator=g).to(torch.int32).view(1, n)
    q = queries(1, 2, 64, 43)
    L = torch.tensor([n * T - 3], dtype=torch.int32, device=cuda)
    sel, cnt = A.select_pages(q.to(cuda), b, ids.to(cuda), L, 700, sink=2, recent=3)
    check_selected(sel, cnt, select_want(q, b, ids.numpy(), [n * T - 3], T, 700, 2, 3))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    bad = ids.clone()
    bad[0, 100] = -5
    bad[0, 200] = n
    sel, cnt = A.select_pages(q.to(cuda), b, bad.to(cuda), L, n - 2, sink=0, recent=0, status=status)
    assert int(status) == N.FLAG_INDEX_RANGE and int(cnt) == n - 2
    assert not ({100, 200} & set(sel[0, 0].tolist()))  # the two that do not exist come last
    status.zero_()
    A.select_pages(q.to(cuda), b, ids.to(cuda), L + 100, 5, status=status)
    assert int(status) == N.FLAG_INDEX_RANGE


def test_selected_attention(cuda):
    """Each key head attends its own pages; padding, wrong positions and an empty list."""
    T, heads, dim, P = 16, 2, 128, 12
    kinds = [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT2]
    c = Cache(cuda, [kinds[i % 4] for i in range(2 * P)], T, heads, dim, 44)
    ids = np.random.default_rng(5).permutation(2 * P).astype(np.int32).reshape(2, P)
    lengths = [P * T - 7, 100]
    q = queries(2, 8, dim, 44)
    sel = torch.full((2, heads, 6), -1, dtype=torch.int32)
    rows = {(0, 0): [0, 3, 11], (0, 1): [1, 2, 5, 7, 8, 11], (1, 0): [], (1, 1): [6]}
    cnt = torch.zeros(2, heads, dtype=torch.int32)
    for (b, h), r in rows.items():
        sel[b, h, :len(r)] = torch.tensor(r, dtype=torch.int32)
        cnt[b, h] = len(r)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    args = (q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda),
            torch.tensor(lengths, dtype=torch.int32, device=cuda))
    out, lse = A.decode_attention(*args, selected=sel.to(cuda), selected_count=cnt.to(cuda), return_lse=True,
                                  status=status)
    lists = [[[(j, c.values[ids[b, j]]) for j in rows[b, h]] for h in range(heads)] for b in range(2)]
    want = O.decode_attention(q.double().numpy(), lists, lengths, T, dim ** -0.5)
    assert int(status) == 0
    check(out, lse, want, dim, 12 * T)
    sel[0, 0, 1] = 40  # a position that the sequence does not have
    lists[0][0] = [e for e in lists[0][0] if e[0] != 3]
    cnt[1, 1] = 9      # more than the list holds: cut, its padding left out
    out, lse = A.decode_attention(*args, selected=sel.to(cuda), selected_count=cnt.to(cuda), return_lse=True,
                                  status=status)
    assert int(status) == N.FLAG_INDEX_RANGE
    check(out, lse, O.decode_attention(q.double().numpy(), lists, lengths, T, dim ** -0.5), dim, 12 * T)
    sel[0, 0, :3] = torch.tensor([3, 0, 3])  # out of order, and a position twice: it counts twice
    lists[0][0] = [(j, c.values[ids[0, j]]) for j in (3, 0, 3)]
    out, lse = A.decode_attention(*args, selected=sel.to(cuda), selected_count=cnt.to(cuda), return_lse=True)
    check(out, lse, O.decode_attention(q.double().numpy(), lists, lengths, T, dim ** -0.5), dim, 12 * T)


# ----------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 1), (4, 1, 3), (9, 2, 1), (64, 1, 1), (2000, 3, 5)])
def test_evict_pages(cuda, budget, sink, recent):
    T, P = 16, 1500
    lengths = [0, 5, 16 * 9, 16 * 9 + 1, 16 * 1500, 23001, 16 * 64]
    g = torch.Generator().manual_seed(50)
    mass = torch.rand(len(lengths), P + 3, generator=g)
    mass[4, ::2] = 0.25                      # ties
    mass[5, 3::5] = float("nan")
    mass[5, 4::50] = -0.0
    mass[5, 7::50] = 0.0
    mass[5, 8::50] = -1.0
    mass[5, 9::50] = float("inf")
    mass[6] = 0.0
    ids = torch.randint(0, 1 << 30, (len(lengths), P + 9), generator=g).to(torch.int32)
    m, i = mass.to(cuda)[:, :P], ids.to(cuda)[:, 2:2 + P]
    L = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    got = A.evict_pages(m, i, L, budget, sink=sink, recent=recent, tokens_per_page=T)
    ids, mass = ids[:, 2:2 + P].numpy(), mass[:, :P].numpy()
    for b, n in enumerate(lengths):
        pages = -(-n // T)
        keep = O.keep_highest(mass[b, :pages].astype(np.float64), budget, sink, recent)
        gone = sorted(set(range(pages)) - set(keep))
        assert got.page_ids[b, :len(keep)].tolist() == ids[b, keep].tolist()
        assert (got.page_ids[b, len(keep):] == -1).all() and (got.page_mass[b, len(keep):] == 0).all()
        assert np.array_equal(got.page_mass[b, :len(keep)].cpu().numpy(), mass[b, keep], equal_nan=True)
        assert got.evicted[b, :len(gone)].tolist() == ids[b, gone].tolist() and (got.evicted[b, len(gone):] == -1).all()
        assert int(got.n_evicted[b]) == len(gone) and int(got.lengths[b]) == n - T * len(gone)


def test_refusals(cuda):
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8], 16, 2, 64, 60)
    ids = torch.zeros(1, 2, dtype=torch.int32, device=cuda)
    L = torch.tensor([16], dtype=torch.int32, device=cuda)
    q = queries(1, 4, 64, 60).to(cuda)
    mass = torch.zeros(1, 2, device=cuda)
    sel, cnt = torch.zeros(1, 2, 1, dtype=torch.int32, device=cuda), torch.ones(1, 2, dtype=torch.int32, device=cuda)

    def no(exc, fn, *a, **k):
        with pytest.raises(exc):
            fn(*a, **k)

    D = A.decode_attention
    no(TypeError, D, q.half(), c.table, c.kv, c.stores, ids, L)
    no(ValueError, D, q[:, :3], c.table, c.kv, c.stores, ids, L)
    no(ValueError, D, q[..., ::2], c.table, c.kv, c.stores, ids, L)
    no(ValueError, D, q.repeat(1, 1, 2), c.table, c.kv, c.stores, ids, L, out=q)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids[0], L)
    no(TypeError, D, q, c.table, c.kv, c.stores, ids.long(), L)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids.cpu(), L)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L.repeat(2))
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, tokens_per_page=0)
    no(N.KernelError, D, q, c.table, c.kv, c.stores, ids, L, tokens_per_page=17)
    no(N.KernelError, D, q, c.table, c.kv, c.stores, ids, L, tokens_per_page=32)
    no(ValueError, D, q, c.table, c.kv, {0: c.stores[1]}, ids, L)
    no(ValueError, D, q, c.table, c.kv, {6: c.stores[1]}, ids, L)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, selected=sel)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, selected=sel, selected_count=cnt, page_mass=mass)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, selected=sel[..., :0], selected_count=cnt)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, selected=sel[:, :1], selected_count=cnt)
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, page_mass=mass[:, :1])
    no(ValueError, D, q, c.table, c.kv, c.stores, ids.expand(2, 2), L.repeat(2),
       page_mass=mass.expand(2, 2))
    no(TypeError, D, q, c.table, c.kv, c.stores, ids, L, status=mass[0, :1])
    no(ValueError, D, q, c.table, c.kv, c.stores, ids, L, tokens_per_page=2 ** 32 + 16)
    b = A.PageBounds.empty(2, 2, 64, cuda)
    no(ValueError, b.update, c.table, c.kv, ids[0], tokens_per_page=2 ** 32 + 16)
    S = A.select_pages
    no(ValueError, S, q, b, ids, L, 0)
    no(ValueError, S, q, b, ids, L, 2, sink=2, recent=1)
    no(ValueError, S, q, b, ids, L, 2, sink=-1)
    no(ValueError, S, q, b, ids, L, 2 ** 32 + 2)
    no(ValueError, S, q, b, ids, L, 2, tokens_per_page=2 ** 32 + 16)
    no(ValueError, S, q[:, :3], b, ids, L, 2)
    no(ValueError, S, torch.zeros(1, 4, 128, dtype=torch.bfloat16, device=cuda), b, ids, L, 2)
    no(ValueError, A.PageBounds, b.codes[..., :32].contiguous(), b.exponents)
    no(ValueError, A.PageBounds, b.codes, b.exponents[:1])
    no(ValueError, A.PageBounds.empty(3, 2, 64, cuda).update, c.table, c.kv, ids[0])
    no(ValueError, A.PageBounds.empty(2, 1, 64, cuda).update, c.table, c.kv, ids[0])
    no(ValueError, b.update, c.table, c.kv, ids[0], valid=L)
    E = A.evict_pages
    no(ValueError, E, mass, ids, L, 2, recent=0)
    no(ValueError, E, mass, ids, L, 2, sink=2, recent=1)
    no(ValueError, E, mass[:, :1], ids, L, 2)
    no(ValueError, E, mass, ids, L, 2 ** 32 + 2)
    no(ValueError, E, mass, ids, L, 2, tokens_per_page=2 ** 32 + 16)
    no(TypeError, E, mass.double(), ids, L, 2)


@pytest.mark.parametrize("tiers,dim,heads", [("nbit4", 128, 8), ("nbit2", 64, 16)])
def test_decode_many_outliers(cuda, tiers, dim, heads):
    """Some pages of 65536 values hold more outliers than a unit carries."""
    c, *_ = run_case(cuda, tiers, 32, heads, heads, dim, [70, 33], 7)
    counts = [int(c.stores[TIER[f]].slot_view()[int(c.table.slot[i])][:4].view(torch.int32)) for i, f in enumerate(c.formats)]
    assert 128 < max(counts) <= CAP


# ----------------------------------------------------------------------------- together
def test_serving_loop(cuda):
    """Pages are bounded while they are bf16, demoted by the migrator, attended with their mass,
    evicted, attended again, and attended by selection: against float64 at every step."""
    from ashkv.contracts.config import ASHKVConfig
    from ashkv.runtime.batch import BatchMigrator
    T, heads, dim, P, B = 16, 2, 128, 20, 3
    row, n = heads * dim, 3 * 20
    g = torch.Generator().manual_seed(70)
    k = torch.randn(n * T, heads, dim, generator=g).bfloat16().to(cuda)
    v = torch.randn(n * T, heads, dim, generator=g).bfloat16().to(cuda)
    table = DevicePageTable.empty(n, cuda)
    table.token_start.copy_(torch.randperm(n, generator=g).to(torch.int32) * T)
    kv = KVLayers([k], [v])
    stores = {1: TierStore(N.PAGE_INT8, n, cuda, T, row), 2: TierStore(N.PAGE_INT4, n, cuda, T, row)}
    lengths = [P * T, 11 * T + 5, 1]
    ids = torch.randperm(n, generator=g).to(torch.int32).view(B, P).to(cuda)
    L = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    # bounds of every full page; they are of the keys as they were before the move
    bounds = A.PageBounds.empty(n, heads, dim, cuda)
    bounds.update(table, kv, ids.view(-1))
    # two thirds of the pages leave the pool, half of those two tiers down; the last pages stay
    mig = BatchMigrator(table, kv, stores, ASHKVConfig(), [(0, 1), (1, 0), (1, 2), (2, 1)], tokens_per_page=T)
    last = {int(ids[b, (x - 1) // T]) for b, x in enumerate(lengths)}
    move = torch.tensor([p for p in range(n) if p % 3 and p not in last], dtype=torch.int32, device=cuda)
    for target, lst in ((1, move), (2, move[::2].contiguous())):
        mig.migrate(lst, torch.tensor([lst.numel()], dtype=torch.int32, device=cuda),
                    torch.full((n,), target, dtype=torch.int8, device=cuda))
        assert (mig.status[:lst.numel()] == N.MIGRATE_OK).all()
    pool = {p: 0 for p in range(n)}
    for p in range(n):
        t, s = int(table.tier[p]), int(table.slot[p])
        if t == 0:
            at = int(table.token_start[p])
            data, fmt = np.concatenate([bits(k[at:at + T]).reshape(-1), bits(v[at:at + T]).reshape(-1)]), N.PAGE_BF16
        else:
            data, fmt = stores[t].slot_view()[s].cpu().numpy(), stores[t].format
        pool[p] = O.page_values(fmt, data, T, heads, dim)
    assert {int(t) for t in table.tier} == {0, 1, 2}
    scale = dim ** -0.5
    mass = torch.zeros(B, P, device=cuda)
    acc = np.zeros((B, P))
    for step in range(2):  # two steps' mass, the first decayed
        q = queries(B, 8, dim, 71 + step, 2.0)
        out, lse = A.decode_attention(q.to(cuda), table, kv, stores, ids, L, page_mass=mass, decay=0.5, return_lse=True)
        lists = [[[(j, pool[int(ids[b, j])]) for j in range(-(-lengths[b] // T))]] * heads for b in range(B)]
        want = O.decode_attention(q.double().numpy(), lists, lengths, T, scale, acc, 0.5)
        check(out, lse, want, dim, P * T, mass, acc, 0.5)
        acc = want["mass"]
    kept = A.evict_pages(mass, ids, L, 8, sink=1, recent=2)
    assert kept.n_evicted.tolist() == [P - 8, 12 - 8, 0] and kept.lengths.tolist() == [8 * T, 7 * T + 5, 1]
    host = mass.cpu().numpy()
    for b in range(B):
        want_ids = [int(ids[b, j]) for j in O.keep_highest(host[b, :-(-lengths[b] // T)].astype(np.float64), 8, 1, 2)]
        assert kept.page_ids[b, :len(want_ids)].tolist() == want_ids
    lengths2 = kept.lengths.tolist()
    lists = [[[(j, pool[int(kept.page_ids[b, j])]) for j in range(-(-lengths2[b] // T))]] * heads for b in range(B)]
    acc = kept.page_mass.double().cpu().numpy()
    out, lse = A.decode_attention(q.to(cuda), table, kv, stores, kept.page_ids, kept.lengths, page_mass=kept.page_mass,
                                  decay=1.0, return_lse=True)
    check(out, lse, O.decode_attention(q.double().numpy(), lists, lengths2, T, scale, acc, 1.0), dim, P * T,
          kept.page_mass, acc, 1.0)
    sel, cnt = A.select_pages(q.to(cuda), bounds, ids, L, 6, sink=1, recent=1)
    check_selected(sel, cnt, select_want(q, bounds, ids.cpu().numpy(), lengths, T, 6, 1, 1))
    out, lse = A.decode_attention(q.to(cuda), table, kv, stores, ids, L, selected=sel, selected_count=cnt, return_lse=True)
    lists = [[[(j, pool[int(ids[b, j])]) for j in sel[b, h, :int(cnt[b, h])].tolist()] for h in range(heads)]
             for b in range(B)]
    check(out, lse, O.decode_attention(q.double().numpy(), lists, lengths, T, scale), dim, 6 * T)


def test_results_do_not_depend_on_the_run(cuda):
    """No sum's order depends on timing: the same call gives the same bits."""
    c = Cache(cuda, [FORMATS["mixed"][i % 4] for i in range(64)], 16, 2, 128, 80)
    ids = torch.randperm(64, generator=torch.Generator().manual_seed(2)).to(torch.int32).view(2, 32).to(cuda)
    L = torch.tensor([512, 300], dtype=torch.int32, device=cuda)
    q = queries(2, 8, 128, 80).to(cuda)
    first = None
    for _ in range(10):
        mass = torch.zeros(2, 32, device=cuda)
        got = (*A.decode_attention(q, c.table, c.kv, c.stores, ids, L, page_mass=mass, return_lse=True), mass)
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))


def test_inputs_written_by_the_kernel_before(cuda):
    """Each call right behind the kernel that writes what it reads (lengths, mass, bounds, scores),
    many times over, against the same calls with the device idle in between."""
    T, heads, dim, P, B = 16, 2, 128, 600, 4
    c = Cache(cuda, [N.PAGE_BF16] * 64, T, heads, dim, 90)
    g = torch.Generator().manual_seed(90)
    ids = torch.randint(0, 64, (B, P), generator=g).to(torch.int32).to(cuda)
    q = queries(B, 8, dim, 90).to(cuda)
    rounds = 12
    lengths = torch.randint(1, P * T, (rounds, B), generator=g).to(torch.int32).to(cuda)
    masses = torch.rand(rounds, B, P, generator=g).to(cuda)
    lists = torch.stack([torch.randperm(64, generator=g) for _ in range(rounds)]).to(torch.int32).to(cuda)

    def run(wait):
        L, mass = torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(B, P, device=cuda)
        bounds, got = A.PageBounds.empty(64, heads, dim, cuda), []
        pause = torch.cuda.synchronize if wait else (lambda: None)
        for r in range(rounds):
            L.copy_(lengths[r]), mass.copy_(masses[r])
            pause()
            got.append(tuple(A.evict_pages(mass, ids, L, 40)))
            c.kv.k[0].neg_(), c.kv.k[1].neg_()
            pause()
            bounds.update(c.table, c.kv, lists[r])
            pause()
            sel, cnt = A.select_pages(q, bounds, ids, L, 33)
            pause()
            got.append((sel, cnt, A.decode_attention(q, c.table, c.kv, None, ids, L, selected=sel, selected_count=cnt)))
            pause()
            got.append((A.decode_attention(q, c.table, c.kv, None, ids, L, page_mass=mass), mass.clone()))
            pause()
            got.append(tuple(A.evict_pages(mass, ids, L, 40)))
            pause()
        torch.cuda.synchronize()
        return got

    want, got = run(True), run(False)  # an even number of sign changes: both start from the same keys
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_decode_the_longest_list(cuda):
    """2^31 - 1 - 2^16 pages of one token; all but the last entry weigh e^-64."""
    most, dim = 2 ** 31 - 1 - 2 ** 16, 64
    k, v = (torch.zeros(2, 1, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    k[1], v[0] = 8.0, 1.0
    v[1] = torch.arange(dim).to(v)
    table = DevicePageTable.empty(2, cuda)
    table.token_start[1] = 1
    ids = torch.zeros(1, most, dtype=torch.int32, device=cuda)
    ids[0, -1] = 1
    L, status = torch.tensor([most], dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = A.decode_attention(torch.ones(1, 1, dim, dtype=torch.bfloat16, device=cuda), table, KVLayers([k], [v]),
                                  None, ids, L, tokens_per_page=1, return_lse=True, status=status)
    # the other entries weigh less than 2^31 e^-64 = 2^(31 - 92.33) < 2^-61 together, their values are at most 1, and
    # v[1]'s whole numbers are bf16 numbers; lse: log2(e), ln 2 and two products are rounded
    assert int(status) == 0 and ((out[0, 0].double() - v[1, 0].double()).abs() <= 2.0 ** -61).all()
    assert abs(float(lse) - 64.0) <= 8 * U * 64.0


@pytest.mark.parametrize("heads_q", [8, 12])
@pytest.mark.parametrize("tiers,power", [(t, e) for t in FORMATS for e in (110, -110)] +
                         [(t, e) for t in ("int8", "fp8", "int4") for e in (125, -125)])
def test_decode_queries_of_any_size(cuda, tiers, power, heads_q):
    """Queries near either end of bf16's range, brought back by the scale (bf16 keys stay where
    an fp32 sum of products does not overflow)."""
    T, heads, dim = 16, 1, 128
    c = Cache(cuda, [FORMATS[tiers][i % len(FORMATS[tiers])] for i in range(8)], T, heads, dim, 91)
    ids = np.arange(8, dtype=np.int32).reshape(1, 8)
    q = queries(1, heads_q, dim, 91).float().mul(2.0 ** power).bfloat16()
    assert torch.isfinite(q).all()
    scale = 0.05 * 2.0 ** -power
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda),
                                  torch.tensor([120], dtype=torch.int32, device=cuda), scale=scale, return_lse=True)
    check(out, lse, O.decode_attention(q.double().numpy(), c.lists(ids, [120]), [120], T, scale), dim, 120)


@pytest.mark.parametrize("heads_q", [8, 12])
@pytest.mark.parametrize("kinds", [[N.PAGE_INT4] * 3, [N.PAGE_INT4, N.PAGE_BF16, N.PAGE_NBIT2], [N.PAGE_NBIT4] * 2])
def test_decode_large_keys(cuda, kinds, heads_q):
    """Keys around 2^97, brought back by the scale."""
    T, heads, dim, scale = 16, 1, 128, 0.5 * 2.0 ** -97
    g = torch.Generator().manual_seed(92)
    pages = torch.randn(len(kinds), 2, T * heads * dim, generator=g)
    pages[:, 0] *= 2.0 ** 97
    c = Cache(cuda, kinds, T, heads, dim, 92, pool_bits=bits(pages.reshape(len(kinds), -1).to(torch.bfloat16)))
    ids, lengths = np.arange(len(kinds), dtype=np.int32)[None], [len(kinds) * T - 3]
    q = queries(1, heads_q, dim, 92)
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda),
                                  torch.tensor(lengths, dtype=torch.int32, device=cuda), scale=scale, return_lse=True)
    check(out, lse, O.decode_attention(q.double().numpy(), c.lists(ids, lengths), lengths, T, scale), dim, lengths[0])


def run_shared(dev, c, heads_q, lengths, seed, ids=None, decay=0.75, scale=None):
    """Sequences over few pages that they share, so many list entries that a worker has several to
    attend one after the other (at most 12 workers on each of 148 SMs for all key heads)."""
    P = max(-(-x // c.T) for x in lengths)
    entries, workers = sum(-(-x // c.T) for x in lengths), 12 * torch.cuda.get_device_properties(dev).multi_processor_count
    assert entries >= 3 * (workers // c.heads)
    g = np.random.default_rng(seed)
    if ids is None:
        ids = g.integers(0, len(c.formats), (len(lengths), P)).astype(np.int32)
    q, acc = queries(len(lengths), heads_q, c.dim, seed), g.random((len(lengths), P), dtype=np.float32)
    mass, status = torch.from_numpy(acc.copy()).to(dev), torch.zeros(1, dtype=torch.int32, device=dev)
    scale = c.dim ** -0.5 if scale is None else scale
    out, lse = A.decode_attention(q.to(dev), c.table, c.kv, c.stores, torch.from_numpy(ids).to(dev),
                                  torch.tensor(lengths, dtype=torch.int32, device=dev), tokens_per_page=c.T, scale=scale,
                                  page_mass=mass, decay=decay, return_lse=True, status=status)
    assert int(status) == 0
    want = O.decode_attention(q.double().numpy(), c.lists(ids, lengths), lengths, c.T, scale, acc, decay)
    check(out, lse, want, c.dim, max(lengths) + 1, mass, acc, decay)


def far_apart(dev, kinds, sizes):
    T, heads, dim = 16, 16, 128
    g = torch.Generator().manual_seed(93)
    pages = torch.randn(len(kinds), 2, T * heads * dim, generator=g)
    pages[:, 1] *= torch.tensor(sizes)[:, None]
    return Cache(dev, kinds, T, heads, dim, 93, pool_bits=bits(pages.reshape(len(kinds), -1).to(torch.bfloat16)))


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("kinds,sizes", [
    ([N.PAGE_BF16, N.PAGE_INT4], [2.0 ** 70, 2.0 ** -40]), ([N.PAGE_INT8, N.PAGE_NBIT4], [1e-5, 2.0 ** 70]),
    ([N.PAGE_NBIT2, N.PAGE_INT8, N.PAGE_BF16], [2.0 ** 70, 1e-5, 1.0]),
    ([N.PAGE_INT4, N.PAGE_BF16, N.PAGE_INT4], [1e-8, 2.0 ** 62, 2.0 ** 100]),
    ([N.PAGE_INT4, N.PAGE_BF16, N.PAGE_INT4], [1e-7, 1e15, 1.0]), ([N.PAGE_INT4] * 3, [3e35, 1e-7, 1e35]),
    ([N.PAGE_INT4, N.PAGE_FP8, N.PAGE_FP8], [1e-7, 1e2, 1.0]), ([N.PAGE_BF16] * 2, [2.0 ** 100, 2.0 ** -60])])
def test_decode_values_of_far_apart_sizes_of_one_worker(cuda, kinds, sizes, group):
    """The power of two that small scales need leaves room for the values of other pages, before and behind them."""
    c = far_apart(cuda, kinds, sizes)
    ids = (np.arange(36 * 10) % len(kinds)).astype(np.int32).reshape(36, 10)
    run_shared(cuda, c, 16 * group, [157] * 36, 93, ids)


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("first", [0, 1])
def test_decode_scales_smaller_than_a_codec_writes(cuda, first, group):
    """INT4 V scales of 2^-60 beside bf16 values of 2^70."""
    T, heads, dim = 16, 16, 128
    c = far_apart(cuda, [N.PAGE_INT4, N.PAGE_BF16], [1.0, 2.0 ** 70])
    slot = c.stores[TIER[N.PAGE_INT4]].slot_view()[int(c.table.slot[0])]
    row = heads * dim
    slot[T * row // 32:2 * T * row // 32].view(torch.bfloat16).fill_(2.0 ** -60)
    c.values[0] = O.page_values(N.PAGE_INT4, slot.cpu().numpy(), T, heads, dim)
    ids = ((first + np.arange(36 * 10)) % 2).astype(np.int32).reshape(36, 10)
    run_shared(cuda, c, heads * group, [157] * 36, 94, ids)


@pytest.mark.parametrize("heads_q", [2, 12])
@pytest.mark.parametrize("at", [0, 3, 21])
def test_decode_an_infinite_value_stays_infinite(cuda, at, heads_q):
    """... in its channel; beside one of the other sign it gives NaN."""
    c = Cache(cuda, [N.PAGE_BF16] * 2, 16, 1, 64, 8)
    ids = torch.arange(2, dtype=torch.int32, device=cuda).view(1, 2)
    L = torch.tensor([30], dtype=torch.int32, device=cuda)
    q = queries(1, heads_q, 64, 8).to(cuda)
    where = [(c.kv.v[int(c.table.layer[p])], int(c.table.token_start[p])) for p in range(2)]
    want = A.decode_attention(q, c.table, c.kv, None, ids, L)
    v, s = where[at // 16]
    v[s + at % 16, 0, 5], v[s + at % 16, 0, 9] = float("inf"), -float("inf")
    out = A.decode_attention(q, c.table, c.kv, None, ids, L)
    assert (out[..., 5] == float("inf")).all() and (out[..., 9] == -float("inf")).all()
    rest = [d for d in range(64) if d not in (5, 9)]
    assert torch.equal(out[..., rest], want[..., rest])
    v, s = where[0]
    v[s + 7, 0, 5] = -float("inf")
    out = A.decode_attention(q, c.table, c.kv, None, ids, L)
    assert torch.isnan(out[..., 5]).all() and (out[..., 9] == -float("inf")).all()


def test_refuses_heads_of_another_size_than_the_pools(cuda):
    c = Cache(cuda, [N.PAGE_BF16], 16, 2, 128, 61)
    ids, L = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.tensor([16], dtype=torch.int32, device=cuda)
    with pytest.raises(ValueError, match="128 channels"):
        A.decode_attention(queries(1, 4, 64, 61).to(cuda), c.table, c.kv, None, ids, L)
    with pytest.raises(ValueError, match="128 channels"):
        A.PageBounds.empty(1, 4, 64, cuda).update(c.table, c.kv, ids[0])
    flat = KVLayers([k.view(k.shape[0], -1) for k in c.kv.k], [v.view(v.shape[0], -1) for v in c.kv.v])  # rows as one
    q = queries(1, 4, 128, 61).to(cuda)
    assert torch.equal(A.decode_attention(q, c.table, flat, None, ids, L), A.decode_attention(q, c.table, c.kv, None, ids, L))


def test_refuses_stores_of_other_pages(cuda):
    """Slots are laid out for one page size; a smaller page fits, but is not what they hold."""
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8], 16, 2, 128, 62)
    ids, L = torch.zeros(1, 2, dtype=torch.int32, device=cuda), torch.tensor([8], dtype=torch.int32, device=cuda)
    q = queries(1, 4, 128, 62).to(cuda)
    A.decode_attention(q, c.table, c.kv, c.stores, ids, L)
    with pytest.raises(N.KernelError, match="laid out for pages of 16 x 256"):
        A.decode_attention(q, c.table, c.kv, c.stores, ids, L, tokens_per_page=8)
    wide = {1: TierStore(N.PAGE_INT8, 2, cuda, 16, 512)}
    with pytest.raises(N.KernelError, match="laid out for pages of 16 x 512"):
        A.decode_attention(q, c.table, c.kv, wide, ids, L)


# ----------------------------------------------------------------------------- every instance of the kernels
STORES = {**FORMATS, "fp8+int4": [N.PAGE_FP8, N.PAGE_INT4]}  # the last: queries in all three forms at once


@pytest.mark.parametrize("tiers", list(STORES))
@pytest.mark.parametrize("dim,heads", [(64, 2), (64, 8), (128, 1), (128, 2)])
@pytest.mark.parametrize("group", [9, 20])
def test_decode_groups_of_all_formats(cuda, tiers, dim, heads, group, monkeypatch):
    monkeypatch.setitem(FORMATS, tiers, STORES[tiers])
    run_case(cuda, tiers, 16, heads * group, heads, dim, [50, 131], 100)


@pytest.mark.parametrize("dim,heads,group", [(64, 1, 12), (64, 3, 9), (128, 5, 11)])
def test_decode_odd_numbers_of_heads(cuda, dim, heads, group):
    run_case(cuda, "bf16", 16, heads * group, heads, dim, [50, 131], 101)


@pytest.mark.parametrize("tiers", list(STORES))
@pytest.mark.parametrize("T", [1, 19])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 3), (64, 10), (128, 12)])
def test_decode_compressed_pages_of_an_odd_number_of_tokens(cuda, tiers, T, dim, group, monkeypatch):
    monkeypatch.setitem(FORMATS, tiers, STORES[tiers])
    heads = 512 // dim
    run_case(cuda, tiers, T, heads * group, heads, dim, [T, 3 * T - 1, 4 * T + 1, 1], 102)


@pytest.mark.parametrize("tiers", list(STORES))
@pytest.mark.parametrize("T,dim,group", [(16, 128, 1), (16, 64, 12), (5, 128, 9), (8, 64, 2), (16, 128, 8)])
def test_decode_several_pages_to_a_worker(cuda, tiers, T, dim, group):
    """Workers that attend many pages of several sequences, some of them empty."""
    heads = 2048 // dim
    kinds = STORES[tiers]
    c = Cache(cuda, [kinds[i % len(kinds)] for i in range(12)], T, heads, dim, 103)
    run_shared(cuda, c, heads * group, [0 if i % 7 == 3 else 1 + (53 * i) % (40 * T) for i in range(30)], 103)


@pytest.mark.parametrize("tiers", ["bf16", "mixed", "fp8+int4"])
@pytest.mark.parametrize("dim,group", [(64, 3), (128, 12)])
def test_decode_selected_several_pages_to_a_worker(cuda, tiers, dim, group):
    T, heads, P, B = 16, 1024 // dim, 60, 24
    kinds = STORES[tiers]
    c = Cache(cuda, [kinds[i % len(kinds)] for i in range(12)], T, heads, dim, 104)
    g = np.random.default_rng(104)
    ids = g.integers(0, 12, (B, P)).astype(np.int32)
    lengths = [int(x) for x in g.integers(1, P * T, B)]
    lengths[5] = 0
    sel, cnt = np.full((B, heads, 40), -1, np.int32), np.zeros((B, heads), np.int32)
    rows = {}
    for b in range(B):
        for h in range(heads):
            pages = -(-lengths[b] // T)
            k = int(g.integers(0, min(40, pages) + 1))
            rows[b, h] = sorted(g.permutation(pages)[:k].tolist())
            sel[b, h, :k], cnt[b, h] = rows[b, h], k
    q, status = queries(B, heads * group, dim, 104), torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = A.decode_attention(q.to(cuda), c.table, c.kv, c.stores, torch.from_numpy(ids).to(cuda),
                                  torch.tensor(lengths, dtype=torch.int32, device=cuda), selected=torch.from_numpy(sel).to(cuda),
                                  selected_count=torch.from_numpy(cnt).to(cuda), return_lse=True, status=status)
    assert int(status) == 0
    lists = [[[(j, c.values[ids[b, j]]) for j in rows[b, h]] for h in range(heads)] for b in range(B)]
    check(out, lse, O.decode_attention(q.double().numpy(), lists, lengths, T, dim ** -0.5), dim, 40 * T)


@pytest.mark.parametrize("pages", [8191, 8192, 8193, 20001])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 1), (300, 2, 5), (8192, 1, 1), (20000, 0, 0)])
def test_select_rows_around_and_beyond_8192(cuda, pages, budget, sink, recent):
    """Rows whose keys do not fit the registers of a CTA are read anew in each round."""
    T, n, heads = 16, 700, 2
    g = torch.Generator().manual_seed(105)
    b = A.PageBounds.empty(n, heads, 64, cuda)
    b.codes.copy_(torch.randint(-127, 128, b.codes.shape, generator=g).sort(2).values.to(torch.int8))
    b.exponents.copy_(torch.randint(-2, 2, (n, heads), generator=g).to(torch.int8))
    ids = torch.randint(0, n, (2, pages), generator=g).to(torch.int32)  # every page about thirty times: ties
    lengths = [pages * T - 3, (pages // 2) * T]
    q = queries(2, 4, 64, 105)
    sel, cnt = A.select_pages(q.to(cuda), b, ids.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda), budget,
                              sink=sink, recent=recent)
    check_selected(sel, cnt, select_want(q, b, ids.numpy(), lengths, T, budget, sink, recent))


@pytest.mark.parametrize("pages", [8192, 8193, 20001])
@pytest.mark.parametrize("budget,sink,recent", [(1, 0, 1), (700, 3, 8), (8192, 1, 1), (20000, 5, 2)])
def test_evict_rows_around_and_beyond_8192(cuda, pages, budget, sink, recent):
    T = 16
    g = torch.Generator().manual_seed(106)
    mass = torch.rand(4, pages, generator=g)
    mass[1, ::2] = 0.25  # ties
    mass[2, 3::5] = float("nan")
    mass[2, 4::50], mass[2, 8::50], mass[2, 9::50] = -0.0, -1.0, float("inf")
    mass[3] = 0.0
    ids = torch.randint(0, 1 << 30, (4, pages), generator=g).to(torch.int32)
    lengths = [pages * T, pages * T - 5, (pages - 1) * T + 1, (pages // 2) * T]
    got = A.evict_pages(mass.to(cuda), ids.to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda), budget, sink=sink,
                        recent=recent)
    for b, n in enumerate(lengths):
        used = -(-n // T)
        keep = O.keep_highest(mass[b, :used].double().numpy(), budget, sink, recent)
        gone = np.setdiff1d(np.arange(used), keep)
        assert np.array_equal(got.page_ids[b, :len(keep)].cpu().numpy(), ids[b, keep].numpy())
        assert np.array_equal(got.page_mass[b, :len(keep)].cpu().numpy(), mass[b, keep].numpy(), equal_nan=True)
        assert (got.page_ids[b, len(keep):] == -1).all() and (got.page_mass[b, len(keep):] == 0).all()
        assert np.array_equal(got.evicted[b, :len(gone)].cpu().numpy(), ids[b, gone].numpy())
        assert (got.evicted[b, len(gone):] == -1).all()
        assert int(got.n_evicted[b]) == len(gone) and int(got.lengths[b]) == n - T * len(gone)


def test_refuses_rows_that_overlap(cuda):
    """Sequences whose ids or masses share memory: two blocks would update one mass."""
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_BF16], 16, 2, 64, 60)
    ids = torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    L, q, mass = torch.full((2,), 16, dtype=torch.int32, device=cuda), queries(2, 4, 64, 60).to(cuda), torch.zeros(2, 2, device=cuda)
    bounds = A.PageBounds.empty(2, 2, 64, cuda)
    for call in (lambda i, m: A.decode_attention(q, c.table, c.kv, c.stores, i, L, page_mass=m),
                 lambda i, m: A.evict_pages(m, i, L, 2)):
        call(ids, mass)
        for i, m in ((ids[:1].expand(2, 2), mass), (ids, mass[:1].expand(2, 2)),
                     (ids, torch.zeros(3, device=cuda).as_strided((2, 2), (1, 1)))):
            with pytest.raises(ValueError, match="rows overlap"):
                call(i, m)
    with pytest.raises(ValueError, match="rows overlap"):
        A.select_pages(q, bounds, ids[:1].expand(2, 2), L, 2)
