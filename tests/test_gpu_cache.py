"""GPU tests of writing tokens into tiered pages and reading them back.

Bytes are compared with the oracle's page codecs, exactly: a token's codes and scale are those of the
page encoded as a whole (INT8 codes may be one apart where the oracle marks a tie of the GPU's
approximate division), every other byte of the stores and the pool stays as it was, and a read gives
the bits that the oracle's page decoder gives."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from test_gpu_attention import CAP, FORMATS, TIER, Cache, bits

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime import cache as C
from ashkv.runtime.batch import DevicePageTable, KVLayers, StepGraph, TierStore

pytestmark = pytest.mark.gpu

SHAPES = [(8, 128), (2, 64), (4, 64), (4, 128), (16, 128)]  # rows of 1024, 128, 256, 512, 2048


def i32(x, dev):
    return torch.as_tensor(np.asarray(x, np.int32)).to(dev)


def starts_of(new):
    return np.concatenate([[0], np.cumsum(new)])


def pool_bits(c):
    return [[bits(x).reshape(-1, c.heads * c.dim) for x in side] for side in (c.kv.k, c.kv.v)]


def row_bytes(fmt, T, row, r):
    """Ranges of a slot's bytes that hold row r of the page."""
    E = 2 * T * row
    if fmt == N.PAGE_INT8:
        c0 = (4 * T + 15) // 16 * 16
        return [(2 * r, 2 * r + 2), (c0 + r * row, c0 + (r + 1) * row)]
    if fmt == N.PAGE_FP8:
        return [(r * row, (r + 1) * row)]
    return [(r * (row // 32), (r + 1) * (row // 32)), (E // 32 + r * (row // 2), E // 32 + (r + 1) * (row // 2))]


def place(c, page):
    t = c.table
    return int(t.tier[page]), int(t.layer[page]), int(t.token_start[page]), int(t.slot[page])


def expect_writes(c, rows, pool, slots):
    """Applies (page, token, K bits, V bits) to copies of the pool and the slots; True: bytes that may be one apart."""
    T, row = c.T, c.heads * c.dim
    ties = {t: np.zeros(s.shape, bool) for t, s in slots.items()}
    for page, t, kb, vb in rows:
        fmt, (tier, layer, start, slot) = c.formats[page], place(c, page)
        if fmt == N.PAGE_BF16:
            pool[0][layer][start + t], pool[1][layer][start + t] = kb, vb
            continue
        image = np.zeros((2, T, row), np.uint16)
        image[0, t], image[1, t] = kb, vb
        data, tie, _ = oracle.page_encode(fmt, image, T, row)
        for r in (t, T + t):
            for a, b in row_bytes(fmt, T, row, r):
                slots[tier][slot, a:b] = data[a:b]
                ties[tier][slot, a:b] = tie[a:b]
    return ties


def slot_bytes(c):
    return {t: s.data[:s.n_slots * s.slot_bytes].view(s.n_slots, -1).cpu().numpy().copy() for t, s in c.stores.items()}


def check_stores(c, want, ties):
    for t, got in slot_bytes(c).items():
        near = np.abs(got.view(np.int8).astype(int) - want[t].view(np.int8)) <= 1
        assert ((got == want[t]) | (ties[t] & near)).all()


def new_rows(n, heads, dim, dev, seed, shift=0):
    """K and V rows as slices of a fused projection; ``shift`` puts them off their alignment."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, 3 * heads * dim + 8 + shift, generator=g) * 2).to(torch.bfloat16)
    x[::5] *= 30
    x = x.to(dev)
    k = x[:, shift:shift + heads * dim].unflatten(1, (heads, dim))
    v = x[:, shift + heads * dim:shift + 2 * heads * dim].unflatten(1, (heads, dim))
    return k, v


def layout(c, lengths, new, ids):
    """(row of the call, page, token) of every new token."""
    out, i = [], 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        for pos in range(n - m, n):
            out.append((i, int(ids[b][pos // c.T]), pos % c.T))
            i += 1
    return out


def write_case(dev, kinds, T, heads, dim, lengths, new, seed, shift=0, flat=False):
    P = max(1, max(-(-x // T) for x in lengths))
    g = np.random.default_rng(seed)
    n = len(lengths) * P
    c = Cache(dev, [kinds[i % len(kinds)] for i in range(n)], T, heads, dim, seed)
    ids = g.permutation(n).astype(np.int32).reshape(len(lengths), P)
    k, v = new_rows(sum(new), heads, dim, dev, seed, shift)
    pool, slots = pool_bits(c), slot_bytes(c)
    kb, vb = bits(k).reshape(sum(new), -1), bits(v).reshape(sum(new), -1)
    ties = expect_writes(c, [(p, t, kb[i], vb[i]) for i, p, t in layout(c, lengths, new, ids)], pool, slots)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    args = (c.table, c.kv, c.stores, i32(ids, dev), i32(lengths, dev), i32(starts_of(new), dev))
    C.write_kv(k.flatten(1) if flat else k, v.flatten(1) if flat else v, *args, tokens_per_page=T, status=status)
    assert int(status) == 0
    for got, want in zip(pool_bits(c), pool):
        for x, y in zip(got, want):
            assert np.array_equal(x, y)
    check_stores(c, slots, ties)
    return c, ids, args, k, v


WRITES = {"bf16": [N.PAGE_BF16], "int8": [N.PAGE_INT8], "fp8": [N.PAGE_FP8], "int4": [N.PAGE_INT4],
          "three": [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT4], "three8": [N.PAGE_FP8, N.PAGE_INT4, N.PAGE_BF16]}


@pytest.mark.parametrize("tiers", list(WRITES))
@pytest.mark.parametrize("heads,dim", SHAPES)
def test_write(cuda, tiers, heads, dim):
    write_case(cuda, WRITES[tiers], 16, heads, dim, [70, 0, 1, 16, 33, 57], [70, 0, 1, 3, 17, 0], 1)


@pytest.mark.parametrize("T,tiers", [(1, "bf16"), (5, "bf16"), (8, "three"), (1, "int8"), (19, "int8"), (12, "int4"),
                                     (32, "three8"), (64, "int8")])
def test_write_page_sizes(cuda, T, tiers):
    write_case(cuda, WRITES[tiers], T, 8, 64, [1, T, T + 1, 3 * T - 1, 90], [1, T, 1, 2 * T, 90], 2)


@pytest.mark.parametrize("tiers", ["bf16", "int8", "fp8", "int4"])
@pytest.mark.parametrize("shift,flat", [(1, False), (4, False), (8, True), (0, True)])
def test_write_strides_and_alignment(cuda, tiers, shift, flat):
    write_case(cuda, WRITES[tiers], 16, 4, 64, [40, 9], [11, 9], 3, shift, flat)


def test_write_many_sequences(cuda):
    """More sequences than a step of the search looks at, most with a token or none."""
    n = 1500
    new = [(i * 7) % 3 for i in range(n)]
    write_case(cuda, WRITES["int8"], 16, 2, 64, [m + i % 20 for i, m in enumerate(new)], new, 4)


@pytest.mark.parametrize("heads,dim,T", [(2, 64, 8), (4, 64, 16), (4, 128, 4)])
def test_many_rows(cuda, heads, dim, T):
    """Enough rows that a warp takes several: they may cross pages and sequences, follow a page that does not exist, and end early."""
    lengths, seqs = 20000 + 3, 2
    P = -(-lengths // T)
    n = 64  # (each stands in many places of the lists)
    c = Cache(cuda, FORMATS["mixed"] * (n // 4), T, heads, dim, 20)
    g = np.random.default_rng(20)
    ids = g.integers(0, n, (seqs, P)).astype(np.int32)
    ids[1, 5::7] = n + 3
    new = [20001, 19990]
    args = (c.table, c.kv, c.stores, i32(ids, cuda), i32([lengths, lengths - 2], cuda), i32(starts_of(new) + 1, cuda), sum(new) + 5)
    out = tuple(torch.full((args[-1], heads, dim), 5.0, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    C.read_kv(*args, tokens_per_page=T, out=out, status=status)
    assert int(status) & N.FLAG_INDEX_RANGE
    pages = np.zeros((n + 4, 2, T, heads * dim), np.uint16)
    for i in range(n):
        pages[i] = page_bits_of(c, i)
    for side in range(2):
        got = bits(out[side]).reshape(-1, heads * dim)
        assert (bits(out[side][:1]) == 0x40A0).all() and (got[1 + sum(new):] == 0x40A0).all()
        at = 1
        for b, (length, m) in enumerate(zip((lengths, lengths - 2), new)):
            pos = np.arange(length - m, length)
            want = pages[np.minimum(ids[b, pos // T], n + 3), side, pos % T]
            assert np.array_equal(got[at:at + m], want)
            at += m


@pytest.mark.parametrize("heads,dim,T,tiers", [(2, 64, 8, "bf16"), (2, 64, 16, "int8"), (4, 64, 16, "int4"), (4, 64, 4, "fp8")])
def test_write_many_rows(cuda, heads, dim, T, tiers):
    """As many rows written, each to a place of its own, as a few at a time write them."""
    seqs, length = 5, 8001
    P = -(-length // T)
    caches = []
    n = seqs * length
    k, v = new_rows(n, heads, dim, cuda, 21)
    ids = i32(np.random.default_rng(21).permutation(seqs * P).reshape(seqs, P), cuda)
    row = heads * dim
    fmt = FORMATS[tiers][0]
    for step in (n, 8001):
        z = torch.zeros(seqs * P, device=cuda)
        tier = torch.full((seqs * P,), TIER.get(fmt, 0), dtype=torch.int8, device=cuda)
        own = torch.arange(seqs * P, dtype=torch.int32, device=cuda)
        table = DevicePageTable(z, z, z, z, tier, torch.zeros_like(own), torch.zeros_like(own), own * T, own)
        pool = [torch.zeros(seqs * P * T, heads, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
        stores = {} if fmt == N.PAGE_BF16 else {TIER[fmt]: TierStore(fmt, seqs * P, cuda, T, row)}
        for s in stores.values():
            s.data.zero_()
        kv = KVLayers(pool[:1], pool[1:])
        for b in range(0, n, step):
            m = min(step, n - b)
            one = slice(b // length, (b + m) // length)
            C.write_kv(k[b:b + m], v[b:b + m], table, kv, stores, ids[one].contiguous(), i32([length] * (m // length), cuda),
                       i32(starts_of([length] * (m // length)), cuda), tokens_per_page=T)
        caches.append((pool, [s.data for s in stores.values()]))
    (pool, data), (pool1, data1) = caches
    for a, b in zip(pool + data, pool1 + data1):
        assert torch.equal(a, b)
    assert any(bool((x != 0).any()) for x in pool + data)


@pytest.mark.parametrize("heads,dim", [(3, 40), (5, 64), (1, 8), (1, 3000)])
def test_rows_of_any_size_in_the_pool(cuda, heads, dim):
    dev, T, n = cuda, 4, 40
    k = torch.zeros(n * T, heads, dim, dtype=torch.bfloat16, device=dev)
    v = torch.zeros_like(k)
    start = i32(np.random.default_rng(0).permutation(n) * T, dev)
    z = torch.zeros(n, device=dev)
    zi = torch.zeros(n, dtype=torch.int32, device=dev)
    table = DevicePageTable(z, z, z, z, zi.to(torch.int8), zi, zi, start, zi)
    ids = torch.arange(n, dtype=torch.int32, device=dev).view(4, 10)
    lengths, new = [40, 13, 0, 7], [40, 5, 0, 7]
    nk = torch.randn(sum(new), heads, dim, device=dev).bfloat16()
    nv = torch.randn(sum(new), heads, dim, device=dev).bfloat16()
    args = (table, KVLayers([k], [v]), None, ids, i32(lengths, dev), i32(starts_of(new), dev))
    C.write_kv(nk, nv, *args, tokens_per_page=T)
    gk, gv = C.read_kv(*args, sum(new), tokens_per_page=T)
    assert torch.equal(gk, nk) and torch.equal(gv, nv)
    assert (k != 0).any(-1).any(-1).sum() == sum(new)


def special_rows(heads, dim, dev):
    x = torch.randn(12, heads, dim, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    x[0] = 0.0
    x[1, 0, 3] = float("nan")
    x[2, 1, 5] = float("inf")
    x[3, 0, 7] = -float("inf")
    x[4] *= 2.0 ** -125
    x[5] *= 2.0 ** 120
    x[6] = float("nan")
    x[7] = 464.0
    x[8] = -480.0
    x[9] = 1e-30
    x[10, :, ::2] = -0.0
    return x.to(dev)


@pytest.mark.parametrize("fmt", [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_FP8, N.PAGE_INT4])
def test_write_special_values(cuda, fmt):
    """NaN, infinities, zeros, subnormal and huge rows are coded as the page codecs code them."""
    T, heads, dim = 16, 2, 128
    c = Cache(cuda, [fmt], T, heads, dim, 3)
    x = special_rows(heads, dim, cuda)
    n = x.shape[0]
    pool, slots = pool_bits(c), slot_bytes(c)
    xb, yb = bits(x).reshape(n, -1), bits(x.flip(0)).reshape(n, -1)
    ties = expect_writes(c, [(0, t, xb[t], yb[t]) for t in range(n)], pool, slots)
    C.write_kv(x, x.flip(0), c.table, c.kv, c.stores, i32([[0]], cuda), i32([n], cuda), i32([0, n], cuda))
    check_stores(c, slots, ties)
    for got, want in zip(pool_bits(c), pool):
        assert all(np.array_equal(a, b) for a, b in zip(got, want))


def page_bits_of(c, page):
    """The bf16 bits that a page decodes to [2, T, row], from the stored bytes."""
    T, row = c.T, c.heads * c.dim
    fmt, (tier, layer, start, slot) = c.formats[page], place(c, page)
    if fmt == N.PAGE_BF16:
        return np.stack([bits(side[layer]).reshape(-1, row)[start:start + T] for side in (c.kv.k, c.kv.v)])
    s = c.stores[tier]
    data = s.data[slot * s.slot_bytes:(slot + 1) * s.slot_bytes].cpu().numpy()
    return oracle.page_decode(fmt, data, T, row, outlier_cap=CAP).reshape(2, T, row)


def check_read(c, lengths, new, ids, k, v):
    decoded = {}
    kb, vb = bits(k).reshape(k.shape[0], -1), bits(v).reshape(k.shape[0], -1)
    for i, page, t in layout(c, lengths, new, ids):
        if page not in decoded:
            decoded[page] = page_bits_of(c, page)
        for got, want in ((kb[i], decoded[page][0, t]), (vb[i], decoded[page][1, t])):
            nan = (want & 0x7FFF) > 0x7F80
            assert np.array_equal(got[~nan], want[~nan]) and ((got[nan] & 0x7FFF) > 0x7F80).all()


@pytest.mark.parametrize("tiers", list(FORMATS))
@pytest.mark.parametrize("heads,dim", SHAPES)
def test_read(cuda, tiers, heads, dim):
    T, lengths, new = 16, [70, 0, 1, 16, 33, 57], [70, 0, 1, 3, 17, 0]
    kinds = FORMATS[tiers]
    c = Cache(cuda, [kinds[i % len(kinds)] for i in range(30)], T, heads, dim, 6)
    ids = np.random.default_rng(6).permutation(30).astype(np.int32).reshape(6, 5)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    k, v = C.read_kv(c.table, c.kv, c.stores, i32(ids, cuda), i32(lengths, cuda), i32(starts_of(new), cuda), sum(new),
                     status=status)
    assert k.shape == (sum(new), heads, dim) and int(status) == 0
    check_read(c, lengths, new, ids, k, v)


@pytest.mark.parametrize("tiers,T", [("nbit4", 4), ("nbit2", 4), ("mixed", 8), ("mixed8", 40), ("int8", 1), ("int8", 19),
                                     ("nbit2", 64)])
def test_read_page_sizes(cuda, tiers, T):
    lengths, new = [1, T, T + 1, 3 * T - 1], [1, T, 1, 2 * T]
    kinds = FORMATS[tiers]
    c = Cache(cuda, [kinds[i % len(kinds)] for i in range(12)], T, 8, 64, 7)
    ids = np.random.default_rng(7).permutation(12).astype(np.int32).reshape(4, 3)
    k, v = C.read_kv(c.table, c.kv, c.stores, i32(ids, cuda), i32(lengths, cuda), i32(starts_of(new), cuda), sum(new),
                     tokens_per_page=T)
    check_read(c, lengths, new, ids, k, v)


@pytest.mark.parametrize("tiers", list(WRITES))
def test_read_gives_what_was_written(cuda, tiers):
    lengths, new = [70, 0, 5, 40], [70, 0, 2, 39]
    c, ids, args, k, v = write_case(cuda, WRITES[tiers], 16, 8, 128, lengths, new, 8)
    gk, gv = C.read_kv(*args, sum(new))
    check_read(c, lengths, new, ids, gk, gv)
    if tiers == "bf16":
        assert torch.equal(gk, k) and torch.equal(gv, v)


def test_rows_of_no_sequence_and_bad_pages(cuda):
    """Padding stays as it was, tokens without a page are left out and flagged, and nothing else is touched."""
    T, heads, dim = 16, 2, 128
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT8, N.PAGE_NBIT2, N.PAGE_BF16, N.PAGE_INT8, N.PAGE_BF16], T, heads, dim, 9)
    c.table.tier[1] = 5            # a tier without a store
    c.table.slot[2] = 100          # a slot outside the store
    c.table.layer[4] = 9           # a layer that does not exist
    c.table.slot[5] = -1
    c.table.token_start[6] = 7 * T - 15
    ids = i32([[0, -1], [7, 0], [1, 0], [2, 0], [4, 0], [5, 0], [6, 0], [0, 0]], cuda)
    lengths = [32, 3, 3, 3, 3, 3, 3, 40]
    new = [16, 3, 3, 3, 3, 3, 3, 8]      # the first: a page id of -1; the last: past the list's end
    n = sum(new)
    rows = torch.randn(n + 5, heads, dim, device=cuda).bfloat16()
    before, slots = pool_bits(c), slot_bytes(c)
    starts = i32(starts_of(new), cuda)
    for b in range(len(lengths)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        one = i32([0, new[b]], cuda)
        C.write_kv(rows[:new[b]], rows[:new[b]], c.table, c.kv, c.stores, ids[b:b + 1], i32(lengths[b:b + 1], cuda), one, status=status)
        assert int(status) == N.FLAG_INDEX_RANGE
        status.zero_()
        k, v = C.read_kv(c.table, c.kv, c.stores, ids[b:b + 1], i32(lengths[b:b + 1], cuda), one, new[b], status=status)
        assert int(status) == N.FLAG_INDEX_RANGE and not k.any() and not v.any()
    C.write_kv(rows, rows, c.table, c.kv, c.stores, ids, i32(lengths, cuda), starts)
    out = torch.full((n + 5, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda), \
        torch.full((n + 5, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda)
    C.read_kv(c.table, c.kv, c.stores, ids, i32(lengths, cuda), starts, n + 5, out=out)
    for x in out:
        assert not x[:n].any() and (x[n:] == 7.0).all()
    # a dithered page takes no single tokens
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    C.write_kv(rows[:2], rows[:2], c.table, c.kv, c.stores, i32([[3]], cuda), i32([5], cuda), i32([0, 2], cuda), status=status)
    assert int(status) == N.FLAG_INDEX_RANGE
    for got, want in zip(pool_bits(c), before):
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
    check_stores(c, slots, {t: np.zeros(s.shape, bool) for t, s in slots.items()})


def test_odd_starts(cuda):
    """Rows before the first start belong to nobody; more rows than tokens are flagged, as are starts that fall."""
    T, heads, dim = 16, 2, 64
    c = Cache(cuda, [N.PAGE_BF16] * 4, T, heads, dim, 10)
    ids, lengths = i32([[0, 1], [2, 3]], cuda), i32([20, 2], cuda)
    out = torch.full((10, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda), \
        torch.full((10, heads, dim), 7.0, dtype=torch.bfloat16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    C.read_kv(c.table, c.kv, None, ids, lengths, i32([3, 5, 9], cuda), 10, out=out, status=status)
    k = out[0].cpu()
    assert (k[:3] == 7.0).all() and (k[9:] == 7.0).all()
    want = torch.from_numpy(page_bits_of(c, 1)[0, 2:4].view(np.int16)).view(torch.bfloat16)
    assert torch.equal(k[3:5].flatten(1), want)
    assert not k[5:7].any() and int(status) == N.FLAG_INDEX_RANGE  # tokens -2 and -1 of the second
    status.zero_()
    C.read_kv(c.table, c.kv, None, ids, lengths, i32([0, 6, 2], cuda), 10, out=out, status=status)
    assert int(status) in (0, N.FLAG_INDEX_RANGE)


def test_slots_beyond_32_bits(cuda):
    T, heads, dim = 16, 8, 128
    c = Cache(cuda, [N.PAGE_INT8] * 2, T, heads, dim, 11)
    need = N.page_slot_bytes(N.PAGE_INT8, T, heads * dim)
    n = (1 << 32) // need + 4
    store = TierStore(N.PAGE_INT8, n, cuda, T, heads * dim)
    c.table.slot.copy_(i32([n - 1, n - 2], cuda))
    stores = {1: store}
    k, v = new_rows(20, heads, dim, cuda, 11)
    args = (c.table, c.kv, stores, i32([[0, 1]], cuda), i32([20], cuda), i32([0, 20], cuda))
    C.write_kv(k, v, *args)
    gk, gv = C.read_kv(*args, 20)
    for got, want in ((gk, k), (gv, v)):
        top = want.float().abs().amax((1, 2), keepdim=True)
        # half a code of the scale (fp16: 2^-11 of it), then a rounding to bf16
        assert ((got.float() - want.float()).abs() <= top * (0.5 / 127 + 2.0 ** -10) + want.float().abs() * 2.0 ** -8).all()


def test_streams_and_graphs(cuda):
    """On a stream of its own, then captured: a graph replays with new rows, lengths, starts and pages in place."""
    T, heads, dim = 16, 8, 128
    c = Cache(cuda, [N.PAGE_INT8, N.PAGE_BF16] * 4, T, heads, dim, 12)
    ids, lengths = i32(np.arange(8).reshape(2, 4), cuda), i32([20, 33], cuda)
    starts = i32([0, 3, 5], cuda)
    k, v = new_rows(8, heads, dim, cuda, 12)
    k, v = k.contiguous(), v.contiguous()
    out = torch.zeros_like(k), torch.zeros_like(v)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))

    def body():
        C.write_kv(k, v, c.table, c.kv, c.stores, ids, lengths, starts)
        C.read_kv(c.table, c.kv, c.stores, ids, lengths, starts, 8, out=out)

    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream(cuda).wait_stream(side)
    idn = ids.cpu().numpy()
    check_read(c, [20, 33], [3, 2], idn, out[0][:5], out[1][:5])
    graph = StepGraph(body, cuda)
    for length, new in (([1, 64], [1, 7]), ([30, 5], [0, 5])):
        lengths.copy_(i32(length, cuda))
        starts.copy_(i32(starts_of(new), cuda))
        k.normal_()
        graph.replay()
        torch.cuda.synchronize()
        m = sum(new)
        check_read(c, length, new, idn, out[0][:m], out[1][:m])
        got = C.read_kv(c.table, c.kv, c.stores, ids, lengths, starts, m)
        assert torch.equal(got[0], out[0][:m]) and torch.equal(got[1], out[1][:m])


def test_nothing_to_do(cuda):
    c = Cache(cuda, [N.PAGE_BF16], 16, 2, 64)
    none = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    C.write_kv(none, none, c.table, c.kv, None, i32([[0]], cuda), i32([3], cuda), i32([0, 0], cuda))
    assert C.read_kv(c.table, c.kv, None, i32([[0]], cuda), i32([3], cuda), i32([0, 0], cuda), 0)[0].shape == (0, 2, 64)
    empty = torch.zeros(0, 4, dtype=torch.int32, device=cuda)
    C.write_kv(none, none, c.table, c.kv, None, empty, i32([], cuda), i32([0], cuda))


def test_refusals(cuda):
    T, heads, dim = 16, 2, 64
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8], T, heads, dim, 13)
    k = torch.zeros(3, heads, dim, dtype=torch.bfloat16, device=cuda)
    ids, lengths, starts = i32([[0, 1]], cuda), i32([20], cuda), i32([0, 3], cuda)

    def write(k=k, v=k, ids=ids, lengths=lengths, starts=starts, stores=c.stores, **more):
        C.write_kv(k, v, c.table, c.kv, stores, ids, lengths, starts, **more)

    def read(ids=ids, lengths=lengths, starts=starts, n=3, **more):
        C.read_kv(c.table, c.kv, c.stores, ids, lengths, starts, n, **more)

    write(), read()
    wide = torch.zeros(3, heads, 2 * dim, dtype=torch.bfloat16, device=cuda)
    for bad in (dict(k=k.float()), dict(k=k.cpu()), dict(v=k[:2]), dict(k=wide), dict(k=wide[..., ::2]), dict(k=k[0]),
                dict(starts=starts[:1]), dict(starts=starts.long()), dict(lengths=lengths.long()), dict(ids=ids.long()),
                dict(ids=ids[0]), dict(starts=starts.cpu()), dict(status=torch.zeros(2, dtype=torch.int32, device=cuda)),
                dict(tokens_per_page=0), dict(k=k.half())):
        with pytest.raises((ValueError, TypeError)):
            write(**bad)
    for bad in (dict(n=-1), dict(starts=starts[:1]), dict(out=(k, k[:2])), dict(out=(k.float(), k)), dict(ids=ids.cpu()),
                dict(out=(torch.zeros(3 * heads * dim + 1, dtype=torch.bfloat16, device=cuda)[1:].view(3, heads, dim), k))):
        with pytest.raises((ValueError, TypeError)):
            read(**bad)
    with pytest.raises(N.KernelError):
        write(tokens_per_page=8)  # the store holds pages of 16
