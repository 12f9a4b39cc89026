"""GPU tests of a decode step with a sliding window and first tokens that stay visible, against float64.

The oracle attends the visible tokens one by one (pages of one token); tolerances are those of
test_gpu_attention.check, which hold for any list of tokens."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as O
from test_gpu_attention import FORMATS, TIER, Cache, check, queries

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime.batch import StepGraph

pytestmark = pytest.mark.gpu


def i32(x, dev):
    return torch.as_tensor(np.asarray(x, np.int32)).to(dev)


def visible(n, window, sinks):
    return [t for t in range(n) if t < sinks or t >= n - window]


def reference(c, ids, q, lengths, window, sinks, acc, decay, scale=None):
    lists = []
    for b, n in enumerate(lengths):
        tokens = []
        for t in visible(n, window, sinks):
            K, V = c.values[ids[b][t // c.T]]
            r = t % c.T
            tokens.append((t, (K[r:r + 1], V[r:r + 1])))
        lists.append([tokens] * c.heads)
    scale = c.dim ** -0.5 if scale is None else scale
    want = O.decode_attention(q, lists, lengths, 1, scale, np.zeros((len(lengths), max(1, max(lengths)))), 1.0)
    mass = acc.astype(np.float64).copy()
    for b, n in enumerate(lengths):
        for j in range(-(-n // c.T)):
            mass[b, j] = decay * acc[b, j] + want["mass"][b, j * c.T:min(n, (j + 1) * c.T)].sum()
    want["mass"] = mass
    return want


def run(dev, kinds, T, heads_q, heads, dim, lengths, window, sinks, seed, decay=0.75, junk=True):
    P = max(1, max(-(-x // T) for x in lengths))
    n = len(lengths) * P
    g = np.random.default_rng(seed)
    c = Cache(dev, [kinds[i] for i in g.integers(0, len(kinds), n)], T, heads, dim, seed)
    ids = g.permutation(n).astype(np.int32).reshape(len(lengths), P)
    q = queries(len(lengths), heads_q, dim, seed, 2.0)
    acc = g.random((len(lengths), P), dtype=np.float32)
    given = ids.copy()
    if junk:  # the entries of pages without a visible token are not looked at
        for b, m in enumerate(lengths):
            used = {t // T for t in visible(m, window, sinks)}
            for j in range(P):
                if j not in used:
                    given[b, j] = (-1, n + 7, 2 ** 31 - 1)[j % 3]
    mass = torch.from_numpy(acc.copy()).to(dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    args = (q.to(dev), c.table, c.kv, c.stores, i32(given, dev), i32(lengths, dev))
    out, lse = A.decode_attention(*args, tokens_per_page=T, window=window, sinks=sinks, page_mass=mass, decay=decay,
                                  return_lse=True, status=status)
    want = reference(c, ids, q.double().numpy(), lengths, window, sinks, acc, decay)
    assert int(status) == 0
    check(out, lse, want, dim, max(lengths) + 1, mass, acc, decay)
    again = A.decode_attention(*args, tokens_per_page=T, window=window, sinks=sinks)  # without mass
    assert torch.equal(again, out)
    return c, ids, q, out


@pytest.mark.parametrize("tiers", list(FORMATS))
@pytest.mark.parametrize("heads_q,heads,dim", [(8, 2, 128), (4, 4, 64), (12, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 5), (64, 0)])
def test_formats(cuda, tiers, heads_q, heads, dim, window, sinks):
    run(cuda, FORMATS[tiers], 16, heads_q, heads, dim, [70, 0, 1, 16, 33, 257], window, sinks, 1)


@pytest.mark.parametrize("window,sinks", [(1, 1), (1, 16), (16, 17), (15, 1), (17, 31), (100, 100), (48, 200), (300, 0),
                                          (2 ** 31 - 1, 0), (1, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("tiers", ["bf16", "mixed"])
def test_borders(cuda, tiers, window, sinks):
    run(cuda, FORMATS[tiers], 16, 4, 2, 128, [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 49, 64, 150], window, sinks, 2)


@pytest.mark.parametrize("T,tiers", [(1, "bf16"), (5, "bf16"), (24, "bf16"), (1000, "bf16"), (8, "mixed"), (18, "int8"),
                                     (20, "int4"), (40, "mixed8"), (64, "int8"), (64, "nbit4")])
@pytest.mark.parametrize("window,sinks", [(3, 0), (33, 2), (70, 50)])
def test_page_sizes(cuda, T, tiers, window, sinks):
    run(cuda, FORMATS[tiers], T, 4, 2, 128, [1, T, T + 1, 3 * T - 1, 150], window, sinks, 3)


@pytest.mark.parametrize("tiers", ["bf16", "int8", "int4"])
def test_long_and_many(cuda, tiers):
    run(cuda, FORMATS[tiers], 16, 4, 2, 64, [5001], 3000, 100, 4)
    run(cuda, FORMATS[tiers], 16, 4, 2, 64, [(37 * i) % 190 for i in range(150)], 50, 4, 5)


def test_a_wide_window_changes_nothing(cuda):
    c, ids, q, _ = run(cuda, FORMATS["mixed"], 16, 8, 2, 128, [130, 17, 64], 40, 3, 6, junk=False)
    args = (q.to(cuda), c.table, c.kv, c.stores, i32(ids, cuda), i32([130, 17, 64], cuda))
    assert torch.equal(A.decode_attention(*args, window=130), A.decode_attention(*args))


@pytest.mark.parametrize("fmt", [N.PAGE_BF16, N.PAGE_FP8, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT4, N.PAGE_NBIT2])
@pytest.mark.parametrize("heads_q", [4, 24])
def test_hidden_tokens_may_hold_anything(cuda, fmt, heads_q):
    """NaN and infinities in the hidden tokens of pages that are read in part change nothing."""
    T, heads, dim, length, window, sinks = 16, 2, 128, 60, 20, 5
    c = Cache(cuda, [fmt] * 4, T, heads, dim, 7)
    ids, L = i32([[0, 1, 2, 3]], cuda), i32([length], cuda)
    q = queries(1, heads_q, dim, 7).to(cuda)
    want = A.decode_attention(q, c.table, c.kv, c.stores, ids, L, window=window, sinks=sinks, return_lse=True)
    row = heads * dim
    for t in sorted(set(range(64)) - set(visible(length, window, sinks))):
        page, r = t // T, t % T
        bad = (0x7FC0, 0x7F80, 0xFF80)[t % 3]
        if fmt == N.PAGE_BF16:
            layer, at = int(c.table.layer[page]), int(c.table.token_start[page]) + r
            for side in (c.kv.k, c.kv.v):
                side[layer][at].view(torch.int16).fill_(bad - 65536 if bad > 32767 else bad)
            continue
        s = c.stores[TIER[fmt]]
        slot = s.data[int(c.table.slot[page]) * s.slot_bytes:][:s.slot_bytes]
        E = 2 * T * row
        for half in (r, T + r):
            if fmt == N.PAGE_INT8:
                slot[2 * half:2 * half + 2].view(torch.int16).fill_((0x7E00, 0x7C00, -1024)[t % 3])
            elif fmt == N.PAGE_FP8:
                slot[half * row:(half + 1) * row].fill_(0x7F)
            elif fmt == N.PAGE_INT4:
                slot[half * row // 32:(half + 1) * row // 32].view(torch.int16).fill_(0x7FC0)
            else:
                slot[16 + half * row // 16:16 + (half + 1) * row // 16].view(torch.int16).fill_(0x7FC0)
    got = A.decode_attention(q, c.table, c.kv, c.stores, ids, L, window=window, sinks=sinks, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_hidden_outliers_stay_hidden(cuda):
    """The outliers of hidden tokens of a dithered page do not come back over the zeros."""
    run(cuda, [N.PAGE_NBIT4], 16, 8, 8, 128, [59, 90], 17, 3, 8)
    run(cuda, [N.PAGE_NBIT2], 16, 8, 8, 128, [59, 90], 5, 20, 9)


def test_bad_pages_count_only_where_seen(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 8, 16, 2, 64, 10)
    ids = np.arange(8, dtype=np.int32)[None]
    q = queries(1, 4, 64, 10)
    mass = torch.ones(1, 8, device=cuda)
    for j, flagged in ((0, True), (1, False), (4, False), (5, True), (7, True)):
        bad = ids.copy()
        bad[0, j] = 99
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        mass.fill_(1.0)
        A.decode_attention(q.to(cuda), c.table, c.kv, None, i32(bad, cuda), i32([125], cuda), window=40, sinks=2,
                           page_mass=mass, decay=0.5, status=status)
        assert bool(int(status)) == flagged
        assert torch.isfinite(mass).all() and (mass[0, [1, 2, 3, 4]] == 0.5).all() and (not flagged or mass[0, j] == 0.5)


def test_a_window_in_a_graph(cuda):
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8, N.PAGE_INT4] * 8, 16, 2, 128, 11)
    ids = np.random.default_rng(11).permutation(24).astype(np.int32).reshape(2, 12)
    q = queries(2, 8, 128, 11).to(cuda)
    L, acc = i32([100, 5], cuda), np.zeros((2, 12), np.float32)
    mass, out = torch.zeros(2, 12, device=cuda), torch.empty_like(q)
    idt = i32(ids, cuda)
    graph = StepGraph(lambda: A.decode_attention(q, c.table, c.kv, c.stores, idt, L, window=33, sinks=4, page_mass=mass,
                                                 out=out), cuda)
    for lengths in ([1, 192], [50, 0], [34, 33]):
        L.copy_(i32(lengths, cuda))
        mass.zero_()
        graph.replay()
        torch.cuda.synchronize()
        lse = A.decode_attention(q, c.table, c.kv, c.stores, idt, L, window=33, sinks=4, return_lse=True)[1]
        want = reference(c, ids, q.cpu().double().numpy(), lengths, 33, 4, acc, 1.0)
        check(out, lse, want, 128, 200, mass, acc, 1.0)


def test_refusals(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 2, 16, 2, 64, 12)
    q, ids, L = queries(1, 4, 64, 12).to(cuda), i32([[0, 1]], cuda), i32([20], cuda)
    sel, cnt = torch.zeros(1, 2, 1, dtype=torch.int32, device=cuda), torch.ones(1, 2, dtype=torch.int32, device=cuda)
    for bad in (dict(window=0), dict(window=-3), dict(window=2 ** 31), dict(window=4, sinks=-1), dict(sinks=2),
                dict(window=4, sinks=2 ** 31), dict(window=4, selected=sel, selected_count=cnt)):
        with pytest.raises(ValueError):
            A.decode_attention(q, c.table, c.kv, None, ids, L, **bad)
