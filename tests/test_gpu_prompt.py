"""GPU tests of the attention of prompts over tiered pages, against float64.

Pages count as the bf16 values that the oracle's page decoders give.  Tolerances, from the arithmetic.
With u = 2^-24, size = max_t |scale| sum_d |q_d k_d| over the tokens that a row sees:
  a score is an fp32 sum of dim exact products on the tensor cores, scaled once: the sum may lose a few
      bits of its running value at each of its dim / 16 steps, |ds| <= (dim + 20) * 4 u * size;
  a weight is then off by a factor of 1 + dp, dp = 2 |ds| + 2^-20 (exp2's approximation, the
      difference to the running maximum);
  it is rounded to bf16 once, by at most 2^-8 of it, the sum of the weights takes it unrounded;
  the product accumulates in fp32 over n tokens, losing at most 4 u a step of 16;
  a weight below 2^-126, fp32's smallest normal number, counts as zero (the largest weight of a row is at least 1, and so
      is what the sums are divided by): the result loses at most 2^-126 * sum_t |v|;
  the result is rounded to bf16: 2^-8 of its value.
So |out - exact| <= 2^-8 |exact| + (2^-8 + 2 dp + n u) * sum_t P |v| + 2^-126 sum_t |v|; of lse: ds + 2^-19 + 8 u |lse|."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from oracle.attention import bf16_to_f64
from test_gpu_attention import CAP, FORMATS, TIER, Cache, bits
from test_gpu_cache import i32, new_rows, place, slot_bytes, starts_of

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime import cache as C
from ashkv.runtime.batch import DevicePageTable, KVLayers, StepGraph, TierStore

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def pages_of(c):
    """The bf16 bits that a page decodes to [2, T, row], from the stored bytes; what is read from the device is kept."""
    T, row, pools, slots, known = c.T, c.heads * c.dim, {}, {}, {}

    def page(i):
        if i not in known:
            fmt, (tier, layer, start, slot) = c.formats[i], place(c, i)
            if fmt == N.PAGE_BF16:
                if layer not in pools:
                    pools[layer] = [bits(side[layer]).reshape(-1, row) for side in (c.kv.k, c.kv.v)]
                known[i] = np.stack([x[start:start + T] for x in pools[layer]])
            else:
                if tier not in slots:
                    slots[tier] = slot_bytes(c)[tier]
                known[i] = oracle.page_decode(fmt, slots[tier][slot], T, row, outlier_cap=CAP).reshape(2, T, row)
        return known[i]
    return page


def tokens_of(c, page, ids, n):
    """K and V [2, n, heads, dim] in 64 bits of the first n tokens of a list."""
    pages = [bf16_to_f64(page(int(j))).reshape(2, c.T, c.heads, c.dim) for j in ids[:-(-n // c.T)]]
    if not pages:
        return np.zeros((2, 0, c.heads, c.dim))
    return np.concatenate(pages, 1)[:, :n]


def seen_tokens(n, new, window, sinks):
    p, t = np.arange(n - new, n)[:, None], np.arange(n)[None]
    seen = t <= p
    if window:
        seen &= (t > p - window) | (t < sinks)
    return seen


def reference(c, ids, q, lengths, new, window=0, sinks=0, scale=None, gone=()):
    """q float64 [rows, heads_q, dim] -> out, lse, and reach and size of the tolerances; pages `gone` do not exist."""
    page = pages_of(c)
    rows, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out, reach, lost = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q)
    lse, size = np.full((rows, hq), -np.inf), np.zeros((rows, hq))
    at = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        if not m:
            continue
        kv = tokens_of(c, page, ids[b], n)
        seen = seen_tokens(n, m, window, sinks) & ~np.isin(np.repeat(ids[b], c.T)[:n], gone)
        kv = np.where(seen.any(0)[:, None, None], kv, 0.0)
        x = slice(at, at + m)
        at += m
        for h in range(hq):
            k, v = kv[0][:, h // (hq // c.heads)], kv[1][:, h // (hq // c.heads)]
            s = np.where(seen, scale * (q[x, h] @ k.T), -np.inf)
            top = s.max(-1, keepdims=True, initial=-np.inf)
            p = np.exp(s - np.where(np.isneginf(top), 0.0, top))
            with np.errstate(divide="ignore"):
                lse[x, h] = np.log(p.sum(-1)) + np.where(np.isneginf(top), 0.0, top)[:, 0]
            p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
            out[x, h], reach[x, h] = p @ v, p @ np.abs(v)
            lost[x, h] = 2.0 ** -126 * (seen @ np.abs(v))
            size[x, h] = np.where(seen, abs(scale) * (np.abs(q[x, h]) @ np.abs(k).T), 0).max(-1, initial=0.0)
    return {"out": out, "lse": lse, "reach": reach, "size": size, "lost": lost}


def check(got, lse, want, dim, n):
    out, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    ds = (dim + 20) * 4 * U * want["size"]
    dp = 2 * ds + 2.0 ** -20
    tol = 2.0 ** -8 * np.abs(want["out"]) + (2.0 ** -8 + 2 * dp + n * U)[..., None] * want["reach"] + want["lost"] + 1e-37
    assert np.isfinite(out).all()
    worst = np.max(np.abs(out - want["out"]) / tol) if out.size else 0.0
    assert worst <= 1.0, f"result off by {worst} of its tolerance"
    none = np.isneginf(want["lse"])
    assert (np.isneginf(l) == none).all()
    t = (ds + 2.0 ** -19 + 8 * U * np.abs(want["lse"], where=~none, out=np.zeros_like(l)))[~none]
    assert (np.abs(l[~none] - want["lse"][~none]) <= t).all()


def rows_of(n, hq, dim, seed, dev, shift=0):
    """Queries as a slice of a fused projection."""
    g = torch.Generator().manual_seed(2000 + seed)
    x = (torch.randn(n, (hq + 2) * dim + shift, generator=g) * 2).to(torch.bfloat16).to(dev)
    return x[:, shift:shift + hq * dim].unflatten(1, (hq, dim))


def run(dev, kinds, T, hq, heads, dim, lengths, new, seed, window=0, sinks=0, scale=None, shift=0, junk=False):
    P = max(1, max(-(-x // T) for x in lengths))
    n = len(lengths) * P
    g = np.random.default_rng(seed)
    c = Cache(dev, [kinds[i] for i in g.integers(0, len(kinds), n)], T, heads, dim, seed)
    ids = g.permutation(n).astype(np.int32).reshape(len(lengths), P)
    given = ids.copy()
    if junk:  # entries of pages that no query sees are not looked at
        for b, (x, m) in enumerate(zip(lengths, new)):
            used = set((np.flatnonzero(seen_tokens(x, m, window, sinks).any(0)) // T).tolist()) if m else set()
            for j in range(P):
                if j not in used:
                    given[b, j] = (-1, n + 7, 2 ** 31 - 1)[j % 3]
    q = rows_of(sum(new), hq, dim, seed, dev, shift)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    args = (c.table, c.kv, c.stores, i32(given, dev), i32(lengths, dev), i32(starts_of(new), dev))
    out, lse = A.prompt_attention(q, *args, tokens_per_page=T, scale=scale, window=window or None, sinks=sinks,
                                  return_lse=True, status=status)
    want = reference(c, ids, q.double().cpu().numpy(), lengths, new, window, sinks, scale)
    assert int(status) == 0
    check(out, lse, want, dim, max(lengths) + 1)
    return c, ids, q, out, lse


def test_smallest(cuda):
    run(cuda, [N.PAGE_BF16], 16, 1, 1, 128, [1], [1], 0)
    run(cuda, [N.PAGE_BF16], 16, 4, 2, 64, [17], [3], 0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,new", [([128], [128]), ([300], [300]), ([260], [5]), ([1000], [600])])
def test_one_sequence(cuda, dim, lengths, new):
    run(cuda, [N.PAGE_BF16], 16, 4, 2, dim, lengths, new, 1)


@pytest.mark.parametrize("tiers", list(FORMATS))
@pytest.mark.parametrize("hq,heads,dim", [(8, 2, 128), (4, 4, 64), (12, 1, 128), (16, 2, 64)])
def test_formats(cuda, tiers, hq, heads, dim):
    run(cuda, FORMATS[tiers], 16, hq, heads, dim, [70, 0, 1, 16, 33, 457], [70, 0, 1, 3, 17, 200], 2)


@pytest.mark.parametrize("tiers", ["bf16", "int8", "mixed", "mixed8"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 17), (64, 0), (127, 3), (128, 128), (129, 200), (300, 140), (5000, 7)])
def test_windows(cuda, tiers, window, sinks):
    run(cuda, FORMATS[tiers], 16, 8, 2, 128, [400, 131, 1, 700], [130, 131, 1, 300], 3, window, sinks, junk=True)


@pytest.mark.parametrize("T,tiers", [(1, "bf16"), (5, "bf16"), (8, "bf16"), (24, "bf16"), (100, "bf16"), (128, "bf16"), (256, "bf16"),
                                     (1000, "bf16"), (2, "int8"), (10, "mixed"), (18, "mixed8"), (40, "fp8"), (126, "int4"),
                                     (64, "nbit2")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 50)])
def test_page_sizes(cuda, T, tiers, window, sinks):
    run(cuda, FORMATS[tiers], T, 4, 2, 128, [300, 5, 129], [200, 5, 7], 4, window, sinks, junk=True)


@pytest.mark.parametrize("hq,heads", [(1, 1), (3, 1), (7, 7), (48, 1), (64, 2), (128, 1), (256, 1), (512, 1), (600, 2)])
@pytest.mark.parametrize("dim,tiers", [(64, "bf16"), (128, "bf16"), (128, "fp8")])
def test_head_layouts(cuda, hq, heads, dim, tiers):
    case = (cuda, FORMATS[tiers], 16, hq, heads, dim, [150, 40, 9], [11, 40, 1], 5, 60, 3)
    if tiers == "fp8" and heads == 7:  # (stores hold rows of 128 .. 2048 values, powers of two)
        with pytest.raises(N.KernelError):
            run(*case)
    else:
        run(*case)


@pytest.mark.parametrize("tiers,n", [("bf16", 200), ("mixed", 200), ("bf16", 1100), ("int8", 1100)])
def test_many_sequences(cuda, tiers, n):
    g = np.random.default_rng(6)
    lengths = g.integers(0, 150 if n < 1000 else 20, n).tolist()
    new = [int(g.integers(0, x + 1)) for x in lengths]
    run(cuda, FORMATS[tiers], 16, 4, 2, 64 if n > 1000 else 128, lengths, new, 6)


@pytest.mark.parametrize("tiers", ["bf16", "int8"])
@pytest.mark.parametrize("lengths,new,window,sinks", [([9000], [3], 0, 0), ([30000], [1], 0, 0), ([5000, 60], [300, 60], 0, 0),
                                                      ([9000, 700], [70, 2], 3000, 500), ([9000], [5], 8000, 0)])
def test_long_contexts(cuda, tiers, lengths, new, window, sinks):
    """Few rows over many tokens: cut, and joined."""
    run(cuda, FORMATS[tiers], 16, 8, 2, 128, lengths, new, 7, window, sinks)


@pytest.mark.parametrize("pages", [55, 56, 57, 63, 64, 65])
def test_around_the_first_cut(cuda, pages):
    run(cuda, FORMATS["bf16"], 16, 8, 2, 128, [16 * pages, 16 * pages - 15], [3, 20], 29)


@pytest.mark.parametrize("tiers", ["bf16", "int4"])
@pytest.mark.parametrize("shift", [1, 4, 8])
def test_query_alignment(cuda, tiers, shift):
    run(cuda, FORMATS[tiers], 16, 8, 2, 128, [100, 33], [50, 33], 8, shift=shift)


def test_query_strides_and_out(cuda):
    """Queries laid out head by head; results into a given tensor; both streams of heads of one token."""
    c, ids, q, out, lse = run(cuda, FORMATS["mixed"], 16, 8, 2, 64, [100, 33], [50, 33], 9)
    args = (c.table, c.kv, c.stores, i32(ids, cuda), i32([100, 33], cuda), i32([0, 50, 83], cuda))
    by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
    to = torch.full_like(out, 7.0)
    assert A.prompt_attention(by_head, *args, out=to) is to and torch.equal(to, out)
    one = q[:, :1].expand(-1, 8, -1)  # a stride of zero
    assert torch.equal(A.prompt_attention(one, *args), A.prompt_attention(one.contiguous(), *args))
    padded = torch.full((2, 19), 2 ** 30, dtype=torch.int32, device=cuda)
    padded[:, 5:5 + ids.shape[1]] = args[3]
    assert torch.equal(A.prompt_attention(q, *args[:3], padded[:, 5:5 + ids.shape[1]], *args[4:]), out)
    wide = torch.empty(83, 8, 192, dtype=torch.bfloat16, device=cuda)[..., :64].copy_(q)
    assert torch.equal(A.prompt_attention(wide, *args), out)


@pytest.mark.parametrize("tiers", ["bf16", "fp8"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0, 2.0 ** -20])
def test_scales(cuda, tiers, scale):
    run(cuda, FORMATS[tiers], 16, 4, 2, 128, [200, 17], [150, 17], 10, 90, 4, scale=scale)


def poison(c, page, r, kind):
    """A token's K and V that are not finite; kind 0: NaN, 1: infinite, 2: -infinite (where the format has such)."""
    T, row = c.T, c.heads * c.dim
    fmt, (tier, layer, start, slot) = c.formats[page], place(c, page)
    if fmt == N.PAGE_BF16:
        for side in (c.kv.k, c.kv.v):
            side[layer][start + r] = (float("nan"), float("inf"), -float("inf"))[kind]
        return
    s = c.stores[tier]
    data, E = s.data[slot * s.slot_bytes:][:s.slot_bytes], 2 * T * row
    for half in (r, T + r):
        if fmt == N.PAGE_INT8:
            data[2 * half:2 * half + 2].view(torch.int16).fill_((0x7E00, 0x7C00, -1024)[kind])
        elif fmt == N.PAGE_FP8:
            data[half * row:(half + 1) * row].fill_((0x7F, 0xFF, 0x7F)[kind])
        elif fmt == N.PAGE_INT4:
            data[half * row // 32:(half + 1) * row // 32].view(torch.int16).fill_((0x7FC0, 0x7F80, -128)[kind])
        else:
            data[16 + half * row // 16:16 + (half + 1) * row // 16].view(torch.int16).fill_((0x7FC0, 0x7F80, -128)[kind])


@pytest.mark.parametrize("fmt", [N.PAGE_BF16, N.PAGE_FP8, N.PAGE_INT8, N.PAGE_INT4, N.PAGE_NBIT4, N.PAGE_NBIT2])
@pytest.mark.parametrize("hq,dim,T", [(4, 128, 16), (24, 64, 16), (4, 128, 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_hidden_tokens_may_hold_anything(cuda, fmt, hq, dim, T, window, sinks):
    """A row that sees no NaN and no infinity is what it is without them; one that sees some is not finite."""
    heads, length, new = 2, 300, 290
    c = Cache(cuda, [fmt] * (-(-length // T)), T, heads, dim, 11)
    ids = np.random.default_rng(11).permutation(len(c.formats)).astype(np.int32)[None]
    q = rows_of(new, hq, dim, 11, cuda)
    want = reference(c, ids, q.double().cpu().numpy(), [length], [new], window, sinks)
    at = [250, 131, 139, 288] if not window else [150, 151, 220, 288]
    for i, t in enumerate(at + list(range(length, len(c.formats) * T))):
        poison(c, int(ids[0, t // T]), t % T, i % 3)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = A.prompt_attention(q, c.table, c.kv, c.stores, i32(ids, cuda), i32([length], cuda), i32([0, new], cuda),
                                  tokens_per_page=T, window=window or None, sinks=sinks, return_lse=True, status=status)
    hit = seen_tokens(length, new, window, sinks)[:, at].any(1)
    assert int(status) == 0 and hit.any() and not hit.all()
    assert not torch.isfinite(out[torch.from_numpy(hit).to(cuda)]).all(-1).any()
    clean = torch.from_numpy(~hit).to(cuda)
    check(out[clean], lse[clean], {k: v[~hit] for k, v in want.items()}, dim, length + 1)


def test_one_infinite_value_comes_through(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 2, 16, 1, 64, 12)
    args = (c.table, c.kv, None, i32([[0, 1]], cuda), i32([32], cuda), i32([0, 20], cuda))
    q = rows_of(20, 2, 64, 12, cuda)
    l, s = int(c.table.layer[0]), int(c.table.token_start[0])
    c.kv.v[l][s + 15, 0, 5] = float("nan")  # position 15; the rows are at 12 .. 31
    out = A.prompt_attention(q, *args)
    assert torch.isnan(out[3:, :, 5]).all() and torch.isfinite(out[:, :, :5]).all() and torch.isfinite(out[:3]).all()
    c.kv.k[l][s:s + 16] = -float("inf")
    one = torch.ones_like(q)
    out, lse = A.prompt_attention(one, *args, return_lse=True)
    assert (out[:3] == 0).all() and torch.isneginf(lse[:4]).all()  # (position 15 sees a NaN, by a weight of zero)


def test_bad_pages_count_only_where_seen(cuda):
    for fmt, T in ((N.PAGE_BF16, 16), (N.PAGE_BF16, 4), (N.PAGE_INT8, 16)):
        c = Cache(cuda, [fmt] * 20, T, 2, 128, 13)
        n, new = 20 * T - 3, 10
        ids = np.random.default_rng(13).permutation(20).astype(np.int32)[None]
        q = rows_of(new, 4, 128, 13, cuda)
        seen = seen_tokens(n, new, 2 * T + 5, 2).any(0)
        for j in range(20):
            for bad in (-1, 20, 2 ** 31 - 1) if j in (0, 19) else (99,):
                given = ids.copy()
                given[0, j] = bad
                status = torch.zeros(1, dtype=torch.int32, device=cuda)
                out, lse = A.prompt_attention(q, c.table, c.kv, c.stores, i32(given, cuda), i32([n], cuda), i32([0, new], cuda),
                                              tokens_per_page=T, window=2 * T + 5, sinks=2, return_lse=True, status=status)
                assert bool(int(status)) == bool(seen[j * T:(j + 1) * T].any())
                want = reference(c, ids, q.double().cpu().numpy(), [n], [new], 2 * T + 5, 2, gone=[ids[0, j]])
                check(out, lse, want, 128, n)


def test_bad_entries_of_the_table(cuda):
    """A page whose tier, layer, rows or slot do not exist counts as absent, and is flagged."""
    for column, value in (("tier", 6), ("tier", -1), ("tier", 3), ("layer", 2), ("layer", -1), ("token_start", -16),
                          ("token_start", 16 * 9 - 15), ("slot", 9), ("slot", -1)):
        for kinds in ([N.PAGE_BF16], [N.PAGE_INT8]):
            if (column in ("layer", "token_start")) != (kinds == [N.PAGE_BF16]) and column != "tier":
                continue
            c = Cache(cuda, kinds * 9, 16, 2, 128, 14)
            ids = np.arange(9, dtype=np.int32)[None]
            q = rows_of(30, 4, 128, 14, cuda)
            want = reference(c, ids, q.double().cpu().numpy(), [140], [30], gone=[3])
            getattr(c.table, column)[3] = value
            status = torch.zeros(1, dtype=torch.int32, device=cuda)
            out, lse = A.prompt_attention(q, c.table, c.kv, c.stores, i32(ids, cuda), i32([140], cuda), i32([0, 30], cuda),
                                          return_lse=True, status=status)
            assert int(status) & N.FLAG_INDEX_RANGE
            check(out, lse, want, 128, 140)


@pytest.mark.parametrize("kinds", [[N.PAGE_BF16], [N.PAGE_INT8]])
def test_rows_of_no_sequence(cuda, kinds):
    """Rows before the first start and behind the last are left as they were, whatever they hold."""
    c = Cache(cuda, kinds * 6, 16, 2, 128, 15)
    ids = np.arange(6, dtype=np.int32).reshape(2, 3)
    q = rows_of(300, 4, 128, 15, cuda).clone()
    q[:3], q[3 + 25:] = float("nan"), float("inf")
    out = torch.full((300, 4, 128), 5.0, dtype=torch.bfloat16, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, lse = A.prompt_attention(q, c.table, c.kv, c.stores, i32(ids, cuda), i32([40, 30], cuda), i32([3, 23, 28], cuda), out=out,
                                  return_lse=True, status=status)
    assert int(status) == 0 and (out[:3] == 5).all() and (out[28:] == 5).all()
    want = reference(c, ids, q[3:28].double().cpu().numpy(), [40, 30], [20, 5])
    check(out[3:28], lse[3:28], want, 128, 40)


def test_odd_starts_and_lengths(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 6, 16, 2, 128, 16)
    ids, q = np.arange(6, dtype=np.int32).reshape(2, 3), rows_of(40, 4, 128, 16, cuda)

    def call(lengths, starts):
        out = torch.full((40, 4, 128), 5.0, dtype=torch.bfloat16, device=cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        out, lse = A.prompt_attention(q, c.table, c.kv, None, i32(ids, cuda), i32(lengths, cuda), i32(starts, cuda), out=out,
                                      return_lse=True, status=status)
        return out, lse, int(status)

    for starts in ([0, 20, 10], [-4, 10, 20], [0, 10, 41], [30, 20, 10], [0, 2 ** 31 - 1, 5]):
        out, _, status = call([40, 40], starts)
        assert status & N.FLAG_INDEX_RANGE and (out == 5).all(), starts
    # more new tokens than a sequence has: those that do not exist have none before them
    out, lse, status = call([10, 20], [0, 15, 20])
    assert status & N.FLAG_INDEX_RANGE
    assert (out[:5] == 0).all() and torch.isneginf(lse[:5]).all()
    want = reference(c, ids, q[5:20].double().cpu().numpy(), [10, 20], [10, 5])
    check(out[5:20], lse[5:20], want, 128, 20)
    # a length beyond the list, or below zero
    out, _, status = call([60, 20], [0, 15, 20])
    assert status & N.FLAG_INDEX_RANGE and torch.isfinite(out).all()
    out, _, status = call([-1, 20], [0, 0, 5])
    assert status & N.FLAG_INDEX_RANGE
    want = reference(c, ids[1:], q[:5].double().cpu().numpy(), [20], [5])
    check(out[:5], call([0, 20], [0, 0, 5])[1][:5], want, 128, 20)


@pytest.mark.parametrize("tiers", list(FORMATS))
@pytest.mark.parametrize("std", [2.0 ** -12, 1.0, 300.0])
@pytest.mark.parametrize("T", [16, 4])
def test_a_token_that_sees_itself_alone_gives_its_values(cuda, tiers, std, T):
    """A weight of one: the decoded bf16 values, bit by bit what a dense read gives."""
    n = 64
    c = Cache(cuda, [FORMATS[tiers][i % len(FORMATS[tiers])] for i in range(n)], T, 4, 128, 27, std=std)
    ids = i32(np.random.default_rng(27).permutation(n)[None], cuda)
    args = (c.table, c.kv, c.stores, ids, i32([n * T], cuda), i32([0, n * T], cuda))
    out = A.prompt_attention(rows_of(n * T, 8, 128, 27, cuda), *args, tokens_per_page=T, window=1, scale=2.0 ** -12)
    keys, values = C.read_kv(*args, n * T, tokens_per_page=T)
    finite = torch.isfinite(keys).all(-1) & torch.isfinite(values).all(-1)  # (FP8 pages hold NaN for values beyond 448)
    assert finite.any() or std > 1
    for h in range(8):
        ok = finite[:, h // 2]
        assert torch.equal(out[ok, h], values[ok, h // 2])


@pytest.mark.parametrize("std,scale", [(2.0 ** 90, 2.0 ** -95), (2.0 ** -100, 1.0), (2.0 ** -60, 2.0 ** 55)])
def test_value_ranges(cuda, std, scale):
    c = Cache(cuda, [N.PAGE_BF16] * 20, 16, 2, 128, 28, std=std)
    ids = np.arange(20, dtype=np.int32)[None]
    q = rows_of(300, 8, 128, 28, cuda)
    out, lse = A.prompt_attention(q, c.table, c.kv, None, i32(ids, cuda), i32([311], cuda), i32([0, 300], cuda), scale=scale,
                                  return_lse=True)
    check(out, lse, reference(c, ids, q.double().cpu().numpy(), [311], [300], scale=scale), 128, 312)


def test_pages_shared_and_listed_twice(cuda):
    c = Cache(cuda, FORMATS["mixed"] * 2, 16, 2, 128, 17)
    ids = np.array([[3, 1, 3, 3, 0], [1, 1, 3, 2, 2]], np.int32)
    q = rows_of(60, 4, 128, 17, cuda)
    out, lse = A.prompt_attention(q, c.table, c.kv, c.stores, i32(ids, cuda), i32([80, 70], cuda), i32([0, 40, 60], cuda),
                                  return_lse=True)
    check(out, lse, reference(c, ids, q.double().cpu().numpy(), [80, 70], [40, 20]), 128, 80)


def test_offsets_beyond_32_bits(cuda):
    """Pool rows and slots more than 2^32 bytes from their base, all in the pool and not."""
    T, heads, dim = 16, 8, 128
    tokens = (1 << 32) // (heads * dim * 2) + 4 * T
    k = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=cuda)
    v = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=cuda)
    c = Cache(cuda, [N.PAGE_BF16, N.PAGE_INT8], T, heads, dim, 18, layers=1)
    far, old = tokens - T, place(c, 0)[2]
    k[far:], v[far:] = c.kv.k[0][old:old + T], c.kv.v[0][old:old + T]
    need = c.stores[1].slot_bytes
    n_slots, slot = (1 << 32) // need + 3, place(c, 1)[3]
    store = TierStore(N.PAGE_INT8, n_slots, cuda, T, heads * dim)
    store.data[(n_slots - 1) * need:n_slots * need].copy_(c.stores[1].data[slot * need:(slot + 1) * need])
    q, ids = rows_of(20, 16, dim, 18, cuda), np.array([[0, 1]], np.int32)
    want = reference(c, ids, q.double().cpu().numpy(), [30], [20])
    c.table.token_start[0], c.table.slot[1] = far, n_slots - 1
    kv = KVLayers([k], [v])
    out, lse = A.prompt_attention(q, c.table, kv, {1: store}, i32(ids, cuda), i32([30], cuda), i32([0, 20], cuda), return_lse=True)
    check(out, lse, want, dim, 30)
    c.table.token_start[1] = far
    c.table.tier[1] = 0
    args = (c.table, kv, None, i32([[1, 0]], cuda), i32([30], cuda), i32([0, 20], cuda))
    out, lse = A.prompt_attention(q, *args, return_lse=True)
    c.table.token_start.fill_(old)
    near = A.prompt_attention(q, c.table, c.kv, *args[2:], return_lse=True)
    assert torch.equal(out, near[0]) and torch.equal(lse, near[1])


@pytest.mark.parametrize("tiers", ["bf16", "mixed"])
def test_streams_and_graphs(cuda, tiers):
    """On a stream of its own, then captured twice: replays with new queries, lengths, starts and pages in place."""
    c = Cache(cuda, [k for k in FORMATS[tiers] for _ in range(24 // len(FORMATS[tiers]))], 16, 2, 128, 19)
    ids = i32(np.random.default_rng(19).permutation(24).reshape(2, 12), cuda)
    lengths, starts, q = i32([100, 40], cuda), i32([0, 60, 100], cuda), rows_of(100, 8, 128, 19, cuda)
    outs = [torch.zeros(100, 8, 128, dtype=torch.bfloat16, device=cuda) for _ in range(2)]

    def body(i, window):
        return lambda: A.prompt_attention(q, c.table, c.kv, c.stores, ids, lengths, starts, window=window, out=outs[i])

    def expect(n, m, window, out):
        lse = A.prompt_attention(q, c.table, c.kv, c.stores, ids, lengths, starts, window=window, return_lse=True)[1]
        rows = sum(m)
        want = reference(c, ids.cpu().numpy(), q[:rows].double().cpu().numpy(), n, m, window or 0)
        check(out[:rows], lse[:rows], want, 128, 192)

    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        body(0, None)()
    torch.cuda.current_stream(cuda).wait_stream(side)
    expect([100, 40], [60, 40], None, outs[0])
    graphs = [StepGraph(body(0, None), cuda), StepGraph(body(1, 33), cuda)]
    for n, m in (([1, 192], [1, 99]), ([30, 5], [0, 5]), ([150, 90], [50, 50])):
        lengths.copy_(i32(n, cuda))
        starts.copy_(i32(starts_of(m), cuda))
        q.normal_()
        ids.copy_(ids.flip(1))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        expect(n, m, None, outs[0])
        expect(n, m, 33, outs[1])


def test_two_streams_at_once(cuda):
    """Calls that run at the same time share nothing."""
    c = Cache(cuda, FORMATS["mixed"] * 40, 16, 2, 128, 20)
    ids, n = i32(np.arange(160).reshape(2, 80), cuda), 1200
    q = [rows_of(n, 8, 128, s, cuda) for s in (20, 21)]
    args = (c.table, c.kv, c.stores, ids, i32([1280, 1200], cuda), i32([0, 700, n], cuda))
    want = [A.prompt_attention(x, *args) for x in q]
    streams = [torch.cuda.Stream(cuda) for _ in q]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, s in zip(q, streams):
            with torch.cuda.stream(s):
                got.append(A.prompt_attention(x, *args))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("tiers", ["bf16", "mixed"])
def test_results_do_not_depend_on_the_run(cuda, tiers):
    """Bit by bit the same, cut items and the order of the pieces included."""
    c = Cache(cuda, FORMATS[tiers] * (600 // len(FORMATS[tiers])), 16, 2, 128, 22)
    ids = i32(np.random.default_rng(22).permutation(600).reshape(2, 300), cuda)
    q = rows_of(410, 8, 128, 22, cuda)
    args = (c.table, c.kv, c.stores, ids, i32([4800, 900], cuda), i32([0, 10, 410], cuda))
    want = A.prompt_attention(q, *args, return_lse=True)
    for _ in range(10):
        got = A.prompt_attention(q, *args, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kinds", [[N.PAGE_BF16], [N.PAGE_INT8], [N.PAGE_BF16, N.PAGE_FP8, N.PAGE_INT4]])
@pytest.mark.parametrize("dim,heads", [(128, 2), (64, 8)])
def test_a_run_together(cuda, kinds, dim, heads):
    """Chunks of prompts and then single tokens, as a server steps: written, attended, read back, in one stream without a wait."""
    T, hq, P, window, sinks = 16, 4 * heads, 40, 100, 4
    c = Cache(cuda, [kinds[i % len(kinds)] for i in range(3 * P)], T, heads, dim, 23)
    ids = np.random.default_rng(23).permutation(3 * P).astype(np.int32).reshape(3, P)
    idt, lengths = i32(ids, cuda), np.zeros(3, int)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    steps = [[300, 0, 17], [130, 260, 1], [1, 1, 1], [1, 1, 1], [5, 3, 2], [1, 0, 64], [1, 1, 1]]
    seen = []
    for i, new in enumerate(steps):
        lengths += new
        n = sum(new)
        k, v = new_rows(n, heads, dim, cuda, 100 + i)
        q = rows_of(n, hq, dim, 200 + i, cuda)
        at = (c.table, c.kv, c.stores, idt, i32(lengths, cuda), i32(starts_of(new), cuda))
        C.write_kv(k, v, *at, status=status)
        full = A.prompt_attention(q, *at, return_lse=True, status=status)
        part = A.prompt_attention(q, *at, window=window, sinks=sinks, return_lse=True, status=status)
        one = A.decode_attention(q, *at[:5], window=window, sinks=sinks, status=status) if new == [1, 1, 1] else None
        back = C.read_kv(*at, n, status=status)
        seen.append((list(lengths), new, q, k, v, full, part, one, back))
    assert int(status) == 0
    # (later steps write later tokens only, so the pages as they are now hold what every step saw)
    for lens, new, q, k, v, full, part, one, back in seen:
        q64 = q.double().cpu().numpy()
        check(*full, reference(c, ids, q64, lens, new), dim, max(lens) + 1)
        want = reference(c, ids, q64, lens, new, window, sinks)
        check(*part, want, dim, max(lens) + 1)
        if one is not None:
            # decode counts the numbers that the codes stand for, a prompt their bf16 roundings: 2^-8 of each value, and of each
            # key, which moves a score by 2^-8 of its size and a weight by a factor of exp of that
            dp = np.expm1(2 * (2.0 ** -8 + (dim + 20) * 4 * U) * want["size"])[..., None]
            bound = 2.0 ** -8 * np.abs(want["out"]) + (2.0 ** -7 + dp) * want["reach"] + want["lost"]
            assert (np.abs(one.double().cpu().numpy() - want["out"]) <= bound).all()
        at = 0
        page = pages_of(c)
        for b, (n, m) in enumerate(zip(lens, new)):
            kv = tokens_of(c, page, ids[b], n)[:, n - m:]
            for got, w in zip(back, kv):
                assert np.array_equal(got[at:at + m].double().cpu().numpy(), w)
            at += m


def test_inputs_written_by_the_kernel_before(cuda):
    """Launches that begin before the one ahead has ended see what it wrote: queries, lists, lengths and starts."""
    c = Cache(cuda, FORMATS["mixed"] * 6, 16, 2, 128, 24)
    q0, ids0 = rows_of(200, 4, 128, 24, cuda).contiguous(), i32(np.arange(24).reshape(2, 12), cuda)
    L0, s0 = i32([190, 130], cuda), i32([0, 100, 200], cuda)
    want = A.prompt_attention(q0, c.table, c.kv, c.stores, ids0, L0, s0)
    q, ids, L, s = torch.zeros_like(q0), torch.zeros_like(ids0), torch.zeros_like(L0), torch.zeros_like(s0)
    for _ in range(20):
        for x in (q, ids, L, s):
            x.zero_()
        A.prompt_attention(q, c.table, c.kv, c.stores, ids, L, s)
        for x, y in ((q, q0), (ids, ids0), (L, L0), (s, s0)):
            x.copy_(y)
        assert torch.equal(A.prompt_attention(q, c.table, c.kv, c.stores, ids, L, s), want)


def test_nothing_to_do(cuda):
    c = Cache(cuda, [N.PAGE_BF16], 16, 2, 64, 25)
    q = rows_of(3, 4, 64, 25, cuda)
    none, one = i32(np.zeros((0, 1)), cuda), i32([[0]], cuda)
    out = torch.full((3, 4, 64), 5.0, dtype=torch.bfloat16, device=cuda)
    A.prompt_attention(q, c.table, c.kv, None, none, i32([], cuda), i32([0], cuda), out=out)
    A.prompt_attention(q, c.table, c.kv, None, one, i32([9], cuda), i32([1, 1], cuda), out=out)
    assert (out == 5).all()
    assert A.prompt_attention(q[:0], c.table, c.kv, None, one, i32([9], cuda), i32([0, 0], cuda)).shape == (0, 4, 64)
    out, lse = A.prompt_attention(q, c.table, c.kv, None, one, i32([0], cuda), i32([0, 3], cuda), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_refusals(cuda):
    c = Cache(cuda, [N.PAGE_BF16] * 2, 16, 2, 64, 26)
    q = rows_of(3, 4, 64, 26, cuda)
    good = dict(q=q, table=c.table, kv=c.kv, stores=None, page_ids=i32([[0, 1]], cuda), lengths=i32([20], cuda),
                starts=i32([0, 3], cuda))
    A.prompt_attention(**good)
    cpu = i32([0, 3], "cpu")
    for bad in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[..., ::2]), dict(q=q[0]), dict(q=q.cpu()),
                dict(window=0), dict(window=-2), dict(sinks=3), dict(window=4, sinks=-1), dict(window=2 ** 31),
                dict(starts=i32([0], cuda)), dict(starts=cpu), dict(starts=torch.tensor([0, 3], device=cuda)),
                dict(lengths=i32([20, 20], cuda)), dict(lengths=torch.tensor([20], device=cuda)),
                dict(page_ids=i32([0, 1], cuda)), dict(page_ids=torch.tensor([[0, 1]], device=cuda)),
                dict(out=q), dict(out=torch.empty(3, 4, 64, device=cuda)), dict(out=q.new_empty(4, 4, 64)),
                dict(out=q.new_empty(3 * 4 * 64 + 1)[1:].view(3, 4, 64)), dict(status=torch.zeros(1, device=cuda)),
                dict(tokens_per_page=0)):
        with pytest.raises((TypeError, ValueError, N.KernelError)):
            A.prompt_attention(**{**good, **bad})
