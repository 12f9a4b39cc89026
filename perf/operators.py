"""The serving operators over tiered KV pages, in their plain form and as calls of the library.

Three groups that work on the pages of one layer of a paged cache (16 tokens a page, rows of
``heads_kv * dim`` values, a page either in the bf16 pool or compressed in its tier's store):

* decode: one new query per sequence attends the sequence's pages wherever their tier keeps them,
  and may add the attention weight that each page drew to a running, decayed mass per page;
* sparse / bounds: 8-bit outward-rounded bounds of the keys of a page, the pages that a query scores
  highest by them, and the same attention over only those pages of each key head;
* evict: the pages of least accumulated mass leave a sequence that is over its budget.

``own`` selects the library's kernels; otherwise elementary torch operations in 32 bits compute the
same from the same inputs.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

T = 16                                        # tokens of a page, as everywhere in this library
BF16, INT8, FP8, INT4, NBIT4, NBIT2 = range(6)  # page formats
TIER_OF = {BF16: 0, INT8: 1, FP8: 1, INT4: 2, NBIT4: 2, NBIT2: 3}
KINDS = {"bf16": [BF16], "int8": [INT8], "fp8": [FP8], "int4": [INT4], "nbit4": [NBIT4],
         "mixed": [BF16, INT8, INT4, NBIT2], "mixed8": [BF16, FP8, NBIT4, NBIT2]}
OUTLIERS, CAP = 96, 128                       # outliers of a dithered page, and the slots' capacity
DECAY = 0.9


def _case(name, kind, seqs, tokens, heads_q, heads_kv, dim, tiers="bf16", ragged=False, mass=False, budget=0,
          sink=1, recent=2):
    return {"name": name, "kind": kind, "seqs": seqs, "tokens": tokens, "heads_q": heads_q, "heads_kv": heads_kv,
            "dim": dim, "tiers": tiers, "ragged": ragged, "mass": mass, "budget": budget, "sink": sink,
            "recent": recent}


def listed():
    return [
        # one short conversation: nothing to read, so the latency of a call counts
        _case("decode-1x257-bf16", "decode", 1, 257, 32, 8, 128),
        # the migration workload's batch, 32 sequences of 8192 tokens, before any page was demoted
        _case("decode-32x8192-bf16", "decode", 32, 8192, 64, 8, 128),
        # the same after demotion to INT8 pages, the mass that feeds the page scores kept up
        _case("decode-32x8192-int8", "decode", 32, 8192, 64, 8, 128, "int8", mass=True),
        # a single long context in INT4 pages, ending inside a page: few rows, one very long axis
        _case("decode-1x131071-int4", "decode", 1, 131071, 32, 8, 128, "int4"),
        # a ragged batch with an idle slot over all four tiers at once
        _case("decode-24-mixed", "decode", 24, 6001, 32, 8, 128, "mixed", ragged=True, mass=True),
        # one rank's two heads of 64 of a batch with FP8 pages
        _case("decode-64-shard-fp8", "decode", 64, 4000, 16, 2, 64, "fp8", ragged=True),
        # one long context, 256 of its pages for each key head
        _case("sparse-1x131072-bf16", "sparse", 1, 131072, 32, 8, 128, budget=256),
        # a ragged batch of long contexts in INT8 pages
        _case("sparse-8x32000-int8", "sparse", 8, 32000, 64, 8, 128, "int8", ragged=True, budget=128, sink=4,
              recent=8),
        # the pages that one step of a batch filled
        _case("bounds-32", "bounds", 1, 32 * T - 5, 8, 8, 128),
        # the pages of a prefill of 32 x 8192 tokens
        _case("bounds-16384", "bounds", 32, 8192, 8, 8, 128),
        # a step of the batch above, a quarter of each sequence leaves
        _case("evict-32x512", "evict", 32, 8192, 8, 8, 128, budget=384),
        # many long sequences at once
        _case("evict-256x8192", "evict", 256, 131072, 8, 8, 128, ragged=True, budget=1024, sink=4, recent=16),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["decode", "decode", "decode", "sparse", "bounds", "evict"])
    heads_q, heads_kv, dim = rng.choice([(32, 8, 128), (64, 8, 128), (8, 8, 64), (16, 2, 64), (8, 1, 128),
                                         (32, 2, 128), (20, 4, 128), (4, 4, 128), (2, 2, 64)])
    row = heads_kv * dim
    if kind == "evict":
        seqs, tokens = size(1, 256), size(1, 131072)
        pages = -(-tokens // T)
        sink, recent = rng.randint(0, 8), rng.randint(1, 16)
        return _case("", kind, seqs, tokens, 8, 8, 128, ragged=rng.random() < 0.7, sink=sink, recent=recent,
                     budget=sink + recent + size(1, max(pages, 2)))
    seqs = size(1, 64)
    most = 262144 * 1024 // max(row, 256) // 2
    tokens = size(1, max(2, min(131072, most // seqs, 262144 // seqs)))
    tiers = rng.choice(["bf16", "int8", "fp8", "int4", "nbit4", "mixed", "mixed8"])
    if kind == "sparse":
        sink, recent = rng.randint(0, 4), rng.randint(1, 8)
        return _case("", kind, seqs, tokens, heads_q, heads_kv, dim, rng.choice(["bf16", "int8", "int4", "mixed"]),
                     ragged=rng.random() < 0.5, sink=sink, recent=recent, budget=sink + recent + size(1, 256))
    return _case("", kind, seqs, tokens, heads_q, heads_kv, dim, "bf16" if kind == "bounds" else tiers,
                 ragged=rng.random() < 0.5, mass=kind == "decode" and rng.random() < 0.5)


# ----------------------------------------------------------------------------- sizes
def _lengths(case):
    """Tokens of each sequence: all alike, or spread over 5 % to 100 % with one idle slot in eight or more."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["tokens"]] * n
    got = [max(1, round(case["tokens"] * (0.05 + 0.95 * ((i * 0.6180339887) % 1.0)))) for i in range(n)]
    got[n // 3] = case["tokens"]
    if n >= 8:
        got[n // 2] = 0
    return got


def _formats(case):
    """Format of every page position [seqs, pages]: the tiers in turn, the page being filled in bf16."""
    lens = _lengths(case)
    P = max(1, max(-(-n // T) for n in lens))
    kinds = np.asarray(KINDS[case["tiers"]])
    k = np.arange(case["seqs"] * P, dtype=np.int64)
    fmt = kinds[((k * 2654435761) >> 7) % len(kinds)].reshape(case["seqs"], P)
    for b, n in enumerate(lens):
        last = (n - 1) // T
        if n:
            fmt[b, last] = BF16
        fmt[b, last + 1:] = BF16
    return fmt, lens, P


def _page_bytes(fmt, row):
    e = 2 * T * row
    return {BF16: 2 * e, INT8: e + 4 * T, FP8: e, INT4: e // 2 + e // 32,
            NBIT4: 16 + e // 16 + e // 2 + 4 * OUTLIERS, NBIT2: 16 + e // 16 + e // 4 + 4 * OUTLIERS}[fmt]


def _slot_bytes(fmt, row):
    e = 2 * T * row
    used = {INT8: (4 * T + 15) // 16 * 16 + e, FP8: e, INT4: e // 32 + e // 2,
            NBIT4: 16 + e // 16 + e // 2 + 4 * CAP, NBIT2: 16 + e // 16 + e // 4 + 4 * CAP}[fmt]
    return (used + 255) // 256 * 256


def work(case):
    row, hq, hkv, d = case["heads_kv"] * case["dim"], case["heads_q"], case["heads_kv"], case["dim"]
    fmt, lens, P = _formats(case)
    pages = [-(-n // T) for n in lens]
    if case["kind"] == "evict":
        n = sum(pages)
        return {"bytes": 8 * n + 16 * case["seqs"] * P + 12 * case["seqs"], "flops": 0}
    if case["kind"] == "bounds":
        n = sum(pages)
        return {"bytes": sum(lens) * row * 2 + n * (2 * row + hkv + 8), "flops": 0}
    io = case["seqs"] * hq * d * 4 + sum(pages) * 20
    if case["kind"] == "decode":
        got = io + (2 * 4 * sum(pages) if case["mass"] else 0)
        for b, n in enumerate(lens):
            full, rest = divmod(n, T)
            got += sum(_page_bytes(int(f), row) * int((fmt[b, :full] == f).sum()) for f in set(fmt[b, :full].tolist()))
            got += 4 * rest * row
        return {"bytes": got, "flops": 4 * hq * d * sum(lens)}
    kept = [min(p, case["budget"]) for p in pages]
    each = float(np.mean([_page_bytes(int(f), row) for f in fmt.reshape(-1)]))
    return {"bytes": io + sum(pages) * (2 * row + hkv) + sum(kept) * (each + 4 * hkv),
            "flops": 4 * hq * d * T * sum(kept) + 4 * hq * d * sum(pages)}


# ----------------------------------------------------------------------------- inputs
def _encode(fmt, n, row, g):
    """Slots [n, bytes] of compressed pages of roughly normal values, straight from codes and scales."""
    dev, e = g.device, 2 * T * row
    out = torch.zeros(n, _slot_bytes(fmt, row), dtype=torch.uint8, device=dev)
    at = 0

    def put(x):
        nonlocal at
        b = x.contiguous().view(torch.uint8).reshape(n, -1)
        out[:, at:at + b.shape[1]] = b
        at += b.shape[1]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float16)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, device=dev, generator=g) * (hi - lo) + lo

    if fmt == INT8:
        put(uniform(2.5, 4.5, n, 2 * T).half())
        at = (4 * T + 15) // 16 * 16
        put((normal(n, e) * 36).round_().clamp_(-127, 127).to(torch.int8))
    elif fmt == FP8:
        put(normal(n, e).to(torch.float8_e4m3fn))
    elif fmt == INT4:
        put(uniform(1.5, 3.0, n, e // 64).bfloat16())
        q = (normal(n, e) * 2.8).round_().clamp_(-7, 7).to(torch.int8) + 8
        put(((q[:, 0::2] << 4) | q[:, 1::2]).to(torch.uint8))
    else:
        bits = 4 if fmt == NBIT4 else 2
        half = (2 ** bits - 1) / 2
        head = torch.zeros(n, 4, dtype=torch.int32, device=dev)
        head[:, 0] = OUTLIERS
        put(head)
        put((uniform(1.5, 2.5, n, e // 32) / half).bfloat16())
        q = (normal(n, e) * (half / 2) + half).round_().clamp_(0, 2 ** bits - 1).to(torch.uint8)
        per = 8 // bits
        word = torch.zeros(n, e // per, dtype=torch.uint8, device=dev)
        for i in range(per):  # the first code in the top bits
            word |= q[:, i::per] << (8 - bits * (i + 1))
        put(word)
        step = e // OUTLIERS
        idx = torch.arange(OUTLIERS, device=dev) * step + torch.randint(0, step, (n, OUTLIERS), device=dev, generator=g)
        val = (normal(n, OUTLIERS).float() * 4).bfloat16().view(torch.int16).to(torch.int64) & 0xFFFF
        put(((idx << 16) | val).to(torch.int32))
    return out


def _inputs(case, seed):
    """Everything the program holds before the call, from the seed alone."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    row = case["heads_kv"] * case["dim"]
    fmt, lens, P = _formats(case)
    n = case["seqs"] * P
    s = {"case": case, "lengths": torch.tensor(lens, dtype=torch.int32, device=dev),
         "page_ids": torch.randperm(n, device=dev, generator=g).to(torch.int32).view(case["seqs"], P)}
    if case["kind"] == "evict":
        # heavy-tailed, as accumulated attention is: most pages draw next to nothing
        s["mass"] = torch.exp(2.0 * torch.randn(case["seqs"], P, device=dev, generator=g))
        s["mass"][:, ::7] = 0.0
        return s
    flat, ids = fmt.reshape(-1), s["page_ids"].reshape(-1).long()
    tier, slot = torch.zeros(n, dtype=torch.int8, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev)
    start = torch.zeros(n, dtype=torch.int32, device=dev)
    s["at"], s["slots"] = {}, {}
    for f in sorted(set(flat.tolist())):
        at = torch.from_numpy(np.flatnonzero(flat == f)).to(dev)
        where = torch.randperm(at.numel(), device=dev, generator=g).to(torch.int32)
        tier[ids[at]] = TIER_OF[f]
        if f == BF16:
            start[ids[at]] = where * T
            pool = (at.numel() * T, case["heads_kv"], case["dim"])
            s["k"] = torch.randn(*pool, device=dev, generator=g, dtype=torch.bfloat16)
            s["v"] = torch.randn(*pool, device=dev, generator=g, dtype=torch.bfloat16)
        else:
            slot[ids[at]] = where
            s["slots"][f] = _encode(f, at.numel(), row, g)
        s["at"][f] = (at, where.long())
    s |= {"tier": tier, "slot": slot, "start": start, "zeros": torch.zeros(n, dtype=torch.int32, device=dev)}
    # a peaked softmax: scores spread over a few units
    s["q"] = (torch.randn(case["seqs"], case["heads_q"], case["dim"], device=dev, generator=g) * 2).bfloat16()
    if case["mass"]:
        s["mass"] = torch.rand(case["seqs"], P, device=dev, generator=g)
    if case["kind"] == "sparse":
        s["codes"], s["exponents"] = _key_bounds(_pages(s)[:, 0], None)
        s["codes"], s["exponents"] = s["codes"][torch.argsort(ids)], s["exponents"][torch.argsort(ids)]
    if case["kind"] == "bounds":
        # every page of every sequence, with the tokens that it holds
        left = s["lengths"][:, None] - T * torch.arange(P, device=dev, dtype=torch.int32)
        s["valid"] = left.clamp(0, T).reshape(-1).contiguous()
        s["codes"] = torch.zeros(n, case["heads_kv"], 2, case["dim"], dtype=torch.int8, device=dev)
        s["exponents"] = torch.zeros(n, case["heads_kv"], dtype=torch.int8, device=dev)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] != "evict":
        s["handle"] = _handle(s)
    return s


def _library():
    """The library's operators (the package lives in a folder of the repository, not on the path)."""
    import sys
    from pathlib import Path
    package = str(Path(__file__).resolve().parent.parent / "ash-kv_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ashkv.runtime import attention
    return attention


def _handle(s):
    """The page table, the pool, the stores and the bounds as a user's program keeps them."""
    PageBounds = _library().PageBounds
    from ashkv.runtime.batch import DevicePageTable, KVLayers, TierStore
    case, dev = s["case"], s["q"].device
    f = s["mass"].reshape(-1) if s["case"]["mass"] else s["zeros"].float()
    table = DevicePageTable(f, f, f, f, s["tier"], s["zeros"], s["zeros"], s["start"], s["slot"])
    kv = KVLayers([s["k"]], [s["v"]])
    stores = {}
    for fmt, data in s["slots"].items():
        cap = CAP if fmt in (NBIT4, NBIT2) else 0
        store = TierStore(fmt, data.shape[0], dev, T, case["heads_kv"] * case["dim"], cap)
        store.data = data.view(-1)
        stores[TIER_OF[fmt]] = store
    bounds = PageBounds(s["codes"], s["exponents"]) if "codes" in s else None
    return table, kv, stores, bounds


# ----------------------------------------------------------------------------- plain forms
def _dequantise(fmt, slots, row):
    """Slots [n, bytes] -> the values their codes stand for [n, 2, T, row] (dithered pages: their bf16 values)."""
    n, e = slots.shape[0], 2 * T * row
    if fmt == INT8:
        at = (4 * T + 15) // 16 * 16
        scale = slots[:, :4 * T].contiguous().view(torch.float16).float()
        return slots[:, at:at + e].view(torch.int8).float().view(n, 2, T, row) * (scale / 127.0).view(n, 2, T, 1)
    if fmt == FP8:
        return slots[:, :e].contiguous().view(torch.float8_e4m3fn).float().view(n, 2, T, row)
    if fmt == INT4:
        scale = slots[:, :e // 32].contiguous().view(torch.bfloat16).float() / 7.0
        c = slots[:, e // 32:e // 32 + e // 2]
        q = torch.stack((c >> 4, c & 15), -1).float() - 8.0
        return (q.view(n, e // 64, 64) * scale[..., None]).view(n, 2, T, row)
    bits = 4 if fmt == NBIT4 else 2
    at = 16 + e // 16
    delta = slots[:, 16:at].contiguous().view(torch.bfloat16).float()
    shifts = torch.arange(8 - bits, -1, -bits, device=slots.device, dtype=torch.uint8)
    q = ((slots[:, at:at + e * bits // 8, None] >> shifts) & (2 ** bits - 1)).float() - (2 ** bits - 1) / 2
    x = (q.reshape(n, e // 32, 32) * delta[..., None]).bfloat16().float().view(n, e)
    at += e * bits // 8
    words = slots[:, at:at + 4 * OUTLIERS].contiguous().view(torch.int32)
    idx = (words.to(torch.int64) >> 16) & 0xFFFF
    return x.scatter(1, idx, (words << 16).view(torch.float32)).view(n, 2, T, row)


def _pages(s):
    """K and V of every page position in 32 bits: [seqs * pages, 2, T, heads_kv, dim]."""
    case = s["case"]
    hkv, d = case["heads_kv"], case["dim"]
    n = s["page_ids"].numel()
    out = torch.empty(n, 2, T, hkv, d, dtype=torch.float32, device=s["q"].device)
    at, where = s["at"][BF16]
    out[at, 0] = s["k"].view(-1, T, hkv, d)[where].float()
    out[at, 1] = s["v"].view(-1, T, hkv, d)[where].float()
    for f, slots in s["slots"].items():
        at, where = s["at"][f]
        out[at] = _dequantise(f, slots[where], hkv * d).view(-1, 2, T, hkv, d)
    return out


def _softmax_rows(scores, values):
    """Rows of masked scores [..., N] and values [..., N, dim] -> weights, result, log of the sum of exponentials."""
    top = scores.amax(-1, keepdim=True)
    safe = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores - safe)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return p, p @ values, (torch.log(total) + safe)[..., 0]


def _decode(s):
    case = s["case"]
    B, P = s["page_ids"].shape
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    kv = _pages(s).view(B, P, 2, T, hkv, d)
    k = kv[:, :, 0].reshape(B, P * T, hkv, d).permute(0, 2, 3, 1)
    v = kv[:, :, 1].reshape(B, P * T, hkv, d).permute(0, 2, 1, 3)
    q = s["q"].float().view(B, hkv, hq // hkv, d)
    inside = torch.arange(P * T, device=q.device)[None] < s["lengths"][:, None]
    scores = ((q @ k) / math.sqrt(d)).masked_fill(~inside[:, None, None], -math.inf)
    p, o, lse = _softmax_rows(scores, v)
    out = {"out": o.reshape(B, hq, d).bfloat16(), "lse": lse.reshape(B, hq)}
    if case["mass"]:
        drawn = p.view(B, hq, P, T).sum((1, 3))
        live = inside.view(B, P, T)[..., 0]
        out["mass"] = torch.where(live, DECAY * s["mass"] + drawn, s["mass"])
    return out


def _exponent(amax):
    """Smallest e >= -100 with amax <= 127 * 2^e (amax finite)."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 127.0 / 128.0, x - 6, x - 7)
    return torch.where(amax > 0, e, torch.full_like(e, -100)).clamp_min(-100)


def _key_bounds(keys, valid):
    """keys [n, T, heads, dim] -> int8 codes [n, heads, 2, dim] of their outward-rounded bounds, exponents [n, heads]."""
    n, t, h, d = keys.shape
    keys = keys.float()
    low, high = keys, keys
    if valid is not None:
        gone = (torch.arange(t, device=keys.device)[None] >= valid[:, None])[:, :, None, None]
        low, high = keys.masked_fill(gone, math.inf), keys.masked_fill(gone, -math.inf)
    b = torch.stack((low.amin(1), high.amax(1)), 2)
    if valid is not None:
        b = torch.where((valid > 0)[:, None, None, None], b, torch.zeros_like(b))
    e = _exponent(b.abs().amax((2, 3)))
    b = torch.ldexp(b.double(), -e[..., None, None])
    return torch.stack((b[:, :, 0].floor(), b[:, :, 1].ceil()), 2).to(torch.int8), e.to(torch.int8)


def _keep_highest(score, n_pages, budget, sink, recent):
    """Per row the first ``sink``, the last ``recent`` and the highest-scored positions up to ``budget``:
    a mask over the positions; of equal scores the lower position wins."""
    P = score.shape[-1]
    j = torch.arange(P, device=score.device)
    n = n_pages.view(-1, *([1] * (score.dim() - 1)))
    score = torch.where((j < sink) | (j >= n - recent), torch.full_like(score, math.inf), score)
    score = torch.where(j < n, score, torch.full_like(score, -math.inf))
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, j.expand_as(order).contiguous())
    return (rank < budget) & (j < n)


def _in_order(mask, width):
    """Positions of each row's true entries, ascending, padded with -1 to ``width``, and their number."""
    P = mask.shape[-1]
    j = torch.arange(P, device=mask.device).expand_as(mask)
    at = torch.sort(torch.where(mask, j, torch.full_like(j, P)), dim=-1).values[..., :width]
    at = torch.nn.functional.pad(at, (0, width - at.shape[-1]), value=P)
    return torch.where(at < P, at, torch.full_like(at, -1)).to(torch.int32), mask.sum(-1).to(torch.int32)


def _select(s):
    case = s["case"]
    B, P = s["page_ids"].shape
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    q = s["q"].float().view(B, hkv, hq // hkv, d)
    eq = _exponent(q.abs().amax(-1))
    q8 = torch.ldexp(q, -eq[..., None]).round()
    ids = s["page_ids"].reshape(-1).long()
    codes = s["codes"][ids].view(B, P, hkv, 2, d).permute(0, 2, 3, 4, 1).float()
    e = s["exponents"][ids].view(B, P, hkv).permute(0, 2, 1).int()
    dots = q8.clamp_max(0) @ codes[:, :, 0] + q8.clamp_min(0) @ codes[:, :, 1]  # whole numbers below 2^24
    score = torch.ldexp(dots.double(), eq[..., None] + e[:, :, None]).float().amax(2)
    pages = (s["lengths"] + T - 1) // T
    return _in_order(_keep_highest(score, pages, case["budget"], case["sink"], case["recent"]), case["budget"])


def _sparse(s):
    case = s["case"]
    B, P = s["page_ids"].shape
    hq, hkv, d, W = case["heads_q"], case["heads_kv"], case["dim"], case["budget"]
    selected, count = _select(s)
    kv = _pages(s).view(B, P, 2, T, hkv, d)
    at = selected.clamp_min(0).long()
    b = torch.arange(B, device=at.device)[:, None, None]
    h = torch.arange(hkv, device=at.device)[None, :, None]
    kv = kv[b, at, :, :, h]                                            # [B, heads, W, 2, T, dim]
    k, v = kv[:, :, :, 0].reshape(B, hkv, W * T, d), kv[:, :, :, 1].reshape(B, hkv, W * T, d)
    token = at[..., None] * T + torch.arange(T, device=at.device)
    inside = (selected >= 0)[..., None] & (token < s["lengths"][:, None, None, None])
    q = s["q"].float().view(B, hkv, hq // hkv, d)
    scores = (q @ k.transpose(-1, -2)) / math.sqrt(d)
    scores = scores.masked_fill(~inside.view(B, hkv, 1, W * T), -math.inf)
    _, o, lse = _softmax_rows(scores, v)
    return {"selected": selected, "count": count, "out": o.reshape(B, hq, d).bfloat16(), "lse": lse.reshape(B, hq)}


def _bounds(s):
    case = s["case"]
    at, where = s["at"][BF16]
    keys = s["k"].view(-1, T, case["heads_kv"], case["dim"])[where]
    ids = s["page_ids"].reshape(-1).long()[at]
    codes, exponents = _key_bounds(keys, s["valid"][at])
    s["codes"].index_copy_(0, ids, codes)
    s["exponents"].index_copy_(0, ids, exponents)
    return {"codes": s["codes"], "exponents": s["exponents"]}


def _evict(s):
    case = s["case"]
    P = s["page_ids"].shape[1]
    pages = (s["lengths"] + T - 1) // T
    keep = _keep_highest(s["mass"], pages, case["budget"], case["sink"], case["recent"])
    live = torch.arange(P, device=keep.device)[None] < pages[:, None]
    kept, n_kept = _in_order(keep, P)
    gone, n_gone = _in_order(live & ~keep, P)
    take = lambda x, at, fill: torch.where(at >= 0, x.gather(1, at.clamp_min(0).long()), torch.full_like(x, fill))  # noqa: E731
    return {"page_ids": take(s["page_ids"], kept, -1), "mass": take(s["mass"], kept, 0.0),
            "lengths": s["lengths"] - T * n_gone, "evicted": take(s["page_ids"], gone, -1), "n_evicted": n_gone}


# ----------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if not own:
        return {"decode": _decode, "sparse": _sparse, "bounds": _bounds, "evict": _evict}[case["kind"]](s)
    A = _library()
    if case["kind"] == "evict":
        got = A.evict_pages(s["mass"], s["page_ids"], s["lengths"], case["budget"], sink=case["sink"],
                            recent=case["recent"], tokens_per_page=T)
        return {"page_ids": got.page_ids, "mass": got.page_mass, "lengths": got.lengths, "evicted": got.evicted,
                "n_evicted": got.n_evicted}
    table, kv, stores, bounds = s["handle"]
    if case["kind"] == "bounds":
        bounds.update(table, kv, s["page_ids"].view(-1), valid=s["valid"], tokens_per_page=T)
        return {"codes": bounds.codes, "exponents": bounds.exponents}
    if case["kind"] == "sparse":
        selected, count = A.select_pages(s["q"], bounds, s["page_ids"], s["lengths"], case["budget"],
                                         sink=case["sink"], recent=case["recent"], tokens_per_page=T)
        out, lse = A.decode_attention(s["q"], table, kv, stores, s["page_ids"], s["lengths"], tokens_per_page=T,
                                      selected=selected, selected_count=count, return_lse=True)
        return {"selected": selected, "count": count, "out": out, "lse": lse}
    mass = s["mass"].clone() if case["mass"] else None  # the program's running mass, kept for the next pass
    out, lse = A.decode_attention(s["q"], table, kv, stores, s["page_ids"], s["lengths"], tokens_per_page=T,
                                  page_mass=mass, decay=DECAY, return_lse=True)
    return {"out": out, "lse": lse} | ({"mass": mass} if case["mass"] else {})


# ----------------------------------------------------------------------------- 64 bits
def _exact_page_values(s, position):
    """K and V of the given page positions [m] in 64 bits, from the stored bytes: [m, 2, T, row]."""
    case = s["case"]
    row = case["heads_kv"] * case["dim"]
    out = torch.zeros(position.numel(), 2, T, row, dtype=torch.float64, device=position.device)
    pid = s["page_ids"].reshape(-1)[position].long()
    tier, start, slot = s["tier"][pid], s["start"][pid].long(), s["slot"][pid].long()
    pick = (tier == 0).nonzero()[:, 0]
    rows = start[pick][:, None] + torch.arange(T, device=pid.device)
    for i, x in enumerate((s["k"], s["v"])):
        out[pick, i] = x.view(-1, row)[rows].double()
    for f, data in s["slots"].items():
        pick = (tier == TIER_OF[f]).nonzero()[:, 0]
        if not pick.numel():
            continue
        b, e = data[slot[pick]], 2 * T * row
        if f == INT8:
            first = 4 * T + (-4 * T) % 16
            x = b[:, first:first + e].contiguous().view(torch.int8).double().view(-1, 2 * T, row)
            x = x * b[:, :4 * T].contiguous().view(torch.float16).double()[..., None] / 127
        elif f == FP8:
            x = b[:, :e].contiguous().view(torch.float8_e4m3fn).double()
        elif f == INT4:
            c = b[:, e // 32:e // 32 + e // 2].to(torch.int64)
            x = torch.empty(b.shape[0], e, dtype=torch.float64, device=b.device)
            x[:, 0::2], x[:, 1::2] = (c // 16 - 8).double(), (c % 16 - 8).double()
            x = x * b[:, :e // 32].contiguous().view(torch.bfloat16).double().repeat_interleave(64, 1) / 7
        else:
            bits = 4 if f == NBIT4 else 2
            levels, first = 1 << bits, 16 + e // 16
            c = b[:, first:first + e * bits // 8].to(torch.int64)
            x = torch.empty(b.shape[0], e, dtype=torch.float64, device=b.device)
            for i in range(8 // bits):
                x[:, i::8 // bits] = (c // levels ** (8 // bits - 1 - i) % levels).double() - (levels - 1) / 2
            x = x * b[:, 16:first].contiguous().view(torch.bfloat16).double().repeat_interleave(32, 1)
            x = x.float().bfloat16().double()  # the product has few enough bits: one rounding
            first += e * bits // 8
            w = b[:, first:first + 4 * OUTLIERS].contiguous().view(torch.int16).view(-1, OUTLIERS, 2)
            x.scatter_(1, w[..., 1].to(torch.int64) & 0xFFFF, w[..., 0].contiguous().view(torch.bfloat16).double())
        out[pick] = x.view(-1, 2, T, row)
    return out


def _exact_attention(s, b, heads, tokens, kv, out, lse, share=None):
    """Query heads ``heads`` of sequence b over the keys and values kv [2, N, dim], N = tokens."""
    q = s["q"][b, heads].double()
    x = q @ kv[0, :tokens].T / math.sqrt(q.shape[-1])
    lse[b, heads] = torch.logsumexp(x, -1)
    w = torch.exp(x - lse[b, heads][:, None])
    out[b, heads] = w @ kv[1, :tokens]
    if share is not None:
        w = torch.nn.functional.pad(w.sum(0), (0, (-tokens) % T))
        share[: w.numel() // T] += w.view(-1, T).sum(-1)


def _exact_power(x):
    """Smallest e >= -100 with max |x| <= 127 * 2^e, over numpy's last axes."""
    e = np.full(x.shape, -100, dtype=np.int64)
    pos = x > 0
    e[pos] = np.maximum(-100, np.ceil(np.log2(x[pos] / 127.0) - 1e-9).astype(np.int64))
    while True:
        more = x > 127.0 * np.exp2(e)
        if not more.any():
            break
        e[more] += 1
    less = (e > -100) & (x <= 127.0 * np.exp2(e - 1.0))
    return e - less


def _exact_kept(score, budget, sink, recent):
    """Positions kept of one row of scores (numpy, length = its pages), ascending."""
    n = len(score)
    forced = [j for j in range(n) if j < sink or j >= n - recent] if n > budget else list(range(n))
    rest = [j for j in np.lexsort((np.arange(n), -score)).tolist() if sink <= j < n - recent] if n > budget else []
    return np.sort(np.asarray(forced + rest[:max(0, budget - len(forced))], dtype=np.int64))


def exact(case, seed):
    s = _inputs(case, seed)
    lens, P, hkv = s["lengths"].tolist(), s["page_ids"].shape[1], case["heads_kv"]
    group = case["heads_q"] // hkv
    if case["kind"] == "evict":
        if case["seqs"] * P > 1 << 19:
            return None
        ids, mass = s["page_ids"].cpu().numpy(), s["mass"].double().cpu().numpy()
        got = {"page_ids": np.full_like(ids, -1), "mass": np.zeros_like(mass), "lengths": np.array(lens, np.int32),
               "evicted": np.full_like(ids, -1), "n_evicted": np.zeros(len(lens), np.int32)}
        for b, n in enumerate(lens):
            pages = -(-n // T)
            keep = _exact_kept(mass[b, :pages], case["budget"], case["sink"], case["recent"])
            gone = np.setdiff1d(np.arange(pages), keep)
            got["page_ids"][b, :len(keep)], got["mass"][b, :len(keep)] = ids[b, keep], mass[b, keep]
            got["evicted"][b, :len(gone)], got["n_evicted"][b] = ids[b, gone], len(gone)
            got["lengths"][b] -= T * len(gone)
        got["mass"] = torch.from_numpy(got["mass"]).float()
        return got
    dev = s["q"].device
    if case["kind"] == "bounds":
        at, where = s["at"][BF16]
        k, left = s["k"].view(-1, T, hkv, case["dim"])[where].double(), s["valid"][at]
        codes, exps = torch.zeros_like(s["codes"]), torch.zeros_like(s["exponents"])
        for m in range(T + 1):  # pages that hold m tokens
            pick = (left == m).nonzero()[:, 0]
            if not pick.numel():
                continue
            x = k[pick, :m] if m else k[pick, :1] * 0
            lo, hi = x.min(1).values, x.max(1).values
            e = _exact_power(torch.maximum(lo.abs(), hi.abs()).amax(-1).cpu().numpy())
            e = torch.from_numpy(e).to(dev)
            unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=dev), e.double())[..., None]
            pid = s["page_ids"].reshape(-1).long()[at[pick]]
            codes[pid] = torch.stack((torch.floor(lo / unit), torch.ceil(hi / unit)), 2).to(torch.int8)
            exps[pid] = e.to(torch.int8)
        return {"codes": codes, "exponents": exps}
    out = torch.zeros(case["seqs"], case["heads_q"], case["dim"], dtype=torch.float64, device=dev)
    lse = torch.full((case["seqs"], case["heads_q"]), -math.inf, dtype=torch.float64, device=dev)
    mass = s["mass"].double() if case["mass"] else None
    W = case["budget"]
    selected = torch.full((case["seqs"], hkv, max(W, 1)), -1, dtype=torch.int32, device=dev)
    count = torch.zeros(case["seqs"], hkv, dtype=torch.int32, device=dev)
    for b, n in enumerate(lens):
        pages = -(-n // T)
        if not n:
            continue
        here = b * P + torch.arange(pages, device=dev)
        if case["kind"] == "decode":
            kv = _exact_page_values(s, here).view(pages, 2, T, hkv, case["dim"]).permute(1, 3, 0, 2, 4)
            share = torch.zeros(pages, dtype=torch.float64, device=dev)
            for h in range(hkv):
                _exact_attention(s, b, slice(h * group, (h + 1) * group), n,
                                 kv[:, h].reshape(2, pages * T, case["dim"]), out, lse, share)
            if mass is not None:
                mass[b, :pages] = DECAY * mass[b, :pages] + share
            continue
        pid = s["page_ids"].reshape(-1)[here].long()
        e = s["exponents"][pid].double()
        for h in range(hkv):
            lo, hi = s["codes"][pid, h, 0].double(), s["codes"][pid, h, 1].double()
            best = torch.full((pages,), -math.inf, dtype=torch.float64, device=dev)
            for i in range(h * group, (h + 1) * group):
                x = s["q"][b, i].double()
                p = float(_exact_power(np.array([float(x.abs().max())]))[0])
                x = torch.round(x / 2.0 ** p)
                dots = torch.maximum(x * lo, x * hi).sum(-1)
                best = torch.maximum(best, dots * torch.exp2(e[:, h] + p))
            keep = torch.from_numpy(_exact_kept(best.cpu().numpy(), W, case["sink"], case["recent"])).to(dev)
            selected[b, h, :keep.numel()], count[b, h] = keep.int(), keep.numel()
            kv = _exact_page_values(s, here[keep]).view(-1, 2, T, hkv, case["dim"])[:, :, :, h].transpose(0, 1)
            last = int(keep[-1]) == pages - 1
            tokens = keep.numel() * T - (pages * T - n if last else 0)
            _exact_attention(s, b, slice(h * group, (h + 1) * group), tokens,
                             kv.reshape(2, -1, case["dim"]), out, lse)
    got = {"out": out, "lse": lse}
    if case["kind"] == "sparse":
        return {"selected": selected, "count": count} | got
    return got | ({"mass": mass} if mass is not None else {})
