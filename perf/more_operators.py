"""Operators around tiered KV pages beyond a decode step, in their plain form and as calls of the library.

A layer of a paged cache: pages of ``page`` tokens, rows of ``heads_kv * dim`` values, a page either in
the bf16 pool or compressed in its tier's store.  Of every sequence the newest ``new`` tokens are the
ones that a pass deals with; their rows follow one another in the inputs and outputs.

* store: the keys and values of new tokens are quantised into the pages they belong to and read back;
* load: the tokens of the sequences are read from their pages into dense bf16 rows;
* prompt: the queries of new tokens attend the sequence up to themselves, all of it or a sliding window
  and the first tokens that stay visible.  Compressed pages count as the bf16 values that they decode to;
* step: one new query per sequence with such a window, and the attention weight that each page drew.
  Compressed pages count as the numbers that their codes stand for.

``own`` selects the library's kernels; otherwise elementary torch operations in 32 bits compute the
same from the same inputs.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BF16, INT8, FP8, INT4, NBIT4, NBIT2 = range(6)  # page formats
TIER_OF = {BF16: 0, INT8: 1, FP8: 1, INT4: 2, NBIT4: 2, NBIT2: 3}
KINDS = {"bf16": [BF16], "int8": [INT8], "fp8": [FP8], "int4": [INT4], "nbit4": [NBIT4],
         "three": [BF16, INT8, INT4], "three8": [BF16, FP8, INT4],
         "mixed": [BF16, INT8, INT4, NBIT2], "mixed8": [BF16, FP8, NBIT4, NBIT2]}
OUTLIERS, CAP = 96, 128                       # outliers of a dithered page, and the slots' capacity
DECAY = 0.9
MOST_SCORES = 1 << 29                         # scores that the plain form holds at a time


def _case(name, kind, seqs, tokens, new, heads_q, heads_kv, dim, tiers="bf16", ragged=False, window=0, sinks=0,
          mass=False, page=16):
    return {"name": name, "kind": kind, "seqs": seqs, "tokens": tokens, "new": new, "heads_q": heads_q,
            "heads_kv": heads_kv, "dim": dim, "tiers": tiers, "ragged": ragged, "window": window, "sinks": sinks,
            "mass": mass, "page": page}


def listed():
    return [
        # what one decode step of a batch adds to its INT8 pages: the latency of the calls counts
        _case("store-32x1-int8", "store", 32, 4000, 1, 64, 8, 128, "int8"),
        # a ragged batch of prompts written where the plan wants their pages: bf16, INT8 and INT4
        _case("store-12x8192-three", "store", 12, 8192, 8192, 32, 8, 128, "three", ragged=True),
        # whole prompts straight into FP8 pages, one rank's two heads of 64
        _case("store-32x8192-shard-fp8", "store", 32, 8192, 8192, 16, 2, 64, "fp8"),
        # one short conversation leaves its INT4 pages
        _case("load-1x301-int4", "load", 1, 301, 301, 32, 8, 128, "int4"),
        # the migration workload's pages in all four tiers, for an engine that wants dense keys and values
        _case("load-16x8192-mixed", "load", 16, 8192, 8192, 8, 8, 128, "mixed"),
        # a turn of a chat: a few new tokens after a short prefix
        _case("prompt-1x40-300-bf16", "prompt", 1, 300, 40, 32, 8, 128),
        # a whole prompt
        _case("prompt-1x8192-bf16", "prompt", 1, 8192, 8192, 32, 8, 128),
        # chunks of long prompts with a sliding window over INT8 pages, ragged
        _case("prompt-4x2048-w4096-int8", "prompt", 4, 32000, 2048, 64, 8, 128, "int8", ragged=True, window=4096,
              sinks=4),
        # five drafted tokens of every sequence are verified over long prefixes in FP8 pages
        _case("prompt-32x5-8192-fp8", "prompt", 32, 8192, 5, 64, 8, 128, "fp8"),
        # a decode step of the migration workload's batch with a window of 1024
        _case("step-32x8192-w1024-bf16", "step", 32, 8192, 1, 64, 8, 128, window=1024, sinks=4, mass=True),
        # a single long context in INT4 pages, a wide window
        _case("step-1x131071-w8192-int4", "step", 1, 131071, 1, 32, 8, 128, "int4", window=8192, sinks=64),
        # a ragged batch with an idle slot over all tiers, one rank's two heads of 64
        _case("step-64x6000-w512-mixed", "step", 64, 6000, 1, 16, 2, 64, "mixed", ragged=True, window=512, sinks=5,
              mass=True),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(["store", "load", "prompt", "prompt", "step"])
    heads_q, heads_kv, dim = rng.choice([(32, 8, 128), (64, 8, 128), (8, 8, 64), (16, 2, 64), (8, 1, 128),
                                         (32, 2, 128), (20, 4, 128), (28, 4, 128), (4, 4, 128), (2, 2, 64)])
    row = heads_kv * dim
    page = rng.choice([p for p in (8, 16, 16, 16, 32, 64) if 512 <= p * row <= 32768])
    seqs, ragged = size(1, 64), rng.random() < 0.6
    window = rng.choice([0, size(1, 8192)]) if kind == "prompt" else size(1, 8192) if kind == "step" else 0
    sinks = rng.choice([0, size(1, 100)]) if window else 0
    if kind in ("store", "load"):
        tokens = size(1, min(32768, 98304 * 512 // max(row, 512) // seqs))
        new = rng.choice([1, tokens, size(1, tokens)])
        tiers = rng.choice(["bf16", "int8", "fp8", "int4", "three", "three8"] + ["nbit4", "mixed", "mixed8"] * (kind == "load"))
    elif kind == "step":
        tokens, new = size(1, max(2, min(131072, 131072 * 1024 // max(row, 512) // seqs))), 1
        tiers = rng.choice(["bf16", "int8", "fp8", "int4", "nbit4", "mixed", "mixed8"])
    else:
        tokens = size(1, max(2, min(32768, 98304 // seqs)))
        # the scores of all new tokens cost no more than the whole prompt's among the listed cases
        new = size(1, max(1, min(tokens, 16384 // seqs, 8192 * 4096 * 4096 // (seqs * heads_q * dim * tokens))))
        tiers = rng.choice(["bf16", "bf16", "int8", "fp8", "int4", "nbit4", "mixed", "mixed8"])
    return _case("", kind, seqs, tokens, new, heads_q, heads_kv, dim, tiers, ragged, window, sinks,
                 kind == "step" and rng.random() < 0.5, page)


# ----------------------------------------------------------------------------- sizes
def _lengths(case):
    """Tokens and new tokens of each sequence: all alike, or spread over 5 % to 100 % with one idle slot in eight or more."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["tokens"]] * n, [min(case["new"], case["tokens"])] * n
    share = [0.05 + 0.95 * ((i * 0.6180339887) % 1.0) for i in range(n)]
    share[n // 3] = 1.0
    lens = [max(1, round(case["tokens"] * x)) for x in share]
    news = [min(m, max(1, round(case["new"] * x))) for m, x in zip(lens, reversed(share))]
    if n >= 8:
        lens[n // 2] = news[n // 2] = 0
    return lens, news


def _formats(case, P):
    """Format of every page position [seqs, P]: the tiers in turn."""
    kinds = np.asarray(KINDS[case["tiers"]])
    k = np.arange(case["seqs"] * P, dtype=np.int64)
    return kinds[((k * 2654435761) >> 7) % len(kinds)].reshape(case["seqs"], P)


def _touched(case, n, new):
    """Page positions of a sequence that a pass deals with, ascending."""
    T = case["page"]
    first, last = n - new, -(-n // T)
    if not new:
        return []
    if case["kind"] in ("store", "load") or case["window"]:
        at = first if case["kind"] in ("store", "load") else max(0, first - case["window"] + 1)
        sinks = -(-min(case["sinks"], n) // T)
        return sorted(set(range(sinks)) | set(range(at // T, last)))
    return list(range(last))


def _page_bytes(fmt, T, row):
    e = 2 * T * row
    return {BF16: 2 * e, INT8: e + 4 * T, FP8: e, INT4: e // 2 + e // 32,
            NBIT4: 16 + e // 16 + e // 2 + 4 * OUTLIERS, NBIT2: 16 + e // 16 + e // 4 + 4 * OUTLIERS}[fmt]


def _slot_bytes(fmt, T, row):
    e = 2 * T * row
    used = {INT8: (4 * T + 15) // 16 * 16 + e, FP8: e, INT4: e // 32 + e // 2,
            NBIT4: 16 + e // 16 + e // 2 + 4 * CAP, NBIT2: 16 + e // 16 + e // 4 + 4 * CAP}[fmt]
    return (used + 255) // 256 * 256


def work(case):
    T, hq, hkv, d = case["page"], case["heads_q"], case["heads_kv"], case["dim"]
    row = hkv * d
    lens, news = _lengths(case)
    fmt = _formats(case, max(1, max(-(-n // T) for n in lens)))
    N, pages, stored, pairs = sum(news), 0, 0.0, 0
    for b, (n, new) in enumerate(zip(lens, news)):
        at = _touched(case, n, new)
        pages += len(at)
        first = n - new
        for j in at:  # the tokens of the page that are read or written
            lo, hi = j * T, min(n, j * T + T)
            if case["kind"] in ("store", "load"):
                used = hi - max(lo, first)
            elif case["window"]:
                used = len(set(range(lo, min(hi, case["sinks"]))) | set(range(max(lo, first - case["window"] + 1), hi)))
            else:
                used = hi - lo
            stored += _page_bytes(int(fmt[b, j]), T, row) * used / T
        if case["kind"] in ("prompt", "step") and new:
            p = np.arange(first, n, dtype=np.int64)
            seen = p + 1
            if case["window"]:
                recent = np.minimum(seen, case["window"])
                seen = recent + np.minimum(seen - recent, case["sinks"])
            pairs += int(seen.sum())
    if case["kind"] == "store":
        return {"bytes": 8 * N * row + 2 * stored + 20 * pages, "flops": 0}
    if case["kind"] == "load":
        return {"bytes": 4 * N * row + stored + 20 * pages, "flops": 0}
    mass = 8 * sum(-(-n // T) for n in lens) if case["mass"] else 0
    return {"bytes": N * hq * (4 * d + 4) + stored + 20 * pages + mass, "flops": 4 * hq * d * pairs}


# ----------------------------------------------------------------------------- inputs
def _encode(fmt, n, T, row, g):
    """Slots [n, bytes] of compressed pages of roughly normal values, straight from codes and scales."""
    dev, e = g.device, 2 * T * row
    out = torch.zeros(n, _slot_bytes(fmt, T, row), dtype=torch.uint8, device=dev)
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
    up = lambda a, dt=torch.int64: torch.as_tensor(np.asarray(a), dtype=dt).to(dev)  # noqa: E731
    T, B, hq, hkv, d = case["page"], case["seqs"], case["heads_q"], case["heads_kv"], case["dim"]
    lens, news = _lengths(case)
    P = max(1, max(-(-n // T) for n in lens))
    fmt, n = _formats(case, P), B * P
    starts = np.concatenate([[0], np.cumsum(news)])
    N, M = int(starts[-1]), max(1, max(news))
    s = {"case": case, "lengths": up(lens, torch.int32), "starts": up(starts, torch.int32), "N": N,
         "page_ids": torch.randperm(n, device=dev, generator=g).to(torch.int32).view(B, P)}
    # where the pages are
    ids = s["page_ids"].reshape(-1).long()
    tier, slot = torch.zeros(n, dtype=torch.int8, device=dev), torch.full((n,), -1, dtype=torch.int32, device=dev)
    start = torch.zeros(n, dtype=torch.int32, device=dev)
    place = torch.zeros(n, dtype=torch.int64, device=dev)  # of a page position: its slot, or its page in the pool
    s["slots"], pool = {}, (T, hkv, d)
    for f in sorted(set(fmt.reshape(-1).tolist())):
        at = torch.from_numpy(np.flatnonzero(fmt.reshape(-1) == f)).to(dev)
        where = torch.randperm(at.numel(), device=dev, generator=g).to(torch.int32)
        tier[ids[at]] = TIER_OF[f]
        place[at] = where.long()
        if f == BF16:
            start[ids[at]] = where * T
            pool = (at.numel() * T, hkv, d)
        else:
            slot[ids[at]] = where
            s["slots"][f] = _encode(f, at.numel(), T, hkv * d, g)
    s["k"] = torch.randn(*pool, device=dev, generator=g, dtype=torch.bfloat16)
    s["v"] = torch.randn(*pool, device=dev, generator=g, dtype=torch.bfloat16)
    s |= {"tier": tier, "slot": slot, "start": start, "zeros": torch.zeros(n, dtype=torch.int32, device=dev)}
    if case["kind"] != "load":
        # the new tokens' rows as a model's fused projection leaves them; scores spread over a few units
        spread = torch.rand(hq + 2 * hkv, d, device=dev, generator=g) * 1.5 + 0.5
        spread[:hq] = 2.0
        at = B if case["kind"] == "step" else N  # (a step has a row for an idle sequence too: a padded batch)
        s["qkv"] = (torch.randn(at, hq + 2 * hkv, d, device=dev, generator=g, dtype=torch.bfloat16) * spread).bfloat16()
    if case["mass"]:
        s["mass"] = torch.rand(B, P, device=dev, generator=g)
    # the plan that the plain form goes by: the touched pages of every sequence, side by side
    touched = [_touched(case, m, k) for m, k in zip(lens, news)]
    V = max(1, max(len(t) for t in touched))
    vis = np.full((B, V), -1, np.int64)
    for b, t in enumerate(touched):
        vis[b, :len(t)] = t
    tok = vis[:, :, None] * T + np.arange(T)
    tok = np.where((vis[:, :, None] >= 0) & (tok < np.asarray(lens)[:, None, None]), tok, -1).reshape(B, V * T)
    s["vis"], s["tok"], s["at"] = up(vis), up(tok), {}
    flat = np.where(vis >= 0, np.arange(B)[:, None] * P + vis, -1).reshape(-1)
    for f in sorted(set(fmt.reshape(-1)[flat[flat >= 0]].tolist())):
        at = np.flatnonzero((flat >= 0) & (fmt.reshape(-1)[np.maximum(flat, 0)] == f))
        s["at"][f] = (up(at), place[up(flat[at])])
    # rows of the new tokens: [seqs, most new], their positions (-1: none), and back
    b_of = np.repeat(np.arange(B), news)
    i_of = np.arange(N) - starts[:-1][b_of]
    pos = np.asarray(lens)[b_of] - np.asarray(news)[b_of] + i_of
    rows, where = np.zeros((B, M), np.int64), np.full((B, M), -1, np.int64)
    rows[b_of, i_of], where[b_of, i_of] = b_of if case["kind"] == "step" else np.arange(N), pos
    s |= {"rows": up(rows), "pos": up(where), "back": up(b_of * M + i_of)}
    if case["kind"] in ("store", "load"):
        first = np.asarray([t[0] if t else 0 for t in touched])
        s["local"] = up(b_of * V * T + pos - first[b_of] * T)  # the token among the touched pages' tokens
    if case["kind"] == "store":
        page = b_of * P + pos // T
        s["put"] = {}
        for f in sorted(set(fmt.reshape(-1)[page].tolist())):
            r = np.flatnonzero(fmt.reshape(-1)[page] == f)
            s["put"][f] = (up(r), place[up(page[r])], up(pos[r] % T))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["handle"] = _handle(s)
    return s


def _handle(s):
    """The library, the page table, the pool and the stores as a user's program keeps them."""
    import sys
    from pathlib import Path
    package = str(Path(__file__).resolve().parent.parent / "ash-kv_b200")  # (a folder of the repository, not on the path)
    if package not in sys.path:
        sys.path.insert(0, package)
    from ashkv.runtime import attention, cache
    from ashkv.runtime.batch import DevicePageTable, KVLayers, TierStore
    case, f = s["case"], s["zeros"].float()
    table = DevicePageTable(f, f, f, f, s["tier"], s["zeros"], s["zeros"], s["start"], s["slot"])
    stores = {}
    for fmt, data in s["slots"].items():
        store = TierStore(fmt, data.shape[0], data.device, case["page"], case["heads_kv"] * case["dim"],
                          CAP if fmt in (NBIT4, NBIT2) else 0)
        store.data = data.view(-1)
        stores[TIER_OF[fmt]] = store
    return attention, cache, table, KVLayers([s["k"]], [s["v"]]), stores


# ----------------------------------------------------------------------------- plain forms
def _dequantise(fmt, slots, T, row):
    """Slots [n, bytes] -> the values their codes stand for [n, 2, T, row] (dithered pages: their bf16 values)."""
    n, e = slots.shape[0], 2 * T * row
    if fmt == INT8:
        at = (4 * T + 15) // 16 * 16
        scale = slots[:, :4 * T].contiguous().view(torch.float16).float()
        return slots[:, at:at + e].view(torch.int8).float().view(n, 2, T, row) * scale.view(n, 2, T, 1) / 127.0
    if fmt == FP8:
        return slots[:, :e].contiguous().view(torch.float8_e4m3fn).float().view(n, 2, T, row)
    if fmt == INT4:
        scale = slots[:, :e // 32].contiguous().view(torch.bfloat16).float()
        c = slots[:, e // 32:e // 32 + e // 2]
        q = torch.stack((c >> 4, c & 15), -1).float() - 8.0
        return (q.view(n, e // 64, 64) * scale[..., None] / 7.0).view(n, 2, T, row)
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


def _pages(s, rounded):
    """K and V of the touched pages [seqs * touched, 2, T, heads_kv, dim] in 32 bits, zeros where there is
    none; ``rounded``: the bf16 values that the pages decode to."""
    case = s["case"]
    T, hkv, d = case["page"], case["heads_kv"], case["dim"]
    out = torch.zeros(s["vis"].numel(), 2, T, hkv, d, dtype=torch.float32, device=s["vis"].device)
    for f, (at, where) in s["at"].items():
        if f == BF16:
            out[at] = torch.stack((s["k"].view(-1, T, hkv, d)[where], s["v"].view(-1, T, hkv, d)[where]), 1).float()
        else:
            x = _dequantise(f, s["slots"][f][where], T, hkv * d)
            out[at] = (x.bfloat16().float() if rounded else x).view(-1, 2, T, hkv, d)
    return out


def _attend(s, rounded):
    """Masked attention of the new tokens' queries: out [N, heads_q, dim], lse [N, heads_q], and the
    weights of a pass that needs them."""
    case = s["case"]
    B, V = s["vis"].shape
    T, hq, hkv, d = case["page"], case["heads_q"], case["heads_kv"], case["dim"]
    G, n, M = hq // hkv, V * T, s["rows"].shape[1]
    kv = _pages(s, rounded).view(B, V, 2, T, hkv, d)
    k = kv[:, :, 0].reshape(B, n, hkv, d).permute(0, 2, 3, 1)
    v = kv[:, :, 1].reshape(B, n, hkv, d).permute(0, 2, 1, 3)
    out = torch.empty(B, M, hq, d, dtype=torch.bfloat16, device=k.device)
    lse = torch.empty(B, M, hq, dtype=torch.float32, device=k.device)
    p = None
    step = max(1, MOST_SCORES // (B * hq * n))
    for i in range(0, M, step):  # as many rows at a time as the scores have room for
        m = min(step, M - i)
        q = s["qkv"][s["rows"][:, i:i + m], :hq].float().view(B, m, hkv, G, d).permute(0, 2, 1, 3, 4)
        pos, tok = s["pos"][:, i:i + m, None], s["tok"][:, None]
        seen = (tok >= 0) & (tok <= pos)
        if case["window"]:
            seen &= (tok > pos - case["window"]) | (tok < case["sinks"])
        scores = ((q.reshape(B, hkv, m * G, d) @ k) / math.sqrt(d)).view(B, hkv, m, G, n)
        scores = scores.masked_fill_(~seen[:, None, :, None], -math.inf)
        top = scores.amax(-1, keepdim=True)
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        p = scores.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        lse[:, i:i + m] = (torch.log(total) + top)[..., 0].permute(0, 2, 1, 3).reshape(B, m, hq)
        p /= torch.where(total > 0, total, torch.ones_like(total))
        o = (p.view(B, hkv, m * G, n) @ v).view(B, hkv, m, G, d)
        out[:, i:i + m] = o.permute(0, 2, 1, 3, 4).reshape(B, m, hq, d).bfloat16()
    return out, lse, p


def _prompt(s):
    out, lse, _ = _attend(s, True)
    return {"out": out.flatten(0, 1)[s["back"]], "lse": lse.flatten(0, 1)[s["back"]]}


def _step(s):
    case = s["case"]
    B, V = s["vis"].shape
    out, lse, p = _attend(s, False)  # a sequence without tokens has a row as well: zeros and -inf
    got = {"out": out[:, 0], "lse": lse[:, 0]}
    if case["mass"]:
        drawn = p.view(B, case["heads_q"], V, case["page"]).sum((1, 3))
        j = torch.arange(s["mass"].shape[1], device=drawn.device)
        live = j * case["page"] < s["lengths"][:, None]
        mass = torch.where(live, DECAY * s["mass"], s["mass"])
        got["mass"] = mass.scatter_add(1, s["vis"].clamp_min(0), torch.where(s["vis"] >= 0, drawn, torch.zeros_like(drawn)))
    return got


def _load(s):
    kv = _pages(s, True).bfloat16().transpose(0, 1).flatten(1, 2)
    return {"k": kv[0][s["local"]], "v": kv[1][s["local"]]}


def _store(s):
    case = s["case"]
    T, hq, hkv, d = case["page"], case["heads_q"], case["heads_kv"], case["dim"]
    row = hkv * d
    e = 2 * T * row
    for f, (r, slot, t) in s["put"].items():
        x = torch.stack((s["qkv"][r, hq:hq + hkv], s["qkv"][r, hq + hkv:]), 1).reshape(-1, 2, row)  # [rows, K and V, row]
        if f == BF16:
            s["k"].view(-1, row)[slot * T + t], s["v"].view(-1, row)[slot * T + t] = x[:, 0], x[:, 1]
            continue
        data = s["slots"][f]
        slot, half, t = slot[:, None], torch.arange(2, device=t.device)[None], t[:, None]
        if f == INT8:
            top = x.float().abs().amax(-1, keepdim=True).clamp_min(1e-8)
            q = (x * 127.0).bfloat16().float() / top
            q = torch.trunc(q + torch.where(q > 0, 0.5, -0.5)).to(torch.int8)
            at = (4 * T + 15) // 16 * 16
            data[:, at:at + e].view(torch.int8).unflatten(1, (2, T, row))[slot, half, t] = q
            data[:, :4 * T].view(torch.float16).unflatten(1, (2, T))[slot, half, t] = top[..., 0].half()
        elif f == FP8:
            data[:, :e].unflatten(1, (2, T, row))[slot, half, t] = x.to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            x = x.float().view(-1, 2, row // 64, 64)
            top = x.abs().amax(-1, keepdim=True).clamp_min(1e-8)
            q = (torch.round(x * 7.0 / top).clamp(-8, 7) + 8).to(torch.uint8).view(-1, 2, row)
            data[:, e // 32:e // 32 + e // 2].unflatten(1, (2, T, row // 2))[slot, half, t] = (q[..., 0::2] << 4) | q[..., 1::2]
            data[:, :e // 32].view(torch.bfloat16).unflatten(1, (2, T, row // 64))[slot, half, t] = top[..., 0].bfloat16()
    return _load(s)


# ----------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if not own:
        return {"store": _store, "load": _load, "prompt": _prompt, "step": _step}[case["kind"]](s)
    A, C, table, kv, stores = s["handle"]
    T, hq, hkv = case["page"], case["heads_q"], case["heads_kv"]
    window = case["window"] or None
    if case["kind"] == "step":
        mass = s["mass"].clone() if case["mass"] else None  # the program's running mass, kept for the next pass
        out, lse = A.decode_attention(s["qkv"][:, :hq], table, kv, stores, s["page_ids"], s["lengths"], tokens_per_page=T,
                                      window=window, sinks=case["sinks"], page_mass=mass, decay=DECAY, return_lse=True)
        return {"out": out, "lse": lse} | ({"mass": mass} if case["mass"] else {})
    if case["kind"] == "prompt":
        out, lse = A.prompt_attention(s["qkv"][:, :hq], table, kv, stores, s["page_ids"], s["lengths"], s["starts"],
                                      tokens_per_page=T, window=window, sinks=case["sinks"], return_lse=True)
        return {"out": out, "lse": lse}
    if case["kind"] == "store":
        C.write_kv(s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:], table, kv, stores, s["page_ids"], s["lengths"],
                   s["starts"], tokens_per_page=T)
    k, v = C.read_kv(table, kv, stores, s["page_ids"], s["lengths"], s["starts"], s["N"], tokens_per_page=T)
    return {"k": k, "v": v}


# ----------------------------------------------------------------------------- 64 bits
def _exact_tokens(s, b, tokens, rounded):
    """K and V [2, m, row] in 64 bits of the given tokens of sequence b, from the stored bytes."""
    case = s["case"]
    T, row = case["page"], case["heads_kv"] * case["dim"]
    e, dev = 2 * T * row, tokens.device
    pid = s["page_ids"][b, tokens // T].long()
    tier, slot, t = s["tier"][pid], s["slot"][pid].long(), tokens % T
    out = torch.zeros(2, tokens.numel(), row, dtype=torch.float64, device=dev)
    pick = (tier == 0).nonzero()[:, 0]
    at = s["start"][pid[pick]].long() + t[pick]
    out[0, pick], out[1, pick] = s["k"].view(-1, row)[at].double(), s["v"].view(-1, row)[at].double()
    for f, data in s["slots"].items():
        pick = (tier == TIER_OF[f]).nonzero()[:, 0]
        if not pick.numel():
            continue
        sl, lines = data[slot[pick]] if f in (NBIT4, NBIT2) else None, slot[pick]
        for half in range(2):
            r = half * T + t[pick]                      # the token's row in its page
            col = torch.arange(row, device=dev)
            if f == INT8:
                first = 4 * T + (-4 * T) % 16
                c = data[lines[:, None], first + r[:, None] * row + col].view(torch.int8).double()
                sc = data[lines[:, None], 2 * r[:, None] + torch.arange(2, device=dev)].contiguous().view(torch.float16)
                x = c * sc.double() / 127
            elif f == FP8:
                x = data[lines[:, None], r[:, None] * row + col].view(torch.float8_e4m3fn).double()
            elif f == INT4:
                c = data[lines[:, None], e // 32 + r[:, None] * (row // 2) + torch.arange(row // 2, device=dev)].long()
                x = torch.stack((c // 16 - 8, c % 16 - 8), -1).flatten(1).double()
                sc = data[lines[:, None], r[:, None] * (row // 32) + torch.arange(row // 32, device=dev)]
                x = x * sc.contiguous().view(torch.bfloat16).double().repeat_interleave(64, 1) / 7
            else:
                bits = 4 if f == NBIT4 else 2
                per, first = 8 // bits, 16 + e // 16
                c = sl.gather(1, first + r[:, None] * (row // per) + torch.arange(row // per, device=dev)).long()
                x = torch.stack([c // 2 ** (bits * (per - 1 - i)) % 2 ** bits for i in range(per)], -1).flatten(1)
                sc = sl.gather(1, 16 + r[:, None] * (row // 16) + torch.arange(row // 16, device=dev))
                x = (x.double() - (2 ** bits - 1) / 2) * sc.view(torch.bfloat16).double().repeat_interleave(32, 1)
                x = x.float().bfloat16().double()  # the product has few enough bits: one rounding
                first += e * bits // 8
                w = sl[:, first:first + 4 * OUTLIERS].contiguous().view(torch.int16).view(-1, OUTLIERS, 2)
                at = (w[..., 1].long() & 0xFFFF) - r[:, None] * row
                i, j = ((at >= 0) & (at < row)).nonzero(as_tuple=True)
                x[i, at[i, j]] = w[i, j, 0].view(torch.bfloat16).double()
            out[half, pick] = x.float().bfloat16().double() if rounded else x
    return out


def _exact_codes(x, f):
    """Rows x [m, row] of bf16 values in 64 bits -> the values that their codes stand for, in 64 bits."""
    if f == BF16:
        return x
    if f == FP8:
        return x.float().to(torch.float8_e4m3fn).double()
    if f == INT8:
        top = x.abs().amax(-1, keepdim=True).clamp_min(1e-8)
        q = (x * 127).float().bfloat16().double() / top
        return torch.sign(q) * torch.floor(q.abs() + 0.5) * top.float().half().double() / 127
    x = x.view(x.shape[0], -1, 64)
    top = x.abs().amax(-1, keepdim=True).clamp_min(1e-8)
    return (torch.round(x * 7 / top) * top.float().bfloat16().double() / 7).flatten(1)


def exact(case, seed):
    s = _inputs(case, seed)
    T, hq, hkv, d = case["page"], case["heads_q"], case["heads_kv"], case["dim"]
    lens, news = _lengths(case)
    starts, dev = s["starts"].tolist(), s["lengths"].device
    if case["kind"] in ("store", "load"):
        k = torch.zeros(2, s["N"], hkv * d, dtype=torch.float64, device=dev)
        if case["kind"] == "store":
            for f, (r, _, _) in s["put"].items():
                for i in range(2):
                    k[i, r] = _exact_codes(s["qkv"][r, hq + i * hkv:hq + (i + 1) * hkv].flatten(1).double(), f)
        else:
            for b, (n, new) in enumerate(zip(lens, news)):
                for t in range(n - new, n, 16384):
                    at = torch.arange(t, min(n, t + 16384), device=dev)
                    row = starts[b] + t - (n - new)
                    k[:, row:row + at.numel()] = _exact_tokens(s, b, at, False)
        return {"k": k[0].view(-1, hkv, d), "v": k[1].view(-1, hkv, d)}
    step = case["kind"] == "step"
    rows = case["seqs"] if step else s["N"]
    out = torch.zeros(rows, hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64, device=dev)
    mass = s["mass"].double() if case["mass"] else None
    for b, (n, new) in enumerate(zip(lens, news)):
        if not new:
            continue
        tokens = torch.arange(n, device=dev)
        if case["window"]:  # the first tokens, and from the first query's window on
            tokens = tokens[(tokens < case["sinks"]) | (tokens >= n - new - case["window"] + 1)]
        kv = _exact_tokens(s, b, tokens, not step).view(2, -1, hkv, d)
        if mass is not None:
            mass[b, :-(-n // T)] *= DECAY
        at = torch.arange(n - new, n, device=dev)[:, None]
        hidden = tokens[None] > at
        if case["window"]:
            hidden |= (tokens[None] <= at - case["window"]) & (tokens[None] >= case["sinks"])
        to = slice(b, b + 1) if step else slice(starts[b], starts[b + 1])
        for h in range(hq):
            q = s["qkv"][to, h].double()
            x = (q @ kv[0, :, h // (hq // hkv)].T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            lse[to, h] = torch.logsumexp(x, -1)
            w = x.sub_(lse[to, h][:, None]).exp_()
            out[to, h] = w @ kv[1, :, h // (hq // hkv)]
            if mass is not None:
                mass[b].index_add_(0, tokens // T, w[0])
    return {"out": out, "lse": lse} | ({"mass": mass} if mass is not None else {})
