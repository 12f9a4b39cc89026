"""GPU tests of the attention of prompts over tiered pages, against float64.

Pages count as the bf16 values that the oracle's page decoders give.  Tolerances, from the arithmetic.
With u = 2^-24, size = max_t |scale| sum_d |q_d k_d| over the tokens that a row sees:
  a score is an fp32 sum of dim exact products on the tensor cores, scaled once: the sum may lose a few
      bits of its running value at each of its dim / 16 steps, |ds| <= (dim + 20) * 4 u * size;
  a weight is then off by a factor of 1 + dp, dp = 2 |ds| + 2^-20 (exp2's approximation, the
      difference to the running maximum);
  it is rounded to bf16 once, by at most 2^-8 of it, the sum of the weights takes it unrounded;
  the product accumulates in fp32 over n tokens, losing at most 4 u a step of 16;
  the result is rounded to bf16: 2^-8 of its value.
So |out - exact| <= 2^-8 |exact| + (2^-8 + 2 dp + n u) * sum_t P |v|; of lse: ds + 2^-19 + 8 u |lse|."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle
from oracle.attention import bf16_to_f64
from test_gpu_attention import CAP, FORMATS, TIER, Cache, bits
from test_gpu_cache import i32, page_bits_of, starts_of

from ashkv import _native as N
from ashkv.runtime import attention as A
from ashkv.runtime import cache as C
from ashkv.runtime.batch import StepGraph

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def tokens_of(c, ids, n):
    """K and V [2, n, heads, dim] in 64 bits of the first n tokens of a list."""
    pages = [bf16_to_f64(page_bits_of(c, int(j))).reshape(2, c.T, c.heads, c.dim) for j in ids[:-(-n // c.T)]]
    if not pages:
        return np.zeros((2, 0, c.heads, c.dim))
    return np.concatenate(pages, 1)[:, :n]


def seen_tokens(n, new, window, sinks):
    p, t = np.arange(n - new, n)[:, None], np.arange(n)[None]
    seen = t <= p
    if window:
        seen &= (t > p - window) | (t < sinks)
    return seen


def reference(c, ids, q, lengths, new, window=0, sinks=0, scale=None):
    """q float64 [rows, heads_q, dim] -> out, lse, and reach and size of the tolerances."""
    rows, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out, reach = np.zeros_like(q), np.zeros_like(q)
    lse, size = np.full((rows, hq), -np.inf), np.zeros((rows, hq))
    at = 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        if not m:
            continue
        kv = tokens_of(c, ids[b], n)
        seen = seen_tokens(n, m, window, sinks)
        x = slice(at, at + m)
        at += m
        for h in range(hq):
            k, v = kv[0][:, h // (hq // c.heads)], kv[1][:, h // (hq // c.heads)]
            s = np.where(seen, scale * (q[x, h] @ k.T), -np.inf)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            lse[x, h] = np.log(p.sum(-1)) + top[:, 0]
            p /= p.sum(-1, keepdims=True)
            out[x, h], reach[x, h] = p @ v, p @ np.abs(v)
            size[x, h] = np.where(seen, abs(scale) * (np.abs(q[x, h]) @ np.abs(k).T), 0).max(-1)
    return {"out": out, "lse": lse, "reach": reach, "size": size}


def check(got, lse, want, dim, n):
    out, l = got.double().cpu().numpy(), lse.double().cpu().numpy()
    ds = (dim + 20) * 4 * U * want["size"]
    dp = 2 * ds + 2.0 ** -20
    tol = 2.0 ** -8 * np.abs(want["out"]) + (2.0 ** -8 + 2 * dp + n * U)[..., None] * want["reach"] + 1e-37
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
