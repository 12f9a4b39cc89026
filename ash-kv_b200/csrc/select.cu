// Which pages of a sequence to attend, and which to drop: int8 bounds of the
// keys of a page (ashkv_page_bounds), the pages whose bounds promise a query
// the highest scores (ashkv_select_pages), and the pages of least accumulated
// attention (ashkv_evict_pages).
//
// The bounds are rounded outwards to int8 with a power-of-two unit per page
// and key head and the query to int8 with one per query head, so a score is a
// whole number below 2^22 times a power of two: exact in fp32 in any order of
// summation, which makes the selection a function of the inputs alone.  sum_d
// max(q lo, q hi) = sum_d max(q, 0) hi + min(q, 0) lo, two int8 dot products.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>

#include "common.cuh"
#include "page_layout.cuh"

namespace ashkv {
namespace {

constexpr float kBf16Max = 3.3895313892515355e38f;
constexpr int kMinExponent = -100;  // also the exponent of an all-zero page

__device__ __forceinline__ void flag(uint32_t* status, uint32_t f) {
  if (status) atomicOr(status, f);
}

// Smallest e >= kMinExponent with amax <= 127 * 2^e, for finite amax >= 0.
__device__ __forceinline__ int bound_exponent(float amax) {
  if (amax == 0.0f) return kMinExponent;
  int x;
  const float m = frexpf(amax, &x);  // amax = m * 2^x, m in [0.5, 1)
  return max(kMinExponent, m > 127.0f / 128.0f ? x - 6 : x - 7);
}

struct BoundsParams {
  const int8_t* tier;
  const int32_t* layer_id;
  const int32_t* token_start;
  int64_t n_pages;
  const uint64_t* layer_k;
  int64_t pool_tokens, row_stride;
  int32_t n_layers, T, heads;
  const int32_t* list;
  const int32_t* count;
  int32_t max_entries;
  const int32_t* valid;
  int8_t* codes;
  int8_t* exponents;
  uint32_t* status;
};

// Bytes of four int8.
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
  return uint32_t(a & 255) | (uint32_t(b & 255) << 8) | (uint32_t(c & 255) << 16) | (uint32_t(d & 255) << 24);
}

__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {  // passes over a NaN
  uint32_t d;
  asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A thread per 8 channels of a listed page: a page's threads read whole rows, 16
// bytes each, eight rows in flight, and keep the channels' extremes as bf16
// pairs; the D / 8 threads of a head share its exponent.  Bound by reading the
// keys once: 16384 pages of 16 x 1024 keys take 93 us, 6.1 TB/s (93 % of a plain
// copy's rate); a warp per page and head, in runs of 256 bytes, took 169.
template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsParams p) {
  constexpr int kHead = D / 8;  // threads of a head
  const int lane = threadIdx.x & 31;
  wait_for_previous();
  const int64_t n = p.count ? min(max(*p.count, 0), p.max_entries) : p.max_entries;
  const int chunks = p.heads * kHead;
  const int64_t items = n * chunks, stride = int64_t(gridDim.x) * 256;
  for (int64_t i0 = int64_t(blockIdx.x) * 256 + (threadIdx.x & ~31); i0 < items; i0 += stride) {  // warp-uniform
    const int64_t i = i0 + lane, entry = i / chunks;
    const int c = int(i - entry * chunks), h = c / kHead;
    const bool on = i < items;  // a head's threads are all on or all off
    const int32_t id = on ? p.list[entry] : -1;
    bool ok = id >= 0 && id < p.n_pages;
    int32_t tier = 0, l = 0, ts = 0;
    int nt = p.T;
    if (ok) {
      tier = p.tier[id];
      l = p.layer_id[id];
      ts = p.token_start[id];
      if (p.valid) nt = max(0, min(p.valid[entry], p.T));
    }
    ok = ok && tier == 0 && l >= 0 && l < p.n_layers && ts >= 0 && int64_t(ts) + p.T <= p.pool_tokens;
    if (on && !ok && c == 0) flag(p.status, ASHKV_FLAG_INDEX_RANGE);
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) { lo[k] = 0x7F807F80u; hi[k] = 0xFF80FF80u; }  // +inf, -inf
    if (ok) {
      const uint16_t* row = reinterpret_cast<const uint16_t*>(p.layer_k[l]) + int64_t(ts) * p.row_stride + c * 8;
      auto take = [&](const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) { lo[k] = min_bf16x2(lo[k], w[k]); hi[k] = max_bf16x2(hi[k], w[k]); }
      };
      int t = 0;
      for (; t + 8 <= nt; t += 8) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = ld_v4(row + (t + u) * p.row_stride);
#pragma unroll
        for (int u = 0; u < 8; ++u) take(v[u]);
      }
      for (; t < nt; ++t) take(ld_v4(row + t * p.row_stride));
    }
    float a[8], b[8], amax = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      a[k] = k & 1 ? bf16hi(lo[k >> 1]) : bf16lo(lo[k >> 1]);
      b[k] = k & 1 ? bf16hi(hi[k >> 1]) : bf16lo(hi[k >> 1]);
      const bool none = a[k] > b[k];  // no number in the channel
      a[k] = none ? 0.0f : fmaxf(fminf(a[k], kBf16Max), -kBf16Max);
      b[k] = none ? 0.0f : fmaxf(fminf(b[k], kBf16Max), -kBf16Max);
      amax = fmaxf(amax, fmaxf(fabsf(a[k]), fabsf(b[k])));
    }
#pragma unroll
    for (int off = kHead / 2; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, off));
    if (!ok) continue;  // (the loop bound is the same for the whole warp)
    const int e = bound_exponent(amax);
    const float unit = __uint_as_float(uint32_t(127 - e) << 23);  // 2^-e, exact: e is in [-100, 122]
    int cl[8], ch[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      // a bound too small for fp32 in these units still rounds outwards
      cl[k] = a[k] < 0.0f ? min(int(floorf(a[k] * unit)), -1) : int(floorf(a[k] * unit));
      ch[k] = b[k] > 0.0f ? max(int(ceilf(b[k] * unit)), 1) : int(ceilf(b[k] * unit));
    }
    int8_t* out = p.codes + (int64_t(id) * p.heads + h) * 2 * D + (c % kHead) * 8;
    *reinterpret_cast<uint2*>(out) = make_uint2(pack4(cl[0], cl[1], cl[2], cl[3]), pack4(cl[4], cl[5], cl[6], cl[7]));
    *reinterpret_cast<uint2*>(out + D) = make_uint2(pack4(ch[0], ch[1], ch[2], ch[3]), pack4(ch[4], ch[5], ch[6], ch[7]));
    if (c % kHead == 0) p.exponents[int64_t(id) * p.heads + h] = int8_t(e);
  }
}

// ---------------------------------------------------------------- scores
struct ScoreParams {
  const uint16_t* q;
  int64_t q_seq_stride, q_head_stride;
  int32_t n_seqs, heads_q, heads, group;
  const int8_t* codes;
  const int8_t* exponents;
  int64_t n_pages;
  const int32_t* page_ids;
  int64_t page_ids_stride;
  int32_t max_pages, T;
  const int32_t* lengths;
  float* scores;  // [n_seqs][heads][max_pages]
  uint32_t* status;
};

__device__ __forceinline__ int pages_of(int32_t length, int max_pages, int T) {
  const int64_t n = length <= 0 ? 0 : (int64_t(length) + T - 1) / T;
  return int(n < max_pages ? n : max_pages);
}

// fl(dot * 2^x), exact but for results outside the normal range: |dot| < 2^22.
__device__ __forceinline__ float times_pow2(int dot, int x) { return scalbnf(float(dot), x); }

constexpr int kScoreWarps = 8;
constexpr int kScorePages = 16;  // pages of a warp, in two halves of 8

// D (16 x 8, int32) += A (16 x 32, int8, row) * B (32 x 8, int8, col): lane (g, t) holds
// A rows g and g + 8 and B column g at k = 4t .. 4t + 3 and 16 more, D rows g and g
// + 8 at columns 2t, 2t + 1.
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

// A CTA per (kScoreWarps * kScorePages page positions, key head, sequence).  The
// group's queries are quantised into shared memory as A operands of 16 rows,
// min(q8, 0) against the lower and max(q8, 0) against the upper bounds; the
// bounds of 8 pages are a B operand straight from global memory, 16 bytes a load
// (thread t takes chunk 4 j + t of a page, its words serving two products of 32).
// Bound by reading the bounds once, and for one sequence by the latency of length,
// ids and bounds: 8192 pages x 8 heads (17 MB) take 9 us; on fp32 FMAs 19.
template <int D>
__global__ void __launch_bounds__(kScoreWarps * 32) select_scores_kernel(const ScoreParams p) {
  constexpr int kChunks = 2 * D / 16;           // 16-byte chunks of a page's bounds
  extern __shared__ __align__(16) uint8_t s_score[];  // [tiles of 16 queries][kChunks][2 products][8 rows][16 B], exponents
  // Neighbouring chunks keep a row in different banks.
  const auto operand_row = [](int tile, int chunk, int product, int row) {
    return ((tile * kChunks + chunk) * 2 + product) * 128 + (row ^ ((2 * chunk + product) & 7)) * 16;
  };
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  wait_for_previous();
  allow_next();
  const int n = pages_of(p.lengths[b], p.max_pages, p.T);
  const int j_cta = blockIdx.x * (kScoreWarps * kScorePages);
  if (j_cta >= n) return;
  const int tiles = (p.group + 15) / 16;
  // page ids and bounds first: they do not depend on the queries
  const int j0 = j_cta + warp * kScorePages;
  int32_t id[2];
  bool ok[2];
  uint4 w[2][kChunks / 4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int j = j0 + 8 * u + g;
    id[u] = j < n ? p.page_ids[b * p.page_ids_stride + j] : -1;
    ok[u] = id[u] >= 0 && id[u] < p.n_pages;
    if (j < n && !ok[u] && t == 0) flag(p.status, ASHKV_FLAG_INDEX_RANGE);
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int8_t* c = p.codes + (int64_t(ok[u] ? id[u] : 0) * p.heads + h) * 2 * D + t * 16;
#pragma unroll
    for (int k = 0; k < kChunks / 4; ++k)
      w[u][k] = ok[u] ? ld_v4(c + 64 * k) : make_uint4(0, 0, 0, 0);
  }
  int e_mine[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) e_mine[u] = ok[u] ? p.exponents[int64_t(id[u]) * p.heads + h] : 0;
  int* s_e = reinterpret_cast<int*>(s_score + size_t(tiles) * kChunks * 256);
  for (int q = warp; q < tiles * 16; q += kScoreWarps) {
    constexpr int N = D / 32;  // channels of a lane: lane * N ..
    float x[N], amax = 0.0f;
    const uint16_t* src = p.q + b * p.q_seq_stride + int64_t(h * p.group + q) * p.q_head_stride + lane * N;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      x[k] = q < p.group ? bf16_to_f32(src[k]) : 0.0f;
      if (!(fabsf(x[k]) <= kBf16Max)) x[k] = 0.0f;
      amax = fmaxf(amax, fabsf(x[k]));
    }
    amax = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax)));
    const int e = bound_exponent(amax);
    const float unit = __uint_as_float(uint32_t(127 - e) << 23);
    if (lane == 0) s_e[q] = e;
    uint32_t low = 0, high = 0;  // this lane's channels against the lower and the upper bounds
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int v = __float2int_rn(x[k] * unit);
      low |= uint32_t(min(v, 0) & 255) << (8 * k);
      high |= uint32_t(max(v, 0)) << (8 * k);
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int at = half * D + lane * N, word = (at >> 2) & 3;
      // operand word order: (row g, row g + 8) of the product's first, of its second word
      uint8_t* to = s_score + operand_row(q >> 4, at >> 4, word >> 1, q & 7) + ((word & 1) * 2 + ((q >> 3) & 1)) * 4 + (at & 3);
      if constexpr (N == 4) *reinterpret_cast<uint32_t*>(to) = half ? high : low;
      else *reinterpret_cast<uint16_t*>(to) = uint16_t(half ? high : low);
    }
  }
  __syncthreads();
  float best[2][2];  // [half][page 2t, 2t + 1]
#pragma unroll
  for (int u = 0; u < 2; ++u) best[u][0] = best[u][1] = -INFINITY;
  for (int m = 0; m < tiles; ++m) {
    int d[2][4] = {};
#pragma unroll
    for (int k = 0; k < kChunks / 4; ++k) {
      const uint4 a0 = *reinterpret_cast<const uint4*>(s_score + operand_row(m, 4 * k + t, 0, g));
      const uint4 a1 = *reinterpret_cast<const uint4*>(s_score + operand_row(m, 4 * k + t, 1, g));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        mma_s8(d[u], a0, w[u][k].x, w[u][k].y);
        mma_s8(d[u], a1, w[u][k].z, w[u][k].w);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int x = 0; x < 4; ++x) {  // row g (+ 8), column 2t + (x & 1)
        const int q = 16 * m + g + 8 * (x >> 1);
        const int e = __shfl_sync(0xFFFFFFFFu, e_mine[u], 4 * (2 * t + (x & 1)));
        if (q < p.group) best[u][x & 1] = fmaxf(best[u][x & 1], times_pow2(d[u][x], e + s_e[q]));
      }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float v = best[u][x];
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
      v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
      const int j = j0 + 8 * u + 2 * t + x;
      const bool exists = __shfl_sync(0xFFFFFFFFu, int(ok[u]), 4 * (2 * t + x));
      if (g == 0 && j < n) p.scores[(int64_t(b) * p.heads + h) * p.max_pages + j] = exists ? v : -INFINITY;
    }
}

// ---------------------------------------------------------------- keep the highest
// fp32 as an unsigned key of the same order; -0 equals +0, NaN is below all.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0u;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr int kKeepThreads = 1024;

constexpr int kKeepWarps = kKeepThreads / 32;
constexpr int kBins = 2048, kDigit = 11;

struct KeepShared {
  uint32_t hist[kBins];
  uint32_t warp_a[kKeepWarps], warp_b[kKeepWarps];
  uint32_t border, need, done;
};

// Sum over the CTA of what the threads before this one hold (and of all of it).
__device__ __forceinline__ uint32_t scan_before(uint32_t v, uint32_t* s_warp, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, inc, off);
    if (lane >= off) inc += x;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  uint32_t w = s_warp[lane], wi = w;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, wi, off);
    if (lane >= off) wi += x;
  }
  total = __shfl_sync(0xFFFFFFFFu, wi, 31);
  return __shfl_sync(0xFFFFFFFFu, wi - w, warp) + inc - v;
}

// One CTA decides for each position j of a row of n scores whether it is kept
// -- the first `sink`, the last `recent`, and of the others the highest, of
// equal ones the first, `budget` in all -- and calls emit(j, kept, rank) with
// its rank among the kept (else among the dropped) in ascending order of j.
// The border score is found by up to three rounds over 11, 11 and 10 bits of
// the keys (a count per value of the digit among the keys that share the digits
// above), fewer where a digit's count ends exactly at the number still wanted.
// Every warp owns a run of positions, 32 at a time.  For the ranks each warp counts
// its run first, so one scan over the warps serves the whole row.  Bound by the
// latency of its rounds: 128 of 8192 pages for 8 rows 15 us on 8 SMs, 1024 of
// up to 8192 for 256 rows (eviction) 24 us.  Digits taken of the distance from the
// lowest key, which spread over more bins, cost the reduction what they save.
//   CACHED: rows of up to kCached * kKeepThreads positions keep their keys in
// registers, longer ones read them anew in each round.  At 8192 positions: 8 rows
// (select, with its attention) 39.4 us and 41.4 read anew, 64 rows 100 and 104, 256
// rows (evict) 28.5 and 30.8; the same at 2048.
constexpr int kCached = 8;
template <bool CACHED, class Emit>
__device__ void keep_highest(const float* score, int n, int budget, int sink, int recent, KeepShared& sm,
                             Emit emit) {
  static_assert(kKeepWarps == 32, "scan_before takes 32 warps");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool all = n <= budget;
  const int lo = all ? n : sink, hi = all ? n : n - recent;  // the positions that compete
  const int steps = (n + kKeepThreads - 1) / kKeepThreads, j_first = warp * steps * 32 + lane;
  const auto competes = [&](int s) { return unsigned(j_first + 32 * s - lo) < unsigned(hi - lo); };
  uint32_t cached[CACHED ? kCached : 1];
  uint32_t alive = 0;  // bit s (CACHED): step s's position competes and shares the border's digits so far
  if constexpr (CACHED) {
#pragma unroll
    for (int s = 0; s < kCached; ++s) {
      cached[s] = 0;
      if (s < steps && competes(s)) {
        cached[s] = order_key(score[j_first + 32 * s]);
        alive |= 1u << s;
      }
    }
  }
  const uint32_t competing = alive;
  uint32_t border = 0xFFFFFFFFu, need = all ? 0u : uint32_t(budget - sink - recent);
  // whether keys equal to the border are all in (then there are no more than wanted above and at it)
  bool whole = false;
  if (need > 0) {
    border = 0;
    for (int i = tid; i < kBins; i += kKeepThreads) sm.hist[i] = 0;
    __syncthreads();
    for (int shift = 32 - kDigit;; shift = shift >= kDigit ? shift - kDigit : 0) {
      // digit: bits [shift, shift + bits); the last round has the 10 lowest
      const int bits = shift == 0 ? 32 - 2 * kDigit : kDigit;
      const uint32_t mask = (1u << bits) - 1u;
      if constexpr (CACHED) {
        if (alive) {
#pragma unroll
          for (int s = 0; s < kCached; ++s)
            if (alive >> s & 1u) atomicAdd(&sm.hist[cached[s] >> shift & mask], 1u);
        }
      } else {
        const uint32_t above_bits = uint32_t(uint64_t(0xFFFFFFFFu) << (shift + bits));
        for (int s = 0; s < steps; ++s) {
          if (!competes(s)) continue;
          const uint32_t k = order_key(score[j_first + 32 * s]);
          if (((k ^ border) & above_bits) == 0) atomicAdd(&sm.hist[k >> shift & mask], 1u);
        }
      }
      __syncthreads();
      // two bins of a thread, from the top
      const uint32_t d0 = kBins - 1 - 2 * tid, v0 = sm.hist[d0], v1 = sm.hist[d0 - 1];
      uint32_t total;
      const uint32_t above = scan_before(v0 + v1, sm.warp_a, total);
      if (above < need && above + v0 + v1 >= need) {  // exactly one thread
        const bool first = above + v0 >= need;
        const uint32_t over = first ? above : above + v0, count = first ? v0 : v1;
        sm.border = border | ((first ? d0 : d0 - 1) << shift);
        sm.need = need - over;
        sm.done = over + count == need;  // every key of this digit is wanted
      }
      sm.hist[d0] = sm.hist[d0 - 1] = 0;
      __syncthreads();
      border = sm.border;
      need = sm.need;
      whole = sm.done;
      if (shift == 0 || whole) break;
      if constexpr (CACHED) {
        if (alive) {
#pragma unroll
          for (int s = 0; s < kCached; ++s)
            if ((cached[s] ^ border) >> shift & mask) alive &= ~(1u << s);
        }
      }
    }
  }
  // Kept for certain (`in`), and at the border, where `need` are still wanted.
  const auto votes = [&](int s, unsigned& in, unsigned& at_border) {
    const int j = j_first + 32 * s;
    bool mid;
    uint32_t k = 0;
    if constexpr (CACHED) {
      mid = competing >> s & 1u;
      k = cached[s];
    } else {
      mid = competes(s);
      if (mid) k = order_key(score[j]);
    }
    in = __ballot_sync(0xFFFFFFFFu, j < n && (!mid || (whole ? k >= border : k > border)));
    at_border = __ballot_sync(0xFFFFFFFFu, mid && !whole && k == border);
  };
  const auto for_steps = [&](auto body) {
    if constexpr (CACHED) {
#pragma unroll
      for (int s = 0; s < kCached; ++s)
        if (s < steps) body(s);
    } else {
      for (int s = 0; s < steps; ++s) body(s);
    }
  };
  uint32_t n_keep = 0, n_eq = 0;
  for_steps([&](int s) {
    unsigned in, at_border;
    votes(s, in, at_border);
    n_keep += __popc(in);
    n_eq += __popc(at_border);
  });
  if (lane == 0) { sm.warp_a[warp] = n_keep; sm.warp_b[warp] = n_eq; }
  __syncthreads();
  uint32_t keep_before = lane < warp ? sm.warp_a[lane] : 0u, eq_before = lane < warp ? sm.warp_b[lane] : 0u;
  keep_before = __reduce_add_sync(0xFFFFFFFFu, keep_before);
  eq_before = __reduce_add_sync(0xFFFFFFFFu, eq_before);
  const unsigned below = (1u << lane) - 1u;
  for_steps([&](int s) {
    unsigned in, at_border;
    votes(s, in, at_border);
    const uint32_t e = eq_before + __popc(at_border & below), kept = keep_before + __popc(in & below) + min(e, need);
    const bool eq = at_border >> lane & 1u, keep = eq ? e < need : in >> lane & 1u;
    const int j = j_first + 32 * s;
    if (j < n) emit(j, keep, keep ? int(kept) : j - int(kept));
    keep_before += __popc(in);
    eq_before += __popc(at_border);
  });
}
template <class Emit>
__device__ __forceinline__ void keep_highest_of(const float* score, int n, int budget, int sink, int recent,
                                                KeepShared& sm, Emit emit) {
  if (n <= kCached * kKeepThreads) keep_highest<true>(score, n, budget, sink, recent, sm, emit);
  else keep_highest<false>(score, n, budget, sink, recent, sm, emit);
}

__global__ void __launch_bounds__(kKeepThreads, 2) select_keep_kernel(const float* scores, const int32_t* lengths,
                                                                      int heads, int max_pages, int T, int budget,
                                                                      int sink, int recent, int32_t* selected,
                                                                      int32_t* count, uint32_t* status) {
  __shared__ KeepShared sm;
  const int64_t row = blockIdx.x;
  const int b = int(row / heads);
  wait_for_previous();
  allow_next();
  const int n = pages_of(lengths[b], max_pages, T);
  int32_t* out = selected + row * budget;
  keep_highest_of(scores + row * max_pages, n, budget, sink, recent, sm, [&](int j, bool kept, int at) {
    if (kept) out[at] = j;
  });
  const int kept = min(n, budget);
  for (int i = kept + threadIdx.x; i < budget; i += kKeepThreads) out[i] = -1;
  if (threadIdx.x == 0) {
    count[row] = kept;
    if (lengths[b] < 0 || int64_t(lengths[b]) > int64_t(max_pages) * T) flag(status, ASHKV_FLAG_INDEX_RANGE);
  }
}

__global__ void __launch_bounds__(kKeepThreads, 2) evict_kernel(
    const float* mass, int64_t mass_stride, const int32_t* page_ids, int64_t page_ids_stride, const int32_t* lengths,
    int max_pages, int T, int budget, int sink, int recent, int32_t* out_ids, float* out_mass, int32_t* out_lengths,
    int32_t* evicted, int32_t* evicted_count) {
  __shared__ KeepShared sm;
  const int64_t b = blockIdx.x;
  wait_for_previous();
  const int n = pages_of(lengths[b], max_pages, T);
  const float* m = mass + b * mass_stride;
  const int32_t* ids = page_ids + b * page_ids_stride;
  int32_t* oi = out_ids + b * max_pages;
  float* om = out_mass + b * max_pages;
  int32_t* ev = evicted + b * max_pages;
  keep_highest_of(m, n, budget, sink, recent, sm, [&](int j, bool kept, int at) {
    const int32_t id = ids[j];  // both loads before a store that they might have to wait for
    const float x = m[j];
    if (kept) {
      oi[at] = id;
      om[at] = x;
    } else {
      ev[at] = id;
    }
  });
  const int kept = min(n, budget), gone = n - kept;
  for (int i = threadIdx.x; i < max_pages; i += kKeepThreads) {
    if (i >= kept) { oi[i] = -1; om[i] = 0.0f; }
    if (i >= gone) ev[i] = -1;
  }
  if (threadIdx.x == 0) {
    const int64_t len = max(0, lengths[b]), most = int64_t(max_pages) * T;
    out_lengths[b] = int32_t((len < most ? len : most) - int64_t(gone) * T);
    evicted_count[b] = gone;
  }
}

ashkv_status_t refuse(const char* what, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", what, why);
  set_message(text);
  return ASHKV_BAD_ARGUMENT;
}

}  // namespace
}  // namespace ashkv

using namespace ashkv;

extern "C" ashkv_status_t ashkv_page_bounds(const ashkv_paged_kv_t* kv, const int32_t* d_list, const int32_t* d_count,
                                            int32_t max_entries, const int32_t* d_valid, int8_t* d_codes,
                                            int8_t* d_exponents, uint32_t* d_status, void* stream) {
  constexpr const char* kName = "ashkv_page_bounds";
  if (!kv) return refuse(kName, "null page description");
  if (kv->head_dim != 64 && kv->head_dim != 128) return refuse(kName, "head_dim must be 64 or 128");
  if (max_entries < 0 || kv->heads_kv <= 0 || kv->heads_kv > 65536 || kv->tokens_per_page <= 0 || kv->n_layers <= 0 ||
      kv->n_pages < 0 || kv->pool_tokens < 0)
    return refuse(kName, "heads_kv, tokens_per_page and n_layers must be positive, sizes not negative");
  if (kv->row_stride < int64_t(kv->heads_kv) * kv->head_dim || kv->row_stride % 8)
    return refuse(kName, "row_stride must be a multiple of 8 and at least heads_kv * head_dim");
  if (max_entries == 0) return ASHKV_OK;
  if (!kv->d_tier || !kv->d_layer_id || !kv->d_token_start || !kv->d_layer_k || !d_list || !d_codes || !d_exponents ||
      !aligned(d_codes, 16))
    return refuse(kName, "null or misaligned device pointer");
  BoundsParams p{kv->d_tier, kv->d_layer_id, kv->d_token_start, kv->n_pages, kv->d_layer_k, kv->pool_tokens,
                 kv->row_stride, kv->n_layers, kv->tokens_per_page, kv->heads_kv, d_list, d_count, max_entries, d_valid,
                 d_codes, d_exponents, d_status};
  const int64_t threads = int64_t(max_entries) * p.heads * (kv->head_dim / 8);
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const unsigned grid = unsigned(std::min<int64_t>((threads + 255) / 256, int64_t(sms) * 8));
  launch_overlapped(kv->head_dim == 64 ? page_bounds_kernel<64> : page_bounds_kernel<128>, dim3(grid), dim3(256), 0,
                    as_stream(stream), p);
  return check_launch(kName);
}

extern "C" int64_t ashkv_select_scratch_floats(int32_t n_seqs, int32_t heads_kv, int32_t max_pages) {
  if (n_seqs < 0 || heads_kv <= 0 || max_pages < 0) return -1;
  return int64_t(n_seqs) * heads_kv * max_pages;
}

extern "C" ashkv_status_t ashkv_select_pages(const void* d_q, int64_t q_seq_stride, int64_t q_head_stride,
                                             int32_t n_seqs, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                                             const int8_t* d_codes, const int8_t* d_exponents, int64_t n_pages,
                                             const int32_t* d_page_ids, int64_t page_ids_stride, int32_t max_pages,
                                             const int32_t* d_lengths, int32_t tokens_per_page, int32_t budget,
                                             int32_t sink, int32_t recent, int32_t* d_selected,
                                             int32_t* d_selected_count, float* d_scratch, uint32_t* d_status,
                                             void* stream) {
  constexpr const char* kName = "ashkv_select_pages";
  if (head_dim != 64 && head_dim != 128) return refuse(kName, "head_dim must be 64 or 128");
  if (n_seqs < 0 || n_seqs > 65535 || max_pages < 0 || n_pages < 0 || heads_q <= 0 || heads_kv <= 0 ||
      heads_kv > 65535 || heads_q % heads_kv || heads_q / heads_kv > 128 || tokens_per_page <= 0)
    return refuse(kName, "bad size (at most 65535 sequences and key heads, 128 query heads to a key head)");
  if (budget < 1 || sink < 0 || recent < 0 || int64_t(sink) + recent > budget)
    return refuse(kName, "budget must be at least 1 and at least sink + recent");
  if (int64_t(n_seqs) * heads_kv > INT_MAX || int64_t(max_pages) + kKeepThreads > INT_MAX)
    return refuse(kName, "too many rows or pages");
  if (n_seqs == 0) return ASHKV_OK;
  if (!d_q || (!d_page_ids && max_pages > 0) || !d_lengths || !d_selected || !d_selected_count || (max_pages > 0 && !d_scratch) ||
      (n_pages > 0 && (!d_codes || !d_exponents)) || !aligned(d_codes, 16))
    return refuse(kName, "null or misaligned device pointer");
  if (page_ids_stride < max_pages) return refuse(kName, "page_ids_stride must hold max_pages entries");
  cudaStream_t st = as_stream(stream);
  const int group = heads_q / heads_kv;
  if (max_pages > 0) {
    ScoreParams p{static_cast<const uint16_t*>(d_q), q_seq_stride, q_head_stride, n_seqs, heads_q, heads_kv, group,
                  d_codes, d_exponents, n_pages, d_page_ids, page_ids_stride, max_pages, tokens_per_page, d_lengths,
                  d_scratch, d_status};
    constexpr int kPages = kScoreWarps * kScorePages;
    const dim3 grid(unsigned((max_pages + kPages - 1) / kPages), unsigned(heads_kv), unsigned(n_seqs));
    const size_t smem = size_t((group + 15) / 16) * 16 * (2 * head_dim + 4);  // at most 128 queries: 33 KB
    launch_overlapped(head_dim == 64 ? select_scores_kernel<64> : select_scores_kernel<128>, grid, dim3(kScoreWarps * 32),
                      smem, st, p);
    const ashkv_status_t rc = check_launch(kName);
    if (rc != ASHKV_OK) return rc;
  }
  launch_overlapped(select_keep_kernel, dim3(unsigned(n_seqs * heads_kv)), dim3(kKeepThreads), 0, st, d_scratch, d_lengths,
                    heads_kv, max_pages, tokens_per_page, budget, sink, recent, d_selected, d_selected_count, d_status);
  return check_launch(kName);
}

extern "C" ashkv_status_t ashkv_evict_pages(const float* d_page_mass, int64_t mass_stride, const int32_t* d_page_ids,
                                            int64_t page_ids_stride, const int32_t* d_lengths, int32_t n_seqs,
                                            int32_t max_pages, int32_t tokens_per_page, int32_t budget, int32_t sink,
                                            int32_t recent, int32_t* d_out_page_ids, float* d_out_mass,
                                            int32_t* d_out_lengths, int32_t* d_evicted, int32_t* d_evicted_count,
                                            void* stream) {
  constexpr const char* kName = "ashkv_evict_pages";
  if (n_seqs < 0 || max_pages < 0 || tokens_per_page <= 0 || int64_t(max_pages) + kKeepThreads > INT_MAX)
    return refuse(kName, "negative size, or too many pages");
  if (sink < 0 || recent < 1 || int64_t(sink) + recent > budget)
    return refuse(kName, "recent must be at least 1 and budget at least sink + recent");
  if (n_seqs == 0) return ASHKV_OK;
  if (!d_lengths || !d_out_lengths || !d_evicted_count ||
      (max_pages > 0 && (!d_page_mass || !d_page_ids || !d_out_page_ids || !d_out_mass || !d_evicted)))
    return refuse(kName, "null device pointer");
  if (page_ids_stride < max_pages || mass_stride < max_pages) return refuse(kName, "row strides must hold max_pages entries");
  launch_overlapped(evict_kernel, dim3(unsigned(n_seqs)), dim3(kKeepThreads), 0, as_stream(stream), d_page_mass, mass_stride,
                    d_page_ids, page_ids_stride, d_lengths, max_pages, tokens_per_page, budget, sink, recent,
                    d_out_page_ids, d_out_mass, d_out_lengths, d_evicted, d_evicted_count);
  return check_launch(kName);
}
