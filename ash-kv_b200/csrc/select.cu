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

// A warp per (listed page, key head): lane l keeps the extremes of channels
// l * D/32 .. over the page's tokens.  Bound by reading the keys once.
template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsParams p) {
  constexpr int N = D / 32, W = N / 2;  // channels, 32-bit words per lane
  const int lane = threadIdx.x & 31;
  const int64_t n = p.count ? min(max(*p.count, 0), p.max_entries) : p.max_entries;
  const int64_t stride = int64_t(gridDim.x) * (blockDim.x >> 5);
  for (int64_t i = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); i < n * p.heads; i += stride) {
    const int64_t entry = i / p.heads;
    const int h = int(i % p.heads);
    const int32_t id = p.list[entry];
    bool ok = id >= 0 && id < p.n_pages && p.tier[id] == 0;
    int32_t l = 0, ts = 0;
    if (ok) {
      l = p.layer_id[id];
      ts = p.token_start[id];
      ok = l >= 0 && l < p.n_layers && ts >= 0 && int64_t(ts) + p.T <= p.pool_tokens;
    }
    if (!ok) {
      if (lane == 0) flag(p.status, ASHKV_FLAG_INDEX_RANGE);
      continue;
    }
    const int nt = p.valid ? max(0, min(p.valid[entry], p.T)) : p.T;
    const uint16_t* k = reinterpret_cast<const uint16_t*>(p.layer_k[l]) + int64_t(ts) * p.row_stride + h * D + lane * N;
    float lo[N], hi[N];
#pragma unroll
    for (int c = 0; c < N; ++c) { lo[c] = INFINITY; hi[c] = -INFINITY; }
    auto take = [&](const uint32_t (&w)[W]) {
#pragma unroll
      for (int c = 0; c < W; ++c) {  // fminf / fmaxf pass over a NaN
        lo[2 * c] = fminf(lo[2 * c], bf16lo(w[c])); hi[2 * c] = fmaxf(hi[2 * c], bf16lo(w[c]));
        lo[2 * c + 1] = fminf(lo[2 * c + 1], bf16hi(w[c])); hi[2 * c + 1] = fmaxf(hi[2 * c + 1], bf16hi(w[c]));
      }
    };
    auto load = [&](int t, uint32_t (&w)[W]) {
      if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(k + t * p.row_stride);
        w[0] = v.x; w[1] = v.y;
      } else {
        w[0] = *reinterpret_cast<const uint32_t*>(k + t * p.row_stride);
      }
    };
    int t = 0;
    for (; t + 8 <= nt; t += 8) {
      uint32_t w[8][W];
#pragma unroll
      for (int u = 0; u < 8; ++u) load(t + u, w[u]);
#pragma unroll
      for (int u = 0; u < 8; ++u) take(w[u]);
    }
    for (; t < nt; ++t) {
      uint32_t w[W];
      load(t, w);
      take(w);
    }
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const bool none = lo[c] > hi[c];  // no number in the channel
      lo[c] = none ? 0.0f : fmaxf(fminf(lo[c], kBf16Max), -kBf16Max);
      hi[c] = none ? 0.0f : fmaxf(fminf(hi[c], kBf16Max), -kBf16Max);
      amax = fmaxf(amax, fmaxf(fabsf(lo[c]), fabsf(hi[c])));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, off));
    const int e = bound_exponent(amax);
    // 2^-e, exact: e is in [-100, 122]
    const float unit = __uint_as_float(uint32_t(127 - e) << 23);
    int cl[4] = {0, 0, 0, 0}, ch[4] = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < N; ++c) {
      // a bound too small for fp32 in these units still rounds outwards
      cl[c] = lo[c] < 0.0f ? min(int(floorf(lo[c] * unit)), -1) : int(floorf(lo[c] * unit));
      ch[c] = hi[c] > 0.0f ? max(int(ceilf(hi[c] * unit)), 1) : int(ceilf(hi[c] * unit));
    }
    int8_t* out = p.codes + (int64_t(id) * p.heads + h) * 2 * D + lane * N;
    if constexpr (N == 4) {
      *reinterpret_cast<uint32_t*>(out) = pack4(cl[0], cl[1], cl[2], cl[3]);
      *reinterpret_cast<uint32_t*>(out + D) = pack4(ch[0], ch[1], ch[2], ch[3]);
    } else {
      *reinterpret_cast<uint16_t*>(out) = uint16_t(pack4(cl[0], cl[1], 0, 0));
      *reinterpret_cast<uint16_t*>(out + D) = uint16_t(pack4(ch[0], ch[1], 0, 0));
    }
    if (lane == 0) p.exponents[int64_t(id) * p.heads + h] = int8_t(e);
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
constexpr int kScorePages = 64;  // pages of a CTA

// A CTA per (kScorePages page positions, key head, sequence).  The group's
// queries are quantised once into shared memory; a warp then takes a page at a
// time, lane l the bytes 4l .. of lo or hi (D = 128: lanes cover lo, then hi).
template <int D>
__global__ void __launch_bounds__(kScoreWarps * 32) select_scores_kernel(const ScoreParams p) {
  constexpr int W = D / 4;  // 32-bit words of one bound
  extern __shared__ uint32_t s_q[];  // [group][2][W]: min(q8, 0), max(q8, 0); then [group] exponents
  const int b = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = pages_of(p.lengths[b], p.max_pages, p.T);
  const int j0 = blockIdx.x * kScorePages;
  if (j0 >= n) return;
  int* s_e = reinterpret_cast<int*>(s_q + p.group * 2 * W);
  for (int g = warp; g < p.group; g += kScoreWarps) {
    const uint16_t* q = p.q + b * p.q_seq_stride + int64_t(h * p.group + g) * p.q_head_stride;
    constexpr int N = D / 32;
    float x[N], amax = 0.0f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      x[c] = bf16_to_f32(q[lane * N + c]);
      if (!(fabsf(x[c]) <= kBf16Max)) x[c] = 0.0f;
      amax = fmaxf(amax, fabsf(x[c]));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, off));
    const int e = bound_exponent(amax);
    const float unit = __uint_as_float(uint32_t(127 - e) << 23);
    int8_t* neg = reinterpret_cast<int8_t*>(s_q + g * 2 * W) + lane * N;
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int v = __float2int_rn(x[c] * unit);
      neg[c] = int8_t(min(v, 0));
      neg[D + c] = int8_t(max(v, 0));
    }
    if (lane == 0) s_e[g] = e;
  }
  __syncthreads();
  const int j1 = min(n, j0 + kScorePages);
  for (int j = j0 + warp; j < j1; j += kScoreWarps) {
    const int32_t id = p.page_ids[b * p.page_ids_stride + j];
    float best = -INFINITY;
    if (id >= 0 && id < p.n_pages) {
      const uint32_t* c = reinterpret_cast<const uint32_t*>(p.codes + (int64_t(id) * p.heads + h) * 2 * D);
      uint32_t w[2 * W / 32];
#pragma unroll
      for (int k = 0; k < 2 * W / 32; ++k) w[k] = c[lane + 32 * k];
      const int e = p.exponents[int64_t(id) * p.heads + h];
      for (int g = 0; g < p.group; ++g) {
        int dot = 0;
#pragma unroll
        for (int k = 0; k < 2 * W / 32; ++k) dot = __dp4a(int(w[k]), int(s_q[g * 2 * W + lane + 32 * k]), dot);
        dot = __reduce_add_sync(0xFFFFFFFFu, dot);
        best = fmaxf(best, times_pow2(dot, e + s_e[g]));
      }
    } else if (lane == 0) {
      flag(p.status, ASHKV_FLAG_INDEX_RANGE);
    }
    if (lane == 0) p.scores[(int64_t(b) * p.heads + h) * p.max_pages + j] = best;
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

struct KeepShared {
  uint32_t hist[256];
  uint32_t warp_a[32], warp_b[32];
  uint32_t prefix, need;
  uint32_t base_eq, base_keep;
};

// One CTA decides for each position j of a row of n scores whether it is kept
// -- the first `sink`, the last `recent`, and of the others the highest, of
// equal ones the first, `budget` in all -- and calls emit(j, kept, rank) with
// its rank among the kept (else among the dropped) in ascending order of j.
// The border score is found by four rounds over 8 bits of the keys each
// (a count per value of the digit among the keys that share the digits above).
template <class Emit>
__device__ void keep_highest(const float* __restrict__ score, int n, int budget, int sink, int recent, KeepShared& sm,
                             Emit emit) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool all = n <= budget;
  const int lo = sink, hi = n - recent;  // the positions that compete
  uint32_t border = 0, need = all ? 0u : uint32_t(budget - sink - recent);
  const bool rank = !all && need > 0;
  if (rank) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) sm.hist[tid] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kKeepThreads) {
        const uint32_t k = order_key(score[j]);
        if (shift == 24 || (k >> (shift + 8)) == (border >> (shift + 8))) atomicAdd(&sm.hist[(k >> shift) & 255u], 1u);
      }
      __syncthreads();
      if (warp == 0) {  // the digit, from the top, at which the count reaches `need`
        uint32_t v[8], sum = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          v[k] = sm.hist[255 - (lane * 8 + k)];
          sum += v[k];
        }
        uint32_t inc = sum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const uint32_t x = __shfl_up_sync(0xFFFFFFFFu, inc, off);
          if (lane >= off) inc += x;
        }
        uint32_t above = inc - sum;
        if (above < need && inc >= need) {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (above < need && above + v[k] >= need) {
              sm.prefix = border | (uint32_t(255 - (lane * 8 + k)) << shift);
              sm.need = need - above;
              break;
            }
            above += v[k];
          }
        }
      }
      __syncthreads();
      border = sm.prefix;
      need = sm.need;
    }
  }
  if (tid == 0) sm.base_eq = sm.base_keep = 0;
  __syncthreads();
  for (int j0 = 0; j0 < n; j0 += kKeepThreads) {
    const int j = j0 + tid;
    const bool on = j < n, mid = on && !all && j >= lo && j < hi;
    const uint32_t k = mid && rank ? order_key(score[j]) : 0u;
    const bool eq = mid && rank && k == border;
    const unsigned me = __ballot_sync(0xFFFFFFFFu, eq);
    if (lane == 0) sm.warp_a[warp] = __popc(me);
    __syncthreads();
    uint32_t before = sm.base_eq, total_eq = sm.base_eq;
    for (int w = 0; w < kKeepThreads / 32; ++w) {
      before += w < warp ? sm.warp_a[w] : 0u;
      total_eq += sm.warp_a[w];
    }
    before += __popc(me & ((1u << lane) - 1u));
    const bool keep = on && (!mid || (rank && (k > border || (eq && before < need))));
    const unsigned mk = __ballot_sync(0xFFFFFFFFu, keep);
    if (lane == 0) sm.warp_b[warp] = __popc(mk);
    __syncthreads();
    uint32_t kept = sm.base_keep, total_keep = sm.base_keep;
    for (int w = 0; w < kKeepThreads / 32; ++w) {
      kept += w < warp ? sm.warp_b[w] : 0u;
      total_keep += sm.warp_b[w];
    }
    kept += __popc(mk & ((1u << lane) - 1u));
    if (on) emit(j, keep, keep ? int(kept) : j - int(kept));
    __syncthreads();
    if (tid == 0) { sm.base_eq = total_eq; sm.base_keep = total_keep; }
    __syncthreads();
  }
}

__global__ void __launch_bounds__(kKeepThreads) select_keep_kernel(const float* __restrict__ scores,
                                                                   const int32_t* __restrict__ lengths, int heads,
                                                                   int max_pages, int T, int budget, int sink,
                                                                   int recent, int32_t* __restrict__ selected,
                                                                   int32_t* __restrict__ count, uint32_t* status) {
  __shared__ KeepShared sm;
  const int64_t row = blockIdx.x;
  const int b = int(row / heads);
  const int n = pages_of(lengths[b], max_pages, T);
  int32_t* out = selected + row * budget;
  keep_highest(scores + row * max_pages, n, budget, sink, recent, sm, [&](int j, bool kept, int at) {
    if (kept) out[at] = j;
  });
  const int kept = min(n, budget);
  for (int i = kept + threadIdx.x; i < budget; i += kKeepThreads) out[i] = -1;
  if (threadIdx.x == 0) {
    count[row] = kept;
    if (lengths[b] < 0 || int64_t(lengths[b]) > int64_t(max_pages) * T) flag(status, ASHKV_FLAG_INDEX_RANGE);
  }
}

__global__ void __launch_bounds__(kKeepThreads) evict_kernel(
    const float* __restrict__ mass, int64_t mass_stride, const int32_t* __restrict__ page_ids, int64_t page_ids_stride,
    const int32_t* __restrict__ lengths, int max_pages, int T, int budget, int sink, int recent,
    int32_t* __restrict__ out_ids, float* __restrict__ out_mass, int32_t* __restrict__ out_lengths,
    int32_t* __restrict__ evicted, int32_t* __restrict__ evicted_count) {
  __shared__ KeepShared sm;
  const int64_t b = blockIdx.x;
  const int n = pages_of(lengths[b], max_pages, T);
  const float* m = mass + b * mass_stride;
  const int32_t* ids = page_ids + b * page_ids_stride;
  int32_t* oi = out_ids + b * max_pages;
  float* om = out_mass + b * max_pages;
  int32_t* ev = evicted + b * max_pages;
  keep_highest(m, n, budget, sink, recent, sm, [&](int j, bool kept, int at) {
    if (kept) {
      oi[at] = ids[j];
      om[at] = m[j];
    } else {
      ev[at] = ids[j];
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
  const int64_t warps = int64_t(max_entries) * p.heads;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const unsigned grid = unsigned(std::min<int64_t>((warps + 7) / 8, int64_t(sms) * 8));
  if (kv->head_dim == 64) page_bounds_kernel<64><<<grid, 256, 0, as_stream(stream)>>>(p);
  else page_bounds_kernel<128><<<grid, 256, 0, as_stream(stream)>>>(p);
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
    const dim3 grid(unsigned((max_pages + kScorePages - 1) / kScorePages), unsigned(heads_kv), unsigned(n_seqs));
    const size_t smem = size_t(group) * (2 * head_dim + 4);
    if (head_dim == 64) select_scores_kernel<64><<<grid, kScoreWarps * 32, smem, st>>>(p);
    else select_scores_kernel<128><<<grid, kScoreWarps * 32, smem, st>>>(p);
    const ashkv_status_t rc = check_launch(kName);
    if (rc != ASHKV_OK) return rc;
  }
  select_keep_kernel<<<unsigned(n_seqs * heads_kv), kKeepThreads, 0, st>>>(
      d_scratch, d_lengths, heads_kv, max_pages, tokens_per_page, budget, sink, recent, d_selected, d_selected_count,
      d_status);
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
  evict_kernel<<<unsigned(n_seqs), kKeepThreads, 0, as_stream(stream)>>>(
      d_page_mass, mass_stride, d_page_ids, page_ids_stride, d_lengths, max_pages, tokens_per_page, budget, sink,
      recent, d_out_page_ids, d_out_mass, d_out_lengths, d_evicted, d_evicted_count);
  return check_launch(kName);
}
