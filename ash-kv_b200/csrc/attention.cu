// Attention of one new token per sequence over paged KV whose pages may be in
// any tier (ashkv_decode_attention).
//
// With s[t] = scale * q . K[t] the result is sum_t 2^(s2[t] - M) V[t] / sum_t
// 2^(s2[t] - M), s2 = s * log2(e), for any M; one pass over the pages keeps a
// running M and the two sums.  The work is split over the length of the pages:
// for each key head the pages of all sequences form one row, cut into equal
// ranges, one warp each, so a batch of one long sequence and a ragged batch
// fill the GPU alike.  A range that reaches into several sequences leaves one
// partial result per sequence (normalised, with its log2-sum); the join kernel
// weighs the partials of each sequence by 2^(their log2-sum - the total).
#include <algorithm>
#include <cstdio>

#include "common.cuh"
#include "fp8_conv.cuh"
#include "page_layout.cuh"

namespace ashkv {
namespace {

constexpr int kWarpsA = 4;          // warps of a CTA, each a worker of its own
constexpr int kWorkersPerSm = 12;   // resident worker warps per SM
constexpr int kQ = 8;               // query heads of one worker
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kJoinThreads = 128;

struct AttnParams {
  // pages
  const int8_t* tier;
  const int32_t* layer_id;
  const int32_t* token_start;
  const int32_t* page_slot;
  int64_t n_pages;
  const uint64_t* layer_k;
  const uint64_t* layer_v;
  int64_t pool_tokens, row_stride;
  int32_t n_layers, T, row_len, outlier_cap;
  Store store[kTiers];
  // the call
  const uint16_t* q;
  int64_t q_seq_stride, q_head_stride;
  int32_t n_seqs, heads_q, heads_kv, group, q_chunks;
  const int32_t* page_ids;
  int64_t page_ids_stride;
  int32_t max_pages;
  const int32_t* lengths;
  const int32_t* selected;
  const int32_t* selected_count;
  int32_t max_selected;
  float scale2;  // scale * log2(e)
  float* mass;
  int64_t mass_stride;
  float decay;
  uint16_t* out;
  float* lse;
  // scratch
  int32_t ranges;     // worker warps per key head and query chunk
  float* part_o;      // [ranges + n_seqs][heads_q][D], each divided by its sum
  float* part_lse2;   // [ranges + n_seqs][heads_q]
  float* page_lse2;   // [n_seqs][max_pages][heads_q], with mass only
  uint32_t* status;
};

__device__ __forceinline__ void flag(uint32_t* status, uint32_t f) {
  if (status) atomicOr(status, f);
}

// Tokens of sequence b that its page list can hold.
__device__ __forceinline__ int64_t seq_tokens(const AttnParams& p, int b) {
  const int64_t len = p.lengths[b], most = int64_t(p.max_pages) * p.T;
  return len < 0 ? 0 : (len > most ? most : len);
}
// Entries of the list that key head hk of sequence b attends.
__device__ __forceinline__ int list_len(const AttnParams& p, int b, int hk) {
  if (p.selected) return max(0, min(p.selected_count[int64_t(b) * p.heads_kv + hk], p.max_selected));
  return int((seq_tokens(p, b) + p.T - 1) / p.T);
}

// Pages of key head hk's lists before sequence b (warp-collective; b <= n_seqs).
__device__ int lists_before(const AttnParams& p, int b, int hk) {
  const int lane = threadIdx.x & 31;
  int sum = 0;
  for (int i = lane; i < b; i += 32) sum += list_len(p, i, hk);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
  return sum;
}
// Pages per range; every range but the last of the row has as many.
__device__ __forceinline__ int range_len(const AttnParams& p, int total) { return max(1, (total + p.ranges - 1) / p.ranges); }

// The page behind list entry i of (sequence b, key head hk).
struct PageRef {
  const uint8_t* k;   // BF16: the K row of the page's first token; else the slot
  const uint8_t* v;   // BF16: the V row
  int32_t format;     // ASHKV_PAGE_*, ASHKV_PAGE_NONE for a page to leave out
  int32_t pos;        // position in the sequence
};
__device__ PageRef resolve(const AttnParams& p, int b, int hk, int i) {
  PageRef r{nullptr, nullptr, ASHKV_PAGE_NONE, i};
  if (p.selected) {
    r.pos = p.selected[(int64_t(b) * p.heads_kv + hk) * p.max_selected + i];
    if (r.pos < 0 || int64_t(r.pos) * p.T >= seq_tokens(p, b)) {
      flag(p.status, ASHKV_FLAG_INDEX_RANGE);
      r.pos = 0;
      return r;
    }
  }
  const int32_t id = p.page_ids[int64_t(b) * p.page_ids_stride + r.pos];
  bool ok = id >= 0 && id < p.n_pages;
  const int t = ok ? p.tier[id] : -1;
  ok = ok && t >= 0 && t < kTiers && (t == 0 || p.store[t].format != ASHKV_PAGE_NONE);
  if (ok && t == 0) {
    const int32_t l = p.layer_id[id], ts = p.token_start[id];
    ok = l >= 0 && l < p.n_layers && ts >= 0 && int64_t(ts) + p.T <= p.pool_tokens;
    if (ok) {
      const int64_t off = int64_t(ts) * p.row_stride * 2;
      r.k = reinterpret_cast<const uint8_t*>(p.layer_k[l]) + off;
      r.v = reinterpret_cast<const uint8_t*>(p.layer_v[l]) + off;
    }
  } else if (ok) {
    const int32_t s = p.page_slot[id];
    ok = s >= 0 && s < p.store[t].n_slots;
    if (ok) r.k = p.store[t].data + int64_t(s) * p.store[t].slot_bytes;
  }
  if (ok) r.format = t == 0 ? ASHKV_PAGE_BF16 : p.store[t].format;
  else flag(p.status, ASHKV_FLAG_INDEX_RANGE);
  return r;
}

// N neighbouring values (columns c .. c + N - 1) of row r of a page (its K rows, then its V rows).
template <int N, int BITS>
__device__ __forceinline__ void nbit_values(const AttnParams& p, const uint8_t* slot, int64_t e, float (&x)[N]) {
  const int64_t E = 2 * int64_t(p.T) * p.row_len;
  const float delta = bf16_to_f32(reinterpret_cast<const uint16_t*>(slot + nbit_delta_off())[e / 32]);
  const uint8_t* codes = slot + nbit_codes_off(E);
  constexpr float half = float((1 << BITS) - 1) * 0.5f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t bit = (e + i) * BITS;
    const int c = (codes[bit >> 3] >> (8 - BITS - int(bit & 7))) & ((1 << BITS) - 1);
    x[i] = bf16_to_f32(f32_to_bf16(__fmul_rn(float(c) - half, delta)));
  }
  const uint32_t* ent = reinterpret_cast<const uint32_t*>(slot + nbit_entries_off(E, BITS));
  uint32_t lo = 0, n = min(*reinterpret_cast<const uint32_t*>(slot), uint32_t(p.outlier_cap));
  for (uint32_t hi = n; lo < hi;) {  // first entry at element e or later
    const uint32_t mid = (lo + hi) / 2;
    if ((ent[mid] >> 16) < uint32_t(e)) lo = mid + 1;
    else hi = mid;
  }
  for (; lo < n && (ent[lo] >> 16) < uint32_t(e) + N; ++lo)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((ent[lo] >> 16) == uint32_t(e) + i) x[i] = bf16_to_f32(uint16_t(ent[lo] & 0xFFFFu));
}
template <int N>
__device__ void page_values(const AttnParams& p, const PageRef& pg, int r, int c, float (&x)[N]) {
  const int64_t e = int64_t(r) * p.row_len + c, E = 2 * int64_t(p.T) * p.row_len;
  switch (pg.format) {
    case ASHKV_PAGE_BF16: {
      const bool isv = r >= p.T;
      const uint16_t* row = reinterpret_cast<const uint16_t*>(isv ? pg.v : pg.k) + int64_t(isv ? r - p.T : r) * p.row_stride + c;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = bf16_to_f32(row[i]);
      break;
    }
    case ASHKV_PAGE_INT8: {
      const float s = f16_to_f32(reinterpret_cast<const uint16_t*>(pg.k)[r]) * (1.0f / 127.0f);
      const int8_t* q = reinterpret_cast<const int8_t*>(pg.k) + int8_codes_offset(p.T) + e;
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = float(q[i]) * s;
      break;
    }
    case ASHKV_PAGE_FP8: {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = bf16lo(bf16x2_from_fp8x2(pg.k[e + i]));
      break;
    }
    case ASHKV_PAGE_INT4: {
      const float s = bf16_to_f32(reinterpret_cast<const uint16_t*>(pg.k)[e / 64]) * (1.0f / 7.0f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint8_t w = pg.k[E / 32 + (e + i) / 2];
        x[i] = float(int((e + i) & 1 ? w & 15 : w >> 4) - 8) * s;
      }
      break;
    }
    case ASHKV_PAGE_NBIT4: nbit_values<N, 4>(p, pg.k, e, x); break;
    default: nbit_values<N, 2>(p, pg.k, e, x); break;
  }
}

// A warp per (range of pages, key head, up to kQ of its query heads).  Lane l
// holds channels l * D/32 .. of the queries and of the results.
template <int D>
__global__ void __launch_bounds__(kWarpsA * 32) decode_partials_kernel(const AttnParams p) {
  constexpr int N = D / 32;
  const int lane = threadIdx.x & 31;
  const int w = int(blockIdx.x) * kWarpsA + int(threadIdx.x >> 5);
  const int cells = p.heads_kv * p.q_chunks;
  const int range = w / cells, cell = w % cells;
  if (range >= p.ranges) return;
  const int hk = cell % p.heads_kv, q0 = (cell / p.heads_kv) * kQ;
  const int nq = min(kQ, p.group - q0), hq0 = hk * p.group + q0;
  const int total = lists_before(p, p.n_seqs, hk), len = range_len(p, total);
  int64_t pos = int64_t(range) * len;
  const int64_t end = min(pos + len, int64_t(total));
  if (pos >= end) return;
  int b = 0, before = 0;
  for (;; ++b) {  // the sequence that the range starts in
    const int n = list_len(p, b, hk);
    if (before + n > pos) break;
    before += n;
  }
  for (; pos < end; ++b) {
    const int n = list_len(p, b, hk);
    if (n == 0) continue;
    const int i0 = int(pos - before), i1 = int(min(int64_t(n), end - before));
    float q[kQ][N], o[kQ][N], m[kQ], l[kQ];
    const int64_t tokens = seq_tokens(p, b);
    for (int g = 0; g < kQ; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.0f;
      for (int i = 0; i < N; ++i) {
        o[g][i] = 0.0f;
        q[g][i] = g < nq ? bf16_to_f32(p.q[b * p.q_seq_stride + (hq0 + g) * p.q_head_stride + lane * N + i]) : 0.0f;
      }
    }
    for (int i = i0; i < i1; ++i) {
      const PageRef pg = resolve(p, b, hk, i);
      const int nt = pg.format == ASHKV_PAGE_NONE ? 0 : int(min(int64_t(p.T), tokens - int64_t(pg.pos) * p.T));
      float pm[kQ], pl[kQ];  // the page's own maximum and sum
      for (int g = 0; g < kQ; ++g) { pm[g] = -INFINITY; pl[g] = 0.0f; }
      for (int t = 0; t < nt; ++t) {
        float k[N], v[N];
        page_values<N>(p, pg, t, hk * D + lane * N, k);
        page_values<N>(p, pg, p.T + t, hk * D + lane * N, v);
        for (int g = 0; g < kQ; ++g) {
          float s = 0.0f;
          for (int c = 0; c < N; ++c) s = fmaf(q[g][c], k[c], s);
          for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, off);
          s *= p.scale2;
          const float mn = fmaxf(m[g], s), ref = mn == -INFINITY ? 0.0f : mn;
          const float a = exp2f(m[g] - ref), e = exp2f(s - ref);
          l[g] = l[g] * a + e;
          for (int c = 0; c < N; ++c) o[g][c] = fmaf(e, v[c], o[g][c] * a);
          m[g] = mn;
          const float pn = fmaxf(pm[g], s), pref = pn == -INFINITY ? 0.0f : pn;
          pl[g] = pl[g] * exp2f(pm[g] - pref) + exp2f(s - pref);
          pm[g] = pn;
        }
      }
      if (p.mass && lane == 0)
        for (int g = 0; g < nq; ++g)
          p.page_lse2[(int64_t(b) * p.max_pages + pg.pos) * p.heads_q + hq0 + g] =
              nt > 0 ? (pm[g] == -INFINITY ? 0.0f : pm[g]) + log2f(pl[g]) : -INFINITY;
    }
    const int64_t slot = int64_t(range + b) * p.heads_q + hq0;
    for (int g = 0; g < nq; ++g) {
      const float inv = l[g] == 0.0f ? 0.0f : 1.0f / l[g];
      for (int c = 0; c < N; ++c) p.part_o[(slot + g) * D + lane * N + c] = o[g][c] * inv;
      if (lane == 0) p.part_lse2[slot + g] = (m[g] == -INFINITY ? 0.0f : m[g]) + log2f(l[g]);
    }
    pos = before + i1;
    before += n;
  }
}

// log2-sum over the partials of (sequence b, query head hq): ranges r0 .. r1.
__device__ __forceinline__ void join_range(const AttnParams& p, int b, int hk, int& r0, int& r1) {
  const int before = lists_before(p, b, hk), n = list_len(p, b, hk);
  int total = before + n;
  const int lane = threadIdx.x & 31;
  int rest = 0;
  for (int i = b + 1 + lane; i < p.n_seqs; i += 32) rest += list_len(p, i, hk);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) rest += __shfl_xor_sync(0xFFFFFFFFu, rest, off);
  total += rest;
  const int len = range_len(p, total);
  r0 = before / len;
  r1 = n == 0 ? r0 - 1 : (before + n - 1) / len;
}
__device__ __forceinline__ float join_lse2(const AttnParams& p, int b, int hq, int r0, int r1) {  // warp-collective
  const int lane = threadIdx.x & 31;
  float m = -INFINITY, l = 0.0f;
  for (int r = r0 + lane; r <= r1; r += 32) {
    const float x = p.part_lse2[int64_t(r + b) * p.heads_q + hq];
    const float mn = x > m || x != x ? x : m, ref = mn == -INFINITY ? 0.0f : mn;
    l = l * exp2f(m - ref) + exp2f(x - ref);
    m = mn;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, off), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, off);
    const float mn = m2 > m || m2 != m2 ? m2 : m, ref = mn == -INFINITY ? 0.0f : mn;
    l = l * exp2f(m - ref) + l2 * exp2f(m2 - ref);
    m = mn;
  }
  return (m == -INFINITY ? 0.0f : m) + log2f(l);  // no tokens: log2(0) = -inf
}

// Blocks 0 .. n_seqs * heads_q - 1: one result row each.  With mass, then
// ceil(max_pages / kJoinThreads) blocks per sequence for its pages' mass.
template <int D>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const AttnParams p) {
  const int tid = threadIdx.x;
  const int64_t n_out = int64_t(p.n_seqs) * p.heads_q;
  if (blockIdx.x < n_out) {
    const int b = int(blockIdx.x / p.heads_q), hq = int(blockIdx.x % p.heads_q);
    if (tid == 0 && hq % p.group == 0) {  // what list_len cut
      const int32_t n = p.selected ? p.selected_count[int64_t(b) * p.heads_kv + hq / p.group] : 0;
      if (p.lengths[b] != seq_tokens(p, b) || n < 0 || n > p.max_selected) flag(p.status, ASHKV_FLAG_INDEX_RANGE);
    }
    int r0, r1;
    join_range(p, b, hq / p.group, r0, r1);
    const float lse2 = join_lse2(p, b, hq, r0, r1);
    if (tid < D) {
      float acc = 0.0f;
      for (int r = r0; r <= r1; ++r) {
        const int64_t at = int64_t(r + b) * p.heads_q + hq;
        const float x = p.part_lse2[at];
        if (x != -INFINITY) acc = fmaf(exp2f(x - lse2), p.part_o[at * D + tid], acc);
      }
      p.out[int64_t(blockIdx.x) * D + tid] = f32_to_bf16(acc);
    }
    if (tid == 0 && p.lse) p.lse[blockIdx.x] = lse2 * kLn2;
    return;
  }
  extern __shared__ float s_lse[];  // [heads_q]
  const int64_t mb = int64_t(blockIdx.x) - n_out;
  const int per = (p.max_pages + kJoinThreads - 1) / kJoinThreads;
  const int b = int(mb / per), j = int(mb % per) * kJoinThreads + tid;
  for (int hq = tid >> 5; hq < p.heads_q; hq += kJoinThreads / 32) {
    int r0, r1;
    join_range(p, b, hq / p.group, r0, r1);
    const float lse2 = join_lse2(p, b, hq, r0, r1);
    if ((tid & 31) == 0) s_lse[hq] = lse2;
  }
  __syncthreads();
  if (int64_t(j) * p.T >= seq_tokens(p, b)) return;
  const float* pl = p.page_lse2 + (int64_t(b) * p.max_pages + j) * p.heads_q;
  float sum = 0.0f;
  for (int h = 0; h < p.heads_q; ++h)
    if (pl[h] != -INFINITY) sum += exp2f(pl[h] - s_lse[h]);
  float* m = p.mass + int64_t(b) * p.mass_stride + j;
  *m = fmaf(p.decay, *m, sum);
}

int ranges_for(int64_t n_seqs, int heads_kv, int q_chunks, int64_t pages_per_list) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t fit = std::max<int64_t>(1, int64_t(sms) * kWorkersPerSm / (int64_t(heads_kv) * q_chunks));
  return int(std::max<int64_t>(1, std::min<int64_t>(fit, n_seqs * pages_per_list)));
}
int q_chunks_for(int heads_q, int heads_kv) { return (heads_q / heads_kv + kQ - 1) / kQ; }

bool row_ok(int64_t row) { return row == 128 || row == 256 || row == 512 || row == 1024 || row == 2048; }

// The page description of a call; the message of what is wrong with it, or nullptr.
const char* copy_pages(const ashkv_paged_kv_t* kv, AttnParams& p) {
  if (!kv) return "null page description";
  if (kv->head_dim != 64 && kv->head_dim != 128) return "head_dim must be 64 or 128";
  if (kv->heads_kv <= 0 || kv->tokens_per_page <= 0 || kv->n_layers <= 0 || kv->n_pages < 0 || kv->pool_tokens < 0 ||
      kv->outlier_cap < 0 || kv->tokens_per_page > 65536 || kv->heads_kv > 65536)
    return "heads_kv, tokens_per_page and n_layers must be positive, sizes not negative";
  const int64_t row = int64_t(kv->heads_kv) * kv->head_dim;
  if (kv->row_stride < row || kv->row_stride % 8) return "row_stride must be a multiple of 8 and at least heads_kv * head_dim";
  if (!kv->d_tier || !kv->d_layer_id || !kv->d_token_start || !kv->d_page_slot || !kv->d_layer_k || !kv->d_layer_v)
    return "null device pointer";
  if (!copy_stores(kv->stores, p.store, true)) return "bad tier store table (store 0 must be the BF16 pool)";
  bool any = false;
  for (int t = 1; t < kTiers; ++t) {
    if (p.store[t].format == ASHKV_PAGE_NONE) continue;
    any = true;
    if (p.store[t].slot_bytes < ashkv_page_slot_bytes(p.store[t].format, kv->tokens_per_page, int32_t(row), kv->outlier_cap))
      return "a tier store's slots are smaller than its format needs";
  }
  const int64_t E = 2 * int64_t(kv->tokens_per_page) * row;
  if (any && (!row_ok(row) || E % 1024 || E > 65536))
    return "with stores heads_kv * head_dim must be 128, 256, 512, 1024 or 2048 and a page a multiple of 1024 and at "
           "most 65536 elements";
  p.tier = kv->d_tier; p.layer_id = kv->d_layer_id; p.token_start = kv->d_token_start; p.page_slot = kv->d_page_slot;
  p.n_pages = kv->n_pages; p.layer_k = kv->d_layer_k; p.layer_v = kv->d_layer_v;
  p.pool_tokens = kv->pool_tokens; p.row_stride = kv->row_stride; p.n_layers = kv->n_layers;
  p.T = kv->tokens_per_page; p.row_len = int32_t(row); p.outlier_cap = kv->outlier_cap; p.heads_kv = kv->heads_kv;
  return nullptr;
}

ashkv_status_t refuse(const char* what, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", what, why);
  set_message(text);
  return ASHKV_BAD_ARGUMENT;
}

template <int D>
ashkv_status_t launch_decode(const AttnParams& p, cudaStream_t st) {
  const int64_t workers = int64_t(p.ranges) * p.heads_kv * p.q_chunks;
  decode_partials_kernel<D><<<unsigned((workers + kWarpsA - 1) / kWarpsA), kWarpsA * 32, 0, st>>>(p);
  int64_t blocks = int64_t(p.n_seqs) * p.heads_q;
  if (p.mass) blocks += int64_t(p.n_seqs) * ((p.max_pages + kJoinThreads - 1) / kJoinThreads);
  decode_join_kernel<D><<<unsigned(blocks), kJoinThreads, p.mass ? size_t(p.heads_q) * 4 : 0, st>>>(p);
  return check_launch("ashkv_decode_attention");
}

}  // namespace
}  // namespace ashkv

using namespace ashkv;

extern "C" int64_t ashkv_decode_scratch_floats(int32_t n_seqs, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                                               int32_t pages_per_list, int32_t with_mass) {
  if (n_seqs < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || head_dim <= 0 || pages_per_list < 0) return -1;
  const int64_t slots = int64_t(ranges_for(n_seqs, heads_kv, q_chunks_for(heads_q, heads_kv), pages_per_list)) + n_seqs;
  int64_t n = slots * heads_q * (int64_t(head_dim) + 1);
  if (with_mass) n += int64_t(n_seqs) * pages_per_list * heads_q;
  return n;
}

extern "C" ashkv_status_t ashkv_decode_attention(
    const ashkv_paged_kv_t* kv, const void* d_q, int64_t q_seq_stride, int64_t q_head_stride, int32_t n_seqs,
    int32_t heads_q, const int32_t* d_page_ids, int64_t page_ids_stride, int32_t max_pages, const int32_t* d_lengths,
    const int32_t* d_selected, const int32_t* d_selected_count, int32_t max_selected, float scale, float* d_page_mass,
    int64_t mass_stride, float decay, void* d_out, float* d_lse, float* d_scratch, uint32_t* d_status, void* stream) {
  constexpr const char* kName = "ashkv_decode_attention";
  AttnParams p{};
  if (const char* why = copy_pages(kv, p)) return refuse(kName, why);
  if (n_seqs < 0 || max_pages < 0 || heads_q <= 0 || heads_q % p.heads_kv)
    return refuse(kName, "negative size, or heads_q not a multiple of heads_kv");
  if (int64_t(n_seqs) * heads_q > (int64_t(1) << 24) || heads_q > 8192) return refuse(kName, "too many query rows");
  const int64_t width = d_selected ? max_selected : max_pages;
  if (width < 0 || int64_t(n_seqs) * width > 0x7FFFFFFFLL || int64_t(n_seqs) * max_pages > 0x7FFFFFFFLL)
    return refuse(kName, "too many list entries");
  if (d_selected && (!d_selected_count || d_page_mass)) return refuse(kName, "d_selected needs its counts and takes no mass");
  if (n_seqs == 0) return ASHKV_OK;
  if (!d_q || (!d_page_ids && max_pages > 0) || !d_lengths || !d_out || !d_scratch || !aligned(d_scratch, 16))
    return refuse(kName, "null or misaligned device pointer");
  if (page_ids_stride < max_pages || (d_page_mass && mass_stride < max_pages))
    return refuse(kName, "row strides must hold max_pages entries");
  p.q = static_cast<const uint16_t*>(d_q);
  p.q_seq_stride = q_seq_stride; p.q_head_stride = q_head_stride;
  p.n_seqs = n_seqs; p.heads_q = heads_q; p.group = heads_q / p.heads_kv;
  p.q_chunks = q_chunks_for(heads_q, p.heads_kv);
  p.page_ids = d_page_ids; p.page_ids_stride = page_ids_stride; p.max_pages = max_pages; p.lengths = d_lengths;
  p.selected = d_selected; p.selected_count = d_selected_count; p.max_selected = max_selected;
  p.scale2 = scale * kLog2e;
  p.mass = d_page_mass; p.mass_stride = mass_stride; p.decay = decay;
  p.out = static_cast<uint16_t*>(d_out); p.lse = d_lse; p.status = d_status;
  p.ranges = ranges_for(n_seqs, p.heads_kv, p.q_chunks, width);
  const int64_t rows = (int64_t(p.ranges) + n_seqs) * heads_q;
  p.part_o = d_scratch;
  p.part_lse2 = p.part_o + rows * kv->head_dim;
  p.page_lse2 = p.part_lse2 + rows;
  return kv->head_dim == 64 ? launch_decode<64>(p, as_stream(stream)) : launch_decode<128>(p, as_stream(stream));
}
