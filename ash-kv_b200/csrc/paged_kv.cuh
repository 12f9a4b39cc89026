// The pages of a call as ashkv_paged_kv_t describes them, and what the operators over page lists share:
// checks of the description, the sequence of a row, the place of a token.
#pragma once

#include <cstdio>

#include "common.cuh"
#include "page_layout.cuh"

namespace ashkv {
namespace {

// Entries of all lists of a call: what is added to a position (ranges, a batch looked up ahead) stays inside an int.
constexpr int64_t kMostEntries = 0x7FFFFFFFLL - 65536;

struct PagedKV {
  const int8_t* tier;
  const int32_t* layer_id;
  const int32_t* token_start;
  const int32_t* page_slot;
  int64_t n_pages;
  const uint64_t* layer_k;
  const uint64_t* layer_v;
  int64_t pool_tokens, row_stride;
  int32_t n_layers, T, row_len, outlier_cap, heads_kv;
  Store store[kTiers];
};

// Sequences and their lists.
struct PageLists {
  const int32_t* page_ids;
  int64_t page_ids_stride;
  int32_t max_pages;
  const int32_t* lengths;
  const int32_t* starts;  // [n_seqs + 1]: rows of the new tokens
  int32_t n_seqs;
  uint32_t* status;
};

__device__ __forceinline__ void flag(uint32_t* status, uint32_t f) {
  if (status) atomicOr(status, f);
}

inline bool row_ok(int64_t row) { return row == 128 || row == 256 || row == 512 || row == 1024 || row == 2048; }

// The page description of a call; the message of what is wrong with it, or nullptr.
template <class P>
const char* copy_pages(const ashkv_paged_kv_t* kv, P& p, bool any_head_dim = false) {
  if (!kv) return "null page description";
  if (!any_head_dim && kv->head_dim != 64 && kv->head_dim != 128) return "head_dim must be 64 or 128";
  if (kv->head_dim <= 0 || kv->head_dim % 8) return "head_dim must be a positive multiple of 8";
  if (kv->heads_kv <= 0 || kv->tokens_per_page <= 0 || kv->n_layers <= 0 || kv->n_pages < 0 || kv->pool_tokens < 0 ||
      kv->outlier_cap < 0 || kv->tokens_per_page > 65536 || kv->heads_kv > 65536)
    return "heads_kv, tokens_per_page and n_layers must be positive, sizes not negative";
  const int64_t row = int64_t(kv->heads_kv) * kv->head_dim;
  if (row > 0x7FFFFFFF || kv->row_stride > 0x3FFFFFFF || kv->tokens_per_page * kv->row_stride > 0x3FFFFFFF)
    return "a page must span less than 2^31 bytes";
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

// Page lists of a call with rows of new tokens.
inline const char* copy_lists(const int32_t* d_page_ids, int64_t page_ids_stride, int32_t max_pages,
                              const int32_t* d_lengths, const int32_t* d_starts, int32_t n_seqs, int64_t n_rows,
                              uint32_t* d_status, PageLists& l) {
  if (n_seqs < 0 || max_pages < 0 || n_rows < 0 || n_rows > kMostEntries || n_seqs > kMostEntries) return "bad size";
  if (int64_t(n_seqs) * max_pages > kMostEntries) return "too many list entries";
  if (n_seqs > 0 && n_rows > 0 && ((!d_page_ids && max_pages > 0) || !d_lengths || !d_starts)) return "null device pointer";
  if (page_ids_stride < max_pages) return "page_ids_stride must hold max_pages entries";
  l = PageLists{d_page_ids, page_ids_stride, max_pages, d_lengths, d_starts, n_seqs, d_status};
  return nullptr;
}

inline ashkv_status_t refuse(const char* what, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", what, why);
  set_message(text);
  return ASHKV_BAD_ARGUMENT;
}

// Launches a kernel over page lists in the manner of launch_overlapped, whose rules it follows.
template <class... Params, class... Args>
cudaError_t launch_paged(void (*kernel)(Params...), int64_t blocks, int threads, size_t smem, void* stream, Args&&... args) {
  return launch_overlapped(kernel, dim3(unsigned(blocks)), dim3(unsigned(threads)), smem, as_stream(stream), args...);
}

// The sequence b with starts[b] <= i < starts[b + 1], or -1 (warp-collective; starts ascend).  A step
// looks at 32 of the starts that are left.
__device__ __forceinline__ int sequence_of(const PageLists& l, int64_t i) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = l.n_seqs;  // how many of starts[1 ..] are at most i lies in [lo, hi]
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32;
    const int64_t k = lo + int64_t(lane) * step;
    const int c = __popc(__ballot_sync(0xFFFFFFFFu, k < hi && l.starts[k + 1] <= i));
    if (step == 1 || c == 0) {
      lo += c;
      break;
    }
    hi = int(min(int64_t(hi), lo + int64_t(c) * step));
    lo += (c - 1) * step + 1;
  }
  if (lo >= l.n_seqs) return -1;
  const int64_t s0 = l.starts[lo], s1 = l.starts[lo + 1];
  if (s0 <= i && i < s1) return lo;
  if (lane == 0 && i >= l.starts[0]) flag(l.status, ASHKV_FLAG_INDEX_RANGE);  // starts that do not ascend
  return -1;
}

// What the table says of a page; of no such page, tier -1.
struct Entry {
  int32_t tier, layer, start, slot;
};
__device__ __forceinline__ Entry entry_of(const PagedKV& p, int32_t id) {
  if (id < 0 || id >= p.n_pages) return Entry{-1, 0, 0, 0};
  return Entry{p.tier[id], p.layer_id[id], p.token_start[id], p.page_slot[id]};
}
// Where a page lies: its format, and its first K and V row in the pool or (k) its slot.  No such page: -1.
struct Place {
  int32_t format;
  uint8_t *k, *v;
};
__device__ __forceinline__ Place place_of(const PagedKV& p, const Entry& e) {
  Place at{-1, nullptr, nullptr};
  const auto [tier, layer, start, slot] = e;
  if (tier == 0) {
    if (layer < 0 || layer >= p.n_layers || start < 0 || int64_t(start) + p.T > p.pool_tokens) return at;
    at.format = ASHKV_PAGE_BF16;
    at.k = reinterpret_cast<uint8_t*>(p.layer_k[layer]) + int64_t(start) * p.row_stride * 2;
    at.v = reinterpret_cast<uint8_t*>(p.layer_v[layer]) + int64_t(start) * p.row_stride * 2;
  } else if (tier > 0 && tier < kTiers) {
    const Store& st = p.store[tier];
    if (st.format == ASHKV_PAGE_NONE || slot < 0 || slot >= st.n_slots) return at;
    at.format = st.format;
    at.k = at.v = st.data + int64_t(slot) * st.slot_bytes;
  }
  return at;
}
__device__ __forceinline__ Place place_of(const PagedKV& p, int32_t id) { return place_of(p, entry_of(p, id)); }

}  // namespace
}  // namespace ashkv
