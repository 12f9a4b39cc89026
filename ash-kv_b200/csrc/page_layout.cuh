// Layout of a page's slot in each tier store (the ASHKV_PAGE_* formats), shared
// by the kernels that read or write pages in place (E elements, offsets in bytes):
//   INT8   [2T fp16 scales | pad to 16 | E int8 codes]           (the hooks' per-token layout)
//   FP8    [E e4m3fn bytes]
//   INT4   [E/64 bf16 scales | E/2 nibble bytes]                 (INT4Codec, group 64)
//   NBIT*  [u32 n_out, 3 x u32 0 | E/32 bf16 delta | E*bits/8 codes | cap x u32 outliers]
//          outlier entry = (element index in the page << 16) | bf16 bits, ascending
#pragma once

#include "common.cuh"

namespace ashkv {

constexpr int kTiers = 6;

// One tier's slots, as ashkv_tier_store_t describes them.
struct Store {
  uint8_t* data;
  int64_t slot_bytes;
  int32_t n_slots;
  int32_t format;
  int32_t* free_stack;
  int32_t* free_top;
};

__host__ __device__ __forceinline__ int64_t int8_codes_offset(int T) { return (4 * int64_t(T) + 15) / 16 * 16; }
__host__ __device__ __forceinline__ int64_t nbit_delta_off() { return 16; }
__host__ __device__ __forceinline__ int64_t nbit_codes_off(int64_t E) { return 16 + E / 16; }
__host__ __device__ __forceinline__ int64_t nbit_entries_off(int64_t E, int bits) {
  return nbit_codes_off(E) + E * bits / 8;
}

// The caller's six stores; false where store 0 is not the BF16 pool or a store is malformed.
inline bool copy_stores(const ashkv_tier_store_t* stores, Store (&out)[kTiers], bool need_data) {
  if (!stores) return false;
  for (int t = 0; t < kTiers; ++t) {
    const ashkv_tier_store_t& s = stores[t];
    out[t] = Store{static_cast<uint8_t*>(s.d_data), s.slot_bytes, s.n_slots, s.format, s.d_free_stack, s.d_free_top};
    if (t == 0) {
      if (s.format != ASHKV_PAGE_BF16) return false;
      continue;
    }
    if (s.format == ASHKV_PAGE_NONE) continue;
    if (s.format < ASHKV_PAGE_INT8 || s.format > ASHKV_PAGE_NBIT2) return false;
    if (s.n_slots < 0 || s.n_slots > 0xFFFFFF || !s.d_free_stack || !s.d_free_top) return false;
    if (need_data && (!s.d_data || !aligned(s.d_data, 16) || s.slot_bytes % 16)) return false;
  }
  return true;
}

// 16-byte asynchronous global -> shared copy: no register staging, so every
// chunk of a page can be in flight at once; cp.async.wait_all completes them.
__device__ __forceinline__ void cp_async16(uint32_t smem_addr, const void* gptr) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_addr), "l"(gptr) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

}  // namespace ashkv
