// Attention of one new token per sequence over paged KV whose pages may be in
// any tier (ashkv_decode_attention).
//
// With s[t] = scale * q . K[t] the result is sum_t 2^(s2[t] - M) V[t] / sum_t
// 2^(s2[t] - M), s2 = s * log2(e), for any M; one pass over the pages keeps a
// running M and the two sums.  The work is split over the length of the pages:
// for each key head the pages of all sequences form one row, cut into equal
// ranges, one worker warp each, so a batch of one long sequence and a ragged
// batch fill the GPU alike.  A range that reaches into several sequences leaves one
// partial result per sequence (normalised, with its log2-sum); the join kernel
// weighs the partials of each sequence by 2^(their log2-sum - the total).
//
// A step reads every page once and uses it for one group of query heads (8 of
// them: 8 operations a byte of bf16, 32 of INT4), so HBM is the bound to aim for,
// and products of 128 rows are not what is missing: the tensor pipe is 10 to 18 % busy with the 16 x 8 ones used here,
// whose operands come from codes in registers.  Measured calls, both kernels:
//   32 x 8192 tokens, 64 / 8 heads of 128:  bf16 184 us (5.8 TB/s, 89 % of a
//     plain copy's rate), INT8 with page mass 137 us (3.9 TB/s; the copies alone
//     run at 5.1, the rest is issue and latency)
//   131071 INT4 tokens, 32 / 8 heads: 75 us (1.9 TB/s; 58 % of the issue slots
//     are used, 48 % of the ALU's: two tokens' nibbles make one operand word)
//   24 ragged sequences over bf16, INT8, INT4 and 2-bit pages: 82 us (the four
//     formats' code does not fit the instruction cache together)
//   64 sequences, 2 heads of 64, FP8: 32 us, of which about 7 pass before the
//     first page arrives (lengths, ids, table, page: loads that wait for another)
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "common.cuh"
#include "nbit_group.cuh"
#include "page_layout.cuh"

namespace ashkv {
namespace {

constexpr int kWarpsA = 4;          // worker warps of a CTA; a fifth warp feeds them
constexpr int kThreadsA = (kWarpsA + 1) * 32;
constexpr int kWorkersPerSm = 12;   // resident worker warps per SM (8 where registers or shared memory leave two CTAs)
constexpr uint32_t kPolls = 1u << 24;  // bounded mbarrier waits
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kJoinThreads = 256;
// Entries of all lists of a call: what is added to a position (ranges, a batch looked up ahead) stays inside an int.
constexpr int64_t kMostEntries = 0x7FFFFFFFLL - 65536;

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
  int32_t* first_range;  // [n_seqs][heads_kv]: the ranges that hold a list's first and last entry
  int32_t* last_range;
  int32_t warp_smem;  // bytes of shared memory of a worker
  int32_t fp8_pages, int_pages;  // whether a store holds FP8, or INT8 or INT4 pages
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

// ---------------------------------------------------------------- tensor-core pieces
// D (16 x 8, fp32) = A (16 x 16, row) * B (16 x 8, col) + (first ? 0 : D).  Lane (g,
// t) = (lane / 4, lane % 4) holds A rows g and g + 8, k = 2t, 2t + 1, 2t + 8, 2t +
// 9 (a.x .. a.w: row g, row g + 8, then the same for the upper k), B column g at
// the same k (b0, b1), and D rows g, g + 8 at columns 2t, 2t + 1.
#define ASHKV_MMA(KIND, C, ...) \
  asm volatile("mma.sync.aligned." KIND " {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, " C ";" __VA_ARGS__)
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, bool first = false) {
  if (first) {
    if constexpr (BF16)
      ASHKV_MMA("m16n8k16.row.col.f32.bf16.bf16.f32", "{%10,%10,%10,%10}", : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
    else
      ASHKV_MMA("m16n8k16.row.col.f32.f16.f16.f32", "{%10,%10,%10,%10}", : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(0.0f));
  } else {
    if constexpr (BF16)
      ASHKV_MMA("m16n8k16.row.col.f32.bf16.bf16.f32", "{%0,%1,%2,%3}", : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
    else
      ASHKV_MMA("m16n8k16.row.col.f32.f16.f16.f32", "{%0,%1,%2,%3}", : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
}
// The same with int8 operands and k = 32: A and B registers hold k = 4t .. 4t + 3, the upper ones 16 more.
__device__ __forceinline__ void mma16832(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, bool first) {
  if (first)
    ASHKV_MMA("m16n8k32.row.col.s32.s8.s8.s32", "{%10,%10,%10,%10}", : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
              : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(0));
  else
    ASHKV_MMA("m16n8k32.row.col.s32.s8.s8.s32", "{%0,%1,%2,%3}", : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
              : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(uint32_t(127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t f32x2_to_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t f32x2_to_bf16x2_down(float lo, float hi) {  // toward zero
  uint32_t r;
  asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" :: "r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// 16 bytes global -> shared; zeros instead when `real` is false (nothing is read then).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" :: "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(dst), "l"(src) : "memory");
}
// Codes as exact fp16 pairs, by putting them into the low bits of 1024.0 (0x6400)
// and subtracting what that adds.
// Bytes (0, 1) or (2, 3) of an int8 word with its sign bits flipped (code + 128):
__device__ __forceinline__ uint32_t int8_pair(uint32_t flipped, uint32_t sel) {
  return add_f16x2(__byte_perm(flipped, 0x64646464u, sel), 0xE480E480u);  // - 1152
}
// Nibbles at bits 0-3 and 16-19, or at bits 4-7 and 20-23, less 8:
__device__ __forceinline__ uint32_t nibble_lo(uint32_t w) { return add_f16x2((w & 0x000F000Fu) | 0x64006400u, 0xE408E408u); }
__device__ __forceinline__ uint32_t nibble_hi(uint32_t w) {  // (1024 + 16 n) / 16 - 72
  return fma_f16x2((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, 0xD480D480u);
}
__device__ __forceinline__ uint32_t fp8_pair(uint32_t c16) {  // two e4m3 bytes -> fp16 pair, exact
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(c16)));
  return h;
}

// Where row r (token of a tile), 16-byte chunk c of a K or V tile of RB bytes a
// row sits in shared memory.  The rows a warp reads together (K: tokens g; V:
// tokens 2t, 2t + 1 and those + 8) fall into different banks.
template <int RB>
__device__ __forceinline__ uint32_t k_off(uint32_t r, uint32_t c) {
  if constexpr (RB >= 128) return r * RB + ((c ^ ((r & 1u) << 2)) << 4);
  else if constexpr (RB == 64) return r * RB + ((c ^ (r & 2u)) << 4);
  else return r * RB + (c << 4);
}
template <int RB>
__device__ __forceinline__ uint32_t v_off(uint32_t r, uint32_t c) {
  if constexpr (RB >= 128) return r * RB + ((c ^ (r & 6u)) << 4);
  const uint32_t q = (r >> 1) | ((r & 1u) << 3);
  if constexpr (RB == 64) return q * RB + ((c ^ (q & 2u)) << 4);
  return q * RB + (c << 4);
}

// ---------------------------------------------------------------- the pages of a worker
constexpr int kRing = 3;  // units in shared memory per worker: one in use, two on their way

// A unit is 16 tokens of a page for one key head: the K or the V rows of a BF16
// page (16 x D bf16), or the codes of both of a compressed page (K first), with
// the scales of those rows beside them: INT8: fp16, K then V, the V rows from the
// last 4-byte boundary on; INT4: a word per row, K then V (D = 64: the row's scale
// for this head is the word's upper half for an odd head).  The K or the V rows of
// a dithered page come as they are (see RawNbit) and are decoded to a BF16 unit
// in place.  A page to leave out takes a unit that nothing is copied to.  A
// header says what the unit is.
template <int D>
struct UnitLayout {  // the ring's data, scales and headers, one after the other
  static constexpr uint32_t kData = 16 * D * 2, kScales = kRing * kData, kHeaders = kScales + kRing * 128,
                            kBytes = kHeaders + kRing * 16;
};
struct Header {
  const uint8_t* slot;  // dithered pages
  uint32_t meta;        // format | rows in use << 8 | flags | first token / 16 << 20
  int32_t pos;          // page position in the sequence
  static constexpr uint32_t kIsV = 1u << 16, kPageEnd = 1u << 17, kSegmentEnd = 1u << 18;
  __device__ __forceinline__ uint32_t format() const { return meta & 0xFFu; }
  __device__ __forceinline__ int rows() const { return int(meta >> 8) & 0xFF; }
};

// A unit of a dithered page as copied: 16 rows of codes, their deltas (D / 32 of a
// row), the slot's first 16 bytes (the number of outliers) and its first outliers.
template <int D, int BITS>
struct RawNbit {
  static constexpr uint32_t kRow = D * BITS / 8, kDeltas = 16 * kRow, kDeltaRow = D / 16, kCount = kDeltas + 16 * kDeltaRow,
                            kEntries = kCount + 16, kMaxEntries = 128;
};
// Decodes such a unit in place into the K or V rows (bf16) of a BF16 unit; slot: the page's.  A group
// of 32 channels at a time and lane, all read before any is written; the outliers overwrite theirs.
// (Out of line: a call costs little beside the decode, and the loop of the other formats stays short.)
template <int D, int BITS>
__device__ __noinline__ void decode_nbit(uint32_t unit, const uint8_t* slot, int T, int row_len, int cap, int hk, bool v,
                                         int t0, int rows) {
  using Raw = RawNbit<D, BITS>;
  constexpr int GPR = D / 32, RB = D * 2, N = GPR / 2;
  constexpr float half = float((1 << BITS) - 1) * 0.5f;
  const int lane = threadIdx.x & 31;
  GroupCodes<BITS> gc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t n = lane + 32 * j, at = unit + n * (4 * BITS);  // group n % GPR of row n / GPR
    if constexpr (BITS == 4) {
      const uint4 x = lds128(at);
      gc[j].w[0] = x.x; gc[j].w[1] = x.y; gc[j].w[2] = x.z; gc[j].w[3] = x.w;
    } else {
      const uint2 x = lds64(at);
      gc[j].w[0] = x.x; gc[j].w[1] = x.y;
    }
    uint16_t d;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(d) : "r"(unit + Raw::kDeltas + n * 2));
    gc[j].delta = bf16_to_f32(d);
  }
  const uint32_t n_out = min(lds32(unit + Raw::kCount), uint32_t(cap));
  uint32_t entry[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) entry[j] = lds32(unit + Raw::kEntries + (lane + 32 * j) * 4);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const uint32_t n = lane + 32 * j, r = n / GPR, k = n % GPR;
    uint32_t o[16];
    group_bf16<BITS>(gc[j], half, o);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 x = int(r) < rows ? make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]) : make_uint4(0, 0, 0, 0);
      sts128(unit + (v ? v_off<RB>(r, 4 * k + c) : k_off<RB>(r, 4 * k + c)), x);
    }
  }
  __syncwarp();
  const uint32_t row0 = uint32_t((v ? T : 0) + t0), shift = 31 - __clz(row_len);  // rows are powers of two
  const auto put = [&](uint32_t e) {
    const uint32_t r = (e >> 16 >> shift) - row0, c = ((e >> 16) & uint32_t(row_len - 1)) - uint32_t(hk * D);
    if (r < uint32_t(rows) && c < uint32_t(D))
      asm volatile("st.shared.u16 [%0], %1;" :: "r"(unit + (v ? v_off<RB>(r, c >> 3) : k_off<RB>(r, c >> 3)) + (c & 7u) * 2u),
                   "h"(static_cast<uint16_t>(e)) : "memory");
  };
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (lane + 32 * j < n_out) put(entry[j]);
  if (n_out > Raw::kMaxEntries) {
    const uint32_t* ent = reinterpret_cast<const uint32_t*>(slot + nbit_entries_off(2 * int64_t(T) * row_len, BITS));
    for (uint32_t j = Raw::kMaxEntries + lane; j < n_out; j += 32) put(ent[j]);
  }
  __syncwarp();
}

// Where a worker's pages begin: sequence b, of whose list `before` entries of the row lie ahead.
struct Share {
  int b, before, pos, end;  // row positions [pos, end)
};

// The producer warp of a CTA sends the units of its four workers, eight lanes for
// each, so that the instructions that find pages and copy rows serve four
// workers at once (they mostly hold four heads of the same pages).  List entries
// are looked up eight at a time, a lane each, in four steps two pages apart
// (position, page id, page-table columns, layer address), so that no step waits
// for the loads of the one before it.
template <int D>
struct Producer {
  using Layout = UnitLayout<D>;
  static constexpr int kLook = 8;
  const AttnParams& p;
  const int hk, sub;      // this lane's worker's key head; lane within the worker's eight
  int b, i, i0, i1;       // its sequence, next list entry, the segment's entries
  int64_t tokens;
  int row_pos, row_end, before;
  bool active;
  int t0;                 // first token of the next unit in its page
  bool second;            // BF16: the V rows are next
  uint32_t slot, phase;
  const uint32_t ring, bars;  // shared addresses: the units; full[kRing], empty[kRing]
  // entry batch0 + sub of the segment, and the one being looked up for the next batch
  const uint8_t *k, *v;
  uint32_t meta;          // format | tokens in use << 8; no tokens: a page to leave out
  int pos, batch0;        // position in the sequence
  int n_pos, n_id, n_tier, n_layer, n_start, n_slot;
  uint64_t n_k, n_v;

  __device__ __forceinline__ Producer(const AttnParams& p_, int hk_, const Share& s, uint32_t ring_, uint32_t bars_)
      : p(p_), hk(hk_), sub(int(threadIdx.x & 7u)), slot(0), phase(0), ring(ring_), bars(bars_) {
    b = s.b; before = s.before; row_pos = s.pos; row_end = s.end;
    active = row_pos < row_end;
  }

  // A segment is the part of the worker's pages that lies in one sequence.
  __device__ void open_segment() {
    int n = 0;
    for (; active; ++b) {
      n = list_len(p, b, hk);
      if (before + n > row_pos) break;
      before += n;
    }
    if (active) {
      i0 = i = row_pos - before;
      i1 = min(n, row_end - before);
      tokens = seq_tokens(p, b);
    } else {
      i0 = i = i1 = 0;
      tokens = 0;
    }
    t0 = 0;
    second = false;
    batch0 = i0 - kLook;
    for (int step = 0; step < 4; ++step) look_up(step);
    take_batch();
  }
  // Steps of the look-up of entry batch0 + kLook + sub.
  __device__ __forceinline__ void look_up(int step) {
    const int e = batch0 + kLook + sub;
    const bool mine = e < i1;
    if (step == 0) {
      n_pos = mine && p.selected ? p.selected[(int64_t(b) * p.heads_kv + hk) * p.max_selected + e] : e;
    } else if (step == 1) {
      const bool ok = mine && n_pos >= 0 && int64_t(n_pos) * p.T < tokens;
      n_id = ok ? p.page_ids[int64_t(b) * p.page_ids_stride + n_pos] : -1;
      if (!ok) n_pos = 0;
    } else if (step == 2) {
      const bool ok = n_id >= 0 && n_id < p.n_pages;
      n_tier = ok ? p.tier[n_id] : -1;
      n_layer = ok ? p.layer_id[n_id] : 0;
      n_start = ok ? p.token_start[n_id] : 0;
      n_slot = ok ? p.page_slot[n_id] : 0;
    } else {
      const bool ok = n_tier == 0 && n_layer >= 0 && n_layer < p.n_layers;
      n_k = ok ? p.layer_k[n_layer] : 0;
      n_v = ok ? p.layer_v[n_layer] : 0;
    }
  }
  // Makes the entry looked up this lane's entry of the current batch (the last step).
  __device__ __forceinline__ void take_batch() {
    batch0 += kLook;
    k = v = nullptr;
    meta = 0;
    pos = n_pos;
    if (batch0 + sub >= i1) return;
    const int n_where = n_tier == 0 ? n_start : n_slot;
    bool ok = n_tier >= 0 && n_tier < kTiers && n_where >= 0;
    if (ok && n_tier == 0) {
      ok = n_layer >= 0 && n_layer < p.n_layers && int64_t(n_where) + p.T <= p.pool_tokens;
      if (ok) {
        const int64_t off = (int64_t(n_where) * p.row_stride + hk * D) * 2;
        k = reinterpret_cast<const uint8_t*>(n_k) + off;
        v = reinterpret_cast<const uint8_t*>(n_v) + off;
        meta = ASHKV_PAGE_BF16;
      }
    } else if (ok) {
      const Store& st = p.store[n_tier];
      ok = st.format != ASHKV_PAGE_NONE && n_where < st.n_slots;
      if (ok) {
        v = k = st.data + int64_t(n_where) * st.slot_bytes;
        meta = uint32_t(st.format);
        if (meta == ASHKV_PAGE_INT8) k += int8_codes_offset(p.T) + hk * D;
        if (meta == ASHKV_PAGE_FP8) k += hk * D;
        if (meta == ASHKV_PAGE_INT4) {
          k += p.T * p.row_len / 16 + hk * (D / 2);  // past E / 32 bytes of scales
          v += hk * D / 32 & ~3;
        }
      }
    }
    if (ok) {
      meta |= uint32_t(min(int64_t(p.T), tokens - int64_t(pos) * p.T)) << 8;
    } else {
      flag(p.status, ASHKV_FLAG_INDEX_RANGE);
      if (p.mass)  // a page that is left out draws nothing
        for (int g = 0; g < p.group; ++g)
          p.page_lse2[(int64_t(b) * p.max_pages + pos) * p.heads_q + hk * p.group + g] = -INFINITY;
    }
  }

  // 16 rows of RB bytes, `step` bytes apart from src on, into a tile by the worker's eight lanes;
  // rows behind `rows` become zeros.
  template <int RB, bool V>
  __device__ __forceinline__ void copy_rows(const uint8_t* src, uint32_t step, int rows, uint32_t tile) const {
    constexpr uint32_t CPR = RB / 16;                     // chunks of a row
    constexpr uint32_t LPR = CPR < 8 ? CPR : 8, RPI = 8 / LPR;  // lanes of a row, rows of one instruction
    const uint32_t r0 = uint32_t(sub) / LPR, c0 = uint32_t(sub) % LPR;
    src += r0 * step + c0 * 16u;
    if (rows >= 16) {
#pragma unroll
      for (uint32_t j = 0; j < 16 / RPI; ++j) {
#pragma unroll
        for (uint32_t c = 0; c < CPR; c += LPR)
          cp_async16(tile + (V ? v_off<RB>(r0 + RPI * j, c0 + c) : k_off<RB>(r0 + RPI * j, c0 + c)), src + c * 16);
        src += RPI * step;
      }
      return;
    }
#pragma unroll 1
    for (uint32_t j = 0; j < 16 / RPI; ++j) {
      const uint32_t r = r0 + RPI * j;
      const bool real = r < uint32_t(rows);
#pragma unroll
      for (uint32_t c = 0; c < CPR; c += LPR)
        cp_async16_or_zero(tile + (V ? v_off<RB>(r, c0 + c) : k_off<RB>(r, c0 + c)),
                           real ? src + uint64_t(RPI * step) * j + c * 16 : k, real);
    }
  }

  // The rows, deltas and first outliers of a dithered page (slot pk) for a unit.
  template <int BITS>
  __device__ __forceinline__ void copy_nbit(const uint8_t* pk, int rows, uint32_t unit) const {
    using Raw = RawNbit<D, BITS>;
    const int64_t E = 2 * int64_t(p.T) * p.row_len;
    const uint32_t row = uint32_t(p.row_len), row0 = uint32_t((second ? p.T : 0) + t0), last = uint32_t(min(rows, 16)) - 1u;
    const uint8_t *codes = pk + nbit_codes_off(E), *deltas = pk + nbit_delta_off();
    constexpr uint32_t CPR = Raw::kRow / 16;
#pragma unroll
    for (uint32_t j = 0; j < 2 * CPR; ++j) {  // (rows not in use: the last one again)
      const uint32_t n = uint32_t(sub) + 8u * j, r = n / CPR, c = n % CPR;
      cp_async16(unit + n * 16u, codes + ((row0 + min(r, last)) * row + hk * D) * BITS / 8u + c * 16u);
    }
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t r = uint32_t(sub) + 8u * j;
      const uint8_t* src = deltas + ((row0 + min(r, last)) * row + hk * D) / 16u;
      if constexpr (D == 128) cp_async8(unit + Raw::kDeltas + r * 8u, src);
      else cp_async4(unit + Raw::kDeltas + r * 4u, src);
    }
    if (sub == 0) cp_async16(unit + Raw::kCount, pk);
    const uint8_t* entries = pk + nbit_entries_off(E, BITS);
    const uint32_t bytes = uint32_t(min(p.outlier_cap, int(Raw::kMaxEntries))) * 4u;  // (slots end on 256 bytes)
#pragma unroll
    for (uint32_t o = 0; o < Raw::kMaxEntries * 4; o += 128)
      if (o + uint32_t(sub) * 16u < bytes) cp_async16(unit + Raw::kEntries + o + uint32_t(sub) * 16u, entries + o + sub * 16);
  }

  __device__ void run() {
    open_segment();
    const uint32_t group = threadIdx.x & 24u;  // first lane of the worker's eight
    const uint8_t *pk = nullptr, *pv = nullptr;  // the current page
    uint32_t pm = 0;
    int pp = 0;
    for (uint32_t sent = 0; __any_sync(0xFFFFFFFFu, active); ++sent) {
      const bool page_start = active && !second && t0 == 0;
      // two pages apart, a step for the next eight entries
      if (page_start && !((i - batch0) & 1)) {
        if (i - batch0 == kLook) take_batch();
        look_up((i - batch0) >> 1);
      }
      if (__any_sync(0xFFFFFFFFu, page_start)) {
        const int src = int(group) + ((i - batch0) & (kLook - 1));  // (inside a page: its own entry again)
        pk = reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(k), src));
        pv = reinterpret_cast<const uint8_t*>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(v), src));
        pm = __shfl_sync(0xFFFFFFFFu, meta, src);
        pp = __shfl_sync(0xFFFFFFFFu, pos, src);
      }
      bool ok = true;
      if (active && sent >= kRing) ok = wait_bar(bars + (kRing + slot) * 8, phase ^ 1u);
      if (!__all_sync(0xFFFFFFFFu, ok)) {
        flag(p.status, ASHKV_FLAG_TIMEOUT);
        for (uint32_t n = sent < kRing ? 0 : sent - kRing; n < sent && active; ++n)  // what is still on its way
          wait_bar(bars + n % kRing * 8, n / kRing & 1u);
        break;
      }
      if (active) {
        const uint32_t format = pm & 0xFFu, T = uint32_t(p.T), row = uint32_t(p.row_len);
        const uint32_t unit = ring + slot * Layout::kData, scales = ring + Layout::kScales + slot * 128;
        const uint32_t full = bars + slot * 8;
        const int left = int(pm >> 8) - t0;
        uint32_t h = format | uint32_t(max(0, min(left, 16))) << 8 | uint32_t(t0) << 16;
        bool done = true;  // with these tokens
        if (left <= 0) {
        } else if (format == ASHKV_PAGE_BF16) {
          const uint32_t step = uint32_t(p.row_stride) * 2u;
          if (second) copy_rows<D * 2, true>(pv + uint32_t(t0) * step, step, left, unit);
          else copy_rows<D * 2, false>(pk + uint32_t(t0) * step, step, left, unit);
          if (second) h |= Header::kIsV;
          done = second;
          second = !second;
        } else if (format < ASHKV_PAGE_NBIT4) {
          const bool int4 = format == ASHKV_PAGE_INT4;
          if (int4) {
            const uint8_t* codes = pk + uint32_t(t0) * (row / 2);
            copy_rows<D / 2, false>(codes, row / 2, left, unit);
            copy_rows<D / 2, true>(codes + T * (row / 2), row / 2, left, unit + 8 * D);
          } else {
            const uint8_t* codes = pk + uint32_t(t0) * row;
            copy_rows<D, false>(codes, row, left, unit);
            copy_rows<D, true>(codes + T * row, row, left, unit + 16 * D);
          }
          if (int4) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
              const uint32_t r = sub + 8u * (j & 1u);
              cp_async4(scales + (16u * (j >> 1) + r) * 4u, pv + (min(uint32_t(t0) + r, T - 1u) + (j >> 1) * T) * (row / 32u));
            }
          } else if (format == ASHKV_PAGE_INT8) {
            // 8 words of K scales, 9 of V scales (all inside the slot: codes follow them)
            const uint8_t* vs = pv + ((T + uint32_t(t0)) * 2u & ~3u);
            if (T % 8u == 0) {  // 16-byte chunks: two of either
              if (sub < 4) cp_async16(scales + sub * 16u, (sub < 2 ? pv + t0 * 2 : vs - 32) + sub * 16);
            } else {
              cp_async4(scales + sub * 4u, pv + t0 * 2 + sub * 4);
              cp_async4(scales + 32u + sub * 4u, vs + sub * 4);
              if (sub == 0) cp_async4(scales + 64u, vs + 32);
            }
          }
        }
        else {
          if (format == ASHKV_PAGE_NBIT4) copy_nbit<4>(pk, left, unit);
          else copy_nbit<2>(pk, left, unit);
          if (second) h |= Header::kIsV;
          done = second;
          second = !second;
        }
        if (done) {
          t0 += 16;
          if (left <= 16) {
            h |= Header::kPageEnd;
            t0 = 0;
            if (++i == i1) h |= Header::kSegmentEnd;
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(full) : "memory");
        if (sub == 0) {
          const uint64_t a = reinterpret_cast<uint64_t>(pk);
          sts128(ring + Layout::kHeaders + slot * 16, make_uint4(uint32_t(a), uint32_t(a >> 32), h, uint32_t(pp)));
          asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(full) : "memory");
        }
        if (++slot == kRing) {
          slot = 0;
          phase ^= 1u;
        }
      }
      const bool ended = active && i == i1;
      if (__any_sync(0xFFFFFFFFu, ended)) {
        if (ended) {
          row_pos = before + i1;
          active = row_pos < row_end;
          open_segment();
        }
        __syncwarp();
      }
    }
    cp_async_wait_all();
  }
  static __device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity) {
    for (uint32_t n = 0; n < kPolls; ++n) {
      uint32_t done;
      asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                   : "=r"(done) : "r"(bar), "r"(parity) : "memory");
      if (done) return true;
    }
    return false;
  }
};

// ---------------------------------------------------------------- the worker
// A warp per (range of pages, key head, up to 8 * NT of its query heads).
//   S (queries x tokens) = Q K^T, then O^T (channels x queries) += V^T P^T.  K rows
// enter the first product as its B operand and the weights leave it laid out as
// the B operand of the second, so nothing is exchanged between lanes; the 16
// rows of A are the channels in the second product.  In the first they hold up
// to 16 queries (NT = 2); for 8 (NT = 1) the upper 8 rows do not idle but hold
// the same queries' next 16 channels (or their next digit, see below), and each
// half of D is read from the product whose B operand matches it.
//   Lane (g, t) owns the scores of query g (and g + 8) and tokens 2t, 2t + 1, 2t +
// 8, 2t + 9 of a tile.  m is the reference of the weights 2^(s - m).  It follows
// the running maximum only when a score lies more than 2^8 above it, which is
// rare after the first tiles, so most tiles reduce nothing across the lanes.
// acc holds sum_t 2^(s - m) * c * v.  The scale of a compressed V row rides on its
// weight and its codes enter the product as whole numbers; the power of two c
// keeps weight * scale inside the fp16 range: c * (largest scale so far) lies in
// [2^6, 2^7], a weight below 2^8, so the operand stays below 2^15 and is off by at
// most 2^-25 / c where fp16 runs out of digits, 2^-31 of a largest value.
template <int D, int NT>
struct Worker {
  static constexpr int MT = D / 16;  // channel tiles of 16
  static constexpr float kUnit8 = 1.0f / 127.0f, kUnit4 = 1.0f / 7.0f;  // a code's value is code * scale * unit
  const AttnParams& p;
  float acc[NT][MT][4];              // [queries 8 n ..][channel tile]: rows g, g + 8, columns (queries) 2t, 2t + 1
  float m[NT], thr[NT], l[NT], ps[NT];  // of query 8 n + g; ps: the page's own sum
  float c;
  float qs_h[NT], qs_i[NT];  // factors from a dot product with the fp16 / whole-number queries to a log2 score
  // The queries in shared memory as A operands: bf16; fp16, scaled by a power of two (FP8 stores
  // only); three int8 digits of whole numbers (INT8 and INT4 stores only).
  uint32_t qb, qh, qi;
  int lane, g, t;
  bool fresh;               // no scale was seen yet
  bool odd_head, odd_pages;

  __device__ __forceinline__ Worker(const AttnParams& p_, uint32_t q_smem, int hk)
      : p(p_), qb(q_smem), qh(q_smem + NT * 8 * D * 2), qi(qh + (p_.fp8_pages ? NT * 8 * D * 2 : 0)),
        lane(threadIdx.x & 31), g(lane >> 2), t(lane & 3), odd_head(hk & 1), odd_pages(p_.T & 1) {}

  // 16-bit queries.  Channels 8 k .. 8 k + 7 (words w = 0 .. 3 of two) serve two products of 16
  // channels, words 0, 1 the first.  NT = 1: one operand (0, 2, 1, 3), the second product's words in
  // rows 8-15; NT = 2: two operands (row g, row g + 8).  Neighbouring rows go to other banks.
  static __device__ __forceinline__ uint32_t q_chunk(uint32_t row, uint32_t chunk, bool wide) {
    return row * (NT * D * 2) + ((chunk ^ (NT == 1 && !wide ? (row & 1u) << 2 : row & 1u)) << 4);
  }
  static __device__ __forceinline__ uint32_t q_word(uint32_t n, uint32_t k, uint32_t w, bool wide) {
    if constexpr (NT == 1) return q_chunk(n, k, wide) + (((w & 1u) << 1) | (w >> 1)) * 4u;
    return q_chunk(n & 7u, 2u * k + (w >> 1), true) + ((w & 1u) * 2u + (n >> 3)) * 4u;
  }
  // Digits.  Channels 16 k .. 16 k + 15 (words of four) serve two products of 32 channels.  NT = 1: the
  // two higher digits as the two halves of the rows, two operands; the lowest like 16-bit words above.
  // NT = 2: two operands for each digit.
  static __device__ __forceinline__ uint32_t digit_chunk(uint32_t row, uint32_t chunk) { return row * (D * 2) + ((chunk ^ (row & 1u)) << 4); }
  static __device__ __forceinline__ uint32_t low_chunk(uint32_t row, uint32_t chunk) {
    return 8 * D * 2 + row * D + (((chunk ^ ((row & 1u) << 2)) & (D / 16 - 1)) << 4);
  }
  static __device__ __forceinline__ uint32_t digit_word(uint32_t digit, uint32_t n, uint32_t k, uint32_t w) {  // digit 0: the highest
    if constexpr (NT == 1) {
      if (digit == 2) return low_chunk(n, k) + (((w & 1u) << 1) | (w >> 1)) * 4u;
      return digit_chunk(n, 2u * k + (w >> 1)) + ((w & 1u) * 2u + digit) * 4u;
    }
    return digit * (16 * D) + digit_chunk(n & 7u, 2u * k + (w >> 1)) + ((w & 1u) * 2u + (n >> 3)) * 4u;
  }
  static __device__ __forceinline__ void sts32(uint32_t a, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" :: "r"(a), "r"(v) : "memory"); }

  __device__ void start(int b, int hq0, int nq) {
    constexpr int N = D / 32;  // channels of a lane here
#pragma unroll
    for (int half = 0; half < NT; ++half)
#pragma unroll 2
    for (int n = 8 * half; n < 8 * half + 8; ++n) {
      uint16_t x[N];
      float amax = 0.0f;
      bool whole = true;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k] = n < nq ? p.q[b * p.q_seq_stride + int64_t(hq0 + n) * p.q_head_stride + lane * N + k] : uint16_t(0);
        const float a = fabsf(bf16_to_f32(x[k]));
        if (a < INFINITY) amax = fmaxf(amax, a);
        else whole = false;
      }
      amax = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax)));
      whole = __all_sync(0xFFFFFFFFu, whole);
      const uint32_t k8 = uint32_t(lane * N) >> 3, w8 = (uint32_t(lane * N) & 7u) >> 1;
#pragma unroll
      for (int k = 0; k < N; k += 2) sts32(qb + q_word(n, k8, w8 + k / 2, false), uint32_t(x[k]) | (uint32_t(x[k + 1]) << 16));
      // the exponent e of the largest value; powers of two around it in two factors, as 2^+-(e + 21) may
      // be no fp32 numbers.  The first takes the values to 2^(e / 2): exact, or nothing is left of values below
      // 2^-126 of the largest.
      const int e = max(int(__float_as_uint(amax) >> 23) - 127, -126), e1 = e >> 1, e2 = e - e1;
      const float up = pow2(e1), down = pow2(-e1);
      const bool mine = (n & 7) == g;
      if (p.fp8_pages) {
        // the largest value to [2^14, 2^15): fp16 then keeps all 8 bits of every value down to
        // 2^-31 of it, exactly
        if (mine) qs_h[half] = p.scale2 * up * pow2(e2 - 14);
        const float down2 = pow2(14 - e2);
#pragma unroll
        for (int k = 0; k < N; k += 2)
          sts32(qh + q_word(n, k8, w8 + k / 2, true),
                f32x2_to_f16x2(bf16_to_f32(x[k]) * down * down2, bf16_to_f32(x[k + 1]) * down * down2));
      }
      if (p.int_pages) {
        // whole numbers below 2^22 as digits of base 256 in [-128, 127] (the highest at most 64): exact
        // down to 2^-14 of the largest value, off by at most 2^-22 of it below
        if (mine) qs_i[half] = whole ? p.scale2 * up * pow2(e2 - 21) : NAN;
        const float down2 = pow2(21 - e2);
        uint32_t d[3] = {0, 0, 0};
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int v = __float2int_rn(bf16_to_f32(x[k]) * down * down2);
          const int v1 = (v + 128) >> 8, v2 = (v1 + 128) >> 8;
          d[0] |= uint32_t(v2 & 255) << (8 * k);
          d[1] |= uint32_t(v1 & 255) << (8 * k);
          d[2] |= uint32_t(v & 255) << (8 * k);
        }
        const uint32_t k16 = uint32_t(lane * N) >> 4, w16 = (uint32_t(lane * N) & 15u) >> 2;
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          const uint32_t at = qi + digit_word(k, n, k16, w16);
          if constexpr (N == 4) sts32(at, d[k]);
          else asm volatile("st.shared.u16 [%0], %1;" :: "r"(at + (lane & 1) * 2), "h"(uint16_t(d[k])) : "memory");
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = 0.0f; thr[n] = -INFINITY; l[n] = 0.0f; ps[n] = 0.0f;
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[n][k][x] = 0.0f;
    }
    c = 0x1p-8f;  // weights reach 2^8: a sum of n bf16 values stays below n times the largest
    fresh = true;
    __syncwarp();
  }

  __device__ __forceinline__ void scale_acc(int n, float f0, float f1) {
#pragma unroll
    for (int k = 0; k < MT; ++k) {
      acc[n][k][0] *= f0; acc[n][k][1] *= f1; acc[n][k][2] *= f0; acc[n][k][3] *= f1;
    }
  }
  // Query 8 n + 2t + j's value of x, which is spread over the owners (8 n + g) of the queries.
  __device__ __forceinline__ float of_column(float x, int j) const { return __shfl_sync(0xFFFFFFFFu, x, 8 * t + 4 * j); }
  static __device__ __forceinline__ float max_over_tokens(float x) {
    x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 1));
    return fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 2));
  }
  static __device__ __forceinline__ float sum_over_tokens(float x) {
    x += __shfl_xor_sync(0xFFFFFFFFu, x, 1);
    return x + __shfl_xor_sync(0xFFFFFFFFu, x, 2);
  }

  // log2 scores of tokens 2t, 2t + 1, 2t + 8, 2t + 9 -> weights 2^(s - m), added up.
  __device__ __forceinline__ void weights(float (&s)[NT][4], int rows) {
    if (rows < 16) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (2 * t + (x & 1) + 8 * (x >> 1) >= rows) s[n][x] = -INFINITY;
    }
    bool over = false;
    float top[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      top[n] = fmaxf(fmaxf(s[n][0], s[n][1]), fmaxf(s[n][2], s[n][3]));
      over |= top[n] > thr[n];
    }
    if (__any_sync(0xFFFFFFFFu, over)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float x = max_over_tokens(top[n]);
        float f = 1.0f;
        if (x > thr[n]) {
          if (thr[n] != -INFINITY) f = ex2(m[n] - x);
          m[n] = x;
          thr[n] = x + 8.0f;
          l[n] *= f;
          ps[n] *= f;
        }
        scale_acc(n, of_column(f, 0), of_column(f, 1));
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] = ex2(s[n][x] - m[n]);
      const float sum = (s[n][0] + s[n][1]) + (s[n][2] + s[n][3]);
      l[n] += sum;
      ps[n] += sum;
    }
  }

  // Makes room for V rows of scale x (this lane's, 0 where it holds none).
  __device__ __forceinline__ void fit_scale(float x) {
    if (!__any_sync(0xFFFFFFFFu, fresh || x * c > 128.0f)) return;
    const float top = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, x > 0.0f ? __float_as_uint(x) : 0u));
    if (top > 0.0f && top < INFINITY) {  // c * top to [2^6, 2^7)
      // (c stops at 2^37, which the smallest scales that the codecs write need, 1e-8 and the least fp16 above 0, so
      // that n weights of up to 2^8 have room beside it for BF16 values up to 2^83 / n; a scale below that is off by
      // up to 2^-62 a token)
      const int e = max(int(__float_as_uint(top) >> 23), 96);
      const float next = __uint_as_float(uint32_t(254 + 6 - e) << 23);
      const float f = next / c;  // a power of two
#pragma unroll
      for (int n = 0; n < NT; ++n) scale_acc(n, f, f);
      c = next;
      fresh = false;
    }
  }
  // Weights times the scales w of the rows of this lane's tokens and a unit (c times what the scales
  // leave out), as the fp16 operand of the product with V.
  static __device__ __forceinline__ void fp16_weights(const float (&s)[NT][4], const float (&w)[4], float unit,
                                                      uint32_t (&b)[NT][2]) {
    float wc[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) wc[x] = w[x] * unit;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      b[n][0] = f32x2_to_f16x2(s[n][0] * wc[0], s[n][1] * wc[1]);
      b[n][1] = f32x2_to_f16x2(s[n][2] * wc[2], s[n][3] * wc[3]);
    }
  }

  // Dot products with the 16-bit queries at q (8-channel chunk k) of 16 channels each, keys (b0, b1)
  // and (b2, b3) of one token half: d takes the first or, with NT = 2, both; e the second with NT = 1.
  template <bool BF16>
  static __device__ __forceinline__ void dot16(float (&d)[4], float (&e)[4], const uint4 (&q)[NT], uint32_t b0, uint32_t b1,
                                               uint32_t b2, uint32_t b3, bool first) {
    mma16816<BF16>(d, q[0], b0, b1, first);
    if constexpr (NT == 1) mma16816<BF16>(e, q[0], b2, b3, first);
    else mma16816<BF16>(d, q[1], b2, b3);
  }
  static __device__ __forceinline__ void gather16(float (&s)[NT][4], const float (&d)[2][4], const float (&e)[2][4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (NT == 1) s[0][x] = d[x >> 1][x & 1] + e[x >> 1][2 + (x & 1)];
      else { s[0][x] = d[x >> 1][x & 1]; s[1][x] = d[x >> 1][2 + (x & 1)]; }
    }
  }
  __device__ __forceinline__ void load_q16(uint4 (&q)[NT], uint32_t base, uint32_t k, bool wide) const {
    if constexpr (NT == 1) q[0] = lds128(base + q_chunk(g, k, wide));
    else { q[0] = lds128(base + q_chunk(g, 2 * k, true)); q[1] = lds128(base + q_chunk(g, 2 * k + 1, true)); }
  }

  // Weights of a tile of BF16 keys.
  __device__ __forceinline__ void bf16_scores(uint32_t tile, int rows, float (&s)[NT][4]) {
    float d[2][4], e[2][4];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      uint4 q[NT];
      load_q16(q, qb, 4 * i + t, false);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 k = lds128(tile + k_off<D * 2>(g + 8 * h, 4 * i + t));
        dot16<true>(d[h], e[h], q, k.x, k.y, k.z, k.w, i == 0);
      }
    }
    gather16(s, d, e);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][x] *= p.scale2;
    weights(s, rows);
  }
  // Adds a tile of BF16 values: the weights in two bf16 parts (8 + 8 bits), as a single one would
  // cost as much accuracy as the rounding of the result.  Both parts of a weight are above 0 (the lower one
  // at least 2^-17 of it), so that an infinite value stays what it is.
  __device__ __forceinline__ void bf16_values(uint32_t tile, const float (&s)[NT][4]) {
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x0 = s[n][2 * h] * c, x1 = s[n][2 * h + 1] * c;
        hi[n][h] = f32x2_to_bf16x2_down(x0, x1);
        lo[n][h] = f32x2_to_bf16x2(fmaxf(x0 - bf16lo(hi[n][h]), x0 * 0x1p-17f), fmaxf(x1 - bf16hi(hi[n][h]), x1 * 0x1p-17f));
      }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      uint32_t v[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 x = lds128(tile + v_off<D * 2>(2 * t + (k & 1) + 8 * (k >> 1), g + 8 * i));
        v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 a = make_uint4(__byte_perm(v[0][w], v[1][w], 0x5410), __byte_perm(v[0][w], v[1][w], 0x7632),
                                   __byte_perm(v[2][w], v[3][w], 0x5410), __byte_perm(v[2][w], v[3][w], 0x7632));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<true>(acc[n][4 * i + w], a, hi[n][0], hi[n][1]);
          mma16816<true>(acc[n][4 * i + w], a, lo[n][0], lo[n][1]);
        }
      }
    }
  }

  // Dot products of int8 keys (64 channels i, this thread's 16 of tokens g and g + 8 in k[0], k[1])
  // with the three digits of the queries: whole numbers below 2^21 each, exact.
  struct Dots {
    int d[3][2][4];  // NT = 1: the higher two digits, the lowest of the first 32 channels, of the second; NT = 2: a digit each
  };
  __device__ __forceinline__ void add_digits(Dots& a, const uint4 (&k)[2], int i, bool first) const {
    if constexpr (NT == 1) {
      const uint4 q0 = lds128(qi + digit_chunk(g, 2 * (4 * i + t))), q1 = lds128(qi + digit_chunk(g, 2 * (4 * i + t) + 1));
      const uint4 ql = lds128(qi + low_chunk(g, 4 * i + t));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mma16832(a.d[0][h], q0, k[h].x, k[h].y, first);
        mma16832(a.d[0][h], q1, k[h].z, k[h].w, false);
        mma16832(a.d[1][h], ql, k[h].x, k[h].y, first);
        mma16832(a.d[2][h], ql, k[h].z, k[h].w, first);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint4 q0 = lds128(qi + j * (16 * D) + digit_chunk(g, 2 * (4 * i + t)));
        const uint4 q1 = lds128(qi + j * (16 * D) + digit_chunk(g, 2 * (4 * i + t) + 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mma16832(a.d[j][h], q0, k[h].x, k[h].y, first);
          mma16832(a.d[j][h], q1, k[h].z, k[h].w, false);
        }
      }
    }
  }
  static __device__ __forceinline__ float dot_value(const Dots& a, int n, int x) {
    const int h = x >> 1, j = x & 1;
    if constexpr (NT == 1)
      return fmaf(float(a.d[0][h][j] * 256 + a.d[0][h][2 + j]), 256.0f, float(a.d[1][h][j] + a.d[2][h][2 + j]));
    return fmaf(float(a.d[0][h][2 * n + j] * 256 + a.d[1][h][2 * n + j]), 256.0f, float(a.d[2][h][2 * n + j]));
  }
  // A tile's row scales of this lane's tokens 2t, 2t + 1, 2t + 8, 2t + 9.
  static __device__ __forceinline__ void fp16_pairs(uint32_t a, uint32_t b, float (&x)[4]) {
    x[0] = f16_to_f32(uint16_t(a)); x[1] = f16_to_f32(uint16_t(a >> 16));
    x[2] = f16_to_f32(uint16_t(b)); x[3] = f16_to_f32(uint16_t(b >> 16));
  }
  __device__ __forceinline__ void int8_scales(uint32_t at, float (&ks)[4], float (&vs)[4]) const {
    at += 4 * t;
    fp16_pairs(lds32(at), lds32(at + 16), ks);
    if (odd_pages)  // the V rows start in the upper half of a word
      fp16_pairs(__byte_perm(lds32(at + 32), lds32(at + 36), 0x5432), __byte_perm(lds32(at + 48), lds32(at + 52), 0x5432), vs);
    else
      fp16_pairs(lds32(at + 32), lds32(at + 48), vs);
  }
  // Rows not in use weigh nothing: 0 for their scales.
  template <int K>
  __device__ __forceinline__ void zero_unused(float (&x)[K][4], int rows) const {
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (2 * t + (y & 1) + 8 * (y >> 1) >= rows)
#pragma unroll
        for (int k = 0; k < K; ++k) x[k][y] = 0.0f;
  }

  // A tile of a page of 8-bit codes, K then V.
  template <bool INT8>
  __device__ __forceinline__ void tile8(uint32_t tile, uint32_t scales, int rows) {
    float s[NT][4], vs[1][4] = {{1.0f, 1.0f, 1.0f, 1.0f}};
    if constexpr (INT8) {
      float ks[4];
      int8_scales(scales, ks, vs[0]);
      if (rows < 16) zero_unused(vs, rows);
      fit_scale(fmaxf(fmaxf(vs[0][0], vs[0][1]), fmaxf(vs[0][2], vs[0][3])) * kUnit8);
      Dots a;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 k[2] = {lds128(tile + k_off<D>(g, 4 * i + t)), lds128(tile + k_off<D>(g + 8, 4 * i + t))};
        add_digits(a, k, i, i == 0);
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][x] = dot_value(a, n, x) * (qs_i[n] * kUnit8 * ks[x]);
    } else {
      fit_scale(1.0f);
      float d[2][4], e[2][4];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        uint4 q[2][NT];
        load_q16(q[0], qh, 2 * (4 * i + t), true);
        load_q16(q[1], qh, 2 * (4 * i + t) + 1, true);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 k = lds128(tile + k_off<D>(g + 8 * h, 4 * i + t));
          dot16<false>(d[h], e[h], q[0], fp8_pair(k.x), fp8_pair(k.x >> 16), fp8_pair(k.y), fp8_pair(k.y >> 16), i == 0);
          dot16<false>(d[h], e[h], q[1], fp8_pair(k.z), fp8_pair(k.z >> 16), fp8_pair(k.w), fp8_pair(k.w >> 16), false);
        }
      }
      gather16(s, d, e);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) s[n][x] *= qs_h[n];
    }
    tile += 16 * D;
    // V's first 64 channels are on their way from shared memory while the scores become weights
    const auto load_v = [&](int i, int k) {
      return lds64(tile + v_off<D>(2 * t + (k & 1) + 8 * (k >> 1), 4 * i + (g >> 1)) + (g & 1) * 8);
    };
    uint2 raw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) raw[k] = load_v(0, k);
    weights(s, rows);
    uint32_t b[NT][2];
    fp16_weights(s, vs[0], INT8 ? c * kUnit8 : c, b);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      uint32_t v[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 x = i == 0 ? raw[k] : load_v(i, k);
        v[k][0] = INT8 ? x.x ^ 0x80808080u : x.x;
        v[k][1] = INT8 ? x.y ^ 0x80808080u : x.y;
      }
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // channels 4w + 2h, + 1: (token, next token) bytes side by side
          const uint32_t lo = __byte_perm(v[0][w], v[1][w], h ? 0x7362 : 0x5140);
          const uint32_t hi = __byte_perm(v[2][w], v[3][w], h ? 0x7362 : 0x5140);
          uint4 a;
          if constexpr (INT8)
            a = make_uint4(int8_pair(lo, 0x4140), int8_pair(lo, 0x4342), int8_pair(hi, 0x4140), int8_pair(hi, 0x4342));
          else
            a = make_uint4(fp8_pair(lo), fp8_pair(lo >> 16), fp8_pair(hi), fp8_pair(hi >> 16));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<false>(acc[n][4 * i + 2 * w + h], a, b[n][0], b[n][1]);
        }
    }
  }

  // Sixteen nibbles (8 bytes: byte j = channel 2j in the high nibble, 2j + 1) as int8 16 * (nibble -
  // 8) in channel order: a nibble in the upper half of a byte with its top bit flipped.
  static __device__ __forceinline__ uint4 nibbles_x16(uint2 w) {
    const uint32_t e0 = (w.x & 0xF0F0F0F0u) ^ 0x80808080u, o0 = ((w.x << 4) & 0xF0F0F0F0u) ^ 0x80808080u;
    const uint32_t e1 = (w.y & 0xF0F0F0F0u) ^ 0x80808080u, o1 = ((w.y << 4) & 0xF0F0F0F0u) ^ 0x80808080u;
    return make_uint4(__byte_perm(e0, o0, 0x5140), __byte_perm(e0, o0, 0x7362), __byte_perm(e1, o1, 0x5140),
                      __byte_perm(e1, o1, 0x7362));
  }

  __device__ __forceinline__ void int4_scales(uint32_t at, float (&x)[D / 64][4]) const {
    const uint2 a = lds64(at), b = lds64(at + 32);
    const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      if constexpr (D == 128) {
        x[0][y] = bf16lo(w[y]);
        x[1][y] = bf16hi(w[y]);
      } else {
        x[0][y] = odd_head ? bf16hi(w[y]) : bf16lo(w[y]);
      }
    }
  }

  // A tile of an INT4 page (scales per 64 channels), K then V.
  __device__ __forceinline__ void tile4(uint32_t tile, uint32_t scales, int rows) {
    constexpr int K = D / 64;
    float ks[K][4], vs[K][4];
    int4_scales(scales + 8 * t, ks);
    int4_scales(scales + 8 * t + 64, vs);
    if (rows < 16) zero_unused(vs, rows);
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) top = fmaxf(top, fmaxf(fmaxf(vs[k][0], vs[k][1]), fmaxf(vs[k][2], vs[k][3])));
    fit_scale(top * kUnit4);
    float s[NT][4];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint4 x[2] = {nibbles_x16(lds64(tile + k_off<D / 2>(g, 2 * k + (t >> 1)) + (t & 1) * 8)),
                          nibbles_x16(lds64(tile + k_off<D / 2>(g + 8, 2 * k + (t >> 1)) + (t & 1) * 8))};
      Dots a;
      add_digits(a, x, k, true);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          // (the factor of the query meets the scale first: a product of up to 2^35 and a scale above 2^93 would overflow)
          const float z = dot_value(a, n, y), f = ks[k][y] * (qs_i[n] * (0.0625f * kUnit4));
          s[n][y] = k ? fmaf(z, f, s[n][y]) : z * f;
        }
    }
    tile += 8 * D;
    // V is on its way from shared memory while the scores become weights
    uint32_t raw[K][4];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        raw[k][j] = lds32(tile + v_off<D / 2>(2 * t + (j & 1) + 8 * (j >> 1), 2 * k + (g >> 2)) + (g & 3) * 4);
    weights(s, rows);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      uint32_t b[NT][2];
      fp16_weights(s, vs[k], c * kUnit4, b);
      const uint32_t (&v)[4] = raw[k];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // bytes 2h, 2h + 1 of both tokens: four channels
        uint32_t lo = __byte_perm(v[0], v[1], h ? 0x7632 : 0x5410), hi = __byte_perm(v[2], v[3], h ? 0x7632 : 0x5410);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint4 a = make_uint4(nibble_hi(lo), nibble_lo(lo), nibble_hi(hi), nibble_lo(hi));
#pragma unroll
          for (int n = 0; n < NT; ++n) mma16816<false>(acc[n][4 * k + 2 * h + w], a, b[n][0], b[n][1]);
          lo >>= 8;
          hi >>= 8;
        }
      }
    }
  }

  // The log2-sum of the page that just ended, for its mass.
  __device__ __forceinline__ void page_sum(int b, int pos, int hq0, int nq) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float sum = sum_over_tokens(ps[n]);
      if (t == 0 && 8 * n + g < nq)
        p.page_lse2[(int64_t(b) * p.max_pages + pos) * p.heads_q + hq0 + 8 * n + g] = m[n] + __log2f(sum);
      ps[n] = 0.0f;
    }
  }
  // The segment's partial result.
  __device__ void finish(int64_t row0, int nq) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float sum = sum_over_tokens(l[n]);
      if (t == 0 && 8 * n + g < nq) p.part_lse2[row0 + 8 * n + g] = m[n] + log2f(sum);
      const float own = sum == 0.0f ? 0.0f : (1.0f / sum) * (1.0f / c);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float inv = of_column(own, j);
        const int q = 8 * n + 2 * t + j;
        if (q >= nq) continue;
        float* o = p.part_o + (row0 + q) * D;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          float x[8];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            x[2 * w] = acc[n][4 * i + w][j] * inv;
            x[2 * w + 1] = acc[n][4 * i + w][2 + j] * inv;
          }
          float4* at = reinterpret_cast<float4*>(o + 64 * i + 8 * g);
          at[0] = make_float4(x[0], x[1], x[2], x[3]);
          at[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
      }
    }
  }
};

// Four workers and a producer, 128 registers a thread, three such CTAs on an SM
// (two with NT = 2).  Why a producer: a worker that copies its own units spent
// about 240 of 550 instructions for a page and head on look-ups and copies; here
// eight lanes for each of four workers issue them once (INT8 135 -> 131 us, FP8 31 -> 23).  Why cp.async and
// not tensor copies: a unit is 1 to 4 KB in runs of 64 to 256 bytes, and one lane
// per worker issuing boxes measured 129 against 128 us (INT8) and 68 against 63
// (131071 INT4 tokens).  A ring of three units leaves two on their way: 24 to an
// SM, 48 to 96 KB, which covers a microsecond of HBM's full rate.
template <int D, int NT>
__global__ void __launch_bounds__(kThreadsA, NT == 1 ? 3 : 2) decode_partials_kernel(const __grid_constant__ AttnParams p) {
  using Layout = UnitLayout<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Share s_share[kWarpsA];
  __shared__ __align__(8) uint64_t s_bars[kWarpsA][2 * kRing];  // full, empty
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cells = p.heads_kv * p.q_chunks;
  // the worker of this warp, or of this lane of the producer
  const int mine = warp < kWarpsA ? warp : lane >> 3;
  const int w = int(blockIdx.x) * kWarpsA + mine;
  const int range = w / cells, cell = w % cells;
  const int hk = cell % p.heads_kv, q0 = (cell / p.heads_kv) * (8 * NT);
  const uint32_t ring = ((smem_u32(smem) + 1023u) & ~1023u) + uint32_t(mine * p.warp_smem), bars = smem_u32(s_bars[mine]);
  wait_for_previous();
  if (warp < kWarpsA) {
    Share sh{0, 0, 0, 0};
    if (range < p.ranges) {
      const int total = lists_before(p, p.n_seqs, hk), len = range_len(p, total);
      const int64_t at = int64_t(range) * len;
      sh.pos = int(min(at, int64_t(total)));
      sh.end = int(min(at + len, int64_t(total)));
      if (sh.pos < sh.end) {  // the sequence that the range starts in
        for (int b0 = 0;; b0 += 32) {
          const int n = b0 + lane < p.n_seqs ? list_len(p, b0 + lane, hk) : 0;
          int upto = n;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const int x = __shfl_up_sync(0xFFFFFFFFu, upto, off);
            if (lane >= off) upto += x;
          }
          const unsigned past = __ballot_sync(0xFFFFFFFFu, sh.before + upto > sh.pos);
          if (past || b0 + 32 >= p.n_seqs) {
            const int l = past ? __ffs(past) - 1 : 31;
            sh.b = b0 + l;
            sh.before += __shfl_sync(0xFFFFFFFFu, upto - n, l);
            break;
          }
          sh.before += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
      }
    }
    if (lane == 0) {
      s_share[warp] = sh;
      for (int k = 0; k < kRing; ++k) {
        mbar_init(&s_bars[warp][k], 9);          // eight lanes' copies and the header
        mbar_init(&s_bars[warp][kRing + k], 1);
      }
      mbar_init_fence();
    }
  }
  __syncthreads();
  allow_next();
  if (warp == kWarpsA) {
    Producer<D>(p, hk, s_share[mine], ring, bars).run();
    return;
  }
  Worker<D, NT> work(p, ring + Layout::kBytes, hk);
  const int nq = min(8 * NT, p.group - q0), hq0 = hk * p.group + q0;
  int b = s_share[warp].b, before = s_share[warp].before, pos = s_share[warp].pos;
  const int end = s_share[warp].end;
  uint32_t slot = 0, phase = 0;
  for (; pos < end; ++b) {
    const int n = list_len(p, b, hk);
    if (n == 0) continue;
    work.start(b, hq0, nq);
    float s[NT][4];  // weights of a BF16 tile between its K and its V unit
    for (bool last = false; !last;) {
      if (!Producer<D>::wait_bar(bars + slot * 8, phase)) {
        flag(p.status, ASHKV_FLAG_TIMEOUT);
        return;
      }
      const uint32_t unit = ring + slot * Layout::kData, scales = ring + Layout::kScales + slot * 128;
      const uint4 h4 = lds128(ring + Layout::kHeaders + slot * 16);
      const Header h{reinterpret_cast<const uint8_t*>(uint64_t(h4.x) | uint64_t(h4.y) << 32), h4.z, int32_t(h4.w)};
      if (h.format() >= ASHKV_PAGE_NBIT4 && h.rows()) {
        const int t0 = int(h.meta >> 20) * 16;
        const bool is_v = h.meta & Header::kIsV;
        if (h.format() == ASHKV_PAGE_NBIT4)
          decode_nbit<D, 4>(unit, h.slot, p.T, p.row_len, p.outlier_cap, hk, is_v, t0, h.rows());
        else
          decode_nbit<D, 2>(unit, h.slot, p.T, p.row_len, p.outlier_cap, hk, is_v, t0, h.rows());
      }
      if (h.rows() == 0) {
      } else if (h.format() == ASHKV_PAGE_INT8) {
        work.template tile8<true>(unit, scales, h.rows());
      } else if (h.format() == ASHKV_PAGE_FP8) {
        work.template tile8<false>(unit, scales, h.rows());
      } else if (h.format() == ASHKV_PAGE_INT4) {
        work.tile4(unit, scales, h.rows());
      } else if (h.meta & Header::kIsV) {
        work.bf16_values(unit, s);
      } else {
        work.bf16_scores(unit, h.rows(), s);
      }
      if (p.mass && (h.meta & Header::kPageEnd) && h.rows()) work.page_sum(b, h.pos, hq0, nq);
      last = h.meta & Header::kSegmentEnd;
      __syncwarp();  // every lane has read the unit
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bars + (kRing + slot) * 8) : "memory");
      if (++slot == kRing) {
        slot = 0;
        phase ^= 1u;
      }
    }
    work.finish(int64_t(range + b) * p.heads_q + hq0, nq);
    if (lane == 0) {
      if (pos == before) p.first_range[int64_t(b) * p.heads_kv + hk] = range;
      if (before + n <= end) p.last_range[int64_t(b) * p.heads_kv + hk] = range;
    }
    before += n;
    pos = before;
  }
}

// The ranges r0 .. r1 that hold pages of (sequence b, key head hk); none: r1 < r0.
__device__ __forceinline__ void partials_of(const AttnParams& p, int b, int hk, int& r0, int& r1) {
  const int64_t at = int64_t(b) * p.heads_kv + hk;
  const bool any = list_len(p, b, hk) > 0;
  r0 = min(max(p.first_range[at], 0), p.ranges - 1);
  r1 = any ? min(max(p.last_range[at], r0), p.ranges - 1) : r0 - 1;
}
// (m, l) <- the log2-sum of (m, l) and (m2, l2): m + log2 l; NaN stays.
__device__ __forceinline__ void merge_lse2(float& m, float& l, float m2, float l2) {
  const float top = m2 > m || m2 != m2 ? m2 : m, ref = top == -INFINITY ? 0.0f : top;
  l = l * ex2(m - ref) + l2 * ex2(m2 - ref);
  m = top;
}
__device__ __forceinline__ float lse2_of(float m, float l) { return (m == -INFINITY ? 0.0f : m) + log2f(l); }

constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kLongRow = 24;  // a row of more partials takes the block's warps together

// A result row, its partials shared by W warps (this one is the first'th; with W = kJoinWarps the
// block's, added through shared memory s_join [kJoinWarps][D]).
template <int D, int W>
__device__ __forceinline__ void join_row(const AttnParams& p, int64_t row, int first, int r0, int r1, float* s_join) {
  static_assert(W == 1 || W == kJoinWarps, "a row has one warp or the block's");
  constexpr int N = D / 32;               // channels of a lane
  constexpr int kAhead = W == 1 ? 6 : 2;  // partials of a warp that are on their way while the total is found
  const int lane = threadIdx.x & 31;
  const int b = int(row / p.heads_q), hq = int(row % p.heads_q);
  if (first == 0 && lane == 0 && hq % p.group == 0) {  // what list_len cut
    const int32_t n = p.selected ? p.selected_count[int64_t(b) * p.heads_kv + hq / p.group] : 0;
    if (p.lengths[b] != seq_tokens(p, b) || n < 0 || n > p.max_selected) flag(p.status, ASHKV_FLAG_INDEX_RANGE);
  }
  const float* lse = p.part_lse2 + int64_t(b) * p.heads_q + hq;  // + r * heads_q
  const float* rows = p.part_o + (int64_t(b) * p.heads_q + hq) * D + lane * N;  // + r * heads_q * D
  const auto load_row = [&](int r, float (&v)[N]) {
    if constexpr (N == 4) {
      const float4 f = *reinterpret_cast<const float4*>(rows + int64_t(r) * p.heads_q * D);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const float2 f = *reinterpret_cast<const float2*>(rows + int64_t(r) * p.heads_q * D);
      v[0] = f.x; v[1] = f.y;
    }
  };
  float ahead[kAhead][N] = {};
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (r0 + first + k * W <= r1) load_row(r0 + first + k * W, ahead[k]);
  float m = -INFINITY, l = 0.0f;
  for (int r = r0 + lane; r <= r1; r += 32) merge_lse2(m, l, lse[int64_t(r) * p.heads_q], 1.0f);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    merge_lse2(m, l, __shfl_xor_sync(0xFFFFFFFFu, m, off), __shfl_xor_sync(0xFFFFFFFFu, l, off));
  const float total = lse2_of(m, l);
  float acc[N] = {};
  const auto add_row = [&](int r, const float (&v)[N]) {
    const float x = lse[int64_t(r) * p.heads_q], w = x == -INFINITY ? 0.0f : ex2(x - total);
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = fmaf(w, v[k], acc[k]);
  };
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (r0 + first + k * W <= r1) add_row(r0 + first + k * W, ahead[k]);
#pragma unroll 4
  for (int r = r0 + first + kAhead * W; r <= r1; r += W) {
    float v[N];
    load_row(r, v);
    add_row(r, v);
  }
  uint16_t* out = p.out + row * D;  // (any alignment of 2 bytes)
  if constexpr (W == 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) out[lane * N + k] = f32_to_bf16(acc[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) s_join[first * D + lane * N + k] = acc[k];
    __syncthreads();
    for (int ch = threadIdx.x; ch < D; ch += kJoinThreads) {
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += s_join[w * D + ch];
      out[ch] = f32_to_bf16(sum);
    }
  }
  if (first == 0 && lane == 0 && p.lse) p.lse[row] = total * kLn2;
}

// The first blocks hold the result rows: W = kJoinWarps: a block for each; W = 1: a
// warp for each, but for the rows of many partials (a long sequence among short
// ones), which the block's warps then take together, one row after the other.
// With mass, then blocks for kMassPages pages of a sequence each: the total
// log2-sum of every head, then a half warp per page over the heads.  Bound by the
// latency of three dependent loads; 4 to 10 us.
constexpr int kMassPages = 64;
template <int D, int W>
__global__ void __launch_bounds__(kJoinThreads) decode_join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int kWarps = kJoinWarps, kRows = kWarps / W;  // rows of a block
  extern __shared__ float s_join[];  // [kWarps][D], or [heads_q] and [2][kJoinThreads]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  wait_for_previous();  // the partials
  const int64_t n_out = int64_t(p.n_seqs) * p.heads_q, out_blocks = (n_out + kRows - 1) / kRows;
  if (blockIdx.x < out_blocks) {
    // a block's rows lie far apart, so that the heads of one long sequence are in as many blocks
    const auto row_of = [&](int k) { return int64_t(blockIdx.x) + k * out_blocks; };
    const auto partials = [&](int64_t row, int& r0, int& r1) {
      partials_of(p, int(row / p.heads_q), int(row % p.heads_q) / p.group, r0, r1);
    };
    int r0 = 0, r1 = -1;
    if constexpr (W == 1) {
      const int64_t row = row_of(warp);
      if (row < n_out) partials(row, r0, r1);
      const bool split = r1 - r0 >= kLongRow;
      if (row < n_out && !split) join_row<D, 1>(p, row, 0, r0, r1, s_join);
      if (!__syncthreads_or(split)) return;
      for (int k = 0; k < kRows && row_of(k) < n_out; ++k) {
        partials(row_of(k), r0, r1);
        if (r1 - r0 < kLongRow) continue;
        join_row<D, kWarps>(p, row_of(k), warp, r0, r1, s_join);
        __syncthreads();  // s_join is read before the next row's sums
      }
    } else {
      partials(row_of(0), r0, r1);
      join_row<D, kWarps>(p, row_of(0), warp, r0, r1, s_join);
    }
    return;
  }
  const int per = (p.max_pages + kMassPages - 1) / kMassPages;
  const int64_t mb = int64_t(blockIdx.x) - out_blocks;
  const int b = int(mb / per), j0 = int(mb % per) * kMassPages;
  const int pages = int((seq_tokens(p, b) + p.T - 1) / p.T), j1 = min(pages, j0 + kMassPages);
  if (j0 >= j1) return;
  float* s_total = s_join;
  for (int h0 = 0; h0 < p.heads_q; h0 += 32) {  // 32 heads at a time, a warp's lanes; the warps share the partials
    const int hq = h0 + lane;
    float m = -INFINITY, l = 0.0f;
    if (hq < p.heads_q) {
      int r0, r1;
      partials_of(p, b, hq / p.group, r0, r1);
#pragma unroll 4
      for (int r = r0 + warp; r <= r1; r += kWarps)
        merge_lse2(m, l, p.part_lse2[int64_t(r + b) * p.heads_q + hq], 1.0f);
    }
    float* s_m = s_join + p.heads_q;
    s_m[tid] = m;
    s_m[kJoinThreads + tid] = l;
    __syncthreads();
    if (warp == 0 && hq < p.heads_q) {
#pragma unroll
      for (int w = 1; w < kWarps; ++w) merge_lse2(m, l, s_m[w * 32 + lane], s_m[kJoinThreads + w * 32 + lane]);
      s_total[hq] = lse2_of(m, l);
    }
    __syncthreads();
  }
  const int half = tid >> 4, sub = tid & 15;
  for (int j = j0 + half; j - half < j1; j += kJoinThreads / 16) {
    float sum = 0.0f;
    if (j < j1) {
      const float* pl = p.page_lse2 + (int64_t(b) * p.max_pages + j) * p.heads_q;
      for (int h = sub; h < p.heads_q; h += 16)
        if (pl[h] != -INFINITY) sum += ex2(pl[h] - s_total[h]);
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
    if (sub == 0 && j < j1) {
      float* at = p.mass + int64_t(b) * p.mass_stride + j;
      *at = fmaf(p.decay, *at, sum);
    }
  }
}

// Ranges that fill the GPU once with `per_sm` workers on an SM.
int ranges_for(int64_t n_seqs, int heads_kv, int q_chunks, int64_t pages_per_list, int per_sm) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const int64_t fit = std::max<int64_t>(1, int64_t(sms) * per_sm / (int64_t(heads_kv) * q_chunks));
  return int(std::max<int64_t>(1, std::min<int64_t>(fit, n_seqs * pages_per_list)));
}
// Query heads of one worker: one or two column tiles.  Two read a page once for up to 16 heads of a
// group but hold twice the sums, so 8 instead of 12 workers fit an SM.  16 x 8192 tokens, 8 key heads:
// groups of 16 take 135 us (bf16), 114 (INT8), 115 (INT4) with two and 152, 128, 131 as two halves of
// 8, groups of 10 bf16 125 and 150; groups of 8 take 106, 79, 78 with one and 122, 102, 103 with two.
int worker_queries(int group) { return group <= 8 ? 8 : 16; }
int q_chunks_for(int heads_q, int heads_kv) {
  const int group = heads_q / heads_kv, n = worker_queries(group);
  return (group + n - 1) / n;
}

bool row_ok(int64_t row) { return row == 128 || row == 256 || row == 512 || row == 1024 || row == 2048; }

// The page description of a call; the message of what is wrong with it, or nullptr.
const char* copy_pages(const ashkv_paged_kv_t* kv, AttnParams& p) {
  if (!kv) return "null page description";
  if (kv->head_dim != 64 && kv->head_dim != 128) return "head_dim must be 64 or 128";
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

ashkv_status_t refuse(const char* what, const char* why) {
  char text[256];
  snprintf(text, sizeof text, "%s: %s", what, why);
  set_message(text);
  return ASHKV_BAD_ARGUMENT;
}

// Warps of a result row in the join.  One warp per row makes eight times fewer CTAs and needs no second
// sum, eight read a row's partials at once.  Calls with one / eight warps, by partials to a row: 1.7 (128 x
// 1024 bf16 tokens, 64 heads) 109 / 129 us; 3.5 (64 x 2048 INT8) 79 / 88; 7 (32 x 8192 bf16) 183 / 186; 9 (24 x
// 8192 INT8) 103.8 / 104.4; 14 (16 x 8192 bf16) 106.6 / 105.3; 28 (8 x 8192) 68.9 / 65.7; 111 (2 x 8192) 41 / 33.
// One sequence of 131072 among 31 of 30 tokens: 219 / 213 (230 if its rows had one warp each).
int join_warps(const AttnParams& p) { return p.ranges <= int64_t(p.n_seqs) * 10 ? 1 : 8; }

template <int D, int NT>
ashkv_status_t launch_decode(AttnParams& p, cudaStream_t st) {
  const int64_t workers = int64_t(p.ranges) * p.heads_kv * p.q_chunks;
  p.warp_smem = int(UnitLayout<D>::kBytes) + NT * 8 * D * (2 + (p.fp8_pages ? 2 : 0) + (p.int_pages ? 3 : 0));
  p.warp_smem = (p.warp_smem + 1023) / 1024 * 1024;
  const int smem = kWarpsA * p.warp_smem + 1024;
  // The attribute is the kernel's on a device and outlasts the call: asked for once with the most that
  // any stores need.
  static std::atomic<bool> allowed[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !allowed[dev].load(std::memory_order_acquire))) {
    constexpr int kMost = kWarpsA * ((int(UnitLayout<D>::kBytes) + NT * 8 * D * 7 + 1023) / 1024 * 1024) + 1024;
    e = cudaFuncSetAttribute(decode_partials_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e == cudaSuccess && dev < 64) allowed[dev].store(true, std::memory_order_release);
  }
  if (e != cudaSuccess) {
    set_error("ashkv_decode_attention (shared memory attribute)", e);
    return ASHKV_LAUNCH_ERROR;
  }
  launch_overlapped(decode_partials_kernel<D, NT>, dim3(unsigned((workers + kWarpsA - 1) / kWarpsA)), dim3(kThreadsA),
                    size_t(smem), st, p);
  const ashkv_status_t rc = check_launch("ashkv_decode_attention");
  if (rc != ASHKV_OK) return rc;
  const int64_t rows = int64_t(p.n_seqs) * p.heads_q;
  const int w = join_warps(p), per_block = kJoinThreads / 32 / w;
  int64_t blocks = (rows + per_block - 1) / per_block;
  size_t join_smem = kJoinThreads / 32 * D * 4;
  if (p.mass) {
    blocks += int64_t(p.n_seqs) * ((p.max_pages + kMassPages - 1) / kMassPages);
    join_smem = std::max(join_smem, size_t(p.heads_q + 2 * kJoinThreads) * 4);
  }
  launch_overlapped(w == 1 ? decode_join_kernel<D, 1> : decode_join_kernel<D, 8>, dim3(unsigned(blocks)), dim3(kJoinThreads),
                    join_smem, st, p);
  return check_launch("ashkv_decode_attention");
}

}  // namespace
}  // namespace ashkv

using namespace ashkv;

extern "C" int64_t ashkv_decode_scratch_floats(int32_t n_seqs, int32_t heads_q, int32_t heads_kv, int32_t head_dim,
                                               int32_t pages_per_list, int32_t with_mass) {
  if (n_seqs < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || head_dim <= 0 || pages_per_list < 0) return -1;
  const int64_t slots = int64_t(ranges_for(n_seqs, heads_kv, q_chunks_for(heads_q, heads_kv), pages_per_list, kWorkersPerSm)) +
                        n_seqs;
  int64_t n = slots * heads_q * (int64_t(head_dim) + 1) + 2 * int64_t(n_seqs) * heads_kv;
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
  if (width < 0 || int64_t(n_seqs) * width > kMostEntries || int64_t(n_seqs) * max_pages > kMostEntries)
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
  for (int t = 1; t < kTiers; ++t) {
    p.fp8_pages |= p.store[t].format == ASHKV_PAGE_FP8;
    p.int_pages |= p.store[t].format == ASHKV_PAGE_INT8 || p.store[t].format == ASHKV_PAGE_INT4;
  }
  const bool two_ctas = worker_queries(p.group) == 16 || (p.fp8_pages && p.int_pages);
  p.ranges = ranges_for(n_seqs, p.heads_kv, p.q_chunks, width, two_ctas ? 2 * kWarpsA : kWorkersPerSm);
  const int64_t rows = (int64_t(p.ranges) + n_seqs) * heads_q;
  p.part_o = d_scratch;
  p.part_lse2 = p.part_o + rows * kv->head_dim;
  p.first_range = reinterpret_cast<int32_t*>(p.part_lse2 + rows);
  p.last_range = p.first_range + int64_t(n_seqs) * p.heads_kv;
  p.page_lse2 = reinterpret_cast<float*>(p.last_range + int64_t(n_seqs) * p.heads_kv);
  cudaStream_t st = as_stream(stream);
  if (worker_queries(p.group) == 8) return kv->head_dim == 64 ? launch_decode<64, 1>(p, st) : launch_decode<128, 1>(p, st);
  return kv->head_dim == 64 ? launch_decode<64, 2>(p, st) : launch_decode<128, 2>(p, st);
}
