// Eight elements of a compressed page -> eight bf16, as the page's codec decodes them: shared by the
// page transcoder (migrate.cu), the dense read (cache.cu) and the attention of prompts (prompt.cu).
#pragma once

#include "common.cuh"
#include "fp8_conv.cuh"
#include "int4_group.cuh"
#include "nbit_group.cuh"
#include "page_layout.cuh"

namespace ashkv {
namespace {

// Eight INT8 codes with scale s -> eight bf16 (the reference decode).
__device__ __forceinline__ uint4 int8_dec8(uint2 cw, float s) {
  const Recip y = make_recip(127.0f);
  const f2 YHI = pk2(y.hi, y.hi), YLO = pk2(y.lo, y.lo), S = pk2(s, s);
  const bool fast = int8_dec_fast(s);
  const uint32_t ww[2] = {cw.x, cw.y};
  uint32_t o[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f2 F0, F1;
    int8x4_to_f2(ww[h], F0, F1);
    if (fast) {
      o[2 * h] = f32x2_to_bf16x2_pk(div2_short(mul2(F0, S), YHI, YLO));
      o[2 * h + 1] = f32x2_to_bf16x2_pk(div2_short(mul2(F1, S), YHI, YLO));
    } else {
      float a, b;
      upk2(F0, a, b);
      o[2 * h] = f32x2_to_bf16x2(__fdiv_rn(__fmul_rn(a, s), 127.0f), __fdiv_rn(__fmul_rn(b, s), 127.0f));
      upk2(F1, a, b);
      o[2 * h + 1] = f32x2_to_bf16x2(__fdiv_rn(__fmul_rn(a, s), 127.0f), __fdiv_rn(__fmul_rn(b, s), 127.0f));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
__device__ __forceinline__ uint4 fp8_dec8(uint2 c) {
  return make_uint4(bf16x2_from_fp8x2(c.x & 0xFFFFu), bf16x2_from_fp8x2(c.x >> 16),
                    bf16x2_from_fp8x2(c.y & 0xFFFFu), bf16x2_from_fp8x2(c.y >> 16));
}
__device__ __forceinline__ uint4 int4_dec8(uint32_t c, uint16_t scale) {
  uint32_t o[4];
  unpack_nibbles8(c, bf16_to_f32(scale), o);
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// Eight dithered codes (BITS = 4: a word; 2: its lower half) with the group's delta, without outliers.
template <int BITS>
__device__ __forceinline__ uint4 nbit_dec8(uint32_t w, uint16_t delta_bits) {
  constexpr float half = float((1 << BITS) - 1) * 0.5f;
  const float delta = bf16_to_f32(delta_bits);
  const f2 DEL = pk2(delta, delta), NH = pk2(-half, -half), N23 = pk2(-8388608.0f, -8388608.0f);
  auto pair = [&](float a, float b) { return f32x2_to_bf16x2_pk(mul2(add2(add2(pk2(a, b), N23), NH), DEL)); };
  uint32_t o[4];
  if constexpr (BITS == 4) {  // byte j = (elem 2j) << 4 | elem 2j+1
    const uint32_t hi = (w >> 4) & 0x0F0F0F0Fu, lo = w & 0x0F0F0F0Fu;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = pair(code_plus_2p23(hi, j), code_plus_2p23(lo, j));
  } else {  // four codes a byte, the first in the top bits
    const uint32_t c0 = (w >> 6) & 0x0303u, c1 = (w >> 4) & 0x0303u, c2 = (w >> 2) & 0x0303u, c3 = w & 0x0303u;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      o[2 * j] = pair(code_plus_2p23(c0, j), code_plus_2p23(c1, j));
      o[2 * j + 1] = pair(code_plus_2p23(c2, j), code_plus_2p23(c3, j));
    }
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace
}  // namespace ashkv
