// Eight-bit blocks: 128 consecutive values of a row (or 128 x 128 values of a
// weight) held as OCP e4m3 with one scale 2^e, e the least integer with
// max |x| <= 448 2^e over the block's finite values, kept as the e8m0 byte
// e + 127 (0 .. 247; 127 for a block of zeros).  The scale is a power of two so
// that dividing by it, multiplying by it again and the matrix instruction's own
// scaling are all exact: the only rounding is that to e4m3 (2^-4 relative, and
// 2^-10 2^e below 2^-6 2^e).  Values that are not finite become e4m3's NaN, and
// leave the rest of their block as it is.
#pragma once
#include "kd_tile.h"

namespace kd {

constexpr int QB = 128;  // values of a block

template <class E>
KD_DEV void unpack8(const u32x4& v, float (&f)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[2 * w] = to_f32<E>(uint16_t(v[w] & 0xFFFFu));
    f[2 * w + 1] = to_f32<E>(uint16_t(v[w] >> 16));
  }
}

KD_DEV float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Bits of max |f| over the finite f; bits of non-negative floats order as they do.
KD_DEV uint32_t finite_max(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __float_as_uint(f[i]) & 0x7FFFFFFFu;
    m = max(m, u < 0x7F800000u ? u : 0u);
  }
  return m;
}

// Maximum over the 16 lanes of a DPP row (all lanes active): exchanges within
// pairs, fours, eights and the row
KD_DEV uint32_t row16_max(uint32_t m) {
  m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0xB1, 0xF, 0xF, true)));   // quad_perm 1 0 3 2
  m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x4E, 0xF, 0xF, true)));   // quad_perm 2 3 0 1
  m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x141, 0xF, 0xF, true)));  // row_half_mirror
  m = max(m, uint32_t(__builtin_amdgcn_mov_dpp(int(m), 0x140, 0xF, 0xF, true)));  // row_mirror
  return m;
}

// The scale's byte for a block whose finite maximum has the bits m: 448 = 1.75 2^8
KD_DEV uint32_t scale_byte(uint32_t m) {
  const int e = int(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return m == 0u ? 127u : uint32_t(max(e, 0));
}
KD_DEV float scale_value(uint32_t byte) {  // 2^(byte - 127); 2^-127 is subnormal
  return __uint_as_float(byte == 0u ? 0x00400000u : byte << 23);
}
KD_DEV float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }  // byte <= 253

// Eight finite values as e4m3 bytes under the scale (round to nearest even; scaled
// values are at most 448).  The conversions divide by the power of two themselves.
typedef short s16x2 __attribute__((ext_vector_type(2)));
KD_DEV u32x2 pack_finite(const float (&f)[8], float scale) {
  u32x2 w;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    s16x2 r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{}, f[4 * k], f[4 * k + 1], scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, f[4 * k + 2], f[4 * k + 3], scale, true);
    w[k] = __builtin_bit_cast(uint32_t, r);
  }
  return w;
}
// Bits of max |f|, NaN and infinities among them (0x7F800000 and above)
KD_DEV uint32_t any_max(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
  return m;
}
// the same of eight bf16 or fp16, as a 16-bit number
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
KD_DEV uint32_t any_max(const u32x4& v) {
  u16x2 m = __builtin_bit_cast(u16x2, v[0] & 0x7FFF7FFFu);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[i] & 0x7FFF7FFFu));
  return max(uint32_t(m[0]), uint32_t(m[1]));
}

// Eight values as e4m3 bytes under the scale whose inverse is inv, NaN where they are not finite
KD_DEV u32x2 pack_e4m3(const float (&f)[8], float inv) {
  float g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool fin = (__float_as_uint(f[i]) & 0x7FFFFFFFu) < 0x7F800000u;
    g[i] = fin ? f[i] * inv : __uint_as_float(0x7FC00000u);
  }
  u32x2 w;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(g[4 * k], g[4 * k + 1], 0, false);
    w[k] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(g[4 * k + 2], g[4 * k + 3], lo, true));
  }
  return w;
}
// and back, without the scale
KD_DEV void unpack_e4m3(const u32x2& w, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[k]), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[k]), true);
    f[4 * k] = lo[0], f[4 * k + 1] = lo[1], f[4 * k + 2] = hi[0], f[4 * k + 3] = hi[1];
  }
}

}  // namespace kd
