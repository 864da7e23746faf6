// 8-bit activation checkpoints: the block format and the row loads / stores shared by its kernels.
//
// A row of C values is cut into blocks of 32 columns.  A block keeps ONE exponent byte b = e + 127 and 32 codes q in [-127, 127]:
//     value = q 2^e,   e = the smallest integer with max|x| <= 127.5 2^e   (kept within [-126, 121]),   q = round_half_even(x 2^-e)
// so a code is off by at most half a step, and a step is less than max|x| / 63.75.
// The step is a power of two on purpose: x 2^-e is exact, so the codes are whole numbers that do not depend on how a division rounds,
// and q 2^e is exact in bfloat16 (7 significant bits) -- the products of the backward pass read the codes as bf16 operands without a
// second rounding.  A block with an infinity or a NaN has b = 255 and stands for NaN in all its 32 columns.
// Magnitudes above 127.5 2^121 (only fp32 inputs have them) keep the largest code.
#pragma once
#include "aql_common.h"

namespace act8 {

constexpr int BLK = 32;

__device__ __forceinline__ uint32_t exp_byte(uint32_t amax_bits) {   // amax_bits: bits of max|x|
  if (amax_bits >= 0x7f800000u) return 255u;
  int b = (int)(amax_bits >> 23) - 6 + ((amax_bits & 0x7fffffu) > 0x7f0000u ? 1 : 0);   // e + 127
  return (uint32_t)min(max(b, 1), 248);
}
__device__ __forceinline__ float inv_step(uint32_t b) { return b == 255u ? 0.f : __uint_as_float((254u - b) << 23); }
__device__ __forceinline__ float step(uint32_t b) { return b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(b << 23); }

// four codes in one word.  The clamp to +-127 steps comes before the scaling (both are exact), then 1.5 2^23 + v / step rounds to the nearest even integer
// and leaves it, in two's complement, in the low byte
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv, float lim) {
  constexpr float MAGIC = 12582912.f;
  const uint32_t ua = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(a, -lim, lim), inv, MAGIC));
  const uint32_t ub = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(b, -lim, lim), inv, MAGIC));
  const uint32_t uc = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(c, -lim, lim), inv, MAGIC));
  const uint32_t ud = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(d, -lim, lim), inv, MAGIC));
  return __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u) | __builtin_amdgcn_perm(ud, uc, 0x04000c0cu);
}
// the eight codes of a chunk whose block has exponent byte b
__device__ __forceinline__ uint2 codes8(const float* v, uint32_t b) {
  const float inv = inv_step(b), lim = 127.f * step(b);
  return make_uint2(codes4(v[0], v[1], v[2], v[3], inv, lim), codes4(v[4], v[5], v[6], v[7], inv, lim));
}
// value of byte i of a word of codes: (code + 128) comes out of one v_cvt_f32_ubyte; both further steps are exact
template <int I>
__device__ __forceinline__ float value(uint32_t w, float st) {
  return ((float)(((w ^ 0x80808080u) >> (8 * I)) & 255u) - 128.f) * st;
}
__device__ __forceinline__ void values4(uint32_t w, float st, float* o) {
  o[0] = value<0>(w, st);
  o[1] = value<1>(w, st);
  o[2] = value<2>(w, st);
  o[3] = value<3>(w, st);
}

// ---- eight consecutive columns of a row, whatever the row's alignment (gfx950 loads and stores 16 bytes at any element address)
struct __attribute__((packed, aligned(2))) U4a2 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(4))) U4a4 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(2))) U2a2 { uint32_t x, y; };

template <class T>
struct Raw8;   // eight elements as loaded
template <>
struct Raw8<bf16_t> {
  uint32_t w[4];
};
template <>
struct Raw8<float> {
  uint32_t w[8];
};

// n = number of live columns of the chunk (<= 0: none, >= 8: all); dead columns read as zero
__device__ __forceinline__ void load_raw(const bf16_t* p, int n, Raw8<bf16_t>& r) {
  if (n >= 8) {
    const U4a2 v = *reinterpret_cast<const U4a2*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = 2 * i < n ? p[2 * i] : 0, hi = 2 * i + 1 < n ? p[2 * i + 1] : 0;
      r.w[i] = lo | (hi << 16);
    }
  }
}
__device__ __forceinline__ void load_raw(const float* p, int n, Raw8<float>& r) {
  if (n >= 8) {
    const U4a4 a = *reinterpret_cast<const U4a4*>(p), b = *reinterpret_cast<const U4a4*>(p + 4);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w, r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i] = i < n ? __float_as_uint(p[i]) : 0u;
  }
}
__device__ __forceinline__ void widen(const Raw8<bf16_t>& r, float* o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = bf16lo(r.w[i]);
    o[2 * i + 1] = bf16hi(r.w[i]);
  }
}
__device__ __forceinline__ void widen(const Raw8<float>& r, float* o) {
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void store8(bf16_t* p, int n, const float* v) {
  if (n >= 8) {
    *reinterpret_cast<U4a2*>(p) = U4a2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = f32_to_bf16(v[i]);
  }
}
__device__ __forceinline__ void store8(float* p, int n, const float* v) {
  if (n >= 8) {
    *reinterpret_cast<U4a4*>(p) = U4a4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    *reinterpret_cast<U4a4*>(p + 4) = U4a4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
}

// max over the four lanes of a quad (the four 8-column chunks of one block) of non-negative float bits
__device__ __forceinline__ uint32_t quad_umax(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false);   // quad_perm [1,0,3,2]
  v = max(v, o);
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false);            // quad_perm [2,3,0,1]
  return max(v, o);
}
// bits of the largest magnitude of eight elements, as fp32
__device__ __forceinline__ uint32_t amax_bits8(const Raw8<float>& r) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, r.w[i] & 0x7fffffffu);
  return m;
}
__device__ __forceinline__ uint32_t amax_bits8(const Raw8<bf16_t>& r) {   // two at a time: magnitudes compare as unsigned integers
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = r.w[i] & 0x7fff7fffu;
    m = __builtin_elementwise_max(m, *reinterpret_cast<const u16x2_t*>(&w));
  }
  return (uint32_t)max(m.x, m.y) << 16;
}

}  // namespace act8
