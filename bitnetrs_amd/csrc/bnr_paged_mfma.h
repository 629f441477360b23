// bnr_paged_mfma.h -- what the paged cache's decode kernels on the matrix cores
// share: loads, and fp32 values as bf16 parts.  Included by the .hip sources only.
#pragma once

#include "bnr_paged.h"

namespace bnr {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// N dwords at p; NT: with the non-temporal hint.  V's loads take whole lines
// and have it; K's take half of each line, the other half comes with the next
// load and is not to be dropped before.  32 sequences of 128 to 4096 bf16 rows:
// 38.4 us; 41.2 with the hint on both, 45.0 on neither.
template <bool NT, int N>
__device__ __forceinline__ void load_bytes(const char *p, unsigned (&r)[N]) {
  const auto load = [](const auto *q) { return NT ? __builtin_nontemporal_load(q) : *q; };
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4 v = load(reinterpret_cast<const u32x4 *>(p + 4 * i));
      r[i] = v.x;
      r[i + 1] = v.y;
      r[i + 2] = v.z;
      r[i + 3] = v.w;
    }
  } else if constexpr (N == 2) {
    const u32x2 v = load(reinterpret_cast<const u32x2 *>(p));
    r[0] = v.x;
    r[1] = v.y;
  } else {
    r[0] = load(reinterpret_cast<const unsigned *>(p));
  }
}

// The upper halves of two floats: a's below b's.
__device__ __forceinline__ unsigned pack_hi(float a, float b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a),
                               0x07060302u);
}

// Three bf16 parts of 8 floats: truncation leaves 8 bits a part, so the parts
// sum to the value.  (Where the value is a product, the compiler may take the
// first rest from it unrounded: a rest of the other sign is less than half of
// the value's last place then.)  kFill: no part is zero or of the other sign,
// down to values of 2^-90: a rest is 2^-40 of the value at least, which no sum
// notices.  An infinity of the other operand then makes the infinity in each
// part's product that it makes with the value, where a zero would make NaN.
struct Parts {
  u32x4 p[3];
};
template <bool kFill>
__device__ __forceinline__ Parts split8(const float (&x)[8]) {
  Parts s;
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = kFill ? fabsf(x[i]) : x[i];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s.p[k][i] = pack_hi(r[2 * i], r[2 * i + 1]);
      if (kFill) s.p[k][i] |= pack_hi(x[2 * i], x[2 * i + 1]) & 0x80008000u;
    }
    if (k < 2)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        r[i] -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, r[i]) & 0xffff0000u);
        if (kFill) r[i] = fmaxf(r[i], fabsf(x[i]) * 0x1p-40f);
      }
  }
  return s;
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

}  // namespace bnr
