// Codes of the quantised cache: 8 bits per value and one fp32 scale per token's row of
// a KV head.  Value = code * scale.
//   e4m3  scale 2^e, the least with amax / 2^e <= 448; code = x / scale rounded to e4m3
//         (OCP).  Floating codes gain nothing from a scale between powers of two, and
//         with a power of two both steps are exact but for the one rounding: a value
//         read back in bf16 is exact, and quantising the read-back row again keeps its values.
//         (Not always its codes: a row whose amax is rounded down to 1.75 * 2^k gets half the
//         scale the next time, and codes of twice the size.)  Where 256 * scale would be
//         beyond the rows' type, its largest values take the code 240.
//   int8  scale amax / 127; code = x * (127 / amax) rounded to a whole number.
// Roundings are to nearest, ties to even.  amax counts as 2^-100 at least, so that scales
// and their inverses are normal numbers.  A row that holds an infinity or a NaN gets the
// scale NaN: each of its values reads as NaN.
#pragma once

#include "kvc_common.h"

namespace kvc {

constexpr int kQuantPage = 16;   // tokens of a block

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

struct RowScale {
  float scale, inverse;
  float most;   // the largest code
};

// amax: the row's largest |x| as fp32 bits (an infinity's or a NaN's if it holds one).
template <int kCode, bool kHalf>
__device__ __forceinline__ RowScale row_scale(uint32_t amax) {
  if (amax >= 0x7f800000u) {
    const float nan = __uint_as_float(0x7fc00000u);
    return {nan, nan, 0.f};
  }
  amax = max(amax, uint32_t(127 - 100) << 23);
  if constexpr (kCode == KVC_CODE_INT8) {
    const float a = __uint_as_float(amax);
    return {a / 127.f, 127.f / a, 127.f};
  } else {
    // 448 = 1.75 * 2^8: amax = m 2^e needs 2^(e-8), and above m = 1.75 twice that.
    const uint32_t e = (amax + 0x1fffffu) >> 23;
    const uint32_t largest = kHalf ? 127 + 16 : 127 + 128;   // amax above 1.75 * 2^15 or 2^127
    return {__uint_as_float((e - 8) << 23), __uint_as_float((262 - e) << 23),
            e == largest ? 240.f : 448.f};
  }
}

// Four codes of x / scale, the first in the low byte.
template <int kCode>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, RowScale s) {
  a *= s.inverse;
  b *= s.inverse;
  c *= s.inverse;
  d *= s.inverse;
  if constexpr (kCode == KVC_CODE_INT8) {
    const uint32_t i = uint32_t(int(rintf(a))), j = uint32_t(int(rintf(b)));
    const uint32_t k = uint32_t(int(rintf(c))), l = uint32_t(int(rintf(d)));
    return (i & 255u) | (j & 255u) << 8 | (k & 255u) << 16 | l << 24;
  } else {
    auto fit = [&](float x) { return __builtin_amdgcn_fmed3f(x, -s.most, s.most); };
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(fit(a), fit(b), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(fit(c), fit(d), r, true));
  }
}

// Code i of a word as a float (exact).
template <int kCode, int i>
__device__ __forceinline__ float decode1(uint32_t w) {
  if constexpr (kCode == KVC_CODE_INT8)
    return float(int8_t(w >> (8 * i)));
  else
    return __builtin_amdgcn_cvt_f32_fp8(int(w), i);
}

// Codes 2h and 2h + 1 of a word as two bf16 or fp16 (exact: a code has at most eight
// significant bits, and an e4m3 code's exponent fits fp16).
template <int kCode, bool kHalf, int h>
__device__ __forceinline__ uint32_t decode2(uint32_t w) {
  if constexpr (kCode == KVC_CODE_INT8) {
    const float a = decode1<kCode, 2 * h>(w), b = decode1<kCode, 2 * h + 1>(w);
    if constexpr (kHalf) {
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    } else {
      bf16x2_t r;
      r[0] = __bf16(a);
      r[1] = __bf16(b);
      return __builtin_bit_cast(uint32_t, r);
    }
  } else if constexpr (kHalf) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, h));
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, h));
  }
}

// Two floats rounded to bf16 or fp16.
template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kHalf) {
    f16x2_t r;
    r[0] = _Float16(a);
    r[1] = _Float16(b);
    return __builtin_bit_cast(uint32_t, r);
  } else {
    bf16x2_t r;
    r[0] = __bf16(a);
    r[1] = __bf16(b);
    return __builtin_bit_cast(uint32_t, r);
  }
}

template <bool kHalf>
__device__ __forceinline__ float unpack_lo(uint32_t w) {
  if constexpr (kHalf)
    return float(__builtin_bit_cast(f16x2_t, w)[0]);
  else
    return bf16lo(w);
}
template <bool kHalf>
__device__ __forceinline__ float unpack_hi(uint32_t w) {
  if constexpr (kHalf)
    return float(__builtin_bit_cast(f16x2_t, w)[1]);
  else
    return bf16hi(w);
}

}  // namespace kvc
