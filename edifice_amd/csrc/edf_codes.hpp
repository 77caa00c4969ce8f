// 8-bit numbers of a paged cache: whole numbers -127 .. 127 (EDF_INT8) or e4m3 floats (EDF_E4M3), in units of a
// float32 scale that the tokens of one page and key head share.
#pragma once

#include "edf_abi.hpp"
#include "edf_common.hpp"
#include "edf_mfma.hpp"

namespace edf {

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// C: the code's kind.  unpack4: four codes as float32, exactly; pack4: four values to codes, ties to even, whole
// numbers saturated, e4m3 for values up to 448 (what a scale leaves).
template <int C> struct Codes;
template <> struct Codes<EDF_INT8> {
  EDF_DEVICE static void unpack4(unsigned c, float* x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (float)(signed char)(c >> (8 * e));
  }
  // eight codes as float16, exactly: 1024 + (c + 128) has the byte in its last bits
  EDF_DEVICE static f16x8 half8(unsigned lo, unsigned hi) {
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const unsigned u = (e < 2 ? lo : hi) ^ 0x80808080u;
      const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, e & 1 ? 0x04030402u : 0x04010400u)) - off;
      y[2 * e] = x[0], y[2 * e + 1] = x[1];
    }
    return y;
  }
  EDF_DEVICE static unsigned pack4(const float* x) {
    unsigned c = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) c |= ((unsigned)(int)clampf(rintf(x[e]), -127.0f, 127.0f) & 255u) << (8 * e);
    return c;
  }
};
template <> struct Codes<EDF_E4M3> {
  EDF_DEVICE static void unpack4(unsigned c, float* x) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  }
  EDF_DEVICE static f16x8 half8(unsigned lo, unsigned hi) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
  EDF_DEVICE static unsigned pack4(const float* x) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true);
  }
};

}  // namespace edf
