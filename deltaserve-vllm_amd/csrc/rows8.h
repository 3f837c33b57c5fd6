// Device side of 8-bit rows (dsb_rows8_* in include/dsb.h): codes with a power-of-two scale per 32
// columns.
//
//   e = the least with max|block| <= M·2^e, M = 448 (e4m3) or 127 (int8), at least −126
//   code = round(v·2^−e) to nearest even; value = code·2^e
//
// Every step but the one rounding is exact: the scale is a shift of the exponent, so codes are the same
// however they are computed, and a value has at most 8 significant bits, so that bf16 holds it. The
// byte of a block is e + 127; a block with an infinity or a NaN has byte 255 and codes 0, and 0 times
// the byte's 2^128 (infinity) is NaN again.
#pragma once

#include "kernels.h"

namespace dsb {

constexpr int kBlock8 = DSB_ROWS8_BLOCK;

// The exponent byte of a block by the bits of its largest magnitude: carries into the exponent where
// the mantissa is past M's.
template <int CODE>
DSB_DEV unsigned scale_byte(unsigned amax) {
  constexpr unsigned kMant = CODE == DSB_DT_E4M3 ? 0x600000u : 0x7e0000u;  // 1.75, 1.984375
  constexpr int kExp = CODE == DSB_DT_E4M3 ? 8 : 6;
  if (amax >= 0x7f800000u) return 255u;
  return (unsigned)max((int)((amax + (0x7fffffu - kMant)) >> 23) - kExp, 1);
}
DSB_DEV float scale_of(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }
// 2^−e of a byte (of 255: anything, its codes are 0).
DSB_DEV float inverse_scale_of(unsigned byte) {
  return __builtin_bit_cast(float, (254u - min(byte, 253u)) << 23);
}

// Four codes of v·inv, in a word.
template <int CODE>
DSB_DEV unsigned encode4(const float* v, float inv) {
  if constexpr (CODE == DSB_DT_E4M3) {
    const unsigned r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, r, true);
  } else {
    // v·inv (exact) + 3·2^22 is rounded to a whole number, whose low byte is the code
    unsigned b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      b[i] = __builtin_bit_cast(unsigned, __builtin_fmaf(v[i], inv, 0x1.8p23f));
    // v_perm_b32: bytes 0 to 3 are the second operand's, 4 to 7 the first's
    const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
    const unsigned hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    return lo | hi;
  }
}
template <int CODE>
DSB_DEV u32x2 encode8(const float v[8], unsigned byte) {
  const float inv = inverse_scale_of(byte);
  const u32x2 c = {encode4<CODE>(v, inv), encode4<CODE>(v + 4, inv)};
  return byte == 255u ? u32x2{0u, 0u} : c;
}
template <int CODE>
DSB_DEV void decode4(unsigned c, float scale, float* v) {
  if constexpr (CODE == DSB_DT_E4M3) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
    const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    v[0] = a[0] * scale;
    v[1] = a[1] * scale;
    v[2] = b[0] * scale;
    v[3] = b[1] * scale;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(c >> (8 * i)) * scale;
  }
}
template <int CODE>
DSB_DEV void decode8(u32x2 c, unsigned byte, float v[8]) {
  const float s = scale_of(byte);
  decode4<CODE>(c[0], s, v);
  decode4<CODE>(c[1], s, v + 4);
}

// The largest over the four lanes that hold a block (8 columns each).
DSB_DEV unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true));  // lanes 1, 0, 3, 2
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true));  // lanes 2, 3, 0, 1
}
DSB_DEV unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// ---- rows of any of the types, 8 columns at a time
struct RowsArg {
  const void* p;
  long ld;  // in elements
  const uint8_t* s;
  long lds;
  int type;  // DSB_DT_*
};
enum { kRowsBF16 = 0, kRowsF32 = 1, kRows8 = 2, kRowsNone = 3 };
inline int rows_kind(int type) {
  return type == DSB_DT_BF16 ? kRowsBF16 : type == DSB_DT_F32 ? kRowsF32 : kRows8;
}

template <int KIND>
struct Raw8 {
  u32x4 a;
  DSB_DEV void load(const RowsArg& r, long row, int c) {
    a = ldg128_nt((const bf16*)r.p + row * r.ld + 8 * c);
  }
  DSB_DEV void get(const RowsArg&, float v[8]) const { unpack8(a, v); }
};
template <>
struct Raw8<kRowsF32> {
  u32x4 a, b;
  DSB_DEV void load(const RowsArg& r, long row, int c) {
    const float* p = (const float*)r.p + row * r.ld + 8 * c;
    a = ldg128_nt(p);
    b = ldg128_nt(p + 4);
  }
  DSB_DEV void get(const RowsArg&, float v[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned x = a[i], y = b[i];
      v[i] = __builtin_bit_cast(float, x);
      v[4 + i] = __builtin_bit_cast(float, y);
    }
  }
};
template <>
struct Raw8<kRows8> {
  u32x2 c;
  unsigned byte;
  DSB_DEV void load(const RowsArg& r, long row, int ch) {
    c = __builtin_nontemporal_load(
        reinterpret_cast<const u32x2*>((const uint8_t*)r.p + row * r.ld + 8 * ch));
    byte = r.s[row * r.lds + (ch >> 2)];
  }
  DSB_DEV void get(const RowsArg& r, float v[8]) const {
    if (r.type == DSB_DT_E4M3)  // the same for all lanes
      decode8<DSB_DT_E4M3>(c, byte, v);
    else
      decode8<DSB_DT_INT8>(c, byte, v);
  }
};
template <>
struct Raw8<kRowsNone> {
  DSB_DEV void load(const RowsArg&, long, int) {}
  DSB_DEV void get(const RowsArg&, float v[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
};

// 8 columns out, past the caches.
DSB_DEV void put8(void* p, long at, bool f32, const float v[8]) {
  if (f32) {
    f32x4* o = reinterpret_cast<f32x4*>((float*)p + at);
    __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, o);
    __builtin_nontemporal_store(f32x4{v[4], v[5], v[6], v[7]}, o + 1);
  } else {
    __builtin_nontemporal_store(pack8(v), reinterpret_cast<u32x4*>((bf16*)p + at));
  }
}

}  // namespace dsb
