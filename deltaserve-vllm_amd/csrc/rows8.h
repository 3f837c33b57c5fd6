// Device side of 8-bit rows (dsb_rows8_* in include/dsb.h): codes with a power-of-two scale per 32
// columns.
//
//   e = the least with max|block| <= M·2^e, M = 448 (e4m3) or 127 (int8), at least −126
//   code = round(v·2^−e) to nearest even, or the code below where that makes 2^128; value = code·2^e
//
// Every step but the one rounding is exact: the scale is a shift of the exponent, so codes are the same
// however they are computed, and a value has at most 8 significant bits, so that bf16 holds it. The
// byte of a block is e + 127; a block with an infinity or a NaN has byte 255 and codes 0, and 0 times
// the byte's 2^128 (infinity) is NaN again.
#pragma once

#include <type_traits>

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
// A block's values are at most M·2^e, so only with the last exponent (which takes M·2^e past fp32) may one round
// to 2^128: there the code below stands for it, 240 (e4m3) or 63 (int8) times the scale. (Saves of 8192 × 1024
// rows, calls in a graph: 7.25 µs, 7.2 without it; in a branch it costs no less.)
template <int CODE>
DSB_DEV u32x2 encode8(const float v[8], unsigned byte) {
  constexpr unsigned kLastByte = CODE == DSB_DT_E4M3 ? 127 + 120 : 127 + 122;
  constexpr float kLast = CODE == DSB_DT_E4M3 ? 0x1.ep127f : 0x1.f8p127f;
  const float inv = inverse_scale_of(byte), most = byte >= kLastByte ? kLast : __builtin_inff();
  float w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __builtin_amdgcn_fmed3f(v[i], -most, most);
  const u32x2 c = {encode4<CODE>(w, inv), encode4<CODE>(w + 4, inv)};
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

// ---- memory
// What a kernel leaves in the caches (the last level, 256 MB, keeps data from one kernel to the next):
//   kNear  loads through them, stores past the L2: inputs of up to a third of the last level, which the
//          kernel before may have left there; stores that stay in the L2 are written back at the kernel's end
//   kFar   loads past them, stores into them: larger inputs, and outputs that fit beside others
//   kPast  both past them: larger outputs
//   kIn    both through them: for stores that cover lines in parts
// µs, near / far / past (MB in, out): RMSNorm of 2048 × 4096 8-bit rows (8, 17) 5.0 / 8 / 8; rotary positions, 40
// heads of 8192 rows (84, 84) 29 / 31 / 34, of 10240 41 / 38 / 42, of 16384 67 / 68 / 65; SwiGLU of 2048 ×
// 14336 (61, 59) 18 / 21 / 23, of 4000 43 / 38 / 42, of 6500 71 / 78 / 68; 4096 × 28672 rows restored (121, 235)
// 70 / 73 / 69. (Three sets of inputs in turn, two of outputs.)
enum { kNear, kFar, kPast, kIn };
inline int cache_of(double in, double out) {
  constexpr double kLast = 256 << 20;
  return in <= kLast / 3 ? kNear : out <= 0.6 * kLast ? kFar : kPast;
}
template <int P, class V>
DSB_DEV V load_as(const void* p) {
  const V* q = reinterpret_cast<const V*>(p);
  if constexpr (P == kNear || P == kIn) return *q;
  return __builtin_nontemporal_load(q);
}
template <int P, class V>
DSB_DEV void store_as(void* p, V v) {
  V* q = reinterpret_cast<V*>(p);
  if constexpr (P == kFar || P == kIn)
    *q = v;
  else
    __builtin_nontemporal_store(v, q);
}
// Accesses of 16 and 8 bytes that need their elements' alignment only.
typedef unsigned u32x4h __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2b __attribute__((ext_vector_type(2), aligned(1)));

// ---- rows of any of the types, 8 columns at a time
struct RowsArg {
  const void* p;
  long ld;  // in elements
  const uint8_t* s;
  long lds;
  int type;  // DSB_DT_*
};
constexpr int kRowsNone = -1;
// Bytes of a column of such rows.
inline double row_bytes(const RowsArg& r) {
  return !r.p ? 0 : r.type == DSB_DT_BF16 ? 2 : r.type == DSB_DT_F32 ? 4 : 1 + 1.0 / kBlock8;
}

DSB_DEV void floats8(u32x4 a, u32x4 b, float v[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned x = a[i], y = b[i];
    v[i] = __builtin_bit_cast(float, x);
    v[4 + i] = __builtin_bit_cast(float, y);
  }
}
// As they lie, of type T.
template <int T>
struct Raw8 {  // 8-bit rows
  u32x2 c;
  unsigned byte;
  template <int P>
  DSB_DEV void load(const RowsArg& r, long row, int ch) {
    c = load_as<P, u32x2>((const uint8_t*)r.p + row * r.ld + 8 * ch);
    byte = r.s[row * r.lds + (ch >> 2)];
  }
  DSB_DEV void get(float v[8]) const { decode8<T>(c, byte, v); }
};
template <>
struct Raw8<DSB_DT_BF16> {
  u32x4 a;
  template <int P>
  DSB_DEV void load(const RowsArg& r, long row, int c) {
    a = load_as<P, u32x4>((const bf16*)r.p + row * r.ld + 8 * c);
  }
  DSB_DEV void get(float v[8]) const { unpack8(a, v); }
};
template <>
struct Raw8<DSB_DT_F32> {
  u32x4 a, b;
  template <int P>
  DSB_DEV void load(const RowsArg& r, long row, int c) {
    const float* p = (const float*)r.p + row * r.ld + 8 * c;
    a = load_as<P, u32x4>(p);
    b = load_as<P, u32x4>(p + 4);
  }
  DSB_DEV void get(float v[8]) const { floats8(a, b, v); }
};
template <>
struct Raw8<kRowsNone> {
  template <int P>
  DSB_DEV void load(const RowsArg&, long, int) {}
  DSB_DEV void get(float v[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
  }
};
template <int K>
using Int = std::integral_constant<int, K>;
// f with the type of rows as a constant.
template <class F>
hipError_t by_type(const RowsArg& r, F f) {
  switch (r.type) {
    case DSB_DT_BF16: return f(Int<DSB_DT_BF16>{});
    case DSB_DT_F32: return f(Int<DSB_DT_F32>{});
    case DSB_DT_E4M3: return f(Int<DSB_DT_E4M3>{});
    default: return f(Int<DSB_DT_INT8>{});
  }
}

// 8 columns out. Of fp32 they are two stores, each of every other 16 bytes of a line over a wave: past the caches, lines
// go out in parts where the second comes late (the join of 8191 × 4096 fp32 rows 78 µs so, 69 into them).
template <int P>
DSB_DEV void put8(void* p, long at, bool f32, const float v[8]) {
  constexpr int F = P == kPast ? kFar : P;
  if (f32) {
    store_as<F>((float*)p + at, f32x4{v[0], v[1], v[2], v[3]});
    store_as<F>((float*)p + at + 4, f32x4{v[4], v[5], v[6], v[7]});
  } else {
    store_as<P>((bf16*)p + at, pack8(v));
  }
}

}  // namespace dsb
