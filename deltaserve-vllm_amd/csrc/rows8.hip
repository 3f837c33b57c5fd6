// Rows in and out of 8 bits (rows8.h says what they are) and SwiGLU with its backward from rows of
// either kind. All of it is bound by its bytes.
//
// A lane holds 8 columns: its loads of 16 bytes (8 of codes) cover whole lines over a wave, and a
// block of 32 columns is four neighbouring lanes, whose maximum takes two DPP steps.
#include "block.h"

namespace dsb {

namespace {

template <int T>
DSB_DEV float widen(const void* p, long i) {
  if constexpr (T == DSB_DT_BF16) return (float)((const bf16*)p)[i];
  if constexpr (T == DSB_DT_F16) return (float)((const _Float16*)p)[i];
  return ((const float*)p)[i];
}
// Rounded to the rows' own type, as their sum is.
template <int T>
DSB_DEV float narrow(float v) {
  if constexpr (T == DSB_DT_BF16) return (float)(bf16)v;
  if constexpr (T == DSB_DT_F16) return (float)(_Float16)v;
  return v;
}
template <int T>
struct In8 {
  u32x4 a, b;
  DSB_DEV void load(const void* p, long i) {
    if constexpr (T == DSB_DT_F32) {
      a = ldg128_nt((const float*)p + i);
      b = ldg128_nt((const float*)p + i + 4);
    } else {
      a = ldg128_nt((const bf16*)p + i);
    }
  }
  DSB_DEV void get(float v[8]) const {
    if constexpr (T == DSB_DT_F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned x = a[i], y = b[i];
        v[i] = __builtin_bit_cast(float, x);
        v[4 + i] = __builtin_bit_cast(float, y);
      }
    } else if constexpr (T == DSB_DT_F16) {
      typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
      const f16x8 h = __builtin_bit_cast(f16x8, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
      unpack8(a, v);
    }
  }
};

// The rows that slot i moves; false: none.
DSB_DEV bool slot_rows(const Save8Args& a, int i, long& s, long& d) {
  s = a.src ? a.src[i] : i;
  d = a.dst ? a.dst[i] : i;
  return d >= 0 && d < a.out_rows && s >= 0 && s < a.x_rows;
}

constexpr int kSaveVec = 2, kSaveRun = 256 * 8 * kSaveVec;
template <int T, int CODE, bool RES>
__global__ __launch_bounds__(256) void save_rows8_kernel(Save8Args a) {
  long s, d;
  if (!slot_rows(a, blockIdx.x, s, d)) return;
  const int c0 = blockIdx.y * kSaveRun + threadIdx.x * 8;
  In8<T> x[kSaveVec], r[kSaveVec];
#pragma unroll
  for (int i = 0; i < kSaveVec; ++i) {
    const int c = c0 + 2048 * i;
    if (c < a.width) {
      x[i].load(a.x, s * a.ldx + c);
      if (RES) r[i].load(a.r, s * a.ldr + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kSaveVec; ++i) {
    const int c = c0 + 2048 * i;
    float v[8] = {};
    unsigned top = 0;
    if (c < a.width) {
      x[i].get(v);
      if (RES) {
        float w[8];
        r[i].get(w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = narrow<T>(v[e] + w[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[e]));
    }
    const unsigned byte = scale_byte<CODE>(quad_max(top));
    if (c < a.width) {
      __builtin_nontemporal_store(encode8<CODE>(v, byte),
                                  reinterpret_cast<u32x2*>(a.codes + d * a.ldc + c));
      if ((threadIdx.x & 3) == 0) a.scales[d * a.lds + c / kBlock8] = (uint8_t)byte;
    }
  }
}

// Any width, strides and alignment: 32 lanes to a block, a column each.
template <int T, int CODE>
__global__ __launch_bounds__(256) void save_rows8_any_kernel(Save8Args a) {
  long s, d;
  if (!slot_rows(a, blockIdx.x, s, d)) return;
  const int lane = threadIdx.x & 31;
  const int nb = (a.width + kBlock8 - 1) / kBlock8;
  for (int b = blockIdx.y * 8 + (threadIdx.x >> 5); b < nb; b += gridDim.y * 8) {
    const int c = b * kBlock8 + lane;
    float v = 0.f;
    if (c < a.width) {
      v = widen<T>(a.x, s * a.ldx + c);
      if (a.r) v = narrow<T>(v + widen<T>(a.r, s * a.ldr + c));
    }
    unsigned top = abs_bits(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    const unsigned byte = scale_byte<CODE>(top);
    if (c < a.width) {
      const float four[4] = {v, 0.f, 0.f, 0.f};
      a.codes[d * a.ldc + c] =
          byte == 255u ? 0 : (uint8_t)encode4<CODE>(four, inverse_scale_of(byte));
      if (lane == 0) a.scales[d * a.lds + b] = (uint8_t)byte;
    }
  }
}

constexpr int kRestoreVec = 4, kRestoreRun = 256 * 8 * kRestoreVec;
template <int CODE, bool F32>
__global__ __launch_bounds__(256) void restore_rows8_kernel(RowsArg q, int width, void* out, long ldo) {
  const long row = blockIdx.x;
  const int c0 = blockIdx.y * kRestoreRun + threadIdx.x * 8;
  Raw8<kRows8> x[kRestoreVec];
#pragma unroll
  for (int i = 0; i < kRestoreVec; ++i)
    if (c0 + 2048 * i < width) x[i].load(q, row, (c0 + 2048 * i) / 8);
#pragma unroll
  for (int i = 0; i < kRestoreVec; ++i) {
    const int c = c0 + 2048 * i;
    if (c < width) {
      float v[8];
      decode8<CODE>(x[i].c, x[i].byte, v);
      put8(out, row * ldo + c, F32, v);
    }
  }
}
template <int CODE, bool F32>
__global__ __launch_bounds__(256) void restore_rows8_any_kernel(RowsArg q, int width, void* out,
                                                                long ldo) {
  const long row = blockIdx.x;
  const uint8_t* p = (const uint8_t*)q.p + row * q.ld;
  for (int c = blockIdx.y * 256 + threadIdx.x; c < width; c += gridDim.y * 256) {
    float v[4];
    decode4<CODE>(p[c], scale_of(q.s[row * q.lds + c / kBlock8]), v);
    if (F32)
      ((float*)out)[row * ldo + c] = v[0];
    else
      ((bf16*)out)[row * ldo + c] = (bf16)v[0];
  }
}

// A lane takes 8 gate and 8 up columns of a row. BWD with σ = σ(gate):
//   dgate = dh·up·σ·(1 + gate·(1 − σ)), dup = dh·gate·σ
constexpr int kGluVec = 2, kGluRun = 256 * 8 * kGluVec;
template <int KIND, int DH>
__global__ __launch_bounds__(256) void swiglu_kernel(SwigluArgs a) {
  const long row = blockIdx.x;
  const int c0 = blockIdx.y * kGluRun + threadIdx.x * 8;
  Raw8<KIND> g[kGluVec], u[kGluVec];
  Raw8<DH> dh[kGluVec];
#pragma unroll
  for (int i = 0; i < kGluVec; ++i) {
    const int c = c0 + 2048 * i;
    if (c < a.I) {
      g[i].load(a.gu, row, c / 8);
      u[i].load(a.gu, row, (a.I + c) / 8);
      dh[i].load(a.dh, row, c / 8);
    }
  }
#pragma unroll
  for (int i = 0; i < kGluVec; ++i) {
    const int c = c0 + 2048 * i;
    if (c >= a.I) continue;
    float gv[8], uv[8], dv[8], og[8], ou[8], h[8];
    g[i].get(a.gu, gv);
    u[i].get(a.gu, uv);
    dh[i].get(a.dh, dv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float sg = sigmoid(gv[e]), silu = gv[e] * sg;
      h[e] = silu * uv[e];
      og[e] = dv[e] * uv[e] * (sg * (1.f + gv[e] * (1.f - sg)));
      ou[e] = dv[e] * silu;
    }
    if (DH != kRowsNone) {
      put8(a.dgu, row * a.lddgu + c, false, og);
      put8(a.dgu, row * a.lddgu + a.I + c, false, ou);
    }
    if (a.h) put8(a.h, row * a.ldh + c, false, h);
  }
}

bool aligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) == 0; }
unsigned runs(int width, int run) { return (unsigned)((width + run - 1) / run); }

}  // namespace

hipError_t save_rows8(const Save8Args& a, hipStream_t s) {
  if (a.count <= 0 || a.width <= 0) return hipSuccess;
  const long es = a.dtype == DSB_DT_F32 ? 4 : 2;
  const bool vec = a.width % 8 == 0 && a.ldx * es % 16 == 0 && (!a.r || a.ldr * es % 16 == 0) &&
                   a.ldc % 8 == 0 && aligned(a.x, 16) && aligned(a.r, 16) && aligned(a.codes, 8);
  const bool e4 = a.code == DSB_DT_E4M3;
  auto go = [&](auto kernel, unsigned gy) {
    hipLaunchKernelGGL(kernel, dim3(a.count, gy), dim3(256), 0, s, a);
    return hipGetLastError();
  };
  auto by_type = [&](auto t) {
    constexpr int T = decltype(t)::value;
    if (!vec) {
      const unsigned gy = runs(a.width, 8 * kBlock8 * 4);
      return e4 ? go(save_rows8_any_kernel<T, DSB_DT_E4M3>, gy)
                : go(save_rows8_any_kernel<T, DSB_DT_INT8>, gy);
    }
    const unsigned gy = runs(a.width, kSaveRun);
    if (a.r)
      return e4 ? go(save_rows8_kernel<T, DSB_DT_E4M3, true>, gy)
                : go(save_rows8_kernel<T, DSB_DT_INT8, true>, gy);
    return e4 ? go(save_rows8_kernel<T, DSB_DT_E4M3, false>, gy)
              : go(save_rows8_kernel<T, DSB_DT_INT8, false>, gy);
  };
  switch (a.dtype) {
    case DSB_DT_BF16: return by_type(std::integral_constant<int, DSB_DT_BF16>{});
    case DSB_DT_F16: return by_type(std::integral_constant<int, DSB_DT_F16>{});
    case DSB_DT_F32: return by_type(std::integral_constant<int, DSB_DT_F32>{});
    default: return hipErrorInvalidValue;
  }
}

hipError_t restore_rows8(const RowsArg& q, int rows, int width, void* out, long ldo, bool f32,
                         hipStream_t s) {
  if (rows <= 0 || width <= 0) return hipSuccess;
  const bool vec = width % 8 == 0 && q.ld % 8 == 0 && aligned(q.p, 8) &&
                   ldo * (f32 ? 4 : 2) % 16 == 0 && aligned(out, 16);
  auto go = [&](auto kernel, unsigned gy) {
    hipLaunchKernelGGL(kernel, dim3(rows, gy), dim3(256), 0, s, q, width, out, ldo);
    return hipGetLastError();
  };
  auto by_code = [&](auto c) {
    constexpr int C = decltype(c)::value;
    if (!vec) {
      const unsigned gy = runs(width, 2048);
      return f32 ? go(restore_rows8_any_kernel<C, true>, gy) : go(restore_rows8_any_kernel<C, false>, gy);
    }
    const unsigned gy = runs(width, kRestoreRun);
    return f32 ? go(restore_rows8_kernel<C, true>, gy) : go(restore_rows8_kernel<C, false>, gy);
  };
  return q.type == DSB_DT_E4M3 ? by_code(std::integral_constant<int, DSB_DT_E4M3>{})
                               : by_code(std::integral_constant<int, DSB_DT_INT8>{});
}

hipError_t swiglu(const SwigluArgs& a, hipStream_t s) {
  if (a.rows <= 0 || a.I <= 0) return hipSuccess;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(a.rows, runs(a.I, kGluRun)), dim3(256), 0, s, a);
    return hipGetLastError();
  };
  auto by_kind = [&](auto k) {
    constexpr int K = decltype(k)::value;
    if (!a.dh.p) return go(swiglu_kernel<K, kRowsNone>);
    return a.dh.type == DSB_DT_F32 ? go(swiglu_kernel<K, kRowsF32>) : go(swiglu_kernel<K, kRowsBF16>);
  };
  return a.gu.type == DSB_DT_BF16 ? by_kind(std::integral_constant<int, kRowsBF16>{})
                                  : by_kind(std::integral_constant<int, kRows8>{});
}

}  // namespace dsb
