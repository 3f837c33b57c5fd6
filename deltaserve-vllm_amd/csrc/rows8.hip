// Rows in and out of 8 bits (rows8.h says what they are) and SwiGLU with its backward from rows of
// either kind. All of it is bound by its bytes.
//
// A lane holds 8 columns: its loads of 16 bytes (8 of codes) cover whole lines over a wave, and a
// block of 32 columns is four neighbouring lanes, whose maximum takes two DPP steps. Rows may start
// anywhere; the last columns of a width that is no multiple of 8 are moved one by one. A workgroup takes
// several narrow rows, or a part of a wide one (Span).
//
// 8192 × 28672 bf16 rows in: 124 µs, 5.7 TB/s; restored 132 µs, 5.4 TB/s (a copy: 4.8); 8192 × 1024 in 5.7 µs,
// 8192 × 28671 147. SwiGLU of 8192 × 14336 8-bit rows 85 µs, its backward with the forward's rows 220 µs, 5.4 TB/s.
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
  template <int P>
  DSB_DEV void load(const void* p, long i) {
    if constexpr (T == DSB_DT_F32) {
      a = load_as<P, u32x4h>((const float*)p + i);
      b = load_as<P, u32x4h>((const float*)p + i + 4);
    } else {
      a = load_as<P, u32x4h>((const bf16*)p + i);
    }
  }
  DSB_DEV void get(float v[8]) const {
    if constexpr (T == DSB_DT_F32) {
      floats8(a, b, v);
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
template <int T>
DSB_DEV void few(const void* p, long i, int count, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < count ? widen<T>(p, i + e) : 0.f;
}

// How 256 threads lie over rows: 2^lanes_log (4 to 256) of them to a row, V runs of 8 columns each.
struct Span {
  int rows, lanes_log;
};
template <int V>
struct Spot {
  long row;
  int column, step;  // of the thread's first run, and between its runs
  DSB_DEV Spot(Span p) {
    row = (long)blockIdx.x * (256 >> p.lanes_log) + (threadIdx.x >> p.lanes_log);
    step = 8 << p.lanes_log;
    column = blockIdx.y * V * step + (threadIdx.x & ((1 << p.lanes_log) - 1)) * 8;
  }
};
// A row's lanes take `runs` of its V before it gets more of them: 2 in the copies, 1 in SwiGLU (µs with 1 / 2:
// saves of 8192 × 1024 6.9 / 5.9; SwiGLU's backward of 8192 × 1000 14.1 / 17.5).
template <int V>
Span span_of(int rows, int width, int runs, dim3& grid) {
  Span p{rows, 2};
  while (p.lanes_log < 8 && (8l * runs << p.lanes_log) < width) ++p.lanes_log;
  const int each = 256 >> p.lanes_log;
  const long run = 8l * V << p.lanes_log;
  grid = dim3((unsigned)((rows + each - 1) / each), (unsigned)((width + run - 1) / run));
  return p;
}

// The rows that slot i moves; false: none.
DSB_DEV bool slot_rows(const Save8Args& a, int i, long& s, long& d) {
  s = a.src ? a.src[i] : i;
  d = a.dst ? a.dst[i] : i;
  return d >= 0 && d < a.out_rows && s >= 0 && s < a.x_rows;
}

constexpr int kSaveVec = 2;
template <int T, int CODE, bool RES, int P>
__global__ __launch_bounds__(256) void save_rows8_kernel(Save8Args a, Span span) {
  const Spot<kSaveVec> at(span);
  long s, d;
  if (at.row >= span.rows || !slot_rows(a, (int)at.row, s, d)) return;  // (a block's lanes are of one row)
  In8<T> x[kSaveVec], r[kSaveVec];
#pragma unroll
  for (int i = 0; i < kSaveVec; ++i) {
    const int c = at.column + at.step * i;
    if (c + 8 <= a.width) {
      x[i].template load<P>(a.x, s * a.ldx + c);
      if (RES) r[i].template load<P>(a.r, s * a.ldr + c);
    }
  }
#pragma unroll
  for (int i = 0; i < kSaveVec; ++i) {
    const int c = at.column + at.step * i, left = a.width - c;
    float v[8] = {}, w[8];
    unsigned top = 0;
    if (left > 0) {
      if (left >= 8) {
        x[i].get(v);
        if (RES) r[i].get(w);
      } else {
        few<T>(a.x, s * a.ldx + c, left, v);
        if (RES) few<T>(a.r, s * a.ldr + c, left, w);
      }
      if (RES) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = narrow<T>(v[e] + w[e]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, abs_bits(v[e]));
    }
    const unsigned byte = scale_byte<CODE>(quad_max(top));
    if (left > 0) {
      const u32x2 code = encode8<CODE>(v, byte);
      uint8_t* o = a.codes + d * a.ldc + c;
      if (left >= 8) {
        store_as<P, u32x2b>(o, code);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < left) o[e] = (uint8_t)(code[e >> 2] >> (8 * (e & 3)));
      }
      if ((threadIdx.x & 3) == 0) a.scales[d * a.lds + c / kBlock8] = (uint8_t)byte;
    }
  }
}

constexpr int kRestoreVec = 4;
template <int CODE, bool F32, int P>
__global__ __launch_bounds__(256) void restore_rows8_kernel(RowsArg q, int width, void* out, long ldo,
                                                            Span span, const int* rows_dev) {
  const Spot<kRestoreVec> at(span);
  const long row = at.row;
  if (row >= (rows_dev ? min(span.rows, *rows_dev) : span.rows)) return;
  const uint8_t* in = (const uint8_t*)q.p + row * q.ld;
  u32x2 x[kRestoreVec];
  unsigned byte[kRestoreVec];
#pragma unroll
  for (int i = 0; i < kRestoreVec; ++i) {
    const int c = at.column + at.step * i;
    if (c + 8 <= width) x[i] = load_as<P, u32x2b>(in + c);
    if (c < width) byte[i] = q.s[row * q.lds + c / kBlock8];
  }
#pragma unroll
  for (int i = 0; i < kRestoreVec; ++i) {
    const int c = at.column + at.step * i, left = width - c;
    float v[8];
    if (left >= 8) {
      decode8<CODE>(x[i], byte[i], v);
      if (F32) {
        store_as<P, u32x4h>((float*)out + row * ldo + c, __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]}));
        store_as<P, u32x4h>((float*)out + row * ldo + c + 4, __builtin_bit_cast(u32x4, f32x4{v[4], v[5], v[6], v[7]}));
      } else {
        store_as<P, u32x4h>((bf16*)out + row * ldo + c, pack8(v));
      }
    } else if (left > 0) {
      u32x2 few = {0u, 0u};
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left) few[e >> 2] |= (unsigned)in[c + e] << (8 * (e & 3));
      decode8<CODE>(few, byte[i], v);
#pragma unroll
      for (int e = 0; e < 7; ++e) {
        if (e < left && F32) ((float*)out)[row * ldo + c + e] = v[e];
        if (e < left && !F32) ((bf16*)out)[row * ldo + c + e] = (bf16)v[e];
      }
    }
  }
}

// A lane takes 8 gate and 8 up columns of a row. With dh and σ = 1 / (1 + exp(−gate)):
//   dgate = dh·up·σ·(1 + gate·(1 − σ)), dup = dh·gate·σ
constexpr int kGluVec = 2;
template <int T, int DH, int P>
__global__ __launch_bounds__(256) void swiglu_kernel(SwigluArgs a, Span span) {
  const Spot<kGluVec> at(span);
  const long row = at.row;
  if (row >= span.rows) return;
  Raw8<T> g[kGluVec], u[kGluVec];
  Raw8<DH> dh[kGluVec];
#pragma unroll
  for (int i = 0; i < kGluVec; ++i) {
    const int c = at.column + at.step * i;
    if (c < a.I) {
      g[i].template load<P>(a.gu, row, c / 8);
      u[i].template load<P>(a.gu, row, (a.I + c) / 8);
      dh[i].template load<P>(a.dh, row, c / 8);
    }
  }
#pragma unroll
  for (int i = 0; i < kGluVec; ++i) {
    const int c = at.column + at.step * i;
    if (c >= a.I) continue;
    float gv[8], uv[8], dv[8], og[8], ou[8], h[8];
    g[i].get(gv);
    u[i].get(uv);
    dh[i].get(dv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float sg = sigmoid(gv[e]), silu = gv[e] * sg;
      h[e] = silu * uv[e];
      og[e] = dv[e] * uv[e] * (sg * (1.f + gv[e] * (1.f - sg)));
      ou[e] = dv[e] * silu;
    }
    if (DH != kRowsNone) {
      put8<P>(a.dgu, row * a.lddgu + c, false, og);
      put8<P>(a.dgu, row * a.lddgu + a.I + c, false, ou);
    }
    if (a.h) put8<P>(a.h, row * a.ldh + c, false, h);
  }
}

template <class F>
hipError_t by_cache(double in, double out, F f) {
  switch (cache_of(in, out)) {
    case kNear: return f(Int<kNear>{});
    case kFar: return f(Int<kFar>{});
    default: return f(Int<kPast>{});
  }
}

}  // namespace

hipError_t save_rows8(const Save8Args& a, hipStream_t s) {
  if (a.count <= 0 || a.width <= 0) return hipSuccess;
  const double n = (double)a.count * a.width, es = a.dtype == DSB_DT_F32 ? 4 : 2;
  const double in = (a.r ? 2 : 1) * es * n;
  // (where a call ends up past both goes by what it reads, at least twice what it writes: kFar / kPast 39 / 41 µs
  // at 149 MB, 2600 × 28672, 60 / 54 at 201 MB, 3500)
  return by_cache(in, in, [&](auto p) {
    constexpr int P = decltype(p)::value;
    auto go = [&](auto kernel) {
      dim3 grid;
      const Span span = span_of<kSaveVec>(a.count, a.width, 2, grid);
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, span);
      return hipGetLastError();
    };
    auto by_code = [&](auto t, auto c) {
      constexpr int T = decltype(t)::value, C = decltype(c)::value;
      return a.r ? go(save_rows8_kernel<T, C, true, P>) : go(save_rows8_kernel<T, C, false, P>);
    };
    auto by_type = [&](auto t) {
      return a.code == DSB_DT_E4M3 ? by_code(t, Int<DSB_DT_E4M3>{}) : by_code(t, Int<DSB_DT_INT8>{});
    };
    switch (a.dtype) {
      case DSB_DT_BF16: return by_type(Int<DSB_DT_BF16>{});
      case DSB_DT_F16: return by_type(Int<DSB_DT_F16>{});
      default: return by_type(Int<DSB_DT_F32>{});
    }
  });
}

hipError_t restore_rows8(const RowsArg& q, int rows, int width, void* out, long ldo, bool f32,
                         hipStream_t s, const int* rows_dev) {
  if (rows <= 0 || width <= 0) return hipSuccess;
  auto run = [&](auto p) {
    constexpr int P = decltype(p)::value;
    auto go = [&](auto kernel) {
      dim3 grid;
      const Span span = span_of<kRestoreVec>(rows, width, 2, grid);
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, q, width, out, ldo, span, rows_dev);
      return hipGetLastError();
    };
    auto by_code = [&](auto c) {
      constexpr int C = decltype(c)::value;
      return f32 ? go(restore_rows8_kernel<C, true, P>) : go(restore_rows8_kernel<C, false, P>);
    };
    return q.type == DSB_DT_E4M3 ? by_code(Int<DSB_DT_E4M3>{}) : by_code(Int<DSB_DT_INT8>{});
  };
  // (results of larger inputs, twice or four times their bytes, fit no cache)
  return cache_of((double)rows * width, 0) == kNear ? run(Int<kNear>{}) : run(Int<kPast>{});
}

hipError_t swiglu(const SwigluArgs& a, hipStream_t s) {
  if (a.rows <= 0 || a.I <= 0) return hipSuccess;
  const double n = (double)a.rows * a.I;
  return by_cache(n * (2 * row_bytes(a.gu) + row_bytes(a.dh)), n * ((a.dh.p ? 4 : 0) + (a.h ? 2 : 0)),
                  [&](auto p) {
    constexpr int P = decltype(p)::value;
    auto go = [&](auto kernel) {
      dim3 grid;
      const Span span = span_of<kGluVec>(a.rows, a.I, 1, grid);
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a, span);
      return hipGetLastError();
    };
    auto by_dh = [&](auto t) {
      constexpr int T = decltype(t)::value;
      if (!a.dh.p) return go(swiglu_kernel<T, kRowsNone, P>);
      return a.dh.type == DSB_DT_F32 ? go(swiglu_kernel<T, DSB_DT_F32, P>)
                                     : go(swiglu_kernel<T, DSB_DT_BF16, P>);
    };
    switch (a.gu.type) {
      case DSB_DT_BF16: return by_dh(Int<DSB_DT_BF16>{});
      case DSB_DT_E4M3: return by_dh(Int<DSB_DT_E4M3>{});
      default: return by_dh(Int<DSB_DT_INT8>{});
    }
  });
}

}  // namespace dsb
