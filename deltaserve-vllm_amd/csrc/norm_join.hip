// The join of a block with the residual stream and the norms around it, and its backward:
//
//   z = y / rms(y) · w_out (or y),  x' = x + α·gate·z,  normed = x' / rms(x') · w_in
//
// with rms(v) = sqrt(mean(v²) + ε); without a block it is an RMSNorm of rows of any type. The
// backward starts from x' and y, as they were kept (8-bit rows among them). With i = 1 / rms(x'),
// j = 1 / rms(y) (1 without w_out), x̂ = x'·i, ŷ = y·j and the gradients dn of normed and dx' of x':
//
//   t = dx' + i·(dn·w_in − x̂·mean(dn·w_in·x̂))      the stream's gradient, before the join too
//   dy = j·(α·gate·t·w_out − ŷ·mean(α·gate·t·w_out·ŷ))   (α·gate·t without w_out)
//   dw_in = Σ dn·x̂,  dw_out = Σ α·gate·t·ŷ,  dgate = Σ α·t·z over what the gate is broadcast over
//
// The second mean needs t, which needs the first, but it is linear in it: with c = gate·w_out,
//   Σ c·y·t = Σ c·y·dx' + i·(Σ c·y·dn·w_in − mean(dn·w_in·x̂)·i·Σ c·y·x')
// so that one pass over a row takes six sums at once and one barrier a row does. All of it is fp32,
// rounded once where it is stored; the kernels are bound by their bytes.
//
// A block of threads takes row after row, two runs of 8 columns a thread; the weights stay in its
// registers and so do its sums over rows, which a second launch adds up over the blocks, in order.
#include <algorithm>
#include <type_traits>

#include "block.h"

namespace dsb {

namespace {

constexpr int kRuns = 2;                       // of 8 columns a thread
constexpr int kMostThreads = 8192 / 8 / kRuns;  // D <= 8192
constexpr int kMostWaves = kMostThreads / 64;

// The sum over a wave, the same for all: within rows of 16 lanes, then over them.
DSB_DEV float wave_total(float v) {
  auto dpp = [](float x, auto ctrl, auto rows) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
        0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  v += dpp(v, integral_constant<int, 0x128>{}, integral_constant<int, 0xf>{});  // row_ror:8
  v += dpp(v, integral_constant<int, 0x124>{}, integral_constant<int, 0xf>{});
  v += dpp(v, integral_constant<int, 0x122>{}, integral_constant<int, 0xf>{});
  v += dpp(v, integral_constant<int, 0x121>{}, integral_constant<int, 0xf>{});
  v += dpp(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast:15
  v += dpp(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast:31
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// K sums over the block, the same for all. red holds two sets of them, taken in turn: a set is
// written again only after the barrier of the call between, which every wave reaches after it has
// read the set, so one barrier a call is enough.
template <int K>
DSB_DEV void block_totals(float (&v)[K], float (&red)[2][kMostWaves][8], int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_total(v[k]);
  const int waves = blockDim.x >> 6;
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int k = 0; k < K; ++k) red[turn][threadIdx.x >> 6][k] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = 0.f;
  for (int w = 0; w < waves; ++w) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += red[turn][w][k];
  }
  turn ^= 1;
}

// Eight of a bf16 vector's elements, or ones.
DSB_DEV void weights8(u32x4 raw, bool have, float v[8]) {
  unpack8(raw, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = have ? v[e] : 1.f;
}

template <int XK, int YK>
__global__ __launch_bounds__(kMostThreads) void join_fwd_kernel(JoinArgs a) {
  __shared__ float red[2][kMostWaves][8];
  int turn = 0;
  const int nch = a.D >> 3;
  const float rD = 1.f / (float)a.D;
  u32x4 wo[kRuns] = {}, wi[kRuns] = {}, gc[kRuns] = {};
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < nch) {
      if (YK != kRowsNone && a.w_out) wo[i] = ldg128(a.w_out + 8 * c);
      if (a.w_in) wi[i] = ldg128(a.w_in + 8 * c);
      if (YK != kRowsNone && a.gate_kind == kGateChannel) gc[i] = ldg128(a.gate + 8 * c);
    }
  }
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Raw8<XK> x[kRuns];
    Raw8<YK> y[kRuns];
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        x[i].load(a.x, row, c);
        y[i].load(a.y, row, c);
        if (YK != kRowsNone && a.gate_kind == kGateFull) gc[i] = ldg128_nt(a.gate + row * a.ldg + 8 * c);
      }
    }
    const float gr = YK != kRowsNone && a.gate_kind == kGateRow ? (float)a.gate[row * a.ldg] : 1.f;
    const bool each = a.gate_kind == kGateChannel || a.gate_kind == kGateFull;
    float j = 1.f;
    if (YK != kRowsNone && a.w_out) {
      float ss[1] = {0.f};
#pragma unroll
      for (int i = 0; i < kRuns; ++i) {
        if (threadIdx.x + i * blockDim.x < nch) {
          float yv[8];
          y[i].get(a.y, yv);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss[0] += yv[e] * yv[e];
        }
      }
      block_totals(ss, red, turn);
      j = rsqrtf(ss[0] * rD + a.eps);
    }
    float xv[kRuns][8], ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        x[i].get(a.x, xv[i]);
        if (YK != kRowsNone) {
          float yv[8], w[8], g[8];
          y[i].get(a.y, yv);
          weights8(wo[i], a.w_out, w);
          weights8(gc[i], each, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            xv[i][e] += a.scale * (g[e] * gr) * (yv[e] * j * w[e]);
            if (XK == kRowsBF16) xv[i][e] = (float)(bf16)xv[i][e];  // the norm is of the rows as they are kept
          }
          put8(a.x_new, row * a.ldxn + 8 * c, XK == kRowsF32, xv[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[0] += xv[i][e] * xv[i][e];
      }
    }
    if (!a.w_in) continue;  // the same for all
    block_totals(ss, red, turn);
    const float inv = rsqrtf(ss[0] * rD + a.eps);
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        float w[8], o[8];
        unpack8(wi[i], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (xv[i][e] * inv) * w[e];
        put8(a.normed, row * a.ldn + 8 * c, false, o);
      }
    }
  }
}

// SUMS: sums over rows too, by block into part [3][gridDim.x][D] (w_in, w_out, gate).
template <int XK, int YK, int GK, bool SUMS>
__global__ __launch_bounds__(kMostThreads) void join_bwd_kernel(JoinArgs a, float* part) {
  constexpr bool Y = YK != kRowsNone;
  __shared__ float red[2][kMostWaves][8];
  int turn = 0;
  const int nch = a.D >> 3;
  const float rD = 1.f / (float)a.D;
  u32x4 wo[kRuns] = {}, wi[kRuns] = {}, gc[kRuns] = {};
  float s_in[kRuns][8] = {}, s_out[kRuns][8] = {}, s_gate[kRuns][8] = {};
#pragma unroll
  for (int i = 0; i < kRuns; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < nch) {
      if (Y && a.w_out) wo[i] = ldg128(a.w_out + 8 * c);
      if (a.w_in) wi[i] = ldg128(a.w_in + 8 * c);
      if (Y && a.gate_kind == kGateChannel) gc[i] = ldg128(a.gate + 8 * c);
    }
  }
  const bool each = a.gate_kind == kGateChannel || a.gate_kind == kGateFull;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Raw8<XK> x[kRuns];
    Raw8<YK> y[kRuns];
    Raw8<GK> dn[kRuns];
    u32x4 ta[kRuns] = {}, tb[kRuns] = {};  // dx', bf16 or fp32
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        if (GK != kRowsNone) x[i].load(a.x, row, c);
        y[i].load(a.y, row, c);
        dn[i].load(a.dn, row, c);
        if (a.dxn.p) {
          if (a.dxn.type == DSB_DT_F32) {
            const float* p = (const float*)a.dxn.p + row * a.dxn.ld + 8 * c;
            ta[i] = ldg128_nt(p);
            tb[i] = ldg128_nt(p + 4);
          } else {
            ta[i] = ldg128_nt((const bf16*)a.dxn.p + row * a.dxn.ld + 8 * c);
          }
        }
        if (Y && a.gate_kind == kGateFull) gc[i] = ldg128_nt(a.gate + row * a.ldg + 8 * c);
      }
    }
    const float gr = Y && a.gate_kind == kGateRow ? (float)a.gate[row * a.ldg] : 1.f;
    auto carried = [&](int i, float v[8]) {
      if (a.dxn.type == DSB_DT_F32) {  // the same for all
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned p = ta[i][e], q = tb[i][e];
          v[e] = __builtin_bit_cast(float, p);
          v[4 + e] = __builtin_bit_cast(float, q);
        }
      } else {
        unpack8(ta[i], v);
      }
    };
    // Σ x'², Σ dn·w_in·x', Σ y², Σ c·y·dx', Σ c·y·dn·w_in, Σ c·y·x'; c without a row's gate
    float s[Y ? 6 : 2] = {};
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      if (threadIdx.x + i * blockDim.x < nch) {
        float xv[8] = {}, dv[8], w[8];
        if (GK != kRowsNone) x[i].get(a.x, xv);
        dn[i].get(a.dn, dv);
        unpack8(wi[i], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          dv[e] *= w[e];
          s[0] += xv[e] * xv[e];
          s[1] += dv[e] * xv[e];
        }
        if constexpr (Y) {
          float yv[8], tv[8], wv[8], gv[8];
          y[i].get(a.y, yv);
          carried(i, tv);
          weights8(wo[i], a.w_out, wv);
          weights8(gc[i], each, gv);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float cy = gv[e] * wv[e] * yv[e];
            s[2] += yv[e] * yv[e];
            s[3] += cy * tv[e];
            s[4] += cy * dv[e];
            s[5] += cy * xv[e];
          }
        }
      }
    }
    block_totals(s, red, turn);
    const float inv = rsqrtf(s[0] * rD + a.eps);
    const float k = s[1] * inv * rD;  // mean(dn·w_in·x̂)
    float j = 1.f, m = 0.f;           // 1 / rms(y), mean(α·gate·t·w_out·ŷ)
    if constexpr (Y) {
      float p = s[3];
      if (GK != kRowsNone) p += inv * (s[4] - k * (inv * s[5]));
      if (a.w_out) {
        j = rsqrtf(s[2] * rD + a.eps);
        m = a.scale * gr * p * j * rD;
      }
      if (a.dgate_row && threadIdx.x == 0) a.dgate_row[row] = a.scale * p * j;
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        float t[8];
        carried(i, t);
        if (GK != kRowsNone) {
          float xv[8], dv[8], w[8];
          x[i].get(a.x, xv);
          dn[i].get(a.dn, dv);
          unpack8(wi[i], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float hat = xv[e] * inv;
            t[e] += (dv[e] * w[e] - hat * k) * inv;
            if (SUMS) s_in[i][e] += dv[e] * hat;
          }
        }
        put8(a.dx, row * a.lddx + 8 * c, a.dx_f32, t);
        if constexpr (Y) {
          float yv[8], wv[8], gv[8], o[8], q[8];
          y[i].get(a.y, yv);
          weights8(wo[i], a.w_out, wv);
          weights8(gc[i], each, gv);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float hat = yv[e] * j, at = a.scale * t[e], dz = gv[e] * gr * at;
            o[e] = a.w_out ? (dz * wv[e] - hat * m) * j : dz;
            q[e] = at * hat * wv[e];
            if (SUMS) {
              s_out[i][e] += dz * hat;
              s_gate[i][e] += q[e];
            }
          }
          put8(a.dy, row * a.lddy + 8 * c, false, o);
          if (a.dgate_full) put8(a.dgate_full, row * a.lddg + 8 * c, false, q);
        }
      }
    }
  }
  if (SUMS) {
    const long plane = (long)gridDim.x * a.D;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        float* p = part + (long)blockIdx.x * a.D + 8 * c;
        auto put = [&](float* o, const float* v) {
          *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
        };
        if (a.dw_in) put(p, s_in[i]);
        if (a.dw_out) put(p + plane, s_out[i]);
        if (a.dgate) put(p + 2 * plane, s_gate[i]);
      }
    }
  }
}

// out[k][c] = Σ_b part[k][b][c]: 32 columns a block, 32 threads to each group of 4 of them.
__global__ __launch_bounds__(256) void join_sums_kernel(const float* __restrict__ part, int blocks,
                                                        int D, float* o0, float* o1, float* o2) {
  float* out = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (!out) return;
  __shared__ f32x4 red[256];
  const int c = blockIdx.x * 32 + (threadIdx.x & 7) * 4, g = threadIdx.x >> 3;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (c < D) {
    const float* p = part + (long)blockIdx.y * blocks * D + c;
#pragma unroll 8
    for (int b = g; b < blocks; b += 32) s += *reinterpret_cast<const f32x4*>(p + (long)b * D);
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 8 && c < D) {
    for (int i = 1; i < 32; ++i) s += red[threadIdx.x + 8 * i];
    *reinterpret_cast<f32x4*>(out + c) = s;
  }
}

int threads_of(int D) { return std::max(64, (D / 8 + kRuns * 64 - 1) / (kRuns * 64) * 64); }
constexpr int kFwdBlocks = 2048, kBwdBlocks = 512;

}  // namespace

hipError_t join_fwd(const JoinArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(std::min(a.rows, kFwdBlocks)), dim3(threads_of(a.D)), 0, s, a);
    return hipGetLastError();
  };
  auto by_x = [&](auto k) {
    constexpr int K = decltype(k)::value;
    return a.y.p ? go(join_fwd_kernel<K, kRowsBF16>) : go(join_fwd_kernel<K, kRowsNone>);
  };
  switch (rows_kind(a.x.type)) {
    case kRowsBF16: return by_x(std::integral_constant<int, kRowsBF16>{});
    case kRowsF32: return by_x(std::integral_constant<int, kRowsF32>{});
    default: return a.y.p ? hipErrorInvalidValue : go(join_fwd_kernel<kRows8, kRowsNone>);
  }
}

int64_t join_bwd_bytes(int rows, int D, int sums) {
  return sums ? 12ll * std::min(rows, kBwdBlocks) * D : 0;
}

hipError_t join_bwd(const JoinArgs& a, void* work, hipStream_t s) {
  const bool sums = a.dw_in || a.dw_out || a.dgate;
  const int blocks = sums ? std::min(a.rows, kBwdBlocks) : std::min(a.rows, kFwdBlocks);
  float* part = (float*)work;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(threads_of(a.D)), 0, s, a, part);
    return hipGetLastError();
  };
  auto by_sums = [&](auto x, auto y, auto g) {
    constexpr int X = decltype(x)::value, Y = decltype(y)::value, G = decltype(g)::value;
    return sums ? go(join_bwd_kernel<X, Y, G, true>) : go(join_bwd_kernel<X, Y, G, false>);
  };
  auto by_g = [&](auto x, auto y) {
    if (!a.dn.p) return by_sums(x, y, std::integral_constant<int, kRowsNone>{});
    return a.dn.type == DSB_DT_F32 ? by_sums(x, y, std::integral_constant<int, kRowsF32>{})
                                   : by_sums(x, y, std::integral_constant<int, kRowsBF16>{});
  };
  auto by_y = [&](auto x) {
    if (!a.y.p) return by_g(x, std::integral_constant<int, kRowsNone>{});
    return a.y.type == DSB_DT_BF16 ? by_g(x, std::integral_constant<int, kRowsBF16>{})
                                   : by_g(x, std::integral_constant<int, kRows8>{});
  };
  if (a.rows > 0) {
    hipError_t e;
    switch (rows_kind(a.x.type)) {
      case kRowsBF16: e = by_y(std::integral_constant<int, kRowsBF16>{}); break;
      case kRowsF32: e = by_y(std::integral_constant<int, kRowsF32>{}); break;
      default: e = by_y(std::integral_constant<int, kRows8>{});
    }
    if (e != hipSuccess) return e;
  }
  if (sums)
    hipLaunchKernelGGL(join_sums_kernel, dim3((a.D + 31) / 32, 3), dim3(256), 0, s, part,
                       std::max(blocks, 0), a.D, a.dw_in, a.dw_out, a.dgate);
  return hipGetLastError();
}

}  // namespace dsb
