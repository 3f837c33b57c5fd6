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
// A block of threads takes row after row, a lane 8 columns (16 or 24 in the forward, which needs few
// registers); the weights stay in its registers and so do its two sums over rows, which a second
// launch adds up over the blocks, in order. In the backward 16 waves a CU cover each other's loads and barriers:
// two rows' loads ahead of one another in fewer waves (16 columns a lane) took 117 to 124 µs
// for 8192 × 4096 8-bit rows with everything on, without them 95, this 91 (95 where results live on, and 6 the
// sums' launch; the bytes take 98 at a copy's rate). Kernel times at that size: forward 47 µs, 5.7 TB/s (fp32
// 70); a norm alone of 8-bit rows 21 µs, its backward with an fp32 gradient 51 µs, 5.9 TB/s.
#include <algorithm>
#include <type_traits>

#include "block.h"

namespace dsb {

namespace {

constexpr int kMostThreads = 1024;  // 8 columns each: D <= 8192
constexpr int kMostWaves = kMostThreads / 64;

template <int CTRL, int ROWS>
DSB_DEV float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(
                 0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
// The sum over each 16 lanes, in all of them.
DSB_DEV float row_total(float v) {
  v = dpp_add<0x128, 0xf>(v);  // row_ror:8, 4, 2, 1
  v = dpp_add<0x124, 0xf>(v);
  v = dpp_add<0x122, 0xf>(v);
  return dpp_add<0x121, 0xf>(v);
}

// K sums over the block, the same for all. red holds two sets of them, taken in turn: a set is
// written again only after the barrier of the call between, which every wave reaches after it has
// read the set, so one barrier a call is enough. (It orders LDS alone: a fence would wait for the row
// before's stores too.)
template <int K>
DSB_DEV void block_totals(float (&v)[K], float (&red)[2][kMostWaves][8], int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = row_total(v[k]);
    v[k] = dpp_add<0x142, 0xa>(v[k]);  // row_bcast:15 into rows 1 and 3
    v[k] = dpp_add<0x143, 0xc>(v[k]);  // row_bcast:31 into rows 2 and 3: lane 63 has all
  }
  const int waves = blockDim.x >> 6, lane = threadIdx.x & 63;
  if (waves == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      v[k] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v[k]), 63));
    return;
  }
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < K; ++k) red[turn][threadIdx.x >> 6][k] = v[k];
  }
  wait_lgkm0();
  lds_barrier();
  const int w = lane & 15;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = w < waves ? red[turn][w][k] : 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = row_total(v[k]);
  turn ^= 1;
}

// Eight of a bf16 vector's elements, or ones.
DSB_DEV void weights8(u32x4 raw, bool have, float v[8]) {
  unpack8(raw, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = have ? v[e] : 1.f;
}

// R runs of 8 columns a thread; XK, YK: the types of x and y.
template <int XK, int YK, int P, int R>
__global__ __launch_bounds__(kMostThreads / 2) void join_fwd_kernel(JoinArgs a) {
  __shared__ float red[2][kMostWaves][8];
  int turn = 0;
  const int nch = a.D >> 3;
  const float rD = 1.f / (float)a.D;
  u32x4 wo[R] = {}, wi[R] = {}, gc[R] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < nch) {
      if (YK != kRowsNone && a.w_out) wo[i] = ldg128(a.w_out + 8 * c);
      if (a.w_in) wi[i] = ldg128(a.w_in + 8 * c);
      if (YK != kRowsNone && a.gate_kind == kGateChannel) gc[i] = ldg128(a.gate + 8 * c);
    }
  }
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Raw8<XK> x[R];
    Raw8<YK> y[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        x[i].template load<P>(a.x, row, c);
        y[i].template load<P>(a.y, row, c);
        if (YK != kRowsNone && a.gate_kind == kGateFull)
          gc[i] = load_as<P, u32x4>(a.gate + row * a.ldg + 8 * c);
      }
    }
    const float gr = YK != kRowsNone && a.gate_kind == kGateRow ? (float)a.gate[row * a.ldg] : 1.f;
    const bool each = a.gate_kind == kGateChannel || a.gate_kind == kGateFull;
    float j = 1.f;
    if (YK != kRowsNone && a.w_out) {
      float ss[1] = {0.f};
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (threadIdx.x + i * blockDim.x < nch) {
          float yv[8];
          y[i].get(yv);
#pragma unroll
          for (int e = 0; e < 8; ++e) ss[0] += yv[e] * yv[e];
        }
      }
      block_totals(ss, red, turn);
      j = rsqrtf(ss[0] * rD + a.eps);
    }
    float xv[R][8], ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        x[i].get(xv[i]);
        if (YK != kRowsNone) {
          float yv[8], w[8], g[8];
          y[i].get(yv);
          weights8(wo[i], a.w_out, w);
          weights8(gc[i], each, g);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            xv[i][e] += a.scale * (g[e] * gr) * (yv[e] * j * w[e]);
            if (XK == DSB_DT_BF16) xv[i][e] = (float)(bf16)xv[i][e];  // the norm is of the rows as they are kept
          }
          put8<P>(a.x_new, row * a.ldxn + 8 * c, XK == DSB_DT_F32, xv[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[0] += xv[i][e] * xv[i][e];
      }
    }
    if (!a.w_in) continue;  // the same for all
    block_totals(ss, red, turn);
    const float inv = rsqrtf(ss[0] * rD + a.eps);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      if (c < nch) {
        float w[8], o[8];
        unpack8(wi[i], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (xv[i][e] * inv) * w[e];
        put8<P>(a.normed, row * a.ldn + 8 * c, false, o);
      }
    }
  }
}

// 8 columns a thread; XT, YT, GT: the types of x', y and dn, FULL: a gate of rows; through: dx is fp32 and
// goes into the caches. With a block its
// sums over rows go into part [2][gridDim.x][D]: Σ dn·x̂, and Σ t·ŷ times a gate that differs by row, of
// which dw_out and a channel gate's dgate are multiples (join_sums_kernel).
template <int XT, int YT, int GT, bool FULL, int P>
__global__ __launch_bounds__(kMostThreads) void join_bwd_kernel(JoinArgs a, float* part, bool through) {
  constexpr bool Y = YT != kRowsNone, N = GT != kRowsNone;
  __shared__ float red[2][kMostWaves][8];
  int turn = 0;
  // threads past the row take its last columns too, and leave them out of sums and results
  const int c = min((int)threadIdx.x, (a.D >> 3) - 1);
  const bool live = threadIdx.x == c;
  const float rD = 1.f / (float)a.D;
  float cw[8];  // w_out·a gate by channel
  u32x4 wi = {};
  if (N) wi = ldg128(a.w_in + 8 * c);
  if constexpr (Y) {
    float g[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) cw[e] = g[e] = 1.f;
    if (a.w_out) unpack8(ldg128(a.w_out + 8 * c), cw);
    if (a.gate_kind == kGateChannel) unpack8(ldg128(a.gate + 8 * c), g);
#pragma unroll
    for (int e = 0; e < 8; ++e) cw[e] *= g[e];
  }
  float s_in[8] = {}, s_out[8] = {};
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    Raw8<XT> x;
    Raw8<YT> y;
    Raw8<GT> dn;
    u32x4 ta = {}, tb = {}, gf;  // dx' (bf16 or fp32), a gate of rows
    if (N) x.template load<P>(a.x, row, c);
    y.template load<P>(a.y, row, c);
    dn.template load<P>(a.dn, row, c);
    if (a.dxn.p) {
      if (a.dxn.type == DSB_DT_F32) {
        const float* p = (const float*)a.dxn.p + row * a.dxn.ld + 8 * c;
        ta = load_as<P, u32x4>(p);
        tb = load_as<P, u32x4>(p + 4);
      } else {
        ta = load_as<P, u32x4>((const bf16*)a.dxn.p + row * a.dxn.ld + 8 * c);
      }
    }
    if (FULL) gf = load_as<P, u32x4>(a.gate + row * a.ldg + 8 * c);
    const float gr = Y && a.gate_kind == kGateRow ? (float)a.gate[row * a.ldg] : 1.f;
    float xv[8], dv[8], yv[8], t[8], w[8], g[8];
    if (N) {
      x.get(xv);
      dn.get(dv);
      unpack8(wi, w);
    }
    if (Y) y.get(yv);
    if (FULL) unpack8(gf, g);
    if (a.dxn.type == DSB_DT_F32)
      floats8(ta, tb, t);
    else
      unpack8(ta, t);
    // Σ x'², Σ dn·w_in·x', Σ y², Σ c·y·dx', Σ c·y·dn·w_in, Σ c·y·x'; c without a row's gate
    float s[Y ? 6 : 2] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (N) {
        s[0] += xv[e] * xv[e];
        s[1] += dv[e] * w[e] * xv[e];
      }
      if constexpr (Y) {
        const float cy = (FULL ? cw[e] * g[e] : cw[e]) * yv[e];
        s[2] += yv[e] * yv[e];
        s[3] += cy * t[e];
        if (N) {
          s[4] += cy * (dv[e] * w[e]);
          s[5] += cy * xv[e];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < (Y ? 6 : 2); ++i) s[i] = live ? s[i] : 0.f;
    block_totals(s, red, turn);
    const float inv = rsqrtf(s[0] * rD + a.eps);
    const float k = s[1] * inv * rD;  // mean(dn·w_in·x̂)
    float j = 1.f, m = 0.f;           // 1 / rms(y), mean(α·gate·t·w_out·ŷ)
    if constexpr (Y) {
      float p = s[3];
      if (N) p += inv * (s[4] - k * (inv * s[5]));
      if (a.w_out) {
        j = rsqrtf(s[2] * rD + a.eps);
        m = a.scale * gr * p * j * rD;
      }
      if (a.dgate_row && threadIdx.x == 0) a.dgate_row[row] = a.scale * p * j;
    }
    if (N) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float hat = xv[e] * inv;
        t[e] += (dv[e] * w[e] - hat * k) * inv;
        if (Y) s_in[e] += dv[e] * hat;
      }
    }
    if (live) {
      if (through)
        put8<kIn>(a.dx, row * a.lddx + 8 * c, true, t);
      else
        put8<P>(a.dx, row * a.lddx + 8 * c, a.dx_f32, t);
    }
    if constexpr (Y) {
      const float to_y = a.scale * gr * j, back = m * j;
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        yv[e] *= j;
        o[e] = (FULL ? cw[e] * g[e] : cw[e]) * t[e] * to_y;
      }
      if (a.w_out) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] -= yv[e] * back;
      }
      if (live) put8<P>(a.dy, row * a.lddy + 8 * c, false, o);
      if (FULL) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          o[e] = a.scale * (t[e] * yv[e]) * cw[e];
          yv[e] *= g[e];
        }
        if (live) put8<P>(a.dgate_full, row * a.lddg + 8 * c, false, o);
      } else if (a.gate_kind == kGateRow) {
#pragma unroll
        for (int e = 0; e < 8; ++e) yv[e] *= gr;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s_out[e] += t[e] * yv[e];
    }
  }
  if constexpr (Y) {
    if (!part || !live) return;
    auto put = [&](float* o, const float* v) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(o + 4) = f32x4{v[4], v[5], v[6], v[7]};
    };
    float* p = part + (long)blockIdx.x * a.D + 8 * c;
    if (a.dw_in) put(p, s_in);
    if (a.dw_out || a.dgate) put(p + (long)gridDim.x * a.D, s_out);
  }
}

// The sums over the blocks, kSumLanes threads to a row of 4 columns each and as many rows at once as a
// workgroup has threads for: dw_in from plane 0; dw_out (times α·a channel gate) and dgate (times
// α·w_out) from plane 1.
constexpr int kSumLanes = 8, kSumThreads = 512;
__global__ __launch_bounds__(kSumThreads) void join_sums_kernel(JoinArgs a, const float* __restrict__ part,
                                                                int blocks) {
  const bool first = blockIdx.y == 0;
  if (first ? !a.dw_in : !a.dw_out && !a.dgate) return;
  __shared__ f32x4 red[kSumThreads];
  const int t = threadIdx.x, c = (blockIdx.x * kSumLanes + t % kSumLanes) * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
  if (c < a.D) {
    const float* p = part + (long)blockIdx.y * blocks * a.D + c;
#pragma unroll 8
    for (int b = t / kSumLanes; b < blocks; b += kSumThreads / kSumLanes)
      s += *reinterpret_cast<const f32x4*>(p + (long)b * a.D);
  }
  red[t] = s;
  __syncthreads();
  if (t < 64) {
    for (int i = 64; i < kSumThreads; i += 64) s += red[t + i];
    red[t] = s;
  }
  __syncthreads();
  if (t >= kSumLanes || c >= a.D) return;
  for (int i = kSumLanes; i < 64; i += kSumLanes) s += red[t + i];
  if (first) {
    *reinterpret_cast<f32x4*>(a.dw_in + c) = s;
    return;
  }
  s *= a.scale;
  auto times = [&](const bf16* v) {
    f32x4 r = s;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] *= v ? (float)v[c + e] : 1.f;
    return r;
  };
  if (a.dw_out) *reinterpret_cast<f32x4*>(a.dw_out + c) = times(a.gate_kind == kGateChannel ? a.gate : nullptr);
  if (a.dgate) *reinterpret_cast<f32x4*>(a.dgate + c) = times(a.w_out);
}

int waves_of(int D, int runs) { return (D / 8 + 64 * runs - 1) / (64 * runs); }
constexpr int kCUs = 256;
// Blocks of a kernel that keeps no sums: of the chip's threads.
int blocks_of(int rows, int waves) { return std::min(rows, (1 << 13) / waves); }
// The forward's runs a thread: two, or three where more of its blocks fit 8 waves that way (8191 × 5120, 5
// waves or 4: 76 or 62 µs; 8192 wide, 8 or 6: 88 or 128; one run each 74 and 101).
int fwd_runs(int D) { return 8 / waves_of(D, 3) > 8 / waves_of(D, 2) ? 3 : 2; }
// With sums, 8 waves a CU, which leave the fewest sums to write out, or two blocks where 16 waves, all
// that fit its registers, hold them: a lone block waits at its barriers. 8192 × 4096, one / two blocks of 8
// waves a CU: 104 / 92 µs; 32768 × 1024, four / eight of two waves, the sums' launch too: 95 / 103.
int sum_blocks(int rows, int D) {
  const int w = waves_of(D, 1);
  const int most = kCUs * std::max(1, std::max(8 / w, std::min(2, 16 / w)));
  // a CU has a block before a block has a second row, whose sums cost nothing more to write out
  return rows <= kCUs ? rows : std::min(std::max(kCUs, (rows + 1) / 2), most);
}

}  // namespace

hipError_t join_fwd(const JoinArgs& a, hipStream_t s) {
  if (a.rows <= 0) return hipSuccess;
  const double in = row_bytes(a.x) + row_bytes(a.y) + (a.gate_kind == kGateFull ? 2 : 0);
  // (kFar is as kPast: 8191 × 4096 bf16 rows, kNear / kFar / kPast 50 / 47 / 47 µs)
  const bool near = cache_of(in * a.rows * a.D, 0) == kNear;
  const int runs = fwd_runs(a.D), waves = waves_of(a.D, runs);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks_of(a.rows, waves)), dim3(64 * waves), 0, s, a);
    return hipGetLastError();
  };
  auto by_cache = [&](auto x, auto y) {
    constexpr int X = decltype(x)::value, Y = decltype(y)::value;
    if (runs == 2) return near ? go(join_fwd_kernel<X, Y, kNear, 2>) : go(join_fwd_kernel<X, Y, kPast, 2>);
    return near ? go(join_fwd_kernel<X, Y, kNear, 3>) : go(join_fwd_kernel<X, Y, kPast, 3>);
  };
  return by_type(a.x, [&](auto x) {
    constexpr int X = decltype(x)::value;
    if constexpr (X == DSB_DT_BF16 || X == DSB_DT_F32)
      if (a.y.p) return by_cache(x, Int<DSB_DT_BF16>{});
    return by_cache(x, Int<kRowsNone>{});
  });
}

int64_t join_bwd_bytes(int rows, int D, int sums) {
  return sums ? 8ll * sum_blocks(rows, D) * D : 0;
}

hipError_t join_bwd(const JoinArgs& a, void* work, hipStream_t s) {
  const bool sums = a.dw_in || a.dw_out || a.dgate, full = a.gate_kind == kGateFull;
  const int waves = waves_of(a.D, 1);
  const int blocks = a.y.p ? sum_blocks(a.rows, a.D) : blocks_of(a.rows, waves);
  float* part = sums ? (float*)work : nullptr;
  const double in = row_bytes(a.x) + row_bytes(a.dn) + row_bytes(a.dxn);
  // (a norm alone; kFar is near kPast: 8192 × 4096 8-bit rows, fp32 gradient, kNear / kFar / kPast 55 / 53 / 52 µs;
  // with a block kNear is as good or better at all sizes: 8192 × 5120 121 / 136 / 132)
  const bool small = cache_of(in * a.rows * a.D, 0) == kNear, near = a.y.p || small;
  // (see put8: 2048 × 4096 8-bit rows 30 µs past the caches, 33 into them; 4096 58.4, 57.4; 12000 146, 141)
  const bool through = a.dx_f32 && !small;
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * waves), 0, s, a, part, through);
    return hipGetLastError();
  };
  auto by_cache = [&](auto x, auto y, auto g, auto f) {
    constexpr int X = decltype(x)::value, Y = decltype(y)::value, G = decltype(g)::value;
    constexpr bool F = decltype(f)::value;
    if constexpr (Y == kRowsNone)
      if (!near) return go(join_bwd_kernel<X, Y, G, F, kPast>);
    return go(join_bwd_kernel<X, Y, G, F, kNear>);
  };
  auto by_gate = [&](auto x, auto y, auto g) {
    return full ? by_cache(x, y, g, std::true_type{}) : by_cache(x, y, g, std::false_type{});
  };
  auto by_y = [&](auto x, auto g) {
    switch (a.y.type) {
      case DSB_DT_BF16: return by_gate(x, Int<DSB_DT_BF16>{}, g);
      case DSB_DT_E4M3: return by_gate(x, Int<DSB_DT_E4M3>{}, g);
      default: return by_gate(x, Int<DSB_DT_INT8>{}, g);
    }
  };
  auto by_g = [&](auto x, auto f) { return a.dn.type == DSB_DT_F32 ? f(x, Int<DSB_DT_F32>{}) : f(x, Int<DSB_DT_BF16>{}); };
  if (a.rows > 0) {
    hipError_t e;
    if (!a.dn.p)  // no norm after: x' is not read
      e = by_y(Int<kRowsNone>{}, Int<kRowsNone>{});
    else if (a.y.p)
      e = by_type(a.x, [&](auto x) { return by_g(x, by_y); });
    else
      e = by_type(a.x, [&](auto x) {
        return by_g(x, [&](auto x1, auto g) { return by_cache(x1, Int<kRowsNone>{}, g, std::false_type{}); });
      });
    if (e != hipSuccess) return e;
  }
  if (sums)
    hipLaunchKernelGGL(join_sums_kernel, dim3((a.D + 4 * kSumLanes - 1) / (4 * kSumLanes), 2), dim3(kSumThreads), 0, s, a, part, blocks);
  return hipGetLastError();
}

}  // namespace dsb
