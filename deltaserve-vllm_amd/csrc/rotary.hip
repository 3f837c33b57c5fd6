// Rotary positions: each pair (p, q) of a head's first `rot` elements, neighbours (2i, 2i + 1) or the
// halves' (i, i + rot / 2), turns by the angle position·inv_freq[i] and is scaled by a factor,
//
//   p' = f·(p·cos − q·sin),  q' = f·(q·cos + p·sin)
//
// and the rest of the head stays as it is. The backward turns by the opposite angle with the same
// factor. Angles are taken in turns, position·(inv_freq / 2π) less its nearest whole number, in 64 bits and rounded
// once, and from there in fp32 with what that rounded off put back: at position 2^20 an fp32 angle is off by up
// to 2^-5 radians, and fp32 results without the last are off by 5.8e-8 (root mean square, relative), with it 4.1e-8.
//
// A wave takes a token, or a part of its heads where there are few tokens. It computes the token's
// cosines and sines once, a pair of them a lane, and keeps them in LDS, where all of its heads read
// them; then a lane moves 8 elements of either member of 8 pairs (halves), of 4 pairs (neighbours) or of what
// stays. Accesses of 16 bytes need their elements' alignment only, so all strides and widths go
// the same way: the last run of a region that is no multiple of 8 starts earlier and overlaps the
// one before. Both compute the same values there; in place, where the first may have written
// already, the second leaves them out. Bound by its bytes: 16384 rows of 40 heads of 128 64 µs, 5.3 TB/s (31 pairs
// of such a head 88 µs; one element at a time it took 212), 256 rows 3.6 µs.
#include <algorithm>
#include <type_traits>

#include "block.h"

namespace dsb {

namespace {

constexpr int kWaves = 4, kMostPairs = DSB_ROTARY_MOST / 2 + 8;  // (a run may read past the last pair)
constexpr int kSlots = 2;  // runs that a lane has in flight

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int T>
struct Elem {
  using type = bf16;
};
template <>
struct Elem<DSB_DT_F16> {
  using type = _Float16;
};
template <>
struct Elem<DSB_DT_F32> {
  using type = float;
};

typedef float f32x4e __attribute__((ext_vector_type(4), aligned(4)));

// 8 elements as they lie, wherever they start.
template <int T>
struct Vec8 {
  u32x4 a, b;
  using E = typename Elem<T>::type;
  template <int P>
  DSB_DEV void load(const E* p) {
    a = load_as<P, u32x4h>(p);
    if constexpr (T == DSB_DT_F32) b = load_as<P, u32x4h>(p + 4);
  }
  template <int P>
  DSB_DEV void store(E* p) const {
    store_as<P, u32x4h>(p, a);
    if constexpr (T == DSB_DT_F32) store_as<P, u32x4h>(p + 4, b);
  }
  DSB_DEV void get(float v[8]) const {
    if constexpr (T == DSB_DT_BF16) {
      unpack8(a, v);
    } else if constexpr (T == DSB_DT_F16) {
      const f16x8 h = __builtin_bit_cast(f16x8, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
      floats8(a, b, v);
    }
  }
  DSB_DEV void set(const float v[8]) {
    if constexpr (T == DSB_DT_BF16) {
      a = pack8(v);
    } else if constexpr (T == DSB_DT_F16) {
      f16x8 h;
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (_Float16)v[i];
      a = __builtin_bit_cast(u32x4, h);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = __builtin_bit_cast(unsigned, v[i]);
        b[i] = __builtin_bit_cast(unsigned, v[4 + i]);
      }
    }
  }
};

// EVEN: the regions are multiples of 8 elements.
// Runs of 8 elements (of all there are, in a region with fewer) of a head: `turned` of them over the
// pairs' first members or, with neighbours (NEXT), over both, and the rest over what stays.
template <int T, bool NEXT, bool EVEN, int P>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(RotaryArgs a, int parts, int per, int turned,
                                                             int slots, unsigned magic) {
  using E = typename Elem<T>::type;
  __shared__ __align__(16) float table[kWaves][2][kMostPairs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long item = (long)blockIdx.x * kWaves + wave;
  const bool live = item < (long)a.n * parts;
  const long t = live ? item / parts : 0;
  const int h0 = live ? (int)(item % parts) * per : 0;
  const int half = a.rot >> 1;
  float *cosv = table[wave][0], *sinv = table[wave][1];
  if (live) {
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[t] : (double)((const int*)a.pos)[t];
    for (int i = lane; i < half; i += 64) {
      // (one fma: the product's own rounding would be 1.9e-7 radians at position 2^31)
      const double u = 2 * __builtin_fma(pos, a.turns[i], -__builtin_rint(pos * a.turns[i]));
      float s, c;
      sincospif((float)u, &s, &c);
      // what the angle lost to fp32, up to 2^-25 half turns, to the first order
      const float d = (float)(u - (double)(float)u) * 3.14159265f;
      const float c1 = a.factor * (c - s * d), s1 = a.factor * (s + c * d);
      cosv[i] = c1;
      sinv[i] = a.inverse ? -s1 : s1;
    }
  }
  __syncthreads();
  if (!live) return;
  const int heads = min(per, a.heads - h0);
  const E* x = (const E*)a.x + t * a.ldx + h0 * a.hx;
  E* y = (E*)a.y + t * a.ldy + h0 * a.hy;
  const int total = heads * slots;
  const bool place = a.x == a.y;
  // elements of a run in the two regions
  const int count1 = EVEN ? 8 : min(8, NEXT ? a.rot : half);
  const int count2 = EVEN ? 8 : min(8, a.hd - a.rot);
  for (int k0 = lane; k0 < total; k0 += 64 * kSlots) {
    Vec8<T> p[kSlots], q[kSlots];
    float pe[8], qe[8];  // of runs of less than 8 elements, which are the whole region
    int slot[kSlots], at[kSlots], from[kSlots];
    const E* xi[kSlots];
    E* yi[kSlots];
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
      const int k = k0 + 64 * u;
      const int h = magic ? (int)__umulhi((unsigned)k, magic) : k;
      const int s = k - h * slots;
      slot[u] = k < total ? s : slots;  // (slots: none)
      const bool turns = s < turned;
      const int length = turns ? (NEXT ? a.rot : half) : a.hd - a.rot;
      const int want = 8 * (turns ? s : s - turned);
      at[u] = EVEN ? want : max(0, min(want, length - 8));
      from[u] = want - at[u];
      xi[u] = x + h * a.hx + at[u] + (turns ? 0 : a.rot);
      yi[u] = y + h * a.hy + at[u] + (turns ? 0 : a.rot);
      if (k < total && (turns || !place) && (turns ? count1 : count2) == 8) {
        p[u].template load<P>(xi[u]);
        if (!NEXT && turns) q[u].template load<P>(xi[u] + half);
      }
    }
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
      if (slot[u] >= slots) continue;
      if (slot[u] >= turned) {
        if (place) continue;
        if (count2 == 8) {
          p[u].template store<P>(yi[u]);
        } else {
          for (int e = 0; e < count2; ++e) yi[u][e] = xi[u][e];
        }
        continue;
      }
      if (count1 == 8) {
        p[u].get(pe);
        if (!NEXT) q[u].get(qe);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          pe[e] = e < count1 ? (float)xi[u][e] : 0.f;
          if (!NEXT) qe[e] = e < count1 ? (float)xi[u][half + e] : 0.f;
        }
      }
      const int pair = NEXT ? at[u] >> 1 : at[u];
#pragma unroll
      for (int b = 0; b < (NEXT ? 1 : 2); ++b) {
        using Four = typename std::conditional<EVEN, f32x4, f32x4e>::type;
        const f32x4 c = *reinterpret_cast<const Four*>(cosv + pair + 4 * b);
        const f32x4 sn = *reinterpret_cast<const Four*>(sinv + pair + 4 * b);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float &f = NEXT ? pe[2 * e] : pe[4 * b + e], &g = NEXT ? pe[2 * e + 1] : qe[4 * b + e];
          const float f0 = f, g0 = g;
          f = f0 * c[e] - g0 * sn[e];
          g = g0 * c[e] + f0 * sn[e];
        }
      }
      const int skip = place ? from[u] : 0;
      if (count1 == 8 && skip == 0) {
        p[u].set(pe);
        p[u].template store<P>(yi[u]);
        if (!NEXT) {
          q[u].set(qe);
          q[u].template store<P>(yi[u] + half);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= skip && e < count1) {
            yi[u][e] = (E)pe[e];
            if (!NEXT) yi[u][half + e] = (E)qe[e];
          }
        }
      }
    }
  }
}

// Waves wanted before a token's heads stay with one of them, enough to fill the chip's 256 CUs with 16 each. µs with
// 1024 / 2048 / 4096 / 8192: 256 rows of 48 heads of 128, 32 turned, 4.1 / 3.7 / 3.6 / 3.7; 504 rows of 40 heads 4.3 / 4.0
// / 3.9 / 3.9; from 4096 rows on no difference.
constexpr long kMostSplit = 4096;

}  // namespace

hipError_t rotary(const RotaryArgs& a, hipStream_t s) {
  if (a.n <= 0 || a.heads <= 0) return hipSuccess;
  const int turned = ((a.interleaved ? a.rot : a.rot / 2) + 7) / 8;
  const bool even = a.rot % (a.interleaved ? 8 : 16) == 0 && (a.hd - a.rot) % 8 == 0;
  const int slots = turned + (a.hd - a.rot + 7) / 8;
  // at least a wave's worth of slots to a part
  const int least = (64 + slots - 1) / slots;
  const long want = std::max(1l, kMostSplit / a.n);
  const int per = (int)std::max<long>(least, (a.heads + want - 1) / want);
  const int parts = (a.heads + per - 1) / per;
  // k / slots for k below per·slots and a wave's step past it: exact while k·slots < 2^32 (0: one slot)
  const unsigned magic = slots == 1 ? 0u : (unsigned)(((1ull << 32) + slots - 1) / slots);
  const unsigned blocks = (unsigned)(((long)a.n * parts + kWaves - 1) / kWaves);
  const double bytes = (double)a.n * a.heads * a.hd * (a.dtype == DSB_DT_F32 ? 4 : 2);
  const int cache = cache_of(bytes, bytes);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, s, a, parts, per, turned, slots, magic);
    return hipGetLastError();
  };
  auto by_cache = [&](auto t, auto next, auto ev) {
    constexpr int T = decltype(t)::value;
    constexpr bool N = decltype(next)::value, E = decltype(ev)::value;
    // runs that start anywhere cover lines in parts: their stores go into the caches (rot 30 of 64 fp32
    // elements, 167 MB: 55 µs past them, 38 so)
    if constexpr (!E)
      return cache == kNear ? go(rotary_kernel<T, N, E, kIn>) : go(rotary_kernel<T, N, E, kFar>);
    else
      return cache == kNear  ? go(rotary_kernel<T, N, E, kNear>)
             : cache == kFar ? go(rotary_kernel<T, N, E, kFar>)
                             : go(rotary_kernel<T, N, E, kPast>);
  };
  using std::false_type;
  using std::true_type;
  auto by_type = [&](auto t) {
    if (even) return a.interleaved ? by_cache(t, true_type{}, true_type{}) : by_cache(t, false_type{}, true_type{});
    return a.interleaved ? by_cache(t, true_type{}, false_type{}) : by_cache(t, false_type{}, false_type{});
  };
  switch (a.dtype) {
    case DSB_DT_BF16: return by_type(std::integral_constant<int, DSB_DT_BF16>{});
    case DSB_DT_F16: return by_type(std::integral_constant<int, DSB_DT_F16>{});
    default: return by_type(std::integral_constant<int, DSB_DT_F32>{});
  }
}

}  // namespace dsb
