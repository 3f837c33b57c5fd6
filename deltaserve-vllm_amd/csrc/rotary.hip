// Rotary positions: each pair (p, q) of a head's first `rot` elements, neighbours (2i, 2i + 1) or the
// halves' (i, i + rot / 2), turns by the angle position·inv_freq[i] and is scaled by a factor,
//
//   p' = f·(p·cos − q·sin),  q' = f·(q·cos + p·sin)
//
// and the rest of the head stays as it is. The backward turns by the opposite angle with the same
// factor. Angles are taken in turns, position·(inv_freq / 2π) in 64 bits less its nearest whole
// number, and from there in fp32: at position 2^20 an fp32 angle is off by up to 2^-5 radians.
//
// A wave takes a token, or a part of its heads where there are few tokens. It computes the token's
// cosines and sines once, a pair of them a lane, and keeps them in LDS, where all of its heads read
// them; then it moves 8 elements of either member of 8 pairs (or 4 pairs of neighbours) a lane. Bound
// by its bytes.
#include <algorithm>
#include <type_traits>

#include "block.h"

namespace dsb {

namespace {

constexpr int kWaves = 4, kMostPairs = DSB_ROTARY_MOST / 2;

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

// 8 elements as they lie.
template <int T>
struct Vec8 {
  u32x4 a, b;
  using E = typename Elem<T>::type;
  DSB_DEV void load(const E* p) {
    a = ldg128_nt(p);
    if constexpr (T == DSB_DT_F32) b = ldg128_nt(p + 4);
  }
  DSB_DEV void store(E* p) const {
    __builtin_nontemporal_store(a, reinterpret_cast<u32x4*>(p));
    if constexpr (T == DSB_DT_F32) __builtin_nontemporal_store(b, reinterpret_cast<u32x4*>(p + 4));
  }
  DSB_DEV void get(float v[8]) const {
    if constexpr (T == DSB_DT_BF16) {
      unpack8(a, v);
    } else if constexpr (T == DSB_DT_F16) {
      const f16x8 h = __builtin_bit_cast(f16x8, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned x = a[i], y = b[i];
        v[i] = __builtin_bit_cast(float, x);
        v[4 + i] = __builtin_bit_cast(float, y);
      }
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

// VEC: 16-byte accesses, `slots` a head: with halves rot / 16 slots of 8 pairs, then 8 elements that
// stay; with neighbours 8 elements each, the first rot / 8 of them turned. Else one pair or element
// a slot.
template <int T, bool NEXT, bool VEC>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(RotaryArgs a, int parts, int per,
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
      const double turn = pos * a.turns[i];
      float s, c;
      sincospif(2.f * (float)(turn - __builtin_rint(turn)), &s, &c);
      cosv[i] = a.factor * c;
      sinv[i] = a.inverse ? -a.factor * s : a.factor * s;
    }
  }
  __syncthreads();
  if (!live) return;
  const int heads = min(per, a.heads - h0);
  const E* x = (const E*)a.x + t * a.ldx + h0 * a.hx;
  E* y = (E*)a.y + t * a.ldy + h0 * a.hy;
  const int total = heads * slots;
  if constexpr (VEC) {
    const int turned = NEXT ? a.rot >> 3 : a.rot >> 4;
    const bool keep = a.x == a.y;  // what stays is there
    constexpr int U = 2;
    for (int k0 = lane; k0 < total; k0 += 64 * U) {
      Vec8<T> p[U], q[U];
      const E* xi[U];
      E* yi[U];
      int s[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + 64 * u;
        const int h = magic ? (int)__umulhi((unsigned)k, magic) : k;
        s[u] = k < total ? k - h * slots : -1;
        const int at = NEXT ? 8 * s[u] : s[u] < turned ? 8 * s[u] : a.rot + 8 * (s[u] - turned);
        xi[u] = x + h * a.hx + at;
        yi[u] = y + h * a.hy + at;
        if (s[u] >= 0 && (s[u] < turned || !keep)) {
          p[u].load(xi[u]);
          if (!NEXT && s[u] < turned) q[u].load(xi[u] + half);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s[u] < 0) continue;
        if (s[u] >= turned) {
          if (!keep) p[u].store(yi[u]);
          continue;
        }
        float pv[8], qv[8];
        p[u].get(pv);
        if constexpr (NEXT) {
          const f32x4 c = *reinterpret_cast<const f32x4*>(cosv + 4 * s[u]);
          const f32x4 sn = *reinterpret_cast<const f32x4*>(sinv + 4 * s[u]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = pv[2 * e], g = pv[2 * e + 1];
            pv[2 * e] = f * c[e] - g * sn[e];
            pv[2 * e + 1] = g * c[e] + f * sn[e];
          }
          p[u].set(pv);
          p[u].store(yi[u]);
        } else {
          q[u].get(qv);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const f32x4 c = *reinterpret_cast<const f32x4*>(cosv + 8 * s[u] + 4 * b);
            const f32x4 sn = *reinterpret_cast<const f32x4*>(sinv + 8 * s[u] + 4 * b);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = pv[4 * b + e], g = qv[4 * b + e];
              pv[4 * b + e] = f * c[e] - g * sn[e];
              qv[4 * b + e] = g * c[e] + f * sn[e];
            }
          }
          p[u].set(pv);
          q[u].set(qv);
          p[u].store(yi[u]);
          q[u].store(yi[u] + half);
        }
      }
    }
  } else {
    for (int k = lane; k < total; k += 64) {
      const int h = magic ? (int)__umulhi((unsigned)k, magic) : k, s = k - h * slots;
      const E* xi = x + h * a.hx;
      E* yi = y + h * a.hy;
      if (s >= half) {
        yi[half + s] = xi[half + s];
      } else {
        const int i0 = NEXT ? 2 * s : s, i1 = NEXT ? 2 * s + 1 : s + half;
        const float p = (float)xi[i0], q = (float)xi[i1], c = cosv[s], sn = sinv[s];
        yi[i0] = (E)(p * c - q * sn);
        yi[i1] = (E)(q * c + p * sn);
      }
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Waves wanted before a token's heads stay with one of them.
constexpr long kMostSplit = 4096;

}  // namespace

hipError_t rotary(const RotaryArgs& a, hipStream_t s) {
  if (a.n <= 0 || a.heads <= 0) return hipSuccess;
  const int es = a.dtype == DSB_DT_F32 ? 4 : 2;
  auto whole = [&](long v) { return v * es % 16 == 0; };
  const bool vec = a.hd % 8 == 0 && a.rot % (a.interleaved ? 8 : 16) == 0 && aligned16(a.x) &&
                   aligned16(a.y) && whole(a.ldx) && whole(a.hx) && whole(a.ldy) && whole(a.hy);
  const int slots = !vec ? a.hd - a.rot / 2 : a.interleaved ? a.hd / 8 : a.rot / 16 + (a.hd - a.rot) / 8;
  // at least a wave's worth of slots to a part
  const int least = (64 + slots - 1) / slots;
  const long want = std::max(1l, kMostSplit / a.n);
  const int per = (int)std::max<long>(least, (a.heads + want - 1) / want);
  const int parts = (a.heads + per - 1) / per;
  // k / slots for k below per·slots and a wave's step past it: exact while k·slots < 2^32 (0: one slot)
  const unsigned magic = slots == 1 ? 0u : (unsigned)(((1ull << 32) + slots - 1) / slots);
  const unsigned blocks = (unsigned)(((long)a.n * parts + kWaves - 1) / kWaves);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, s, a, parts, per, slots, magic);
    return hipGetLastError();
  };
  auto by_type = [&](auto t) {
    constexpr int T = decltype(t)::value;
    if (a.interleaved) return vec ? go(rotary_kernel<T, true, true>) : go(rotary_kernel<T, true, false>);
    return vec ? go(rotary_kernel<T, false, true>) : go(rotary_kernel<T, false, false>);
  };
  switch (a.dtype) {
    case DSB_DT_BF16: return by_type(std::integral_constant<int, DSB_DT_BF16>{});
    case DSB_DT_F16: return by_type(std::integral_constant<int, DSB_DT_F16>{});
    case DSB_DT_F32: return by_type(std::integral_constant<int, DSB_DT_F32>{});
    default: return hipErrorInvalidValue;
  }
}

}  // namespace dsb
