// Clip by group and AdamW over many tensors, moments in 8 or 32 bits.
//
//   g' = g·min(1, max_norm / (‖group‖ + 1e-6))
//   m' = β1·m + (1 − β1)·g',  v' = β2·v + (1 − β2)·g'²
//   w' = w − lr·wd·w − (lr / bc1)·m' / (sqrt(v') / sqrt(bc2) + ε),  bc_i = 1 − β_i^t
//
// 8 bits. Blocks of 256 elements share two fp32 scales: m = code·m_scale and
// sqrt(v) = code·r_scale, codes e4m3 (3 mantissa bits, largest 448, smallest 2^-9).
// The square root halves the exponents that v takes, so a block holds v over 11
// decades. m moves by a tenth of the gradient a step and is rounded to nearest
// (half a step, 2^-4 relative). sqrt(v) falls by at most 0.05 % a step (β2 = 0.999), far
// below half a step of 6 to 12 %: to nearest it would never fall, so it is rounded up or
// down at random in proportion to where it lies, and the mean moves as it should. It
// is never rounded to 0 from above, where m / (0 + ε) would leap. The step uses m' and
// v' before they are rounded. The moments take the formula's operations one by one in fp32,
// each to nearest, so that their codes are those that elementary operations give, bit for
// bit: a code on the other side of where two meet (one in a million with fused operations) is
// a step of 6 to 12 % that later updates show.
//
// Range. Blocks whose largest |m| or sqrt(v) is below 2^-100 are held as zeros. The squares
// are taken in fp32: gradients (after the clip) and sqrt(v) lose bits in v below 2^-63 and
// count as 0 there below 2^-74.5, and from 2^64 on v is infinite; the root is to nearest for v
// from 2^-100 on.
//
// A workgroup takes a chunk of 4096 elements, a wave 4 blocks, 16 lanes a block:
// loads of 16 bytes a lane cover whole 256-byte runs, and the block's
// maxima are 4 DPP steps. The step is bound by its bytes, which nothing reads again:
// its loads and stores bypass the caches, where they only push out what the norm's pass
// left of the gradients (54 M fp32 elements with fp32 moments 320 → 259 µs, 6.7 TB/s;
// 252 M bf16 ones with 8-bit moments 575 → 515; 84 M fp32 ones, no clip, 252 → 230; the
// stores alone 321, 592, 272, the moments' loads alone 312, 571, 241). The norm's pass
// reads through them (past them: 285, 556).
#include <cmath>
#include <type_traits>

#include "feedback.h"

namespace dsb {

namespace {

constexpr int kBlock = DSB_ADAM_BLOCK, kChunk = DSB_ADAM_CHUNK;
constexpr int kThreads = kChunk / 16;  // of a chunk's workgroup in the step
constexpr float kTiny = 0x1p-100f;
// Words of shared memory by block: its codes, and the gap that spreads a wave's four blocks
// over the banks.
constexpr int kTurn = kBlock / 4 + 16;

struct Hyper {
  float b1, ob1, b2, ob2;  // β and 1 − β, each rounded once from 64 bits
  float decay;             // 1 − lr·wd
  float step_size, rbc2;   // lr / bc1, 1 / sqrt(bc2)
  float eps;
  unsigned key;
};

__host__ __device__ inline unsigned mix32(unsigned x) {
  x ^= x >> 16;
  x *= 0x6a09e667u;  // the first bits of sqrt(2) and sqrt(3)
  x ^= x >> 15;
  x *= 0xbb67ae85u;
  return x ^ (x >> 16);
}
constexpr unsigned kGolden = 0x9e3779b9u;

__host__ __device__ inline Hyper make_hyper(double lr, double beta1, double beta2, double eps,
                                            double wd, int64_t step, unsigned seed) {
  const double bc1 = -expm1((double)step * log(beta1)), bc2 = -expm1((double)step * log(beta2));
  Hyper h;
  h.b1 = (float)beta1;
  h.ob1 = (float)(1.0 - beta1);
  h.b2 = (float)beta2;
  h.ob2 = (float)(1.0 - beta2);
  h.decay = (float)(1.0 - lr * wd);
  h.step_size = (float)(lr / bc1);
  h.rbc2 = (float)(1.0 / sqrt(bc2));
  h.eps = (float)eps;
  h.key = mix32(seed + (unsigned)step * kGolden);
  return h;
}

// Tensors' addresses come from a table in memory, of which the compiler does not know that they
// are device memory: without these casts every access is a flat one, which waits on the LDS
// counter too.
template <class T>
using Global = __attribute__((address_space(1))) T;
template <class T>
DSB_DEV T gload(const void* p, int e) {
  return reinterpret_cast<const Global<T>*>((unsigned long)p)[e];
}
template <class T>
DSB_DEV void gstore(void* p, int e, T v) {
  reinterpret_cast<Global<T>*>((unsigned long)p)[e] = v;
}

typedef unsigned u32x4h __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32x2h __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

template <bool NT, class T>
DSB_DEV T load_at(unsigned long at) {
  const auto* q = reinterpret_cast<const Global<T>*>(at);
  return NT ? __builtin_nontemporal_load(q) : *q;
}
template <int E>
using Run = unsigned __attribute__((ext_vector_type(E)));
// G runs of E (4 or 8) consecutive elements of a chunk, from e, e + step, ..., as they lie (bf16:
// two to a word), zeros past its `count`, wherever they start (these loads need their elements'
// alignment only). The type is tested once and what is left of a last run comes after, so that
// all the loads are on their way together. NT: loads past the caches.
template <bool WHOLE, bool BF, bool NT, int E, int G>
DSB_DEV void load_runs(Run<E> (&o)[G], const void* p, int e, int step, int count) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int at = e + step * g;
    const unsigned long a = (unsigned long)p + (BF ? 2l : 4l) * at;
    if (WHOLE || at + E <= count) {
      if (BF && E == 8) {
        const u32x4h x = load_at<NT, u32x4h>(a);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[g][i] = x[i];
      } else if (BF) {
        const u32x2h x = load_at<NT, u32x2h>(a);
        o[g][0] = x[0];
        o[g][1] = x[1];
      } else {
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
          const u32x4u x = load_at<NT, u32x4u>(a + 16 * h);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[g][4 * h + i] = x[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) o[g][i] = 0;
    }
  }
  if (!WHOLE) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int at = e + step * g;
      if (at < count && at + E > count) {
#pragma unroll
        for (int i = 0; i < E - 1; ++i)
          if (at + i < count) {
            if (BF)
              o[g][i / 2] |= (unsigned)gload<uint16_t>(p, at + i) << (16 * (i & 1));
            else
              o[g][i] = gload<unsigned>(p, at + i);
          }
      }
    }
  }
}
template <bool NT, int E, int G>
DSB_DEV void load_runs(Run<E> (&o)[G], const void* p, int e, int step, int count, bool bf) {
  if (count == kChunk) {
    if (bf)
      load_runs<true, true, NT>(o, p, e, step, count);
    else
      load_runs<true, false, NT>(o, p, e, step, count);
  } else {
    if (bf)
      load_runs<false, true, NT>(o, p, e, step, count);
    else
      load_runs<false, false, NT>(o, p, e, step, count);
  }
}
// Element i of a run.
template <int E>
DSB_DEV float value(Run<E> o, int i, bool bf) {
  const unsigned two = o[i / 2], one = o[i];
  const unsigned x = i & 1 ? two & 0xffff0000u : two << 16;
  return __builtin_bit_cast(float, bf ? x : one);
}
// A run's elements times a power of two.
template <int E>
DSB_DEV void rescale(Run<E>& o, float by, bool bf) {
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const float a = value(o, i, bf) * by, b = value(o, i + 1, bf) * by;
    if (bf) {
      o[i / 2] = (unsigned)__builtin_bit_cast(uint16_t, (bf16)a) |
                 (unsigned)__builtin_bit_cast(uint16_t, (bf16)b) << 16;
    } else {
      o[i] = __builtin_bit_cast(unsigned, a);
      o[i + 1] = __builtin_bit_cast(unsigned, b);
    }
  }
}
// A run of E elements from e, past the caches.
template <int E>
DSB_DEV void store_run(void* p, int e, int count, bool bf, const float (&v)[E]) {
  if (e + E <= count) {
    if (bf) {
      const unsigned long a = (unsigned long)p + 2l * e;
      if constexpr (E == 8)
        __builtin_nontemporal_store((u32x4h)pack8(v), reinterpret_cast<Global<u32x4h>*>(a));
      else
        __builtin_nontemporal_store(
            __builtin_bit_cast(u32x2, bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]}),
            reinterpret_cast<Global<u32x2h>*>(a));
    } else {
#pragma unroll
      for (int h = 0; h < E / 4; ++h)
        __builtin_nontemporal_store(
            f32x4u{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]},
            reinterpret_cast<Global<f32x4u>*>((unsigned long)p + 4l * (e + 4 * h)));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < E - 1; ++i)
    if (e + i < count) {
      if (bf)
        gstore(p, e + i, (bf16)v[i]);
      else
        gstore(p, e + i, v[i]);
    }
}

// The moments: kernel arguments, aligned.
template <class T>
DSB_DEV T nt_load(const void* base, long at) {
  return __builtin_nontemporal_load(reinterpret_cast<const T*>(base) + at);
}
template <class T>
DSB_DEV void nt_store(void* base, long at, T v) {
  __builtin_nontemporal_store(v, reinterpret_cast<T*>(base) + at);
}
// The largest of the 16 lanes of a block, as unsigned bits (of magnitudes: NaN wins).
DSB_DEV unsigned max16(unsigned x) {
  auto step = [&](auto ctrl) {
    const unsigned y =
        __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, 0xf, 0xf, false);
    x = max(x, y);
  };
  step(std::integral_constant<int, 0xB1>{});   // lanes 1 0 3 2 of each four
  step(std::integral_constant<int, 0x4E>{});   // 2 3 0 1
  step(std::integral_constant<int, 0x141>{});  // mirrored within 8
  step(std::integral_constant<int, 0x140>{});  // within 16
  return x;
}
DSB_DEV unsigned mag(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }

DSB_DEV unsigned pack4_e4m3(const float* x) {
  unsigned r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
}
DSB_DEV void unpack4_e4m3(unsigned c, float* x) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
  x[0] = a[0];
  x[1] = a[1];
  x[2] = b[0];
  x[3] = b[1];
}

// x in [0, 448] onto the e4m3 grid, up with the chance (x − below) / step: 16 random
// bits (their middle) added under the three mantissa bits, the rest cut off. Below
// 2^-6 the grid's step stays 2^-9: 2^-6 is added first.
DSB_DEV float round_random(float x, unsigned r16) {
  const float off = x < 0x1p-6f ? 0x1p-6f : 0.f;
  const unsigned y = __builtin_bit_cast(unsigned, x + off) + ((r16 << 4) | 8u);
  const float q = __builtin_bit_cast(float, y & 0xfff00000u) - off;
  return x > 0.f ? fmaxf(q, 0x1p-9f) : 0.f;
}

}  // namespace

__global__ void adam_hyper_kernel(const float* lr_dev, const int64_t* step_dev, double lr,
                                  int64_t step, double beta1, double beta2, double eps, double wd,
                                  unsigned seed, Hyper* out) {
  *out = make_hyper(lr_dev ? (double)*lr_dev : lr, beta1, beta2, eps, wd,
                    step_dev ? *step_dev : step, seed);
}

// Σ g² of a chunk, in 64 bits (gradients of any finite size): a wave to a chunk, all its loads
// of 16 bytes a lane in flight at once.
__global__ __launch_bounds__(256) void adam_sumsq_kernel(const dsb_adam_chunk* __restrict__ chunks,
                                                         int nchunks,
                                                         double* __restrict__ partial) {
  const int c = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
  if (c >= nchunks) return;
  const dsb_adam_chunk t = chunks[c];
  const bool bf = (t.dtypes >> 8) == DSB_DT_BF16;
  double s = 0.0;
  if (t.count == kChunk) {
    if (bf) {
      u32x4 v[kChunk / 512];
#pragma unroll
      for (int k = 0; k < kChunk / 512; ++k)
        v[k] = load_at<false, u32x4h>((unsigned long)t.g + 16 * (64 * k + l));
#pragma unroll
      for (int k = 0; k < kChunk / 512; ++k) {
        float g[8];
        unpack8(v[k], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) s += (double)g[i] * (double)g[i];
      }
    } else {
      u32x4u v[kChunk / 256];
#pragma unroll
      for (int k = 0; k < kChunk / 256; ++k)
        v[k] = load_at<false, u32x4u>((unsigned long)t.g + 16 * (64 * k + l));
#pragma unroll
      for (int k = 0; k < kChunk / 256; ++k) {
        const f32x4 g = __builtin_bit_cast(f32x4, (u32x4)v[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s += (double)g[i] * (double)g[i];
      }
    }
  } else {
    for (int k0 = 0; k0 < kChunk / 256; k0 += 4) {
      Run<4> v[4];
      load_runs<false, 4>(v, t.g, 256 * k0 + 4 * l, 256, t.count, bf);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double g = value(v[k], i, bf);
          s += g * g;
        }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (l == 0) partial[c] = s;
}

// The sum over a block of NT threads, the same for all.
template <int NT>
DSB_DEV double block_sum64(double s, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) s += red[i];
  return s;
}
// The clip's factor, in two where one would leave fp32's normal range: g·first·second.
struct Clip {
  float first, second;
};
// With 8 bits a reciprocal and a product in fp32, each rounded (as elementary operations give it),
// else the quotient in 64 bits. A norm near or past fp32's range, or a factor that small, takes the
// quotient and leaves 2^-64 of it to a factor of its own.
template <int BITS>
DSB_DEV Clip clip_factor(double norm, double max_norm) {
  if (BITS == 8 && norm <= 0x1p100 && norm <= 0x1p100 * max_norm) {
    const float f = 1.f / ((float)norm + 1e-6f) * (float)max_norm;
    return Clip{1.f, f > 1.f ? 1.f : f};
  }
  const double c = max_norm / (norm + 1e-6);  // (NaN stays)
  if (c < 0x1p-100) return Clip{0x1p-64f, (float)(c * 0x1p64)};
  return Clip{1.f, c > 1.0 ? 1.f : (float)c};
}
// x / s to nearest, from inv = 1 / s to nearest: what the product leaves over, times inv. (s and
// the largest x are not near the smallest numbers, so that the rest is exact.)
DSB_DEV float divided(float x, float s, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, s, x), inv, q);
}
// sqrt(v) to nearest, by Tuckerman's test: the instruction is off by at most a step, and a
// neighbour s' of its s is the nearer one where v − s·s' says so (not with 0, infinity or NaN,
// where s stays). Below v = 2^-100 that difference may underflow.
DSB_DEV float root(float v) {
  const float s = __builtin_amdgcn_sqrtf(v);
  const float down = __builtin_bit_cast(float, __builtin_bit_cast(int, s) - 1);
  const float up = __builtin_bit_cast(float, __builtin_bit_cast(int, s) + 1);
  const float below = fmaf(-down, s, v), above = fmaf(-up, s, v);
  return above > 0.f ? up : below <= 0.f ? down : s;
}
// β·x + (1 − β)·y, every operation rounded.
DSB_DEV float blend(float b, float x, float ob, float y) {
#pragma clang fp contract(off)
  return b * x + ob * y;
}

// One block per group: its chunks' sums in a fixed order, the norm and the factor.
template <int BITS>
__global__ __launch_bounds__(1024) void adam_norm_kernel(const int* __restrict__ group_chunks,
                                                         const double* __restrict__ partial,
                                                         double max_norm, float* __restrict__ norms,
                                                         Clip* __restrict__ coef) {
  __shared__ double red[16];
  const int c0 = group_chunks[blockIdx.x], c1 = group_chunks[blockIdx.x + 1];
  double s = 0.0;
#pragma unroll 4
  for (int c = c0 + threadIdx.x; c < c1; c += 1024) s += partial[c];
  const double norm = sqrt(block_sum64<1024>(s, red));
  if (threadIdx.x == 0) {
    norms[blockIdx.x] = (float)norm;
    coef[blockIdx.x] = clip_factor<BITS>(norm, max_norm);
  }
}

// How a step's blocks get their group's clip factor: none, from adam_norm_kernel, or each from
// its group's sums.
enum { CLIP_NONE, CLIP_GIVEN, CLIP_SUM };
struct ClipArgs {
  int how;
  const Clip* coef;
  const int* group_chunks;
  int ngroups;
  const double* partial;
  double max_norm;
  float* norms;
};

namespace {

struct AdamKernelArgs {
  const dsb_adam_chunk* chunks;
  Hyper hv;
  const Hyper* hp;
  ClipArgs clip;
  void *mp, *vp;
  float *m_scale, *r_scale;
};

// A chunk; turn: kTurn words of shared memory of the lane's block. A lane holds E elements at
// a time: 16-byte accesses to fp32 weights, gradients or moments with 4, to bf16 ones with 8.
template <int BITS, int E>
DSB_DEV void adam_chunk(const AdamKernelArgs& a, const dsb_adam_chunk& t, int chunk, double* red,
                        unsigned* turn, bool wbf, bool gbf) {
  constexpr int G = 16 / E;
  const ClipArgs& clip = a.clip;
  const int l16 = threadIdx.x & 15, qb = threadIdx.x >> 4;  // 16 blocks of 256 per chunk
  const bool live = qb * kBlock < t.count;                  // the 16 lanes of a block together
  const int e0 = qb * kBlock + E * l16;  // and 16·E on, G times
  const long b = t.block + qb, s0 = b * kBlock + E * l16;
  const double mine =
      clip.how == CLIP_SUM && t.c0 + (int)threadIdx.x < t.c1 ? clip.partial[t.c0 + threadIdx.x] : 0.0;
  Run<E> graw[G], wraw[G];
  unsigned mc[G][E / 4], rc[G][E / 4];
  float m[G][E], r[G][E];
  float ms = 0.f, rs = 0.f;
  if (live) {
    load_runs<true, E>(graw, t.g, e0, 16 * E, t.count, gbf);
    load_runs<true, E>(wraw, t.w, e0, 16 * E, t.count, wbf);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      const long s = s0 + 16 * E * k;
      if constexpr (BITS == 32) {
#pragma unroll
        for (int h = 0; h < E / 4; ++h) {
          const f32x4 x = nt_load<f32x4>(a.mp, s / 4 + h), y = nt_load<f32x4>(a.vp, s / 4 + h);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            m[k][4 * h + i] = x[i];
            r[k][4 * h + i] = y[i];
          }
        }
      } else if constexpr (E == 8) {
        const u32x2 x = nt_load<u32x2>(a.mp, s / 8), y = nt_load<u32x2>(a.vp, s / 8);
        mc[k][0] = x[0];
        mc[k][1] = x[1];
        rc[k][0] = y[0];
        rc[k][1] = y[1];
      } else {
        mc[k][0] = nt_load<unsigned>(a.mp, s / 4);
        rc[k][0] = nt_load<unsigned>(a.vp, s / 4);
      }
    }
    if constexpr (BITS == 8) {
      ms = a.m_scale[b];
      rs = a.r_scale[b];
    }
  }
  Clip cf{1.f, 1.f};
  if (clip.how == CLIP_GIVEN) {
    cf = clip.coef[t.group];
  } else if (clip.how == CLIP_SUM) {
    const double norm = sqrt(block_sum64<kThreads>(mine, red));
    cf = clip_factor<BITS>(norm, clip.max_norm);
    if (chunk == t.c0 && threadIdx.x == 0) clip.norms[t.group] = (float)norm;
    if (chunk == 0)  // groups without elements
      for (int g = threadIdx.x; g < clip.ngroups; g += kThreads)
        if (clip.group_chunks[g] == clip.group_chunks[g + 1]) clip.norms[g] = 0.f;
  }
  if (!live) return;
  if (cf.first != 1.f) {  // rare
#pragma unroll
    for (int k = 0; k < G; ++k) rescale(graw[k], cf.first, gbf);
  }
  Hyper h = a.hv;
  if (a.hp) h = *a.hp;
  unsigned mtop = 0, rtop = 0;
#pragma unroll
  for (int k = 0; k < G; ++k) {
    if constexpr (BITS == 8) {
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        unpack4_e4m3(mc[k][q], m[k] + 4 * q);
        unpack4_e4m3(rc[k][q], r[k] + 4 * q);
      }
    }
    float w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float gi = value(graw[k], i, gbf) * cf.second, wi = value(wraw[k], i, wbf);
      if constexpr (BITS == 8) {
        const float ro = r[k][i] * rs;
        m[k][i] = blend(h.b1, m[k][i] * ms, h.ob1, gi);
        r[k][i] = root(blend(h.b2, ro * ro, h.ob2, gi * gi));
        mtop = max(mtop, mag(m[k][i]));
        rtop = max(rtop, mag(r[k][i]));
        w[i] = wi * h.decay -
               h.step_size * m[k][i] * __builtin_amdgcn_rcpf(r[k][i] * h.rbc2 + h.eps);
      } else {
        const float v = h.b2 * r[k][i] + h.ob2 * (gi * gi);
        m[k][i] = h.b1 * m[k][i] + h.ob1 * gi;
        r[k][i] = v;
        w[i] = wi * h.decay -
               h.step_size * m[k][i] *
                   __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * h.rbc2 + h.eps);
      }
    }
    store_run(t.w, e0 + 16 * E * k, t.count, wbf, w);
    if constexpr (BITS == 32) {
      const long s = s0 + 16 * E * k;
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        nt_store(a.mp, s / 4 + q, f32x4{m[k][4 * q], m[k][4 * q + 1], m[k][4 * q + 2], m[k][4 * q + 3]});
        nt_store(a.vp, s / 4 + q, f32x4{r[k][4 * q], r[k][4 * q + 1], r[k][4 * q + 2], r[k][4 * q + 3]});
      }
    }
  }
  if constexpr (BITS == 8) {
    const float mt = __builtin_bit_cast(float, max16(mtop));
    const float rt = __builtin_bit_cast(float, max16(rtop));
    // not below kTiny (so NaN and infinity show in the scale)
    const float unit = mt * (1.f / 448.f), im = mt < kTiny ? 0.f : 1.f / unit;
    const float ir = rt < kTiny ? 0.f : 1.f / rt * 448.f;
    const unsigned key = mix32(h.key ^ mix32((unsigned)b));
#pragma unroll
    for (int k = 0; k < G; ++k) {
      float q[E], p[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        q[i] = fminf(fmaxf(divided(m[k][i], unit, im), -448.f), 448.f);
        p[i] = fminf(r[k][i] * ir, 448.f);
      }
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const unsigned x = mix32(key + (unsigned)(8 * E * k + E / 2 * l16 + j) * kGolden);
        p[2 * j] = round_random(p[2 * j], x & 0xffffu);
        p[2 * j + 1] = round_random(p[2 * j + 1], x >> 16);
      }
      const long s = s0 + 16 * E * k;
      if constexpr (E == 8) {
        nt_store(a.mp, s / 8, u32x2{pack4_e4m3(q), pack4_e4m3(q + 4)});
        nt_store(a.vp, s / 8, u32x2{pack4_e4m3(p), pack4_e4m3(p + 4)});
      } else {
        turn[16 * k + l16] = pack4_e4m3(q);
        rc[k][0] = pack4_e4m3(p);
      }
    }
    if constexpr (E == 4) {
      // 16 codes to a lane: a wave's leave in whole lines (from where they are made, 64 bytes a
      // block at a time, 9 % more bytes were written; 84 M elements 230 → 216 µs)
      auto turned = [&] {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const u32x4 x = *reinterpret_cast<const u32x4*>(turn + 4 * l16);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return x;
      };
      const long s = b * (kBlock / 16) + l16;
      nt_store(a.mp, s, turned());
#pragma unroll
      for (int k = 0; k < G; ++k) turn[16 * k + l16] = rc[k][0];
      nt_store(a.vp, s, turned());
    }
    if (l16 == 0) {
      a.m_scale[b] = mt < kTiny ? 0.f : unit;
      a.r_scale[b] = rt < kTiny ? 0.f : rt * (1.f / 448.f);
    }
  }
}

}  // namespace

// A block per chunk. With 8-bit moments the element types are constants of the code (2.3 M fp32
// elements: 15.3 → 14.8 µs; with 32 bits 258 → 261, where they stay variables), and a lane takes
// 8 elements at a time of bf16 weights and gradients (252 M: 508 → 494 µs), else 4 (84 M fp32
// ones with 8: 230 → 265). 84 M elements, no clip, weights and gradients fp32 / bf16 / bf16 and
// fp32 / fp32 and bf16: 215 / 147 / 163 / 192 µs with 8 bits (6.3 / 5.8 / 6.2 / 6.2 TB/s), 381 /
// 301 / 331 / 353 with 32 (6.1 to 6.2).
template <int BITS>
__global__ __launch_bounds__(kThreads) void adam_kernel(AdamKernelArgs a) {
  __shared__ double red[kThreads / 64];
  __shared__ __align__(16) unsigned turn[kTurn * kChunk / kBlock];
  const int chunk = blockIdx.x;
  const dsb_adam_chunk t = a.chunks[chunk];
  unsigned* mine = turn + kTurn * (threadIdx.x >> 4);
  const bool wbf = (t.dtypes & 255) == DSB_DT_BF16, gbf = (t.dtypes >> 8) == DSB_DT_BF16;
  if constexpr (BITS == 32)
    adam_chunk<32, 4>(a, t, chunk, red, mine, wbf, gbf);
  else if (wbf && gbf)
    adam_chunk<8, 8>(a, t, chunk, red, mine, true, true);
  else if (wbf)
    adam_chunk<8, 4>(a, t, chunk, red, mine, true, false);
  else if (gbf)
    adam_chunk<8, 4>(a, t, chunk, red, mine, false, true);
  else
    adam_chunk<8, 4>(a, t, chunk, red, mine, false, false);
}

int64_t adam_bytes(int nchunks, int ngroups) {
  return 256 + ((int64_t)nchunks * 8 + 255) / 256 * 256 +
         ((int64_t)ngroups * (int64_t)sizeof(Clip) + 255) / 256 * 256;
}

hipError_t adam_step(const AdamArgs& a, void* work, hipStream_t s) {
  Hyper* hp = (Hyper*)work;
  double* partial = (double*)((char*)work + 256);
  Clip* coef = (Clip*)((char*)partial + ((int64_t)a.nchunks * 8 + 255) / 256 * 256);
  const bool dev = a.lr_dev || a.step_dev, clip = a.max_norm >= 0;
  Hyper hv{};
  if (dev)
    hipLaunchKernelGGL(adam_hyper_kernel, dim3(1), dim3(1), 0, s, a.lr_dev, a.step_dev, a.lr, a.step,
                       a.beta1, a.beta2, a.eps, a.wd, a.seed, hp);
  else
    hv = make_hyper(a.lr, a.beta1, a.beta2, a.eps, a.wd, a.step, a.seed);
  ClipArgs c{CLIP_NONE, coef, a.group_chunks, a.ngroups, partial, a.max_norm, a.norms};
  if (clip) {
    if (a.nchunks > 0)
      hipLaunchKernelGGL(adam_sumsq_kernel, dim3((a.nchunks + 3) / 4), dim3(256), 0, s, a.chunks,
                         a.nchunks, partial);
    // Groups of at most 256 chunks (a million elements) are added up by each of their blocks,
    // which saves a launch (2.3 M elements in 28 groups: 14.6 µs, about 2 more with it); a thread of a
    // block reads one sum.
    c.how = a.most_chunks <= kThreads && a.nchunks > 0 ? CLIP_SUM : CLIP_GIVEN;
    if (c.how == CLIP_GIVEN)
      hipLaunchKernelGGL(a.bits == 8 ? adam_norm_kernel<8> : adam_norm_kernel<32>, dim3(a.ngroups), dim3(1024), 0, s, a.group_chunks, partial,
                         a.max_norm, a.norms, coef);
  }
  const AdamKernelArgs k{a.chunks, hv, dev ? hp : nullptr, c, a.m, a.v, a.m_scale, a.r_scale};
  if (a.nchunks > 0) {
    if (a.bits == 8)
      hipLaunchKernelGGL(adam_kernel<8>, dim3(a.nchunks), dim3(kThreads), 0, s, k);
    else
      hipLaunchKernelGGL(adam_kernel<32>, dim3(a.nchunks), dim3(kThreads), 0, s, k);
  }
  return hipGetLastError();
}

}  // namespace dsb
