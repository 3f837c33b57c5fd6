// Losses of training from feedback over a packing of sequences, each with its
// gradient with respect to the rows' log probabilities: a preference loss over
// pairs of sequences and a clipped policy loss with a KL term, and the labels that
// the log probabilities are taken of.
//
// Both are bound by their bytes (9 to 21 a row) where the batch is large and by
// launches where it is small, so:
//   * a batch of few rows is one launch of one workgroup, the sums by sequence in LDS;
//   * a large one takes two (a block to a pair) or three where sequences are long (by
//     tile, by pair, by tile), and for the policy loss what the mask's count needs, the
//     gradients with partial sums, and their total;
//   * rows are read and written four at a time wherever they start (16-byte accesses need
//     4-byte alignment only), several such groups in flight per thread, with no test of the
//     array's end but for a range's last three rows;
//   * sums over rows are held in 64 bits and added in a fixed order.
// The value of an unscored row is never used in arithmetic: it is replaced by 0
// first, so infinities and NaN there do not spread.
#include <algorithm>
#include <type_traits>

#include "feedback.h"

namespace dsb {

namespace {

constexpr int kChunkRows = DSB_CHUNK_ROWS;
// Batches of one workgroup: at most this many rows (two groups of four per thread), tiles
// and sequences. µs of the kernels, one workgroup / as larger batches: preference loss, 4
// sequences of 512 rows 4.5 / 5.8, 16 of 256 5.3 / 5.8, 32 of 128 7.3 / 5.8, 8 of 1024 5.7 / 6.3, 2 of
// 4096 9.2 / 10.2; policy loss by sequence, 4 of 512 6.5 / 13.8, 16 of 256 9.1 / 18.6, 8 of 1024
// 14.1 / 18.9, 2 of 4096 13.4 / 18.7, by token 5.2 / 11.0, 6.4 / 13.6, 8.0 / 13.8, 8.0 / 13.8. (32 short
// sequences take a second round of the 16 waves; the policy loss sets the border.)
constexpr int kSmallRows = 8192, kSmallTiles = 64, kSmallSeqs = 512;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned u32u __attribute__((aligned(1)));
template <int K>
using Int = std::integral_constant<int, K>;

DSB_DEV double wave_sumd(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
DSB_DEV int wave_sumi(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// K sums over a block of NT threads at once, the same for all; red: K · NT / 64 doubles,
// for one use.
template <int NT, int K>
DSB_DEV void block_sums(double (&v)[K], double* red) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = wave_sumd(v[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) red[(threadIdx.x >> 6) * K + k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = 0.0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v[k] += red[i * K + k];
  }
}
template <int NT>
DSB_DEV double block_sumd(double v, double* red) {
  double s[1] = {v};
  block_sums<NT>(s, red);
  return s[0];
}

// Rows r .. r+k-1 (k <= 4; Int<4>: one access), zeros after them. NT: past the caches.
template <bool NT = false, class K>
DSB_DEV f32x4 get4(const float* p, int r, K k) {
  if constexpr (std::is_same<K, Int<4>>::value) {
    const auto* q = reinterpret_cast<const f32x4u*>(p + r);
    return NT ? __builtin_nontemporal_load(q) : *q;
  } else {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < k) o[i] = p[r + i];
    return o;
  }
}
template <bool NT = false, class K>
DSB_DEV void put4(float* p, int r, K k, f32x4 v) {
  if constexpr (std::is_same<K, Int<4>>::value) {
    auto* q = reinterpret_cast<f32x4u*>(p + r);
    if (NT)
      __builtin_nontemporal_store((f32x4u)v, q);
    else
      *q = v;
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < k) p[r + i] = v[i];
  }
}
// Bit i: byte i of x is not zero.
DSB_DEV unsigned bytes4(unsigned x) {
  const unsigned y = (((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u;
  return (y >> 7 | y >> 14 | y >> 21 | y >> 28) & 15u;
}
template <class K>
DSB_DEV unsigned mask4(const uint8_t* p, int r, K k) {
  if constexpr (std::is_same<K, Int<4>>::value) {
    return *reinterpret_cast<const u32u*>(p + r);
  } else {
    unsigned o = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < k) o |= (unsigned)p[r + i] << (8 * i);
    return o;
  }
}

// Rows [r0, r1) by NT threads in groups of four from r0 on: load(r, k) for U groups of a
// thread at a time, then use(r, k, its value) for each; k is Int<4>, or 1 to 3 for what is left
// at the end. (Groups past the end load the last one again, so that the loads of a batch have
// no branch between them.)
template <int NT, int U, class L, class F>
DSB_DEV void for_rows(int r0, int r1, int tid, L&& load, F&& use) {
  const int full = (r1 - r0) >> 2;
  for (int g = tid; g < full; g += NT * U) {
    decltype(load(0, Int<4>{})) x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load(r0 + 4 * min(g + u * NT, full - 1), Int<4>{});
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (g + u * NT < full) use(r0 + 4 * (g + u * NT), Int<4>{}, x[u]);
  }
  const int r = r0 + 4 * full;
  if (r < r1 && tid == full % NT) use(r, r1 - r, load(r, r1 - r));
}

struct Tile {
  int r0, r1, seq;
};
DSB_DEV Tile get_tile(const dsb_pack_plan& p, int t) {
  const int4 v = reinterpret_cast<const int4*>(p.tiles)[t];
  return Tile{v.x, v.y, v.z};
}

// The values that a preference loss reads of a group. What is not given is read from the log
// probabilities instead and not used: a load without a branch.
struct PrefRows {
  f32x4 a, b;
  unsigned m;
};
struct PrefIn {
  const float *logp, *ref;
  const uint8_t* mask;
  template <class K>
  DSB_DEV PrefRows operator()(int r, K k) const {
    return PrefRows{get4(logp, r, k), get4(ref ? ref : logp, r, k), (*this).marks(r, k)};
  }
  template <class K>
  DSB_DEV unsigned marks(int r, K k) const {
    return mask4(mask ? mask : (const uint8_t*)logp, r, k);
  }
  DSB_DEV double diff(const PrefRows& x, int i) const {
    return (double)x.a[i] - (ref ? (double)x.b[i] : 0.0);
  }
};

// One pair from its sequences' sums and counts: the loss, the rewards and each
// scored row's gradient by sequence.
struct Pair {
  double loss;
  float reward[2], coef[2];
};
DSB_DEV Pair pair_eval(const PrefHyper& h, int npairs, const double (&sum)[2], const int (&cnt)[2]) {
  const double per[2] = {h.average ? (double)max(cnt[0], 1) : 1.0,
                         h.average ? (double)max(cnt[1], 1) : 1.0};
  const double s[2] = {sum[0] / per[0], sum[1] / per[1]};
  const double d = s[0] - s[1], z = h.beta * d - h.margin;
  Pair o;
  double g;  // d loss / d (s_0 − s_1)
  if (h.kind == DSB_PREF_SIGMOID) {
    const double e = exp(-fabs(z)), l = log1p(e), q = 1.0 / (1.0 + e);
    const double up = z >= 0 ? q : e * q, down = z >= 0 ? e * q : q;  // σ(z), σ(−z)
    // a term of weight 0 stays out: it may be infinite
    o.loss = (h.smooth < 1.0 ? (1.0 - h.smooth) * (fmax(-z, 0.0) + l) : 0.0) +
             (h.smooth > 0.0 ? h.smooth * (fmax(z, 0.0) + l) : 0.0);
    g = h.beta * (h.smooth * up - (1.0 - h.smooth) * down);
  } else if (h.kind == DSB_PREF_HINGE) {
    o.loss = z >= 1.0 ? 0.0 : 1.0 - z;
    g = z >= 1.0 ? 0.0 : z < 1.0 ? -h.beta : z;
  } else {
    const double t = d - 0.5 / h.beta;
    o.loss = t * t;
    g = 2.0 * t;
  }
  g *= h.grad_scale / npairs;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o.reward[i] = (float)(h.beta * s[i]);
    o.coef[i] = (float)((i ? -g : g) / per[i]);
  }
  return o;
}

}  // namespace

// ---------------------------------------------------------------- labels
//
// A wave to a tile. 16 M rows in 4096 sequences 108 µs (2.8 TB/s), 1 M in 1000 8.5, 8192 in 32 3.0
// (10.5 with the host).

__global__ __launch_bounds__(256) void labels_kernel(const int64_t* __restrict__ ids,
                                                     const uint8_t* __restrict__ mask,
                                                     dsb_pack_plan p, int64_t* __restrict__ labels,
                                                     uint8_t* __restrict__ rows) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  const Tile tl = get_tile(p, t);
  const int last = p.starts[tl.seq + 1] - 1;
#pragma unroll 4
  for (int r = tl.r0 + lane; r < tl.r1; r += 64) {
    int64_t v = -1;
    if (r < last && (!mask || mask[r + 1])) v = max(ids[r + 1], (int64_t)-1);
    labels[r] = v;
    rows[r] = v >= 0;
  }
}

// ---------------------------------------------------------------- preference loss

namespace {

// One wave: Σ (logp − ref) and the count over the scored rows of a tile; last: the last row of
// its sequence.
DSB_DEV double tile_sum(const PrefIn& in, const Tile& t, int last, int lane, int* count) {
  double s = 0.0;
  int c = 0;
  for_rows<64, 4>(t.r0, t.r1, lane, in, [&](int r, auto k, const PrefRows& x) {
    const unsigned m = bytes4(x.m);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool on = i < k && (in.mask ? m >> i & 1 : r + i != last);
      s += on ? in.diff(x, i) : 0.0;
      c += on;
    }
  });
  *count = wave_sumi(c);
  return wave_sumd(s);
}

// One wave: a tile's rows of the gradient. Large batches store it past the caches (4096 pairs of
// 1024 rows by pair: 18.4 → 17.5 µs; their loads past them too 18.3).
template <bool NT>
DSB_DEV void tile_grads(const PrefIn& in, const Tile& t, int last, float coef, float* dlogp,
                        int lane) {
  for_rows<64, 4>(
      t.r0, t.r1, lane, [&](int r, auto k) { return in.marks(r, k); },
      [&](int r, auto k, unsigned x) {
        const unsigned m = bytes4(x);
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = (in.mask ? m >> i & 1 : r + i != last) ? coef : 0.f;
        put4<NT>(dlogp, r, k, v);
      });
}

// A pair from its tiles' sums and counts, one after the other by one lane: 16 sequences of 1 M rows
// (256 tiles each) 87 µs, 2 of 8 M 369.
DSB_DEV Pair pair_of_tiles(const dsb_pack_plan& p, const PrefHyper& h, int i, const double* sums,
                           const int* counts) {
  double s[2] = {0.0, 0.0};
  int c[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int t = p.seq_tile[2 * i + k]; t < p.seq_tile[2 * i + k + 1]; ++t) {
      s[k] += sums[t];
      c[k] += counts[t];
    }
  return pair_eval(h, p.nseq / 2, s, c);
}

}  // namespace

__global__ __launch_bounds__(1024) void pref_small_kernel(PrefIn in, dsb_pack_plan p, PrefHyper h,
                                                          float* loss, float* rewards,
                                                          float* dlogp) {
  __shared__ double sums[kSmallTiles], red[16];
  __shared__ int counts[kSmallTiles];
  __shared__ float coef[kSmallSeqs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int t = wave; t < p.ntiles; t += 16) {
    const Tile tl = get_tile(p, t);
    int c;
    const double s = tile_sum(in, tl, p.starts[tl.seq + 1] - 1, lane, &c);
    if (lane == 0) {
      sums[t] = s;
      counts[t] = c;
    }
  }
  __syncthreads();
  const int npairs = p.nseq / 2;
  double total = 0.0;
  if ((int)threadIdx.x < npairs) {  // at most kSmallSeqs / 2 of 1024
    const int i = threadIdx.x;
    const Pair o = pair_of_tiles(p, h, i, sums, counts);
    total = o.loss;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      rewards[2 * i + k] = o.reward[k];
      coef[2 * i + k] = o.coef[k];
    }
  }
  total = block_sumd<1024>(total, red);  // its barrier publishes coef too
  if (threadIdx.x == 0) *loss = (float)(total / npairs);
  for (int t = wave; t < p.ntiles; t += 16) {
    const Tile tl = get_tile(p, t);
    tile_grads<false>(in, tl, p.starts[tl.seq + 1] - 1, coef[tl.seq], dlogp, lane);
  }
}

// NT threads per pair, whose rows lie together: both sums, the pair, its rows' gradient; NB / NT
// pairs to a block. Sequences of one tile, so that a count fits 16 bits. One wave evaluates the
// block's pairs, a lane each.
template <int NT, int NB>
__global__ __launch_bounds__(NB) void pref_pair_kernel(PrefIn in, dsb_pack_plan p, PrefHyper h,
                                                       float* rewards, float* dlogp,
                                                       double* losses) {
  static_assert(DSB_TILE_ROWS < 1 << 16, "counts");
  constexpr int P = NB / NT, WP = NT / 64;  // pairs of a block, waves of a pair
  __shared__ double sums[2][P][WP];
  __shared__ int counts[P][WP];
  __shared__ float both[P][2];
  const int q = threadIdx.x / NT, i = blockIdx.x * P + q, tid = threadIdx.x % NT;
  const int npairs = p.nseq / 2;
  int a = 0, b = 0, c = 0;
  if (i < npairs) {
    a = p.starts[2 * i];
    b = p.starts[2 * i + 1];
    c = p.starts[2 * i + 2];
  }
  double s[2] = {0.0, 0.0};
  int cnt = 0;  // of the first sequence, and of the second 16 bits up
  for_rows<NT, NT == 64 ? 4 : 2>(a, c, tid, in, [&](int r, auto k, const PrefRows& x) {
    const unsigned m = bytes4(x.m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool second = r + j >= b;
      const bool on = j < k && (in.mask ? m >> j & 1 : r + j != b - 1 && r + j != c - 1);
      const double d = on ? in.diff(x, j) : 0.0;
      s[0] += second ? 0.0 : d;
      s[1] += second ? d : 0.0;
      cnt += on ? second ? 1 << 16 : 1 : 0;
    }
  });
  s[0] = wave_sumd(s[0]);
  s[1] = wave_sumd(s[1]);
  cnt = wave_sumi(cnt);
  if ((tid & 63) == 0) {
    sums[0][q][tid >> 6] = s[0];
    sums[1][q][tid >> 6] = s[1];
    counts[q][tid >> 6] = cnt;
  }
  __syncthreads();
  const int e = threadIdx.x, ei = blockIdx.x * P + e;
  if (e < P && ei < npairs) {
    s[0] = s[1] = 0.0;
    cnt = 0;
#pragma unroll
    for (int k = 0; k < WP; ++k) {
      s[0] += sums[0][e][k];
      s[1] += sums[1][e][k];
      cnt += counts[e][k];
    }
    const int n[2] = {cnt & 0xffff, cnt >> 16};
    const Pair o = pair_eval(h, npairs, s, n);
    losses[ei] = o.loss;
    rewards[2 * ei] = o.reward[0];
    rewards[2 * ei + 1] = o.reward[1];
    both[e][0] = o.coef[0];
    both[e][1] = o.coef[1];
  }
  __syncthreads();
  const float d0 = both[q][0], d1 = both[q][1];
  for_rows<NT, NT == 64 ? 4 : 2>(
      a, c, tid, [&](int r, auto k) { return in.marks(r, k); },
      [&](int r, auto k, unsigned x) {
        const unsigned m = bytes4(x);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool on = in.mask ? m >> j & 1 : r + j != b - 1 && r + j != c - 1;
          v[j] = on ? r + j >= b ? d1 : d0 : 0.f;
        }
        put4<true>(dlogp, r, k, v);
      });
}

__global__ __launch_bounds__(1024) void pref_total_kernel(const double* losses, int npairs,
                                                          float* loss) {
  __shared__ double red[16];
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < npairs; i += 1024) s += losses[i];
  s = block_sumd<1024>(s, red);
  if (threadIdx.x == 0) *loss = (float)(s / npairs);
}

__global__ __launch_bounds__(256) void pref_sums_kernel(PrefIn in, dsb_pack_plan p, double* sums,
                                                        int* counts) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  const Tile tl = get_tile(p, t);
  int c;
  const double s = tile_sum(in, tl, p.starts[tl.seq + 1] - 1, lane, &c);
  if (lane == 0) {
    sums[t] = s;
    counts[t] = c;
  }
}

__global__ __launch_bounds__(256) void pref_pairs_kernel(dsb_pack_plan p, PrefHyper h,
                                                         const double* sums, const int* counts,
                                                         float* rewards, float* coef,
                                                         double* partial) {
  __shared__ double red[4];
  const int i = blockIdx.x * 256 + threadIdx.x;
  double l = 0.0;
  if (i < p.nseq / 2) {
    const Pair o = pair_of_tiles(p, h, i, sums, counts);
    l = o.loss;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      rewards[2 * i + k] = o.reward[k];
      coef[2 * i + k] = o.coef[k];
    }
  }
  l = block_sumd<256>(l, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = l;
}

// Block 0: the loss; the others: the gradients, a wave to a tile.
__global__ __launch_bounds__(256) void pref_grads_kernel(PrefIn in, dsb_pack_plan p,
                                                         const float* coef, const double* partial,
                                                         int nparts, float* loss, float* dlogp) {
  if (blockIdx.x == 0) {
    __shared__ double red[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += partial[i];
    s = block_sumd<256>(s, red);
    if (threadIdx.x == 0) *loss = (float)(s / (p.nseq / 2));
    return;
  }
  const int t = (blockIdx.x - 1) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  const Tile tl = get_tile(p, t);
  tile_grads<true>(in, tl, p.starts[tl.seq + 1] - 1, coef[tl.seq], dlogp, lane);
}

// ---------------------------------------------------------------- policy loss

namespace {

// The sequence in [lo, hi] that holds row r: the last one that starts at or before it.
DSB_DEV int seq_of(const int* starts, int lo, int hi, int r) {
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (starts[mid] <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

struct RowOut {
  float pol, kl, grad;
  bool clipped;
};
// One scored row. The border tests take logp − old in 64 bits, where it is exact.
// e^u − 1 − u cancels for small u: |u| < 1 takes u²·Σ u^k / (k + 2)! (k <= 9, off by
// 2^-24), which gives e^u − 1 = u + that too. PAST: as in policy_rows4.
template <bool PAST>
DSB_DEV RowOut policy_row(const PolicyHyper& h, float lp, float old, float ref, bool has_ref,
                          float A) {
  RowOut o;
  const double d = (double)lp - (double)old;
  const float rho = expf((float)d);
  float gain = rho * A;
  if (PAST && rho == INFINITY && d < INFINITY) {
    // the product may be 0 or small: e^d = 2^k · 2^f, k last
    const double t = d * 1.4426950408889634074, k = rint(t);
    gain = ldexpf(exp2f((float)(t - k)) * A, (int)fmin(k, 1e6));
  }
  const bool high = d > h.log_high && A > 0.f, low = d < h.log_low && A < 0.f;
  o.clipped = high || low;
  o.pol = -(high ? h.high * A : low ? h.low * A : gain);
  o.grad = o.clipped ? 0.f : -gain;
  o.kl = 0.f;
  if (has_ref) {
    // with a coefficient of 0 only the KL itself is wanted, and may be infinite
    const float u = (float)((double)ref - (double)lp);
    float dkl;
    if (h.kl == DSB_KL_K3) {
      float em1, val;
      if (fabsf(u) < 1.f) {
        float q = 1.f / 39916800.f;
        q = q * u + 1.f / 3628800.f;
        q = q * u + 1.f / 362880.f;
        q = q * u + 1.f / 40320.f;
        q = q * u + 1.f / 5040.f;
        q = q * u + 1.f / 720.f;
        q = q * u + 1.f / 120.f;
        q = q * u + 1.f / 24.f;
        q = q * u + 1.f / 6.f;
        q = q * u + 0.5f;
        val = u * u * q;
        em1 = u + val;
      } else {
        em1 = expf(u) - 1.f;
        val = em1 == INFINITY ? em1 : em1 - u;
      }
      o.kl = val;
      dkl = em1;
    } else {
      o.kl = 0.5f * u * u;
      dkl = u;
    }
    if (h.kl_coef != 0.f) o.grad -= h.kl_coef * dkl;
  }
  return o;
}

struct PolicySums {
  double pol = 0.0, kl = 0.0;
  int clipped = 0, count = 0;
};
struct Rows {
  f32x4 lp, old, ref, adv;
  unsigned m;
};
// As PrefIn: what is not given is read from the log probabilities and not used.
struct PolicyIn {
  const float *logp, *old, *ref, *adv;
  const uint8_t* mask;
  bool adv_rows;
  template <bool NT = false, class K>
  DSB_DEV Rows load(int r, K k) const {
    return Rows{get4<NT>(logp, r, k), get4<NT>(old, r, k), get4<NT>(ref ? ref : logp, r, k),
                get4<NT>(adv_rows ? adv : logp, r, k),
                mask4(mask ? mask : (const uint8_t*)logp, r, k)};
  }
};
// Rows r .. r+k-1 of the batch, in sequences [lo, hi] of `starts`. weight(seq): a scored row's
// weight in the loss. PAST: the ratio may be past fp32. Where one was, the thread's policy sum is not a
// finite number and its rows are gone over again (tested in each row or group, 16 M rows take
// 1.2 to 1.4 µs more).
template <bool PAST, class K, class W>
DSB_DEV void policy_rows4(const PolicyIn& in, const int* starts, const PolicyHyper& h, int r, K k,
                          const Rows& x, int lo, int hi, bool need_seq, W&& weight, float* dlogp,
                          PolicySums& sums) {
  int seq = need_seq ? seq_of(starts, lo, hi, r) : 0;
  int end = need_seq ? starts[seq + 1] : 0;
  const unsigned m = bytes4(x.m);
  f32x4 g = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= k) break;
    if (need_seq)
      while (r + i >= end) end = starts[++seq + 1];
    if (in.mask ? m >> i & 1 : r + i + 1 < end) {
      const RowOut o = policy_row<PAST>(h, x.lp[i], x.old[i], x.ref[i], in.ref != nullptr,
                                        in.adv_rows ? x.adv[i] : in.adv[seq]);
      const float w = weight(seq);
      g[i] = w * o.grad * (float)h.grad_scale;
      sums.pol += (double)w * (double)o.pol;
      sums.kl += (double)w * (double)o.kl;
      sums.clipped += o.clipped;
      ++sums.count;
    }
  }
  put4(dlogp, r, k, g);
}

// {loss, policy, kl, clipped share}
DSB_DEV void policy_out(float* out, const PolicyHyper& h, double pol, double kl, double clipped,
                        double count) {
  out[0] = (float)(h.kl_coef != 0.f ? pol + (double)h.kl_coef * kl : pol);
  out[1] = (float)pol;
  out[2] = (float)kl;
  out[3] = count > 0 ? (float)(clipped / count) : 0.f;
}

}  // namespace

__global__ __launch_bounds__(1024) void policy_small_kernel(PolicyIn in, dsb_pack_plan p,
                                                            PolicyHyper h, bool need_seq,
                                                            float* out, float* dlogp) {
  __shared__ int cnt[kSmallSeqs], starts[kSmallSeqs + 1];
  __shared__ double red[16 * 4];
  __shared__ int total_s, nonempty_s;
  const int tid = threadIdx.x;
  // a thread's groups, tid and tid + 1024, are on their way while the sequences are counted;
  // the rows of the last group (fewer than 4) are one thread's
  Rows x[2];
  int left[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 4 * (tid + 1024 * j);
    left[j] = min(max(p.n - r, 0), 4);
    if (left[j] == 4)
      x[j] = in.load(r, Int<4>{});
    else if (left[j] > 0)
      x[j] = in.load(r, left[j]);
  }
  if (need_seq)
    for (int s = tid; s <= p.nseq; s += 1024) starts[s] = p.starts[s];
  if (tid == 0) total_s = nonempty_s = 0;
  const bool by_seq = h.reduction == DSB_REDUCE_SEQUENCE;
  double total = p.npred, nonempty = p.nonempty;
  if (by_seq && in.mask)
    for (int s = tid; s < p.nseq; s += 1024) cnt[s] = 0;
  __syncthreads();
  if (by_seq && in.mask) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 4 * (tid + 1024 * j);
      const unsigned on = left[j] > 0 ? bytes4(x[j].m) : 0;
      if (!on) continue;
      int s = seq_of(starts, 0, p.nseq - 1, r);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (on >> i & 1) {
          while (r + i >= starts[s + 1]) ++s;
          if (atomicAdd(&cnt[s], 1) == 0) atomicAdd(&nonempty_s, 1);
        }
    }
    __syncthreads();
    nonempty = nonempty_s;
  } else if (by_seq) {
    for (int s = tid; s < p.nseq; s += 1024) cnt[s] = max(starts[s + 1] - starts[s] - 1, 0);
    __syncthreads();
  } else if (h.reduction == DSB_REDUCE_TOKEN && in.mask) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) c += left[j] > 0 ? __popc(bytes4(x[j].m)) : 0;
    c = wave_sumi(c);
    if ((tid & 63) == 0 && c) atomicAdd(&total_s, c);
    __syncthreads();
    total = total_s;
  }
  const float all = h.reduction == DSB_REDUCE_TOKEN ? (float)(1.0 / fmax(total, 1.0))
                                                    : (float)h.inv_divisor;
  auto weight = [&](int s) {
    return by_seq ? (float)(1.0 / ((double)max(cnt[s], 1) * fmax(nonempty, 1.0))) : all;
  };
  PolicySums sums;
  auto rows = [&](auto past) {
    constexpr bool PAST = decltype(past)::value;
    sums = PolicySums{};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 4 * (tid + 1024 * j);
      if (left[j] == 4)
        policy_rows4<PAST>(in, starts, h, r, Int<4>{}, x[j], 0, p.nseq - 1, need_seq, weight, dlogp,
                           sums);
      else if (left[j] > 0)
        policy_rows4<PAST>(in, starts, h, r, left[j], x[j], 0, p.nseq - 1, need_seq, weight, dlogp,
                           sums);
    }
  };
  rows(std::false_type{});
  if (!(fabs(sums.pol) < INFINITY)) rows(std::true_type{});
  double v[4] = {sums.pol, sums.kl, (double)sums.clipped, (double)sums.count};
  block_sums<1024>(v, red);
  if (tid == 0) policy_out(out, h, v[0], v[1], v[2], v[3]);
}

// Scored rows of the mask: one count per block, blocks striding over the rows 16 at a time.
__global__ __launch_bounds__(256) void count_rows_kernel(const uint8_t* mask, int n, int* counts) {
  typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(1)));
  __shared__ double red[4];
  const int groups = n >> 4, stride = 256 * gridDim.x;
  int c = 0;
  for (int g = blockIdx.x * 256 + threadIdx.x; g < groups; g += 4 * stride) {
    u32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      v[u] = *reinterpret_cast<const u32x4u*>(mask + 16L * min((long)g + (long)u * stride, groups - 1L));
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        c += (long)g + (long)u * stride < groups ? __popc(bytes4(v[u][i])) : 0;
  }
  if (blockIdx.x == 0 && (int)threadIdx.x < (n & 15)) c += mask[16 * groups + threadIdx.x] != 0;
  const double t = block_sumd<256>((double)c, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)t;
}

// A wave per tile: its scored rows.
__global__ __launch_bounds__(256) void count_tiles_kernel(const uint8_t* mask, dsb_pack_plan p,
                                                          int* counts) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  const Tile tl = get_tile(p, t);
  int c = 0;
  for_rows<64, 4>(
      tl.r0, tl.r1, lane, [&](int r, auto k) { return mask4(mask, r, k); },
      [&](int, auto, unsigned x) { c += __popc(bytes4(x)); });
  c = wave_sumi(c);
  if (lane == 0) counts[t] = c;
}

// A thread per sequence: 1 / its scored rows, and how many sequences of the block have any.
__global__ __launch_bounds__(256) void seq_weights_kernel(bool masked, dsb_pack_plan p,
                                                          const int* tile_counts, double* inv,
                                                          int* nonempty) {
  __shared__ double red[4];
  const int s = blockIdx.x * 256 + threadIdx.x;
  int c = 0;
  if (s < p.nseq) {
    if (masked)
      for (int t = p.seq_tile[s]; t < p.seq_tile[s + 1]; ++t) c += tile_counts[t];
    else
      c = max(p.starts[s + 1] - p.starts[s] - 1, 0);
    inv[s] = 1.0 / max(c, 1);
  }
  const double t = block_sumd<256>(c > 0 ? 1.0 : 0.0, red);
  if (threadIdx.x == 0) nonempty[blockIdx.x] = (int)t;
}

struct PolicyPart {
  double pol, kl;
  int clipped, count;
};

// A block per DSB_CHUNK_ROWS rows. 16 M rows in 4096 sequences, with a reference, all launches:
// token mean, advantages by row 70 µs, by sequence 74; sequence mean 86 and 84 (two launches more,
// and each group's sequence is searched for in memory). parts: the counts whose sum is the number of scored
// rows (token) or of sequences with some (sequence); none where the host knows it.
__global__ __launch_bounds__(256) void policy_kernel(PolicyIn in, dsb_pack_plan p, PolicyHyper h,
                                                     bool need_seq, const int* parts, int nparts,
                                                     const double* inv, float* dlogp,
                                                     PolicyPart* partial) {
  __shared__ double red[4], red4[4 * 4];
  double total = h.reduction == DSB_REDUCE_SEQUENCE ? p.nonempty : p.npred;
  if (parts) {
    double c = 0.0;
#pragma unroll 2
    for (int i = threadIdx.x; i < nparts; i += 256) c += parts[i];
    total = block_sumd<256>(c, red);
  }
  const double itot = 1.0 / fmax(total, 1.0);
  const float all = h.reduction == DSB_REDUCE_TOKEN ? (float)itot : (float)h.inv_divisor;
  const int lo = p.chunk_seq[blockIdx.x], hi = p.chunk_seq[blockIdx.x + 1];
  auto weight = [&](int s) {
    return h.reduction == DSB_REDUCE_SEQUENCE ? (float)(inv[s] * itot) : all;
  };
  PolicySums sums;
  const int r0 = blockIdx.x * kChunkRows, r1 = min(p.n - r0, kChunkRows) + r0;
  // rows are read once, past the caches (16 M rows with a reference and advantages by row: 80.9
  // → 70.6 µs; the gradients past them too 72.3)
  auto rows = [&](auto past) {
    sums = PolicySums{};
    for_rows<256, 2>(
        r0, r1, threadIdx.x, [&](int r, auto k) { return in.load<true>(r, k); },
        [&](int r, auto k, const Rows& x) {
          policy_rows4<decltype(past)::value>(in, p.starts, h, r, k, x, lo, hi, need_seq, weight,
                                              dlogp, sums);
        });
  };
  rows(std::false_type{});
  if (!(fabs(sums.pol) < INFINITY)) rows(std::true_type{});
  double v[4] = {sums.pol, sums.kl, (double)sums.clipped, (double)sums.count};
  block_sums<256>(v, red4);
  if (threadIdx.x == 0)
    partial[blockIdx.x] = PolicyPart{v[0], v[1], (int)v[2], (int)v[3]};
}

__global__ __launch_bounds__(1024) void policy_total_kernel(const PolicyPart* partial, int nparts,
                                                            PolicyHyper h, float* out) {
  __shared__ double red[16 * 4];
  double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (int i = threadIdx.x; i < nparts; i += 1024) {
    const PolicyPart q = partial[i];
    v[0] += q.pol;
    v[1] += q.kl;
    v[2] += q.clipped;
    v[3] += q.count;
  }
  block_sums<1024>(v, red);
  if (threadIdx.x == 0) policy_out(out, h, v[0], v[1], v[2], v[3]);
}

// ---------------------------------------------------------------- launches

namespace {

constexpr int kCountBlocks = 512;

struct LossWork {
  double* sums;      // by tile
  int* counts;       // by tile, or by counting block
  double* seq;       // by sequence
  double* partial;   // by block of pairs
  int* nonempty;     // by block of sequences
  PolicyPart* part;  // by chunk
};
LossWork loss_layout(const dsb_pack_plan& p, void* base, int64_t* bytes) {
  int64_t at = 0;
  auto take = [&](int64_t n) {
    char* r = base ? (char*)base + at : nullptr;
    at += (n + 255) / 256 * 256;
    return r;
  };
  const int64_t sb = (p.nseq + 255) / 256 + 1;
  LossWork w;
  w.sums = (double*)take(8 * (int64_t)p.ntiles);
  w.counts = (int*)take(4 * std::max<int64_t>(p.ntiles, kCountBlocks));
  w.seq = (double*)take(8 * (int64_t)p.nseq);
  w.partial = (double*)take(8 * sb);
  w.nonempty = (int*)take(4 * sb);
  w.part = (PolicyPart*)take((int64_t)sizeof(PolicyPart) * ((p.n + kChunkRows - 1) / kChunkRows));
  *bytes = at;
  return w;
}

bool small_batch(const dsb_pack_plan& p) {
  return p.n <= kSmallRows && p.ntiles <= kSmallTiles && p.nseq <= kSmallSeqs;
}

}  // namespace

int64_t loss_bytes(const dsb_pack_plan& p) {
  if (small_batch(p)) return 0;
  int64_t b;
  loss_layout(p, nullptr, &b);
  return b;
}

hipError_t next_token_labels(const int64_t* ids, const uint8_t* mask, const dsb_pack_plan& p,
                             int64_t* labels, uint8_t* rows, hipStream_t s) {
  if (p.ntiles > 0)
    hipLaunchKernelGGL(labels_kernel, dim3((p.ntiles + 3) / 4), dim3(256), 0, s, ids, mask, p,
                       labels, rows);
  return hipGetLastError();
}

hipError_t preference_loss(const float* logp, const float* ref, const uint8_t* mask,
                           const dsb_pack_plan& p, const PrefHyper& h, float* loss, float* rewards,
                           float* dlogp, void* work, hipStream_t s) {
  const PrefIn in{logp, ref, mask};
  if (small_batch(p)) {
    hipLaunchKernelGGL(pref_small_kernel, dim3(1), dim3(1024), 0, s, in, p, h, loss, rewards, dlogp);
    return hipGetLastError();
  }
  int64_t bytes;
  const LossWork w = loss_layout(p, work, &bytes);
  if (p.longest <= DSB_TILE_ROWS) {
    const int pairs = p.nseq / 2;
    auto go = [&](auto nt, auto nb) {
      constexpr int NT = decltype(nt)::value, NB = decltype(nb)::value;
      hipLaunchKernelGGL((pref_pair_kernel<NT, NB>), dim3((pairs + NB / NT - 1) / (NB / NT)),
                         dim3(NB), 0, s, in, p, h, rewards, dlogp, w.seq);
    };
    // Four waves to a pair up to where they fill the device (8192 waves), then two, then one.
    // µs by waves per pair 4 / 2 / 1 and in three launches by tile, ragged sequences: 256
    // pairs of 1000 rows 7.3 / 8.6 / 10.9 / 9.2, 2000 of 4000 26.7 / 28.5 / 35.1 / 29.1, 4096 of
    // 1024 19.8 / 17.2 / 19.0 / 20.4, 16384 of 256 42.4 / 30.1 / 26.9 / 33.0.
    if (pairs <= 2048)
      go(Int<256>{}, Int<256>{});
    else if (pairs <= 8192)
      go(Int<128>{}, Int<512>{});
    else
      go(Int<64>{}, Int<256>{});
    hipLaunchKernelGGL(pref_total_kernel, dim3(1), dim3(1024), 0, s, w.seq, pairs, loss);
    return hipGetLastError();
  }
  const int tb = (p.ntiles + 3) / 4, pb = (p.nseq / 2 + 255) / 256;
  if (tb > 0)
    hipLaunchKernelGGL(pref_sums_kernel, dim3(tb), dim3(256), 0, s, in, p, w.sums, w.counts);
  float* coef = (float*)w.seq;
  hipLaunchKernelGGL(pref_pairs_kernel, dim3(pb), dim3(256), 0, s, p, h, w.sums, w.counts, rewards,
                     coef, w.partial);
  hipLaunchKernelGGL(pref_grads_kernel, dim3(1 + tb), dim3(256), 0, s, in, p, coef, w.partial, pb, loss,
                     dlogp);
  return hipGetLastError();
}

hipError_t policy_loss(const float* logp, const float* old, const float* ref, const float* adv,
                       const uint8_t* mask, const dsb_pack_plan& p, const PolicyHyper& h, float* out,
                       float* dlogp, void* work, hipStream_t s) {
  const PolicyIn in{logp, old, ref, adv, mask, h.adv_rows};
  const bool by_seq = h.reduction == DSB_REDUCE_SEQUENCE, need_seq = by_seq || !h.adv_rows || !mask;
  if (small_batch(p)) {
    hipLaunchKernelGGL(policy_small_kernel, dim3(1), dim3(1024), 0, s, in, p, h, need_seq, out,
                       dlogp);
    return hipGetLastError();
  }
  int64_t bytes;
  const LossWork w = loss_layout(p, work, &bytes);
  const int* parts = nullptr;
  int nparts = 0;
  if (by_seq) {
    nparts = (p.nseq + 255) / 256;
    if (mask && p.ntiles > 0)
      hipLaunchKernelGGL(count_tiles_kernel, dim3((p.ntiles + 3) / 4), dim3(256), 0, s, mask, p,
                         w.counts);
    hipLaunchKernelGGL(seq_weights_kernel, dim3(nparts), dim3(256), 0, s, mask != nullptr, p,
                       w.counts, w.seq, w.nonempty);
    parts = w.nonempty;
  } else if (h.reduction == DSB_REDUCE_TOKEN && mask) {
    nparts = kCountBlocks;
    hipLaunchKernelGGL(count_rows_kernel, dim3(nparts), dim3(256), 0, s, mask, p.n, w.counts);
    parts = w.counts;
  }
  const int chunks = (p.n + kChunkRows - 1) / kChunkRows;
  if (chunks > 0)
    hipLaunchKernelGGL(policy_kernel, dim3(chunks), dim3(256), 0, s, in, p, h, need_seq, parts,
                       nparts, w.seq, dlogp, w.part);
  hipLaunchKernelGGL(policy_total_kernel, dim3(1), dim3(1024), 0, s, w.part, chunks, h, out);
  return hipGetLastError();
}

}  // namespace dsb
