// Losses of training from feedback over a packing of sequences, each with its
// gradient with respect to the rows' log probabilities: a preference loss over
// pairs of sequences and a clipped policy loss with a KL term, and the labels that
// the log probabilities are taken of.
//
// Both are bound by their bytes (9 to 21 a row) where the batch is large and by
// launches where it is small, so:
//   * a batch of few rows is one launch of one workgroup, the sums by sequence in
//     LDS; a large one takes three (sums by tile; by pair or sequence; gradients,
//     with the loss), or two where no mask has to be counted;
//   * a row's values are read four at a time where they are aligned, and written
//     once, the gradient's zeros on unscored rows included;
//   * sums over rows are held in 64 bits and added in a fixed order.
// The value of an unscored row is never used in arithmetic: it is replaced by 0
// first, so infinities and NaN there do not spread.
#include <algorithm>

#include "feedback.h"

namespace dsb {

namespace {

constexpr int kChunkRows = DSB_CHUNK_ROWS;
// Batches of one workgroup: at most this many rows, tiles and sequences.
constexpr int kSmallRows = 8192, kSmallTiles = 64, kSmallSeqs = 512;

DSB_DEV double wave_sumd(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// Sum over a block of NT threads; red: NT / 64 doubles.
template <int NT>
DSB_DEV double block_sumd(double v, double* red) {
  v = wave_sumd(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t += red[i];
  __syncthreads();
  return t;
}

// Rows r .. r+3 (r a multiple of 4) of an fp32 array of n rows.
DSB_DEV f32x4 rows4(const float* p, int r, int n, bool vec) {
  if (vec && r + 4 <= n) return *reinterpret_cast<const f32x4*>(p + r);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + i < n) o[i] = p[r + i];
  return o;
}
// Which of rows r .. r+3 a mask of n rows sets (bits 0 .. 3).
DSB_DEV unsigned mask4(const uint8_t* p, int r, int n, bool vec) {
  unsigned o = 0;
  if (vec && r + 4 <= n) {
    const unsigned v = *reinterpret_cast<const unsigned*>(p + r);
#pragma unroll
    for (int i = 0; i < 4; ++i) o |= (v >> (8 * i) & 255u ? 1u : 0u) << i;
    return o;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (r + i < n && p[r + i]) o |= 1u << i;
  return o;
}
// Bits of rows r .. r+3 that lie in [a, b).
DSB_DEV unsigned within4(int r, int a, int b) {
  unsigned o = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) o |= (r + i >= a && r + i < b ? 1u : 0u) << i;
  return o;
}
DSB_DEV void put4(float* p, int r, unsigned which, bool vec, f32x4 v) {
  if (vec && which == 15u) {
    *reinterpret_cast<f32x4*>(p + r) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (which >> i & 1) p[r + i] = v[i];
}
DSB_DEV bool al16(const void* p) { return ((unsigned long)p & 15) == 0; }
DSB_DEV bool al4(const void* p) { return ((unsigned long)p & 3) == 0; }

struct Tile {
  int r0, r1, seq;
};
DSB_DEV Tile get_tile(const dsb_pack_plan& p, int t) {
  const int4 v = reinterpret_cast<const int4*>(p.tiles)[t];
  return Tile{v.x, v.y, v.z};
}
// Scored rows among r .. r+3 of the tile.
DSB_DEV unsigned scored4(const dsb_pack_plan& p, const Tile& t, int r, const uint8_t* mask,
                         bool mvec) {
  if (mask) return mask4(mask, r, p.n, mvec) & within4(r, t.r0, t.r1);
  return within4(r, t.r0, min(t.r1, p.starts[t.seq + 1] - 1));
}

// One wave: Σ (logp − ref) and the count over the scored rows of a tile.
DSB_DEV double tile_sum(const dsb_pack_plan& p, const Tile& t, const float* logp, const float* ref,
                        const uint8_t* mask, int lane, int* count) {
  const bool v0 = al16(logp), v1 = al16(ref), vm = al4(mask);
  double s = 0.0;
  int c = 0;
#pragma unroll 4
  for (int r = (t.r0 & ~3) + 4 * lane; r < t.r1; r += 256) {
    const unsigned on = scored4(p, t, r, mask, vm);
    const f32x4 a = rows4(logp, r, p.n, v0);
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (ref) b = rows4(ref, r, p.n, v1);
#pragma unroll
    for (int i = 0; i < 4; ++i) s += on >> i & 1 ? (double)a[i] - (double)b[i] : 0.0;
    c += __popc(on);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
  *count = c;
  return wave_sumd(s);
}

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
    o.loss = (1.0 - h.smooth) * (fmax(-z, 0.0) + l) + h.smooth * (fmax(z, 0.0) + l);
    g = h.beta * (h.smooth * up - (1.0 - h.smooth) * down);
    if (z != z) o.loss = z;
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

// One wave: a tile's rows of the gradient.
DSB_DEV void tile_grads(const dsb_pack_plan& p, const Tile& t, float coef, const uint8_t* mask,
                        float* dlogp, int lane) {
  const bool vd = al16(dlogp), vm = al4(mask);
#pragma unroll 4
  for (int r = (t.r0 & ~3) + 4 * lane; r < t.r1; r += 256) {
    const unsigned on = scored4(p, t, r, mask, vm);
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = on >> i & 1 ? coef : 0.f;
    put4(dlogp, r, within4(r, t.r0, t.r1), vd, v);
  }
}

}  // namespace

// ---------------------------------------------------------------- labels

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

__global__ __launch_bounds__(1024) void pref_small_kernel(const float* logp, const float* ref,
                                                          const uint8_t* mask, dsb_pack_plan p,
                                                          PrefHyper h, float* loss, float* rewards,
                                                          float* dlogp) {
  __shared__ double sums[kSmallTiles], red[16];
  __shared__ int counts[kSmallTiles];
  __shared__ float coef[kSmallSeqs];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int t = wave; t < p.ntiles; t += 16) {
    int c;
    const double s = tile_sum(p, get_tile(p, t), logp, ref, mask, lane, &c);
    if (lane == 0) {
      sums[t] = s;
      counts[t] = c;
    }
  }
  __syncthreads();
  const int npairs = p.nseq / 2;
  double total = 0.0;
  for (int i = threadIdx.x; i < npairs; i += 1024) {
    double s[2] = {0.0, 0.0};
    int c[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      for (int t = p.seq_tile[2 * i + k]; t < p.seq_tile[2 * i + k + 1]; ++t) {
        s[k] += sums[t];
        c[k] += counts[t];
      }
    const Pair o = pair_eval(h, npairs, s, c);
    total += o.loss;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      rewards[2 * i + k] = o.reward[k];
      coef[2 * i + k] = o.coef[k];
    }
  }
  total = block_sumd<1024>(total, red);  // its barriers publish coef too
  if (threadIdx.x == 0) *loss = (float)(total / npairs);
  for (int t = wave; t < p.ntiles; t += 16) {
    const Tile tl = get_tile(p, t);
    tile_grads(p, tl, coef[tl.seq], mask, dlogp, lane);
  }
}

__global__ __launch_bounds__(256) void pref_sums_kernel(const float* logp, const float* ref,
                                                        const uint8_t* mask, dsb_pack_plan p,
                                                        double* sums, int* counts) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  int c;
  const double s = tile_sum(p, get_tile(p, t), logp, ref, mask, lane, &c);
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
  const int i = blockIdx.x * 256 + threadIdx.x, npairs = p.nseq / 2;
  double l = 0.0;
  if (i < npairs) {
    double s[2] = {0.0, 0.0};
    int c[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      for (int t = p.seq_tile[2 * i + k]; t < p.seq_tile[2 * i + k + 1]; ++t) {
        s[k] += sums[t];
        c[k] += counts[t];
      }
    const Pair o = pair_eval(h, npairs, s, c);
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
__global__ __launch_bounds__(256) void pref_grads_kernel(const uint8_t* mask, dsb_pack_plan p,
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
  tile_grads(p, tl, coef[tl.seq], mask, dlogp, lane);
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
// 2^-24), which gives e^u − 1 = u + that too.
DSB_DEV RowOut policy_row(const PolicyHyper& h, float lp, float old, float ref, bool has_ref,
                          float A) {
  RowOut o;
  const double d = (double)lp - (double)old;
  const float rho = expf((float)d), gain = rho * A;
  const bool high = d > h.log_high && A > 0.f, low = d < h.log_low && A < 0.f;
  o.clipped = high || low;
  o.pol = -(high ? h.high * A : low ? h.low * A : gain);
  o.grad = o.clipped ? 0.f : -gain;
  o.kl = 0.f;
  if (has_ref) {
    const float u = (float)((double)ref - (double)lp);
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
        val = em1 - u;
      }
      o.kl = val;
      o.grad -= h.kl_coef * em1;
    } else {
      o.kl = 0.5f * u * u;
      o.grad -= h.kl_coef * u;
    }
  }
  return o;
}

struct PolicyIn {
  const float *logp, *old, *ref, *adv;
  const uint8_t* mask;
};
struct PolicySums {
  double pol = 0.0, kl = 0.0;
  int clipped = 0, count = 0;
};

// Rows r .. r+3 of the batch, in sequences [lo, hi]. weight(seq): a scored row's weight
// in the loss.
template <class W>
DSB_DEV void policy_rows4(const PolicyIn& in, const dsb_pack_plan& p, const PolicyHyper& h, int r,
                          int lo, int hi, bool need_seq, W&& weight, float* dlogp,
                          PolicySums& sums) {
  const f32x4 a = rows4(in.logp, r, p.n, al16(in.logp)), b = rows4(in.old, r, p.n, al16(in.old));
  f32x4 c = {0.f, 0.f, 0.f, 0.f}, A = c;
  if (in.ref) c = rows4(in.ref, r, p.n, al16(in.ref));
  if (h.adv_rows) A = rows4(in.adv, r, p.n, al16(in.adv));
  unsigned on = 15u;
  if (in.mask) on = mask4(in.mask, r, p.n, al4(in.mask));
  int seq = need_seq ? seq_of(p.starts, lo, hi, r) : 0;
  int end = need_seq ? p.starts[seq + 1] : 0;
  f32x4 g = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (r + i >= p.n) break;
    if (need_seq)
      while (r + i >= end) end = p.starts[++seq + 1];
    const bool live = in.mask ? on >> i & 1 : r + i + 1 < end;
    if (live) {
      const RowOut o = policy_row(h, a[i], b[i], c[i], in.ref != nullptr,
                                  h.adv_rows ? A[i] : in.adv[seq]);
      const float w = weight(seq);
      g[i] = w * o.grad * (float)h.grad_scale;
      sums.pol += (double)w * (double)o.pol;
      sums.kl += (double)w * (double)o.kl;
      sums.clipped += o.clipped;
      ++sums.count;
    }
  }
  put4(dlogp, r, within4(r, 0, p.n), al16(dlogp), g);
}

// {loss, policy, kl, clipped share}
DSB_DEV void policy_out(float* out, const PolicyHyper& h, double pol, double kl, double clipped,
                        double count) {
  out[0] = (float)(pol + (double)h.kl_coef * kl);
  out[1] = (float)pol;
  out[2] = (float)kl;
  out[3] = count > 0 ? (float)(clipped / count) : 0.f;
}

}  // namespace

__global__ __launch_bounds__(1024) void policy_small_kernel(PolicyIn in, dsb_pack_plan p,
                                                            PolicyHyper h, bool need_seq,
                                                            float* out, float* dlogp) {
  __shared__ int cnt[kSmallSeqs + 1];
  __shared__ double red[16];
  __shared__ int total_s, nonempty_s;
  const int tid = threadIdx.x;
  double total = p.npred, nonempty = p.nonempty;
  if (h.reduction == DSB_REDUCE_SEQUENCE) {
    for (int s = tid; s < p.nseq; s += 1024)
      cnt[s] = in.mask ? 0 : max(p.starts[s + 1] - p.starts[s] - 1, 0);
    if (tid == 0) nonempty_s = 0;
    __syncthreads();
    if (in.mask) {
      for (int r = 4 * tid; r < p.n; r += 4096) {
        const unsigned on = mask4(in.mask, r, p.n, al4(in.mask));
        if (!on) continue;
        int s = seq_of(p.starts, 0, p.nseq - 1, r);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (on >> i & 1) {
            while (r + i >= p.starts[s + 1]) ++s;
            atomicAdd(&cnt[s], 1);
          }
      }
      __syncthreads();
      for (int s = tid; s < p.nseq; s += 1024)
        if (cnt[s]) atomicAdd(&nonempty_s, 1);
      __syncthreads();
      nonempty = nonempty_s;
    }
  } else if (h.reduction == DSB_REDUCE_TOKEN && in.mask) {
    if (tid == 0) total_s = 0;
    __syncthreads();
    int c = 0;
    for (int r = 4 * tid; r < p.n; r += 4096) c += __popc(mask4(in.mask, r, p.n, al4(in.mask)));
    atomicAdd(&total_s, c);
    __syncthreads();
    total = total_s;
  }
  const float all = h.reduction == DSB_REDUCE_TOKEN ? (float)(1.0 / fmax(total, 1.0))
                                                    : (float)h.inv_divisor;
  PolicySums sums;
  for (int r = 4 * tid; r < p.n; r += 4096) {
    auto weight = [&](int s) {
      return h.reduction == DSB_REDUCE_SEQUENCE
                 ? (float)(1.0 / ((double)max(cnt[s], 1) * fmax(nonempty, 1.0)))
                 : all;
    };
    policy_rows4(in, p, h, r, 0, p.nseq - 1, need_seq, weight, dlogp, sums);
  }
  const double pol = block_sumd<1024>(sums.pol, red), kl = block_sumd<1024>(sums.kl, red);
  const double cl = block_sumd<1024>(sums.clipped, red), n = block_sumd<1024>(sums.count, red);
  if (tid == 0) policy_out(out, h, pol, kl, cl, n);
}

// Scored rows of the mask: one count per block of 256, blocks striding over the rows.
__global__ __launch_bounds__(256) void count_rows_kernel(const uint8_t* mask, int n, int* counts) {
  __shared__ double red[4];
  const bool vec = al16(mask);
  int c = 0;
  for (long r = 16 * ((long)blockIdx.x * 256 + threadIdx.x); r < n; r += 16L * 256 * gridDim.x) {
    if (vec && r + 16 <= n) {
      const u32x4 v = ldg128(mask + r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        unsigned x = v[i];  // a bit per nonzero byte
        x |= x >> 4;
        x |= x >> 2;
        x |= x >> 1;
        c += __popc(x & 0x01010101u);
      }
    } else {
      for (int i = 0; i < 16 && r + i < n; ++i) c += mask[r + i] != 0;
    }
  }
  const double t = block_sumd<256>((double)c, red);
  if (threadIdx.x == 0) counts[blockIdx.x] = (int)t;
}

// A wave per tile: its scored rows.
__global__ __launch_bounds__(256) void count_tiles_kernel(const uint8_t* mask, dsb_pack_plan p,
                                                          int* counts) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (t >= p.ntiles) return;
  const Tile tl = get_tile(p, t);
  const bool vm = al4(mask);
  int c = 0;
#pragma unroll 4
  for (int r = (tl.r0 & ~3) + 4 * lane; r < tl.r1; r += 256)
    c += __popc(mask4(mask, r, p.n, vm) & within4(r, tl.r0, tl.r1));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
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

// A block per DSB_CHUNK_ROWS rows. parts: the counts whose sum is the number of scored
// rows (token) or of sequences with some (sequence); none where the host knows it.
__global__ __launch_bounds__(256) void policy_kernel(PolicyIn in, dsb_pack_plan p, PolicyHyper h,
                                                     bool need_seq, const int* parts, int nparts,
                                                     const double* inv, float* dlogp,
                                                     PolicyPart* partial) {
  __shared__ double red[4];
  double total = h.reduction == DSB_REDUCE_SEQUENCE ? p.nonempty : p.npred;
  if (parts) {
    double c = 0.0;
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
#pragma unroll
  for (int k = 0; k < kChunkRows / 1024; ++k) {
    const int r = blockIdx.x * kChunkRows + k * 1024 + 4 * threadIdx.x;
    if (r < p.n) policy_rows4(in, p, h, r, lo, hi, need_seq, weight, dlogp, sums);
  }
  const double pol = block_sumd<256>(sums.pol, red), kl = block_sumd<256>(sums.kl, red);
  const double cl = block_sumd<256>(sums.clipped, red), n = block_sumd<256>(sums.count, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = PolicyPart{pol, kl, (int)cl, (int)n};
}

__global__ __launch_bounds__(1024) void policy_total_kernel(const PolicyPart* partial, int nparts,
                                                            PolicyHyper h, float* out) {
  __shared__ double red[16];
  double pol = 0.0, kl = 0.0, cl = 0.0, n = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 1024) {
    const PolicyPart q = partial[i];
    pol += q.pol;
    kl += q.kl;
    cl += q.clipped;
    n += q.count;
  }
  pol = block_sumd<1024>(pol, red);
  kl = block_sumd<1024>(kl, red);
  cl = block_sumd<1024>(cl, red);
  n = block_sumd<1024>(n, red);
  if (threadIdx.x == 0) policy_out(out, h, pol, kl, cl, n);
}

// ---------------------------------------------------------------- launches

namespace {

constexpr int kCountBlocks = 256;

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
  *bytes = at + 256;
  return w;
}

bool small_batch(const dsb_pack_plan& p) {
  return p.n <= kSmallRows && p.ntiles <= kSmallTiles && p.nseq <= kSmallSeqs;
}

}  // namespace

int64_t loss_bytes(const dsb_pack_plan& p) {
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
  if (small_batch(p)) {
    hipLaunchKernelGGL(pref_small_kernel, dim3(1), dim3(1024), 0, s, logp, ref, mask, p, h, loss,
                       rewards, dlogp);
    return hipGetLastError();
  }
  int64_t bytes;
  const LossWork w = loss_layout(p, work, &bytes);
  const int tb = (p.ntiles + 3) / 4, pb = (p.nseq / 2 + 255) / 256;
  if (tb > 0)
    hipLaunchKernelGGL(pref_sums_kernel, dim3(tb), dim3(256), 0, s, logp, ref, mask, p, w.sums,
                       w.counts);
  float* coef = (float*)w.seq;
  hipLaunchKernelGGL(pref_pairs_kernel, dim3(pb), dim3(256), 0, s, p, h, w.sums, w.counts, rewards,
                     coef, w.partial);
  hipLaunchKernelGGL(pref_grads_kernel, dim3(1 + tb), dim3(256), 0, s, mask, p, coef, w.partial, pb,
                     loss, dlogp);
  return hipGetLastError();
}

hipError_t policy_loss(const float* logp, const float* old, const float* ref, const float* adv,
                       const uint8_t* mask, const dsb_pack_plan& p, const PolicyHyper& h, float* out,
                       float* dlogp, void* work, hipStream_t s) {
  const PolicyIn in{logp, old, ref, adv, mask};
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
