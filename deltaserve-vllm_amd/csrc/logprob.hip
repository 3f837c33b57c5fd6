// Log probabilities of labels through the LM head, and their gradient:
//   x_v = h·W_v, other = log Σ_{v ≠ t} exp(x_v), logp = −log(1 + exp(other − x_t))
//   dH = g·(W_t − Σ_v p_v·W_v) = g·(1 − p_t)·(W_t − Σ_{v ≠ t} q_v·W_v),
//   q_v = exp(x_v − other), 1 − p_t = 1 − exp(logp)
// for the label t and upstream gradient g of each row. The label's term is kept
// out of the sums, so both hold their relative precision where p_t is near 1.
//
// Rows that are not scored (a prompt's, a sequence's last) and, in the backward,
// rows with g = 0 (clipped) or 1 − p_t = 0 are left out of the products: their
// indices are compacted on the device, the others' rows copied together (n·D of
// traffic against 2·D·V flops a row), and the products run over the device's count.
// The forward is one product over the whole vocabulary whose epilogue keeps only a
// sum per row and run of columns: no logits are stored. The backward's softmax
// reference, `other`, is exact and known, so its vocabulary chunks need no
// rescaling between the logits product and the dH product (head.hip).
#include "feedback.h"
#include "gemm_nt.h"

namespace dsb {

namespace {

// Limit on a run's Σ exp(logit − ref), as for the cross-entropy head: above it
// (a logit more than about 40 over the label's) the run takes its own maximum.
constexpr float kRunLimit = 0x1p57f;

// Probabilities held at a time (1 GiB of bf16), and the most K slices of the dH product.
constexpr long kProbElems = 1L << 29;
constexpr int kMaxSlices = 8;

struct LPStat {
  float ref, sum;  // Σ exp(logit − ref) over a run, the label left out
};

// Per run of TN columns and row: LPStat into stats[run · cap + m] (the 16 rows of
// a fragment are neighbours, so a store is one 128-byte line) and the label's logit
// into tgt[m]. A lane holds 4·FN columns of a row.
struct EpiLogProb {
  LPStat* stats;
  int cap, V;
  const float* ref;
  const int* labels;
  float* tgt;
  template <int FM, int FN, int WM, int WN>
  DSB_DEV void run(const f32x4 (&acc)[FM][FN], int mw, int nw, int M, int lane, int,
                   void*) const {
    constexpr int TN = FN * 16;
    if (nw >= V || mw >= M) return;
    const int l16 = lane & 15, lq = lane >> 4;
    const bool whole = nw + TN <= V;
    LPStat* out = stats + (long)(nw / TN) * cap;
    float ref0[FM];
    int tcol[FM];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int m = min(mw + fm * 16 + l16, M - 1);
      ref0[fm] = ref[m];
      tcol[fm] = labels[m] - nw;
    }
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      if (mw + fm * 16 >= M) break;
      const float tl = (float)(tcol[fm] - 4 * lq);
      auto take = [&](float r, auto skips) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int fn = 0; fn < FN; ++fn)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float e = __expf(acc[fm][fn][i] - r);
            if (!whole) e = nw + fn * 16 + 4 * lq + i < V ? e : 0.f;
            if (decltype(skips)::value) e = (float)(fn * 16 + i) == tl ? 0.f : e;
            part[i] += e;
          }
        float v = (part[0] + part[1]) + (part[2] + part[3]);
        v += __shfl_xor(v, 16, 64);
        return LPStat{r, v + __shfl_xor(v, 32, 64)};
      };
      const int m = mw + fm * 16 + l16;
      LPStat st = take(ref0[fm], std::false_type{});
      if (__any(!(st.sum <= kRunLimit) || (unsigned)tcol[fm] < (unsigned)TN)) {
        // rare: a row with its label in the run, or past the limit
        float v = -INFINITY, xt = 0.f;
#pragma unroll
        for (int fn = 0; fn < FN; ++fn)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc[fm][fn][i];
            const bool mine = (float)(fn * 16 + i) == tl;
            if (mine) xt = x;
            v = !mine && (whole || nw + fn * 16 + 4 * lq + i < V) ? fmaxf(v, x) : v;
          }
        const int tc = tcol[fm];
        if ((unsigned)tc < (unsigned)TN && ((tc >> 2) & 3) == lq && m < M) tgt[m] = xt;
        v = fmaxf(v, __shfl_xor(v, 16, 64));
        v = fmaxf(v, __shfl_xor(v, 32, 64));
        st = take(st.sum <= kRunLimit ? st.ref : fmaxf(st.ref, v), std::true_type{});
      }
      if (lq == 0 && m < M) out[m] = st;
    }
  }
};

// The backward's probabilities of chunk [c0, c0 + Vc): P[m, j] = bf16(exp(logit − ref))
// with ref = the log-sum-exp of the row's words but the label, so each is at most 1 and
// they sum to 1, the label's as zero; columns [Vc, Nc8) as zero too. Per run of TN columns
// the sum of the rounded values goes to rsum[m · runs + run] (products with ones on the
// matrix cores). Only runs that hold a label (one in V / TN of a row's) test their columns
// for it; its exponential, which may be infinite, is left out by a select.
struct EpiProb {
  float* rsum;
  int runs;
  bf16* P;
  long ldp;
  int c0, Vc, Nc8;
  const float* ref;
  const int* labels;
  template <int FM, int FN, int WM, int WN>
  DSB_DEV void run(const f32x4 (&acc)[FM][FN], int mw, int nw, int M, int lane, int wave,
                   void* smem) const {
    constexpr int TN = FN * 16, PITCH = TN + 8, CG = TN / 8;
    if (nw >= Vc || mw >= M) return;
    const int l16 = lane & 15, lq = lane >> 4;
    const bool whole = nw + TN <= Vc;
    bf16* buf = reinterpret_cast<bf16*>(smem) + wave * 32 * PITCH;
    float ref0[FM];
    int tcol[FM];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int m = min(mw + fm * 16 + l16, M - 1);
      ref0[fm] = ref[m];
      tcol[fm] = labels[m] - (c0 + nw);
    }
#pragma unroll
    for (int b = 0; b < FM / 2; ++b) {
      if (mw + b * 32 >= M) break;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int fm = 2 * b + h;
        bf16x4 pk[FN];
        const float tl = (float)(tcol[fm] - 4 * lq);
        auto take = [&](auto skips) {
#pragma unroll
          for (int fn = 0; fn < FN; ++fn)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float e = __expf(acc[fm][fn][i] - ref0[fm]);
              if (!whole) e = nw + fn * 16 + 4 * lq + i < Vc ? e : 0.f;
              if (decltype(skips)::value) e = (float)(fn * 16 + i) == tl ? 0.f : e;
              pk[fn][i] = (bf16)e;
            }
        };
        if (__any((unsigned)tcol[fm] < (unsigned)TN))
          take(std::true_type{});
        else
          take(std::false_type{});
        f32x4 r = {0.f, 0.f, 0.f, 0.f};
        const bf16 o = (bf16)1.f;
        const bf16x8 ones = {o, o, o, o, o, o, o, o};
#pragma unroll
        for (int fn = 0; fn < FN; fn += 2)
          r = mfma16(ones, __builtin_shufflevector(pk[fn], pk[fn + 1], 0, 1, 2, 3, 4, 5, 6, 7), r);
#pragma unroll
        for (int fn = 0; fn < FN; ++fn)
          *reinterpret_cast<bf16x4*>(buf + (16 * h + l16) * PITCH + fn * 16 + 4 * lq) = pk[fn];
        const int m = mw + fm * 16 + l16;
        if (lq == 0 && m < M) rsum[(long)m * runs + (c0 + nw) / TN] = r[0];
      }
#pragma unroll
      for (int it = 0; it < 32 * CG / 64; ++it) {
        const int c = lane + 64 * it, row = c / CG, m = mw + b * 32 + row;
        const int n = nw + (c % CG) * 8;
        const u32x4 v = *reinterpret_cast<const u32x4*>(buf + row * PITCH + (c % CG) * 8);
        if (m < M && n < Nc8) stg128(P + (long)m * ldp + n, v);
      }
    }
  }
};

constexpr int lp_run(int cfg) {
  return cfg == GEMM_BIG ? 128 : cfg == GEMM_NARROW || cfg == GEMM_SKINNY ? 32 : 64;
}

// The logits products' tile: by cost, `ob` bytes stored per logit.
int lp_cfg(int n, int D, int V, double ob) {
  int best = GEMM_BIG;
  double bt = 0;
  for (int cfg = 0; cfg < kGemmCfgs; ++cfg) {
    const double c = gemm_cost(n, V, D, ob, cfg, 1);
    if (bt == 0 || c < bt) {
      bt = c;
      best = cfg;
    }
  }
  return best;
}

// Workspace pieces, 256-byte aligned; with a null base only the size is meant.
struct Carve {
  char* p;
  size_t at = 0;
  template <class T>
  T* take(size_t count) {
    T* r = p ? reinterpret_cast<T*>(p + at) : nullptr;
    at += (count * sizeof(T) + 255) / 256 * 256;
    return r;
  }
};

// The backward's products: `vchunk` columns of the vocabulary at a time (a multiple of
// 256), the tile of the logits product and the width of its runs, and the tile and most K
// slices of the dH product.
struct LPPlan {
  int vchunk, prob_cfg, run, runs, dh_cfg, dh_bm, dh_bn, dh_ks;
  long part_elems;
};
LPPlan lp_plan(int n, int D, int V) {
  LPPlan q{};
  const long vr = ((long)V + 255) / 256 * 256;
  const long units = (vr * n + kProbElems - 1) / kProbElems;
  q.vchunk = (int)((vr / 256 + units - 1) / units * 256);
  q.prob_cfg = lp_cfg(n, D, q.vchunk, 2.0);
  q.run = lp_run(q.prob_cfg);
  q.runs = (V + q.run - 1) / q.run;
  // accumulators of all slices: three times the rows, and up to eight slices
  q.dh_ks = kMaxSlices;
  q.part_elems = (n > 2048 ? 3L : (long)kMaxSlices) * n * D;
  double bt = 0;
  for (int cfg = 0; cfg < kGemmCfgs; ++cfg) {
    const GemmTile t = gemm_tile(cfg);
    const int ks = live_split(n, D, q.vchunk, t.bm, t.bn, q.dh_ks, q.part_elems);
    const long blocks = (long)((n + t.bm - 1) / t.bm) * ((D + t.bn - 1) / t.bn) * ks;
    const double steps = ((q.vchunk + 63) / 64 + ks - 1) / ks;
    const double c = std::max(std::ceil((double)blocks / kGemmCus) * steps * t.step,
                              2.0 * q.vchunk * ((double)n + D) / 6.8e6) +
                     4.0 * ks * n * D / 3.9e6;
    if (bt == 0 || c < bt) {
      bt = c;
      q.dh_cfg = cfg;
      q.dh_bm = t.bm;
      q.dh_bn = t.bn;
    }
  }
  return q;
}

struct LPWork {
  int* count;   // scored rows
  int* rows;    // [n] their rows in order
  int* place;   // [n] a row's place among them, −1: unscored, −2: label past V
  int* labels;  // by place, as below
  float* ref;
  float* tgt;
  bf16* X;      // [n, D] the scored rows
  LPStat* stats;
  // backward
  float* rsum;   // [n, runs]
  bf16* P;       // [n, vchunk]
  float* part;   // the dH product's accumulators
  LPPlan plan;
};

LPWork lp_layout(int n, int D, int V, bool backward, void* base, size_t* bytes) {
  Carve c{(char*)base};
  LPWork w{};
  const size_t N = (size_t)n;
  w.count = c.take<int>(1);
  w.rows = c.take<int>(N);
  w.place = c.take<int>(N);
  w.labels = c.take<int>(N);
  w.ref = c.take<float>(N);
  w.tgt = c.take<float>(N);
  w.X = c.take<bf16>(N * D);
  if (!backward) {
    const int run = lp_run(lp_cfg(n, D, V, 0.0));
    w.stats = c.take<LPStat>(N * ((V + run - 1) / run));
  } else {
    w.plan = lp_plan(n, D, V);
    w.rsum = c.take<float>(N * w.plan.runs);
    w.P = c.take<bf16>(N * w.plan.vchunk);
    w.part = c.take<float>((size_t)w.plan.part_elems);
  }
  *bytes = c.at;
  return w;
}

}  // namespace

// Single block: the scored rows' indices in order and their count. A row is scored
// when 0 <= label < V and, with dlogp, dlogp ≠ 0 and logp < 0 (NaN: scored). Without
// dlogp the other rows' outputs are written here: 0, or NaN for a label past V.
__global__ __launch_bounds__(1024) void lp_rows_kernel(const int64_t* __restrict__ labels, int n,
                                                       int V, const float* __restrict__ dlogp,
                                                       const float* __restrict__ logp_in,
                                                       float* __restrict__ logp,
                                                       float* __restrict__ other, LPWork w) {
  __shared__ int tot[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int r0 = 0; r0 < n; r0 += 1024) {
    const int r = r0 + tid;
    int state = -1;
    if (r < n) {
      const int64_t lab = labels[r];
      if (lab >= V)
        state = -2;
      else if (lab >= 0)
        state = !dlogp || !(dlogp[r] == 0.f || logp_in[r] >= 0.f) ? 0 : -1;
      if (state == -2 && dlogp && dlogp[r] == 0.f) state = -1;
    }
    const unsigned long long live = __ballot(state == 0);
    if (lane == 0) tot[wave] = __popcll(live);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      before += i < wave ? tot[i] : 0;
      all += tot[i];
    }
    if (r < n) {
      const int at = base + before + __popcll(live & ((1ull << lane) - 1));
      if (state == 0) w.rows[at] = r;
      w.place[r] = state == 0 ? at : state;
      if (!dlogp && state < 0) {
        const float v = state == -2 ? NAN : 0.f;
        logp[r] = v;
        other[r] = v;
      }
    }
    base += all;
    __syncthreads();
  }
  if (tid == 0) *w.count = base;
}

// One wave per scored row: the row copied to its place, its label, and its softmax
// reference: forward the dot with W[label], backward the forward's `other`.
__global__ __launch_bounds__(256) void lp_gather_kernel(const bf16* __restrict__ H, long ldh,
                                                        const bf16* __restrict__ W,
                                                        const int64_t* __restrict__ labels, int D,
                                                        const float* __restrict__ other,
                                                        LPWork w) {
  const int m = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
  if (m >= *w.count) return;
  const int r = w.rows[m], lab = (int)labels[r];
  const bf16 *x = H + (long)r * ldh, *wt = W + (long)lab * D;
  bf16* o = w.X + (long)m * D;
  float dot = 0.f;
  for (int k = l; k < D / 8; k += 64) {
    const u32x4 v = ldg128(x + 8 * k);
    stg128(o + 8 * k, v);
    if (!other) {
      float xf[8], wf[8];
      unpack8(v, xf);
      unpack8(ldg128(wt + 8 * k), wf);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot += xf[e] * wf[e];
    }
  }
  if (!other) dot = wave_sum(dot);
  if (l == 0) {
    w.labels[m] = lab;
    w.ref[m] = other ? other[r] : dot;
  }
}

// 16 scored rows per block, 16 threads' shares of the runs each: the runs' sums
// brought to one reference M, then logp and other = M + ln L.
__global__ __launch_bounds__(256) void lp_finish_kernel(LPWork w, int cap, int runs,
                                                        float* __restrict__ logp,
                                                        float* __restrict__ other) {
  __shared__ float ms[16][17], ls[16][17];
  const int i = threadIdx.x & 15, part = threadIdx.x >> 4, m = blockIdx.x * 16 + i;
  const int M = *w.count;
  if ((int)blockIdx.x * 16 >= M) return;  // uniform
  const float ref = m < M ? w.ref[m] : 0.f;
  float mx = ref, L = 0.f;
  if (m < M) {
#pragma unroll 4
    for (int t = part; t < runs; t += 16) {
      const LPStat s = w.stats[(long)t * cap + m];
      if (s.ref == mx) {
        L += s.sum;
      } else {
        const float mn = fmaxf(mx, s.ref);
        L = L * __expf(mx - mn) + s.sum * __expf(s.ref - mn);
        mx = mn;
      }
    }
  }
  ms[part][i] = mx;
  ls[part][i] = L;
  __syncthreads();
  if (part || m >= M) return;
  for (int k = 1; k < 16; ++k) mx = fmaxf(mx, ms[k][i]);
  L = 0.f;
  for (int k = 0; k < 16; ++k) L += ls[k][i] * __expf(ms[k][i] - mx);
  const float xt = w.tgt[m], d = xt - mx, et = __expf(d);
  const int r = w.rows[m];
  // log(1 + L/e_t), exact in L where the sum would round it away
  logp[r] = -(L < et ? log1pf(L / et) : logf(et + L) - d);
  other[r] = mx + logf(L);
}

// One wave per row: dH = g·(1 − p_t)·(W_t − acc/R) with R = Σ of the probabilities as
// bf16 holds them (their common rounding falls out), acc the sum of the K slices'
// accumulators; zeros for rows left out, NaN for a label past V. The row is rounded
// once, to the output's type.
__global__ __launch_bounds__(256) void lp_dh_kernel(const bf16* __restrict__ W, int n, int D,
                                                    LPWork a, const float* __restrict__ logp,
                                                    const float* __restrict__ g, void* out,
                                                    long ldo, bool f32) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
  if (r >= n) return;
  const int m = a.place[r], M = *a.count;
  const LPPlan& q = a.plan;
  float f = m == -2 ? NAN : 0.f, R = 0.f;
  const bf16* w = W;
  const float* src = a.part;
  int ks = 1;
  if (m >= 0) {
    for (int j = l; j < q.runs; j += 64) R += a.rsum[(long)m * q.runs + j];
    R = wave_sum(R);
    f = -expm1f(logp[r]) * g[r] / R;
    w += (long)a.labels[m] * D;
    src += (long)m * D;
    ks = live_split(M, D, q.vchunk, q.dh_bm, q.dh_bn, q.dh_ks, q.part_elems);
  }
  const long plane = (long)M * D;
  for (int k = l; k < D / 8; k += 64) {
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = f;
    if (m >= 0) {
      float wf[8];
      unpack8(ldg128(w + 8 * k), wf);
      f32x4 x0 = *reinterpret_cast<const f32x4*>(src + 8 * k);
      f32x4 x1 = *reinterpret_cast<const f32x4*>(src + 8 * k + 4);
#pragma unroll 4
      for (int z = 1; z < ks; ++z) {
        x0 += *reinterpret_cast<const f32x4*>(src + z * plane + 8 * k);
        x1 += *reinterpret_cast<const f32x4*>(src + z * plane + 8 * k + 4);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = (wf[e] * R - x0[e]) * f;
        o[4 + e] = (wf[4 + e] * R - x1[e]) * f;
      }
    }
    if (f32) {
      float* d = (float*)out + (long)r * ldo + 8 * k;
      *reinterpret_cast<f32x4*>(d) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(d + 4) = f32x4{o[4], o[5], o[6], o[7]};
    } else {
      stg128((bf16*)out + (long)r * ldo + 8 * k, pack8(o));
    }
  }
}

int64_t logprob_bytes(int n, int D, int V, bool backward) {
  size_t b = 0;
  lp_layout(n, D, V, backward, nullptr, &b);
  return (int64_t)b;
}

#define LPCK(x)                          \
  do {                                   \
    const hipError_t _e = (x);           \
    if (_e != hipSuccess) return _e;     \
  } while (0)

hipError_t token_logprobs(const bf16* normed, long ldh, const bf16* W, const int64_t* labels, int n,
                          int D, int V, float* logp, float* other, void* work, hipStream_t s) {
  size_t bytes = 0;
  const LPWork w = lp_layout(n, D, V, false, work, &bytes);
  hipLaunchKernelGGL(lp_rows_kernel, dim3(1), dim3(1024), 0, s, labels, n, V,
                     (const float*)nullptr, (const float*)nullptr, logp, other, w);
  hipLaunchKernelGGL(lp_gather_kernel, dim3((n + 3) / 4), dim3(256), 0, s, normed, ldh, W, labels, D,
                     (const float*)nullptr, w);
  LPCK(hipGetLastError());
  const int cfg = lp_cfg(n, D, V, 0.0), run = lp_run(cfg);
  GemmProblem p{w.X, (long)D, W, (long)D, nullptr, 0, nullptr, 0, n, V, D, 0, w.count};
  p.live = 1;
  LPCK(launch_gemm(p, EpiLogProb{w.stats, n, V, w.ref, w.labels, w.tgt}, s, cfg));
  hipLaunchKernelGGL(lp_finish_kernel, dim3((n + 15) / 16), dim3(256), 0, s, w, n,
                     (V + run - 1) / run, logp, other);
  return hipGetLastError();
}

hipError_t token_logprobs_bwd(const bf16* normed, long ldh, const bf16* W, const int64_t* labels,
                              int n, int D, int V, const float* logp, const float* other,
                              const float* dlogp, void* dH, long lddh, bool out_f32, void* work,
                              hipStream_t s) {
  size_t bytes = 0;
  LPWork w = lp_layout(n, D, V, true, work, &bytes);
  hipLaunchKernelGGL(lp_rows_kernel, dim3(1), dim3(1024), 0, s, labels, n, V, dlogp, logp,
                     (float*)nullptr, (float*)nullptr, w);
  hipLaunchKernelGGL(lp_gather_kernel, dim3((n + 3) / 4), dim3(256), 0, s, normed, ldh, W, labels, D,
                     other, w);
  LPCK(hipGetLastError());
  const LPPlan& q = w.plan;
  for (int c0 = 0; c0 < V; c0 += q.vchunk) {
    const int Vc = std::min(q.vchunk, V - c0), Nc8 = (Vc + 7) / 8 * 8;
    GemmProblem p{w.X, (long)D, W + (long)c0 * D, (long)D, nullptr, 0, nullptr, 0,
                  n,   Vc,      D,                0,       w.count};
    p.live = 1;
    LPCK(launch_gemm(p,
                     EpiProb{w.rsum, q.runs, w.P, (long)q.vchunk, c0, Vc, Nc8, w.ref, w.labels}, s,
                     q.prob_cfg));
    // the head read in place as the [K, N] operand; each slice adds up its own partial
    GemmProblem h{w.P, (long)q.vchunk, W + (long)c0 * D, (long)D, nullptr, 0, nullptr, 0,
                  n,   D,              Nc8,              0,       w.count};
    h.b_kn = 1;
    h.kb_rows = Vc;
    h.part = w.part;
    h.part_acc = c0 > 0 ? 1 : 0;
    h.live = 1;
    h.live_k = q.vchunk;
    h.live_ks = q.dh_ks;
    h.live_elems = q.part_elems;
    LPCK(launch_gemm(h, EpiF32{w.part, (long)D, D, 0}, s, q.dh_cfg));
  }
  hipLaunchKernelGGL(lp_dh_kernel, dim3((n + 3) / 4), dim3(256), 0, s, W, n, D, w, logp, dlogp, dH,
                     lddh, out_f32);
  return hipGetLastError();
}

}  // namespace dsb
