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

// Bounds on a run's Σ exp(logit − ref), ref being about the label's logit: past them (a logit
// more than about 40 over the label's, or all more than about 44 under it) the run takes its own
// maximum, the label's left out. Above the lower one what underflows in a run, 128 terms below
// 2^-126, is less than 2^-55 of its sum.
constexpr float kRunLimit = 0x1p57f, kRunFloor = 0x1p-64f;
constexpr float kRefOver = 39.5f, kRefUnder = -44.4f;  // ln of the two
constexpr float kNoWord = -0x1p126f;  // under every logit

// Probabilities held at a time: 1 GiB of bf16. Fewer chunks have fewer half-filled last
// rounds of tiles and read and write the dH accumulators less often.
constexpr long kProbElems = 1L << 29;
// and at most this many columns: 256 rows of them stay within 32-bit byte offsets
constexpr long kMaxChunk = 1L << 21;
// Every product takes 256 × 256 tiles (with lp_narrow's last ones), also over few rows, though a
// tile multiplies all its rows, scored or not (5120 × 151936: 398 GFLOP, 290 µs at the rate of a large
// product). µs at 256 × 256 / 256 × 128 / 128 × 128 tiles, forward and gradient:
//   149 rows × 5120 × 151936   338 / 393 / 498    679 / 717 / 1138
//   504 × 1024 × 151936        170 / 211 / 255    335 / 365 / 498
//   113 × 4096 × 128256        211 / 255 / 203    417 / 462 / 424
//   64 × 5120 × 151936         309 / 373 / 291    620 / 670 / 592
//   16 × 5120 × 151936         297 / 360 / 269    590 / 641 / 539
//   16 × 1024 × 151936          79 /  95 /  72    180 / 198 / 131
// so half as tall ones would be ahead by 4 to 27 % up to 64 scored rows. That number is the
// device's, and the tile is chosen on the host.
constexpr int kRun = 128;  // columns of a wave's tile
// K slices of the dH product, most: 8 tiles (500 rows × 1024) fill the CUs 32 times
// (349 µs; 16 slices 414, 8 580; before the probabilities' stores went past the caches).
constexpr int kMaxSlices = 32;
// Up to this many rows each block of the gather counts the scored rows before its own, which
// saves a launch (1024 × 151936, forward: 504 rows 162 → 158 µs, 1024 226 → 224; 2048, as
// many rows to count, 424 → 421, its gradient 829 → 833).
constexpr int kAloneRows = 1024;

// An accumulator's value, read from its AGPR here: left to itself the compiler reads all 256
// at the start of the epilogue and spills what else is live. (volatile: stays behind the
// wait for the last products.)
DSB_DEV float acc_read(const float& a) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(a));
  return v;
}

struct LPStat {
  float ref, sum;  // Σ exp(logit − ref) over a run, the label left out; 0: no other word in it
};

// Per run of TN columns and row: LPStat into stats[run · cap + m] (the 16 rows of
// a fragment are neighbours, so a store is one 128-byte line) and the label's logit
// into tgt[m]. A lane holds 4·FN columns of a row.
template <bool STREAM>
struct EpiLogProb {
  static constexpr bool kLive = true, kStreamB = STREAM;
  __host__ __device__ int most_slices(int, int) const { return 1; }
  DSB_DEV int slices(int, int, int, int) const { return 1; }
  DSB_DEV const EpiLogProb& at(int, int, int) const { return *this; }
  LPStat* stats;
  int cap, V;  // V: the product's columns, from c0 of the vocabulary on
  const float* ref;
  const int* labels;
  float* tgt;
  int c0;
  template <int FM, int FN, int WM, int WN>
  DSB_DEV void run(const f32x4 (&acc)[FM][FN], int mw, int nw, int M, int lane, int,
                   void*) const {
    constexpr int TN = FN * 16;
    if (nw >= V || mw >= M) return;
    const int l16 = lane & 15, lq = lane >> 4;
    const bool whole = nw + TN <= V;
    LPStat* out = stats + (long)(nw / TN) * cap;
    // a fragment's references and labels are loaded during the one before (all of them ahead
    // spill)
    float ref1 = ref[min(mw + l16, M - 1)];
    int lab1 = labels[min(mw + l16, M - 1)];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      if (mw + fm * 16 >= M) break;
      const float ref0 = ref1;
      const int tc = lab1 - (c0 + nw);
      ref1 = ref[min(mw + fm * 16 + 16 + l16, M - 1)];
      lab1 = labels[min(mw + fm * 16 + 16 + l16, M - 1)];
      const float tl = (float)(tc - 4 * lq);
      auto take = [&](float r, auto skips) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int fn = 0; fn < FN; ++fn)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = acc_read(acc[fm][fn][i]) - r;
            // the label's own column by a factor of 0 (as tests the masks of 128 columns spill):
            // it may be any height above r, so its e is bounded (the others' are below the bound;
            // a NaN stays)
            if (decltype(skips)::value) x = x > 64.f ? 64.f : x;
            float e = __expf(x);
            if (!whole) e = nw + fn * 16 + 4 * lq + i < V ? e : 0.f;
            if (decltype(skips)::value) e *= fminf(fabsf((float)(fn * 16 + i) - tl), 1.f);
            part[i] += e;
          }
        float v = (part[0] + part[1]) + (part[2] + part[3]);
        v += __shfl_xor(v, 16, 64);
        return LPStat{r, v + __shfl_xor(v, 32, 64)};
      };
      const int m = mw + fm * 16 + l16;
      LPStat st = take(ref0, std::false_type{});
      if (__any(!(st.sum <= kRunLimit && st.sum >= kRunFloor) || (unsigned)tc < (unsigned)TN)) {
        // rare: a row with its label in the run, or past the bounds; v: the most of the others (the
        // label's column by kNoWord under it, as tests the masks spill)
        float v = kNoWord, xt = 0.f;
#pragma unroll
        for (int fn = 0; fn < FN; ++fn)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc_read(acc[fm][fn][i]);
            const float at = (float)(fn * 16 + i);
            const float u = x + fmaf(fminf(fabsf(at - tl), 1.f), -kNoWord, kNoWord);
            v = whole || nw + fn * 16 + 4 * lq + i < V ? fmaxf(v, u) : v;
            xt = at == tl ? x : xt;
          }
        if ((unsigned)tc < (unsigned)TN && ((tc >> 2) & 3) == lq && m < M) tgt[m] = xt;
        v = fmaxf(v, __shfl_xor(v, 16, 64));
        v = fmaxf(v, __shfl_xor(v, 32, 64));
        const bool moves = v > ref0 + kRefOver || (v < ref0 + kRefUnder && v > 0.5f * kNoWord);
        st = take(moves ? v : ref0, std::true_type{});
      }
      if (lq == 0 && m < M) out[m] = st;
      // one fragment's values at a time: with several in flight the registers spill
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// The backward's probabilities of chunk [c0, c0 + Vc): P[m, j] = bf16(exp(logit − ref))
// with ref = the log-sum-exp of the row's words but the label, so each is at most 1 and
// they sum to 1, the label's as zero; columns [Vc, Nc8) as zero too. Per run of TN columns
// the sum of the rounded values goes to rsum[m · runs + run] (products with ones on the
// matrix cores). Only runs that hold a label (one in V / TN of a row's) test their columns
// for it; its exponential, which may be infinite, is left out by a select.
template <bool STREAM>
struct EpiProb {
  static constexpr bool kLive = true, kStreamB = STREAM;
  __host__ __device__ int most_slices(int, int) const { return 1; }
  DSB_DEV int slices(int, int, int, int) const { return 1; }
  DSB_DEV const EpiProb& at(int, int, int) const { return *this; }
  float* rsum;  // the chunk's first run of row 0
  int runs;     // row pitch
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
    // e^(x − ref) = 2^(x·log2(e) − ref·log2(e)) with one multiply-add: what the second
    // product's rounding changes is a factor of the whole row, which the division by R takes out
    constexpr float kLog2e = 1.44269504088896340736f;
    float ref2[FM];
    int tcol[FM];
#pragma unroll
    for (int fm = 0; fm < FM; ++fm) {
      const int m = min(mw + fm * 16 + l16, M - 1);
      ref2[fm] = -ref[m] * kLog2e;
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
              float e = __builtin_amdgcn_exp2f(fmaf(acc_read(acc[fm][fn][i]), kLog2e, ref2[fm]));
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
        if (lq == 0 && m < M) rsum[(long)m * runs + nw / TN] = r[0];
      }
#pragma unroll
      for (int it = 0; it < 32 * CG / 64; ++it) {
        const int c = lane + 64 * it, row = c / CG, m = mw + b * 32 + row;
        const int n = nw + (c % CG) * 8;
        const u32x4 v = *reinterpret_cast<const u32x4*>(buf + row * PITCH + (c % CG) * 8);
        // past the caches: the next tiles' panels stay (500 rows × 1024 × 151936: 334 → 322 µs;
        // the dH product's accumulators, read at once, lose by it: 347)
        if (m < M && n < Nc8)
          __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(P + (long)m * ldp + n));
      }
    }
  }
};

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

// The backward's chunks of the vocabulary (`vchunk` columns, a multiple of 256) and the
// room of the dH product's accumulators, all slices together: 2^24 elements are a tile for
// each CU; half as many again, or three times n rows where that is more.
struct LPPlan {
  int vchunk;
  long part_elems;
};
LPPlan lp_plan(int n, int D, int V) {
  const long blocks = ((long)V + 255) / 256;
  const long units = std::max((blocks * 256 * n + kProbElems - 1) / kProbElems,
                              (blocks + kMaxChunk / 256 - 1) / (kMaxChunk / 256));
  LPPlan q;
  q.vchunk = (int)((blocks + units - 1) / units * 256);
  q.part_elems = std::min((long)kMaxSlices * n * D, std::max(3L << 23, 3L * n * D));
  return q;
}

// Columns, the last ones of the vocabulary, that the forward's product takes in 256 × 128
// tiles: over one block of rows the head is streamed by whole rounds of the device's CUs, and
// where the last round of 256 × 256 tiles is at most half full, half-wide ones fill it better
// (5120 × 151936, 82 tiles in the third round: 149 rows 361 → 338 µs, 16 rows 309 → 297; 1024 wide
// 16 rows 81 → 79).
int lp_narrow(int n, int V) {
  const int tiles = (V + 255) / 256, last = tiles % kGemmCus;
  return n <= 256 && tiles > kGemmCus && last > 0 && last <= kGemmCus / 2
             ? V - (tiles - last) * 256
             : 0;
}

struct LPWork {
  int* count;   // scored rows
  int* rows;    // [n] their rows in order
  int* place;   // [n] a row's place among them, −1: unscored, −2: label past V
  int* labels;  // by place, as below
  float* ref;
  float* tgt;
  bf16* X;      // [n, D] the scored rows
  int runs;       // of all columns
  int narrow;     // columns that the narrower tiles take (lp_narrow)
  LPStat* stats;  // forward: [runs, n]
  // backward
  float* rsum;   // [n, runs]
  bf16* P;       // [n, vchunk]
  float* part;   // the dH product's accumulators
  LPPlan plan;
};

// The dH product's epilogue; its K slices at any live row count.
template <bool STREAM = false>
__host__ __device__ inline EpiLivePart<STREAM> lp_part(const LPWork& w, int accumulate) {
  return EpiLivePart<STREAM>{w.part, accumulate, w.plan.vchunk, kMaxSlices, w.plan.part_elems};
}

LPWork lp_layout(int n, int D, int V, bool backward, void* base, size_t* bytes) {
  Carve c{(char*)base};
  LPWork w{};
  const size_t N = (size_t)n;
  w.narrow = backward ? 0 : lp_narrow(n, V);
  w.runs = (V - w.narrow + kRun - 1) / kRun + (w.narrow + kRun / 2 - 1) / (kRun / 2);
  w.count = c.take<int>(1);
  w.rows = c.take<int>(N);
  w.place = c.take<int>(N);
  w.labels = c.take<int>(N);
  w.ref = c.take<float>(N);
  w.tgt = c.take<float>(N);
  w.X = c.take<bf16>(N * D);
  if (!backward) {
    w.stats = c.take<LPStat>(N * w.runs);
  } else {
    w.plan = lp_plan(n, D, V);
    w.rsum = c.take<float>(N * w.runs);
    w.P = c.take<bf16>(N * w.plan.vchunk);
    w.part = c.take<float>((size_t)w.plan.part_elems);
  }
  *bytes = c.at;
  return w;
}

}  // namespace

// A row is scored (0) when 0 <= label < V and, with dlogp, dlogp ≠ 0 and logp < 0 (NaN: scored);
// −2: its label is past V, −1 otherwise.
DSB_DEV int lp_state(int64_t lab, int V, float g, float p) {
  return lab < 0 || g == 0.f ? -1 : lab >= V ? -2 : p >= 0.f ? -1 : 0;
}
// Single block, four rows to a thread: the scored rows' indices in order and their count.
// Without dlogp the other rows' outputs are written here: 0, or NaN for a label past V.
__global__ __launch_bounds__(1024) void lp_rows_kernel(const int64_t* __restrict__ labels, int n,
                                                       int V, const float* __restrict__ dlogp,
                                                       const float* __restrict__ logp_in,
                                                       float* __restrict__ logp,
                                                       float* __restrict__ other, LPWork w) {
  __shared__ int tot[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int r0 = 0; r0 < n; r0 += 4096) {
    const int r = r0 + 4 * tid;
    int64_t lab[4];
    float g[4], p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = r + i < n;
      lab[i] = in ? labels[r + i] : -1;
      g[i] = in && dlogp ? dlogp[r + i] : 1.f;
      p[i] = in && dlogp ? logp_in[r + i] : -1.f;
    }
    int state[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      state[i] = lp_state(lab[i], V, g[i], p[i]);
      mine += state[i] == 0;
    }
    int before = mine;  // of the wave's lanes up to this one
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o, 64);
      before += lane >= o ? x : 0;
    }
    if (lane == 63) tot[wave] = before;
    __syncthreads();
    int all = 0, at = base + before - mine;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      at += i < wave ? tot[i] : 0;
      all += tot[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (r + i >= n) break;
      w.place[r + i] = state[i] == 0 ? at : state[i];
      if (state[i] == 0) w.rows[at++] = r + i;
      if (!dlogp && state[i] < 0) {
        const float v = state[i] == -2 ? NAN : 0.f;
        logp[r + i] = v;
        other[r + i] = v;
      }
    }
    base += all;
    __syncthreads();
  }
  if (tid == 0) *w.count = base;
}

// One block per scored row: the row copied to its place, its label, and its softmax
// reference: forward the dot with W[label], backward the forward's `other`. ALONE: one
// per row, with lp_rows_kernel's part for it.
template <bool ALONE>
__global__ __launch_bounds__(256) void lp_gather_kernel(const bf16* __restrict__ H, long ldh,
                                                        const bf16* __restrict__ W,
                                                        const int64_t* __restrict__ labels, int n,
                                                        int D, int V,
                                                        const float* __restrict__ dlogp,
                                                        const float* __restrict__ logp_in,
                                                        const float* __restrict__ other,
                                                        float* __restrict__ logp_out,
                                                        float* __restrict__ other_out, LPWork w) {
  __shared__ float red[4];
  int m = blockIdx.x, r = m;
  if constexpr (ALONE) {
    auto state = [&](int q) {
      return lp_state(labels[q], V, dlogp ? dlogp[q] : 1.f, dlogp ? logp_in[q] : -1.f);
    };
    const int mine = state(r);
    float before = 0.f;  // exact
#pragma unroll
    for (int i = 0; i < kAloneRows / 256; ++i) {
      const int q = 256 * i + threadIdx.x;
      if (q < r) before += state(q) == 0 ? 1.f : 0.f;
    }
    m = (int)block_sum<256>(before, red);
    if (threadIdx.x == 0) {
      w.place[r] = mine == 0 ? m : mine;
      if (mine == 0) w.rows[m] = r;
      if (r == n - 1) *w.count = m + (mine == 0);
      if (mine < 0 && !dlogp) logp_out[r] = other_out[r] = mine == -2 ? NAN : 0.f;
    }
    if (mine < 0) return;
  } else {
    if (m >= *w.count) return;
    r = w.rows[m];
  }
  const int lab = (int)labels[r];
  const bf16 *x = H + (long)r * ldh, *wt = W + (long)lab * D;
  bf16* o = w.X + (long)m * D;
  float dot = 0.f;
  for (int k = threadIdx.x; k < D / 8; k += 256) {
    const u32x4 v = ldg128(x + 8 * k);
    if (!other) {
      float xf[8], wf[8];
      unpack8(v, xf);
      unpack8(ldg128(wt + 8 * k), wf);
#pragma unroll
      for (int e = 0; e < 8; ++e) dot += xf[e] * wf[e];
    }
    stg128(o + 8 * k, v);
  }
  if (!other) dot = block_sum<256>(dot, red);
  if (threadIdx.x == 0) {
    w.labels[m] = lab;
    w.ref[m] = other ? other[r] : dot;
  }
}

// 16 scored rows per block, 64 threads' shares of the runs each: the runs' sums brought to
// one reference M, then logp and other = M + ln L. Nearly always every run has the row's own
// reference, and its sums are added as they are.
__global__ __launch_bounds__(1024) void lp_finish_kernel(LPWork w, int cap,
                                                         float* __restrict__ logp,
                                                         float* __restrict__ other) {
  __shared__ float ms[64][17], ls[64][17];
  const int i = threadIdx.x & 15, part = threadIdx.x >> 4, m = blockIdx.x * 16 + i;
  const int M = *w.count;
  if ((int)blockIdx.x * 16 >= M) return;  // uniform
  const float ref = m < M ? w.ref[m] : 0.f;
  float mx = -INFINITY, L = 0.f;
  if (m < M) {
    bool other_ref = false;
#pragma unroll 8
    for (int t = part; t < w.runs; t += 64) {
      const LPStat s = w.stats[(long)t * cap + m];
      L += s.sum;
      other_ref |= s.ref != ref;
    }
    if (!other_ref) {
      mx = L == 0.f ? mx : ref;
    } else {
      L = 0.f;
      for (int t = part; t < w.runs; t += 64) {
        const LPStat s = w.stats[(long)t * cap + m];
        if (s.sum == 0.f) continue;  // no word but the label: its reference is none
        const float mn = fmaxf(mx, s.ref);
        L = L * __expf(mx - mn) + s.sum * __expf(s.ref - mn);
        mx = mn;
      }
    }
  }
  ms[part][i] = mx;
  ls[part][i] = L;
  __syncthreads();
  if (part >= 4) return;  // the first wave: 4 threads to a row, in a fixed order
  for (int k = 0; k < 64; ++k) mx = fmaxf(mx, ms[k][i]);
  L = 0.f;
  for (int k = part; k < 64; k += 4) L += ls[k][i] == 0.f ? 0.f : ls[k][i] * __expf(ms[k][i] - mx);
  L += __shfl_xor(L, 16, 64);
  L += __shfl_xor(L, 32, 64);
  if (part || m >= M) return;
  const float xt = w.tgt[m], d = xt - mx, et = __expf(d);
  const int r = w.rows[m];
  // log(1 + L/e_t), exact in L where the sum would round it away; 1/e_t in two factors, as it
  // underflows before the quotient where the label is far above the rest (e_t infinite)
  const float h = __expf(-0.5f * d);
  logp[r] = -(L < et ? log1pf(L * h * h) : logf(et + L) - d);
  other[r] = mx + logf(L);
}

// One block per row: dH = g·(1 − p_t)·(W_t − acc/R) with R = Σ of the probabilities as bf16
// holds them (their common rounding falls out), acc the sum of the K slices' accumulators;
// zeros for rows left out, NaN for a label past V. The row is rounded once, to the output's
// type.
__global__ __launch_bounds__(256) void lp_dh_kernel(const bf16* __restrict__ W, int D, LPWork a,
                                                    const float* __restrict__ logp,
                                                    const float* __restrict__ g, void* out,
                                                    long ldo, bool f32) {
  __shared__ float red[4];
  const int r = blockIdx.x, tid = threadIdx.x;
  const int m = a.place[r], M = *a.count;
  float f = m == -2 ? NAN : 0.f, R = 0.f;
  const bf16* w = W;
  const float* src = a.part;
  int ks = 1;
  if (m >= 0) {
    for (int j = tid; j < a.runs; j += 256) R += a.rsum[(long)m * a.runs + j];
    R = block_sum<256>(R, red);
    f = -expm1f(logp[r]) * g[r] / R;
    w += (long)a.labels[m] * D;
    src += (long)m * D;
    ks = lp_part(a, 0).slices(M, D, 256, 256);
  }
  const long plane = (long)M * D;
  for (int k = tid; k < D / 8; k += 256) {
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

// The scored rows, gathered.
static hipError_t lp_gather(const bf16* H, long ldh, const bf16* W, const int64_t* labels, int n,
                            int D, int V, const float* dlogp, const float* logp,
                            const float* other, float* logp_out, float* other_out,
                            const LPWork& w, hipStream_t s) {
  if (n > kAloneRows)
    hipLaunchKernelGGL(lp_rows_kernel, dim3(1), dim3(1024), 0, s, labels, n, V, dlogp, logp, logp_out,
                       other_out, w);
  hipLaunchKernelGGL(n > kAloneRows ? lp_gather_kernel<false> : lp_gather_kernel<true>, dim3(n),
                     dim3(256), 0, s, H, ldh, W, labels, n, D, V, dlogp, logp, other, logp_out,
                     other_out, w);
  return hipGetLastError();
}

// Over one block of rows (n <= 256) each block of the products reads columns of the head of its
// own: past the caches (µs, through them → past them: 149 rows × 5120 × 151936 forward 349 → 335,
// gradient 711 → 690; 113 × 4096 × 128256 219 → 214, 443 → 429).
hipError_t token_logprobs(const bf16* normed, long ldh, const bf16* W, const int64_t* labels, int n,
                          int D, int V, float* logp, float* other, void* work, hipStream_t s) {
  size_t bytes = 0;
  const LPWork w = lp_layout(n, D, V, false, work, &bytes);
  LPCK(lp_gather(normed, ldh, W, labels, n, D, V, nullptr, nullptr, nullptr, logp, other, w, s));
  const int V1 = V - w.narrow;
  GemmProblem p{w.X, (long)D, W, (long)D, nullptr, 0, nullptr, 0, n, V1, D, 0, w.count};
  if (n > 256) {
    const EpiLogProb<false> epi{w.stats, n, V1, w.ref, w.labels, w.tgt, 0};
    LPCK((launch_gemm_cfg<256, 256, 2, 2>(p, epi, s)));
  } else {
    EpiLogProb<true> epi{w.stats, n, V1, w.ref, w.labels, w.tgt, 0};
    LPCK((launch_gemm_cfg<256, 256, 2, 2>(p, epi, s)));
    if (w.narrow) {
      p.B = W + (long)V1 * D;
      p.N = w.narrow;
      epi.stats += (long)(V1 / kRun) * n;
      epi.V = w.narrow;
      epi.c0 = V1;
      LPCK((launch_gemm_cfg<256, 128, 2, 2, 3, 3>(p, epi, s)));
    }
  }
  hipLaunchKernelGGL(lp_finish_kernel, dim3((n + 15) / 16), dim3(1024), 0, s, w, n, logp, other);
  return hipGetLastError();
}

hipError_t token_logprobs_bwd(const bf16* normed, long ldh, const bf16* W, const int64_t* labels,
                              int n, int D, int V, const float* logp, const float* other,
                              const float* dlogp, void* dH, long lddh, bool out_f32, void* work,
                              hipStream_t s) {
  size_t bytes = 0;
  const LPWork w = lp_layout(n, D, V, true, work, &bytes);
  LPCK(lp_gather(normed, ldh, W, labels, n, D, V, dlogp, logp, other, nullptr, nullptr, w, s));
  const int vchunk = w.plan.vchunk;
  for (int c0 = 0; c0 < V; c0 += vchunk) {
    const int Vc = std::min(vchunk, V - c0), Nc8 = (Vc + 7) / 8 * 8;
    const bf16* Wc = W + (long)c0 * D;
    GemmProblem p{w.X, (long)D, Wc, (long)D, nullptr, 0, nullptr, 0, n, Vc, D, 0, w.count};
    auto logits = [&](auto stream) {
      const EpiProb<decltype(stream)::value> epi{w.rsum + c0 / kRun, w.runs, w.P,   (long)vchunk, c0,
                                                 Vc,                 Nc8,    w.ref, w.labels};
      return launch_gemm_cfg<256, 256, 2, 2>(p, epi, s);
    };
    LPCK(n > 256 ? logits(std::false_type{}) : logits(std::true_type{}));
    // the head read in place as the [K, N] operand; each slice adds up its own partial
    GemmProblem h{w.P, (long)vchunk, Wc, (long)D, nullptr, 0, nullptr, 0, n, D, Nc8, 0, w.count};
    h.b_kn = 1;
    h.kb_rows = Vc;
    LPCK((n > 256 ? launch_gemm_cfg<256, 256, 2, 2>(h, lp_part<false>(w, c0 > 0), s)
                  : launch_gemm_cfg<256, 256, 2, 2>(h, lp_part<true>(w, c0 > 0), s)));
  }
  hipLaunchKernelGGL(lp_dh_kernel, dim3(n), dim3(256), 0, s, W, D, w, logp, dlogp, dH, lddh, out_f32);
  return hipGetLastError();
}

}  // namespace dsb
