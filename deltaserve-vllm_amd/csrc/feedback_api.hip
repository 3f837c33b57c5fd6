// C-ABI of the operators for training from feedback and of the AdamW step with
// 8- or 32-bit moments: argument checks, packing plans (host) and launches. The
// calls only enqueue; nothing here allocates, throws or waits.
#include <cmath>

#include "feedback.h"

using namespace dsb;

namespace {

int bad(const char* what, const char* why) {
  set_error("%s: %s", what, why);
  return -1;
}
int launched(const char* what, hipError_t e) {
  if (e == hipSuccess) return 0;
  set_error("%s failed: %s", what, hipGetErrorString(e));
  return -1;
}
bool misaligned(const void* p, unsigned to) { return ((uintptr_t)p & (to - 1)) != 0; }

const char* check_plan(const dsb_pack_plan* p) {
  if (!p || p->nseq < 0 || p->n < 0 || p->ntiles < 0) return "bad plan";
  if (!p->tiles || !p->seq_tile || !p->starts || !p->chunk_seq) return "the plan has no tables";
  return nullptr;
}

int64_t plan_part(int64_t elems) { return (elems + 3) / 4 * 4; }

// A launch holds fewer than 2^32 threads: blocks of 256 up to this many.
constexpr int64_t kMostBlocks = (1 << 24) - 1;
// Sequences and tiles of a plan, which take a wave each.
constexpr int64_t kMostSeqs = 4 * kMostBlocks - 8;

const char* check_head(int n, int D, int V) {
  if (n < 0 || n > kMostBlocks || V < 2 || D < 8 || D % 8 || D > 65536 || V > (1 << 24))
    return "n below 2^24, D a multiple of 8 up to 65536 and V from 2 to 2^24 are taken";
  if (((int64_t)n + 255) / 256 * ((V + 255) / 256) > kMostBlocks)
    return "n / 256 times V / 256 must be below 2^24";
  return nullptr;
}
const char* check_logprob(const void* normed, int64_t ldh, const void* lm_w, const int64_t* labels,
                          int n, int D, int V) {
  if (const char* e = check_head(n, D, V)) return e;
  if (ldh < D || ldh % 8) return "ldh must be a multiple of 8 and >= D";
  if (n > 0 && (!normed || !lm_w || !labels)) return "null argument";
  if (misaligned(normed, 16) || misaligned(lm_w, 16)) return "normed and lm_w must be 16-byte aligned";
  return nullptr;
}
const char* check_work(const void* work, int64_t have, int64_t need) {
  if (need == 0) return nullptr;
  if (have < need || !work) return "the workspace is too small";
  if (misaligned(work, 256)) return "the workspace must be 256-byte aligned";
  return nullptr;
}

}  // namespace

extern "C" {

int dsb_op_logprob_workspace(int n, int D, int V, int backward, int64_t* bytes) {
  const char* what = "dsb_op_logprob_workspace";
  if (!bytes) return bad(what, "null argument");
  if (const char* e = check_head(n, D, V)) return bad(what, e);
  *bytes = n ? logprob_bytes(n, D, V, backward != 0) : 0;
  return 0;
}

int dsb_op_token_logprobs(const void* normed, int64_t ldh, const void* lm_w, const int64_t* labels,
                          int n, int D, int V, float* logp, float* other, void* work,
                          int64_t work_bytes, void* stream) {
  const char* what = "dsb_op_token_logprobs";
  if (const char* e = check_logprob(normed, ldh, lm_w, labels, n, D, V)) return bad(what, e);
  if (n == 0) return 0;
  if (!logp || !other) return bad(what, "null argument");
  if (const char* e = check_work(work, work_bytes, logprob_bytes(n, D, V, false))) return bad(what, e);
  return launched(what, token_logprobs((const bf16*)normed, ldh, (const bf16*)lm_w, labels, n, D, V,
                                       logp, other, work, (hipStream_t)stream));
}

int dsb_op_token_logprobs_bwd(const void* normed, int64_t ldh, const void* lm_w,
                              const int64_t* labels, int n, int D, int V, const float* logp,
                              const float* other, const float* dlogp, void* dH, int64_t lddh,
                              int out_f32, void* work, int64_t work_bytes, void* stream) {
  const char* what = "dsb_op_token_logprobs_bwd";
  if (const char* e = check_logprob(normed, ldh, lm_w, labels, n, D, V)) return bad(what, e);
  if (n == 0) return 0;
  if (!logp || !other || !dlogp || !dH) return bad(what, "null argument");
  if (lddh < D || lddh % 8 || misaligned(dH, 16))
    return bad(what, "lddh must be a multiple of 8 and >= D, dH 16-byte aligned");
  if (const char* e = check_work(work, work_bytes, logprob_bytes(n, D, V, true))) return bad(what, e);
  return launched(what, token_logprobs_bwd((const bf16*)normed, ldh, (const bf16*)lm_w, labels, n, D,
                                           V, logp, other, dlogp, dH, lddh, out_f32 != 0, work,
                                           (hipStream_t)stream));
}

int dsb_plan_sizes(const int32_t* seq_lens, int nseq, dsb_pack_plan* plan, int64_t* elems) {
  const char* what = "dsb_plan_sizes";
  if (!plan || !elems || nseq < 0 || (nseq > 0 && !seq_lens)) return bad(what, "bad argument");
  int64_t n = 0, tiles = 0, npred = 0, nonempty = 0, longest = 0;
  for (int i = 0; i < nseq; ++i) {
    const int64_t len = seq_lens[i];
    if (len < 0) return bad(what, "a sequence's length is negative");
    n += len;
    tiles += (len + DSB_TILE_ROWS - 1) / DSB_TILE_ROWS;
    npred += len > 1 ? len - 1 : 0;
    nonempty += len > 1;
    longest = len > longest ? len : longest;
  }
  if (n > 0x7fffffffLL - DSB_CHUNK_ROWS) return bad(what, "the sequences hold too many rows");
  if (nseq > kMostSeqs || tiles > kMostSeqs) return bad(what, "there are too many sequences");
  plan->ntiles = (int)tiles;
  plan->nseq = nseq;
  plan->n = (int)n;
  plan->npred = (int)npred;
  plan->nonempty = (int)nonempty;
  plan->longest = (int)longest;
  *elems = plan_part(4 * tiles) + 2 * plan_part(nseq + 1) +
           plan_part((n + DSB_CHUNK_ROWS - 1) / DSB_CHUNK_ROWS + 1);
  return 0;
}

int dsb_plan_fill(const int32_t* seq_lens, dsb_pack_plan* plan, int32_t* tables,
                  const void* device_base) {
  const char* what = "dsb_plan_fill";
  if (!plan || !tables || (plan->nseq > 0 && !seq_lens)) return bad(what, "null argument");
  const int64_t chunks = ((int64_t)plan->n + DSB_CHUNK_ROWS - 1) / DSB_CHUNK_ROWS;
  const int64_t o1 = plan_part(4 * (int64_t)plan->ntiles), o2 = o1 + plan_part(plan->nseq + 1),
                o3 = o2 + plan_part(plan->nseq + 1);
  int32_t *tile = tables, *seq_tile = tables + o1, *starts = tables + o2, *chunk = tables + o3;
  int at = 0, nt = 0, c = 0;
  for (int i = 0; i < plan->nseq; ++i) {
    const int len = seq_lens[i];
    if (len < 0 || len > plan->n - at) return bad(what, "the lengths are not the plan's");
    starts[i] = at;
    seq_tile[i] = nt;
    for (int r = 0; r < len; r += DSB_TILE_ROWS, ++nt) {
      if (nt >= plan->ntiles) return bad(what, "the lengths are not the plan's");
      int32_t* t = tile + 4 * (int64_t)nt;
      t[0] = at + r;
      t[1] = at + (len - r < DSB_TILE_ROWS ? len : r + DSB_TILE_ROWS);
      t[2] = i;
      t[3] = 0;
    }
    at += len;
    for (; c < chunks && (int64_t)c * DSB_CHUNK_ROWS < at; ++c) chunk[c] = i;
  }
  if (at != plan->n || nt != plan->ntiles) return bad(what, "the lengths are not the plan's");
  starts[plan->nseq] = at;
  seq_tile[plan->nseq] = nt;
  chunk[chunks] = plan->nseq > 0 ? plan->nseq - 1 : 0;
  const int32_t* d = (const int32_t*)device_base;
  plan->tiles = d;
  plan->seq_tile = d + o1;
  plan->starts = d + o2;
  plan->chunk_seq = d + o3;
  return 0;
}

int dsb_op_next_token_labels(const int64_t* ids, const uint8_t* mask, const dsb_pack_plan* plan,
                             int64_t* labels, uint8_t* rows, void* stream) {
  const char* what = "dsb_op_next_token_labels";
  if (const char* e = check_plan(plan)) return bad(what, e);
  if (plan->n == 0) return 0;
  if (!ids || !labels || !rows) return bad(what, "null argument");
  return launched(what, next_token_labels(ids, mask, *plan, labels, rows, (hipStream_t)stream));
}

int dsb_op_loss_workspace(const dsb_pack_plan* plan, int64_t* bytes) {
  if (!plan || !bytes) return bad("dsb_op_loss_workspace", "null argument");
  *bytes = loss_bytes(*plan);
  return 0;
}

int dsb_op_preference_loss(const float* logp, const float* ref, const uint8_t* mask,
                           const dsb_pack_plan* plan, int kind, double beta, double smooth,
                           double margin, int average, double grad_scale, float* loss,
                           float* rewards, float* dlogp, void* work, int64_t work_bytes,
                           void* stream) {
  const char* what = "dsb_op_preference_loss";
  if (const char* e = check_plan(plan)) return bad(what, e);
  if (plan->nseq < 2 || plan->nseq % 2) return bad(what, "the plan must hold pairs of sequences");
  if (kind < DSB_PREF_SIGMOID || kind > DSB_PREF_IPO) return bad(what, "unknown kind");
  if (!(beta > 0) || !std::isfinite(beta)) return bad(what, "beta must be positive and finite");
  if (!(smooth >= 0 && smooth <= 1) || !std::isfinite(margin))
    return bad(what, "label smoothing lies in [0, 1], the margin is finite");
  if (smooth != 0 && kind != DSB_PREF_SIGMOID) return bad(what, "smoothing is the sigmoid loss's");
  if (margin != 0 && kind == DSB_PREF_IPO) return bad(what, "the ipo loss has no margin");
  if (!loss || !rewards || (plan->n > 0 && (!logp || !dlogp))) return bad(what, "null argument");
  if (misaligned(logp, 4) || misaligned(ref, 4) || misaligned(dlogp, 4))
    return bad(what, "a pointer is not aligned to its type");
  if (const char* e = check_work(work, work_bytes, loss_bytes(*plan))) return bad(what, e);
  const PrefHyper h{kind, beta, smooth, margin, grad_scale, average != 0};
  return launched(what, preference_loss(logp, ref, mask, *plan, h, loss, rewards, dlogp, work,
                                        (hipStream_t)stream));
}

int dsb_op_policy_loss(const float* logp, const float* old_logp, const float* ref,
                       const float* adv, int adv_rows, const uint8_t* mask,
                       const dsb_pack_plan* plan, double clip_low, double clip_high,
                       double kl_coef, int kl, int reduction, double divisor, double grad_scale,
                       float* out, float* dlogp, void* work, int64_t work_bytes, void* stream) {
  const char* what = "dsb_op_policy_loss";
  if (const char* e = check_plan(plan)) return bad(what, e);
  if (!(clip_low >= 0 && clip_low <= 1) || !(clip_high >= 0))
    return bad(what, "clip_low lies in [0, 1], clip_high is not negative");
  if (kl != DSB_KL_K3 && kl != DSB_KL_K2) return bad(what, "unknown kl estimate");
  if (reduction < DSB_REDUCE_TOKEN || reduction > DSB_REDUCE_SUM) return bad(what, "unknown reduction");
  if (!std::isfinite(kl_coef) || (kl_coef != 0 && !ref && plan->n > 0))
    return bad(what, "kl_coef must be finite, and 0 without ref");
  if (reduction == DSB_REDUCE_SUM && !(divisor > 0)) return bad(what, "the divisor must be positive");
  if (!out || (plan->n > 0 && (!logp || !old_logp || !adv || !dlogp))) return bad(what, "null argument");
  if (misaligned(logp, 4) || misaligned(old_logp, 4) || misaligned(ref, 4) || misaligned(adv, 4) ||
      misaligned(dlogp, 4))
    return bad(what, "a pointer is not aligned to its type");
  if (const char* e = check_work(work, work_bytes, loss_bytes(*plan))) return bad(what, e);
  PolicyHyper h{};
  h.log_high = log1p(clip_high);
  h.log_low = log1p(-clip_low);
  h.high = (float)(1.0 + clip_high);
  h.low = (float)(1.0 - clip_low);
  h.kl_coef = (float)kl_coef;
  h.kl = kl;
  h.reduction = reduction;
  h.inv_divisor = reduction == DSB_REDUCE_SUM ? 1.0 / divisor : 1.0;
  h.grad_scale = grad_scale;
  h.adv_rows = adv_rows != 0;
  return launched(what, policy_loss(logp, old_logp, ref, adv, mask, *plan, h, out, dlogp, work,
                                    (hipStream_t)stream));
}

int dsb_op_adam_workspace(int nchunks, int ngroups, int64_t* bytes) {
  if (!bytes || nchunks < 0 || nchunks > kMostBlocks || ngroups < 0)
    return bad("dsb_op_adam_workspace", "bad argument");
  *bytes = adam_bytes(nchunks, ngroups);
  return 0;
}

int dsb_op_adam_step(const dsb_adam_chunk* chunks, int nchunks, const int32_t* group_chunks,
                     int ngroups, int most_chunks, void* m, void* v, float* m_scale,
                     float* r_scale, int bits, double lr, double beta1, double beta2, double eps,
                     double weight_decay, double max_norm, int64_t step, uint32_t seed,
                     const float* lr_dev, const int64_t* step_dev, float* norms, void* work,
                     int64_t work_bytes, void* stream) {
  const char* what = "dsb_op_adam_step";
  if (nchunks < 0 || nchunks > kMostBlocks || ngroups < 1 || most_chunks < 0 || most_chunks > nchunks)
    return bad(what, "bad sizes");
  if (bits != 8 && bits != 32) return bad(what, "the moments have 8 or 32 bits");
  if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1))
    return bad(what, "beta1 and beta2 lie in [0, 1)");
  if (!(eps >= 0) || !std::isfinite(eps) || !std::isfinite(weight_decay) || !std::isfinite(lr))
    return bad(what, "eps, weight_decay and lr must be finite, eps not negative");
  if (!step_dev && step < 1) return bad(what, "step counts from 1");
  if (std::isnan(max_norm)) return bad(what, "max_norm is NaN");
  if (max_norm >= 0 && (!norms || !group_chunks)) return bad(what, "null argument");
  if (nchunks > 0 && (!chunks || !m || !v || (bits == 8 && (!m_scale || !r_scale))))
    return bad(what, "null argument");
  if (misaligned(m, 16) || misaligned(v, 16)) return bad(what, "the moments must be 16-byte aligned");
  if (const char* e = check_work(work, work_bytes, adam_bytes(nchunks, ngroups))) return bad(what, e);
  AdamArgs a{};
  a.chunks = chunks;
  a.nchunks = nchunks;
  a.group_chunks = group_chunks;
  a.ngroups = ngroups;
  a.most_chunks = most_chunks;
  a.m = m;
  a.v = v;
  a.m_scale = m_scale;
  a.r_scale = r_scale;
  a.bits = bits;
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.wd = weight_decay;
  a.max_norm = max_norm;
  a.step = step;
  a.seed = seed;
  a.lr_dev = lr_dev;
  a.step_dev = step_dev;
  a.norms = norms;
  return launched(what, adam_step(a, work, (hipStream_t)stream));
}

}  // extern "C"
