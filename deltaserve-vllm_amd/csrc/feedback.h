// Internal launch API of the operators for training from feedback (token log
// probabilities, preference and policy losses) and of the AdamW step with 8-
// or 32-bit moments.
#pragma once

#include "kernels.h"

namespace dsb {

// ---- logprob.hip
// Bytes of workspace for n rows (backward: of the gradient too).
int64_t logprob_bytes(int n, int D, int V, bool backward);
hipError_t token_logprobs(const bf16* normed, long ldh, const bf16* W, const int64_t* labels, int n,
                          int D, int V, float* logp, float* other, void* work, hipStream_t s);
hipError_t token_logprobs_bwd(const bf16* normed, long ldh, const bf16* W, const int64_t* labels,
                              int n, int D, int V, const float* logp, const float* other,
                              const float* dlogp, void* dH, long lddh, bool out_f32, void* work,
                              hipStream_t s);

// ---- seqloss.hip
struct PrefHyper {
  int kind;  // DSB_PREF_*
  double beta, smooth, margin, grad_scale;
  bool average;
};
struct PolicyHyper {
  double log_high, log_low;  // log(1 + clip_high), log(1 − clip_low)
  float high, low;           // the ratio's bounds
  float kl_coef;
  int kl;         // DSB_KL_*
  int reduction;  // DSB_REDUCE_*
  double inv_divisor, grad_scale;
  bool adv_rows;
};
int64_t loss_bytes(const dsb_pack_plan& p);
hipError_t next_token_labels(const int64_t* ids, const uint8_t* mask, const dsb_pack_plan& p,
                             int64_t* labels, uint8_t* rows, hipStream_t s);
hipError_t preference_loss(const float* logp, const float* ref, const uint8_t* mask,
                           const dsb_pack_plan& p, const PrefHyper& h, float* loss, float* rewards,
                           float* dlogp, void* work, hipStream_t s);
hipError_t policy_loss(const float* logp, const float* old, const float* ref, const float* adv,
                       const uint8_t* mask, const dsb_pack_plan& p, const PolicyHyper& h, float* out,
                       float* dlogp, void* work, hipStream_t s);

// ---- adamw.hip
struct AdamArgs {
  const dsb_adam_chunk* chunks;
  int nchunks;
  const int* group_chunks;  // [ngroups + 1] first chunk of each group
  int ngroups, most_chunks;
  void *m, *v;              // 8 bits: e4m3 codes of m and of sqrt(v); 32 bits: fp32 m and v
  float *m_scale, *r_scale;
  int bits;
  double lr, beta1, beta2, eps, wd, max_norm;  // max_norm < 0: no clip
  int64_t step;
  unsigned seed;
  const float* lr_dev;      // null, or the learning rate and the step count on the device
  const int64_t* step_dev;
  float* norms;             // [ngroups] (with a clip)
};
int64_t adam_bytes(int nchunks, int ngroups);
hipError_t adam_step(const AdamArgs& a, void* work, hipStream_t s);

}  // namespace dsb
