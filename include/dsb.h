/* dsb.h — C-ABI of the MI355X (gfx950) DeltaServe LoRA-SFT backward.
 *
 * One shared library, libdsb.so, loaded by ctypes into the backward child
 * (PyTorch-ROCm owns device memory and the LoRA master tensors). Plain
 * pointers and sizes only; every device pointer is a HIP device address.
 * Every function returns 0 on success and non-zero on failure, with the
 * message available from dsb_last_error().
 *
 * Reference interface replaced (paths relative to the reference checkout):
 *   the cycle  LoraSftTrainerService.process_backward
 *              deltaserve-plugin/deltaserve/bwd_services/common/trainer.py:503-678
 *   its state  LoraSftTrainerService._build_state           trainer.py:112-296
 *   its math   bwd_services/llama3.py:62-219, qwen3.py:68-204,
 *              common/{ops,attention,ffn,head}.py
 */
#ifndef DSB_H_
#define DSB_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DSB_ABI_VERSION 5

enum { DSB_FAMILY_LLAMA3 = 0, DSB_FAMILY_QWEN3 = 1 };
enum { DSB_ROPE_DEFAULT = 0, DSB_ROPE_LINEAR = 1, DSB_ROPE_LLAMA3 = 2 };
enum {
  DSB_PROJ_Q = 0, DSB_PROJ_K = 1, DSB_PROJ_V = 2, DSB_PROJ_O = 3,
  DSB_PROJ_GATE = 4, DSB_PROJ_UP = 5, DSB_PROJ_DOWN = 6, DSB_NUM_PROJ = 7
};
/* element types of the capture entry points and of rows (the last two: 8-bit rows, below) */
enum { DSB_DT_BF16 = 0, DSB_DT_F16 = 1, DSB_DT_F32 = 2, DSB_DT_E4M3 = 3, DSB_DT_INT8 = 4 };
/* dsb_desc.flags */
/* DSB_FLAG_SERIAL_LAYERS: run each layer's recompute right before its
   backward on the cycle's stream, instead of beside the previous layer's
   backward on a second stream (the default for models of more than one layer
   whose s_max · hidden is at most 2^24; results are the same either way). */
enum { DSB_FLAG_GRAPH = 1u, DSB_FLAG_NO_CLIP = 2u, DSB_FLAG_KTIMING = 4u,
       DSB_FLAG_SERIAL_LAYERS = 8u };

typedef struct dsb_handle dsb_handle;

/* Model and trainer constants: the backward `meta` dict of
 * deltaserve-plugin/deltaserve/ft_meta.py:131-213 plus the AdamW settings of
 * trainer.py:252-256. head_dim 128 or 64; lora_rank in [1, 64] (the rank-r
 * kernels run at the rank rounded up (a multiple of 8, 16 or 32), on zero-padded bf16
 * copies of A and B, and store the adapter's own r rows of each gradient);
 * hidden <= 8192. */
typedef struct dsb_desc {
  int32_t abi_version;       /* DSB_ABI_VERSION */
  int32_t family;            /* DSB_FAMILY_* (Qwen3 adds per-head q/k RMSNorm) */
  int32_t n_layers, hidden, n_heads, n_kv_heads, head_dim, intermediate, vocab;
  int32_t lora_rank;
  float lora_scaling;        /* alpha / r */
  float rms_eps;
  float rope_theta;
  int32_t rope_type;         /* DSB_ROPE_* (ops.py:26-57) */
  float rope_factor, rope_low_freq_factor, rope_high_freq_factor, rope_orig_max_pos;
  int32_t s_max;             /* token capacity of one cycle (max_saved_finetuning_tokens) */
  int32_t max_seqs;          /* sequence capacity of one cycle (s_max admits any packing) */
  float beta1, beta2, adam_eps, weight_decay, max_grad_norm;
  uint32_t flags;            /* DSB_FLAG_* */
  int32_t vocab_chunk;       /* LM-head vocab columns per chunk and pause point, a multiple
                                of 256 (0: 16384, the reference's VOCAB_CHUNK, head.py:25,
                                several chunks at a time over few rows) */
  int32_t gemm_tile;         /* dense-product tile: 0 by shape, else 256, 128 or 64 */
} dsb_desc;

/* Frozen bf16 base weights of one decoder layer, borrowed (the IPC-shared
 * vLLM tensors of trainer.py:201-218: fused qkv_proj and gate_up_proj). */
typedef struct dsb_layer_weights {
  const void* qkv;      /* [q + 2kv, D] */
  const void* o;        /* [D, q] */
  const void* gate_up;  /* [2I, D] (gate rows first) */
  const void* down;     /* [D, I] */
  const void* in_ln;    /* [D] */
  const void* post_ln;  /* [D] */
  const void* q_norm;   /* [head_dim] (Qwen3) or NULL */
  const void* k_norm;   /* [head_dim] (Qwen3) or NULL */
} dsb_layer_weights;

/* One LoRA projection: fp32 PEFT masters A [r, in], B [out, r] and their
 * gradient buffers (torch-owned; the cycle writes the clipped gradient). */
typedef struct dsb_lora_tensors {
  float* A;
  float* B;
  float* gA;
  float* gB;
} dsb_lora_tensors;

/* The captured-activation store (accumulate.py:236-252): per-layer residual
 * inputs and the pre-final-norm residual, bf16 [s_max + 1, D] rows of stride
 * `ld`, and the token ids int64 [s_max]. Only rows [0, n) are read.
 * mlp_gate_up (NULL when not captured): the optional per-layer gate‖up save
 * point, bf16 [s_max + 1, 2·intermediate] (gate columns first) of row stride
 * ld_gate_up; when bound, the cycle takes gate and up from it instead of
 * recomputing the gate_up product (llama3.py:63-72, ffn.py:18-26). */
typedef struct dsb_activations {
  const void* const* layer_in;  /* n_layers pointers */
  const void* final_in;
  const int64_t* input_ids;
  int64_t ld;
  const void* const* mlp_gate_up;  /* n_layers pointers, or NULL */
  int64_t ld_gate_up;
  /* The optional q/k/v save point (all three or none; accumulate.py:213-226):
   * bf16 [s_max + 1, q | kv | kv] per layer, row strides ld_q / ld_k / ld_v.
   * Llama-3 saves q and k after RoPE, Qwen3 before its q/k-norm
   * (family.py:75-84). When bound, the Q/K/V projection is not recomputed
   * (llama3.py:118-126, qwen3.py:90-96): Llama-3 attends the saved rows
   * directly, Qwen3 re-applies the q/k-norm and RoPE to them. The callers
   * pass them only when the worker's save_attn_qkv is on (trainer.py:539-544). */
  const void* const* attn_q;
  const void* const* attn_k;
  const void* const* attn_v;
  int64_t ld_q, ld_k, ld_v;
  /* The optional attention-context save point, bf16 [s_max + 1, q]: the O
   * projection's input (llama3.py:128-132). The attention forward still
   * runs, since the backward takes its softmax statistics and rowsum(dO∘O)
   * from it. */
  const void* const* attn_ctx;
  int64_t ld_ctx;
  /* The optional post-attention residual save point, bf16 [s_max + 1, D]:
   * used in place of the O projection and the residual add
   * (llama3.py:134-141; passed when save_resid_mid is on, trainer.py:552). */
  const void* const* resid_mid;
  int64_t ld_resid_mid;
} dsb_activations;

/* Per-cycle device timing (ms), filled by dsb_step when requested. */
typedef struct dsb_cycle_info {
  float gpu_ms;
  int32_t graph;       /* 1 if the cycle replayed the captured hipGraph */
  int32_t n_valid;
} dsb_cycle_info;

/* Creates the backward state (replaces _build_state's dims/optimizer part,
 * trainer.py:112-256). */
int dsb_create(const dsb_desc* desc, dsb_handle** out);
void dsb_destroy(dsb_handle* h);
/* Message of the last failure on this thread (h may be NULL). */
const char* dsb_last_error(const dsb_handle* h);

/* Binds layer `layer`'s base weights (trainer.py:201-218). Makes the
 * transposed copies the dX products read, once, after waiting for all work
 * already issued to the device (the weights may still be in flight on the
 * caller's streams). */
int dsb_bind_weights(dsb_handle* h, int layer, const dsb_layer_weights* w);
/* Binds the LM head [vocab, D] and the final RMSNorm weight [D] (trainer.py:194-195);
 * waits for the device like dsb_bind_weights. */
int dsb_bind_head(dsb_handle* h, const void* lm_head, const void* final_norm);
/* Binds one LoRA projection (trainer.py:231-243); proj is DSB_PROJ_*. Any
 * subset of the seven projections may be bound per layer (the reference's
 * ld.get(proj) may be None, trainer.py:457-460); unbound ones stay frozen. */
int dsb_bind_lora(dsb_handle* h, int layer, int proj, const dsb_lora_tensors* t);
/* Binds the shared activation buffers (base.py:438-461 share_activations). */
int dsb_bind_activations(dsb_handle* h, const dsb_activations* a);
/* The same with the layers' inputs, their gate‖up, or both in 8 bits (the formats are described
 * with dsb_save_rows8): n_layers descriptors each, or NULL; `a` then holds NULL in their place. The cycle restores a
 * layer's rows to bf16, exactly, when it recomputes the layer, and is that of a bf16 store of these
 * values bit for bit. No counterpart in the reference, whose store is bf16. */
typedef struct dsb_rows8 {
  const void* codes;
  const uint8_t* scales;
  int64_t ld, ld_scales;
  int32_t type; /* DSB_DT_E4M3 or DSB_DT_INT8 */
  int32_t pad;
} dsb_rows8;
int dsb_bind_activations8(dsb_handle* h, const dsb_activations* a, const dsb_rows8* layer_in,
                          const dsb_rows8* mlp_gate_up);

/* One backward cycle + AdamW step (+ the served-slot publish when slots are
 * bound, dsb_bind_served): trainer.py:503-678.
 * seq_lens: host int32[nseq] in request order, summing to n <= s_max.
 * lr: this cycle's learning rate; step: the optimizer step count t >= 1.
 * stream: the caller's hipStream_t (work is ordered after it and it waits
 * for the cycle). Writes the mean loss and the number of predicting rows. */
int dsb_step(dsb_handle* h, const int32_t* seq_lens, int nseq, int n, float lr, int64_t step,
             void* stream, float* loss, int* n_valid, dsb_cycle_info* info);

/* The same cycle in segments, for the GPU-yield contract of the reference's
 * BackwardService._maybe_pause (bwd_services/base.py:148-208), which the
 * reference calls once per vocab chunk in both LM-head passes (head.py:78-80,
 * :92-94) and at every layer boundary (llama3.py:342-344). With C =
 * ceil(vocab / vocab_chunk): segments 0 .. C-1 are the head's LSE pass, one
 * vocab chunk each; C .. 2C-1 its gradient pass (the two products of a chunk
 * run in segments 2c and 2c+1; with vocab_chunk = 0 and few rows, chunks are
 * computed together, and the segments between a group's two products are
 * pause points without work); 2C .. 2C+L-1 the decoder
 * layers from the last to the first; 2C+L (the last) the clip, AdamW and
 * publish. dsb_step_begin stages the
 * cycle (like dsb_step's first half); dsb_step_segment launches segment `seg`
 * (in order, each its own captured graph) and, when run_ahead > 0, keeps the
 * host at most run_ahead segments ahead of the GPU: the reference's
 * backward_run_ahead_boundaries event ring (base.py:155-183). dsb_step_end
 * waits for the cycle and reports like dsb_step. The caller's pause check
 * runs between dsb_step_segment calls, outside any captured region. Results
 * equal dsb_step's bit for bit (same kernels, same order). */
int dsb_num_segments(const dsb_handle* h);
int dsb_step_begin(dsb_handle* h, const int32_t* seq_lens, int nseq, int n, float lr,
                   int64_t step, void* stream);
int dsb_step_segment(dsb_handle* h, int seg, int run_ahead);
int dsb_step_end(dsb_handle* h, void* stream, float* loss, int* n_valid, dsb_cycle_info* info);

/* Served-slot publish, replacing LoraSftTrainerService._publish_to_served
 * (trainer.py:760-802): binds the bf16 rows of vLLM's stacked LoRA buffers
 * for one projection, a_slot = lora_a_stacked[slot, 0] ([r, in], row stride
 * lda) and b_slot = lora_b_stacked[slot, 0] ([out, r], row stride ldb).
 * Every cycle then ends by writing clamp(A, ±6.5e4) and clamp(s·B, ±6.5e4),
 * cast to bf16, into every bound slot, inside its graph after AdamW. NULL
 * slots unbind. dsb_publish writes them once outside a cycle (the
 * switch_adapter path, trainer.py:721-724). */
int dsb_bind_served(dsb_handle* h, int layer, int proj, void* a_slot, int64_t lda, void* b_slot,
                    int64_t ldb);
int dsb_publish(dsb_handle* h, void* stream);

/* Per-kernel-class timing. While enabled (DSB_FLAG_KTIMING at create, or
 * dsb_set_kernel_timing), each cycle replays the captured kernel sequence
 * eagerly on its stream with a HIP event pair around every kernel, and adds
 * the elapsed time and the launch's algorithmic flops / HBM bytes (evaluated
 * for the cycle's live n and packing) to its class. dsb_kernel_stats returns
 * the number of classes (idx < 0 only counts). No counterpart in the
 * reference (it times whole cycles with CUDA events, base.py:528-534); used
 * by bench.py for per-class rooflines. */
int dsb_set_kernel_timing(dsb_handle* h, int on);
int dsb_kernel_stats(const dsb_handle* h, int idx, char* name, int name_len, int64_t* calls,
                     double* total_ms, double* flops, double* bytes);
int dsb_kernel_stats_reset(dsb_handle* h);

/* Zeroes the AdamW moments and sets the weight decay: the fresh optimizer
 * of LoraSftTrainerService.switch_adapter (trainer.py:725-731). The masters
 * keep their addresses, so a captured graph stays valid. */
int dsb_reset_optimizer(dsb_handle* h, float weight_decay);

/* Integer packing of a cycle, host only (trainer.py:510-518, head.py:63-72):
 * positions[n], pred[n] (1 if row t predicts ids[t+1]), returns n_valid or -1. */
int dsb_pack(const int32_t* seq_lens, int nseq, int n, int32_t* positions, int32_t* pred);

/* RoPE inverse frequencies [head_dim/2] (ops.py:26-57), host only. */
int dsb_rope_inv_freq(int head_dim, float theta, int rope_type, float factor, float low,
                      float high, float orig_max, float* out);

/* ---- the forward-side capture (the serving worker's half of the handoff) ----
 *
 * dsb_capture_index replaces ActivationAccumulator.arm_op_step
 * (accumulate.py:324-343), host only: for a step whose finetuning rows sit at
 * `positions` [num_ft] of the flat batch, fills the fixed-length index pair
 * src/dst [max_saved] (n = min(num_ft, max_saved - offset) rows: src[i] =
 * positions[i], dst[i] = offset + i; the rest src 0, dst max_saved, the
 * scratch row). Returns n, or -1 on bad arguments.
 *
 * dsb_save_rows replaces the save op torch.ops.vllm.dserve_save_rows
 * (ft_save_op.py:72-93): buf[dst[i]] = bf16(x[src[i]] (+ r[src[i]], added in
 * x's dtype)) for i < count, x/r of element type x_dtype (DSB_DT_*), rows of
 * `width` elements; buf is a bf16 store [buf_rows = max_saved + 1, ldbuf].
 * Slots pointing at the scratch row (dst == buf_rows - 1), and slots whose
 * src lies outside x's x_rows rows (where the reference's index_select would
 * raise a device-side assert), are skipped. Only
 * enqueues on `stream` (no host synchronisation), so it can be captured in a
 * graph and replayed with refreshed device indices.
 *
 * dsb_save_ids: the final save point's token ids (accumulate.py:598-622):
 * out[dst[i]] = ids[src[i]] for dst[i] < out_len and src[i] < ids_len;
 * stream-ordered likewise. */
int dsb_capture_index(const int64_t* positions, int num_ft, int offset, int max_saved,
                      int64_t* src, int64_t* dst);
int dsb_save_rows(const void* x, int64_t ldx, const void* r, int64_t ldr, int64_t x_rows,
                  int x_dtype, const int64_t* src, const int64_t* dst, int count, int width,
                  void* buf, int64_t ldbuf, int64_t buf_rows, void* stream);
int dsb_save_ids(const int64_t* ids, int64_t ids_len, const int64_t* src, const int64_t* dst,
                 int count, int64_t* out, int64_t out_len, void* stream);

/* ---- single-op entry points (synchronous on `stream`) ----
 *
 * Their scratch memory comes from a pool per device that keeps up to 512 MiB
 * between calls (and 16 MiB of pinned host memory in all); a block serves one
 * call at a time. dsb_release_workspaces gives back what is kept and not in
 * use by a running call. */
int dsb_release_workspaces(void);

/* C = A·Bᵀ (+ A2·B2ᵀ) [+ R]; out_f32 selects fp32 C (accumulate adds to C).
 * b_kn: B and B2 are stored [K, N] (a weight in its own [out, in] layout read
 * by the backward's C = dY·W; N a multiple of 8) instead of [N, K].
 * cfg: -1 (or -2) the tile and the K split the cycle would take for the shape
 * (the least estimated time); 0/1/2 force 256/128/64-wide tiles, 3 a 256x128
 * and 4 a 128x64 one, without a split; -3 256-wide tiles with K split over
 * those of a partly filled last round of the device's compute units (plain
 * launch when there is no such tail). */
int dsb_op_gemm(const void* A, int64_t lda, const void* B, int64_t ldb, const void* A2,
                int64_t lda2, const void* B2, int64_t ldb2, int M, int N, int K1, int K2,
                void* C, int64_t ldc, int out_f32, int accumulate, const void* R, int64_t ldr,
                int b_kn, int cfg, void* stream);
/* dsb_gemm_plan (host only): the tile (cfg 0 to 4) and the number of K slices
 * that a product M × N × K with `out_bytes` read and written per output element
 * takes where it may split. dsb_op_gemm_split: dsb_op_gemm with the tile (0 to
 * 4) and 2 to 16 K slices of it given; N a multiple of 8. */
int dsb_gemm_plan(int M, int N, int K, double out_bytes, int* tile, int* slices);
int dsb_op_gemm_split(const void* A, int64_t lda, const void* B, int64_t ldb, const void* A2,
                      int64_t lda2, const void* B2, int64_t ldb2, int M, int N, int K1, int K2,
                      void* C, int64_t ldc, int out_f32, int accumulate, const void* R, int64_t ldr,
                      int b_kn, int tile, int slices, void* stream);
/* Gate‖up product with the SwiGLU forward in its epilogue (the recompute of
 * ffn.py:25-26, frozen gate_up_proj plus its LoRA term; silu as ffn.py:40-41): GU[m, :] = bf16(A·Bᵀ + A2·B2ᵀ)
 * with B [2I, K1] = gate rows then up rows (GU = [gate | up], ld ldgu), and,
 * when H is non-null, H[m, f] = bf16(silu(gate)·up) of the bf16-rounded
 * halves. I a multiple of 64. */
int dsb_op_gemm_glu(const void* A, int64_t lda, const void* B, int64_t ldb, const void* A2,
                    int64_t lda2, const void* B2, int64_t ldb2, int M, int I, int K1, int K2,
                    void* GU, int64_t ldgu, void* H, int64_t ldh, void* stream);
/* ops.py:84-88 */
int dsb_op_rmsnorm(const void* x, int64_t ldx, const void* w, void* y, int64_t ldy, int rows,
                   int D, float eps, void* stream);
/* ops.py:91-100, plus the bf16 residual add of llama3.py:205 / ffn.py:47-48. */
int dsb_op_rmsnorm_bwd(const void* x, int64_t ldx, const void* g, int g_f32, int64_t ldg,
                       const void* w, const void* resid, int64_t ldr, void* out, int64_t ldo,
                       int rows, int D, float eps, void* stream);
/* The same with the gradient as `parts` fp32 planes, `plane` elements apart,
 * added in order (the K slices of the product that made it). */
int dsb_op_rmsnorm_bwd_parts(const void* x, int64_t ldx, const float* g, int64_t ldg, int parts,
                             int64_t plane, const void* w, const void* resid, int64_t ldr, void* out,
                             int64_t ldo, int rows, int D, float eps, void* stream);
/* ops.py:60-65 cos/sin table [n, head_dim/2] fp32 from int32 positions. */
int dsb_op_rope_table(const int32_t* pos, int n, const float* inv_freq, int half, float* cos_out,
                      float* sin_out, void* stream);
/* ops.py:68-73 (+ qwen3.py:96-107 when norm weights are given). */
int dsb_op_rope(const void* qkv_pre, int64_t ldin, void* qk_out, int64_t ldout,
                const float* cos_t, const float* sin_t, int n, int Hq, int Hkv, int head_dim,
                const void* q_norm, const void* k_norm, float eps, void* stream);
/* ops.py:76-81 (+ qwen3.py:133-144), in place on g. */
int dsb_op_rope_bwd(void* g, int64_t ldg, const void* qkv_pre, int64_t ldp, const float* cos_t,
                    const float* sin_t, int n, int Hq, int Hkv, int head_dim, const void* q_norm,
                    const void* k_norm, float eps, void* stream);
/* attention.py:20-45; o32 [n, Hq*head_dim] fp32 and lse [Hq, n] (log2 domain)
 * out; head_dim 128 or 64. */
int dsb_op_attn_fwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                    int64_t ldv, void* ctx, int64_t ldc, float* o32, float* lse,
                    const int32_t* seq_lens, int nseq, int Hq, int Hkv, int head_dim,
                    void* stream);
/* attention.py:48-112 given the forward's o32/lse. */
int dsb_op_attn_bwd(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                    int64_t ldv, const float* o32, const float* lse, const void* dout,
                    int64_t lddo, void* dq, int64_t lddq, void* dk, int64_t lddk, void* dv,
                    int64_t lddv, const int32_t* seq_lens, int nseq, int Hq, int Hkv,
                    int head_dim, void* stream);
/* head.py:42-100 from the normed rows: loss, n_valid and dH [n, D] fp32
 * (grad wrt the normed rows; the final-norm backward is dsb_op_rmsnorm_bwd),
 * streaming the vocabulary in chunks of vocab_chunk columns (a multiple of
 * 256; 0: 16384). */
int dsb_op_head(const void* normed, int64_t ldh, const void* lm_w, const int64_t* ids,
                const int32_t* seq_lens, int nseq, int n, int D, int V, int vocab_chunk,
                float* dH, float* loss, int* n_valid, void* stream);
/* grad_A / grad_B of ops.py:143-144: out = scale · Pᵀ·X over n rows, P bf16
 * [n, R] (rows of out in groups of rg written to outs[j / rg]; transpose_out
 * writes out[c, j]). */
int dsb_op_lora_tn(const void* P, int64_t ldp, const void* X, int64_t ldx, int n, int R, int C,
                   float scale, float* out0, float* out1, float* out2, int rg, int transpose_out,
                   void* stream);
/* Z / grad_Z of ops.py:141-142: Z = bf16(X·Bᵀ), X [n, K], B [R, K]. */
int dsb_op_lora_skinny(const void* X, int64_t ldx, const void* B, int64_t ldb, int n, int R, int K,
                       void* Z, int64_t ldz, void* stream);
/* One pass of dsb_op_lora_dual: grad_Z and grad_B of ops.py:142 and :144
 * from one pass over gy = G [n, C]: gZ = bf16(G·BTᵀ) with BT = (s·B)ᵀ [r, C]
 * (ld ldbt), and gB[c, j] = scale · sum_t G[t, c]·Z[t, j] (fp32 [C, r], or
 * [r, C] when transpose_out = 0; the same pass over xin with BT = A and
 * Z = grad_Z gives ops.py:141 Z and :143 grad_A). C, ldg, ldbt multiples of 8. */
typedef struct dsb_dual_pass {
  const void* G; int64_t ldg;
  const void* Z; int64_t ldz;
  const void* BT; int64_t ldbt;
  int32_t C;
  float scale;
  void* gZ; int64_t ldgz;
  float* gB;
  int32_t transpose_out;
} dsb_dual_pass;
/* 1 to 3 passes of rank r in {16, 32} over n rows in one launch (the cycle
 * batches q, k and v this way). The row count is read from device memory,
 * as in the cycle, and the token-split partials are laid out for n_alloc >= n
 * rows. */
int dsb_op_lora_dual(const dsb_dual_pass* passes, int count, int n, int n_alloc, int r,
                     void* stream);
/* dsb_op_lora_dual without any allocation, for callers that cannot call
 * hipMalloc (code under HIP graph capture, tight serving loops). No
 * counterpart in the reference. The row count n is a launch argument, the
 * partial sums live in a 64 MiB device array of the library (one per GPU,
 * held until the process ends; a request needing more fails with an error),
 * and the call only enqueues on `stream` (no synchronisation). Every call on
 * one GPU shares that GPU's array: calls that overlap on one GPU race. */
int dsb_op_lora_dual_noalloc(const dsb_dual_pass* passes, int count, int n, int n_alloc, int r,
                             void* stream);
/* trainer.py:624-636 + :668 on a flat tensor list: per-group clip then AdamW. */
int dsb_op_clip_adamw(float* const* w, float* const* g, float* const* m, float* const* v,
                      const int32_t* numel, const int32_t* group, int ntensors, int ngroups,
                      float lr, float beta1, float beta2, float eps, float wd, int64_t step,
                      float max_norm, int do_clip, void* stream);

/* ---- training from feedback: stream-ordered ops that only enqueue
 *
 * No counterpart in the reference, whose backward trains on next-token
 * cross-entropy alone. They allocate nothing and do not synchronise, so they
 * can be captured into a graph and replayed; `work` is device scratch of at
 * least the bytes that the matching *_workspace call gives, 256-byte aligned,
 * and belongs to the call until its work on `stream` is done. The stream's
 * device has to be the current one. */

/* Log probabilities of labels: row t of normed [n, D] (bf16, row stride ldh)
 * against the LM head lm_w [V, D], labels int64 [n]; a negative label leaves the
 * row unscored, one >= V gives NaN. logp[t] = log softmax(h·Wᵀ)[label] and
 * other[t] = log Σ_{v ≠ label} exp(h·W_v), fp32 [n], 0 on unscored rows. D (up to
 * 65536) and ldh multiples of 8, V from 2 to 2^24, n below 2^24 and so is
 * ceil(n / 256)·ceil(V / 256). */
int dsb_op_logprob_workspace(int n, int D, int V, int backward, int64_t* bytes);
int dsb_op_token_logprobs(const void* normed, int64_t ldh, const void* lm_w, const int64_t* labels,
                          int n, int D, int V, float* logp, float* other, void* work,
                          int64_t work_bytes, void* stream);
/* The gradient of Σ_t dlogp[t]·logp[t] with respect to the rows, given the
 * forward's logp and other: dH [n, D] bf16 or (out_f32) fp32, row stride lddh (a
 * multiple of 8). Unscored rows and rows with dlogp = 0 get zeros and cost no
 * product. The probabilities are rounded to bf16, with either output type. */
int dsb_op_token_logprobs_bwd(const void* normed, int64_t ldh, const void* lm_w,
                              const int64_t* labels, int n, int D, int V, const float* logp,
                              const float* other, const float* dlogp, void* dH, int64_t lddh,
                              int out_f32, void* work, int64_t work_bytes, void* stream);

/* A packing of nseq sequences over n rows on the device, built once per packing
 * by dsb_plan_sizes and dsb_plan_fill (host) and copied there: int32 tables, each
 * 16-byte aligned. tiles: (first row, end row, sequence, 0) of every run of at most
 * DSB_TILE_ROWS rows of a sequence; seq_tile [nseq + 1]: a sequence's first tile;
 * starts [nseq + 1]: its first row; chunk_seq [ceil(n / DSB_CHUNK_ROWS) + 1]: the
 * sequence that holds row DSB_CHUNK_ROWS·c (the last entry: nseq − 1). npred:
 * rows that are not the last of their sequence; nonempty: sequences with one; longest: the
 * most rows of a sequence. */
enum { DSB_TILE_ROWS = 4096, DSB_CHUNK_ROWS = 4096 };
typedef struct dsb_pack_plan {
  const int32_t* tiles;
  const int32_t* seq_tile;
  const int32_t* starts;
  const int32_t* chunk_seq;
  int32_t ntiles, nseq, n, npred, nonempty, longest;
} dsb_pack_plan;
/* Host only. seq_lens int32 [nseq], each >= 0, their sum at most 2^31 − 4097, the
 * sequences and their tiles below 2^26 − 12: the counts of the plan (its pointers untouched) and the int32 elements of all four tables. */
int dsb_plan_sizes(const int32_t* seq_lens, int nseq, dsb_pack_plan* plan, int64_t* elems);
/* Host only. Fills `tables` (host memory of `elems` int32) and the plan's pointers,
 * as offsets from `device_base`, where the caller copies it. */
int dsb_plan_fill(const int32_t* seq_lens, dsb_pack_plan* plan, int32_t* tables,
                  const void* device_base);

/* labels[t] = ids[t + 1] where row t has a next token in its sequence and mask[t + 1]
 * (uint8 by token; null: all) is set, else −1; rows[t] (uint8) = labels[t] >= 0. */
int dsb_op_next_token_labels(const int64_t* ids, const uint8_t* mask, const dsb_pack_plan* plan,
                             int64_t* labels, uint8_t* rows, void* stream);

/* 0 for a batch that one workgroup takes (work may be null then). */
int dsb_op_loss_workspace(const dsb_pack_plan* plan, int64_t* bytes);
/* Preference loss over pairs: sequences 2i (preferred) and 2i + 1 of the plan.
 * s_y = Σ over the scored rows of y of (logp − ref) (its mean with `average`; 0 where
 * none is scored), z = beta·(s_2i − s_2i+1) − margin,
 *   DSB_PREF_SIGMOID: (1 − smooth)·softplus(−z) + smooth·softplus(z)
 *   DSB_PREF_HINGE:   max(0, 1 − z)
 *   DSB_PREF_IPO:     (s_2i − s_2i+1 − 1/(2·beta))²
 * and loss = the mean over pairs. Scored rows: mask [n] (uint8) or, null, every row
 * but the last of its sequence; what lies in the others is not used. ref null: 0.
 * Writes loss (fp32 scalar), rewards [nseq] = beta·s and dlogp [n] = grad_scale ·
 * dloss/dlogp (0 on unscored rows). */
enum { DSB_PREF_SIGMOID = 0, DSB_PREF_HINGE = 1, DSB_PREF_IPO = 2 };
int dsb_op_preference_loss(const float* logp, const float* ref, const uint8_t* mask,
                           const dsb_pack_plan* plan, int kind, double beta, double smooth,
                           double margin, int average, double grad_scale, float* loss,
                           float* rewards, float* dlogp, void* work, int64_t work_bytes,
                           void* stream);
/* Clipped policy loss: with ρ = exp(logp − old) and the row's advantage A,
 *   policy = −min(ρ·A, clamp(ρ, 1 − clip_low, 1 + clip_high)·A)
 *   kl (ref given): DSB_KL_K3 e^u − 1 − u, DSB_KL_K2 u²/2, u = ref − logp
 * reduced over the scored rows (as above) by DSB_REDUCE_TOKEN (mean over rows),
 * _SEQUENCE (mean over the sequences with scored rows of their rows' mean) or _SUM
 * (sum / divisor). adv is fp32 [n] (adv_rows) or [nseq]. Writes out[4] = {policy +
 * kl_coef·kl, policy, kl, share of scored rows whose ratio is clipped} and dlogp [n] =
 * grad_scale · d out[0] / dlogp. With kl_coef = 0 the reference enters out[2] alone, also where
 * its term is infinite. */
enum { DSB_KL_K3 = 0, DSB_KL_K2 = 1 };
enum { DSB_REDUCE_TOKEN = 0, DSB_REDUCE_SEQUENCE = 1, DSB_REDUCE_SUM = 2 };
int dsb_op_policy_loss(const float* logp, const float* old_logp, const float* ref,
                       const float* adv, int adv_rows, const uint8_t* mask,
                       const dsb_pack_plan* plan, double clip_low, double clip_high,
                       double kl_coef, int kl, int reduction, double divisor, double grad_scale,
                       float* out, float* dlogp, void* work, int64_t work_bytes, void* stream);

/* Up to DSB_ADAM_CHUNK elements of one tensor of an AdamW step, from a multiple of that: their
 * address in the weights and in the gradients (element types by dtypes: DSB_DT_BF16 or
 * DSB_DT_F32, w + 256·g; aligned to their type), the first of their blocks of DSB_ADAM_BLOCK
 * elements in the moments (a tensor starts on a block), their number, their group and that
 * group's chunks, c0 to c1 - 1. */
enum { DSB_ADAM_BLOCK = 256, DSB_ADAM_CHUNK = 4096 };
typedef struct dsb_adam_chunk {
  void* w;
  const void* g;
  int64_t block;
  int32_t count;
  int32_t group;
  int32_t c0, c1;
  int32_t dtypes;
  int32_t pad;
} dsb_adam_chunk;
/* Clip by group and AdamW over many tensors (the arithmetic of dsb_op_clip_adamw; the
 * gradients are left as they are). chunks, in order of their groups, and group_chunks
 * [ngroups + 1] (first chunk of each group) live on the device; most_chunks: those of the
 * largest group. nchunks is below 2^24.
 * bits 32: m and v fp32 by block. bits 8: m holds e4m3 codes of m / m_scale and v those
 * of sqrt(v) / r_scale, scales fp32 by block, the block's largest magnitude / 448; m is
 * rounded to nearest, sqrt(v) up or down at random in proportion (a function of seed, step,
 * block and element) and never down to 0 from above it. The step itself uses the moments
 * before they are rounded. max_norm < 0: no clip, norms unused; else norms [ngroups]
 * gets each group's gradient norm, summed in 64 bits (infinite past fp32; the clip is not). The
 * clip's factor is taken in 64 bits, with bits 8 as a reciprocal times max_norm in fp32. lr_dev / step_dev: when set, the learning rate (fp32)
 * and the step count (int64) are read on the device, for a captured step. */
int dsb_op_adam_workspace(int nchunks, int ngroups, int64_t* bytes);
int dsb_op_adam_step(const dsb_adam_chunk* chunks, int nchunks, const int32_t* group_chunks,
                     int ngroups, int most_chunks, void* m, void* v, float* m_scale,
                     float* r_scale, int bits, double lr, double beta1, double beta2, double eps,
                     double weight_decay, double max_norm, int64_t step, uint32_t seed,
                     const float* lr_dev, const int64_t* step_dev, float* norms, void* work,
                     int64_t work_bytes, void* stream);

/* ---- a decoder block's memory-bound operators, with its activations kept in 8 bits
 *
 * No counterpart in the reference, which keeps activations in bf16 and knows the pre-norm block with
 * rotate-half positions alone. Stream-ordered like the ops above: they allocate nothing and do
 * not synchronise, `work` is scratch of at least the bytes that the *_workspace call gives. The
 * stream's device has to be the current one. Row counts are below 2^24; strides count elements. Outputs
 * overlap neither each other nor an input, but where a call says so.
 *
 * 8-bit rows (types DSB_DT_E4M3 and DSB_DT_INT8): codes of one byte, and a byte per
 * DSB_ROWS8_BLOCK columns of a row, from the row's first, the exponent of their scale + 127. A value is
 * code·2^(byte − 127); byte 255 makes NaN of a code of 0, and byte 0, which saving never writes, 0. Saving
 * takes the least exponent, at least −126, that brings the block's largest magnitude to at most 448 (e4m3) or 127 (int8) and rounds to the nearest code, ties to
 * even, but to the code below where the nearest one's value is 2^128: finite values stay finite. A block that holds an
 * infinity or a NaN is kept as NaN whole. */
enum { DSB_ROWS8_BLOCK = 32 };
/* dsb_save_rows into 8-bit rows: codes (row stride ldc) and scales (ldsc) of buf_rows rows, the last of
 * them the scratch row. src and dst null: rows 0 to count − 1 of x into those of the buffer, the last one
 * included. Any width, strides and alignment. A row that dst names twice (but the scratch row) is
 * undefined: its codes and scales may be of either source. */
int dsb_save_rows8(const void* x, int64_t ldx, const void* r, int64_t ldr, int64_t x_rows, int x_dtype,
                   const int64_t* src, const int64_t* dst, int count, int width, void* codes,
                   int64_t ldc, uint8_t* scales, int64_t ldsc, int code, int64_t buf_rows, void* stream);
/* The values of 8-bit rows [rows, width], bf16 (exact, but for subnormals) or fp32. */
int dsb_op_restore_rows8(const void* codes, int64_t ldc, const uint8_t* scales, int64_t ldsc, int code,
                         int rows, int width, void* out, int64_t ldo, int out_f32, void* stream);
/* h [rows, I] = bf16(silu(gate)·up) of gate‖up rows [rows, 2I], bf16 or 8-bit (gu_type; scales null for
 * bf16); and their gradient dgu [rows, 2I] (bf16) for dh (bf16 or fp32), with h too unless it is null.
 * I a multiple of 8; bf16 and fp32 rows 16-byte aligned with strides of whole 16 bytes, codes 8-byte aligned
 * with strides of a multiple of 8. */
int dsb_op_swiglu(const void* gu, int64_t ldgu, const uint8_t* gu_scales, int64_t ldsc, int gu_type,
                  int rows, int I, void* h, int64_t ldh, void* stream);
int dsb_op_swiglu_bwd(const void* gu, int64_t ldgu, const uint8_t* gu_scales, int64_t ldsc, int gu_type,
                      int rows, int I, const void* dh, int64_t lddh, int dh_f32, void* dgu,
                      int64_t lddgu, void* h, int64_t ldh, void* stream);
/* The join of a block's output y with the residual stream x and the norms around it, by row:
 *   z = y / rms(y)·w_out (y where w_out is null),  x_new = x + scale·gate·z,
 *   normed = x_new / rms(x_new)·w_in,  rms(v) = sqrt(mean(v²) + eps)
 * x and x_new bf16 or fp32 (x_type), y, normed and the weights [D] bf16, the gate bf16 [D] (DSB_GATE_CHANNEL),
 * a value a row, ldg apart (_ROW), or rows of stride ldg (_FULL). w_in and normed null: no norm after. y null: a
 * norm alone of x, which may then be 8-bit rows; x_new, w_out and the gate are null. D a multiple
 * of 8 up to 8192, alignment as for SwiGLU. normed is of x_new as it is kept. */
enum { DSB_GATE_NONE = 0, DSB_GATE_CHANNEL = 1, DSB_GATE_ROW = 2, DSB_GATE_FULL = 3 };
int dsb_op_norm_join(const void* x, int64_t ldx, const uint8_t* x_scales, int64_t ldxs, int x_type,
                     const void* y, int64_t ldy, const void* w_out, const void* w_in, const void* gate,
                     int64_t ldg, int gate_kind, double scale, double eps, int rows, int D, void* x_new,
                     int64_t ldxn, void* normed, int64_t ldn, void* stream);
/* Its backward from x_new (bf16, fp32 or 8-bit rows) and y (bf16 or 8-bit rows), given the gradients dn of
 * normed and dxn of x_new (bf16 or fp32 each; null: zeros; dn null: w_in and x_new are not used):
 *   dx (bf16 or fp32, of x and of x_new's whole), dy (bf16), dw_out and dw_in fp32 [D] (null: not wanted),
 *   dgate: fp32 [D], fp32 [rows] or bf16 rows of stride lddg, as the gate's kind is; null (not wanted) for the
 *   first two, a gate of rows always gets its own.
 * y null: the gradient of a norm alone, without dw_in. `sums`: whether any of dw_out, dw_in and a channel
 * gate's dgate is wanted; they are added over rows in fp32 in a fixed order. */
int dsb_op_norm_join_workspace(int rows, int D, int sums, int64_t* bytes);
int dsb_op_norm_join_bwd(const void* x_new, int64_t ldx, const uint8_t* x_scales, int64_t ldxs,
                         int x_type, const void* y, int64_t ldy, const uint8_t* y_scales, int64_t ldys,
                         int y_type, const void* dn, int64_t lddn, int dn_f32, const void* dxn,
                         int64_t lddxn, int dxn_f32, const void* w_out, const void* w_in,
                         const void* gate, int64_t ldg, int gate_kind, double scale, double eps,
                         int rows, int D, void* dx, int64_t lddx, int dx_f32, void* dy, int64_t lddy,
                         void* dgate, int64_t lddg, float* dw_out, float* dw_in, void* work,
                         int64_t work_bytes, void* stream);
/* Rotary positions: element h·hx + i of row t of x (head h, row stride ldx, of x_dtype) into y likewise,
 * the pairs (2i, 2i + 1) (interleaved) or (i, i + rot / 2) of the first `rot` elements of a head
 * turned by pos[t]·2π·turns[i] and scaled by `factor`, the others as they are. turns: fp64 [rot / 2];
 * pos: int32, or int64 (pos64). inverse: turned back, which with the same factor is
 * the gradient. y may be x; they do not overlap otherwise. rot is even, head_dim at most DSB_ROTARY_MOST, n
 * below 2^24, heads·head_dim up to 2^20. pos·turns is reduced with one rounding, in 64 bits:
 * angles are exact to fp32 for positions below 2^31 in size. */
enum { DSB_ROTARY_MOST = 1024 };
int dsb_op_rotary(const void* x, int64_t ldx, int64_t hx, void* y, int64_t ldy, int64_t hy, int dtype,
                  const void* pos, int pos64, const double* turns, double factor, int n, int heads,
                  int head_dim, int rot, int interleaved, int inverse, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSB_H_ */
