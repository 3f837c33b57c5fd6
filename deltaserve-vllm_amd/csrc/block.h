// Internal launch API of a decoder block's memory-bound operators: 8-bit rows, SwiGLU, the join of a
// block with the norms around it, rotary positions.
#pragma once

#include "kernels.h"
#include "rows8.h"

namespace dsb {

// ---- rows8.hip
struct Save8Args {
  const void* x; long ldx;
  const void* r; long ldr;     // or null
  long x_rows;
  int dtype;                   // of x and r: DSB_DT_BF16, _F16 or _F32
  const int64_t *src, *dst;    // null: row i into row i
  int count, width;
  uint8_t* codes; long ldc;
  uint8_t* scales; long lds;
  int code;                    // DSB_DT_E4M3 or _INT8
  long out_rows;               // rows that may be written
};
hipError_t save_rows8(const Save8Args& a, hipStream_t s);
// rows_dev (or null): rows past *rows_dev are left as they are.
hipError_t restore_rows8(const RowsArg& q, int rows, int width, void* out, long ldo, bool f32,
                         hipStream_t s, const int* rows_dev = nullptr);
// h = silu(gate)·up of gate‖up rows, and with dh (bf16 or fp32) its gradient dgu; h or dgu null: not
// wanted.
struct SwigluArgs {
  RowsArg gu;
  RowsArg dh;
  bf16* dgu; long lddgu;
  bf16* h; long ldh;
  int rows, I;
};
hipError_t swiglu(const SwigluArgs& a, hipStream_t s);

// ---- norm_join.hip
enum { kGateNone = DSB_GATE_NONE, kGateChannel = DSB_GATE_CHANNEL, kGateRow = DSB_GATE_ROW,
       kGateFull = DSB_GATE_FULL };
struct JoinArgs {
  RowsArg x;                   // the stream before (forward) or after (backward) the join
  RowsArg y;                   // the block's output; p null: a norm alone
  const bf16 *w_out, *w_in;    // or null
  const bf16* gate; long ldg;
  int gate_kind;
  float scale, eps;
  int rows, D;
  // forward
  void* x_new; long ldxn;      // in x's type
  bf16* normed; long ldn;
  // backward
  RowsArg dn, dxn;             // p null: zeros
  void* dx; long lddx; bool dx_f32;
  bf16* dy; long lddy;
  bf16* dgate_full; long lddg;
  float* dgate_row;
  float *dw_in, *dw_out, *dgate;  // sums over rows, or null
};
hipError_t join_fwd(const JoinArgs& a, hipStream_t s);
int64_t join_bwd_bytes(int rows, int D, int sums);
hipError_t join_bwd(const JoinArgs& a, void* work, hipStream_t s);

// ---- rotary.hip
struct RotaryArgs {
  const void* x; long ldx, hx;  // row and head strides in elements
  void* y; long ldy, hy;
  int dtype;
  const void* pos;
  bool pos64;
  const double* turns;          // [rot / 2] turns (of 2π) a position
  float factor;
  int n, heads, hd, rot;
  bool interleaved, inverse;
};
hipError_t rotary(const RotaryArgs& a, hipStream_t s);

}  // namespace dsb
