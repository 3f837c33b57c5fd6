// C-ABI of a decoder block's memory-bound operators (8-bit rows, SwiGLU, the join of a block with its
// norms, rotary positions): argument checks and launches. The calls only enqueue; nothing here
// allocates, throws or waits.
#include <cmath>

#include "block.h"

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

// A launch holds fewer than 2^32 threads a dimension: rows with a block of 256 each.
constexpr int kMostRows = (1 << 24) - 1;
bool is_code(int type) { return type == DSB_DT_E4M3 || type == DSB_DT_INT8; }

// Rows that are read or written 8 columns at a time; `types`: a mask of DSB_DT_* that are taken.
const char* check_rows(const RowsArg& r, int rows, long width, unsigned types) {
  if (r.type < 0 || r.type > DSB_DT_INT8 || !(types >> r.type & 1)) return "rows of that type are not taken";
  if (rows == 0) return nullptr;
  if (!r.p) return "null argument";
  if (r.ld < width) return "a row stride is less than its width";
  if (is_code(r.type)) {
    if (!r.s || r.lds < (width + kBlock8 - 1) / kBlock8) return "8-bit rows need a scale byte per 32 columns";
    if (r.ld % 8 || misaligned(r.p, 8)) return "codes must be 8-byte aligned, their row stride a multiple of 8";
  } else {
    if (r.ld % (r.type == DSB_DT_F32 ? 4 : 8) || misaligned(r.p, 16))
      return "rows must be 16-byte aligned, their stride a multiple of 16 bytes";
  }
  return nullptr;
}
constexpr unsigned type_bit(int t) { return 1u << t; }
constexpr unsigned kHalf = type_bit(DSB_DT_BF16), kFloats = kHalf | type_bit(DSB_DT_F32),
                   kCodes = type_bit(DSB_DT_E4M3) | type_bit(DSB_DT_INT8);
RowsArg plain(const void* p, int64_t ld, bool f32) {
  return RowsArg{p, (long)ld, nullptr, 0, f32 ? DSB_DT_F32 : DSB_DT_BF16};
}

const char* check_join(const JoinArgs& a, bool has_y) {
  if (a.rows < 0 || a.rows > kMostRows || a.D < 8 || a.D > 8192 || a.D % 8)
    return "rows below 2^24 and D a multiple of 8 up to 8192 are taken";
  if (!(a.eps >= 0) || !std::isfinite(a.eps) || !std::isfinite(a.scale))
    return "eps and scale must be finite, eps not negative";
  if (a.gate_kind < kGateNone || a.gate_kind > kGateFull) return "unknown kind of gate";
  if (a.rows == 0) return nullptr;  // (an empty array may be null)
  if ((a.gate_kind != kGateNone) != (a.gate != nullptr)) return "the gate and its kind do not match";
  if (!has_y && (a.w_out || a.gate)) return "w_out and the gate are the block's, which is not given";
  if (misaligned(a.w_out, 16) || misaligned(a.w_in, 16)) return "weights must be 16-byte aligned";
  if (a.gate_kind == kGateChannel && misaligned(a.gate, 16)) return "the gate must be 16-byte aligned";
  if (a.gate_kind == kGateRow && (misaligned(a.gate, 2) || a.ldg < 1)) return "bad gate";
  if (a.gate_kind == kGateFull) return check_rows(plain(a.gate, a.ldg, false), a.rows, a.D, kHalf);
  return nullptr;
}

}  // namespace

extern "C" {

int dsb_save_rows8(const void* x, int64_t ldx, const void* r, int64_t ldr, int64_t x_rows, int x_dtype,
                   const int64_t* src, const int64_t* dst, int count, int width, void* codes,
                   int64_t ldc, uint8_t* scales, int64_t ldsc, int code, int64_t buf_rows,
                   void* stream) {
  const char* what = "dsb_save_rows8";
  if (x_dtype != DSB_DT_BF16 && x_dtype != DSB_DT_F16 && x_dtype != DSB_DT_F32)
    return bad(what, "x must be bf16, fp16 or fp32");
  if (!is_code(code)) return bad(what, "the code is e4m3 or int8");
  if (count < 0 || count > kMostRows || width < 0 || x_rows < 0 || buf_rows < 0 || width > (1 << 26))
    return bad(what, "bad sizes");
  if (!src != !dst) return bad(what, "src and dst are given together or not at all");
  if (!src && (count > x_rows || count > buf_rows)) return bad(what, "count is past the rows");
  if (count == 0 || width == 0) return 0;
  if ((x_rows > 0 && !x) || (buf_rows > 0 && (!codes || !scales))) return bad(what, "null argument");
  const unsigned es = x_dtype == DSB_DT_F32 ? 4 : 2;
  if (misaligned(x, es) || misaligned(r, es)) return bad(what, "a pointer is not aligned to its type");
  if (ldx < width || (r && ldr < width) || ldc < width || ldsc < ((int64_t)width + kBlock8 - 1) / kBlock8)
    return bad(what, "a row stride is less than its width");
  const Save8Args a{x, (long)ldx, r, (long)ldr, (long)x_rows, x_dtype, src, dst, count, width,
                    (uint8_t*)codes, (long)ldc, scales, (long)ldsc, code,
                    (long)(src ? buf_rows - 1 : buf_rows)};
  return launched(what, save_rows8(a, (hipStream_t)stream));
}

int dsb_op_restore_rows8(const void* codes, int64_t ldc, const uint8_t* scales, int64_t ldsc, int code,
                         int rows, int width, void* out, int64_t ldo, int out_f32, void* stream) {
  const char* what = "dsb_op_restore_rows8";
  if (!is_code(code)) return bad(what, "the code is e4m3 or int8");
  if (rows < 0 || rows > kMostRows || width < 0 || width > (1 << 26)) return bad(what, "bad sizes");
  if (rows == 0 || width == 0) return 0;
  if (!codes || !scales || !out) return bad(what, "null argument");
  if (ldc < width || ldo < width || ldsc < ((int64_t)width + kBlock8 - 1) / kBlock8)
    return bad(what, "a row stride is less than its width");
  if (misaligned(out, out_f32 ? 4 : 2)) return bad(what, "a pointer is not aligned to its type");
  const RowsArg q{codes, (long)ldc, scales, (long)ldsc, code};
  return launched(what, restore_rows8(q, rows, width, out, ldo, out_f32 != 0, (hipStream_t)stream));
}

int dsb_op_swiglu(const void* gu, int64_t ldgu, const uint8_t* gu_scales, int64_t ldsc, int gu_type,
                  int rows, int I, void* h, int64_t ldh, void* stream) {
  const char* what = "dsb_op_swiglu";
  if (rows < 0 || rows > kMostRows || I < 8 || I % 8 || I > (1 << 25))
    return bad(what, "rows below 2^24 and I a multiple of 8 up to 2^25 are taken");
  SwigluArgs a{};
  a.gu = RowsArg{gu, (long)ldgu, gu_scales, (long)ldsc, gu_type};
  if (const char* e = check_rows(a.gu, rows, 2l * I, kHalf | kCodes)) return bad(what, e);
  if (const char* e = check_rows(plain(h, ldh, false), rows, I, kHalf)) return bad(what, e);
  a.h = (bf16*)h;
  a.ldh = ldh;
  a.rows = rows;
  a.I = I;
  return launched(what, swiglu(a, (hipStream_t)stream));
}

int dsb_op_swiglu_bwd(const void* gu, int64_t ldgu, const uint8_t* gu_scales, int64_t ldsc, int gu_type,
                      int rows, int I, const void* dh, int64_t lddh, int dh_f32, void* dgu,
                      int64_t lddgu, void* h, int64_t ldh, void* stream) {
  const char* what = "dsb_op_swiglu_bwd";
  if (rows < 0 || rows > kMostRows || I < 8 || I % 8 || I > (1 << 25))
    return bad(what, "rows below 2^24 and I a multiple of 8 up to 2^25 are taken");
  SwigluArgs a{};
  a.gu = RowsArg{gu, (long)ldgu, gu_scales, (long)ldsc, gu_type};
  a.dh = plain(dh, lddh, dh_f32 != 0);
  if (const char* e = check_rows(a.gu, rows, 2l * I, kHalf | kCodes)) return bad(what, e);
  if (const char* e = check_rows(a.dh, rows, I, kFloats)) return bad(what, e);
  if (const char* e = check_rows(plain(dgu, lddgu, false), rows, 2l * I, kHalf)) return bad(what, e);
  if (h)
    if (const char* e = check_rows(plain(h, ldh, false), rows, I, kHalf)) return bad(what, e);
  a.dgu = (bf16*)dgu;
  a.lddgu = lddgu;
  a.h = (bf16*)h;
  a.ldh = ldh;
  a.rows = rows;
  a.I = I;
  return launched(what, swiglu(a, (hipStream_t)stream));
}

int dsb_op_norm_join(const void* x, int64_t ldx, const uint8_t* x_scales, int64_t ldxs, int x_type,
                     const void* y, int64_t ldy, const void* w_out, const void* w_in, const void* gate,
                     int64_t ldg, int gate_kind, double scale, double eps, int rows, int D, void* x_new,
                     int64_t ldxn, void* normed, int64_t ldn, void* stream) {
  const char* what = "dsb_op_norm_join";
  JoinArgs a{};
  a.x = RowsArg{x, (long)ldx, x_scales, (long)ldxs, x_type};
  a.y = plain(y, ldy, false);
  a.w_out = (const bf16*)w_out;
  a.w_in = (const bf16*)w_in;
  a.gate = (const bf16*)gate;
  a.ldg = ldg;
  a.gate_kind = gate_kind;
  a.scale = (float)scale;
  a.eps = (float)eps;
  a.rows = rows;
  a.D = D;
  a.x_new = x_new;
  a.ldxn = ldxn;
  a.normed = (bf16*)normed;
  a.ldn = ldn;
  const bool alone = x_new == nullptr;
  if (const char* e = check_join(a, !alone)) return bad(what, e);
  if (rows == 0) return 0;
  if (const char* e = check_rows(a.x, rows, D, alone ? kFloats | kCodes : kFloats)) return bad(what, e);
  if (alone && y) return bad(what, "x_new is null");
  if (!w_in != !normed) return bad(what, "w_in and normed are given together or not at all");
  if (alone && !w_in) return bad(what, "null argument");
  if (!alone) {
    if (const char* e = check_rows(a.y, rows, D, kHalf)) return bad(what, e);
    if (const char* e = check_rows(plain(x_new, ldxn, x_type == DSB_DT_F32), rows, D, kFloats))
      return bad(what, e);
  }
  if (normed)
    if (const char* e = check_rows(plain(normed, ldn, false), rows, D, kHalf)) return bad(what, e);
  return launched(what, join_fwd(a, (hipStream_t)stream));
}

int dsb_op_norm_join_workspace(int rows, int D, int sums, int64_t* bytes) {
  const char* what = "dsb_op_norm_join_workspace";
  if (!bytes || rows < 0 || rows > kMostRows || D < 8 || D > 8192 || D % 8) return bad(what, "bad argument");
  *bytes = join_bwd_bytes(rows, D, sums != 0);
  return 0;
}

int dsb_op_norm_join_bwd(const void* x_new, int64_t ldx, const uint8_t* x_scales, int64_t ldxs,
                         int x_type, const void* y, int64_t ldy, const uint8_t* y_scales, int64_t ldys,
                         int y_type, const void* dn, int64_t lddn, int dn_f32, const void* dxn,
                         int64_t lddxn, int dxn_f32, const void* w_out, const void* w_in,
                         const void* gate, int64_t ldg, int gate_kind, double scale, double eps,
                         int rows, int D, void* dx, int64_t lddx, int dx_f32, void* dy, int64_t lddy,
                         void* dgate, int64_t lddg, float* dw_out, float* dw_in, void* work,
                         int64_t work_bytes, void* stream) {
  const char* what = "dsb_op_norm_join_bwd";
  JoinArgs a{};
  a.x = RowsArg{x_new, (long)ldx, x_scales, (long)ldxs, x_type};
  a.y = RowsArg{y, (long)ldy, y_scales, (long)ldys, y_type};
  a.w_out = (const bf16*)w_out;
  a.w_in = (const bf16*)w_in;
  a.gate = (const bf16*)gate;
  a.ldg = ldg;
  a.gate_kind = gate_kind;
  a.scale = (float)scale;
  a.eps = (float)eps;
  a.rows = rows;
  a.D = D;
  a.dn = plain(dn, lddn, dn_f32 != 0);
  a.dxn = plain(dxn, lddxn, dxn_f32 != 0);
  a.dx = dx;
  a.lddx = lddx;
  a.dx_f32 = dx_f32 != 0;
  a.dy = (bf16*)dy;
  a.lddy = lddy;
  a.dw_in = dw_in;
  a.dw_out = dw_out;
  const bool has_y = dy != nullptr;
  if (const char* e = check_join(a, has_y)) return bad(what, e);
  if (gate_kind == kGateChannel) a.dgate = (float*)dgate;
  if (gate_kind == kGateRow) a.dgate_row = (float*)dgate;
  if (gate_kind == kGateFull) a.dgate_full = (bf16*)dgate;
  a.lddg = lddg;
  if (dgate && gate_kind == kGateNone) return bad(what, "dgate without a gate");
  if (dgate == nullptr && gate_kind == kGateFull && rows > 0) return bad(what, "null argument");
  if (rows > 0 && !has_y && dw_in) return bad(what, "dw_in comes with a block");
  if ((dw_in && !w_in) || (dw_out && !w_out)) return bad(what, "a weight's gradient without the weight");
  if (misaligned(dw_in, 16) || misaligned(dw_out, 16) || misaligned(a.dgate, 16) || misaligned(a.dgate_row, 4))
    return bad(what, "gradients of vectors must be 16-byte aligned");
  if (rows > 0) {
    if (!dn != !w_in) return bad(what, "dn and w_in are given together or not at all");
    if (!dn && !dxn) return bad(what, "there is no gradient to start from");
    if (!has_y && !dn) return bad(what, "there is neither a block nor a norm");
    if (y && !has_y) return bad(what, "dy is null");
    if (dn)
      if (const char* e = check_rows(a.x, rows, D, kFloats | kCodes)) return bad(what, e);
    if (has_y)
      if (const char* e = check_rows(a.y, rows, D, kHalf | kCodes)) return bad(what, e);
    if (dn)
      if (const char* e = check_rows(a.dn, rows, D, kFloats)) return bad(what, e);
    if (dxn)
      if (const char* e = check_rows(a.dxn, rows, D, kFloats)) return bad(what, e);
    if (const char* e = check_rows(plain(dx, lddx, a.dx_f32), rows, D, kFloats)) return bad(what, e);
    if (has_y)
      if (const char* e = check_rows(plain(dy, lddy, false), rows, D, kHalf)) return bad(what, e);
    if (a.dgate_full)
      if (const char* e = check_rows(plain(dgate, lddg, false), rows, D, kHalf)) return bad(what, e);
  }
  const int64_t need = join_bwd_bytes(rows, D, a.dw_in || a.dw_out || a.dgate);
  if (need && (work_bytes < need || !work)) return bad(what, "the workspace is too small");
  if (need && misaligned(work, 16)) return bad(what, "the workspace must be 16-byte aligned");
  return launched(what, join_bwd(a, work, (hipStream_t)stream));
}

int dsb_op_rotary(const void* x, int64_t ldx, int64_t hx, void* y, int64_t ldy, int64_t hy, int dtype,
                  const void* pos, int pos64, const double* turns, double factor, int n, int heads,
                  int head_dim, int rot, int interleaved, int inverse, void* stream) {
  const char* what = "dsb_op_rotary";
  if (dtype != DSB_DT_BF16 && dtype != DSB_DT_F16 && dtype != DSB_DT_F32)
    return bad(what, "x must be bf16, fp16 or fp32");
  if (rot < 2 || rot % 2 || rot > head_dim || head_dim > DSB_ROTARY_MOST)
    return bad(what, "rot must be even, from 2 to the head's width, which is at most 1024");
  if (n < 0 || n > kMostRows || heads < 0 || (int64_t)heads * head_dim > (1 << 20))
    return bad(what, "n must be below 2^24, heads times head_dim at most 2^20");
  if (!std::isfinite((float)factor)) return bad(what, "the factor must be finite");
  if (n == 0 || heads == 0) return 0;
  if (!x || !y || !pos || !turns) return bad(what, "null argument");
  const unsigned es = dtype == DSB_DT_F32 ? 4 : 2;
  if (misaligned(x, es) || misaligned(y, es) || misaligned(pos, pos64 ? 8 : 4) || misaligned(turns, 8))
    return bad(what, "a pointer is not aligned to its type");
  if (x == y && (ldx != ldy || hx != hy)) return bad(what, "in place the strides are the same");
  // rows of heads or heads of rows: the outer stride spans all of the inner one
  const bool rows_out = ldy >= (__int128)(heads - 1) * hy + head_dim,
             heads_out = hy >= (__int128)(n - 1) * ldy + head_dim;
  if ((n > 1 && ldy < head_dim) || (heads > 1 && hy < head_dim) ||
      (n > 1 && heads > 1 && !rows_out && !heads_out))
    return bad(what, "the heads of y overlap");
  RotaryArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.hx = hx;
  a.y = y;
  a.ldy = ldy;
  a.hy = hy;
  a.dtype = dtype;
  a.pos = pos;
  a.pos64 = pos64 != 0;
  a.turns = turns;
  a.factor = (float)factor;
  a.n = n;
  a.heads = heads;
  a.hd = head_dim;
  a.rot = rot;
  a.interleaved = interleaved != 0;
  a.inverse = inverse != 0;
  return launched(what, rotary(a, (hipStream_t)stream));
}

}  // extern "C"
