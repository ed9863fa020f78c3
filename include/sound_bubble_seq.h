/* sound_bubble_seq.h -- C ABI of the sequence-block operators of libsoundbubble_hip.so (gfx950 / MI355X): layer norm, gated
 * linear recurrence and AdamW over many tensors.
 *
 * Conventions as in sound_bubble_hip.h: device pointers owned by the caller, no allocation, no synchronisation, asynchronous on
 * `stream`, scratch passed in, 0 on success, -(hipError_t) on a launch error, -1000-x on a bad argument.  Element types are
 * named by SB_F32 / SB_BF16 / SB_F16; strides are in elements; pointers need the alignment of their element type only.
 * Every sum has an order that the sizes alone fix: the same call gives the same bits.
 */
#ifndef SOUND_BUBBLE_SEQ_H
#define SOUND_BUBBLE_SEQ_H
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

enum { SB_F32 = 0, SB_BF16 = 1, SB_F16 = 2 };

/* ---- layer norm over the last axis: rows x n ----
 *   y = (x - mean) * rstd * w + b,  mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps)
 * w, b (nullable) of type wtype, which is xtype or SB_F32.  mean, rstd: fp32 [rows] (nullable: not stored).
 * x rows are ldx apart (y dense). */
typedef struct {
  int64_t rows, n, ldx;
  int xtype, wtype;
  float eps;
  const void* x; const void* w; const void* b;
  void* y; float* mean; float* rstd;
} sb_layer_norm_args;
int sb_layer_norm_fwd(const sb_layer_norm_args* a, void* stream);

/* Backward: with xh = (x - mean) rstd, q = dy * w:  dx = rstd (q - mean(q) - xh mean(q xh)),  dw = sum_rows dy xh,  db = sum_rows dy.
 * dx dense; dw, db (nullable) of type wtype, stored (not added).  scratch: sb_layer_norm_bwd_scratch(rows, n, xtype) floats,
 * needed when dw or db is asked for. */
typedef struct {
  int64_t rows, n, ldx, lddy;
  int xtype, wtype;
  const void* x; const void* dy; const void* w; const float* mean; const float* rstd;
  void* dx; void* dw; void* db; float* scratch;
} sb_layer_norm_bwd_args;
int64_t sb_layer_norm_bwd_scratch(int64_t rows, int64_t n, int xtype);
int sb_layer_norm_bwd(const sb_layer_norm_bwd_args* a, void* stream);

/* ---- gated linear recurrence over the middle axis of [outer, steps, inner] ----
 *   form SB_SCAN_DECAY:    h_t = g_t h_{t-1} + x_t       (products of 16 gates in a row have to stay within float32)
 *   form SB_SCAN_SIGMOID:  h_t = s(g_t) h_{t-1} + (1 - s(g_t)) x_t,  s the logistic function
 * x of type xtype, gate of type gtype (xtype or SB_F32); h has x's type; h0 (nullable: zeros), h_last fp32 [outer, inner].
 * x / gate / dh: outer stride so_*, step stride st_*, inner axis dense.  h, dx, dgate dense.
 * reverse: the walk starts at the last step.  len (nullable, int64 [outer], clamped to 0 .. steps): steps at and after a sequence's
 * length leave its state alone; h, dx, dgate are 0 there and what x, gate and dh hold there is not used.
 * states: fp32 [chunks, outer, inner] (nullable in inference), the state in front of every chunk of steps, from which the backward
 * pass makes h again.  scratch: sb_gated_scan_plan's floats (0: NULL is fine). */
enum { SB_SCAN_DECAY = 0, SB_SCAN_SIGMOID = 1 };
typedef struct {
  int64_t outer, steps, inner;
  int xtype, gtype, form, reverse;
  const void* x; int64_t so_x, st_x;
  const void* gate; int64_t so_g, st_g;
  const float* h0; const int64_t* len;
  void* h; float* h_last; float* states; float* scratch;
} sb_gated_scan_args;
typedef struct {
  int64_t outer, steps, inner;
  int xtype, gtype, form, reverse;
  const void* x; int64_t so_x, st_x;
  const void* gate; int64_t so_g, st_g;
  const void* dh; int64_t so_d, st_d;         /* nullable: no gradient for the outputs */
  const float* dlast;                         /* [outer, inner], nullable */
  const int64_t* len; const float* states;
  void* dx; void* dgate; float* dh0;          /* dh0 nullable */
  float* scratch;
} sb_gated_scan_bwd_args;
/* -> chunks of the states buffer and floats of scratch of the two passes */
int sb_gated_scan_plan(int64_t outer, int64_t steps, int64_t inner, int xtype, int64_t* chunks, int64_t* fwd_scratch, int64_t* bwd_scratch);
int sb_gated_scan_fwd(const sb_gated_scan_args* a, void* stream);
int sb_gated_scan_bwd(const sb_gated_scan_bwd_args* a, void* stream);
/* one step: state[r, i] (fp32, dense) = a state + b, y = state in x's type; x / gate rows ld_x / ld_g apart */
int sb_gated_scan_step(const void* x, const void* gate, float* state, void* y, int64_t rows, int64_t inner, int64_t ld_x, int64_t ld_g,
                       int xtype, int gtype, int form, void* stream);

/* ---- AdamW over many tensors (torch.optim.AdamW without amsgrad) ----
 *   g = grad * gscale * min(1, clip / (|grad| gscale + 1e-6))            (clip = 0: g = grad * gscale)
 *   m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
 *   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 * The states of all tensors are one buffer each; tensor i starts at a multiple of SB_ADAMW_BLOCK elements, first_block * SB_ADAMW_BLOCK.
 * 16-bit parameters: master (fp32, same layout) is updated and p is its rounding.
 * bits = 8: m holds E4M3 codes, v E5M2 codes, with one E8M0 scale per block and state (m_scale, v_scale): the smallest 2^k that holds
 * the block's largest magnitude (448 * 2^k, 57344 * 2^k).  A code is rounded up where the part cut off plus a dither reaches 1 -- a hash of the
 * element's place in the buffer, t and seed -- so that states drift by less than a code's spacing without bias; v > 0 never becomes 0.
 * A block with a NaN or an infinity gets the NaN scale (0xFF).
 * eps may be 0: a v that is not 0 in float32 counts in the update, subnormal ones too.  No two tensors may share memory.
 * t: step (> 0), or *step_dev; lr: *lr_dev where lr_dev is given. */
#define SB_ADAMW_BLOCK 256
#define SB_ADAMW_MAX 112          /* tensors of one launch */
#define SB_ADAMW_NORM_SLOTS 512   /* doubles of the norm's partial sums */
typedef struct { void* p; const void* g; int64_t n; int32_t first_block; int32_t first_chunk; } sb_adamw_tensor;
typedef struct {
  sb_adamw_tensor t[SB_ADAMW_MAX];
  int32_t count, ptype, gtype, bits;
  void* m; void* v; void* m_scale; void* v_scale; float* master;
  double lr, beta1, beta2, eps, weight_decay;
  const float* lr_dev; const int32_t* step_dev;
  int32_t step; uint32_t seed;
  float gscale, clip;
  const double* norm_part; int32_t norm_slots;     /* clip > 0: all slots that sb_adamw_norm filled */
  const int* guard; int* skipped;                  /* as in sb_adam_step_guarded; skipped is counted up by the launch whose `last` is set */
  int32_t last;
} sb_adamw_args;
/* sums of squares of the gradients of a->t into norm_part[slot0 .. slot0 + slots) (first_chunk is used, states are not) */
int sb_adamw_norm(const sb_adamw_args* a, double* norm_part, int slot0, int slots, void* stream);
int sb_adamw_step(const sb_adamw_args* a, void* stream);
/* elements of a chunk: sb_adamw_tensor.first_chunk counts ceil(n / this) over the launch's tensors */
int sb_adamw_chunk(void);

#ifdef __cplusplus
}
#endif
#endif
