/*
 * diffphore_train.h - C ABI of the training operators (libdiffphore_train.so): layer norm, attention over packed complexes, AdamW.
 *
 * They stand beside the forward-only layers of diffphore_amd.h and share its conventions:
 *   - every pointer is a DEVICE pointer owned by the caller; the library never allocates, frees or synchronises; all work is enqueued on the
 *     hipStream_t passed as `void*`, and every entry point may be captured into a graph.
 *   - return 0 on success, negative DP_E_* on bad arguments, positive hipError_t on a launch failure.  Never throws.
 *   - values are fp32 or bf16 (the two model precisions of the framework); sums, statistics and optimiser arithmetic are held in 32 bits or more.
 *   - results do not depend on the order in which workgroups run: no floating-point atomics.
 *   - thread-compatible: no mutable globals.
 * A library of its own, so that the sampling library's ABI and the measurements keyed to its sources are not touched by changes here.
 */
#ifndef DIFFPHORE_TRAIN_H
#define DIFFPHORE_TRAIN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DPT_ABI_VERSION 1

/* return codes: those of diffphore_amd.h */
#define DPT_OK 0
#define DPT_E_BADARG (-1)
#define DPT_E_UNSUPPORTED (-2)
#define DPT_E_TOOLARGE (-3)

enum DptType { DPT_F32 = 0, DPT_BF16 = 1 };

int dpt_abi_version(void);
/* sizes of the structs below, for bindings to check their mirrors: DptAttnArgs, DptAdamWArgs */
int dpt_struct_sizes(int32_t* out, int32_t n);

/* ---- layer norm -----------------------------------------------------------------------------------------------------------------------------
 * y = (x - mean) rstd weight + bias over the last dimension; x, y, dy, dx: [rows, width] with unit stride inside a row and row strides in elements.
 * weight / bias may be NULL (1 and 0).  wtype: the type of weight and bias (and of their gradients); fp32, or the type of x.
 * Width 1 .. dpt_layer_norm_max_width().  rows = 0 is allowed (the gradients of weight and bias are then 0). */
int dpt_layer_norm_max_width(void);
int dpt_layer_norm_fwd(int32_t type, int32_t wtype, int64_t rows, int32_t width, const void* x, int64_t x_stride, const void* weight, const void* bias,
                       float eps, void* y, int64_t y_stride, float* mean, float* rstd, void* stream);
/* dweight / dbias may be NULL (not wanted); ws: dpt_layer_norm_ws_bytes(rows, width) bytes, unless both are NULL */
size_t dpt_layer_norm_ws_bytes(int64_t rows, int32_t width);
int dpt_layer_norm_bwd(int32_t type, int32_t wtype, int64_t rows, int32_t width, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                       const float* mean, const float* rstd, const void* weight, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                       void* ws, size_t ws_bytes, void* stream);

/* ---- attention over packed complexes --------------------------------------------------------------------------------------------------------
 * Complex b owns the query rows q_ptr[b] .. q_ptr[b+1] and the key rows k_ptr[b] .. k_ptr[b+1] (CSR offsets, as DpBatch.lig_ptr / ph_ptr) and the
 * pairs pair_ptr[b] .. pair_ptr[b+1], query-major.  Query head h reads key head h / (heads / kv_heads).
 *   s_ij = scale q_i . k_j + bias[h, pair(b, i, j)];  m_i = max_j s_ij;  l_i = sum_j exp(s_ij - m_i);  out_i = sum_j exp(s_ij - m_i) v_j / l_i
 * causal: key j of a complex is seen by query i iff j <= i + n_keys - n_queries.  A bias of -inf takes the pair out.  A row that sees nothing:
 * out = 0, m = -inf, l = 0, dq = 0.  As in every product of probabilities and values, a NaN or inf in v of a pair that is taken out still reaches
 * the rows of its tile that see other keys (0 x NaN), and in the backward pass one in q, k or dout.  A row whose scores are NaN has l = NaN. */
#define DPT_ATTN_MAX_ROWS (0x7fffffff - 1024) /* most rows of q (max_nq times the heads that share a key head, too) and of k */

typedef struct DptAttnArgs {
  int32_t type;                    /* DptType of q, k, v, bias, out, dout and the gradients */
  int32_t B, heads, kv_heads, dim; /* dim 1 .. 128 */
  int32_t causal;
  int32_t n_q, n_k;                /* rows of q and k */
  int32_t max_nq, max_nk;          /* largest complex */
  int64_t n_pairs;
  float scale;                     /* 2^-126 .. 2^126 */
  int32_t splits;                  /* ranges of keys (backward: of rows, too) per workgroup that are joined afterwards, up to 64; 0 = chosen by the library */
  /* strides in elements; the last dimension has unit stride */
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, dout_row, dout_head, bias_head, bias_pair;
  const int32_t *q_ptr, *k_ptr;    /* [B+1] */
  const int64_t* pair_ptr;         /* [B+1] */
  const int32_t* order;            /* [B] the complexes, most pairs first: the order in which their row blocks are started */
  const void *q, *k, *v, *bias;    /* [n_q, heads, dim], [n_k, kv_heads, dim] x2, [heads, n_pairs] or NULL */
  void* out;                       /* [n_q, heads, dim] contiguous (forward: written; backward: read) */
  float* stats;                    /* [2, heads, n_q]: m, then l */
  const void* dout;
  void *dq, *dk, *dv, *dbias;      /* contiguous, as q, k, v, bias; dbias NULL iff bias is NULL or its gradient is not wanted */
  void* ws;                        /* dpt_attn_ws_bytes() bytes, 16-byte aligned */
  size_t ws_bytes;
} DptAttnArgs;

size_t dpt_attn_ws_bytes(const DptAttnArgs* a, int32_t backward);
int dpt_attn_fwd(const DptAttnArgs* a, void* stream);
int dpt_attn_bwd(const DptAttnArgs* a, void* stream);

/* ---- AdamW over many tensors ----------------------------------------------------------------------------------------------------------------
 *   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2  with g = grad_scale * gradient
 *   p = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps);   ema = d ema + (1 - d) p
 * State lives in flat buffers: tensor i owns the 256-element blocks first_block[i] .. first_block[i+1]; what pads its last block stays 0.
 * state_bits 8: m = a c|c| / 127^2 (c int8), v = a (c / 255)^4 (c uint8, never 0 where v > 0) with one fp32 scale a per block, its largest
 * magnitude; codes are the nearest on the curve's axis.  A block whose new m or v is not finite gets the scale NaN.
 * type BF16: the parameters are the roundings of fp32 masters. */
#define DPT_ADAMW_BLOCK 256
#define DPT_ADAMW_MAX_TENSORS 400  /* tensors per call; the host splits longer lists (`last` on the last call of a step) */

/* where a block's elements are; one record per block, held on the device */
typedef struct DptAdamWBlock {
  uint64_t param;                  /* address of the block's first parameter */
  int32_t tensor, index;           /* its tensor, and its number inside it */
  int32_t left;                    /* elements of the tensor from the block's first on, 256 at most */
  float decay;                     /* factor of weight_decay: 1 or 0 */
  int32_t pad_[2];
} DptAdamWBlock;

typedef struct DptAdamWArgs {
  int32_t type, grad_type;         /* fp32/fp32, bf16/bf16 or bf16/fp32 */
  int32_t state_bits;              /* 8 or 32 */
  int32_t n_tensors;               /* of this call */
  int32_t block0, n_blocks;        /* the blocks of this call's tensors */
  int32_t last;                    /* advance the step counter afterwards */
  double lr, beta1, beta2, eps, weight_decay, ema_decay;
  const float* lr_dev;             /* NULL, or the learning rate (then `lr` is not read) */
  const float* grad_scale;         /* NULL, or the factor of the gradients */
  const DptAdamWBlock* blocks;     /* [all blocks] */
  int32_t tensor0, pad_;           /* this call's first tensor */
  float* master;                   /* bf16: [all blocks * 256] */
  float* ema;                      /* NULL or [all blocks * 256] */
  void *exp_avg, *exp_avg_sq;      /* [all blocks * 256] fp32, or int8 / uint8 */
  float *exp_avg_scale, *exp_avg_sq_scale; /* 8 bits: [all blocks] */
  double* counter;                 /* [4]: steps done, b1^t, b2^t of them, and a ticket (uint32) that is 0 between calls */
} DptAdamWArgs;

/* grads: HOST array of n_tensors device pointers (copied into the launch) */
int dpt_adamw_step(const DptAdamWArgs* a, const void* const* grads, void* stream);
/* the fp32 values that 8-bit states stand for */
int dpt_adamw_moments(const void* exp_avg, const float* exp_avg_scale, const void* exp_avg_sq, const float* exp_avg_sq_scale, int32_t n_blocks,
                      float* m, float* v, void* stream);

#ifdef __cplusplus
}
#endif
#endif
