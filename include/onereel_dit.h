/*
 * onereel_dit.h: C ABI of libonereel_dit.so, the linear layers (bf16 and 4-bit), norms and fused elementwise kernels of the
 * Wan-shaped DiT block, and the clipping of its gradients
 * (onereel_amd/wan_dit.py): a random-init model that runs the scene-attention processors end to end so that a
 * denoising step's time can be measured. These kernels are not on the scene-attention path (libonereel_hip.so,
 * include/onereel_hip.h); the library links against libonereel_hip.so and reports errors through its or_last_error.
 *
 * Conventions as in onereel_hip.h: caller-owned device memory, bf16 as uint16_t bits, rows with a row stride in
 * elements, every launch on the given stream (a hipStream_t, NULL = the null stream); 0 on success, -1 for a bad
 * argument, -2 for a HIP error.
 */
#ifndef ONEREEL_DIT_H
#define ONEREEL_DIT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Replaces the LayerNorm + modulation chains of the Wan transformer block the reference's processors run in
 * (diffusers' WanTransformerBlock, third-party; installed at src/onereel/models/wan.py:77-108): per bf16 row of C
 * elements, y = (x - mean) * rstd, then * weight, + bias, * (1 + scale), + shift for each of those fp32 [C] vectors
 * that is not NULL, in that order and in fp32; out = bf16(y). */
int or_layernorm_modulate(const void* x, void* out, int64_t n_rows, int32_t C, int64_t x_row_stride,
                          int64_t out_row_stride, float eps, const float* weight, const float* bias, const float* scale,
                          const float* shift, void* stream);

/* Replaces the block's residual adds (same block): x = bf16(float(x) + float(a) * gate), gate fp32 [C], or
 * x = bf16(float(x) + float(a)) when gate is NULL; in place on x. */
int or_gated_residual(void* x, const void* a, const float* gate, int64_t n_rows, int32_t C, int64_t x_row_stride,
                      int64_t a_row_stride, void* stream);

/* Replaces a residual add of the block followed by the next LayerNorm + modulation (the same block, or the next
 * block's first norm): or_gated_residual on x, then or_layernorm_modulate of the updated x into out, with the same
 * results bit for bit, in one pass over the rows when C <= 4096 (two passes above). out must be neither x nor a. */
int or_residual_layernorm_modulate(void* x, const void* a, const float* gate, void* out, int64_t n_rows, int32_t C,
                                   int64_t x_row_stride, int64_t a_row_stride, int64_t out_row_stride, float eps,
                                   const float* weight, const float* bias, const float* scale, const float* shift,
                                   void* stream);

/* norms of or_block_norm */
#define OR_NORM_NONE 0
#define OR_NORM_LAYER 1       /* (v - mean v) / sqrt(mean (v - mean v)^2 + eps) */
#define OR_NORM_RMS 2         /* v / sqrt(mean v^2 + eps) */

/* Arguments of or_block_norm: h = residual_scale x + gate post_norm(a) post_weight and
 * n = (norm(h) weight + bias) (1 + scale) + shift, per row, fp32 inside; h is rounded once, and n comes from h before that.
 * Without a (then without gate, post_norm, post_weight and h) n is that of x itself. */
typedef struct or_block_norm_args {
  const void* x;              /* [n_rows, C], row stride x_row_stride */
  const void* a;              /* optional [n_rows, C], row stride a_row_stride: the sub-block's output */
  void* h;                    /* [n_rows, C], contiguous; with a */
  void* n;                    /* [n_rows, C], contiguous */
  const float* gate;          /* optional [n_rows / rows_per_group, C]: one vector for rows_per_group consecutive rows */
  const float* post_weight;   /* optional [C] */
  const float* weight;        /* optional [C] */
  const float* bias;          /* optional [C] */
  const float* scale;         /* optional [n_rows / rows_per_group, C] */
  const float* shift;         /* optional [n_rows / rows_per_group, C] */
  int64_t n_rows;             /* up to 2^30 */
  int64_t rows_per_group;     /* divides n_rows */
  int64_t x_row_stride;       /* elements; multiples of 8 */
  int64_t a_row_stride;
  int32_t C;                  /* a multiple of 8 up to 8192 */
  int32_t type;               /* OR_TYPE_* of x, a, h and n */
  int32_t norm;               /* OR_NORM_LAYER or OR_NORM_RMS */
  int32_t post_norm;          /* OR_NORM_* */
  float eps;
  float residual_scale;
} or_block_norm_args;

/* Replaces the residual add of the Wan transformer block and the norm with modulation that follows it (diffusers'
 * WanTransformerBlock, third-party; the blocks the processors are installed in, src/onereel/models/wan.py:77-108), as
 * or_residual_layernorm_modulate does in place, for training (nothing is updated in place), with gate, scale and shift for every
 * group of rows, RMS norms, a norm of the sub-block's output, and all three element types. One launch. Rows and parameters lie at
 * 16-byte aligned addresses. */
int or_block_norm(const or_block_norm_args* args, void* stream);

/* Arguments of or_block_norm_bwd: the gradient of one or_block_norm call. h is the call's h (its x without a). */
typedef struct or_block_norm_bwd_args {
  const void* dh;             /* optional [n_rows, C]: the gradient of h from what else read it; with a */
  const void* dn;             /* [n_rows, C] */
  const void* h;              /* [n_rows, C] */
  const void* a;              /* the call's a or NULL */
  void* dx;                   /* [n_rows, C], contiguous */
  void* da;                   /* [n_rows, C], contiguous; with a */
  const float* gate;          /* the call's parameters */
  const float* post_weight;
  const float* weight;
  const float* bias;
  const float* scale;
  float* dgate;               /* each optional: [n_rows / rows_per_group, C], */
  float* dpost_weight;        /* [C], */
  float* dweight;             /* [C], */
  float* dbias;               /* [C], */
  float* dscale;              /* [n_rows / rows_per_group, C], */
  float* dshift;              /* [n_rows / rows_per_group, C] */
  int64_t n_rows;
  int64_t rows_per_group;
  int64_t dh_row_stride;      /* elements; multiples of 8 */
  int64_t dn_row_stride;
  int64_t h_row_stride;
  int64_t a_row_stride;
  int32_t C;
  int32_t type;               /* OR_TYPE_* of dh, dn, h, a, dx and da */
  int32_t norm;
  int32_t post_norm;
  float eps;
  float residual_scale;
  void* workspace;            /* device scratch of or_block_norm_bwd_workspace_size() bytes; with one of the sums over rows */
  int64_t workspace_bytes;
} or_block_norm_bwd_args;

/* Bytes of device workspace or_block_norm_bwd needs for the sums over rows. Negative for sizes it refuses. */
int64_t or_block_norm_bwd_workspace_size(int64_t n_rows, int64_t rows_per_group, int32_t C);

/* The gradient of or_block_norm. Sums are fp32 in a fixed order; dx and da are rounded once. With 0 rows nothing is written.
 * One launch; with sums over rows up to three. Rows, parameters and the parameters' gradients lie at 16-byte aligned addresses. */
int or_block_norm_bwd(const or_block_norm_bwd_args* args, void* stream);

/* activations of or_linear */
#define OR_ACT_NONE 0
#define OR_ACT_GELU_TANH 1    /* 0.5 z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) */
#define OR_ACT_SILU 2         /* z / (1 + exp(-z)) */

/* Arguments of or_linear: y = residual + gate * act(z), z = x weight^T + bias, fp32 from the bf16 operands to the one
 * rounding of y (and of z, when it is kept). */
typedef struct or_linear_args {
  const void* x;            /* bf16 [n_rows, n_in], row stride x_row_stride */
  const void* weight;       /* bf16 [n_out, n_in], row stride weight_row_stride */
  const void* bias;         /* optional fp32 [n_out] (bf16 with bias_bf16) */
  const void* gate;         /* optional fp32 [n_out] (bf16 with gate_bf16), the same for every row */
  const void* residual;     /* optional bf16 [n_rows, n_out], row stride residual_row_stride; may be y itself */
  void* y;                  /* bf16 [n_rows, n_out], row stride y_row_stride */
  void* preactivation;      /* optional bf16 [n_rows, n_out], contiguous: z, for or_linear_bwd */
  int64_t n_rows;
  int64_t x_row_stride;     /* elements; multiples of 8 up to 2^21 */
  int64_t weight_row_stride;
  int64_t residual_row_stride;
  int64_t y_row_stride;
  int32_t n_in;             /* multiples of 8 up to 2^21 */
  int32_t n_out;
  int32_t activation;       /* OR_ACT_* */
  int32_t bias_bf16;
  int32_t gate_bf16;
  void* workspace;          /* device scratch of or_linear_workspace_size() bytes */
  int64_t workspace_bytes;
} or_linear_args;

/* Bytes of device workspace or_linear needs: fp32 partial products where the call has so few tiles that n_in is split
 * over several work-groups, 0 for others. Negative for sizes it refuses. */
int64_t or_linear_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out);

/* Replaces the Linear layers of the Wan transformer block with what follows them (diffusers' WanTransformerBlock and its
 * feed forward, third-party; the blocks the processors are installed in, src/onereel/models/wan.py:77-108): bias,
 * activation, the block's gate and its residual add in the product's epilogue. One launch, or two where n_in is split. */
int or_linear(const or_linear_args* args, void* stream);

/* Arguments of or_linear_bwd: the gradients of one or_linear call, each optional (NULL: not computed). The gradient of the
 * residual is dy itself. */
typedef struct or_linear_bwd_args {
  const void* dy;            /* bf16 [n_rows, n_out], row stride dy_row_stride */
  const void* x;             /* the call's x (for dweight) */
  const void* weight;        /* its weight (for dx) */
  const void* preactivation; /* its preactivation, contiguous (for an activation, and for dgate) */
  const void* gate;          /* its gate or NULL */
  void* dx;                  /* bf16 [n_rows, n_in], contiguous */
  void* dweight;             /* bf16 [n_out, n_in], contiguous */
  float* dbias;              /* fp32 [n_out] */
  float* dgate;              /* fp32 [n_out] */
  int64_t n_rows;
  int64_t dy_row_stride;     /* elements; multiples of 8 up to 2^21 */
  int64_t x_row_stride;
  int64_t weight_row_stride;
  int32_t n_in;
  int32_t n_out;
  int32_t activation;
  int32_t gate_bf16;
  void* workspace;           /* device scratch of or_linear_bwd_workspace_size() bytes */
  int64_t workspace_bytes;
} or_linear_bwd_args;

/* Bytes of device workspace or_linear_bwd needs; scaled: whether the call has an activation or a gate. Negative for sizes it
 * refuses. */
int64_t or_linear_bwd_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t scaled);

/* The gradient of or_linear: dz = dy * gate * act'(z), dx = dz weight, dweight = dz^T x, dbias = sum of dz over rows and
 * dgate = sum of dy * act(z) over rows. Sums are fp32 in a fixed order; dx and dweight are rounded to bf16 once, and dz is
 * rounded to bf16 as an operand of their products (not in dbias). Up to five launches. */
int or_linear_bwd(const or_linear_bwd_args* args, void* stream);

/* How a product is computed at these sizes: product 0 is or_linear's, 1 and 2 are or_linear_bwd's dx and dweight. tile: rows
 * and columns of a work-group's tile (256, 128 or 64; 0: or_linear's kernels for few rows), buffers: LDS buffers of its ring
 * (0 with them), split: parts of the summed axis. Host only. */
int or_linear_plan(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t product, int32_t* tile, int32_t* buffers,
                   int32_t* split);

/* Rows of n elements (a multiple of 32) in microscaled 4-bit floating point (OCP MXFP4): n / 32 scales, each the biased exponent of a
 * power of two s for 32 elements (255: NaN), and n / 2 bytes of codes, two e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) in
 * each with the even element in the low half. A block's s is 2^(floor(log2 max|x|) - 2), at least 2^-127; an element is the value
 * nearest to x / s, ties to the even code, past 6 as 6; a block with an infinity or a NaN gets the scale 255. x: n_rows up to 2^30 of
 * n up to 2^21 elements of OR_TYPE_*, row stride in elements (a multiple of 8); codes and scales contiguous. */
int or_mx_quantize(const void* x, int64_t n_rows, int32_t n, int64_t x_row_stride, int32_t type, void* codes, void* scales,
                   void* stream);

/* The values that codes and scales stand for, into contiguous rows of OR_TYPE_* elements. */
int or_mx_dequantize(const void* codes, const void* scales, int64_t n_rows, int32_t n, int32_t type, void* out, void* stream);

/* Arguments of or_mx_linear: or_linear with x and the weight in 4 bits. */
typedef struct or_mx_linear_args {
  const void* x;              /* bf16 [n_rows, n_in], row stride x_row_stride, quantised by the call; or NULL, then */
  const void* x_codes;        /* [n_rows, n_in / 2] and */
  const void* x_scales;       /* [n_rows, n_in / 32], contiguous */
  const void* weight_codes;   /* [n_out, n_in / 2], contiguous */
  const void* weight_scales;  /* [n_out, n_in / 32], contiguous */
  const void* bias;           /* optional fp32 [n_out] (bf16 with bias_bf16) */
  const void* gate;           /* optional fp32 [n_out] (bf16 with gate_bf16) */
  const void* residual;       /* optional bf16 [n_rows, n_out], row stride residual_row_stride; may be y itself */
  void* y;                    /* bf16 [n_rows, n_out], row stride y_row_stride */
  int64_t n_rows;             /* up to 2^30 */
  int64_t x_row_stride;       /* elements; multiples of 8 */
  int64_t residual_row_stride;
  int64_t y_row_stride;
  int32_t n_in;               /* a multiple of 32 up to 2^21 */
  int32_t n_out;              /* a multiple of 8 up to 2^21 */
  int32_t activation;         /* OR_ACT_* */
  int32_t bias_bf16;
  int32_t gate_bf16;
  void* workspace;            /* device scratch of or_mx_linear_workspace_size() bytes */
  int64_t workspace_bytes;
} or_mx_linear_args;

/* Bytes of device workspace or_mx_linear needs (quantized: x comes in 4 bits). Negative for sizes it refuses. */
int64_t or_mx_linear_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t quantized);

/* How or_mx_linear computes a product of these sizes, as or_linear_plan tells of or_linear: tile (256, 128 or 64; 0: the kernel for
 * few rows), LDS buffers of its ring (0 with that), parts of n_in. Host only. */
int or_mx_linear_plan(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t* tile, int32_t* buffers, int32_t* split);

/* Replaces the Linear layers of the Wan transformer block with what follows them, as or_linear does (diffusers'
 * WanTransformerBlock, third-party; the blocks the processors are installed in, src/onereel/models/wan.py:77-108), for inference
 * with 4-bit weights and activations: y = residual + gate * act(x weight^T + bias) of the values in 4 bits, fp32 from the products to
 * the one rounding of y. */
int or_mx_linear(const or_mx_linear_args* args, void* stream);

/* Arguments of or_clip. The arrays lie in host memory and are read before the call returns. */
typedef struct or_clip_args {
  const void* const* x;       /* [n_tensors] device addresses of contiguous elements, aligned to their type */
  const int64_t* numel;       /* [n_tensors], 0 to 2^40 */
  const int32_t* type;        /* [n_tensors] OR_TYPE_* */
  void* const* out;           /* optional [n_tensors] device addresses: x's own (in place) or memory that no x shares; NULL: the
                                 norm alone */
  const int32_t* out_type;    /* optional [n_tensors] OR_TYPE_* of out (NULL: as type; that of x where out is x) */
  int64_t n_tensors;
  double max_norm;            /* 0 or more */
  float* norm;                /* device: the norm of all x before scaling */
  void* workspace;            /* device scratch of or_clip_workspace_size() bytes */
  int64_t workspace_bytes;
} or_clip_args;

/* Bytes of device workspace or_clip needs for these tensors. Negative for arguments it refuses. */
int64_t or_clip_workspace_size(const or_clip_args* args);

/* The clipping of a training step's gradients, which the reference, an inference system, leaves to its trainer (torch's
 * clip_grad_norm_): norm = sqrt(sum of all x^2) and out = x min(1, max_norm / (norm + 1e-6)); in place, nothing is written where
 * that factor is 1. Squares are summed in fp64 in a fixed order. Two launches for each 128 tensors. */
int or_clip(const or_clip_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ONEREEL_DIT_H */
