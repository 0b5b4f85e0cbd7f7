/*
 * onereel_dit.h: C ABI of libonereel_dit.so, the linear layers and fused elementwise kernels of the Wan-shaped DiT block
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

#ifdef __cplusplus
}
#endif

#endif /* ONEREEL_DIT_H */
