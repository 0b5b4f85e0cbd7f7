// Microscaled 4-bit floating point (OCP MXFP4) for the linear layers of the DiT block: quantisation, reading back, and the product of
// 4-bit rows with the epilogue of the bf16 layers. Built into libonereel_dit.so (include/onereel_dit.h).
//
//   a row is divided into blocks of 32 elements; s = 2^(floor(log2(max |x|)) - 2) of a block, at least 2^-127, held as its
//   biased exponent in 8 bits (e8m0); an element is held as the e2m1 value (0, 0.5, 1, 1.5, 2, 3, 4, 6, and a sign) nearest to
//   x / s, ties to the even code, values past 6 as 6, two to a byte with the even element in the low half
//   y = residual + gate * act(x^ W^T + b)    with x^ and W the values that codes and scales stand for
//
// A block that holds an infinity or a NaN gets the scale 255, which stands for NaN, and all that is computed from it is NaN.
// x / s is exact (a power of two), so the choice of the code has no rounding but its own, and no result depends on the order of
// anything. The products of codes are exact too; sums and scales are the matrix cores', in fp32.
#include <algorithm>

#include "rows.h"
#include "tiles.h"

namespace onereel {

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 32;

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------------------------------------------------------
// quantisation

struct QuantizeArgs {
  const void* x;
  uint8_t *codes, *scales;             // [rows][K / 2], [rows][K / 32]
  int64_t rows, x_stride;
  int K;
};

// the e8m0 scale of a block from the bits of its largest magnitude, and what its elements are multiplied by
__device__ __forceinline__ uint32_t scale_of(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}
__device__ __forceinline__ float inverse_of(uint32_t scale) { return __uint_as_float((254u - min(scale, 253u)) << 23); }

__device__ __forceinline__ uint32_t code_of(float v) {
  const float m = fabsf(v);
  const uint32_t c = (m > 0.25f) + (m >= 0.75f) + (m > 1.25f) + (m >= 1.75f) + (m > 2.5f) + (m >= 3.5f) + (m > 5.0f);
  return c | (__float_as_uint(v) >> 28 & 8u);
}

// the largest over 4 neighbouring lanes
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, false));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, false));
}

// 8 elements a lane, 4 lanes a block
template <typename T>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(QuantizeArgs g) {
  const int per = g.K / 8;
  const int64_t total = g.rows * per;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per;
    const int c = (int)(i - row * per);
    Piece<T, 8> p;
    float v[8];
    p.load(g.x, row * g.x_stride + 8 * c);
    p.get(v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
    const uint32_t scale = scale_of(quad_max(top));
    const float inverse = inverse_of(scale);
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) codes |= code_of(v[k] * inverse) << (4 * k);
    ((uint32_t*)g.codes)[i] = scale == 255 ? 0 : codes;
    if ((c & 3) == 0) g.scales[i >> 2] = (uint8_t)scale;
  }
}

// what a scale stands for
__device__ __forceinline__ float unit_of(uint32_t scale) {
  return __uint_as_float(scale == 255 ? 0x7fc00000u : scale == 0 ? 0x00400000u : scale << 23);
}

__device__ __forceinline__ float value_of(uint32_t code) {
  const uint32_t m = code & 7u;
  const float f = m < 2 ? 0.5f * (float)m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
  return code & 8u ? -f : f;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(const uint32_t* codes, const uint8_t* scales, void* out, int64_t total) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const uint32_t c = codes[i];
    const float unit = unit_of(scales[i >> 2]);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = value_of(c >> (4 * k) & 15u) * unit;
    Piece<T, 8>::store(out, 8 * i, v);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// product

struct MxArgs {
  const uint8_t *a, *a_scales, *b, *b_scales;   // x and W
  int64_t I;
  int J, K;
  Epilogue e;
};

// A wavefront takes 32 rows of x and 32 columns; W's rows are the rows of the matrix tile, so that a lane holds runs of 4 columns
// of one row.
__global__ __launch_bounds__(64) void mx_small_kernel(MxArgs g) {
  __shared__ float st[32 * 36];
  const int lane = threadIdx.x, l32 = lane & 31, h = lane >> 5;
  const int64_t tiles_j = (g.J + 31) / 32, i0 = blockIdx.x / tiles_j * 32;
  const int j0 = (int)(blockIdx.x % tiles_j) * 32;
  const int64_t ar = min(i0 + l32, g.I - 1), br = min(j0 + l32, g.J - 1);
  f32x16 acc = {};
  for (int k = 32 * h; k < g.K + 32 * h; k += 64) {
    const bool in = k < g.K;
    i32x8 a = {}, b = {};
    int as = 0, bs = 0;
    if (in) {
      const u32x4 x = *(const u32x4*)(g.a + ar * (g.K / 2) + k / 2), w = *(const u32x4*)(g.b + br * (g.K / 2) + k / 2);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        a[t] = (int)x[t];
        b[t] = (int)w[t];
      }
      as = g.a_scales[ar * (g.K / 32) + k / 32];
      bs = g.b_scales[br * (g.K / 32) + k / 32];
    }
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, acc, 4, 4, 0, bs, 0, as);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *(f32x4*)(st + l32 * 36 + 8 * q + 4 * h) = f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  for (int x = lane; x < 128; x += 64) {
    const int64_t row = i0 + x / 4;
    const int col = j0 + 8 * (x % 4);
    if (row >= g.I || col >= g.J) continue;
    float v[8];
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = st[x / 4 * 36 + 8 * (x % 4) + t];
    finish8(g.e, row, col, g.J, v);
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
constexpr int64_t kMaxStride = 1 << 21;

int check_rows(const char* what, int64_t rows, int32_t K) {
  if (rows < 0 || rows > (int64_t)1 << 30) return fail_arg("%s: 0 to 2^30 rows (got %lld)", what, (long long)rows);
  if (K < kBlock || K % kBlock || K > kMaxStride) return fail_arg("%s: rows of a multiple of 32 elements up to 2^21 (got %d)", what, K);
  return 0;
}

int check_product(const char* what, int64_t M, int32_t K, int32_t N) {
  if (int rc = check_rows(what, M, K)) return rc;
  if (N < 8 || N % 8 || N > kMaxStride) return fail_arg("%s: n_out must be a multiple of 8 up to 2^21 (got %d)", what, N);
  return 0;
}

unsigned blocks_for(int64_t total) { return (unsigned)std::min<int64_t>((total + kThreads - 1) / kThreads, 256 * 32); }

void launch_quantize(const QuantizeArgs& g, int type, hipStream_t st) {
  const dim3 grid(blocks_for(g.rows * (g.K / 8)));
  if (type == OR_TYPE_BF16) hipLaunchKernelGGL(mx_quantize_kernel<Bf16>, grid, dim3(kThreads), 0, st, g);
  else if (type == OR_TYPE_FP16) hipLaunchKernelGGL(mx_quantize_kernel<_Float16>, grid, dim3(kThreads), 0, st, g);
  else hipLaunchKernelGGL(mx_quantize_kernel<float>, grid, dim3(kThreads), 0, st, g);
}

int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int or_mx_quantize(const void* x, int64_t n_rows, int32_t n, int64_t x_row_stride, int32_t type, void* codes,
                              void* scales, void* stream) {
  if (!known_type(type)) return fail_arg("or_mx_quantize: unknown element type %d", type);
  if (int rc = check_rows("or_mx_quantize", n_rows, n)) return rc;
  if (n_rows == 0) return 0;
  if (!x || !codes || !scales) return fail_arg("or_mx_quantize: x, codes and scales are required");
  if (!al16(x) || !al16(codes) || x_row_stride < n || x_row_stride % 8)
    return fail_arg("or_mx_quantize: 16-byte aligned x and codes, rows a multiple of 8 elements apart that cover n");
  launch_quantize(QuantizeArgs{x, (uint8_t*)codes, (uint8_t*)scales, n_rows, x_row_stride, n}, type, (hipStream_t)stream);
  return check_hip(hipGetLastError(), "mx_quantize_kernel launch");
}

extern "C" int or_mx_dequantize(const void* codes, const void* scales, int64_t n_rows, int32_t n, int32_t type, void* out,
                                void* stream) {
  if (!known_type(type)) return fail_arg("or_mx_dequantize: unknown element type %d", type);
  if (int rc = check_rows("or_mx_dequantize", n_rows, n)) return rc;
  if (n_rows == 0) return 0;
  if (!codes || !scales || !out || !al16(codes) || !al16(out))
    return fail_arg("or_mx_dequantize: 16-byte aligned codes and out, and scales, are required");
  const int64_t total = n_rows * (n / 8);
  const dim3 grid(blocks_for(total));
  hipStream_t st = (hipStream_t)stream;
  const uint32_t* c = (const uint32_t*)codes;
  const uint8_t* s = (const uint8_t*)scales;
  if (type == OR_TYPE_BF16) hipLaunchKernelGGL(mx_dequantize_kernel<Bf16>, grid, dim3(kThreads), 0, st, c, s, out, total);
  else if (type == OR_TYPE_FP16) hipLaunchKernelGGL(mx_dequantize_kernel<_Float16>, grid, dim3(kThreads), 0, st, c, s, out, total);
  else hipLaunchKernelGGL(mx_dequantize_kernel<float>, grid, dim3(kThreads), 0, st, c, s, out, total);
  return check_hip(hipGetLastError(), "mx_dequantize_kernel launch");
}

extern "C" int64_t or_mx_linear_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t quantized) {
  if (int rc = check_product("or_mx_linear_workspace_size", n_rows, n_in, n_out)) return rc;
  return quantized ? 0 : round256(n_rows * (n_in / 2)) + round256(n_rows * (n_in / 32));
}

extern "C" int or_mx_linear(const or_mx_linear_args* p, void* stream) {
  if (!p) return fail_arg("or_mx_linear: args is NULL");
  const or_mx_linear_args& x = *p;
  if (int rc = check_product("or_mx_linear", x.n_rows, x.n_in, x.n_out)) return rc;
  if (x.activation != OR_ACT_NONE && x.activation != OR_ACT_GELU_TANH && x.activation != OR_ACT_SILU)
    return fail_arg("or_mx_linear: unknown activation %d", x.activation);
  if (x.n_rows == 0) return 0;
  const bool quantized = !x.x;
  if (quantized && (!x.x_codes || !x.x_scales)) return fail_arg("or_mx_linear: x, or x_codes and x_scales, are required");
  if (!x.weight_codes || !x.weight_scales || !x.y) return fail_arg("or_mx_linear: weight_codes, weight_scales and y are required");
  if (!quantized && (x.x_row_stride < x.n_in || x.x_row_stride % 8)) return fail_arg("or_mx_linear: rows of x must be a multiple of 8 elements apart and cover n_in");
  if (x.y_row_stride < x.n_out || x.y_row_stride % 8 || (x.residual && (x.residual_row_stride < x.n_out || x.residual_row_stride % 8)))
    return fail_arg("or_mx_linear: rows of y and the residual must be a multiple of 8 elements apart and cover n_out");
  if (!al16(x.x) || !al16(x.x_codes) || !al16(x.weight_codes) || !al16(x.bias) || !al16(x.gate) || !al16(x.residual) || !al16(x.y))
    return fail_arg("or_mx_linear: pointers must be 16-byte aligned");
  const int64_t need = or_mx_linear_workspace_size(x.n_rows, x.n_in, x.n_out, quantized);
  if (need > 0 && (!x.workspace || !al16(x.workspace) || x.workspace_bytes < need))
    return fail_arg("or_mx_linear: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  MxArgs g = {};
  g.a = (const uint8_t*)x.x_codes;
  g.a_scales = (const uint8_t*)x.x_scales;
  if (!quantized) {
    uint8_t* codes = (uint8_t*)x.workspace;
    uint8_t* scales = codes + round256(x.n_rows * (x.n_in / 2));
    launch_quantize(QuantizeArgs{x.x, codes, scales, x.n_rows, x.x_row_stride, x.n_in}, OR_TYPE_BF16, st);
    g.a = codes;
    g.a_scales = scales;
  }
  g.b = (const uint8_t*)x.weight_codes;
  g.b_scales = (const uint8_t*)x.weight_scales;
  g.I = x.n_rows;
  g.J = x.n_out;
  g.K = x.n_in;
  g.e = Epilogue{(uint16_t*)x.y, x.y_row_stride, nullptr, x.bias, x.gate, x.bias_bf16, x.gate_bf16, (const uint16_t*)x.residual,
                 x.residual_row_stride, x.activation};
  const int64_t tiles = (g.I + 31) / 32 * ((g.J + 31) / 32);
  if (tiles > (int64_t)1 << 26) return fail_arg("or_mx_linear: too many tiles");
  hipLaunchKernelGGL(mx_small_kernel, dim3((unsigned)tiles), dim3(64), 0, st, g);
  return check_hip(hipGetLastError(), "or_mx_linear launch");
}
