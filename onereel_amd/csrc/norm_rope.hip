// Fused RMSNorm + interleaved RoPE of the Wan self-attention's queries and keys, one launch for both.
//
// Reference: _qk (src/onereel/models/wan.py:64-74), compiled there with torch.compile: per token row x [C] (C = H * D,
// the norm spans every head, diffusers' 'rms_norm_across_heads'):
//   y = x / sqrt(mean(x^2) + eps) * w
// then per head, for the interleaved pairs (2i, 2i+1) of its D dims, with c = cos[row, 2i] and s = sin[row, 2i+1]
// (cos[..., 0::2], sin[..., 1::2]):
//   out[2i] = y[2i] c - y[2i+1] s,   out[2i+1] = y[2i] s + y[2i+1] c,
// cast to bf16 (type_as(x)). Here the whole chain is fp32 with one rounding at the end, as the compiled graph computes
// it; the bf16 input is read once and the bf16 output written once.
//
// HBM-bound: 2 * C * 2 bytes per row and tensor, plus the row's cos / sin entries (2 * D * 4 bytes, shared by its
// heads). One wavefront per row: each lane holds C / 512 16-byte chunks, the sum of squares is reduced across the
// wavefront, and every lane's chunks sit at the same dims of their heads (512 elements = a whole number of heads for
// D dividing 512), so each lane loads its cos / sin entries once per row.
#include <math.h>

#include "common.h"

namespace onereel {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxChunks = 16;   // rows up to 64 lanes * 16 chunks * 8 = 8192 elements

struct NormRopeArgs {
  const uint16_t* x[2];
  uint16_t* out[2];
  const uint16_t* w[2];          // bf16 [C]
  int64_t x_stride[2], out_stride[2];
  const float* cos_t;
  const float* sin_t;
  const int32_t* rope_row;       // per token row, or NULL: the token row itself
  int64_t n_rows, n_rope_rows;
  int C, D;
  float eps;
};

// One row's inputs: its bf16 words, and this lane's cos / sin entries (d0 = 8 lane mod D, pairs 2p, 2p + 1).
template <int NCH>
struct RowIn {
  u32x4 x[NCH];
  float c[4], s[4];
};

template <int NCH>
__device__ __forceinline__ void load_row(const NormRopeArgs& g, int which, int64_t r, int lane, RowIn<NCH>& in) {
  const uint16_t* xp = g.x[which] + r * g.x_stride[which];
#pragma unroll
  for (int i = 0; i < NCH; ++i) in.x[i] = *(const u32x4*)(xp + 8 * (lane + 64 * i));
  const int rr = g.rope_row ? g.rope_row[r] : (int)r;
  const int d0 = (8 * lane) % g.D;
  const bool rot = rr >= 0 && rr < g.n_rope_rows;   // rows outside the table (or no table) are not rotated
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    in.c[p] = rot ? g.cos_t[(int64_t)rr * g.D + d0 + 2 * p] : 1.0f;
    in.s[p] = rot ? g.sin_t[(int64_t)rr * g.D + d0 + 2 * p + 1] : 0.0f;
  }
}

template <int NCH>
__device__ __forceinline__ void norm_rope_row(const NormRopeArgs& g, int which, int64_t r, int lane,
                                              const RowIn<NCH>& in, const uint16_t* w) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float a = bf2f((uint16_t)(in.x[i][p] & 0xffffu)), b = bf2f((uint16_t)(in.x[i][p] >> 16));
      ss += a * a + b * b;
    }
  }
  const float inv = 1.0f / sqrtf(wave_sum(ss) / (float)g.C + g.eps);
  uint16_t* op = g.out[which] + r * g.out_stride[which];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int e = 8 * (lane + 64 * i);
    const u32x4 wv = *(const u32x4*)(w + e);
    u32x4 o;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
#pragma clang fp contract(off)
      const float y0 = bf2f((uint16_t)(in.x[i][p] & 0xffffu)) * inv * bf2f((uint16_t)(wv[p] & 0xffffu));
      const float y1 = bf2f((uint16_t)(in.x[i][p] >> 16)) * inv * bf2f((uint16_t)(wv[p] >> 16));
      o[p] = pack2(y0 * in.c[p] - y1 * in.s[p], y0 * in.s[p] + y1 * in.c[p]);
    }
    __builtin_nontemporal_store(o, (u32x4*)(op + e));
  }
}

// blockIdx.y picks q or k. The block stages its weight row in LDS; each wavefront takes one row at a time, and the
// other wavefronts of its SIMD cover the load latency.
template <int NCH>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs g) {
  __shared__ __attribute__((aligned(16))) uint16_t wl[64 * 8 * NCH];
  const int lane = threadIdx.x & 63;
  const int which = blockIdx.y;
  for (int e = 8 * threadIdx.x; e < g.C; e += 8 * kThreads) *(u32x4*)(wl + e) = *(const u32x4*)(g.w[which] + e);
  __syncthreads();
  const int64_t stride = (int64_t)gridDim.x * kWaves;
  for (int64_t r = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6); r < g.n_rows; r += stride) {
    RowIn<NCH> a;
    load_row<NCH>(g, which, r, lane, a);
    norm_rope_row<NCH>(g, which, r, lane, a, wl);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// The gradient. With n = x inv, y = n w, out = R y (R the rotation) and dout:
//   g = R^T dout: g[2i] = dout[2i] c + dout[2i+1] s, g[2i+1] = dout[2i+1] c - dout[2i] s
//   dw = sum over rows of g n,   dx = inv (t - n mean(t n)) with t = g w
// fp32 inside, dx rounded to bf16 once, dw fp32. HBM-bound: x and dout are read once and dx is written once, 6 bytes an
// element. One wavefront per row, as forward; a wavefront adds up dw of its rows in registers, the block's four
// wavefronts add theirs in LDS, and every block writes one fp32 row of partial sums, which a second launch adds up. Rows
// and partial sums are dealt out by index, so the sums' order, and their bits, do not depend on scheduling.
// q and k together: 12 720 rows of 2048 57 to 67 us (4.7 to 5.5 TB/s), two wavefronts a SIMD; 29 040 rows of the 24 heads x 128 of
// the Wan-shaped DiT 210 us (5.1 TB/s) and 12 720 of 4096 136 (4.6) with one; rows of 8192 do not fit a wavefront's registers
// beside their dw and spill: 6000 of them 547 us (1.1 TB/s).
constexpr int kBwdBlocks = 512;      // blocks of q, and of k: 2 x 4 MB of partial sums at C = 2048
constexpr int kSumWaves = 16;

struct NormRopeBwdArgs {
  const uint16_t* dy[2];
  const uint16_t* x[2];
  const uint16_t* w[2];
  uint16_t* dx[2];
  float* dw[2];
  int64_t dy_stride[2], x_stride[2];
  float* part;                       // [2][blocks][C]
  const float* cos_t;
  const float* sin_t;
  const int32_t* rope_row;
  int64_t n_rows, n_rope_rows;
  int C, D, blocks;
  float eps;
};

template <int NCH>
__global__ __launch_bounds__(kThreads) void norm_rope_bwd_kernel(NormRopeBwdArgs g) {
  constexpr int kC = 512 * NCH;
  __shared__ __attribute__((aligned(16))) float sum[kC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y;
  const uint16_t* wp = g.w[which];
  u32x4 wv[NCH];
  float dw[NCH][8];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    wv[i] = *(const u32x4*)(wp + 8 * (lane + 64 * i));
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
  }
  const int d0 = (8 * lane) % g.D;
  const int64_t step = (int64_t)gridDim.x * kWaves;
  for (int64_t r = (int64_t)blockIdx.x * kWaves + wave; r < g.n_rows; r += step) {
    const uint16_t* xp = g.x[which] + r * g.x_stride[which];
    const uint16_t* dp = g.dy[which] + r * g.dy_stride[which];
    u32x4 x[NCH], d[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) x[i] = *(const u32x4*)(xp + 8 * (lane + 64 * i));
#pragma unroll
    for (int i = 0; i < NCH; ++i) d[i] = *(const u32x4*)(dp + 8 * (lane + 64 * i));
    const int64_t rr = g.rope_row ? g.rope_row[r] : r;
    const bool rot = rr >= 0 && rr < g.n_rope_rows;
    float c[4], s[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      c[p] = rot ? g.cos_t[rr * g.D + d0 + 2 * p] : 1.0f;
      s[p] = rot ? g.sin_t[rr * g.D + d0 + 2 * p + 1] : 0.0f;
    }
    float ss = 0.0f, tx = 0.0f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float x0 = bf2f((uint16_t)(x[i][p] & 0xffffu)), x1 = bf2f((uint16_t)(x[i][p] >> 16));
        const float e0 = bf2f((uint16_t)(d[i][p] & 0xffffu)), e1 = bf2f((uint16_t)(d[i][p] >> 16));
        const float t0 = (e0 * c[p] + e1 * s[p]) * bf2f((uint16_t)(wv[i][p] & 0xffffu));
        const float t1 = (e1 * c[p] - e0 * s[p]) * bf2f((uint16_t)(wv[i][p] >> 16));
        ss += x0 * x0 + x1 * x1;
        tx += t0 * x0 + t1 * x1;
      }
    const float inv = 1.0f / sqrtf(wave_sum(ss) / (float)kC + g.eps);
    const float k = wave_sum(tx) / (float)kC * inv * inv;    // mean(t n) inv
    uint16_t* op = g.dx[which] + r * kC;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      u32x4 o;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float x0 = bf2f((uint16_t)(x[i][p] & 0xffffu)), x1 = bf2f((uint16_t)(x[i][p] >> 16));
        const float e0 = bf2f((uint16_t)(d[i][p] & 0xffffu)), e1 = bf2f((uint16_t)(d[i][p] >> 16));
        const float g0 = e0 * c[p] + e1 * s[p], g1 = e1 * c[p] - e0 * s[p];
        dw[i][2 * p] += g0 * (x0 * inv);
        dw[i][2 * p + 1] += g1 * (x1 * inv);
        const float t0 = g0 * bf2f((uint16_t)(wv[i][p] & 0xffffu)), t1 = g1 * bf2f((uint16_t)(wv[i][p] >> 16));
        o[p] = pack2(inv * (t0 - x0 * k), inv * (t1 - x1 * k));
      }
      __builtin_nontemporal_store(o, (u32x4*)(op + 8 * (lane + 64 * i)));
    }
  }
  for (int turn = 0; turn < kWaves; ++turn) {
    if (wave == turn)
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          f32x4* at = (f32x4*)(sum + 8 * (lane + 64 * i) + e);
          const f32x4 v = {dw[i][e], dw[i][e + 1], dw[i][e + 2], dw[i][e + 3]};
          *at = turn ? *at + v : v;
        }
    __syncthreads();
  }
  float* out = g.part + ((int64_t)which * g.blocks + blockIdx.x) * kC;
  for (int e = 4 * threadIdx.x; e < kC; e += 4 * kThreads) *(f32x4*)(out + e) = *(const f32x4*)(sum + e);
}

// dw: 64 columns a block, the blocks' rows of partial sums dealt out to 16 wavefronts
__global__ __launch_bounds__(64 * kSumWaves) void norm_rope_dw_kernel(NormRopeBwdArgs g) {
  __shared__ float sum[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y, col = blockIdx.x * 64 + lane;
  const float* p = g.part + (int64_t)which * g.blocks * g.C + col;
  float v = 0.0f;
#pragma unroll 8
  for (int b = wave; b < g.blocks; b += kSumWaves) v += p[(int64_t)b * g.C];
  sum[wave][lane] = v;
  __syncthreads();
  if (wave == 0) {
    v = 0.0f;
    for (int i = 0; i < kSumWaves; ++i) v += sum[i][lane];
    g.dw[which][col] = v;
  }
}

int bwd_blocks(int64_t n_rows) {
  const int64_t b = (n_rows + kWaves - 1) / kWaves;
  return (int)(b < kBwdBlocks ? b : kBwdBlocks);
}

bool bad_widths(int32_t C, int32_t D) {
  return D < 8 || D % 8 || 512 % D || C % 512 || C < 512 || C > 64 * 8 * kMaxChunks;
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int or_rmsnorm_rope(const void* q, const void* k, const void* wq, const void* wk, int64_t q_row_stride,
                               int64_t k_row_stride, int64_t n_rows, int32_t C, int32_t D, float eps,
                               const float* cos_table, const float* sin_table, const int32_t* rope_row,
                               int64_t n_rope_rows, void* q_out, void* k_out, int64_t qo_row_stride,
                               int64_t ko_row_stride, void* stream) {
  if (n_rows < 0) return fail_arg("or_rmsnorm_rope: n_rows < 0");
  if (D < 8 || D % 8 || 512 % D || C % 512 || C < 512 || C > 64 * 8 * kMaxChunks)
    return fail_arg("or_rmsnorm_rope: need D a multiple of 8 dividing 512 and C a multiple of 512 up to %d "
                    "(C=%d D=%d)", 64 * 8 * kMaxChunks, C, D);
  if (n_rows == 0) return 0;
  if (!q || !wq || !q_out) return fail_arg("or_rmsnorm_rope: q, wq and q_out are required");
  if (n_rope_rows > 0 && (!cos_table || !sin_table))
    return fail_arg("or_rmsnorm_rope: n_rope_rows > 0 needs the cos / sin tables");
  if (n_rope_rows < 0) return fail_arg("or_rmsnorm_rope: n_rope_rows < 0");
  if (k && (!wk || !k_out)) return fail_arg("or_rmsnorm_rope: k needs wk and k_out");
  if (q_row_stride < C || qo_row_stride < C || (k && (k_row_stride < C || ko_row_stride < C)))
    return fail_arg("or_rmsnorm_rope: row strides must cover C elements");
  const uintptr_t al = (uintptr_t)q | (uintptr_t)wq | (uintptr_t)q_out | (uintptr_t)(k ? k : q) |
                       (uintptr_t)(wk ? wk : wq) | (uintptr_t)(k_out ? k_out : q_out);
  if ((al & 15u) || q_row_stride % 8 || qo_row_stride % 8 || (k && (k_row_stride % 8 || ko_row_stride % 8)))
    return fail_arg("or_rmsnorm_rope: pointers must be 16-byte aligned and row strides multiples of 8 elements");
  NormRopeArgs g;
  g.x[0] = (const uint16_t*)q;
  g.x[1] = (const uint16_t*)(k ? k : q);
  g.out[0] = (uint16_t*)q_out;
  g.out[1] = (uint16_t*)(k ? k_out : q_out);
  g.w[0] = (const uint16_t*)wq;
  g.w[1] = (const uint16_t*)(k ? wk : wq);
  g.x_stride[0] = q_row_stride;
  g.x_stride[1] = k ? k_row_stride : q_row_stride;
  g.out_stride[0] = qo_row_stride;
  g.out_stride[1] = k ? ko_row_stride : qo_row_stride;
  g.cos_t = cos_table;
  g.sin_t = sin_table;
  g.rope_row = rope_row;
  g.n_rows = n_rows;
  g.n_rope_rows = n_rope_rows;
  g.C = C;
  g.D = D;
  g.eps = eps;
  int64_t blocks = (n_rows + kWaves - 1) / kWaves;
  if (blocks > 256 * 8) blocks = 256 * 8;
  const dim3 grid((unsigned)blocks, k ? 2 : 1);
  hipStream_t st = (hipStream_t)stream;
  switch (C / 512) {
    case 1: hipLaunchKernelGGL(norm_rope_kernel<1>, grid, dim3(kThreads), 0, st, g); break;
    case 2: hipLaunchKernelGGL(norm_rope_kernel<2>, grid, dim3(kThreads), 0, st, g); break;
    case 3: hipLaunchKernelGGL(norm_rope_kernel<3>, grid, dim3(kThreads), 0, st, g); break;
    case 4: hipLaunchKernelGGL(norm_rope_kernel<4>, grid, dim3(kThreads), 0, st, g); break;
    case 5: hipLaunchKernelGGL(norm_rope_kernel<5>, grid, dim3(kThreads), 0, st, g); break;
    case 6: hipLaunchKernelGGL(norm_rope_kernel<6>, grid, dim3(kThreads), 0, st, g); break;
    case 8: hipLaunchKernelGGL(norm_rope_kernel<8>, grid, dim3(kThreads), 0, st, g); break;
    case 12: hipLaunchKernelGGL(norm_rope_kernel<12>, grid, dim3(kThreads), 0, st, g); break;
    case 16: hipLaunchKernelGGL(norm_rope_kernel<16>, grid, dim3(kThreads), 0, st, g); break;
    default: return fail_arg("or_rmsnorm_rope: C=%d not instantiated (512 x {1..6, 8, 12, 16})", C);
  }
  return check_hip(hipGetLastError(), "norm_rope_kernel launch");
}

extern "C" int64_t or_rmsnorm_rope_bwd_workspace_size(int64_t n_rows, int32_t C) {
  if (n_rows < 0 || C < 512 || C > 64 * 8 * kMaxChunks || C % 512)
    return fail_arg("or_rmsnorm_rope_bwd_workspace_size: need n_rows >= 0 and C a multiple of 512 up to %d",
                    64 * 8 * kMaxChunks);
  return 2 * (int64_t)(bwd_blocks(n_rows) + 1) * C * 4;
}

extern "C" int or_rmsnorm_rope_bwd(const void* dq, const void* dk, const void* q, const void* k, const void* wq,
                                   const void* wk, int64_t dq_row_stride, int64_t dk_row_stride, int64_t q_row_stride,
                                   int64_t k_row_stride, int64_t n_rows, int32_t C, int32_t D, float eps,
                                   const float* cos_table, const float* sin_table, const int32_t* rope_row,
                                   int64_t n_rope_rows, void* q_grad, void* k_grad, float* wq_grad, float* wk_grad,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  if (n_rows < 0) return fail_arg("or_rmsnorm_rope_bwd: n_rows < 0");
  if (bad_widths(C, D))
    return fail_arg("or_rmsnorm_rope_bwd: need D a multiple of 8 dividing 512 and C a multiple of 512 up to %d "
                    "(C=%d D=%d)", 64 * 8 * kMaxChunks, C, D);
  if (n_rope_rows < 0) return fail_arg("or_rmsnorm_rope_bwd: n_rope_rows < 0");
  if (n_rope_rows > 0 && (!cos_table || !sin_table))
    return fail_arg("or_rmsnorm_rope_bwd: n_rope_rows > 0 needs the cos / sin tables");
  if (!wq || !wq_grad || (n_rows > 0 && (!dq || !q || !q_grad)))
    return fail_arg("or_rmsnorm_rope_bwd: dq, q, wq, q_grad and wq_grad are required");
  const bool both = wk != nullptr;
  if (both && (!wk_grad || (n_rows > 0 && (!dk || !k || !k_grad))))
    return fail_arg("or_rmsnorm_rope_bwd: wk needs dk, k, k_grad and wk_grad");
  if (dq_row_stride < C || q_row_stride < C || (both && (dk_row_stride < C || k_row_stride < C)))
    return fail_arg("or_rmsnorm_rope_bwd: row strides must cover C elements");
  uintptr_t al = (uintptr_t)dq | (uintptr_t)q | (uintptr_t)wq | (uintptr_t)q_grad | (uintptr_t)wq_grad |
                 (uintptr_t)workspace;
  if (both) al |= (uintptr_t)dk | (uintptr_t)k | (uintptr_t)wk | (uintptr_t)k_grad | (uintptr_t)wk_grad;
  if ((al & 15u) || dq_row_stride % 8 || q_row_stride % 8 || (both && (dk_row_stride % 8 || k_row_stride % 8)))
    return fail_arg("or_rmsnorm_rope_bwd: pointers must be 16-byte aligned and row strides multiples of 8 elements");
  const int64_t need = or_rmsnorm_rope_bwd_workspace_size(n_rows, C);
  if (!workspace || workspace_bytes < need)
    return fail_arg("or_rmsnorm_rope_bwd: a workspace of %lld bytes is needed", (long long)need);
  NormRopeBwdArgs g = {};
  const void* in[2][3] = {{dq, q, wq}, {dk, k, wk}};
  void* out[2] = {q_grad, k_grad};
  float* dw[2] = {wq_grad, wk_grad};
  const int64_t strides[2][2] = {{dq_row_stride, q_row_stride}, {dk_row_stride, k_row_stride}};
  for (int i = 0; i < (both ? 2 : 1); ++i) {
    g.dy[i] = (const uint16_t*)in[i][0];
    g.x[i] = (const uint16_t*)in[i][1];
    g.w[i] = (const uint16_t*)in[i][2];
    g.dx[i] = (uint16_t*)out[i];
    g.dw[i] = dw[i];
    g.dy_stride[i] = strides[i][0];
    g.x_stride[i] = strides[i][1];
  }
  g.part = (float*)workspace;
  g.cos_t = cos_table;
  g.sin_t = sin_table;
  g.rope_row = rope_row;
  g.n_rows = n_rows;
  g.n_rope_rows = n_rope_rows;
  g.C = C;
  g.D = D;
  g.blocks = bwd_blocks(n_rows);
  g.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)g.blocks, both ? 2 : 1);
  if (g.blocks > 0) switch (C / 512) {
    case 1: hipLaunchKernelGGL(norm_rope_bwd_kernel<1>, grid, dim3(kThreads), 0, st, g); break;
    case 2: hipLaunchKernelGGL(norm_rope_bwd_kernel<2>, grid, dim3(kThreads), 0, st, g); break;
    case 3: hipLaunchKernelGGL(norm_rope_bwd_kernel<3>, grid, dim3(kThreads), 0, st, g); break;
    case 4: hipLaunchKernelGGL(norm_rope_bwd_kernel<4>, grid, dim3(kThreads), 0, st, g); break;
    case 5: hipLaunchKernelGGL(norm_rope_bwd_kernel<5>, grid, dim3(kThreads), 0, st, g); break;
    case 6: hipLaunchKernelGGL(norm_rope_bwd_kernel<6>, grid, dim3(kThreads), 0, st, g); break;
    case 8: hipLaunchKernelGGL(norm_rope_bwd_kernel<8>, grid, dim3(kThreads), 0, st, g); break;
    case 12: hipLaunchKernelGGL(norm_rope_bwd_kernel<12>, grid, dim3(kThreads), 0, st, g); break;
    case 16: hipLaunchKernelGGL(norm_rope_bwd_kernel<16>, grid, dim3(kThreads), 0, st, g); break;
    default: return fail_arg("or_rmsnorm_rope_bwd: C=%d not instantiated (512 x {1..6, 8, 12, 16})", C);
  }
  hipLaunchKernelGGL(norm_rope_dw_kernel, dim3((unsigned)(C / 64), both ? 2 : 1), dim3(64 * kSumWaves), 0, st, g);
  return check_hip(hipGetLastError(), "norm_rope_bwd launch");
}
