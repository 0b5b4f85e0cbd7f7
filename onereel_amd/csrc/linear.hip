// Linear layers of the DiT block for gfx950: y = residual + gate * act(x W^T + b) with everything after the product in its
// epilogue, and the gradient of it. bf16 operands, fp32 accumulation, one rounding.
//
//   z = x W^T + b      y = residual + gate * act(z)
//   dz = dy * gate * act'(z)    dx = dz W    dW = dz^T x    db = sum dz    dgate = sum dy * act(z)   (sums over rows)
//
// One product kernel for the three layouts: C[i][j] = sum_k A(i, k) B(j, k), where an operand's rows are contiguous either
// along k (x and W forward, dz in dx) or along their own index (W in dx, dz and x in dW).
// - A work-group owns a TI x TJ tile, each of its wavefronts (8 of 128 x 64 in a 256 x 256 tile, 4 in smaller ones) a part
//   of it in fp32 accumulators. Steps of 64 k of both operands go into a ring of LDS buffers by LDS DMA. An operand
//   contiguous along k is read as it lies (16 bytes a lane); the others are read by transposing LDS reads. XOR swizzles of
//   the 16-byte chunks keep both free of bank conflicts. The fragments of half a step are read while the other half is
//   multiplied, so that the matrix cores run through the one barrier of a step.
// - C's columns j are the rows of the MFMA tiles, so that a lane holds runs of 4 columns of one row; the epilogue brings
//   32 rows at a time through LDS into rows of 16-byte pieces, with the residual read and the results written in whole
//   lines.
// - Rows and columns past an operand's end load as zeros through the buffer descriptor (and an offset out of its range
//   for the pieces past the end of a row that is not the last), so ragged sizes take the same path.
// - Tiles of 256 x 256 are bound by the matrix cores; smaller tiles and a k axis split over several work-groups (fp32
//   partial products, added in order by the epilogue's own launch) fill the GPU when there are few tiles. Few rows of
//   x take kernels of their own that stream W once, bound by HBM.
// Measured (bf16, fp32 sums): 12720 x 2048 -> 8192 with bias, GELU and the pre-activation written 420 to 467 us, the product
// alone 377 (a library product of that size, without epilogue, 344); dx 371 us (library 356), dW 320 (library 364). The matrix
// pipes are busy 61 % of the cycles with that epilogue, 66 % in dx and 78 % in dW.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "tiles.h"

namespace onereel {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxStride = 1 << 21;

// ------------------------------------------------------------------------------------------------------------------
// products

// sums over rows from dz_kernel's partial ones: [2][chunks][n], db and dgate
struct SumArgs {
  const float* part;
  float* out[2];                     // each optional
  int chunks, n;
  int blocks;                        // work-groups ahead of a product's that take them; 0: none
};

struct GemmArgs {
  Operand a, b;
  int64_t I;                         // rows of C
  int J;                             // columns of C, a multiple of 8
  int64_t K;
  int split;                         // parts of the k axis
  int tiles_i, tiles_j;
  float* part;                       // [split][I][J] when split > 1
  Epilogue e;
  SumArgs sums;
};

// 64 columns of one sum for every 4 wavefronts, which deal out its partial rows; st: 64 floats a wavefront
template <int WAVES>
__device__ __forceinline__ void column_sums(const SumArgs& g, int block, float* st) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, unit = block * (WAVES / 4) + wave / 4;
  const int which = unit & 1, col = (unit >> 1) * 64 + lane;
  float* out = which ? g.out[1] : g.out[0];
  const bool in = out && col < g.n;
  float v = 0.0f;
  if (in) {
    const float* p = g.part + (int64_t)which * g.chunks * g.n + col;
#pragma unroll 16
    for (int b = wave % 4; b < g.chunks; b += 4) v += p[(int64_t)b * g.n];
  }
  st[wave * 64 + lane] = v;
  __syncthreads();
  if (wave % 4 == 0 && in) out[col] = (v + st[(wave + 1) * 64 + lane]) + (st[(wave + 2) * 64 + lane] + st[(wave + 3) * 64 + lane]);
}

template <int TI, int TJ, int WJ, int NB, bool TRA, bool TRB>
__global__ __launch_bounds__(128 * WJ) __attribute__((amdgpu_waves_per_eu(NB * (TI + TJ) * kStep * 2 > 81920 && WJ == 2 ? 1 : 2, 2))) void gemm_kernel(GemmArgs g) {
  constexpr int kThr = 128 * WJ;
  using TA = Tile<TI, TRA, kThr, 2>;
  using TB = Tile<TJ, TRB, kThr, WJ>;
  constexpr int FI = TA::F, FJ = TB::F, BUF = TA::BYTES + TB::BYTES;
  constexpr int kPad = TJ / WJ + 4;                        // floats per staged row of the epilogue
  constexpr int kStage = 2 * WJ * 32 * kPad * 4;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[NB * BUF > kStage ? NB * BUF : kStage];
  if ((int)blockIdx.x < g.sums.blocks) {   // a multiple of 8 of them, so that the others keep their XCDs
    column_sums<2 * WJ>(g.sums, blockIdx.x, (float*)lds);
    return;
  }
  int ti, tj, part;
  if (!tile_of(g, (int)blockIdx.x - g.sums.blocks, ti, tj, part)) return;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = w / WJ, wj = w % WJ;
  const int64_t i0 = (int64_t)ti * TI, j0 = (int64_t)tj * TJ;
  const int64_t steps = (g.K + kStep - 1) / kStep;
  const int k0 = (int)(steps * part / g.split * kStep), k1 = (int)min(steps * (part + 1) / g.split * kStep, g.K);

  TA la;
  TB lb;
  la.init(tid, g.a.stride);
  lb.init(tid, g.b.stride);
  Frag<TI, TRA, kThr, 2> fa;
  Frag<TJ, TRB, kThr, WJ> fb;
  fa.init(lane, wi);
  fb.init(lane, wj);
  const uint32_t base = lds_addr(lds), m0 = base + w * 1024;
  la.start(g.a, i0, g.I, k0, k1);
  lb.start(g.b, j0, g.J, k0, k1);
  f32x16 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  // Two sets of fragments, of 32 k each: one is read while the other is multiplied, across the barrier too, so that no
  // wavefront waits for LDS after it. One barrier per 64 k: every wavefront has read the buffer that the next load
  // overwrites, and every wavefront's part of the next one has arrived, asked for 64 (NB - 1) k ago. The order of reads, loads
  // and products is set here, FJ products at a time: left alone the compiler reads every fragment just before its use.
  constexpr int kLoads = TA::LOADS + TB::LOADS, kFrags = 2 * (FI + FJ), kGroups = 2 * FI;
  using FA = Frag<TI, TRA, kThr, 2>;
  using FB = Frag<TJ, TRB, kThr, WJ>;
  bf16x8 a[2][2][FI], b[2][2][FJ];
  uint32_t pa[FA::P], pb[FB::P];
  auto load = [&](int i, uint32_t buf) {
    if (i < TA::LOADS) la.one(i, m0 + buf);
    else lb.one(i - TA::LOADS, m0 + buf + TA::BYTES);
  };
  auto read = [&](int x, auto s_) {   // fragment x of set s (half s of a buffer)
    constexpr int s = decltype(s_)::value;
    if (x < 2 * FJ) b[s][x / FJ][x % FJ] = FB::template read<s>(pb, x / FJ, x % FJ);
    else a[s][(x - 2 * FJ) / FI][(x - 2 * FJ) % FI] = FA::template read<s>(pa, (x - 2 * FJ) / FI, (x - 2 * FJ) % FI);
  };
  auto half = [&](auto s_, uint32_t next, auto loads_, uint32_t buf) {   // multiplies set s, reads set 1 - s from `next`
    constexpr int s = decltype(s_)::value, kL = decltype(loads_)::value ? (kLoads + kGroups - 1) / kGroups : 0;
    constexpr int kR = (kFrags + kGroups - 1) / kGroups;
    fa.template aim<1 - s>(base + next, pa);
    fb.template aim<1 - s>(base + next + TA::BYTES, pb);
#pragma unroll
    for (int q = 0; q < kGroups; ++q) {
#pragma unroll
      for (int i = q * kL; i < (q + 1) * kL && i < kLoads; ++i) load(i, buf);
#pragma unroll
      for (int x = q * kR; x < (q + 1) * kR && x < kFrags; ++x) read(x, std::integral_constant<int, 1 - s>{});
#pragma unroll
      for (int j = 0; j < FJ; ++j)
        acc[q % FI][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[s][q / FI][j], a[s][q / FI][q % FI], acc[q % FI][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  uint32_t cur = 0;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    la.prepare();
    lb.prepare();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(i, n * BUF);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NB - 1) * kLoads) : "memory");
  fa.template aim<0>(base, pa);
  fb.template aim<0>(base + TA::BYTES, pb);
#pragma unroll
  for (int x = 0; x < kFrags; ++x) read(x, std::integral_constant<int, 0>{});
#pragma unroll 1
  for (int k = k0; k < k1; k += kStep) {
    half(std::integral_constant<int, 0>{}, cur, std::false_type{}, 0);
    la.prepare();
    lb.prepare();
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * kLoads) : "memory");
    const uint32_t next = cur + BUF == NB * BUF ? 0 : cur + BUF;
    half(std::integral_constant<int, 1>{}, next, std::true_type{}, cur);
    cur = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the loads past the end, before the buffers are used again
  __syncthreads();

  // epilogue: 32 rows at a time through this wavefront's part of LDS
  const int l32 = lane & 31, h = lane >> 5;
  float* st = (float*)lds + w * 32 * kPad;
  constexpr int LPR = TJ / WJ / 8;                          // lanes per row of 16-byte pieces
  const int64_t ib = i0 + wi * (TI / 2);
  const int64_t jc = j0 + wj * (TJ / WJ) + (lane % LPR) * 8;
#pragma unroll
  for (int i = 0; i < FI; ++i) {
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)(st + l32 * kPad + 32 * j + 8 * q + 4 * h) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int r = lane / LPR; r < 32; r += 64 / LPR) {
      const int64_t row = ib + 32 * i + r;
      const f32x4 x = *(const f32x4*)(st + r * kPad + (lane % LPR) * 8), y = *(const f32x4*)(st + r * kPad + (lane % LPR) * 8 + 4);
      if (row < g.I && jc < g.J) {
        if (g.split > 1) {
          float* p = g.part + ((int64_t)part * g.I + row) * g.J + jc;
          *(f32x4*)p = x;
          *(f32x4*)(p + 4) = y;
        } else {
          float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
          finish8(g.e, row, (int)jc, g.J, v);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// the parts of a split product, added in order, and the epilogue
__global__ __launch_bounds__(kThreads) void join_kernel(GemmArgs g) {
  const int64_t n8 = g.I * g.J / 8, step = (int64_t)gridDim.x * kThreads;
  for (int64_t x = (int64_t)blockIdx.x * kThreads + threadIdx.x; x < n8; x += step) {
    f32x4 lo = {}, hi = {};
    for (int p = 0; p < g.split; ++p) {
      const float* at = g.part + (int64_t)p * g.I * g.J + x * 8;
      lo += *(const f32x4*)at;
      hi += *(const f32x4*)(at + 4);
    }
    float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    finish8(g.e, x * 8 / g.J, (int)(x * 8 % g.J), g.J, v);
  }
}

// Loads of 16 bytes at a lane's byte offset, zeros where it has none: by way of a buffer descriptor, since with a branch around
// each load they wait for one another.
struct Rows {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Rows(const uint16_t* p, int64_t rows, int64_t stride, int width)
      : r(__builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)((rows - 1) * stride * 2) + width * 2, 0x00020000)) {}
  __device__ __forceinline__ u32x4 at(uint32_t off, bool in) const {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, in ? off : 0x80000000u, 0, 0));
  }
};

// N sums of a lane's own over all lanes, a half of them kept at each distance D, 32 to 1: at[0] of what a lane then holds
template <int N, int D, int ALL>
__device__ __forceinline__ void fold(float (&acc)[ALL], int lane, int& at) {
  if constexpr (N > 1) {
    const bool high = lane & D;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float mine = high ? acc[N / 2 + i] : acc[i], other = high ? acc[i] : acc[N / 2 + i];
      acc[i] = mine + __shfl_xor(other, D);
    }
    at += high ? N / 2 : 0;
  } else {
    acc[0] += __shfl_xor(acc[0], D);
  }
  if constexpr (D > 1) fold<(N > 1 ? N / 2 : 1), D / 2>(acc, lane, at);
}

// M rows of x, 1 to 4: a work-group takes 8 columns, its wavefronts deal out k in pieces of 512 and read each column's row of W
// in whole kilobytes; products on the vector units, sums over lanes by halves. Bound by HBM: one
// row to 12288 columns from 2048, W in no cache, 11.6 us (4.3 TB/s), on the matrix cores (below) 14.7; 2 rows of 7680 to 856 columns 6.2 and 11.3,
// 4 rows of 8192 to 2048 11.5 and 13.4; 8 rows of 2048 to 12288 16.8 and 16.4, so up to 4.
constexpr int kRowWaves = 4, kFewRows = 4;
template <int M>
__global__ __launch_bounds__(64 * kRowWaves) void rows_kernel(GemmArgs g) {
  constexpr int P = M == 3 ? 4 : M;   // the sums over lanes are dealt out by halves
  __shared__ float sum[kRowWaves][P * 8];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, j0 = blockIdx.x * 8, K = (int)g.K;
  const Rows wr(g.b.p + (int64_t)j0 * g.b.stride, 8, g.b.stride, K), xr(g.a.p, g.I, g.a.stride, K);
  const uint32_t ws = (uint32_t)g.b.stride * 2, xs = (uint32_t)g.a.stride * 2;
  float acc[P * 8] = {};
  for (int k0 = w * 512; k0 < K; k0 += kRowWaves * 512) {
    const uint32_t k = k0 + lane * 8;
    const bool in = k < (uint32_t)K;
    u32x4 wf[8], xf[M];
#pragma unroll
    for (int j = 0; j < 8; ++j) wf[j] = wr.at(j * ws + k * 2, in);
#pragma unroll
    for (int m = 0; m < M; ++m) xf[m] = xr.at(m * xs + k * 2, in);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w0 = bf2f((uint16_t)(wf[j][i] & 0xffffu)), w1 = bf2f((uint16_t)(wf[j][i] >> 16));
#pragma unroll
        for (int m = 0; m < M; ++m) {
          acc[m * 8 + j] = fmaf(bf2f((uint16_t)(xf[m][i] & 0xffffu)), w0, acc[m * 8 + j]);
          acc[m * 8 + j] = fmaf(bf2f((uint16_t)(xf[m][i] >> 16)), w1, acc[m * 8 + j]);
        }
      }
  }
  int at = 0;
  fold<P * 8, 32>(acc, lane, at);
  sum[w][at] = acc[0];
  __syncthreads();
  if (threadIdx.x < g.I) {
    float v[8] = {};
    for (int i = 0; i < kRowWaves; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += sum[i][threadIdx.x * 8 + e];
    finish8(g.e, threadIdx.x, j0, g.J, v);
  }
}

// 5 to 16 MB rows of x: a work-group takes 16 columns and reads their rows of W once, its wavefronts dealing out k in
// pieces of 128; no LDS but for the sum of the wavefronts. A load takes 64 contiguous bytes of each of W's 16 rows, the next
// one the other half of their lines (with 64 bytes a lane instead, 16 from each of 64 places a load, 33 us for 32 rows of 2048
// to 12288 columns, so 23). A CU takes 14 bytes a clock this way, whatever is in flight: it is for calls that have little to
// read a CU, and the tiles take the others (plan_of).
constexpr int kSkinnyWaves = 8;
template <int MB>
__global__ __launch_bounds__(64 * kSkinnyWaves) void skinny_kernel(GemmArgs g) {
  __shared__ float sum[kSkinnyWaves][16 * MB][17];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  const int j0 = blockIdx.x * 16;
  const int K = (int)g.K;
  f32x4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = f32x4{0, 0, 0, 0};
  const uint16_t* wp = g.b.p + (int64_t)min(j0 + l16, g.J - 1) * g.b.stride;
  for (int k0 = w * 128; k0 < K; k0 += kSkinnyWaves * 128) {
    u32x4 wf[4], xf[MB][4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = k0 + 32 * s + 8 * q;
      const bool in = k < K;
      wf[s] = in ? *(const u32x4*)(wp + k) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const int r = 16 * m + l16;
        xf[m][s] = in && r < g.I ? *(const u32x4*)(g.a.p + r * g.a.stride + k) : u32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int m = 0; m < MB; ++m)
        acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wf[s]),
                                                         __builtin_bit_cast(bf16x8, xf[m][s]), acc[m], 0, 0, 0);
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[w][16 * m + l16][4 * q + i] = acc[m][i];
  __syncthreads();
  for (int x = threadIdx.x; x < 32 * MB; x += 64 * kSkinnyWaves) {
    const int r = x >> 1, c = 8 * (x & 1);
    if (r >= g.I || j0 + c >= g.J) continue;
    float v[8] = {};
    for (int i = 0; i < kSkinnyWaves; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += sum[i][r][c + e];
    finish8(g.e, r, j0 + c, g.J, v);
  }
}

// ------------------------------------------------------------------------------------------------------------------
// dz = dy * gate * act'(z) and the sums over rows db = sum dz, dgate = sum dy * act(z): 256 columns x 8 to 128 rows a
// work-group, 8 columns a lane; the work-groups' partial sums are added up in order by work-groups ahead of the first product's
// (a launch of their own took 4 us, and 3 of the host: 333 x 1000 -> 2048 27.9 us in a graph, so 26.0). HBM-bound with
// many rows; with few of them by the latency of a work-group's rows, so they are dealt to 1024 work-groups or more.
// dz is rounded to bf16, since it is an operand of the bf16 matrix cores: dx and dW are 0.0023 of their norm off, 0.0017 with
// dz in fp32. The sums over rows take it before that rounding.
struct DzArgs {
  const uint16_t *dy, *z;
  int64_t dy_stride;
  const void* gate;
  int gate_bf16;
  uint16_t* dz;                      // optional
  float* part;                       // [2][chunks][N]: db, dgate
  float *db, *dgate;                 // optional
  int64_t M;
  int N, act, chunks, chunk_rows;
};

__global__ __launch_bounds__(kThreads) void dz_kernel(DzArgs g) {
  __shared__ float sum[2][8][256];
  const int c = threadIdx.x & 31, rr = threadIdx.x >> 5, col = blockIdx.x * 256 + c * 8;
  const int64_t r0 = (int64_t)blockIdx.y * g.chunk_rows, r1 = min(r0 + g.chunk_rows, g.M);
  float db[8] = {}, dg[8] = {}, gate[8];
  const bool in = col < g.N;
#pragma unroll
  for (int i = 0; i < 8; ++i) gate[i] = 1.0f;
  if (in && g.gate) load8(g.gate, g.gate_bf16, col, gate);
  if (in)
    for (int64_t r = r0 + rr; r < r1; r += 8) {
      const u32x4 y = *(const u32x4*)(g.dy + r * g.dy_stride + col);
      const u32x4 z = g.z ? *(const u32x4*)(g.z + r * g.N + col) : u32x4{0, 0, 0, 0};
      float dz[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = bf2f((uint16_t)(i & 1 ? y[i / 2] >> 16 : y[i / 2] & 0xffffu));
        const float zz = bf2f((uint16_t)(i & 1 ? z[i / 2] >> 16 : z[i / 2] & 0xffffu));
        float f, d;
        act_grad(zz, g.act, f, d);
        dg[i] += e * f;
        dz[i] = g.act == OR_ACT_NONE ? e * gate[i] : e * gate[i] * d;
        db[i] += dz[i];
      }
      if (g.dz)
        *(u32x4*)(g.dz + r * g.N + col) = u32x4{pack2(dz[0], dz[1]), pack2(dz[2], dz[3]), pack2(dz[4], dz[5]), pack2(dz[6], dz[7])};
    }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum[0][rr][c * 8 + i] = db[i];
    sum[1][rr][c * 8 + i] = dg[i];
  }
  __syncthreads();
  const int x = blockIdx.x * 256 + threadIdx.x;
  if (x >= g.N) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!(which ? g.dgate : g.db)) continue;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sum[which][i][threadIdx.x];
    g.part[((int64_t)which * g.chunks + blockIdx.y) * g.N + x] = v;
  }
}

__global__ __launch_bounds__(kThreads) void column_sum_kernel(SumArgs g) {
  __shared__ float st[kThreads];
  column_sums<kThreads / 64>(g, blockIdx.x, st);
}

// ------------------------------------------------------------------------------------------------------------------
// which kernel a product takes, and its workspace
struct Plan {
  int tile;                          // 256, 128 or 64; 0: the skinny kernel
  int tiles_i, tiles_j, split;
  int64_t part_bytes;
};

// The tile and the parts of k that a product takes least time with, by what a step of 64 k was measured to take a round of
// work-groups: 1.6 us with a 256 x 256 tile on every CU (8192^3: 815 to 930 us); 1.05 us with two of 128 x 128 (1024 x 8192 x
// 2048: 39 us), 0.6 us with one, whose four buffers then fit (512 x 8192 x 2048: 22.5 us, 27.9 with two); 0.43 and 0.32 us
// with two of 64 x 64 and one (128 x 8192 x 2048: 11 us). A work-group's start and epilogue count as 3 steps. Parts of k add
// the launch that joins them and its traffic (1536 x 8192 in 2 parts: 19 us).
constexpr int kCUs = 256;
constexpr int64_t kMaxBlocks = ((int64_t)1 << 23) - (1 << 17);   // of 512 threads: a grid, sums over rows included, has under 2^32
Plan plan_of(int64_t I, int64_t J, int64_t K, bool rows_of_k) {
  Plan p = {};
  p.split = 1;
  if (rows_of_k && I <= kFewRows) return p;
  const int64_t steps = (K + kStep - 1) / kStep;
  double best = 1e300;
  for (int tile : {256, 128, 64}) {
    const int64_t ti = (I + tile - 1) / tile, tj = (J + tile - 1) / tile;
    for (int split : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
      if (split > 1 && steps / split < 4) break;
      if (ti * tj * split > kMaxBlocks) break;
      const int64_t n = ti * tj * split, two = (n + 2 * kCUs - 1) / (2 * kCUs);
      const double step = tile == 256 ? 1.6 * ((n + kCUs - 1) / kCUs)
                          : tile == 128 ? (n <= kCUs ? 0.6 : 1.05 * two) : (n <= kCUs ? 0.32 : 0.43 * two);
      const double time = step * ((steps + split - 1) / split + 3) + (split > 1 ? 3 + (8.0 * split + 2) * I * J / 8e6 : 0);
      if (time < best) {
        best = time;
        p.tile = tile;
        p.tiles_i = (int)ti;
        p.tiles_j = (int)tj;
        p.split = split;
      }
    }
  }
  // up to 32 rows the kernel for them, by what 1024 k of 16 columns take a CU; the tiles' times above are those of full ones,
  // bound by the matrix cores (us, skinny / tiles: 16 rows of 2048 to 2048 columns 6.7 / 9.5, of 8192 18.5 / 16.1; 32 of 512 to
  // 512 4.2 / 5.5, of 2048 to 12288 22.6 / 14.5, of 7680 to 64 21.6 / 12.3)
  if (rows_of_k && I <= 32) {
    const int64_t groups = (J + 15) / 16, a_cu = (groups + kCUs - 1) / kCUs;
    if (1.2 + (double)((K + 1023) / 1024 * a_cu) * (I <= 16 ? 2.2 : a_cu > 1 ? 3.2 : 2.7) <
        1.2 * best + (p.split > 1 ? 4 : 1)) {
      p.tile = 0;
      p.split = 1;
    }
  }
  p.part_bytes = p.split > 1 ? (int64_t)p.split * I * J * 4 : 0;
  return p;
}

// LDS buffers of the ring: four where a CU has one work-group, with the room of two
int buffers_of(int tile, int64_t work_groups) { return tile == 64 || (tile == 128 && work_groups <= kCUs) ? 4 : 2; }

int sum_blocks(int n, int waves) { return (2 * ((n + 63) / 64) * 4 / waves + 7) / 8 * 8; }

template <bool TRA, bool TRB>
void launch_tiles(GemmArgs g, int tile, hipStream_t st) {
  const int64_t n = (int64_t)g.tiles_i * g.tiles_j * g.split;
  if (g.sums.part) g.sums.blocks = sum_blocks(g.sums.n, tile == 256 ? 8 : 4);
  const dim3 grid((unsigned)((n + 7) / 8 * 8 + g.sums.blocks));
  if (tile == 256) hipLaunchKernelGGL((gemm_kernel<256, 256, 4, 2, TRA, TRB>), grid, dim3(512), 0, st, g);
  else if (tile == 128 && buffers_of(tile, n) == 4) hipLaunchKernelGGL((gemm_kernel<128, 128, 2, 4, TRA, TRB>), grid, dim3(kThreads), 0, st, g);
  else if (tile == 128) hipLaunchKernelGGL((gemm_kernel<128, 128, 2, 2, TRA, TRB>), grid, dim3(kThreads), 0, st, g);
  else hipLaunchKernelGGL((gemm_kernel<64, 64, 2, 4, TRA, TRB>), grid, dim3(kThreads), 0, st, g);
}

void launch_product(GemmArgs g, bool tra, bool trb, float* part, hipStream_t st) {
  const Plan p = plan_of(g.I, g.J, g.K, !tra && !trb);
  if (p.tile == 0) {
    if (g.I <= kFewRows) {
      const dim3 grid((unsigned)(g.J / 8)), block(64 * kRowWaves);
      switch (g.I) {
        case 1: hipLaunchKernelGGL(rows_kernel<1>, grid, block, 0, st, g); break;
        case 2: hipLaunchKernelGGL(rows_kernel<2>, grid, block, 0, st, g); break;
        case 3: hipLaunchKernelGGL(rows_kernel<3>, grid, block, 0, st, g); break;
        default: hipLaunchKernelGGL(rows_kernel<4>, grid, block, 0, st, g);
      }
      return;
    }
    const dim3 grid((unsigned)((g.J + 15) / 16));
    if (g.I <= 16) hipLaunchKernelGGL(skinny_kernel<1>, grid, dim3(64 * kSkinnyWaves), 0, st, g);
    else hipLaunchKernelGGL(skinny_kernel<2>, grid, dim3(64 * kSkinnyWaves), 0, st, g);
    return;
  }
  g.tiles_i = p.tiles_i;
  g.tiles_j = p.tiles_j;
  g.split = p.split;
  g.part = part;
  if (!tra && !trb) launch_tiles<false, false>(g, p.tile, st);
  else if (!tra) launch_tiles<false, true>(g, p.tile, st);
  else launch_tiles<true, true>(g, p.tile, st);
  if (p.split > 1) {
    const int64_t blocks = std::min<int64_t>((g.I * g.J / 8 + kThreads - 1) / kThreads, 8192);
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, st, g);
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

int check_sizes(const char* what, int64_t M, int32_t N, int32_t K, int32_t act) {
  if (M < 0 || M > (int64_t)1 << 30) return fail_arg("%s: 0 to 2^30 rows (got %lld)", what, (long long)M);
  if (N < 8 || N % 8 || K < 8 || K % 8 || N > kMaxStride || K > kMaxStride)
    return fail_arg("%s: n_in and n_out must be multiples of 8 up to 2^21 (got %d and %d)", what, K, N);
  if (act != OR_ACT_NONE && act != OR_ACT_GELU_TANH && act != OR_ACT_SILU) return fail_arg("%s: unknown activation %d", what, act);
  for (int64_t width : {N, K})
    if ((M + 255) / 256 * ((width + 255) / 256) > kMaxBlocks) return fail_arg("%s: too many tiles", what);
  return 0;
}

int bad_stride(const char* what, int64_t stride, int64_t width) {
  if (stride < width || stride % 8 || stride > kMaxStride)
    return fail_arg("%s: row strides must be multiples of 8 elements that cover a row, up to 2^21", what);
  return 0;
}

// rows of a work-group of dz_kernel: a multiple of the 8 it takes at once, and at most 65535 groups of them
int chunk_rows_of(int64_t M, int32_t N) {
  const int64_t chunks = (1024 + (N + 255) / 256 - 1) / ((N + 255) / 256);
  const int64_t rows = ((M + chunks - 1) / chunks + 7) / 8 * 8;
  return (int)std::max<int64_t>({8, std::min<int64_t>(rows, 128), (M + 65534) / 65535 + 7 & ~(int64_t)7});
}

struct BwdLayout {
  int64_t dz, sums, part, bytes;
};
BwdLayout bwd_layout(int64_t M, int32_t N, int32_t K, bool makes_dz) {
  BwdLayout l;
  l.dz = 0;
  l.sums = makes_dz ? round256(M * N * 2) : 0;
  const int rows = chunk_rows_of(M, N);
  const int64_t chunks = (M + rows - 1) / rows;
  l.part = l.sums + round256(2 * chunks * N * 4);
  l.bytes = l.part + round256(std::max(plan_of(M, K, N, false).part_bytes, plan_of(N, K, M, false).part_bytes)) + 256;
  return l;
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int64_t or_linear_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out) {
  if (int rc = check_sizes("or_linear_workspace_size", n_rows, n_out, n_in, OR_ACT_NONE)) return rc;
  return plan_of(n_rows, n_out, n_in, true).part_bytes;
}

extern "C" int or_linear_plan(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t product, int32_t* tile, int32_t* buffers,
                              int32_t* split) {
  if (int rc = check_sizes("or_linear_plan", n_rows, n_out, n_in, OR_ACT_NONE)) return rc;
  if (product < 0 || product > 2 || !tile || !buffers || !split)
    return fail_arg("or_linear_plan: product must be 0, 1 or 2, and tile, buffers and split are required");
  const Plan p = product == 0 ? plan_of(n_rows, n_out, n_in, true)
                 : product == 1 ? plan_of(n_rows, n_in, n_out, false) : plan_of(n_out, n_in, n_rows, false);
  *tile = p.tile;
  *buffers = p.tile ? buffers_of(p.tile, (int64_t)p.tiles_i * p.tiles_j * p.split) : 0;
  *split = p.split;
  return 0;
}

extern "C" int or_linear(const or_linear_args* p, void* stream) {
  if (!p) return fail_arg("or_linear: args is NULL");
  const or_linear_args& x = *p;
  if (int rc = check_sizes("or_linear", x.n_rows, x.n_out, x.n_in, x.activation)) return rc;
  if (x.n_rows == 0) return 0;
  if (!x.x || !x.weight || !x.y) return fail_arg("or_linear: x, weight and y are required");
  if (int rc = bad_stride("or_linear: x", x.x_row_stride, x.n_in)) return rc;
  if (int rc = bad_stride("or_linear: weight", x.weight_row_stride, x.n_in)) return rc;
  if (int rc = bad_stride("or_linear: y", x.y_row_stride, x.n_out)) return rc;
  if (x.residual)
    if (int rc = bad_stride("or_linear: residual", x.residual_row_stride, x.n_out)) return rc;
  if (!al16(x.x) || !al16(x.weight) || !al16(x.bias) || !al16(x.gate) || !al16(x.residual) || !al16(x.y) ||
      !al16(x.preactivation))
    return fail_arg("or_linear: pointers must be 16-byte aligned");
  const int64_t need = or_linear_workspace_size(x.n_rows, x.n_in, x.n_out);
  if (need > 0 && (!x.workspace || !al16(x.workspace) || x.workspace_bytes < need))
    return fail_arg("or_linear: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  GemmArgs g = {};
  g.a = Operand{(const uint16_t*)x.x, x.x_row_stride};
  g.b = Operand{(const uint16_t*)x.weight, x.weight_row_stride};
  g.I = x.n_rows;
  g.J = x.n_out;
  g.K = x.n_in;
  g.e = Epilogue{(uint16_t*)x.y, x.y_row_stride, (uint16_t*)x.preactivation, x.bias, x.gate, x.bias_bf16, x.gate_bf16,
                 (const uint16_t*)x.residual, x.residual_row_stride, x.activation};
  launch_product(g, false, false, (float*)x.workspace, (hipStream_t)stream);
  return check_hip(hipGetLastError(), "or_linear launch");
}

extern "C" int64_t or_linear_bwd_workspace_size(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t scaled) {
  if (int rc = check_sizes("or_linear_bwd_workspace_size", n_rows, n_out, n_in, OR_ACT_NONE)) return rc;
  return bwd_layout(n_rows, n_out, n_in, scaled != 0).bytes;
}

extern "C" int or_linear_bwd(const or_linear_bwd_args* p, void* stream) {
  if (!p) return fail_arg("or_linear_bwd: args is NULL");
  const or_linear_bwd_args& x = *p;
  if (int rc = check_sizes("or_linear_bwd", x.n_rows, x.n_out, x.n_in, x.activation)) return rc;
  const bool scaled = x.activation != OR_ACT_NONE || x.gate;
  if (x.n_rows > 0 && !x.dy) return fail_arg("or_linear_bwd: dy is required");
  if (x.dx && !x.weight) return fail_arg("or_linear_bwd: dx needs the weight");
  if (x.dweight && x.n_rows > 0 && !x.x) return fail_arg("or_linear_bwd: dweight needs x");
  if (x.dgate && !x.gate) return fail_arg("or_linear_bwd: dgate needs the gate");
  if ((x.activation != OR_ACT_NONE || x.dgate) && x.n_rows > 0 && !x.preactivation)
    return fail_arg("or_linear_bwd: an activation's gradient and dgate need the pre-activation");
  if (int rc = bad_stride("or_linear_bwd: dy", x.dy_row_stride, x.n_out)) return rc;
  if (x.x)
    if (int rc = bad_stride("or_linear_bwd: x", x.x_row_stride, x.n_in)) return rc;
  if (x.weight)
    if (int rc = bad_stride("or_linear_bwd: weight", x.weight_row_stride, x.n_in)) return rc;
  if (!al16(x.dy) || !al16(x.x) || !al16(x.weight) || !al16(x.preactivation) || !al16(x.gate) || !al16(x.dx) ||
      !al16(x.dweight) || !al16(x.dbias) || !al16(x.dgate))
    return fail_arg("or_linear_bwd: pointers must be 16-byte aligned");
  const BwdLayout l = bwd_layout(x.n_rows, x.n_out, x.n_in, scaled);
  if (!x.workspace || !al16(x.workspace) || x.workspace_bytes < l.bytes)
    return fail_arg("or_linear_bwd: a 16-byte aligned workspace of %lld bytes is needed", (long long)l.bytes);
  hipStream_t st = (hipStream_t)stream;
  char* ws = (char*)x.workspace;
  const bool sums = x.dbias || x.dgate, products = x.dx || x.dweight;
  if (!sums && !products) return 0;
  Operand dz{(const uint16_t*)x.dy, x.dy_row_stride};
  SumArgs s = {};   // ride along with the first product's launch
  if (sums || (scaled && products)) {
    DzArgs d = {};
    d.dy = (const uint16_t*)x.dy;
    d.dy_stride = x.dy_row_stride;
    d.z = x.activation != OR_ACT_NONE || x.dgate ? (const uint16_t*)x.preactivation : nullptr;
    d.gate = x.gate;
    d.gate_bf16 = x.gate_bf16;
    d.dz = scaled && products ? (uint16_t*)(ws + l.dz) : nullptr;
    d.part = (float*)(ws + l.sums);
    d.db = x.dbias;
    d.dgate = x.dgate;
    d.M = x.n_rows;
    d.N = x.n_out;
    d.act = x.activation;
    d.chunk_rows = chunk_rows_of(x.n_rows, x.n_out);
    d.chunks = (int)((x.n_rows + d.chunk_rows - 1) / d.chunk_rows);
    if (d.chunks > 0)
      hipLaunchKernelGGL(dz_kernel, dim3((unsigned)((x.n_out + 255) / 256), (unsigned)d.chunks), dim3(kThreads), 0, st, d);
    if (sums) s = SumArgs{d.part, {x.dbias, x.dgate}, d.chunks, x.n_out, 0};
    if (d.dz) dz = Operand{d.dz, x.n_out};
  }
  if (x.dx && x.n_rows > 0) {
    GemmArgs g = {};
    g.a = dz;
    g.b = Operand{(const uint16_t*)x.weight, x.weight_row_stride};
    g.I = x.n_rows;
    g.J = x.n_in;
    g.K = x.n_out;
    g.sums = s;
    s = {};
    g.e.y = (uint16_t*)x.dx;
    g.e.y_stride = x.n_in;
    launch_product(g, false, true, (float*)(ws + l.part), st);
  }
  if (x.dweight) {
    GemmArgs g = {};
    g.a = dz;
    g.b = Operand{(const uint16_t*)x.x, x.x_row_stride};
    g.I = x.n_out;
    g.J = x.n_in;
    g.K = x.n_rows;
    g.sums = s;
    s = {};
    g.e.y = (uint16_t*)x.dweight;
    g.e.y_stride = x.n_in;
    launch_product(g, true, true, (float*)(ws + l.part), st);
  }
  if (s.part) hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)sum_blocks(s.n, kThreads / 64)), dim3(kThreads), 0, st, s);
  return check_hip(hipGetLastError(), "or_linear_bwd launch");
}
