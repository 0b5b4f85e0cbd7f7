// Rotary positions with several axes (time, row, column of a video's tokens) from the positions themselves, alone or behind the
// RMSNorm over all heads of the Wan self-attention's queries and keys, and the gradients of both.
//
// Reference: WanRotaryPosEmbed's split of a head's dims over frame, row and column, whose tables the processors get
// (rotary_emb, src/onereel/models/wan.py:91-99), and _qk (wan.py:64-74). Here no table exists: of a token at position pos[axis],
//
//   pair j of the head: axis a and index i within it (n_a dims, n_a / 2 pairs, in order of the axes)
//   angle = pos[a] theta_a^(-2 i / n_a)
//   (y0, y1) -> (y0 cos - y1 sin, y0 sin + y1 cos),  (y0, y1) = elements (2 j, 2 j + 1), or (j, j + R / 2) of the R = sum n_a
//   rotated dims; the dims past R stay as they are
//
// with y = x / sqrt(mean(x^2) + eps) w in the normed form. Its gradient, g = R^T dout, n = x inv, t = g w:
//   dw = sum over rows of g n,   dx = inv (t - n mean(t n))
//
// Angles are taken in turns, pos[a] * (theta_a^(-2 i / n_a) / (2 pi)) in fp64, of which the whole turns are dropped before the
// rest goes to fp32: a position of 1e6 in fp32 would be off by a tenth of a turn's hundredth, as the angle of a table made in
// fp32 is. All else is fp32 with one rounding of the result.
//
// HBM-bound: rows are read once and written once. The cosines and sines of a batch of tokens go through LDS, one of a token's
// pairs a thread, since the heads share them; in the normed form they are ready at the barrier that the rows' sums need anyway.
// 12720 tokens of 16 heads of 128 in bf16, q and k, among other work: normed 38.2 us for 208 MB (5.4 TB/s, the rate of a copy of 1 GB
// here 5.15 to 5.5), its gradient 65.5 us for 313 MB (61 in the first launch, 5.1 TB/s, and 5 in the sum of dw); one tensor rotated
// alone 19 us for 104 MB, either way (5.5 TB/s), of 63600 tokens 106 us (4.9). A call for few
// tokens is the launch: 5.2 us on the GPU for 333 tokens of 5 heads of 96 in fp32, 12.6 with the host.
#include <math.h>

#include <algorithm>

#include "rows.h"

namespace onereel {

namespace {

constexpr int kMaxAxes = 4;
constexpr int kMaxPairs = 256;         // of a head of 512 dims
constexpr int kMaxWaves = 16;
constexpr int kRows = 2;               // rows of a batch in the normed form
constexpr int kThreads = 256;

struct Axes {
  const void* position;                // [n_positions][n_axes], int32 or fp32
  int64_t n_positions;                 // row r of a tensor lies at position row r % n_positions
  int n_axes, whole, pairs;            // pairs: R / 2
  int first[kMaxAxes + 1];             // first pair of each axis
  double log2_theta[kMaxAxes];
};

// turns of pair j per unit of its position
__device__ __forceinline__ double frequency(const Axes& x, int j) {
  int a = 0;
#pragma unroll
  for (int i = 1; i < kMaxAxes; ++i) a = i < x.n_axes && j >= x.first[i] ? i : a;
  const int n = x.first[a + 1] - x.first[a];
  return exp2(-(double)(j - x.first[a]) / (double)n * x.log2_theta[a]) * 0.15915494309189533577;
}

// cosine and sine of pair j at a row's positions, `turn` being its frequency; 1 and 0 past the rotated pairs
__device__ __forceinline__ float2 angle_of(const Axes& x, int64_t row, int j, double turn) {
  if (j >= x.pairs) return make_float2(1.0f, 0.0f);
  int a = 0;
#pragma unroll
  for (int i = 1; i < kMaxAxes; ++i) a = i < x.n_axes && j >= x.first[i] ? i : a;
  const int64_t at = (row < x.n_positions ? row : row % x.n_positions) * x.n_axes + a;   // the division is for batches alone
  const double p = x.whole ? (double)((const int32_t*)x.position)[at] : (double)((const float*)x.position)[at];
  double turns = p * turn;
  turns -= rint(turns);
  float s, c;
  sincospif(2.0f * (float)turns, &s, &c);
  return make_float2(c, s);
}

// Where a unit of 4 pairs lies in a head of D dims: elements lo .. lo + 3 and hi .. hi + 3, first pair j. Interleaved units are
// 8 consecutive elements; of half-split heads the units past the rotated dims are such too, whose pairs are not rotated.
template <bool HALF>
__device__ __forceinline__ void unit_of(const Axes& x, int u, int& lo, int& hi, int& j) {
  j = 4 * u;
  if (HALF && j < x.pairs) {
    lo = j;
    hi = j + x.pairs;
  } else {
    lo = 8 * u;
    hi = lo + 4;
  }
}

// a unit's 8 values: v[0..3] and v[4..7] are its two pieces
template <typename T, bool HALF>
struct Unit {
  Piece<T, HALF ? 4 : 8> p[HALF ? 2 : 1];
  __device__ __forceinline__ void zero() {
    p[0].zero();
    if constexpr (HALF) p[1].zero();
  }
  __device__ __forceinline__ void load(const void* x, int64_t at, int lo, int hi) {
    p[0].load(x, at + lo);
    if constexpr (HALF) p[1].load(x, at + hi);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    if constexpr (HALF) {
      p[0].get(f);
      p[1].get(f + 4);
    } else {
      p[0].get(f);
    }
  }
  static __device__ __forceinline__ void store(void* x, int64_t at, int lo, int hi, const float (&f)[8]) {
    if constexpr (HALF) {
      Piece<T, 4>::store(x, at + lo, f);
      Piece<T, 4>::store(x, at + hi, f + 4);
    } else {
      Piece<T, 8>::store(x, at + lo, f);
    }
  }
};

// The first `left` pairs of a unit, rotated by their angles (sign 1) or back (-1). The others are left as they are: a product with a
// sine of 0 would make a NaN of an infinity beside them.
template <bool HALF>
__device__ __forceinline__ void turn8(float (&v)[8], const float2* angle, int left, float sign) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = angle[i].x, s = sign * angle[i].y;
    float& a = v[HALF ? i : 2 * i];
    float& b = v[HALF ? 4 + i : 2 * i + 1];
    const float x = a * c - b * s, y = a * s + b * c;
    const bool turned = i < left;
    a = turned ? x : a;
    b = turned ? y : b;
  }
}

struct RotateArgs {
  Axes axes;
  const void* x;
  void* out;                           // [rows][H][D]
  int64_t rows, row_stride, head_stride;
  int H, D, batch;                     // tokens of a batch
  float sign;
};

// The rotation alone: a work-group takes `batch` tokens at a time, whose angles it puts into LDS, and then their units.
template <typename T, bool HALF>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(RotateArgs g) {
  extern __shared__ __attribute__((aligned(16))) float2 angle[];      // [batch][D / 2]
  __shared__ double turn[kMaxPairs];
  const int half = g.D / 2, units = g.D / 8, of_token = units * g.H;
  for (int j = threadIdx.x; j < g.axes.pairs; j += kThreads) turn[j] = frequency(g.axes, j);
  const int64_t batches = (g.rows + g.batch - 1) / g.batch;
  for (int64_t b = blockIdx.x; b < batches; b += gridDim.x) {
    const int64_t r0 = b * g.batch;
    const int n = (int)min((int64_t)g.batch, g.rows - r0);
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kThreads) {
      const int t = i / half, j = i - t * half;
      angle[i] = angle_of(g.axes, r0 + t, j, j < g.axes.pairs ? turn[j] : 0.0);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * of_token; i += kThreads) {
      const int t = i / of_token, k = i - t * of_token, h = k / units;
      int lo, hi, j;
      unit_of<HALF>(g.axes, k - h * units, lo, hi, j);
      Unit<T, HALF> x;
      float v[8];
      x.load(g.x, (r0 + t) * g.row_stride + h * g.head_stride, lo, hi);
      x.get(v);
      turn8<HALF>(v, angle + t * half + j, g.axes.pairs - j, g.sign);
      Unit<T, HALF>::store(g.out, ((r0 + t) * g.H + h) * g.D, lo, hi, v);
    }
  }
}

struct NormedArgs {
  Axes axes;
  const void* x[2];
  const void* dy[2];                   // gradient only
  void* out[2];                        // contiguous: the rotated rows, or dx
  const void* w[2];
  float* dw[2];
  float* part;                         // [2][blocks][C]
  int64_t rows, x_stride[2], dy_stride[2];
  int C, D, blocks;
  float eps;
};

// the wavefronts' shares, one to each of 16 lanes
__device__ __forceinline__ float sum_shares(const float* s, int waves) {
  const int w = threadIdx.x & 15;
  return row_sum(w < waves ? s[w] : 0.0f);
}

// blockIdx.y picks q or k. A thread has one unit of every row; the work-group takes kRows rows at a time, so that their loads are under
// way together.
template <typename T, bool HALF>
__global__ __launch_bounds__(1024) void norm_rope_axes_kernel(NormedArgs g) {
  __shared__ float2 angle[2][kRows][kMaxPairs];
  __shared__ double turn[kMaxPairs];
  __shared__ float share[2][kRows][kMaxWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, which = blockIdx.y;
  const int half = g.D / 2, units = g.D / 8, h = threadIdx.x / units;
  const bool in = 8 * (int)threadIdx.x < g.C;
  const float a_column = 1.0f / (float)g.C;
  int lo, hi, j;
  unit_of<HALF>(g.axes, threadIdx.x - h * units, lo, hi, j);
  lo += h * g.D;
  hi += h * g.D;
  float w[8] = {};
  if (in) {
    Unit<T, HALF> p;
    p.load(g.w[which], 0, lo, hi);
    p.get(w);
  }
  for (int p = threadIdx.x; p < g.axes.pairs; p += blockDim.x) turn[p] = frequency(g.axes, p);
  __syncthreads();
  int now = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < g.rows; r0 += (int64_t)gridDim.x * kRows, now ^= 1) {
    Unit<T, HALF> x[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      x[k].zero();
      if (in && r0 + k < g.rows) x[k].load(g.x[which], (r0 + k) * g.x_stride[which], lo, hi);
    }
    for (int i = threadIdx.x; i < kRows * half; i += blockDim.x) {
      const int k = i / half, p = i - k * half;
      angle[now][k][p] = angle_of(g.axes, min(r0 + k, g.rows - 1), p, p < g.axes.pairs ? turn[p] : 0.0);
    }
    float v[kRows][8];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      x[k].get(v[k]);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += v[k][i] * v[k][i];
      ss = wave_sum(ss);
      if (lane == 0) share[now][k][wave] = ss;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const float inv = rsqrtf(sum_shares(share[now][k], waves) * a_column + g.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] *= inv * w[i];
      if (in && r0 + k < g.rows) {
        turn8<HALF>(v[k], angle[now][k] + j, g.axes.pairs - j, 1.0f);
        Unit<T, HALF>::store(g.out[which], (r0 + k) * g.C, lo, hi, v[k]);
      }
    }
  }
}

// (One row at a time, its loads and angles under way ahead of the last one's sums and one barrier a row: 70.5 us, two rows and two barriers 69.2 then, for q and k of
// 12720 rows of 2048.)
template <typename T, bool HALF>
__global__ __launch_bounds__(1024) void norm_rope_axes_bwd_kernel(NormedArgs g) {
  __shared__ float2 angle[2][kRows][kMaxPairs];
  __shared__ double turn[kMaxPairs];
  __shared__ float share[2][kRows][kMaxWaves], share_x[2][kRows][kMaxWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, which = blockIdx.y;
  const int half = g.D / 2, units = g.D / 8, h = threadIdx.x / units;
  const bool in = 8 * (int)threadIdx.x < g.C;
  const float a_column = 1.0f / (float)g.C;
  int lo, hi, j;
  unit_of<HALF>(g.axes, threadIdx.x - h * units, lo, hi, j);
  lo += h * g.D;
  hi += h * g.D;
  float w[8] = {}, dw[8] = {};
  if (in) {
    Unit<T, HALF> p;
    p.load(g.w[which], 0, lo, hi);
    p.get(w);
  }
  for (int p = threadIdx.x; p < g.axes.pairs; p += blockDim.x) turn[p] = frequency(g.axes, p);
  __syncthreads();
  int now = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < g.rows; r0 += (int64_t)gridDim.x * kRows, now ^= 1) {
    Unit<T, HALF> x[kRows], d[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      x[k].zero();
      d[k].zero();
      if (in && r0 + k < g.rows) {
        x[k].load(g.x[which], (r0 + k) * g.x_stride[which], lo, hi);
        d[k].load(g.dy[which], (r0 + k) * g.dy_stride[which], lo, hi);
      }
    }
    for (int i = threadIdx.x; i < kRows * half; i += blockDim.x) {
      const int k = i / half, p = i - k * half;
      angle[now][k][p] = angle_of(g.axes, min(r0 + k, g.rows - 1), p, p < g.axes.pairs ? turn[p] : 0.0);
    }
    // the angles first: the sum of t n needs the gradient turned back
    __syncthreads();
    float v[kRows][8], e[kRows][8];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      x[k].get(v[k]);
      d[k].get(e[k]);
      turn8<HALF>(e[k], angle[now][k] + (in ? j : 0), g.axes.pairs - j, -1.0f);
      float ss = 0.0f, tx = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        ss += v[k][i] * v[k][i];
        tx += e[k][i] * w[i] * v[k][i];
      }
      ss = wave_sum(ss);
      tx = wave_sum(tx);
      if (lane == 0) {
        share[now][k][wave] = ss;
        share_x[now][k][wave] = tx;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const float inv = rsqrtf(sum_shares(share[now][k], waves) * a_column + g.eps);
      const float m = sum_shares(share_x[now][k], waves) * a_column * inv * inv;    // mean(t n) inv
      const bool row = in && r0 + k < g.rows;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[i] += row ? e[k][i] * (v[k][i] * inv) : 0.0f;
        e[k][i] = inv * (e[k][i] * w[i] - v[k][i] * m);
      }
      if (row) Unit<T, HALF>::store(g.out[which], (r0 + k) * g.C, lo, hi, e[k]);
    }
  }
  if (!in) return;
  float* out = g.part + ((int64_t)which * g.blocks + blockIdx.x) * g.C;
  *(f32x4*)(out + lo) = f32x4{dw[0], dw[1], dw[2], dw[3]};
  *(f32x4*)(out + hi) = f32x4{dw[4], dw[5], dw[6], dw[7]};
}

// dw: 64 columns a block, the work-groups' rows of sums dealt out to 16 wavefronts
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void norm_rope_axes_dw_kernel(NormedArgs g) {
  __shared__ float sum[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, which = blockIdx.y, col = blockIdx.x * 64 + lane;
  float v = 0.0f;
  if (col < g.C) {
    const float* p = g.part + (int64_t)which * g.blocks * g.C + col;
#pragma unroll 8
    for (int b = wave; b < g.blocks; b += kSumWaves) v += p[(int64_t)b * g.C];
  }
  sum[wave][lane] = v;
  __syncthreads();
  if (wave != 0 || col >= g.C) return;
  v = 0.0f;
  for (int i = 0; i < kSumWaves; ++i) v += sum[i][lane];
  g.dw[which][col] = v;
}

constexpr int kBwdBlocks = 512;        // of q, and of k

int bwd_blocks(int64_t rows) {
  // each of its threads adds up the rows it takes one after the other, 256 of them at most
  return (int)std::min<int64_t>((rows + kRows - 1) / kRows, std::max<int64_t>(kBwdBlocks, (rows + 255) / 256));
}

int read_axes(const char* what, const or_rope_axes* p, int D, Axes& x) {
  if (!p) return fail_arg("%s: axes is NULL", what);
  if (p->n_axes < 1 || p->n_axes > kMaxAxes) return fail_arg("%s: 1 to %d axes (got %d)", what, kMaxAxes, p->n_axes);
  if (D < 8 || D % 8 || D > 2 * kMaxPairs) return fail_arg("%s: heads of a multiple of 8 dims up to %d (got %d)", what, 2 * kMaxPairs, D);
  if (p->pairs != OR_PAIRS_INTERLEAVED && p->pairs != OR_PAIRS_HALF) return fail_arg("%s: unknown pairs %d", what, p->pairs);
  int64_t sum = 0;
  for (int a = 0; a < p->n_axes; ++a) {
    if (p->dims[a] < 2 || p->dims[a] % 2 || p->dims[a] > D) return fail_arg("%s: an axis takes an even count of dims up to the head's (got %d)", what, p->dims[a]);
    if (!(p->theta[a] > 0) || !isfinite(p->theta[a])) return fail_arg("%s: theta must be finite and positive", what);
    x.first[a] = (int)(sum / 2);
    x.log2_theta[a] = log2(p->theta[a]);
    sum += p->dims[a];
  }
  if (sum > D) return fail_arg("%s: the axes take %lld of %d dims", what, (long long)sum, D);
  if (p->pairs == OR_PAIRS_HALF && sum % 8) return fail_arg("%s: half-split pairs need a multiple of 8 rotated dims (got %lld)", what, (long long)sum);
  for (int a = p->n_axes; a <= kMaxAxes; ++a) x.first[a] = (int)(sum / 2);
  x.position = p->positions;
  x.n_positions = p->n_positions;
  x.n_axes = p->n_axes;
  x.whole = p->positions_fp32 ? 0 : 1;
  x.pairs = (int)(sum / 2);
  return 0;
}

int check_positions(const char* what, const or_rope_axes* p, int64_t rows) {
  if (!p->positions || ((uintptr_t)p->positions & 3)) return fail_arg("%s: 4-byte aligned positions are required", what);
  if (p->n_positions < 1 || rows % p->n_positions) return fail_arg("%s: the %lld positions must divide the %lld rows", what, (long long)p->n_positions, (long long)rows);
  return 0;
}

int check_rows(const char* what, int64_t rows) {
  if (rows < 0 || rows > (int64_t)1 << 30) return fail_arg("%s: 0 to 2^30 rows (got %lld)", what, (long long)rows);
  return 0;
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

template <typename T>
void launch(const RotateArgs& g, bool half, unsigned blocks, size_t lds, hipStream_t st) {
  if (half) hipLaunchKernelGGL((rope_axes_kernel<T, true>), dim3(blocks), dim3(kThreads), lds, st, g);
  else hipLaunchKernelGGL((rope_axes_kernel<T, false>), dim3(blocks), dim3(kThreads), lds, st, g);
}

template <typename T>
void launch_normed(const NormedArgs& g, bool half, bool bwd, dim3 grid, dim3 block, hipStream_t st) {
  if (bwd) {
    if (half) hipLaunchKernelGGL((norm_rope_axes_bwd_kernel<T, true>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((norm_rope_axes_bwd_kernel<T, false>), grid, block, 0, st, g);
  } else {
    if (half) hipLaunchKernelGGL((norm_rope_axes_kernel<T, true>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((norm_rope_axes_kernel<T, false>), grid, block, 0, st, g);
  }
}

int check_normed(const char* what, int64_t rows, int32_t C, int32_t D, int32_t type) {
  if (!known_type(type)) return fail_arg("%s: unknown element type %d", what, type);
  if (int rc = check_rows(what, rows)) return rc;
  if (D < 8 || D % 8 || C < D || C % D || C > 8192) return fail_arg("%s: rows of whole heads up to 8192 elements (C=%d D=%d)", what, C, D);
  return 0;
}

int bad_stride(const char* what, const void* p, int64_t stride, int C) {
  if (!p) return fail_arg("%s is required", what);
  if (!al16(p) || stride < C || stride % 8) return fail_arg("%s: 16-byte aligned rows, a multiple of 8 elements apart, that cover C", what);
  return 0;
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int or_rope_axes_rotate(const or_rope_axes* axes, const void* x, void* out, int64_t n_rows, int32_t H, int32_t D,
                                   int64_t row_stride, int64_t head_stride, int32_t type, int32_t inverse, void* stream) {
  const char* what = "or_rope_axes_rotate";
  RotateArgs g = {};
  if (int rc = read_axes(what, axes, D, g.axes)) return rc;
  if (!known_type(type)) return fail_arg("%s: unknown element type %d", what, type);
  if (int rc = check_rows(what, n_rows)) return rc;
  if (H < 1 || H > 4096) return fail_arg("%s: 1 to 4096 heads (got %d)", what, H);
  if (n_rows == 0) return 0;
  if (int rc = check_positions(what, axes, n_rows)) return rc;
  if (!x || !out || !al16(x) || !al16(out) || row_stride % 8 || head_stride % 8 || row_stride < 0 || head_stride < 0)
    return fail_arg("%s: 16-byte aligned x and out, strides of multiples of 8 elements", what);
  g.x = x;
  g.out = out;
  g.rows = n_rows;
  g.row_stride = row_stride;
  g.head_stride = head_stride;
  g.H = H;
  g.D = D;
  g.sign = inverse ? -1.0f : 1.0f;
  // a batch of about 1024 units, its angles in up to 32 KB
  g.batch = (int)std::max<int64_t>(1, std::min<int64_t>({1024 / ((int64_t)H * D / 8), 8192 / D, n_rows}));
  const int64_t batches = (n_rows + g.batch - 1) / g.batch;
  const unsigned blocks = (unsigned)std::min<int64_t>(batches, 256 * 8);
  const size_t lds = (size_t)g.batch * (D / 2) * sizeof(float2);
  const bool half = axes->pairs == OR_PAIRS_HALF;
  hipStream_t st = (hipStream_t)stream;
  if (type == OR_TYPE_BF16) launch<Bf16>(g, half, blocks, lds, st);
  else if (type == OR_TYPE_FP16) launch<_Float16>(g, half, blocks, lds, st);
  else launch<float>(g, half, blocks, lds, st);
  return check_hip(hipGetLastError(), "rope_axes_kernel launch");
}

extern "C" int or_rmsnorm_rope_axes(const or_rope_axes* axes, const void* q, const void* k, const void* wq, const void* wk,
                                    int64_t q_row_stride, int64_t k_row_stride, int64_t n_rows, int32_t C, int32_t D,
                                    int32_t type, float eps, void* q_out, void* k_out, void* stream) {
  const char* what = "or_rmsnorm_rope_axes";
  NormedArgs g = {};
  if (int rc = check_normed(what, n_rows, C, D, type)) return rc;
  if (int rc = read_axes(what, axes, D, g.axes)) return rc;
  if (n_rows == 0) return 0;
  if (int rc = check_positions(what, axes, n_rows)) return rc;
  const void* in[2][3] = {{q, wq, q_out}, {k, wk, k_out}};
  const int64_t strides[2] = {q_row_stride, k_row_stride};
  const int n = k ? 2 : 1;
  for (int i = 0; i < n; ++i) {
    if (int rc = bad_stride(i ? "or_rmsnorm_rope_axes: k" : "or_rmsnorm_rope_axes: q", in[i][0], strides[i], C)) return rc;
    if (!in[i][1] || !in[i][2] || !al16(in[i][1]) || !al16(in[i][2]))
      return fail_arg("%s: 16-byte aligned weights and outputs are required", what);
    g.x[i] = in[i][0];
    g.w[i] = in[i][1];
    g.out[i] = const_cast<void*>(in[i][2]);
    g.x_stride[i] = strides[i];
  }
  g.rows = n_rows;
  g.C = C;
  g.D = D;
  g.eps = eps;
  const dim3 grid((unsigned)std::min<int64_t>((n_rows + kRows - 1) / kRows, 256 * 8), n), block((unsigned)((C / 8 + 63) / 64 * 64));
  const bool half = axes->pairs == OR_PAIRS_HALF;
  hipStream_t st = (hipStream_t)stream;
  if (type == OR_TYPE_BF16) launch_normed<Bf16>(g, half, false, grid, block, st);
  else if (type == OR_TYPE_FP16) launch_normed<_Float16>(g, half, false, grid, block, st);
  else launch_normed<float>(g, half, false, grid, block, st);
  return check_hip(hipGetLastError(), "norm_rope_axes_kernel launch");
}

extern "C" int64_t or_rmsnorm_rope_axes_bwd_workspace_size(int64_t n_rows, int32_t C) {
  const char* what = "or_rmsnorm_rope_axes_bwd_workspace_size";
  if (int rc = check_rows(what, n_rows)) return rc;
  if (C < 8 || C % 8 || C > 8192) return fail_arg("%s: rows of a multiple of 8 elements up to 8192 (C=%d)", what, C);
  return 2 * (int64_t)bwd_blocks(n_rows) * C * 4;
}

extern "C" int or_rmsnorm_rope_axes_bwd(const or_rope_axes* axes, const void* dq, const void* dk, const void* q, const void* k,
                                        const void* wq, const void* wk, int64_t dq_row_stride, int64_t dk_row_stride,
                                        int64_t q_row_stride, int64_t k_row_stride, int64_t n_rows, int32_t C, int32_t D,
                                        int32_t type, float eps, void* q_grad, void* k_grad, float* wq_grad, float* wk_grad,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "or_rmsnorm_rope_axes_bwd";
  NormedArgs g = {};
  if (int rc = check_normed(what, n_rows, C, D, type)) return rc;
  if (int rc = read_axes(what, axes, D, g.axes)) return rc;
  const int n = wk ? 2 : 1;
  const void* in[2][3] = {{dq, q, wq}, {dk, k, wk}};
  void* out[2] = {q_grad, k_grad};
  float* dw[2] = {wq_grad, wk_grad};
  const int64_t strides[2][2] = {{dq_row_stride, q_row_stride}, {dk_row_stride, k_row_stride}};
  for (int i = 0; i < n; ++i) {
    if (!in[i][2] || !dw[i] || !al16(in[i][2]) || ((uintptr_t)dw[i] & 3)) return fail_arg("%s: 16-byte aligned weights and their gradients are required", what);
    if (n_rows > 0) {
      for (int t = 0; t < 2; ++t)
        if (int rc = bad_stride(t ? "or_rmsnorm_rope_axes_bwd: q, k" : "or_rmsnorm_rope_axes_bwd: dq, dk", in[i][t], strides[i][t], C)) return rc;
      if (!out[i] || !al16(out[i])) return fail_arg("%s: 16-byte aligned q_grad and k_grad are required", what);
    }
    g.dy[i] = in[i][0];
    g.x[i] = in[i][1];
    g.w[i] = in[i][2];
    g.out[i] = out[i];
    g.dw[i] = dw[i];
    g.dy_stride[i] = strides[i][0];
    g.x_stride[i] = strides[i][1];
  }
  if (n_rows > 0)
    if (int rc = check_positions(what, axes, n_rows)) return rc;
  const int64_t need = or_rmsnorm_rope_axes_bwd_workspace_size(n_rows, C);
  if (need > 0 && (!workspace || !al16(workspace) || workspace_bytes < need))
    return fail_arg("%s: a 16-byte aligned workspace of %lld bytes is needed", what, (long long)need);
  g.part = (float*)workspace;
  g.rows = n_rows;
  g.C = C;
  g.D = D;
  g.blocks = bwd_blocks(n_rows);
  g.eps = eps;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)g.blocks, n), block((unsigned)((C / 8 + 63) / 64 * 64));
  const bool half = axes->pairs == OR_PAIRS_HALF;
  if (g.blocks > 0) {
    if (type == OR_TYPE_BF16) launch_normed<Bf16>(g, half, true, grid, block, st);
    else if (type == OR_TYPE_FP16) launch_normed<_Float16>(g, half, true, grid, block, st);
    else launch_normed<float>(g, half, true, grid, block, st);
  }
  hipLaunchKernelGGL(norm_rope_axes_dw_kernel, dim3((unsigned)((C + 63) / 64), n), dim3(64 * kSumWaves), 0, st, g);
  return check_hip(hipGetLastError(), "norm_rope_axes_bwd launch");
}
