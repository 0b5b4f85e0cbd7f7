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
//
// Quantising and reading back are HBM-bound: 8192 x 2048 in bf16 9.4 and 8.8 us for 42 MB (4.5 and 4.8 TB/s). The product of few rows
// reads W once (1 x 2048 -> 12288 7.6 us for 13 MB, a launch and its latency; 12 with the host), that of many is bound by the matrix
// cores and by what feeds them from LDS: 8192^3 in 260 to 270 us (4.1 PFLOP/s; matrix pipes busy 55% of the time at 1.82 GHz; of an
// earlier 288 without loads from HBM 236, without reads of LDS 255, with neither 204, the bare matrix instructions 193), 12720 x 2048 ->
// 8192 with bias and GELU in 171, where the 7 rounds of tiles (6.25 of them full) each pay an epilogue and a start for 8 steps, and 16 to
// 19 for the launch ahead of it, which quantises x (the call 183; with x in 4 bits 174).
#include <algorithm>
#include <type_traits>

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

// the e8m0 scale of a block from the fp32 bits of its largest magnitude
__device__ __forceinline__ uint32_t scale_of(uint32_t top) {
  const uint32_t e = top >> 23;
  return e == 255 ? 255 : e > 2 ? e - 2 : 0;
}

// what a scale stands for
__device__ __forceinline__ float unit_of(uint32_t scale) {
  return __uint_as_float(scale == 255 ? 0x7fc00000u : scale == 0 ? 0x00400000u : scale << 23);
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// Largest magnitude of 8 elements, as bits that compare like it (those of a NaN are the largest): 16-bit types two a register, of
// which the larger is taken at the end; the lanes of a block are joined before that.
template <typename T>
struct Top {
  static __device__ __forceinline__ uint32_t of(const Piece<T, 8>& p) {
    const u32x4 r = __builtin_bit_cast(u32x4, p.r);
    const uint32_t m = 0x7fff7fffu;
    return max16(max16(r[0] & m, r[1] & m), max16(r[2] & m, r[3] & m));
  }
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max16(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t v) {
    const uint32_t x = max(v & 0xffffu, v >> 16);
    return sizeof(T) == 2 && __is_same(T, Bf16) ? x << 16 : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)x));
  }
};
template <>
struct Top<float> {
  static __device__ __forceinline__ uint32_t of(const Piece<float, 8>& p) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) v = max(v, __float_as_uint(p.r[i / 4][i % 4]) & 0x7fffffffu);
    return v;
  }
  static __device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b) { return max(a, b); }
  static __device__ __forceinline__ uint32_t bits(uint32_t v) { return v; }
};

// The codes of 8 elements. The conversion divides by the scale's power of two and rounds to nearest, ties to even, past 6 to 6.
__device__ __forceinline__ uint32_t codes_of(const Piece<Bf16, 8>& p, float unit) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const uint32_t w[4] = {p.r[0], p.r[1], p.r[2], p.r[3]};
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[0]), unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[1]), unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[2]), unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2, w[3]), unit, 3);
}
__device__ __forceinline__ uint32_t codes_of(const Piece<_Float16, 8>& p, float unit) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, half2{p.r[0], p.r[1]}, unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, half2{p.r[2], p.r[3]}, unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, half2{p.r[4], p.r[5]}, unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(c, half2{p.r[6], p.r[7]}, unit, 3);
}
__device__ __forceinline__ uint32_t codes_of(const Piece<float, 8>& p, float unit) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, p.r[0][0], p.r[0][1], unit, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, p.r[0][2], p.r[0][3], unit, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, p.r[1][0], p.r[1][1], unit, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, p.r[1][2], p.r[1][3], unit, 3);
}

// 8 elements of a block that 4 neighbouring lanes share
template <typename T>
__device__ __forceinline__ void quantize8(const Piece<T, 8>& p, uint32_t& codes, uint32_t& scale) {
  uint32_t top = Top<T>::of(p);
  top = Top<T>::join(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xf, 0xf, false));   // quad_perm 1032
  top = Top<T>::join(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xf, 0xf, false));   // quad_perm 2301
  scale = scale_of(Top<T>::bits(top));
  codes = scale == 255 ? 0 : codes_of(p, unit_of(scale));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(QuantizeArgs g) {
  const int per = g.K / 8;
  const int64_t total = g.rows * per;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per;
    const int c = (int)(i - row * per);
    Piece<T, 8> p;
    uint32_t codes, scale;
    p.load(g.x, row * g.x_stride + 8 * c);
    quantize8(p, codes, scale);
    ((uint32_t*)g.codes)[i] = codes;
    if ((c & 3) == 0) g.scales[i >> 2] = (uint8_t)scale;
  }
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

// x / d for x < 2^31 as x m / 2^shift: m = ceil(2^(31 + s) / d) with 2^s >= d is off by less than 2^s / d of what could show
// (the compiler's division by a number known at run time alone is some 40 instructions, one after the other, and a work-group's
// place among the tiles takes five: 12720 x 2048 -> 8192 166.7 us with them, 165.4 so)
struct Divisor {
  uint32_t m, shift;
};

constexpr uint32_t kGroup = 8;         // rows of tiles that share their operands' rows in the L2

struct MxArgs {
  const void* x;                       // bf16, for the kernels of few rows; else NULL
  int64_t x_stride;
  const uint8_t *a, *a_scales, *b, *b_scales;   // x and W; for the tiles the scales as mx_prepare_kernel lays them out
  int64_t I;
  int J, K;
  int split, tiles_i, tiles_j;
  Divisor by_split, by_group, by_rest;   // of kGroup rows of tiles, and of the rest of the rows
  int64_t a_rows, b_rows;              // rows of the scales' layout
  float* part;                         // [split][I][J] when split > 1
  Epilogue e;
};

// Up to 16 MB rows of x: a work-group takes 16 columns and reads their rows of W once, its wavefronts dealing out k in pieces of
// 256; nothing goes through LDS but the sum of the wavefronts. A lane's part of a step of 128 elements is one block of W (16 bytes of one of
// 16 rows) and one of x, which it quantises by itself where x comes in bf16: every work-group does that anew, which costs less than
// a launch.
constexpr int kRowWaves = 8;
template <int MB, bool BF16>
__global__ __launch_bounds__(64 * kRowWaves) void mx_rows_kernel(MxArgs g) {
  __shared__ float sum[kRowWaves][16 * MB][17];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15, q = lane >> 4;
  const int j0 = blockIdx.x * 16, blocks = g.K / kBlock;
  const int64_t wr = min(j0 + l16, g.J - 1);
  const uint8_t *wp = g.b + wr * (g.K / 2), *ws = g.b_scales + wr * blocks;
  f32x4 acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = f32x4{0, 0, 0, 0};
  for (int s0 = 8 * w; s0 < blocks; s0 += 8 * kRowWaves) {
    u32x4 wf[2], xf[MB][2];
    uint32_t wsc[2], xsc[MB][2];
    Piece<Bf16, 8> p[MB][2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int b = s0 + 4 * t + q;
      const bool in = b < blocks;
      wf[t] = in ? *(const u32x4*)(wp + b * 16) : u32x4{0, 0, 0, 0};
      wsc[t] = in ? ws[b] : 0;
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const int64_t r = 16 * m + l16;
        const bool here = in && r < g.I;
        if constexpr (BF16) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            p[m][t][c].zero();
            if (here) p[m][t][c].load(g.x, r * g.x_stride + b * 32 + 8 * c);
          }
        } else {
          xf[m][t] = here ? *(const u32x4*)(g.a + r * (g.K / 2) + b * 16) : u32x4{0, 0, 0, 0};
          xsc[m][t] = here ? g.a_scales[r * blocks + b] : 0;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const i32x8 wv = {(int)wf[t][0], (int)wf[t][1], (int)wf[t][2], (int)wf[t][3]};
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        if constexpr (BF16) {
          using X = Top<Bf16>;
          const uint32_t top = X::join(X::join(X::of(p[m][t][0]), X::of(p[m][t][1])), X::join(X::of(p[m][t][2]), X::of(p[m][t][3])));
          xsc[m][t] = scale_of(X::bits(top));
          const float unit = unit_of(xsc[m][t]);
#pragma unroll
          for (int c = 0; c < 4; ++c) xf[m][t][c] = xsc[m][t] == 255 ? 0 : codes_of(p[m][t][c], unit);
        }
        const i32x8 xv = {(int)xf[m][t][0], (int)xf[m][t][1], (int)xf[m][t][2], (int)xf[m][t][3]};
        acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[m], 4, 4, 0, (int)wsc[t], 0, (int)xsc[m][t]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[w][16 * m + l16][4 * q + i] = acc[m][i];
  __syncthreads();
  for (int x = threadIdx.x; x < 32 * MB; x += 64 * kRowWaves) {
    const int r = x >> 1, c = 8 * (x & 1);
    if (r >= g.I || j0 + c >= g.J) continue;
    float v[8] = {};
    for (int i = 0; i < kRowWaves; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += sum[i][r][c + e];
    finish8(g.e, r, j0 + c, g.J, v);
  }
}

// The tiles' scales. A step of kSB bytes of a row has 8 blocks, 4 of them for the lanes of each half h of a wavefront (lanes 32 h ..),
// which multiply blocks h, 2 + h, .. of their rows, 32 apart. So the scales of 128 rows lie as [step][row % 32][h][row / 32 % 4][4]:
// a step's lie together, and a lane reads those of 4 (or 2, or 1) of its rows at once. Blocks past the end of a row get the scale 0:
// what their place holds in LDS are zeros, but not every scale keeps a zero a zero.
constexpr int kScaleRows = 128;
constexpr int kSB = 128, kStepElements = 2 * kSB, kStepBlocks = kSB / 16;
constexpr int KS = kSB / 32;           // of them, those of one half of the lanes: products of 64 elements in a step

// One operand's tile of N rows x kSB bytes in LDS, chunk c (16 bytes, a block) of row r at position c ^ swz(r). A load of the
// work-group takes ROWS rows; a lane's place among them is the same in each.
template <int N, int THREADS>
struct MxTile {
  static constexpr int BYTES = N * kSB, ROWS = THREADS / kStepBlocks, LOADS = N / ROWS;
  static constexpr int SCALES = (N > kScaleRows ? N : kScaleRows) * kStepBlocks;   // whole groups of rows
  static constexpr int SCALE_LOADS = (SCALES + 4 * THREADS - 1) / (4 * THREADS);
  static __device__ __forceinline__ int swz(int r) { return (r >> 1) & 7; }
  static_assert(LOADS >= 1 && N % ROWS == 0 && ROWS % 16 == 0, "tile");   // 16 rows: the swizzle's period
  const uint8_t *p, *s;
  int rows, left, wide;                // rows that end the tile; bytes of k left, and of this step
  uint32_t row_bytes;
  int64_t scale_pitch;
  __device__ __forceinline__ void start(const uint8_t* codes, const uint8_t* scales, int64_t scale_rows, uint32_t stride, int64_t n0,
                                        int64_t n, int step0, int end) {
    row_bytes = stride;
    p = codes + n0 * stride + (int64_t)step0 * kSB;
    s = scales + ((int64_t)step0 * scale_rows + n0 / kScaleRows * kScaleRows) * kStepBlocks;
    scale_pitch = scale_rows * kStepBlocks;
    rows = (int)min(n - n0, (int64_t)N);
    left = end - step0 * kSB;
    wide = 0;
  }
  // the step to load from now on
  __device__ __forceinline__ void step() { wide = min(max(left, 0), kSB); }
  __device__ __forceinline__ void next() {
    p += kSB;
    s += scale_pitch;
    left -= kSB;
  }
  __device__ __forceinline__ i32x4 codes(int i) const {
    const int n = rows - i * ROWS;
    return descriptor((const uint16_t*)(p + (int64_t)i * ROWS * row_bytes), n > 0 && wide > 0 ? (int32_t)((uint32_t)(n - 1) * row_bytes) + wide : 0);
  }
  __device__ __forceinline__ i32x4 scales() const { return descriptor((const uint16_t*)s, wide > 0 ? SCALES : 0); }
};

// 4 bytes a lane
__device__ __forceinline__ void dma4(const i32x4& r, uint32_t off, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(r),
               "s"(__builtin_amdgcn_readfirstlane(m0))
               : "memory");
}

template <int TI, int TJ, int WI, int WJ, int NB>
struct MxShape {
  static constexpr int THREADS = 64 * WI * WJ;
  using TA = MxTile<TI, THREADS>;
  using TB = MxTile<TJ, THREADS>;
  static constexpr int FI = TI / WI / 32, FJ = TJ / WJ / 32;
  static constexpr int SCALE_A = 4 * THREADS * TA::SCALE_LOADS, SCALE_B = 4 * THREADS * TB::SCALE_LOADS;   // bytes that their loads write
  static constexpr int BUF = TA::BYTES + TB::BYTES + SCALE_A + SCALE_B;
  static constexpr int PAD = TJ / WJ + 4;                 // floats per staged row of the epilogue
  static constexpr int STAGE = WI * WJ * 32 * PAD * 4, LDS = NB * BUF > STAGE ? NB * BUF : STAGE;
  static_assert(kScaleRows % (32 * FI) == 0 && kScaleRows % (32 * FJ) == 0, "a wavefront's rows share a group of scales");
};

// Tile and steps of the k axis that a place in the order of the tiles stands for. The work-groups of one XCD (index modulo 8) take
// consecutive places, and groups of 8 rows of tiles share their operands' rows in its L2. There are under 2^31 places.
struct Place {
  int ti, tj, part, first, last;
};
__device__ __forceinline__ uint32_t quotient(uint32_t x, const Divisor& d) { return (uint32_t)(((uint64_t)x * d.m) >> d.shift); }
__device__ __forceinline__ bool place_of(const MxArgs& g, uint32_t block, int steps, Place& p) {
  const uint32_t n = (uint32_t)g.tiles_i * g.tiles_j * g.split, per = (n + 7) / 8, j = block >> 3;
  uint32_t x = (block & 7) * per + j;
  if (j >= per || x >= n) return false;
  p.part = 0;
  p.first = 0;
  p.last = steps;
  if (g.split > 1) {
    const uint32_t q = quotient(x, g.by_split);
    p.part = (int)(x - q * g.split);
    p.first = (int)quotient((uint32_t)steps * p.part, g.by_split);
    p.last = (int)quotient((uint32_t)steps * (p.part + 1), g.by_split);
    x = q;
  }
  const uint32_t group = quotient(x, g.by_group), in = x - group * kGroup * g.tiles_j, left = g.tiles_i - group * kGroup;
  const uint32_t row = left >= kGroup ? in / kGroup : quotient(in, g.by_rest), high = min(kGroup, left);
  p.ti = (int)(group * kGroup + in - row * high);
  p.tj = (int)row;
  return true;
}

// The epilogue of 8 columns for several rows: the columns' parameters are read once.
struct Finish {
  float bias[8], gate[8];
  __device__ __forceinline__ void start(const Epilogue& e, int col) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bias[i] = 0.0f;
      gate[i] = 1.0f;
    }
    if (e.bias) load8(e.bias, e.bias_bf16, col, bias);
    if (e.gate) load8(e.gate, e.gate_bf16, col, gate);
  }
  __device__ __forceinline__ void finish(const Epilogue& e, int64_t row, int col, float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    if (e.act == OR_ACT_GELU_TANH) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = gelu(v[i]);
    } else if (e.act == OR_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = silu(v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= gate[i];
    if (e.residual) {
      const u32x4 r = *(const u32x4*)(e.residual + row * e.residual_stride + col);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] += bf2f((uint16_t)(r[i] & 0xffffu));
        v[2 * i + 1] += bf2f((uint16_t)(r[i] >> 16));
      }
    }
    *(u32x4*)(e.y + row * e.y_stride + col) = u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
  }
};

// The structure of the bf16 product (linear.hip): a ring of NB buffers filled by LDS DMA, one barrier a step, two sets of
// fragments, one read while the other is multiplied. A lane's 16 bytes of a row are one block, its scale a byte of a register.
template <int TI, int TJ, int WI, int WJ, int NB>
__global__ __launch_bounds__(64 * WI * WJ) __attribute__((amdgpu_waves_per_eu(1, 2))) void mx_tile_kernel(MxArgs g) {
  using S = MxShape<TI, TJ, WI, WJ, NB>;
  using TA = typename S::TA;
  using TB = typename S::TB;
  constexpr int FI = S::FI, FJ = S::FJ, HK = KS / 2;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[S::LDS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = w / WJ, wj = w % WJ, l32 = lane & 31, h = lane >> 5;
  const int row_bytes = g.K / 2, steps = (row_bytes + kSB - 1) / kSB;

  Place work;
  if (!place_of(g, blockIdx.x, steps, work)) return;
  TA la;
  TB lb;
  const int end = min(work.last * kSB, row_bytes);
  la.start(g.a, g.a_scales, g.a_rows, row_bytes, (int64_t)work.ti * TI, g.I, work.first, end);
  lb.start(g.b, g.b_scales, g.b_rows, row_bytes, (int64_t)work.tj * TJ, g.J, work.first, end);
  auto next_step = [&] {
    la.step();
    lb.step();
  };

  const uint32_t base = lds_addr(lds), m0 = base + w * 1024, m0s = base + TA::BYTES + TB::BYTES + w * 256;
  const int chunk = (tid % kStepBlocks) ^ TA::swz(tid / kStepBlocks);
  const uint32_t off = (uint32_t)(tid / kStepBlocks) * (uint32_t)row_bytes + chunk * 16;
  // addresses of the fragments of a buffer: one a step of 64 elements, the blocks of 32 rows are immediates from it
  const int swz = TA::swz(l32);
  uint32_t at[KS];
#pragma unroll
  for (int k = 0; k < KS; ++k) at[k] = l32 * kSB + ((2 * k + h) ^ swz) * 16;
  const uint32_t at_a = base + wi * (TI / WI) * kSB, at_b = base + TA::BYTES + wj * (TJ / WJ) * kSB;
  // a wavefront's rows from `row` on in their group of 128
  auto scale_at = [&](int row) { return (row / kScaleRows) * kScaleRows * kStepBlocks + (l32 * 2 + h) * 4 * KS + row % kScaleRows / 32 * KS; };
  const uint32_t at_sa = base + TA::BYTES + TB::BYTES + scale_at(wi * (TI / WI) + (work.ti * (TI % kScaleRows)) % kScaleRows);
  const uint32_t at_sb = base + TA::BYTES + TB::BYTES + S::SCALE_A + scale_at(wj * (TJ / WJ) + (work.tj * (TJ % kScaleRows)) % kScaleRows);

  f32x16 acc[FI][FJ];
  auto clear = [&] {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  };
  clear();

  constexpr int kCodes = TA::LOADS + TB::LOADS, kLoads = kCodes + TA::SCALE_LOADS + TB::SCALE_LOADS;
  constexpr int kFrags = HK * (FI + FJ), kGroups = HK * FI;
  u32x4 a[2][HK][FI], b[2][HK][FJ];
  auto load = [&](int i, uint32_t buf) {
    constexpr int T = S::THREADS;
    const uint32_t o = chunk * 16 < la.wide ? off : 0x80000000u;
    if (i < TA::LOADS) {
      dma16(la.codes(i), o, m0 + buf + i * T * 16);
    } else if (i < kCodes) {
      dma16(lb.codes(i - TA::LOADS), o, m0 + buf + TA::BYTES + (i - TA::LOADS) * T * 16);
    } else if (i < kCodes + TA::SCALE_LOADS) {
      const int x = i - kCodes;
      dma4(la.scales(), 4 * (tid + x * T), m0s + buf + x * 4 * T);
    } else {
      const int x = i - kCodes - TA::SCALE_LOADS;
      dma4(lb.scales(), 4 * (tid + x * T), m0s + buf + S::SCALE_A + x * 4 * T);
    }
  };
  typedef const __attribute__((address_space(3))) u32x4 lds_u32x4;
  uint32_t pa[HK], pb[HK];
  auto aim = [&](auto s_, uint32_t buf) {
    constexpr int s = decltype(s_)::value;
#pragma unroll
    for (int k = 0; k < HK; ++k) {
      pa[k] = at_a + buf + at[s * HK + k];
      pb[k] = at_b + buf + at[s * HK + k];
      asm volatile("" : "+v"(pa[k]), "+v"(pb[k]));
    }
  };
  auto read = [&](int x, auto s_) {    // fragment x of set s
    constexpr int s = decltype(s_)::value;
    if (x < HK * FJ) b[s][x / FJ][x % FJ] = *(lds_u32x4*)(uintptr_t)(pb[x / FJ] + x % FJ * 32 * kSB);
    else a[s][(x - HK * FJ) / FI][(x - HK * FJ) % FI] = *(lds_u32x4*)(uintptr_t)(pa[(x - HK * FJ) / FI] + (x - HK * FJ) % FI * 32 * kSB);
  };
  // KS bytes of each block of 32 rows, packed
  constexpr int WA = FI * KS / 4, WB = FJ * KS / 4;
  uint32_t sa[WA], sb[WB], na[WA], nb[WB];
  auto words = [](uint32_t at, auto n_, uint32_t* v) {
    constexpr int n = decltype(n_)::value;
    typedef uint32_t vec __attribute__((ext_vector_type(n)));
    typedef const __attribute__((address_space(3))) vec lds_vec;
    const vec x = *(lds_vec*)(uintptr_t)at;
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = x[i];
  };
  auto read_scales = [&](uint32_t buf) {
    words(at_sa + buf, std::integral_constant<int, WA>{}, na);
    words(at_sb + buf, std::integral_constant<int, WB>{}, nb);
  };
  auto take_scales = [&] {
#pragma unroll
    for (int i = 0; i < WA; ++i) sa[i] = na[i];
#pragma unroll
    for (int i = 0; i < WB; ++i) sb[i] = nb[i];
  };
  auto multiply = [&](auto s_, auto k_, auto i_, auto j_) {
    constexpr int s = decltype(s_)::value, k = decltype(k_)::value, i = decltype(i_)::value, j = decltype(j_)::value;
    constexpr int ba = i * KS + s * HK + k, bb = j * KS + s * HK + k;
    const u32x4 x = a[s][k][i], y = b[s][k][j];
    const i32x8 xa = {(int)x[0], (int)x[1], (int)x[2], (int)x[3]}, yb = {(int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(yb, xa, acc[i][j], 4, 4, bb % 4, (int)sb[bb / 4], ba % 4, (int)sa[ba / 4]);
  };
  auto half = [&](auto s_, uint32_t next, auto loads_, uint32_t buf) {
    constexpr int s = decltype(s_)::value, kL = decltype(loads_)::value ? (kLoads + kGroups - 1) / kGroups : 0;
    constexpr int kR = (kFrags + kGroups - 1) / kGroups;
    aim(std::integral_constant<int, 1 - s>{}, next);
    if (s == 1) read_scales(next);
    auto group = [&](auto q_) {
      constexpr int q = decltype(q_)::value;
#pragma unroll
      for (int i = q * kL; i < (q + 1) * kL && i < kLoads; ++i) load(i, buf);
#pragma unroll
      for (int x = q * kR; x < (q + 1) * kR && x < kFrags; ++x) read(x, std::integral_constant<int, 1 - s>{});
      multiply(s_, std::integral_constant<int, q / FI>{}, std::integral_constant<int, q % FI>{}, std::integral_constant<int, 0>{});
      if constexpr (FJ > 1) multiply(s_, std::integral_constant<int, q / FI>{}, std::integral_constant<int, q % FI>{}, std::integral_constant<int, 1>{});
      static_assert(FJ <= 2, "columns of a wavefront");
      __builtin_amdgcn_sched_barrier(0);
    };
    group(std::integral_constant<int, 0>{});
    group(std::integral_constant<int, 1>{});
    if constexpr (kGroups > 2) group(std::integral_constant<int, 2>{});
    if constexpr (kGroups > 2) group(std::integral_constant<int, 3>{});
    if constexpr (kGroups > 4) {
      group(std::integral_constant<int, 4>{});
      group(std::integral_constant<int, 5>{});
      group(std::integral_constant<int, 6>{});
      group(std::integral_constant<int, 7>{});
    }
    static_assert(kGroups == 2 || kGroups == 4 || kGroups == 8, "groups of products");
    if (s == 1) take_scales();
  };
  uint32_t cur = 0;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    next_step();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load(i, n * S::BUF);
    la.next();
    lb.next();
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NB - 1) * kLoads) : "memory");
  aim(std::integral_constant<int, 0>{}, 0);
#pragma unroll
  for (int x = 0; x < kFrags; ++x) read(x, std::integral_constant<int, 0>{});
  read_scales(0);
  take_scales();
#pragma unroll 1
  for (int k = work.first; k < work.last; ++k) {
    half(std::integral_constant<int, 0>{}, cur, std::false_type{}, 0);
    next_step();
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * kLoads) : "memory");
    const uint32_t next = cur + S::BUF == NB * S::BUF ? 0 : cur + S::BUF;
    half(std::integral_constant<int, 1>{}, next, std::true_type{}, cur);
    la.next();
    lb.next();
    cur = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the loads past the end, before the buffers are used again
  __syncthreads();

  // Epilogue: 32 rows at a time through this wavefront's part of LDS, into whole lines. (8 columns of a row from two lanes' registers
  // instead, without LDS, write 32 bytes of each of 32 rows at a time: 8192^3 300 to 336 us.) A lane keeps its columns.
  float* st = (float*)lds + w * 32 * S::PAD;
  constexpr int LPR = TJ / WJ / 8;                          // lanes per row of 16-byte pieces
  const int64_t ib = (int64_t)work.ti * TI + wi * (TI / WI);
  const int64_t jc = (int64_t)work.tj * TJ + wj * (TJ / WJ) + (lane % LPR) * 8;
  const bool in = jc < g.J;
  Finish f;
  if (g.split == 1) f.start(g.e, in ? (int)jc : 0);
#pragma unroll
  for (int i = 0; i < FI; ++i) {
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)(st + l32 * S::PAD + 32 * j + 8 * q + 4 * h) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = lane / LPR; r < 32; r += 64 / LPR) {
      const int64_t row = ib + 32 * i + r;
      const f32x4 x = *(const f32x4*)(st + r * S::PAD + (lane % LPR) * 8), y = *(const f32x4*)(st + r * S::PAD + (lane % LPR) * 8 + 4);
      if (in && row < g.I) {
        if (g.split > 1) {
          float* p = g.part + ((int64_t)work.part * g.I + row) * g.J + jc;
          *(f32x4*)p = x;
          *(f32x4*)(p + 4) = y;
        } else {
          float v[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
          f.finish(g.e, row, (int)jc, v);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// the parts of a split product, added in order, and the epilogue
__global__ __launch_bounds__(kThreads) void mx_join_kernel(MxArgs g) {
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

// What the tiles read, in one launch: x in 4 bits with its scales in their layout (or those of an x that comes in 4 bits), and W's
// scales in theirs
struct PrepareArgs {
  QuantizeArgs q;                      // x NULL: scales only, from q.scales
  uint8_t* a_scales;
  const uint8_t* w_scales;
  uint8_t* b_scales;
  int64_t a_rows, b_rows;
  int n_out, a_blocks, steps;          // a_blocks: work-groups that take x; steps of 256 elements
};

// One unit is 32 rows (8 neighbouring ones of each 32 of 128) x 256 elements: rows r0 + l + 32 f, whose scales lie together in each
// step. They are collected in LDS in that order.
constexpr int kUnitBytes = 8 * 2 * 4 * KS;
__device__ __forceinline__ int unit_place(int l, int f, int block) { return ((l * 2 + (block & 1)) * 4 + f) * KS + (block >> 1); }

__global__ __launch_bounds__(kThreads) void mx_prepare_kernel(PrepareArgs g) {
  __shared__ __attribute__((aligned(16))) uint8_t st[kUnitBytes];
  const bool weights = (int)blockIdx.x >= g.a_blocks;
  const int64_t rows = weights ? g.n_out : g.q.rows, all = weights ? g.b_rows : g.a_rows;
  const int blocks = g.q.K / kBlock, tid = threadIdx.x, work_groups = weights ? (int)gridDim.x - g.a_blocks : g.a_blocks;
  for (int64_t unit = weights ? (int)blockIdx.x - g.a_blocks : (int)blockIdx.x; unit < all / 32 * g.steps; unit += work_groups) {
    const int step = (int)(unit % g.steps);
    // group of 128 rows, and the first of 8 rows in each 32 of it
    const int64_t u = unit / g.steps, r0 = u / 4 * kScaleRows + u % 4 * 8;
    if (weights || !g.q.x) {
      const uint8_t* from = weights ? g.w_scales : g.q.scales;
      const int f = tid >> 6, l = tid >> 3 & 7, k = tid & 7, block = 8 * step + k;
      const int64_t row = r0 + l + 32 * f;
      st[unit_place(l, f, k)] = row < rows && block < blocks ? from[row * blocks + block] : 0;
    } else {
      const int l = tid >> 5, c = tid & 31, at = 256 * step + 8 * c;
      const bool in = at < g.q.K;        // all four lanes of a block, or none
      Piece<Bf16, 8> p[4];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        p[f].zero();
        const int64_t row = r0 + l + 32 * f;
        if (in && row < rows) p[f].load(g.q.x, row * g.q.x_stride + at);
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int64_t row = r0 + l + 32 * f;
        uint32_t codes, scale;
        quantize8(p[f], codes, scale);
        if (in && row < rows) ((uint32_t*)g.q.codes)[row * (g.q.K / 8) + at / 8] = codes;
        if ((c & 3) == 0) st[unit_place(l, f, c >> 2)] = in && row < rows ? (uint8_t)scale : 0;
      }
    }
    __syncthreads();
    uint8_t* to = (weights ? g.b_scales : g.a_scales) + (step * all + r0 / kScaleRows * kScaleRows) * kStepBlocks + r0 % kScaleRows * 8 * KS;
    if (tid < kUnitBytes / 4) ((uint32_t*)to)[tid] = ((const uint32_t*)st)[tid];
    __syncthreads();
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
constexpr int64_t kMaxStride = 1 << 21;
constexpr int kFewRows = 32;
constexpr int kCUs = 256;
constexpr int64_t kMaxBlocks = (int64_t)1 << 22;   // of 512 threads: a grid has under 2^32

int check_rows(const char* what, int64_t rows, int32_t K) {
  if (rows < 0 || rows > (int64_t)1 << 30) return fail_arg("%s: 0 to 2^30 rows (got %lld)", what, (long long)rows);
  if (K < kBlock || K % kBlock || K > kMaxStride) return fail_arg("%s: rows of a multiple of 32 elements up to 2^21 (got %d)", what, K);
  return 0;
}

int check_product(const char* what, int64_t M, int32_t K, int32_t N) {
  if (int rc = check_rows(what, M, K)) return rc;
  if (N < 8 || N % 8 || N > kMaxStride) return fail_arg("%s: n_out must be a multiple of 8 up to 2^21 (got %d)", what, N);
  if ((M + 255) / 256 * ((N + (int64_t)255) / 256) > kMaxBlocks) return fail_arg("%s: too many tiles", what);
  return 0;
}

Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while (1u << s < d) ++s;
  return Divisor{(uint32_t)((((uint64_t)1 << (31 + s)) + d - 1) / d), 31 + s};
}

unsigned blocks_for(int64_t total) { return (unsigned)std::min<int64_t>((total + kThreads - 1) / kThreads, 256 * 32); }

void launch_quantize(const QuantizeArgs& g, int type, hipStream_t st) {
  const dim3 grid(blocks_for(g.rows * (g.K / 8)));
  if (type == OR_TYPE_BF16) hipLaunchKernelGGL(mx_quantize_kernel<Bf16>, grid, dim3(kThreads), 0, st, g);
  else if (type == OR_TYPE_FP16) hipLaunchKernelGGL(mx_quantize_kernel<_Float16>, grid, dim3(kThreads), 0, st, g);
  else hipLaunchKernelGGL(mx_quantize_kernel<float>, grid, dim3(kThreads), 0, st, g);
}

int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// ------------------------------------------------------------------------------------------------------------------
// which kernel a product takes, and its workspace
struct Plan {
  int tile;                            // 0: the kernel for few rows
  int tiles_i, tiles_j, split;
};

constexpr int kTileRows = 256;         // the scales' layouts come in whole tiles of any size

// The tile and the parts of k that a product takes least time with, by what a step of 256 k was measured to take a round of
// work-groups, and their start and epilogue in such steps (us): 2.1 (steps + 3.6) with a 256 x 256 tile on every CU (8192^3 300, 12720 x
// 256 -> 8192 73); 1.2 (steps + 3.8) with two of 128 x 128 a CU and 0.65 (steps + 7) with one, whose four buffers then fit (4096 x
// 2048 -> 2048 22, 1024 x 8192 -> 2048 30); 0.5 (steps + 5.9) and 0.42 (steps + 2.6) with two of 64 x 64 and one (1024 x 8192 -> 2048 26, 333
// x 8192 -> 2048 19). Parts of k add the launch that joins them and its traffic (64 x 8192 -> 512 in 4 parts 12.0, in one 16.3).
double time_of(int tile, int64_t n, double steps) {
  const int64_t one = (n + kCUs - 1) / kCUs, two = (n + 2 * kCUs - 1) / (2 * kCUs);
  if (tile == 256) return 2.1 * (steps + 3.6) * one;
  if (tile == 128) return n <= kCUs ? 0.65 * (steps + 7) : 1.2 * (steps + 3.8) * two;
  return n <= kCUs ? 0.42 * (steps + 2.6) : 0.5 * (steps + 5.9) * two;
}

Plan plan_of(int64_t I, int64_t J, int64_t K) {
  Plan p = {};
  double best = 1e300;
  const int64_t steps = (K + kStepElements - 1) / kStepElements;
  for (int tile : {256, 128, 64}) {
    const int64_t ti = (I + tile - 1) / tile, tj = (J + tile - 1) / tile;
    for (int split : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (split > 1 && steps / split < 4) break;
      const int64_t n = ti * tj * split;
      if (n > kMaxBlocks) break;
      const double time = time_of(tile, n, (double)((steps + split - 1) / split)) + (split > 1 ? 3 + (8.0 * split + 2) * I * J / 4e6 : 0);
      if (time < best) {
        best = time;
        p = Plan{tile, (int)ti, (int)tj, split};
      }
    }
  }
  // Up to 32 rows the kernel for them, by what 2048 k of 16 columns take a CU for that many rows; the tiles' launches and the one
  // ahead of them take 2 us more than its own (us, it and the tiles: one row of 2048 to 12288 columns 7.5 and 10.4, of 8192 to 2048 8.6
  // and 12.1; 16 rows of 2048 to 12288 11.4 and 10.4, of 512 to 512 4.0 and 7.1; 32 of 512 to 512 4.8 and 7.4, of 8192 to 512 23 and 12).
  if (I <= kFewRows) {
    const int64_t a_cu = ((J + 15) / 16 + kCUs - 1) / kCUs;
    if (std::max(0.5, K / 2048.0) * a_cu * (1.5 + 0.11 * I) < best + 2.2) p = Plan{0, 0, 0, 1};
  }
  return p;
}

// LDS buffers of the ring: four where a CU has one work-group, with the room of two
int buffers_of(int tile, int64_t work_groups) { return tile == 64 || (tile == 128 && work_groups <= kCUs) ? 4 : 2; }

struct Layout {
  int64_t codes, a_scales, b_scales, part, bytes;
  int64_t a_rows, b_rows;
  int steps;
};
Layout layout_of(const Plan& p, int64_t M, int64_t N, int64_t K, bool quantized) {
  Layout l = {};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t x = at;
    at += round256(bytes);
    return x;
  };
  if (p.tile) {
    l.steps = (int)((K + kStepElements - 1) / kStepElements);
    l.a_rows = (M + kTileRows - 1) / kTileRows * kTileRows;
    l.b_rows = (N + kTileRows - 1) / kTileRows * kTileRows;
    if (!quantized) l.codes = take(M * (K / 2));
    l.a_scales = take(l.a_rows * l.steps * kStepBlocks);
    l.b_scales = take(l.b_rows * l.steps * kStepBlocks);
    if (p.split > 1) l.part = take((int64_t)p.split * M * N * 4);
  }
  l.bytes = at;
  return l;
}

template <int TI, int TJ, int WI, int WJ, int NB>
void launch_tiles(const MxArgs& g, unsigned blocks, hipStream_t st) {
  hipLaunchKernelGGL((mx_tile_kernel<TI, TJ, WI, WJ, NB>), dim3(blocks), dim3(64 * WI * WJ), 0, st, g);
}

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
  return layout_of(plan_of(n_rows, n_out, n_in), n_rows, n_out, n_in, quantized != 0).bytes;
}

extern "C" int or_mx_linear_plan(int64_t n_rows, int32_t n_in, int32_t n_out, int32_t* tile, int32_t* buffers, int32_t* split) {
  if (int rc = check_product("or_mx_linear_plan", n_rows, n_in, n_out)) return rc;
  if (!tile || !buffers || !split) return fail_arg("or_mx_linear_plan: tile, buffers and split are required");
  const Plan p = plan_of(n_rows, n_out, n_in);
  *tile = p.tile;
  *buffers = p.tile ? buffers_of(p.tile, (int64_t)p.tiles_i * p.tiles_j * p.split) : 0;
  *split = p.split;
  return 0;
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
  char* ws = (char*)x.workspace;
  const Plan plan = plan_of(x.n_rows, x.n_out, x.n_in);
  const Layout l = layout_of(plan, x.n_rows, x.n_out, x.n_in, quantized);
  MxArgs g = {};
  g.I = x.n_rows;
  g.J = x.n_out;
  g.K = x.n_in;
  g.a = quantized ? (const uint8_t*)x.x_codes : (const uint8_t*)ws + l.codes;
  g.b = (const uint8_t*)x.weight_codes;
  g.e = Epilogue{(uint16_t*)x.y, x.y_row_stride, nullptr, x.bias, x.gate, x.bias_bf16, x.gate_bf16, (const uint16_t*)x.residual,
                 x.residual_row_stride, x.activation};
  const QuantizeArgs q = {x.x, (uint8_t*)ws + l.codes, quantized ? (uint8_t*)x.x_scales : (uint8_t*)ws + l.a_scales, x.n_rows, x.x_row_stride, x.n_in};
  if (!plan.tile) {
    g.x = x.x;
    g.x_stride = x.x_row_stride;
    g.a_scales = (const uint8_t*)x.x_scales;
    g.b_scales = (const uint8_t*)x.weight_scales;
    const dim3 grid((unsigned)((g.J + 15) / 16)), block(64 * kRowWaves);
    if (g.I <= 16 && quantized) hipLaunchKernelGGL((mx_rows_kernel<1, false>), grid, block, 0, st, g);
    else if (g.I <= 16) hipLaunchKernelGGL((mx_rows_kernel<1, true>), grid, block, 0, st, g);
    else if (quantized) hipLaunchKernelGGL((mx_rows_kernel<2, false>), grid, block, 0, st, g);
    else hipLaunchKernelGGL((mx_rows_kernel<2, true>), grid, block, 0, st, g);
    return check_hip(hipGetLastError(), "mx_rows_kernel launch");
  }
  PrepareArgs r = {};
  r.q = q;
  r.a_scales = (uint8_t*)ws + l.a_scales;
  r.w_scales = (const uint8_t*)x.weight_scales;
  r.b_scales = (uint8_t*)ws + l.b_scales;
  r.a_rows = l.a_rows;
  r.b_rows = l.b_rows;
  r.n_out = x.n_out;
  r.steps = l.steps;
  const int64_t a_units = l.a_rows / 32 * r.steps, w_units = l.b_rows / 32 * r.steps;
  r.a_blocks = (int)std::min<int64_t>(a_units, kMaxBlocks);
  const unsigned w_blocks = (unsigned)std::min<int64_t>(w_units, kMaxBlocks);
  hipLaunchKernelGGL(mx_prepare_kernel, dim3(r.a_blocks + w_blocks), dim3(kThreads), 0, st, r);
  g.a_scales = r.a_scales;
  g.b_scales = r.b_scales;
  g.a_rows = l.a_rows;
  g.b_rows = l.b_rows;
  g.part = (float*)(ws + l.part);
  g.split = plan.split;
  g.by_split = divisor(plan.split);
  g.by_group = divisor(kGroup * plan.tiles_j);
  g.by_rest = divisor(std::max(1u, plan.tiles_i % kGroup));
  g.tiles_i = plan.tiles_i;
  g.tiles_j = plan.tiles_j;
  // (The rows of a last round that fills few CUs in smaller tiles, in a launch after the others': 12720 x 2048 -> 8192, 1600 tiles in 6.25
  // rounds, 155 and 13 us, one launch 171.)
  const int64_t n = (int64_t)g.tiles_i * g.tiles_j * g.split;
  const unsigned blocks = (unsigned)((n + 7) / 8 * 8);
  if (plan.tile == 256) launch_tiles<256, 256, 2, 4, 2>(g, blocks, st);
  else if (plan.tile == 128 && buffers_of(plan.tile, n) == 4) launch_tiles<128, 128, 2, 2, 4>(g, blocks, st);
  else if (plan.tile == 128) launch_tiles<128, 128, 2, 2, 2>(g, blocks, st);
  else launch_tiles<64, 64, 2, 2, 4>(g, blocks, st);
  if (g.split > 1) {
    const int64_t joins = std::min<int64_t>((g.I * g.J / 8 + kThreads - 1) / kThreads, 8192);
    hipLaunchKernelGGL(mx_join_kernel, dim3((unsigned)joins), dim3(kThreads), 0, st, g);
  }
  return check_hip(hipGetLastError(), "or_mx_linear launch");
}
