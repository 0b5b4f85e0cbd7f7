// What the linear layers' products have in common: the epilogue (bias, activation, gate, residual), tiles of an operand in LDS by
// LDS DMA, the fragments that the matrix cores take from them, and the order of the tiles.
#pragma once

#include <math.h>

#include "../../include/onereel_dit.h"
#include "common.h"

namespace onereel {

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) bf16x4 lds_bf16x4;

constexpr int kStep = 64;            // k per LDS buffer

// ------------------------------------------------------------------------------------------------------------------
// epilogue
struct Epilogue {
  uint16_t* y;
  int64_t y_stride;
  uint16_t* z;                       // optional: the pre-activation, [rows, cols] contiguous
  const void* bias;                  // optional [cols], fp32 or bf16
  const void* gate;                  // optional [cols], fp32 or bf16
  int bias_bf16, gate_bf16;
  const uint16_t* residual;          // optional
  int64_t residual_stride;
  int act;
};

// 8 columns of a parameter
__device__ __forceinline__ void load8(const void* p, int bf16, int col, float (&v)[8]) {
  if (bf16) {
    const u32x4 r = *(const u32x4*)((const uint16_t*)p + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf2f((uint16_t)(r[i] & 0xffffu));
      v[2 * i + 1] = bf2f((uint16_t)(r[i] >> 16));
    }
  } else {
    const f32x4 a = *(const f32x4*)((const float*)p + col), b = *(const f32x4*)((const float*)p + col + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < 4 ? a[i] : b[i - 4];
  }
}

// 1 / (1 + 2^x) with v_exp_f32 and v_rcp_f32, good to 2^-22 (a full division costs the epilogue of a 256 x 256 tile as
// much again as the rest of a GELU: the layer of 12720 x 2048 -> 8192 478 us with it, 455 so; the activation asked for once
// for 8 columns and its constants folded, 480 and 466 in turn)
__device__ __forceinline__ float falling(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x)); }
constexpr float kLog2e = 1.44269504088896340736f;
__device__ __forceinline__ float logistic(float x) { return falling(x * -kLog2e); }

// 0.5 z (1 + tanh u) = z / (1 + exp(-2 u)), u = sqrt(2 / pi) (z + 0.044715 z^3)
constexpr float kGelu1 = 2 * 0.7978845608028654f, kGelu3 = kGelu1 * 0.044715f;
__device__ __forceinline__ float gelu(float z) { return z * falling(z * fmaf(-kLog2e * kGelu3, z * z, -kLog2e * kGelu1)); }
__device__ __forceinline__ float silu(float z) { return z * logistic(z); }

// act(z) and act'(z). The derivative is taken at z clamped to where it has reached 0 or 1 in fp32, so that nothing is 0 * inf:
// +-20 for GELU (within exp(-600) of it), +-100 for SiLU, whose derivative falls as z exp(z) only: -3.9e-8 at -20.
__device__ __forceinline__ void act_grad(float z, int act, float& f, float& d) {
  f = z;
  d = 1.0f;
  if (act == OR_ACT_NONE) return;
  const float far = act == OR_ACT_SILU ? 100.0f : 20.0f, c = fminf(fmaxf(z, -far), far);
  if (act == OR_ACT_SILU) {
    const float p = logistic(c);
    d = p + c * p * (1.0f - p);
  } else {
    const float u = c * (kGelu1 + kGelu3 * c * c), p = logistic(u), q = logistic(-u);
    d = p + c * p * q * (kGelu1 + 3.0f * kGelu3 * c * c);
  }
  if (z != z) d = z;
  f = act == OR_ACT_SILU ? silu(z) : gelu(z);
}

// 8 columns col .. of one row from the fp32 products v
__device__ __forceinline__ void finish8(const Epilogue& e, int64_t row, int col, int cols, float (&v)[8]) {
  float t[8];
  if (e.bias) {
    load8(e.bias, e.bias_bf16, col, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += t[i];
  }
  if (e.z) *(u32x4*)(e.z + row * cols + col) = u32x4{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
  if (e.act == OR_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gelu(v[i]);
  } else if (e.act == OR_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = silu(v[i]);
  }
  if (e.gate) {
    load8(e.gate, e.gate_bf16, col, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= t[i];
  }
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

// ------------------------------------------------------------------------------------------------------------------
// tiles

struct Operand {
  const uint16_t* p;
  int64_t stride;                    // elements between its rows (rows of i or j, or rows of k when transposed)
};

__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)(uintptr_t)(const lds_void*)p; }

__device__ __forceinline__ void dma16(const i32x4& r, uint32_t off, uint32_t m0) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r),
               "s"(__builtin_amdgcn_readfirstlane(m0))
               : "memory");
}

__device__ __forceinline__ i32x4 descriptor(const uint16_t* p, int32_t bytes) {
  const uint64_t b = (uint64_t)p;
  return i32x4{__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)b),
               __builtin_amdgcn_readfirstlane((int32_t)(uint32_t)(b >> 32)), __builtin_amdgcn_readfirstlane(bytes),
               0x00020000};
}

// One operand's tile of N rows x kStep in LDS. TR false: N rows of 64 k (128 bytes each); TR true: 64 rows of k of N
// elements. Chunk c (16 bytes) of row r lies at position c ^ swz(r).
template <int N, bool TR, int THREADS, int WAVES>
struct Tile {
  static constexpr int CH = TR ? N / 8 : kStep / 8;      // chunks per row
  static constexpr int BYTES = N * kStep * 2;
  static constexpr int LOADS = BYTES / 16 / THREADS;    // DMA loads per lane
  static constexpr int W = N / WAVES, F = W / 32;            // a wavefront's share and its blocks of 32
  static_assert(LOADS >= 1, "tile");

  static __device__ __forceinline__ int swz(int r) {
    if constexpr (!TR) return (r >> 1) & 7;
    else if constexpr (CH == 8) return ((r >> 1) & 1) << 2;
    else return (r & 3) << 2;
  }
  uint32_t off[LOADS];               // byte offset of each load from the tile's first element
  int chunk[LOADS];                  // its column of the row, in chunks
  __device__ __forceinline__ void init(int tid, int64_t stride) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int x = i * THREADS + tid, r = x / CH, c = (x % CH) ^ swz(r);
      off[i] = (uint32_t)(r * stride * 2 + c * 16);
      chunk[i] = c;
    }
  }
  // steps of k to load: the rows (or columns) n0 .. of n of the operand, from k0 to k1
  const uint16_t* p;
  int64_t pitch;                     // elements from one step to the next
  int other, left;                   // rows that end the tile (TR: columns), k left
  int64_t row_bytes;
  __device__ __forceinline__ void start(const Operand& o, int64_t n0, int64_t n, int k0, int k1) {
    p = o.p + (TR ? k0 * o.stride + n0 : n0 * o.stride + k0);
    pitch = TR ? kStep * o.stride : kStep;
    other = (int)min(n - n0, (int64_t)N);
    left = k1 - k0;
    row_bytes = o.stride * 2;
  }
  // a step's loads, one at a time: prepare(), one(0 .. LOADS - 1), then the next step
  i32x4 desc;
  int wide;
  __device__ __forceinline__ void prepare() {
    const int ks = min(max(left, 0), kStep), rows = TR ? ks : other;
    wide = TR ? other : ks;
    desc = descriptor(p, ks > 0 ? (int32_t)((rows - 1) * row_bytes) + wide * 2 : 0);
    p += pitch;
    left -= kStep;
  }
  __device__ __forceinline__ void one(int i, uint32_t m0) const {
    dma16(desc, chunk[i] * 8 < wide ? off[i] : 0x80000000u, m0 + i * THREADS * 16);
  }
};

// operand fragments of a wavefront: block f of 32 rows, step ks of 16 k (8 (lane / 32) + 0 .. 7 of them in this lane)
template <int N, bool TR, int THREADS, int WAVES>
struct Frag {
  static constexpr int FS = TR ? (N / WAVES / 32) : kStep / 16;
  uint32_t at[FS];                   // TR: one per block of 32, else one per step
  __device__ __forceinline__ void init(int lane, int half) {
    using T = Tile<N, TR, THREADS, WAVES>;
    const int l32 = lane & 31, h = lane >> 5, r = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
    for (int x = 0; x < FS; ++x) {
      if constexpr (TR) {
        const int row = 8 * h + (r >> 2), c = (half * T::W + 32 * x) / 8 + 2 * g + ((r >> 1) & 1);
        at[x] = row * N * 2 + (c ^ T::swz(row)) * 16 + (r & 1) * 8;
      } else {
        const int row = half * T::W + l32;
        at[x] = row * kStep * 2 + ((2 * x + h) ^ T::swz(row)) * 16;
      }
    }
  }
  // Addresses of one half (32 k) of the buffer at `buf`, one vector register each (kept from being rebuilt out of scalar sums
  // for every read); the blocks (or steps) are immediates from it.
  static constexpr int F = N / WAVES / 32, P = TR ? F : 2;
  template <int HALF>
  __device__ __forceinline__ void aim(uint32_t buf, uint32_t (&p)[P]) const {
#pragma unroll
    for (int x = 0; x < P; ++x) {
      p[x] = buf + at[TR ? x : 2 * HALF + x];
      asm volatile("" : "+v"(p[x]));
    }
  }
  template <int HALF>
  static __device__ __forceinline__ bf16x8 read(const uint32_t (&p)[P], int ks, int f) {
    if constexpr (TR) {
      u32x2 x[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        x[t] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                             (lds_bf16x4*)(uintptr_t)(p[f] + (32 * HALF + 16 * ks + 4 * t) * N * 2)));
      return __builtin_bit_cast(bf16x8, u32x4{x[0][0], x[0][1], x[1][0], x[1][1]});
    } else {
      return *(const __attribute__((address_space(3))) bf16x8*)(uintptr_t)(p[ks] + f * 32 * kStep * 2);
    }
  }
};

// Tiles in groups of 8 rows of tiles: the work-groups of one XCD (index modulo 8) take consecutive tiles, which share
// their operands' rows in that XCD's L2.
template <typename G>
__device__ __forceinline__ bool tile_of(const G& g, int block, int& ti, int& tj, int& part) {
  const int64_t n = (int64_t)g.tiles_i * g.tiles_j * g.split, per = (n + 7) / 8, j = block >> 3;
  int64_t x = (block & 7) * per + j;
  if (j >= per || x >= n) return false;
  part = (int)(x % g.split);
  x /= g.split;
  constexpr int kGroup = 8;
  const int64_t group = x / ((int64_t)kGroup * g.tiles_j), in = x % ((int64_t)kGroup * g.tiles_j);
  const int high = min(kGroup, g.tiles_i - (int)group * kGroup);
  ti = (int)(group * kGroup + in % high);
  tj = (int)(in / high);
  return true;
}

}  // namespace
}  // namespace onereel
