// The norms before and after a sub-block (attention, feed forward), fused with its gate and residual, and their gradient. Built
// into libonereel_dit.so (include/onereel_dit.h). Per row of C elements, in fp32, with one vector of gate, scale and shift for
// every group of `per` consecutive rows (a frame, a scene, or all rows):
//
//   p = Post(a) * wp        h = r x + gate p        n = (Norm(h) w + b) (1 + scale) + shift
//
// Norm is (v - m) / sqrt(mean (v - m)^2 + eps) (layer) or v / sqrt(mean v^2 + eps) (RMS), Post one of them or nothing. h is
// rounded once, and n comes from h before that rounding. The gradient reads the rounded h and a (xh, ah: what the two norms
// make of them, s and sa the factors they multiply by):
//
//   t = dn W, W = w (1 + scale)         d = dh + s (t - mean t - xh mean(t xh))        dx = r d
//   u = d G,  G = gate wp               da = sa (u - mean u - ah mean(u ah))           (without Post: da = u)
//   A = sum dn xh, B = sum dn, D = sum d ah over the rows of a group:
//   dshift = B, dscale = w A + b B, dgate = wp D;   dw = sum (1 + scale) A, db = sum (1 + scale) B, dwp = sum gate D over groups
//
// (the terms mean t and mean u are the layer norm's alone). Three column sums serve all six parameters' gradients.
//
// HBM-bound: x and a are read and h and n written once, h, a, dh and dn are read and dx and da written once. A work-group takes
// rows of one group, each of its threads 8 columns of them, so that the parameters stay in registers, folded into two or three
// vectors; a row's sums go over lanes within a wavefront, then through LDS: one barrier a row, since each wavefront
// hands on its own mean and the squares around that, which are joined without cancellation. In the gradient a thread adds up its
// columns' A, B and D over its work-group's rows, in a fixed order; a second launch joins the work-groups' sums, unless there are so
// many groups that each is one work-group's, which then makes the group's gradients by itself. 12720 x 2048 in bf16
// with gate, scale and shift of 8 groups, among other work: forward 40.3 us for 208 MB (5.2 TB/s, the rate of a copy of 1 GB here
// 5.15 to 5.5); gradient 70.2 us for 313 MB, 65 of them in the first launch (4.8 TB/s) and 5 in the column sums.
#include <math.h>

#include <algorithm>

#include "../../include/onereel_dit.h"
#include "rows.h"

namespace onereel {

namespace {

constexpr int kMaxC = 8192;            // 1024 threads of 8 columns
constexpr int kMaxWaves = 16;
constexpr int kCUs = 256, kBwdBlocks = 512;
constexpr int kMaxPartRows = 256;      // rows whose sums a thread adds up one after the other

struct NormArgs {
  const void *x, *a;
  void *h, *n;
  const float *gate, *post_weight, *weight, *bias, *scale, *shift;   // gate, scale, shift: [groups][C]
  int64_t per, x_stride, a_stride;
  int64_t spans;                       // groups x parts
  int C, parts, norm, post;            // parts: work-groups of a group of rows
  float eps, r;
};

// 8 columns of a vector of parameters, or `other` where there is none
__device__ __forceinline__ void param8(const float* p, int64_t at, bool in, float other, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = other;
  if (p && in) {
    const f32x4 a = *(const f32x4*)(p + at), b = *(const f32x4*)(p + at + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < 4 ? a[i] : b[i - 4];
  }
}

// a wavefront's columns of a row of C: their mean and the sum of squares around it (RMS: around 0), and what else it hands on
struct Share {
  float mean, square, t, tx;
};

// columns of wavefront w of a row of C
__device__ __forceinline__ int wave_columns(int C, int w) { return min(512, C - 512 * w); }

__device__ __forceinline__ void moments(const float (&v)[8], bool in, float a_column, int norm, Share& s) {
  float sum = 0.0f;
  s.mean = 0.0f;
  if (norm == OR_NORM_LAYER) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += v[i];
    s.mean = wave_sum(in ? sum : 0.0f) * a_column;
    sum = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += (v[i] - s.mean) * (v[i] - s.mean);
  s.square = wave_sum(in ? sum : 0.0f);
}

// The wavefronts' shares are joined by 16 lanes, each with one of them (every 16 lanes of every wavefront do the same): one read of
// LDS and sums over lanes. (Loops over the shares, one read after the other: 4096 x
// 8192 63.9 us, so 55.4, with a norm ahead 98 and 62; the gradient of 12720 x 4096 147 and 137, with a norm ahead of 2048 91 and 76.)
struct Joiner {
  int wave, waves;
  float columns, a_column;             // of the lane's share, 0 past the last; 1 / C
  __device__ __forceinline__ Joiner(int C) : wave(threadIdx.x & 15), waves(blockDim.x >> 6), a_column(1.0f / (float)C) {
    columns = wave < waves ? (float)wave_columns(C, wave) : 0.0f;
  }
  __device__ __forceinline__ Share take(const Share* s) const { return wave < waves ? s[wave] : Share{}; }
  // mean and 1 / sqrt(mean square + eps) of a row
  __device__ __forceinline__ void moments(const Share& s, float eps, float& mean, float& inv) const {
    mean = row_sum(s.mean * columns) * a_column;
    const float d = s.mean - mean;
    inv = rsqrtf(row_sum(s.square + d * d * columns) * a_column + eps);
  }
};

// the rows [first, last) of work-group b
struct Span {
  int64_t group, first, last;
  int part;
};
__device__ __forceinline__ Span span_of(int64_t block, int parts, int64_t per) {
  Span s;
  s.group = block / parts;
  s.part = (int)(block - s.group * parts);
  s.first = s.group * per + per * s.part / parts;
  s.last = s.group * per + per * (s.part + 1) / parts;
  return s;
}

// What a row has beside x: nothing, a sub-block's output, or one with a norm of its own
enum { kNoResidual, kResidual, kPostNorm };

// Work-groups of up to N threads take one row after the other, the next one's loads under way ahead of a row's sums. (Two rows a
// barrier and no loads ahead: 41.6 us for 12720 x 2048 with gate, scale and shift of 8 groups, the gradient 75.9.)
template <typename T, int KIND, int N>
__global__ __launch_bounds__(N) void block_norm_kernel(NormArgs g) {
  __shared__ Share post_share[2][kMaxWaves], share[2][kMaxWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = 8 * threadIdx.x, C = g.C;
  const bool in = col < C;
  const float a_column = 1.0f / (float)wave_columns(C, wave);
  const Joiner join(C);
  int turn = 0;
  for (int64_t span = blockIdx.x; span < g.spans; span += gridDim.x) {
    const Span s = span_of(span, g.parts, g.per);
    const int64_t at = s.group * C + col;
    Piece<T, 8> x, a;
    auto load = [&](int64_t r) {
      if (in) {
        x.load(g.x, r * g.x_stride + col);
        if constexpr (KIND != kNoResidual) a.load(g.a, r * g.a_stride + col);
      }
    };
    x.zero();
    a.zero();
    load(s.first);
    float G[8], W[8], B[8], t[8];
    if constexpr (KIND != kNoResidual) param8(g.gate, at, in, 1.0f, G);
    if constexpr (KIND == kPostNorm) {
      param8(g.post_weight, col, in, 1.0f, t);
#pragma unroll
      for (int i = 0; i < 8; ++i) G[i] *= t[i];
    }
    param8(g.weight, col, in, 1.0f, W);
    param8(g.bias, col, in, 0.0f, B);
    param8(g.scale, at, in, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      W[i] *= 1.0f + t[i];
      B[i] *= 1.0f + t[i];
    }
    param8(g.shift, at, in, 0.0f, t);
#pragma unroll
    for (int i = 0; i < 8; ++i) B[i] += t[i];
    for (int64_t r = s.first; r < s.last; ++r, turn ^= 1) {
      float h[8], mean, inv;
      Share m;
      x.get(h);
      if constexpr (KIND != kNoResidual) {
        float p[8];
        a.get(p);
        if (r + 1 < s.last) load(r + 1);
        if constexpr (KIND == kPostNorm) {
          moments(p, in, a_column, g.post, m);
          if (lane == 0) post_share[turn][wave] = m;
          __syncthreads();
          join.moments(join.take(post_share[turn]), g.eps, mean, inv);
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = (p[i] - mean) * inv;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = g.r * h[i] + p[i] * G[i];
        if (in) Piece<T, 8>::store(g.h, r * C + col, h);
      } else if (r + 1 < s.last) {
        load(r + 1);
      }
      moments(h, in, a_column, g.norm, m);
      if (lane == 0) share[turn][wave] = m;
      __syncthreads();
      join.moments(join.take(share[turn]), g.eps, mean, inv);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = (h[i] - mean) * inv * W[i] + B[i];
      if (in) Piece<T, 8>::store(g.n, r * C + col, h);
    }
  }
}

struct NormBwdArgs {
  const void *dh, *dn, *h, *a;         // dh optional
  void *dx, *da;
  const float *gate, *post_weight, *weight, *bias, *scale;
  float *dgate, *dpost_weight, *dweight, *dbias, *dscale, *dshift;   // each optional
  float* part;                         // [groups * parts][3][C]: A, B, D
  float* terms;                        // [n_terms][3][C] of dweight, dbias, dpost_weight: of a group, or (alone) of a work-group
  int64_t n_terms;
  int64_t per, groups, dh_stride, dn_stride, h_stride, a_stride;
  int C, parts, norm, post;
  unsigned blocks;
  bool alone;
  float eps, r;
};

__device__ __forceinline__ void put8(float* p, const float (&v)[8]) {
  *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
  *(f32x4*)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
}

// The gradients of a group's own 8 columns from their sums, and their terms of the weights' gradients, added up in LDS
__device__ __forceinline__ void alone8(const NormBwdArgs& g, int64_t at, int col, const float (&A)[8], const float (&B)[8],
                                       const float (&D)[8], float* term) {
  float x[8], y[8];
  if (g.dshift) put8(g.dshift + at, B);
  if (g.dscale) {
    param8(g.weight, col, true, 1.0f, x);
    param8(g.bias, col, true, 0.0f, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * A[i] + y[i] * B[i];
    put8(g.dscale + at, x);
  }
  if (g.dgate) {
    param8(g.post_weight, col, true, 1.0f, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= D[i];
    put8(g.dgate + at, x);
  }
  if (!g.terms) return;
  param8(g.scale, at, true, 0.0f, x);
  param8(g.gate, at, true, 1.0f, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    term[col + i] += (1.0f + x[i]) * A[i];
    term[g.C + col + i] += (1.0f + x[i]) * B[i];
    term[2 * g.C + col + i] += y[i] * D[i];
  }
}

// ALONE: a group has one work-group, which makes its gradients by itself
template <typename T, int KIND, int N, bool ALONE>
__global__ __launch_bounds__(N) void block_norm_bwd_kernel(NormBwdArgs g) {
  __shared__ Share share[2][kMaxWaves], post_share[2][kMaxWaves];
  __shared__ float back[2][kMaxWaves][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = 8 * threadIdx.x, C = g.C;
  const bool in = col < C;
  const float a_column = 1.0f / (float)wave_columns(C, wave);
  const Joiner join(C);
  extern __shared__ __attribute__((aligned(16))) float term[];        // alone: [3][C], each thread's columns its own
  if (ALONE && g.terms && in) {
#pragma unroll
    for (int i = 0; i < 3; ++i) *(f32x4*)(term + i * C + col) = *(f32x4*)(term + i * C + col + 4) = f32x4{0, 0, 0, 0};
  }
  int turn = 0;
  for (int64_t span = blockIdx.x; span < g.groups * g.parts; span += gridDim.x) {
    const Span s = span_of(span, g.parts, g.per);
    const int64_t at = s.group * C + col;
    struct Row {
      Piece<T, 8> h, n, d, a;
    } now, next;
    auto load = [&](Row& to, int64_t r) {
      if (in) {
        to.h.load(g.h, r * g.h_stride + col);
        to.n.load(g.dn, r * g.dn_stride + col);
        if constexpr (KIND != kNoResidual) {
          if (g.dh) to.d.load(g.dh, r * g.dh_stride + col);
          to.a.load(g.a, r * g.a_stride + col);
        }
      }
    };
    next.h.zero();
    next.n.zero();
    next.d.zero();
    next.a.zero();
    load(next, s.first);
    float G[8], W[8], v[8], A[8], B[8], D[8];
    if constexpr (KIND != kNoResidual) param8(g.gate, at, in, 1.0f, G);
    if constexpr (KIND == kPostNorm) {
      param8(g.post_weight, col, in, 1.0f, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) G[i] *= v[i];
    }
    param8(g.weight, col, in, 1.0f, W);
    param8(g.scale, at, in, 0.0f, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      W[i] *= 1.0f + v[i];
      A[i] = B[i] = D[i] = 0.0f;
    }
    for (int64_t r = s.first; r < s.last; ++r, turn ^= 1) {
      now = next;
      if (r + 1 < s.last) load(next, r + 1);
      float h[8], n[8], t = 0.0f, tx = 0.0f, sum = 0.0f, mean, inv;
      Share m = {};
      now.h.get(h);
      now.n.get(n);
      if (g.norm == OR_NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum += h[i];
          t += n[i] * W[i];
        }
        wave_sums(in ? sum : 0.0f, in ? t : 0.0f, m.mean, m.t);
        m.mean *= a_column;
        sum = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float c = h[i] - m.mean;
        sum += c * c;
        tx += n[i] * W[i] * c;
      }
      wave_sums(in ? sum : 0.0f, in ? tx : 0.0f, m.square, m.tx);
      if (lane == 0) share[turn][wave] = m;
      float a[8];
      if constexpr (KIND != kNoResidual) now.a.get(a);
      if constexpr (KIND == kPostNorm) {
        moments(a, in, a_column, g.post, m);
        if (lane == 0) post_share[turn][wave] = m;
      }
      __syncthreads();
      m = join.take(share[turn]);
      join.moments(m, g.eps, mean, inv);
      t = g.norm == OR_NORM_LAYER ? row_sum(m.t) * join.a_column : 0.0f;
      tx = row_sum(m.tx + (m.mean - mean) * m.t) * inv * join.a_column;
      float d[8];
      now.d.get(d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = (h[i] - mean) * inv;
        A[i] += n[i] * xh;
        B[i] += n[i];
        d[i] += inv * (n[i] * W[i] - t - xh * tx);
      }
      if constexpr (KIND == kNoResidual) {
        if (in) Piece<T, 8>::store(g.dx, r * C + col, d);
      } else {
        float u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          u[i] = d[i] * G[i];
          h[i] = g.r * d[i];
        }
        if (in) Piece<T, 8>::store(g.dx, r * C + col, h);
        if constexpr (KIND == kPostNorm) {
          join.moments(join.take(post_share[turn]), g.eps, mean, inv);
          float su = 0.0f, sux = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] = (a[i] - mean) * inv;
            su += u[i];
            sux += u[i] * a[i];
          }
          wave_sums(in ? su : 0.0f, in ? sux : 0.0f, su, sux);
          if (lane == 0) {
            back[turn][wave][0] = su;
            back[turn][wave][1] = sux;
          }
          __syncthreads();
          const bool has = join.wave < join.waves;
          su = g.post == OR_NORM_LAYER ? row_sum(has ? back[turn][join.wave][0] : 0.0f) * join.a_column : 0.0f;
          sux = row_sum(has ? back[turn][join.wave][1] : 0.0f) * join.a_column;
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = inv * (u[i] - su - a[i] * sux);
        }
        if (in) Piece<T, 8>::store(g.da, r * C + col, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) D[i] += d[i] * a[i];
      }
    }
    if (!in) continue;
    if constexpr (ALONE) {
      alone8(g, at, col, A, B, D, term);
      continue;
    }
    if (!g.part) continue;
    float* out = g.part + span * 3 * C + col;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *(f32x4*)(out + i) = f32x4{A[i], A[i + 1], A[i + 2], A[i + 3]};
      *(f32x4*)(out + C + i) = f32x4{B[i], B[i + 1], B[i + 2], B[i + 3]};
      *(f32x4*)(out + 2 * C + i) = f32x4{D[i], D[i + 1], D[i + 2], D[i + 3]};
    }
  }
  if (!ALONE || !g.terms || !in) return;
  float* out = g.terms + (int64_t)blockIdx.x * 3 * C + col;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    *(f32x4*)(out + i * C) = *(f32x4*)(term + i * C + col);
    *(f32x4*)(out + i * C + 4) = *(f32x4*)(term + i * C + col + 4);
  }
}

// The groups' sums of 64 columns, those of a group's work-groups dealt out to WAVES of 16 wavefronts: all of them, or one for up to 8
// work-groups (the whole gradient of 240 groups of 53 x 2048 with 3 each 81.5 us, so, 93.9 with 4 wavefronts a group; 80 of 20 x 4096
// 29.9 and 35.3). Then its parameters' gradients, or their terms. (16 columns a work-group and four times as many of them: 7.2 us, so
// 5.1, for 8 groups of 64 work-groups and 2048 columns.)
constexpr int kSumWaves = 16;
template <int WAVES>
__global__ __launch_bounds__(64 * kSumWaves) void block_norm_sums_kernel(NormBwdArgs g) {
  __shared__ float sum[3][kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave / WAVES * WAVES, col = blockIdx.x * 64 + lane;
  for (int64_t base = (int64_t)blockIdx.y * (kSumWaves / WAVES); base < g.groups; base += (int64_t)gridDim.y * (kSumWaves / WAVES)) {
    const int64_t group = base + wave / WAVES;
    const bool in = col < g.C && group < g.groups;
    float v[3] = {};
    if (in) {
      const float* p = g.part + group * g.parts * 3 * g.C + col;
#pragma unroll 8
      for (int b = wave - first; b < g.parts; b += WAVES)
#pragma unroll
        for (int i = 0; i < 3; ++i) v[i] += p[((int64_t)b * 3 + i) * g.C];
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) sum[i][wave][lane] = v[i];
    __syncthreads();
    if (wave == first && in) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        v[i] = 0.0f;
        for (int w = 0; w < WAVES; ++w) v[i] += sum[i][first + w][lane];
      }
      const int64_t at = group * g.C + col;
      const float w = g.weight ? g.weight[col] : 1.0f, b = g.bias ? g.bias[col] : 0.0f, e = g.scale ? 1.0f + g.scale[at] : 1.0f;
      const float gate = g.gate ? g.gate[at] : 1.0f, wp = g.post_weight ? g.post_weight[col] : 1.0f;
      if (g.dscale) g.dscale[at] = w * v[0] + b * v[1];
      if (g.dshift) g.dshift[at] = v[1];
      if (g.dgate) g.dgate[at] = wp * v[2];
      const float term[3] = {e * v[0], e * v[1], gate * v[2]};
      if (g.groups == 1) {
        if (g.dweight) g.dweight[col] = term[0];
        if (g.dbias) g.dbias[col] = term[1];
        if (g.dpost_weight) g.dpost_weight[col] = term[2];
      } else if (g.terms) {
#pragma unroll
        for (int i = 0; i < 3; ++i) g.terms[(group * 3 + i) * g.C + col] = term[i];
      }
    }
    __syncthreads();
  }
}

// the sums of the terms
__global__ __launch_bounds__(64 * kSumWaves) void block_norm_weights_kernel(NormBwdArgs g) {
  __shared__ float sum[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane, which = blockIdx.y;
  float* out = which == 0 ? g.dweight : which == 1 ? g.dbias : g.dpost_weight;
  if (!out) return;
  float v = 0.0f;
  if (col < g.C) {
#pragma unroll 8
    for (int64_t b = wave; b < g.n_terms; b += kSumWaves) v += g.terms[(b * 3 + which) * g.C + col];
  }
  sum[wave][lane] = v;
  __syncthreads();
  if (wave != 0 || col >= g.C) return;
  v = 0.0f;
  for (int w = 0; w < kSumWaves; ++w) v += sum[w][lane];
  out[col] = v;
}

bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
int threads_of(int C) { return (C / 8 + 63) / 64 * 64; }

// Work-groups of a group of `per` rows, up to `most` a CU: as many as keep a CU shortest, of whose wavefronts it has room for 16 at a
// time, a work-group's own start being worth a row. What a row takes follows the wavefronts on the fullest of the four SIMDs, and is
// no shorter than with `least` on each, which the loads under way need.
// (768 work-groups and more for the forward, 512 for the gradient, rounded up to whole ones a group, on the left: 113 groups of 189 x
// 2424 with a norm ahead 117 and 102 us, 4096 x 8192 64 and 55; gradients of 24 groups of 880 x 1536 106 and 92, 100 of 200 x 2048 131
// and 118, 4096 x 8192 111 and 95. Up to four a CU for the gradient: 24 of 880 x 1536 105.)
int64_t parts_of(int64_t per, int64_t groups, int C, int least, int most) {
  const int64_t waves = threads_of(C) / 64, at_once = std::max<int64_t>(1, 16 / waves);
  const auto load = [&](int64_t n) { return n ? std::max<int64_t>(least, (n * waves + 3) / 4) : 0; };
  int64_t best = 1, shortest = INT64_MAX;
  for (int k = 1; k <= most; ++k) {
    const int64_t parts = std::min(per, kCUs * k / groups);
    if (parts < 1) continue;
    const int64_t a_cu = (parts * groups + kCUs - 1) / kCUs;
    const int64_t cost = (a_cu / at_once * load(at_once) + load(a_cu % at_once)) * ((per + parts - 1) / parts + 1);
    if (cost < shortest) {
      shortest = cost;
      best = parts;
    }
    if (parts == per) break;
  }
  return best;
}

int check_sizes(const char* what, int64_t rows, int64_t per, int32_t C, int32_t type) {
  if (!known_type(type)) return fail_arg("%s: unknown element type %d", what, type);
  if (C < 8 || C % 8 || C > kMaxC) return fail_arg("%s: rows of a multiple of 8 elements up to %d (got %d)", what, kMaxC, C);
  if (rows < 0 || rows > (int64_t)1 << 30) return fail_arg("%s: 0 to 2^30 rows (got %lld)", what, (long long)rows);
  if (rows > 0 && (per < 1 || rows % per)) return fail_arg("%s: rows_per_group must divide the rows", what);
  return 0;
}

int check_norms(const char* what, int norm, int post) {
  if (norm != OR_NORM_LAYER && norm != OR_NORM_RMS) return fail_arg("%s: norm must be OR_NORM_LAYER or OR_NORM_RMS", what);
  if (post != OR_NORM_NONE && post != OR_NORM_LAYER && post != OR_NORM_RMS) return fail_arg("%s: unknown post_norm %d", what, post);
  return 0;
}

int bad_rows(const char* what, const void* p, int64_t stride, int C) {
  if (!p) return fail_arg("%s is required", what);
  if (!al16(p) || stride < C || stride % 8) return fail_arg("%s: 16-byte aligned rows, a multiple of 8 elements apart, that cover C", what);
  return 0;
}

// Work-groups of the gradient. Each writes 3 sums of C columns, which the second launch reads, so there are as few as keep the
// GPU's loads in flight; and no thread adds up more than kMaxPartRows rows in a row.
//
// A group of few rows is one work-group's where the rows that this takes one after the other cost less than a second launch over
// many groups' sums, a row about as much as 24 groups (in one work-group each and divided, us: 300 groups of 20 x 2048 46 and 51, 100 of
// 4 x 8192 32 and 36; 160 of 12 x 512 17.5 and 15.2, 80 of 20 x 4096 40 and 30, 99 of 13 x 5432 73 and 57). From 256 rows on a
// work-group has two or more (333 x 1000 in 167 work-groups 12.5 us, 333 13.8; 512 x 2048 14.7, 19.6; 76 x 3584 in 38 13.2, 76 12.3).
int64_t bwd_parts(int64_t per, int64_t groups, int C) {
  const int64_t rows = per * groups, turns = (rows + kBwdBlocks - 1) / kBwdBlocks;
  if (groups > 1 && (per - turns) * 24 <= groups) return (per + kMaxPartRows - 1) / kMaxPartRows;
  const int64_t parts = std::min(parts_of(per, groups, C, 2, 3), rows < 256 ? per : (per + 1) / 2);
  return std::max(parts, (per + kMaxPartRows - 1) / kMaxPartRows);
}

constexpr int64_t kMaxBlocks = 1 << 20;   // of up to 1024 threads: a grid has under 2^32 of them

// Where the gradient's sums lie in the workspace: those of the work-groups, unless each group has but one, and the terms of the
// weights' gradients. A group that is one work-group's has its gradients from there: 12720 x 2048 in 1590 groups 94 us, in as many as
// rows 203 (467 and 3180 through the second launch); 1024 or 2048 work-groups instead of 512 93 and 235, 99 and 206.
struct BwdPlan {
  int64_t groups, parts, blocks, part_bytes, n_terms, bytes;
  bool alone;
};
BwdPlan bwd_plan(int64_t rows, int64_t per, int C) {
  BwdPlan p = {};
  p.groups = rows / per;
  p.parts = bwd_parts(per, p.groups, C);
  p.alone = p.groups > 1 && p.parts == 1;
  p.blocks = std::min({p.groups * p.parts, p.alone ? std::max<int64_t>(kBwdBlocks, p.groups / kMaxPartRows) : kMaxBlocks, kMaxBlocks});
  p.part_bytes = p.alone ? 0 : p.groups * p.parts * 3 * C * 4;
  p.n_terms = p.alone ? p.blocks : p.groups > 1 ? p.groups : 0;
  p.bytes = p.part_bytes + p.n_terms * 3 * C * 4;
  return p;
}

template <typename T, int KIND, int N>
void launch_kind(const NormArgs& g, hipStream_t st) {
  const dim3 grid((unsigned)std::min(g.spans, kMaxBlocks)), block((unsigned)threads_of(g.C));
  hipLaunchKernelGGL((block_norm_kernel<T, KIND, N>), grid, block, 0, st, g);
}

template <typename T, int KIND, int N>
void launch_kind(const NormBwdArgs& g, hipStream_t st) {
  const dim3 grid(g.blocks), block((unsigned)threads_of(g.C));
  if (g.alone) hipLaunchKernelGGL((block_norm_bwd_kernel<T, KIND, N, true>), grid, block, g.terms ? 3 * g.C * 4 : 0, st, g);
  else hipLaunchKernelGGL((block_norm_bwd_kernel<T, KIND, N, false>), grid, block, 0, st, g);
}

template <typename T, int KIND, typename G>
void launch_width(const G& g, hipStream_t st) {
  const int n = threads_of(g.C);
  if (n <= 256) launch_kind<T, KIND, 256>(g, st);
  else if (n <= 512) launch_kind<T, KIND, 512>(g, st);
  else launch_kind<T, KIND, 1024>(g, st);
}

template <typename T, typename G>
void launch_type(const G& g, hipStream_t st) {
  if (!g.a) launch_width<T, kNoResidual>(g, st);
  else if (g.post == OR_NORM_NONE) launch_width<T, kResidual>(g, st);
  else launch_width<T, kPostNorm>(g, st);
}

template <typename G>
void launch(const G& g, int type, hipStream_t st) {
  if (type == OR_TYPE_BF16) launch_type<Bf16>(g, st);
  else if (type == OR_TYPE_FP16) launch_type<_Float16>(g, st);
  else launch_type<float>(g, st);
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int or_block_norm(const or_block_norm_args* p, void* stream) {
  if (!p) return fail_arg("or_block_norm: args is NULL");
  const or_block_norm_args& x = *p;
  if (int rc = check_sizes("or_block_norm", x.n_rows, x.rows_per_group, x.C, x.type)) return rc;
  if (int rc = check_norms("or_block_norm", x.norm, x.post_norm)) return rc;
  if (x.n_rows == 0) return 0;
  if (int rc = bad_rows("or_block_norm: x", x.x, x.x_row_stride, x.C)) return rc;
  if (int rc = bad_rows("or_block_norm: n", x.n, x.C, x.C)) return rc;
  if (x.a) {
    if (int rc = bad_rows("or_block_norm: a", x.a, x.a_row_stride, x.C)) return rc;
    if (int rc = bad_rows("or_block_norm: h", x.h, x.C, x.C)) return rc;
  } else if (x.gate || x.post_weight || x.post_norm != OR_NORM_NONE) {
    return fail_arg("or_block_norm: gate, post_norm and post_weight belong to a");
  }
  if (x.post_weight && x.post_norm == OR_NORM_NONE) return fail_arg("or_block_norm: post_weight belongs to a post_norm");
  if (!al16(x.gate) || !al16(x.post_weight) || !al16(x.weight) || !al16(x.bias) || !al16(x.scale) || !al16(x.shift))
    return fail_arg("or_block_norm: parameters must be 16-byte aligned");
  NormArgs g = {};
  g.x = x.x;
  g.a = x.a;
  g.h = x.h;
  g.n = x.n;
  g.gate = x.gate;
  g.post_weight = x.post_weight;
  g.weight = x.weight;
  g.bias = x.bias;
  g.scale = x.scale;
  g.shift = x.shift;
  g.per = x.rows_per_group;
  g.x_stride = x.x_row_stride;
  g.a_stride = x.a_row_stride;
  g.C = x.C;
  g.norm = x.norm;
  g.post = x.post_norm;
  g.eps = x.eps;
  g.r = x.residual_scale;
  const int64_t groups = x.n_rows / g.per;
  g.parts = (int)parts_of(g.per, groups, g.C, 3, 12);
  g.spans = groups * g.parts;
  hipStream_t st = (hipStream_t)stream;
  launch(g, x.type, st);
  return check_hip(hipGetLastError(), "block_norm_kernel launch");
}

extern "C" int64_t or_block_norm_bwd_workspace_size(int64_t n_rows, int64_t rows_per_group, int32_t C) {
  if (int rc = check_sizes("or_block_norm_bwd_workspace_size", n_rows, rows_per_group, C, OR_TYPE_BF16)) return rc;
  if (n_rows == 0) return 0;
  return bwd_plan(n_rows, rows_per_group, C).bytes;
}

extern "C" int or_block_norm_bwd(const or_block_norm_bwd_args* p, void* stream) {
  if (!p) return fail_arg("or_block_norm_bwd: args is NULL");
  const or_block_norm_bwd_args& x = *p;
  if (int rc = check_sizes("or_block_norm_bwd", x.n_rows, x.rows_per_group, x.C, x.type)) return rc;
  if (int rc = check_norms("or_block_norm_bwd", x.norm, x.post_norm)) return rc;
  if (x.n_rows == 0) return 0;
  if (int rc = bad_rows("or_block_norm_bwd: h", x.h, x.h_row_stride, x.C)) return rc;
  if (int rc = bad_rows("or_block_norm_bwd: dn", x.dn, x.dn_row_stride, x.C)) return rc;
  if (int rc = bad_rows("or_block_norm_bwd: dx", x.dx, x.C, x.C)) return rc;
  if (x.a) {
    if (int rc = bad_rows("or_block_norm_bwd: a", x.a, x.a_row_stride, x.C)) return rc;
    if (int rc = bad_rows("or_block_norm_bwd: da", x.da, x.C, x.C)) return rc;
    if (x.dh)
      if (int rc = bad_rows("or_block_norm_bwd: dh", x.dh, x.dh_row_stride, x.C)) return rc;
  } else if (x.gate || x.post_weight || x.post_norm != OR_NORM_NONE || x.dh || x.dgate || x.dpost_weight) {
    return fail_arg("or_block_norm_bwd: dh, gate, post_norm and post_weight belong to a");
  }
  if (x.post_weight && x.post_norm == OR_NORM_NONE) return fail_arg("or_block_norm_bwd: post_weight belongs to a post_norm");
  if (!al16(x.gate) || !al16(x.post_weight) || !al16(x.weight) || !al16(x.bias) || !al16(x.scale))
    return fail_arg("or_block_norm_bwd: parameters must be 16-byte aligned");
  if (!al16(x.dgate) || !al16(x.dpost_weight) || !al16(x.dweight) || !al16(x.dbias) || !al16(x.dscale) || !al16(x.dshift))
    return fail_arg("or_block_norm_bwd: the parameters' gradients must be 16-byte aligned");
  const BwdPlan plan = bwd_plan(x.n_rows, x.rows_per_group, x.C);
  const int64_t need = plan.bytes;
  const bool sums = x.dgate || x.dpost_weight || x.dweight || x.dbias || x.dscale || x.dshift;
  if (sums && (!x.workspace || !al16(x.workspace) || x.workspace_bytes < need))
    return fail_arg("or_block_norm_bwd: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  NormBwdArgs g = {};
  g.dh = x.dh;
  g.dn = x.dn;
  g.h = x.h;
  g.a = x.a;
  g.dx = x.dx;
  g.da = x.da;
  g.gate = x.gate;
  g.post_weight = x.post_weight;
  g.weight = x.weight;
  g.bias = x.bias;
  g.scale = x.scale;
  g.dgate = x.dgate;
  g.dpost_weight = x.dpost_weight;
  g.dweight = x.dweight;
  g.dbias = x.dbias;
  g.dscale = x.dscale;
  g.dshift = x.dshift;
  g.per = x.rows_per_group;
  g.groups = plan.groups;
  g.dh_stride = x.dh_row_stride;
  g.dn_stride = x.dn_row_stride;
  g.h_stride = x.h_row_stride;
  g.a_stride = x.a_row_stride;
  g.C = x.C;
  g.parts = (int)plan.parts;
  g.blocks = (unsigned)plan.blocks;
  g.alone = plan.alone && sums;
  g.norm = x.norm;
  g.post = x.post_norm;
  g.eps = x.eps;
  g.r = x.residual_scale;
  if (sums && !g.alone) g.part = (float*)x.workspace;
  const bool weights = x.dweight || x.dbias || x.dpost_weight;
  g.n_terms = plan.n_terms;
  if (weights && g.groups > 1) g.terms = (float*)((char*)x.workspace + plan.part_bytes);
  hipStream_t st = (hipStream_t)stream;
  launch(g, x.type, st);
  const unsigned columns = (unsigned)((g.C + 63) / 64);
  if (g.part) {
    const int waves = g.parts > 8 ? kSumWaves : 1;
    const dim3 grid(columns, (unsigned)std::min<int64_t>((g.groups * waves + kSumWaves - 1) / kSumWaves, 4096));
    if (waves == kSumWaves) hipLaunchKernelGGL(block_norm_sums_kernel<kSumWaves>, grid, dim3(64 * kSumWaves), 0, st, g);
    else hipLaunchKernelGGL(block_norm_sums_kernel<1>, grid, dim3(64 * kSumWaves), 0, st, g);
  }
  if (g.terms) hipLaunchKernelGGL(block_norm_weights_kernel, dim3(columns, 3), dim3(64 * kSumWaves), 0, st, g);
  return check_hip(hipGetLastError(), "or_block_norm_bwd launch");
}
