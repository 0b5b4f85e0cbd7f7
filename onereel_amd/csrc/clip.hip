// The global norm of many gradients and their clipping. Built into libonereel_dit.so (include/onereel_dit.h).
//
//   norm = sqrt(sum over all tensors and elements of g^2),   c = min(1, max_norm / (norm + 1e-6)),   out = c g
//
// HBM-bound: every gradient is read once for the norm and, where c is below 1 or out is not g, once more and written once.
// Squares are added up in fp64 from the first one on (the vector units take them faster than HBM brings the elements), so that
// neither large gradients overflow nor the order of a thousand million terms matters. Each work-group writes one partial sum, and
// every work-group of the second kernel adds all of them up in the same order: no atomics, and no launch between the two.
//
// A launch takes the addresses and lengths of up to kTensors tensors as its arguments, so nothing is copied to the device ahead
// of it. Its work-groups deal out the tensors' elements evenly, whatever their sizes: pieces of kPiece elements, a tensor's last
// one shorter, numbered through all tensors of the launch; a work-group takes consecutive pieces.
#include <math.h>

#include <algorithm>

#include "../../include/onereel_dit.h"
#include "rows.h"

namespace onereel {

namespace {

constexpr int kThreads = 512;
constexpr int kTensors = 128;          // of a launch: 128 x (8 + 8 + 8 + 4) bytes of arguments
constexpr int kPiece = 8 * kThreads;   // elements
constexpr int kBlocks = 512;           // work-groups of a launch at most: two a CU

struct Tensors {
  const void* x[kTensors];
  void* out[kTensors];                 // clipping only
  int64_t n[kTensors];
  int32_t first[kTensors + 1];         // first piece
  uint8_t type[kTensors];              // low half: of x, high half: of out
  int count, blocks;
};

struct ClipArgs {
  double* part;                        // [blocks of all launches]
  int64_t parts;
  float* norm;
  double max_norm;
};

// the tensor that piece p belongs to
__device__ __forceinline__ int tensor_of(const Tensors& t, int64_t p) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= p) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int64_t piece_of(const Tensors& t, int64_t block) {
  return (int64_t)t.first[t.count] * block / t.blocks;
}

// 8 elements at x + at, fewer at the tensor's end; whole pieces of aligned tensors in wide loads
template <typename T>
__device__ __forceinline__ void get8(const T* x, int64_t at, int64_t n, bool wide, float (&v)[8]) {
  if (wide && at + 8 <= n) {
    Piece<T, 8> p;
    p.load(x, at);
    p.get(v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.0f;
    if (at + i < n) {
      if constexpr (sizeof(T) == 4) v[i] = x[at + i];
      else if constexpr (__is_same(T, Bf16)) v[i] = bf2f(x[at + i].u);
      else v[i] = (float)x[at + i];
    }
  }
}

template <typename T>
__device__ __forceinline__ void put8(T* x, int64_t at, int64_t n, bool wide, const float (&v)[8]) {
  if (wide && at + 8 <= n) {
    Piece<T, 8>::store(x, at, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (at + i < n) {
      if constexpr (sizeof(T) == 4) x[at + i] = v[i];
      else if constexpr (__is_same(T, Bf16)) x[at + i].u = f2bf(v[i]);
      else x[at + i] = (_Float16)v[i];
    }
}

__device__ __forceinline__ void get(int type, const void* x, int64_t at, int64_t n, float (&v)[8]) {
  const bool wide = ((uintptr_t)x & 15) == 0;
  if (type == OR_TYPE_BF16) get8((const Bf16*)x, at, n, wide, v);
  else if (type == OR_TYPE_FP16) get8((const _Float16*)x, at, n, wide, v);
  else get8((const float*)x, at, n, wide, v);
}

__device__ __forceinline__ double wave_sum64(double v) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// sum over the work-group, in every thread
__device__ __forceinline__ double block_sum(double v, double* shared) {
  v = wave_sum64(v);
  if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
  for (int w = 0; w < kThreads / 64; ++w) v += shared[w];
  return v;
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(Tensors t, double* part) {
  __shared__ double shared[kThreads / 64];
  const int64_t last = piece_of(t, blockIdx.x + 1);
  int64_t p = piece_of(t, blockIdx.x);
  int k = tensor_of(t, p);
  double sum = 0.0;
  while (p < last) {
    while (t.first[k + 1] <= p) ++k;
    const int64_t end = min(last, (int64_t)t.first[k + 1]), n = t.n[k];
    for (; p < end; ++p) {
      float v[8];
      get(t.type[k] & 15, t.x[k], (p - t.first[k]) * kPiece + 8 * threadIdx.x, n, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (double)v[i] * (double)v[i];
    }
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// the norm from the partial sums, by every work-group in the same order
__device__ __forceinline__ double norm_of(const ClipArgs& c, double* shared) {
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < c.parts; i += kThreads) sum += c.part[i];
  return sqrt(block_sum(sum, shared));
}

__global__ __launch_bounds__(kThreads) void norm_kernel(ClipArgs c) {
  __shared__ double shared[kThreads / 64];
  const double norm = norm_of(c, shared);
  if (threadIdx.x == 0) *c.norm = (float)norm;
}

__global__ __launch_bounds__(kThreads) void clip_kernel(Tensors t, ClipArgs c) {
  __shared__ double shared[kThreads / 64];
  const double norm = norm_of(c, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm) *c.norm = (float)norm;
  // the comparison keeps a NaN, as min(1, NaN) of torch's clamp does: gradients with a NaN among them all become NaN
  const double ratio = c.max_norm / (norm + 1e-6);
  const float factor = ratio > 1.0 ? 1.0f : (float)ratio;
  const int64_t last = piece_of(t, blockIdx.x + 1);
  int64_t p = piece_of(t, blockIdx.x);
  int k = tensor_of(t, p);
  while (p < last) {
    while (t.first[k + 1] <= p) ++k;
    const int64_t end = min(last, (int64_t)t.first[k + 1]), n = t.n[k];
    if (factor == 1.0f && t.out[k] == t.x[k]) {
      p = end;
      continue;
    }
    for (; p < end; ++p) {
      float v[8];
      const int64_t at = (p - t.first[k]) * kPiece + 8 * threadIdx.x;
      get(t.type[k] & 15, t.x[k], at, n, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= factor;
      void* o = t.out[k];
      const bool wide = ((uintptr_t)o & 15) == 0;
      const int type = t.type[k] >> 4;
      if (type == OR_TYPE_BF16) put8((Bf16*)o, at, n, wide, v);
      else if (type == OR_TYPE_FP16) put8((_Float16*)o, at, n, wide, v);
      else put8((float*)o, at, n, wide, v);
    }
  }
}

int check_tensors(const char* what, const or_clip_args& a) {
  if (a.n_tensors < 0) return fail_arg("%s: n_tensors < 0", what);
  if (a.n_tensors > 0 && (!a.x || !a.numel || !a.type)) return fail_arg("%s: x, numel and type are required", what);
  for (int64_t i = 0; i < a.n_tensors; ++i) {
    const int size = known_type(a.type[i]) ? type_size(a.type[i]) : 0;
    if (!size) return fail_arg("%s: unknown element type %d of tensor %lld", what, a.type[i], (long long)i);
    if (a.numel[i] < 0 || a.numel[i] > (int64_t)1 << 40) return fail_arg("%s: tensor %lld has %lld elements", what, (long long)i, (long long)a.numel[i]);
    if (a.numel[i] > 0 && (!a.x[i] || (uintptr_t)a.x[i] % size)) return fail_arg("%s: the address of tensor %lld is not that of its type", what, (long long)i);
    if (a.out) {
      const int out_type = a.out_type ? a.out_type[i] : a.type[i];
      if (!known_type(out_type)) return fail_arg("%s: unknown element type %d of output %lld", what, out_type, (long long)i);
      if (a.numel[i] > 0 && a.out[i] == a.x[i] && out_type != a.type[i]) return fail_arg("%s: output %lld is its tensor and has another type", what, (long long)i);
      if (a.numel[i] > 0 && (!a.out[i] || (uintptr_t)a.out[i] % type_size(out_type))) return fail_arg("%s: the address of output %lld is not that of its type", what, (long long)i);
    }
  }
  return 0;
}

int64_t pieces_of(int64_t n) { return (n + kPiece - 1) / kPiece; }

// Work-groups of a launch: as many as a second reader of their partial sums may cost, each with two pieces or more
int blocks_of(int64_t pieces) { return (int)std::max<int64_t>(1, std::min<int64_t>(kBlocks, (pieces + 1) / 2)); }

// the launches' tensors, one after the other; f(tensors) for each. A tensor of 2^31 pieces or more, and a launch of so many, are
// divided.
template <typename F>
int64_t each_launch(const or_clip_args& a, const F& f) {
  constexpr int64_t kMost = (int64_t)1 << 30;   // pieces of a launch
  int64_t launches = 0;
  Tensors t;
  t.count = 0;
  t.first[0] = 0;
  auto flush = [&] {
    if (!t.count) return;
    t.blocks = blocks_of(t.first[t.count]);
    f(t);
    ++launches;
    t.count = 0;
  };
  for (int64_t i = 0; i < a.n_tensors; ++i) {
    if (a.numel[i] == 0) continue;
    int64_t at = 0;
    while (at < a.numel[i]) {
      if (t.count == kTensors || (t.count && t.first[t.count] == kMost)) flush();
      const int64_t n = std::min(a.numel[i] - at, (kMost - t.first[t.count]) * kPiece);
      const int size = type_size(a.type[i]), out_type = a.out_type ? a.out_type[i] : a.type[i];
      t.x[t.count] = (const char*)a.x[i] + at * size;
      t.out[t.count] = a.out ? (char*)a.out[i] + at * type_size(out_type) : nullptr;
      t.n[t.count] = n;
      t.type[t.count] = (uint8_t)(a.type[i] | out_type << 4);
      t.first[t.count + 1] = (int32_t)(t.first[t.count] + pieces_of(n));
      ++t.count;
      at += n;
    }
  }
  flush();
  return launches;
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int64_t or_clip_workspace_size(const or_clip_args* p) {
  if (!p) return fail_arg("or_clip_workspace_size: args is NULL");
  if (int rc = check_tensors("or_clip_workspace_size", *p)) return rc;
  int64_t parts = 0;
  each_launch(*p, [&](const Tensors& t) { parts += t.blocks; });
  return parts * 8;
}

extern "C" int or_clip(const or_clip_args* p, void* stream) {
  if (!p) return fail_arg("or_clip: args is NULL");
  const or_clip_args& a = *p;
  const int64_t need = or_clip_workspace_size(p);
  if (need < 0) return (int)need;
  if (!a.norm || ((uintptr_t)a.norm & 3)) return fail_arg("or_clip: norm is required");
  if (a.out && !(a.max_norm >= 0)) return fail_arg("or_clip: max_norm must be 0 or more");
  if (need > 0 && (!a.workspace || ((uintptr_t)a.workspace & 15) || a.workspace_bytes < need))
    return fail_arg("or_clip: a 16-byte aligned workspace of %lld bytes is needed", (long long)need);
  hipStream_t st = (hipStream_t)stream;
  ClipArgs c = {};
  c.part = (double*)a.workspace;
  c.parts = need / 8;
  c.norm = a.norm;
  c.max_norm = a.max_norm;
  double* part = c.part;
  each_launch(a, [&](const Tensors& t) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(t.blocks), dim3(kThreads), 0, st, t, part);
    part += t.blocks;
  });
  if (!a.out || c.parts == 0) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, c);
  } else {
    each_launch(a, [&](const Tensors& t) {
      hipLaunchKernelGGL(clip_kernel, dim3(t.blocks), dim3(kThreads), 0, st, t, c);
      c.norm = nullptr;   // the first launch has written it
    });
  }
  return check_hip(hipGetLastError(), "or_clip launch");
}
