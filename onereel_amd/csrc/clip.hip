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
//
// 1.13e9 bf16 elements in 810 tensors, clipped into others: 1355 us for three passes over 2.27 GB (5.0 TB/s, the
// rate of a copy of 1 GB here 5.15 to 5.5); scaled in place 1443, in place under the limit 511, the norm alone 448. 240 fp32 tensors of
// up to 40000 elements, in two launches of each kernel: 94 us, which is the host's checks and addresses; 7.4, 5.2, 3.9 and 4.6 us on the
// GPU.
#include <math.h>

#include <algorithm>
#include <exception>
#include <vector>

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

// Pieces [p, end) of a tensor of n elements, several at a time where they are whole: the loads of all of them first
constexpr int kAtOnce = 4;

template <typename T>
__device__ __forceinline__ double squares(const T* x, int64_t n, int64_t p, int64_t end) {
  const bool wide = ((uintptr_t)x & 15) == 0;
  double sum = 0.0;
  float v[8];
  auto add = [&] {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += (double)v[i] * (double)v[i];
  };
  const int64_t whole = wide ? min(end, n / kPiece) : 0;
  for (; p + kAtOnce <= whole; p += kAtOnce) {
    Piece<T, 8> r[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) r[k].load(x, (p + k) * kPiece + 8 * threadIdx.x);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      r[k].get(v);
      add();
    }
  }
  for (; p < end; ++p) {
    get8(x, p * kPiece + 8 * threadIdx.x, n, wide, v);
    add();
  }
  return sum;
}

__global__ __launch_bounds__(kThreads) void grad_norm_kernel(Tensors t, double* part) {
  __shared__ double shared[kThreads / 64];
  const int64_t last = piece_of(t, blockIdx.x + 1);
  int64_t p = piece_of(t, blockIdx.x);
  double sum = 0.0;
  for (int k = tensor_of(t, p); p < last; ++k) {
    const int64_t at = t.first[k], end = min(last, (int64_t)t.first[k + 1]), n = t.n[k];
    const int type = t.type[k] & 15;
    if (type == OR_TYPE_BF16) sum += squares((const Bf16*)t.x[k], n, p - at, end - at);
    else if (type == OR_TYPE_FP16) sum += squares((const _Float16*)t.x[k], n, p - at, end - at);
    else sum += squares((const float*)t.x[k], n, p - at, end - at);
    p = end;
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

// Pieces [first, p) of a tensor, from the last one down
template <typename T, typename O>
__device__ __forceinline__ void scale(const T* x, O* out, int64_t n, int64_t first, int64_t p, float factor) {
  const bool wide = ((uintptr_t)x & 15) == 0, wide_out = ((uintptr_t)out & 15) == 0;
  float v[8];
  auto one = [&](int64_t q) {
    const int64_t at = q * kPiece + 8 * threadIdx.x;
    get8(x, at, n, wide, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= factor;
    put8(out, at, n, wide_out, v);
  };
  const int64_t whole = wide && wide_out ? n / kPiece : 0;
  for (; p > first && p > whole; --p) one(p - 1);
  for (; p - kAtOnce >= first; p -= kAtOnce) {
    Piece<T, 8> r[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) r[k].load(x, (p - 1 - k) * kPiece + 8 * threadIdx.x);
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      r[k].get(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= factor;
      Piece<O, 8>::store(out, (p - 1 - k) * kPiece + 8 * threadIdx.x, v);
    }
  }
  for (; p > first; --p) one(p - 1);
}

template <typename T>
__device__ __forceinline__ void scale_into(const T* x, void* out, int type, int64_t n, int64_t first, int64_t p, float factor) {
  if (type == OR_TYPE_BF16) scale(x, (Bf16*)out, n, first, p, factor);
  else if (type == OR_TYPE_FP16) scale(x, (_Float16*)out, n, first, p, factor);
  else scale(x, (float*)out, n, first, p, factor);
}

// The launches, tensors and pieces in the opposite order of the first kernel's: what that has read last is still in the last-level
// cache.
__global__ __launch_bounds__(kThreads) void clip_kernel(Tensors t, ClipArgs c) {
  __shared__ double shared[kThreads / 64];
  const double norm = norm_of(c, shared);
  if (blockIdx.x == 0 && threadIdx.x == 0 && c.norm) *c.norm = (float)norm;
  // the comparison keeps a NaN, as min(1, NaN) of torch's clamp does: gradients with a NaN among them all become NaN
  const double ratio = c.max_norm / (norm + 1e-6);
  const float factor = ratio > 1.0 ? 1.0f : (float)ratio;
  const int64_t first = piece_of(t, blockIdx.x);
  int64_t p = piece_of(t, blockIdx.x + 1);
  for (int k = tensor_of(t, p - 1); p > first; --k) {
    const int64_t at = t.first[k], begin = max(first, at), n = t.n[k];
    if (factor != 1.0f || t.out[k] != t.x[k]) {
      const int type = t.type[k] & 15, to = t.type[k] >> 4;
      if (type == OR_TYPE_BF16) scale_into((const Bf16*)t.x[k], t.out[k], to, n, begin - at, p - at, factor);
      else if (type == OR_TYPE_FP16) scale_into((const _Float16*)t.x[k], t.out[k], to, n, begin - at, p - at, factor);
      else scale_into((const float*)t.x[k], t.out[k], to, n, begin - at, p - at, factor);
    }
    p = begin;
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

// What is written shares memory neither with other such tensors nor with what is read, but for the tensor that it takes the place of.
int check_apart(const or_clip_args& a) {
  struct Span {
    uintptr_t first, last;
    bool writes;
  };
  std::vector<Span> spans;
  spans.reserve(2 * a.n_tensors);
  for (int64_t i = 0; i < a.n_tensors; ++i) {
    if (a.numel[i] == 0) continue;
    const uintptr_t x = (uintptr_t)a.x[i], o = (uintptr_t)a.out[i];
    spans.push_back({o, o + a.numel[i] * type_size(a.out_type ? a.out_type[i] : a.type[i]), true});
    if (o != x) spans.push_back({x, x + a.numel[i] * type_size(a.type[i]), false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& p, const Span& q) { return p.first < q.first; });
  uintptr_t end = 0, written = 0;
  for (const Span& s : spans) {
    if (s.first < (s.writes ? end : written)) return fail_arg("or_clip: tensors that are written must not share memory with one another or with what is read");
    end = std::max(end, s.last);
    if (s.writes) written = std::max(written, s.last);
  }
  return 0;
}

int64_t pieces_of(int64_t n) { return (n + kPiece - 1) / kPiece; }

// Work-groups of a launch: as many as a second reader of their partial sums may cost
int blocks_of(int64_t pieces) { return (int)std::min<int64_t>(kBlocks, pieces); }

// the launches' tensors. A tensor with more pieces than a launch numbers is divided.
std::vector<Tensors> launches_of(const or_clip_args& a) {
  constexpr int64_t kMost = (int64_t)1 << 30;   // pieces of a launch
  std::vector<Tensors> all;
  for (int64_t i = 0; i < a.n_tensors; ++i) {
    const int size = type_size(a.type[i]), out_type = a.out_type ? a.out_type[i] : a.type[i];
    for (int64_t at = 0; at < a.numel[i];) {
      if (all.empty() || all.back().count == kTensors || all.back().first[all.back().count] == kMost) {
        all.emplace_back();
        all.back().count = all.back().first[0] = 0;
      }
      Tensors& t = all.back();
      const int64_t n = std::min(a.numel[i] - at, (kMost - t.first[t.count]) * kPiece);
      t.x[t.count] = (const char*)a.x[i] + at * size;
      t.out[t.count] = a.out ? (char*)a.out[i] + at * type_size(out_type) : nullptr;
      t.n[t.count] = n;
      t.type[t.count] = (uint8_t)(a.type[i] | out_type << 4);
      t.first[t.count + 1] = (int32_t)(t.first[t.count] + pieces_of(n));
      ++t.count;
      t.blocks = blocks_of(t.first[t.count]);
      at += n;
    }
  }
  return all;
}

// how many partial sums there are
int64_t parts_of(const std::vector<Tensors>& launches) {
  int64_t n = 0;
  for (const Tensors& t : launches) n += t.blocks;
  return n;
}

}  // namespace
}  // namespace onereel

using namespace onereel;

extern "C" int64_t or_clip_workspace_size(const or_clip_args* p) try {
  if (!p) return fail_arg("or_clip_workspace_size: args is NULL");
  if (int rc = check_tensors("or_clip_workspace_size", *p)) return rc;
  return parts_of(launches_of(*p)) * 8;
} catch (const std::exception& e) {
  return fail_arg("or_clip_workspace_size: %s", e.what());
}

extern "C" int or_clip(const or_clip_args* p, void* stream) try {
  if (!p) return fail_arg("or_clip: args is NULL");
  const or_clip_args& a = *p;
  if (int rc = check_tensors("or_clip", a)) return rc;
  if (a.out)
    if (int rc = check_apart(a)) return rc;
  if (!a.norm || ((uintptr_t)a.norm & 3)) return fail_arg("or_clip: norm is required");
  if (a.out && !(a.max_norm >= 0)) return fail_arg("or_clip: max_norm must be 0 or more");
  const std::vector<Tensors> launches = launches_of(a);
  ClipArgs c = {};
  c.parts = parts_of(launches);
  if (c.parts > 0 && (!a.workspace || ((uintptr_t)a.workspace & 15) || a.workspace_bytes < c.parts * 8))
    return fail_arg("or_clip: a 16-byte aligned workspace of %lld bytes is needed", (long long)c.parts * 8);
  c.part = (double*)a.workspace;
  c.norm = a.norm;
  c.max_norm = a.max_norm;
  hipStream_t st = (hipStream_t)stream;
  double* part = c.part;
  for (const Tensors& t : launches) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(t.blocks), dim3(kThreads), 0, st, t, part);
    part += t.blocks;
  }
  if (!a.out || launches.empty()) {
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, st, c);
  } else {
    for (auto t = launches.rbegin(); t != launches.rend(); ++t) {
      hipLaunchKernelGGL(clip_kernel, dim3(t->blocks), dim3(kThreads), 0, st, *t, c);
      c.norm = nullptr;   // the first launch writes it
    }
  }
  return check_hip(hipGetLastError(), "or_clip launch");
} catch (const std::exception& e) {
  return fail_arg("or_clip: %s", e.what());
}
