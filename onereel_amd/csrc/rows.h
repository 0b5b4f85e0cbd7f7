// Rows of bf16, fp16 or fp32 elements in pieces of 8 and 4, as fp32 in registers; sums over a work-group.
#pragma once

#include "common.h"

namespace onereel {

// the element types of the row kernels (OR_TYPE_*)
struct Bf16 {
  uint16_t u;
};
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

// N (8 or 4) consecutive elements as they lie in memory; a piece of 8 lies at a 16-byte aligned address, one of 4 at an 8-byte
// aligned one
template <typename T, int N>
struct Piece;

template <>
struct Piece<Bf16, 8> {
  u32x4 r;
  __device__ __forceinline__ void load(const void* p, int64_t at) { r = *(const u32x4*)((const uint16_t*)p + at); }
  __device__ __forceinline__ void zero() { r = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf2f((uint16_t)(r[i] & 0xffffu));
      f[2 * i + 1] = bf2f((uint16_t)(r[i] >> 16));
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float (&f)[8]) {
    const u32x4 o = {pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])};
    __builtin_nontemporal_store(o, (u32x4*)((uint16_t*)p + at));
  }
};

template <>
struct Piece<Bf16, 4> {
  u32x2v r;
  __device__ __forceinline__ void load(const void* p, int64_t at) { r = *(const u32x2v*)((const uint16_t*)p + at); }
  __device__ __forceinline__ void zero() { r = u32x2v{0, 0}; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f[2 * i] = bf2f((uint16_t)(r[i] & 0xffffu));
      f[2 * i + 1] = bf2f((uint16_t)(r[i] >> 16));
    }
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float* f) {
    __builtin_nontemporal_store(u32x2v{pack2(f[0], f[1]), pack2(f[2], f[3])}, (u32x2v*)((uint16_t*)p + at));
  }
};

template <>
struct Piece<_Float16, 8> {
  half8 r;
  __device__ __forceinline__ void load(const void* p, int64_t at) { r = *(const half8*)((const _Float16*)p + at); }
  __device__ __forceinline__ void zero() { r = half8{}; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)r[i];
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float (&f)[8]) {
    half8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (_Float16)f[i];
    __builtin_nontemporal_store(o, (half8*)((_Float16*)p + at));
  }
};

template <>
struct Piece<_Float16, 4> {
  half4 r;
  __device__ __forceinline__ void load(const void* p, int64_t at) { r = *(const half4*)((const _Float16*)p + at); }
  __device__ __forceinline__ void zero() { r = half4{}; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)r[i];
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float* f) {
    half4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (_Float16)f[i];
    __builtin_nontemporal_store(o, (half4*)((_Float16*)p + at));
  }
};

template <>
struct Piece<float, 4> {
  f32x4 r;
  __device__ __forceinline__ void load(const void* p, int64_t at) { r = *(const f32x4*)((const float*)p + at); }
  __device__ __forceinline__ void zero() { r = f32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = r[i];
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float* f) {
    __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, (f32x4*)((float*)p + at));
  }
};

template <>
struct Piece<float, 8> {
  f32x4 r[2];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    r[0] = *(const f32x4*)((const float*)p + at);
    r[1] = *(const f32x4*)((const float*)p + at + 4);
  }
  __device__ __forceinline__ void zero() { r[0] = r[1] = f32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = r[i / 4][i % 4];
  }
  static __device__ __forceinline__ void store(void* p, int64_t at, const float (&f)[8]) {
    __builtin_nontemporal_store(f32x4{f[0], f[1], f[2], f[3]}, (f32x4*)((float*)p + at));
    __builtin_nontemporal_store(f32x4{f[4], f[5], f[6], f[7]}, (f32x4*)((float*)p + at + 4));
  }
};

// sum over 16 neighbouring lanes, the same in each of them
__device__ __forceinline__ float row_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));   // quad_perm 1032
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));   // quad_perm 2301
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // row_half_mirror
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, false));  // row_mirror
  return v;
}

// sums of two values over the 64 lanes of a wavefront, the same in each of them: the halves swap one for the other, so that one
// register goes through the rest for both
__device__ __forceinline__ void wave_sums(float a, float b, float& sum_a, float& sum_b) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  const float v = row_sum(__uint_as_float(p[0]) + __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float r = __uint_as_float(q[0]) + __uint_as_float(q[1]);
  sum_a = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(r), 0));
  sum_b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(r), 32));
}

inline int type_size(int type) { return type == OR_TYPE_FP32 ? 4 : 2; }
inline bool known_type(int type) { return type == OR_TYPE_BF16 || type == OR_TYPE_FP16 || type == OR_TYPE_FP32; }

}  // namespace onereel
