// attnres_layers.h - element types, loads and sums shared by the kernels of the
// layers (attnres_norm.hip, attnres_embedding.hip, attnres_loss.hip).
#ifndef ATTNRES_LAYERS_H
#define ATTNRES_LAYERS_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "attnres_layers_hip.h"

namespace attnres_hip {

// Records the calling thread's error message and returns `code` (attnres_hip.hip).
int layer_error(int code, const char* fmt, ...);
// The status of the launches just made.
int layer_launch_status(const char* what);

namespace layers {

constexpr int kBlock = 256;
constexpr int kVec = 8;  // elements per chunk

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Bf16 { uint16_t bits; };
struct F16 { uint16_t bits; };

inline int64_t dtype_size(int dtype) { return dtype == ATTNRES_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == ATTNRES_BF16 || dtype == ATTNRES_F16 || dtype == ATTNRES_F32; }

// Two FP32 values to packed 16-bit ones (low element first), to nearest even.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, Bf16>) {
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  } else {
    const f16x2 v = {static_cast<_Float16>(lo), static_cast<_Float16>(hi)};
    return __builtin_bit_cast(uint32_t, v);
  }
}

template <class T>
__device__ __forceinline__ float to_f32(T x) {
  if constexpr (std::is_same_v<T, float>) {
    return x;
  } else if constexpr (std::is_same_v<T, Bf16>) {
    return __uint_as_float(static_cast<uint32_t>(x.bits) << 16);
  } else {
    return static_cast<float>(__builtin_bit_cast(_Float16, x.bits));
  }
}

template <class T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (std::is_same_v<T, float>) {
    return x;
  } else {
    return T{static_cast<uint16_t>(pack2<T>(x, 0.0f) & 0xffffu)};
  }
}

// Eight elements at element alignment: one 16-byte access (two for FP32).
// gfx950 takes global accesses at any alignment; rows that start off a 16-byte
// boundary need no path of their own.
struct __attribute__((packed, aligned(2))) Raw16 { u32x4 v; };
struct __attribute__((packed, aligned(4))) Raw32 { f32x4 v; };

template <class T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (std::is_same_v<T, float>) {
    const f32x4 a = reinterpret_cast<const Raw32*>(p)->v, b = reinterpret_cast<const Raw32*>(p + 4)->v;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
  } else {
    const u32x4 w = reinterpret_cast<const Raw16*>(p)->v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[2 * e] = to_f32(T{static_cast<uint16_t>(w[e] & 0xffffu)});
      x[2 * e + 1] = to_f32(T{static_cast<uint16_t>(w[e] >> 16)});
    }
  }
}

template <class T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (std::is_same_v<T, float>) {
    reinterpret_cast<Raw32*>(p)->v = f32x4{x[0], x[1], x[2], x[3]};
    reinterpret_cast<Raw32*>(p + 4)->v = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    reinterpret_cast<Raw16*>(p)->v = w;
  }
}

// Elements c .. c+7 of a row of `width` elements; those past its end read as 0 and
// are not written.
template <class T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int width, float* x) {
  if (c + kVec <= width) {
    load8(row + c, x);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = c + e < width ? to_f32(row[c + e]) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void store_chunk(T* row, int c, int width, const float* x) {
  if (c + kVec <= width) {
    store8(row + c, x);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (c + e < width) row[c + e] = from_f32<T>(x[e]);
    }
  }
}

// Sum over groups of LANES lanes of a wavefront (LANES a power of two <= 64), in
// every lane of the group; the tree's order is fixed.
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int step = LANES / 2; step > 0; step >>= 1) x += __shfl_xor(x, step, 64);
  return x;
}

}  // namespace layers
}  // namespace attnres_hip

#endif  // ATTNRES_LAYERS_H
