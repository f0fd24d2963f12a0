// attnres_layers.h - element types, loads and sums shared by the kernels of the
// layers and of the optimizer (attnres_{norm,embedding,loss,ffn,adamw}.hip).
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
// Results from here on are stored past the caches: beside what they are made of they do not stay in the 256 MB of
// the last one anyway.
constexpr int64_t kPastCaches = int64_t{128} << 20;

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

// `past`: past the caches, for results too large to stay in them.
template <class T>
__device__ __forceinline__ void store8(T* p, const float* x, bool past = false) {
  if constexpr (std::is_same_v<T, float>) {
    const f32x4 a = {x[0], x[1], x[2], x[3]}, b = {x[4], x[5], x[6], x[7]};
    if (past) {
      __builtin_nontemporal_store(a, &reinterpret_cast<Raw32*>(p)->v);
      __builtin_nontemporal_store(b, &reinterpret_cast<Raw32*>(p + 4)->v);
    } else {
      reinterpret_cast<Raw32*>(p)->v = a;
      reinterpret_cast<Raw32*>(p + 4)->v = b;
    }
  } else {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
    if (past) {
      __builtin_nontemporal_store(w, &reinterpret_cast<Raw16*>(p)->v);
    } else {
      reinterpret_cast<Raw16*>(p)->v = w;
    }
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
__device__ __forceinline__ void store_chunk(T* row, int c, int width, const float* x, bool past = false) {
  if (c + kVec <= width) {
    store8(row + c, x, past);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (c + e < width) row[c + e] = from_f32<T>(x[e]);
    }
  }
}

// The same eight elements as they lie, for loads that are under way while others are worked on.
template <class T>
struct Chunk {
  u32x4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* row, int c, int width) {
    if (c + kVec <= width) {
#pragma unroll
      for (size_t k = 0; k < sizeof(T) / 2; ++k) w[k] = reinterpret_cast<const Raw16*>(row + c)[k].v;
    } else {
      float x[kVec];
      load_chunk(row, c, width, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (std::is_same_v<T, float>) {
          w[0][e] = __float_as_uint(x[e]);
          w[1][e] = __float_as_uint(x[4 + e]);
        } else {
          w[0][e] = pack2<T>(x[2 * e], x[2 * e + 1]);
        }
      }
    }
  }
  // Eight elements that are read once, and not from the caches.
  __device__ __forceinline__ void load_past(const T* from) {
#pragma unroll
    for (size_t k = 0; k < sizeof(T) / 2; ++k) w[k] = __builtin_nontemporal_load(&reinterpret_cast<const Raw16*>(from)[k].v);
  }
  __device__ __forceinline__ void unpack(float* x) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (std::is_same_v<T, float>) {
        x[e] = __uint_as_float(w[0][e]);
        x[4 + e] = __uint_as_float(w[1][e]);
      } else {
        x[2 * e] = to_f32(T{static_cast<uint16_t>(w[0][e] & 0xffffu)});
        x[2 * e + 1] = to_f32(T{static_cast<uint16_t>(w[0][e] >> 16)});
      }
    }
  }
};

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// Sum over groups of 16 lanes or a whole wavefront, the same bits in every lane of the
// group: quad permutations and row mirrors within 16 lanes, lane reads across them.
template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
  static_assert(LANES == 16 || LANES == 64, "a DPP row or a wavefront");
  x += dpp<0xb1>(x);   // quad_perm [1,0,3,2]
  x += dpp<0x4e>(x);   // quad_perm [2,3,0,1]
  x += dpp<0x141>(x);  // row_half_mirror
  x += dpp<0x140>(x);  // row_mirror
  if constexpr (LANES == 16) return x;
  return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

}  // namespace layers
}  // namespace attnres_hip

#endif  // ATTNRES_LAYERS_H
