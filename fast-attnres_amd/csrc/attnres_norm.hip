// attnres_norm.hip - layer norm, forward and backward, for gfx950.
//
// A row x of width D:  m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps),
// h = (x - m) r, out = h w + b.  With g = dO w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum_rows dO h,  db = sum_rows dO.
//
// Memory bound: the forward reads x and writes out, the backward reads x and dO
// and writes dx, with about one FP32 operation per byte.  A row stays in the
// registers of its lanes between its sums and its output, so each is read once.
// Statistics are FP32, the variance a second sum over the centred row in
// registers (no difference of squares).

#include "attnres_layers.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

constexpr int kNormBlocks = 512;  // most workgroups of the backward: two per CU; each writes one partial row
                                  // of dw and of db

// Sum over the lanes of a row: a part of a wavefront, or a whole workgroup of
// WAVES wavefronts per row (`scratch` holds one value per wavefront).
template <int LANES>
__device__ __forceinline__ float row_sum(float x, float* scratch) {
  if constexpr (LANES <= 64) {
    return group_sum<LANES>(x);
  } else {
    constexpr int kWaves = LANES / 64;
    const float wave = group_sum<64>(x);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x / 64] = wave;
    __syncthreads();
    const int first = threadIdx.x / LANES * kWaves;
    float total = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) total += scratch[first + k];
    return total;
  }
}

template <int LANES, int CH, class X, class P>
__global__ void __launch_bounds__(kBlock) attnres_norm_fwd_kernel(const X* __restrict__ x, int64_t x_stride, int64_t rows, int width,
                                                                  const P* __restrict__ weight, const P* __restrict__ bias,
                                                                  float eps, X* __restrict__ out, float* __restrict__ stats) {
  __shared__ float scratch[2][kBlock / 64];
  const int lane = threadIdx.x % LANES;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kBlock / LANES) + threadIdx.x / LANES;
  if (LANES <= 64 && row >= rows) return;  // a whole-workgroup row always exists
  const X* from = x + row * x_stride;
  float v[CH][kVec];
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) load_chunk(from, (k * LANES + lane) * kVec, width, v[k]);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += v[k][e];
  }
  const float mean = row_sum<LANES>(sum, scratch[0]) / static_cast<float>(width);
  float square = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float c = (k * LANES + lane) * kVec + e < width ? v[k][e] - mean : 0.0f;
      v[k][e] = c;
      square += c * c;
    }
  }
  const float rstd = 1.0f / sqrtf(row_sum<LANES>(square, scratch[1]) / static_cast<float>(width) + eps);
  if (stats != nullptr && lane == 0) {
    stats[row] = mean;
    stats[rows + row] = rstd;
  }
  X* to = out + row * width;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c = (k * LANES + lane) * kVec;
    if (c >= width) break;
    float w[kVec], b[kVec];
    if (weight != nullptr) load_chunk(weight, c, width, w);
    if (bias != nullptr) load_chunk(bias, c, width, b);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      float y = v[k][e] * rstd;
      if (weight != nullptr) y *= w[e];
      if (bias != nullptr) y += b[e];
      v[k][e] = y;
    }
    store_chunk(to, c, width, v[k]);
  }
}

// The backward: each group of lanes walks over rows, adding up dw and db of its
// own columns in registers; the groups of a workgroup meet in LDS once, at the end,
// and the workgroup writes one partial row of each.
constexpr int kBwdBlock = 512;

template <int LANES, int CH, class X, class P, bool PARAMS>
__global__ void __launch_bounds__(kBwdBlock) attnres_norm_bwd_kernel(
    const X* __restrict__ grad_out, const X* __restrict__ x, int64_t x_stride, int64_t rows, int width,
    const P* __restrict__ weight, const float* __restrict__ stats, X* __restrict__ grad_x, float* __restrict__ partial) {
  constexpr int kGroups = kBwdBlock / LANES;
  __shared__ float scratch[2][2][kBwdBlock / 64];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  float w[CH][kVec], dw[CH][kVec], db[CH][kVec];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (weight != nullptr) load_chunk(weight, (k * LANES + lane) * kVec, width, w[k]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if (weight == nullptr) w[k][e] = 1.0f;
      dw[k][e] = db[k][e] = 0.0f;
    }
  }
  const float inv = 1.0f / static_cast<float>(width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int parity = 0;
  // the same number of trips in every group of the workgroup: row_sum may hold a barrier
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups; base < rows; base += step, parity ^= 1) {
    const int64_t row = base + group;
    const bool live = row < rows;
    const int64_t at = live ? row : rows - 1;
    const float mean = stats[at], rstd = stats[rows + at];
    float h[CH][kVec], g[CH][kVec];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * LANES + lane) * kVec;
      load_chunk(x + at * x_stride, c, width, h[k]);
      load_chunk(grad_out + at * width, c, width, g[k]);
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        h[k][e] = (h[k][e] - mean) * rstd;
        if constexpr (PARAMS) {
          dw[k][e] += live ? g[k][e] * h[k][e] : 0.0f;
          db[k][e] += live ? g[k][e] : 0.0f;
        }
        g[k][e] *= w[k][e];
        s1 += g[k][e];
        s2 += g[k][e] * h[k][e];
      }
    }
    if (grad_x == nullptr) continue;  // the same for every thread
    s1 = row_sum<LANES>(s1, scratch[parity][0]) * inv;
    s2 = row_sum<LANES>(s2, scratch[parity][1]) * inv;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * LANES + lane) * kVec;
      if (c >= width) break;
      float d[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) d[e] = rstd * (g[k][e] - s1 - h[k][e] * s2);
      store_chunk(grad_x + row * width, c, width, d);
    }
  }
  if constexpr (PARAMS) {
    __shared__ float part[kGroups][LANES * kVec];
    for (int which = 0; which < 2; ++which) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kVec; ++e) part[group][lane * kVec + e] = which == 0 ? dw[k][e] : db[k][e];
        __syncthreads();
        for (int c = threadIdx.x; c < LANES * kVec; c += kBwdBlock) {
          float total = 0.0f;
          for (int j = 0; j < kGroups; ++j) total += part[j][c];
          const int col = k * LANES * kVec + c;
          if (col < width) partial[(static_cast<int64_t>(blockIdx.x) * 2 + which) * width + col] = total;
        }
      }
    }
  }
}

// Column sums of the partial rows [blocks][2][width]: workgroups of 32 columns
// by 32 row groups, each adding every 32nd row in order, then the groups in order.
constexpr int kSumCols = 32, kSumGroups = 32;

template <class P>
__global__ void __launch_bounds__(kSumCols* kSumGroups) attnres_norm_sum_kernel(const float* __restrict__ partial, int blocks, int width,
                                                                               P* __restrict__ grad_weight, P* __restrict__ grad_bias) {
  __shared__ float sums[kSumGroups][kSumCols];
  const int c = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
  const int col = blockIdx.x * kSumCols + c;  // of 2 * width: dw, then db
  const int at = col < 2 * width ? col : 2 * width - 1;
  float total = 0.0f;
#pragma unroll 8
  for (int r = g; r < blocks; r += kSumGroups) total += partial[static_cast<int64_t>(r) * 2 * width + at];
  sums[g][c] = total;
  __syncthreads();
  if (g != 0 || col >= 2 * width) return;
  total = 0.0f;
#pragma unroll
  for (int j = 0; j < kSumGroups; ++j) total += sums[j][c];
  P* to = col < width ? grad_weight : grad_bias;
  if (to != nullptr) to[col < width ? col : col - width] = from_f32<P>(total);
}

// Rows of up to 128 elements take 16 lanes, up to 4096 (forward) or 1024 (backward)
// a wavefront, wider ones a workgroup part of 256 lanes.
template <int LANES, int CH, class X, class P>
void launch_fwd(const X* x, int64_t x_stride, int64_t rows, int width, const P* weight, const P* bias, float eps, X* out,
                float* stats, hipStream_t stream) {
  constexpr int kRows = kBlock / LANES;
  const dim3 grid(static_cast<unsigned>((rows + kRows - 1) / kRows));
  hipLaunchKernelGGL((attnres_norm_fwd_kernel<LANES, CH, X, P>), grid, dim3(kBlock), 0, stream, x, x_stride, rows, width,
                     weight, bias, eps, out, stats);
}

template <class X, class P>
void norm_forward(const void* x, int64_t x_stride, int64_t rows, int width, const void* weight, const void* bias, float eps,
                  void* out, float* stats, hipStream_t stream) {
  const auto call = [&](auto launch) {
    launch(static_cast<const X*>(x), x_stride, rows, width, static_cast<const P*>(weight), static_cast<const P*>(bias), eps,
           static_cast<X*>(out), stats, stream);
  };
  if (width <= 128) return call(launch_fwd<16, 1, X, P>);
  if (width <= 512) return call(launch_fwd<64, 1, X, P>);
  if (width <= 1024) return call(launch_fwd<64, 2, X, P>);
  if (width <= 2048) return call(launch_fwd<64, 4, X, P>);
  if (width <= 4096) return call(launch_fwd<64, 8, X, P>);
  return call(launch_fwd<256, 4, X, P>);
}

int64_t bwd_blocks(int64_t rows, int64_t width) {
  const int groups = kBwdBlock / (width <= 128 ? 16 : width <= 1024 ? 64 : 256);
  return std::min<int64_t>((rows + groups - 1) / groups, kNormBlocks);
}

template <int LANES, int CH, class X, class P>
void launch_bwd(const X* grad_out, const X* x, int64_t x_stride, int64_t rows, int width, const P* weight, const float* stats,
                X* grad_x, float* partial, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(bwd_blocks(rows, width)));
  if (partial != nullptr) {
    hipLaunchKernelGGL((attnres_norm_bwd_kernel<LANES, CH, X, P, true>), grid, dim3(kBwdBlock), 0, stream, grad_out, x,
                       x_stride, rows, width, weight, stats, grad_x, partial);
  } else {
    hipLaunchKernelGGL((attnres_norm_bwd_kernel<LANES, CH, X, P, false>), grid, dim3(kBwdBlock), 0, stream, grad_out, x,
                       x_stride, rows, width, weight, stats, grad_x, partial);
  }
}

template <class X, class P>
void norm_backward(const void* grad_out, const void* x, int64_t x_stride, int64_t rows, int width, const void* weight,
                   const float* stats, void* grad_x, void* grad_weight, void* grad_bias, float* partial, hipStream_t stream) {
  if (rows > 0) {
    const auto call = [&](auto launch) {
      launch(static_cast<const X*>(grad_out), static_cast<const X*>(x), x_stride, rows, width, static_cast<const P*>(weight),
             stats, static_cast<X*>(grad_x), partial, stream);
    };
    if (width <= 128) call(launch_bwd<16, 1, X, P>);
    else if (width <= 512) call(launch_bwd<64, 1, X, P>);
    else if (width <= 1024) call(launch_bwd<64, 2, X, P>);
    else if (width <= 2048) call(launch_bwd<256, 1, X, P>);
    else if (width <= 4096) call(launch_bwd<256, 2, X, P>);
    else if (width <= 6144) call(launch_bwd<256, 3, X, P>);
    else call(launch_bwd<256, 4, X, P>);
  }
  if (grad_weight != nullptr || grad_bias != nullptr) {  // zeros when there are no rows
    const dim3 grid(static_cast<unsigned>((2 * width + kSumCols - 1) / kSumCols));
    hipLaunchKernelGGL((attnres_norm_sum_kernel<P>), grid, dim3(kSumCols * kSumGroups), 0, stream, partial,
                       static_cast<int>(rows > 0 ? bwd_blocks(rows, width) : 0), width, static_cast<P*>(grad_weight),
                       static_cast<P*>(grad_bias));
  }
}

constexpr int64_t kMaxRows = int64_t{1} << 31;  // of a launch's grid

int check_norm(int64_t rows, int64_t width, int64_t x_stride, int dtype, int param_dtype) {
  if (rows < 0 || rows > kMaxRows) return layer_error(ATTNRES_ERR_SHAPE, "rows=%lld outside 0..2^31", (long long)rows);
  if (width < 1 || width > ATTNRES_MAX_WIDTH) {
    return layer_error(ATTNRES_ERR_SHAPE, "width=%lld outside 1..%d", (long long)width, ATTNRES_MAX_WIDTH);
  }
  if (x_stride < 0) return layer_error(ATTNRES_ERR_STRIDE, "x_stride=%lld is negative", (long long)x_stride);
  if (!dtype_known(dtype)) return layer_error(ATTNRES_ERR_SHAPE, "unknown dtype %d", dtype);
  if (param_dtype != dtype && param_dtype != ATTNRES_F32) {
    return layer_error(ATTNRES_ERR_SHAPE, "weight and bias must have the rows' dtype or FP32");
  }
  return ATTNRES_OK;
}

template <class F>
void with_types(int dtype, int param_dtype, F f) {
  if (dtype == ATTNRES_F32) return f(float{}, float{});
  if (dtype == ATTNRES_BF16) return param_dtype == ATTNRES_F32 ? f(Bf16{}, float{}) : f(Bf16{}, Bf16{});
  return param_dtype == ATTNRES_F32 ? f(F16{}, float{}) : f(F16{}, F16{});
}

}  // namespace
}  // namespace layers
}  // namespace attnres_hip

using namespace attnres_hip;
using namespace attnres_hip::layers;

extern "C" {

int attnres_hip_layer_norm_forward(const void* x, int64_t x_stride, int64_t rows, int64_t width, int dtype,
                                   const void* weight, const void* bias, int param_dtype, float eps, void* out,
                                   float* stats, void* stream) {
  if (const int status = check_norm(rows, width, x_stride, dtype, param_dtype)) return status;
  if (!(eps >= 0.0f) || eps > 3.0e38f) return layer_error(ATTNRES_ERR_SCALAR, "eps must be finite and not negative");
  if (rows == 0) return ATTNRES_OK;
  if (x == nullptr || out == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "x or out is NULL");
  with_types(dtype, param_dtype, [&](auto xt, auto pt) {
    norm_forward<decltype(xt), decltype(pt)>(x, x_stride, rows, static_cast<int>(width), weight, bias, eps, out, stats,
                                             static_cast<hipStream_t>(stream));
  });
  return layer_launch_status("layer norm forward");
}

int64_t attnres_hip_layer_norm_workspace_elems(int64_t rows, int64_t width) {
  if (rows < 0 || rows > kMaxRows || width < 1 || width > ATTNRES_MAX_WIDTH) return -1;
  return bwd_blocks(rows, width) * 2 * width;
}

int attnres_hip_layer_norm_backward(const void* grad_out, const void* x, int64_t x_stride, int64_t rows, int64_t width,
                                    int dtype, const void* weight, int param_dtype, const float* stats, void* grad_x,
                                    void* grad_weight, void* grad_bias, float* workspace, int64_t workspace_elems,
                                    void* stream) {
  if (const int status = check_norm(rows, width, x_stride, dtype, param_dtype)) return status;
  const bool params = grad_weight != nullptr || grad_bias != nullptr;
  if (rows > 0 && (grad_out == nullptr || x == nullptr || stats == nullptr)) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "grad_out, x or stats is NULL");
  }
  const int64_t need = attnres_hip_layer_norm_workspace_elems(rows, width);
  if (params && rows > 0 && (workspace == nullptr || workspace_elems < need)) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "workspace of %lld elements, %lld needed", (long long)workspace_elems,
                       (long long)need);
  }
  if (!params && (grad_x == nullptr || rows == 0)) return ATTNRES_OK;
  with_types(dtype, param_dtype, [&](auto xt, auto pt) {
    norm_backward<decltype(xt), decltype(pt)>(grad_out, x, x_stride, rows, static_cast<int>(width), weight, stats, grad_x,
                                              grad_weight, grad_bias, params ? workspace : nullptr,
                                              static_cast<hipStream_t>(stream));
  });
  return layer_launch_status("layer norm backward");
}

}  // extern "C"
