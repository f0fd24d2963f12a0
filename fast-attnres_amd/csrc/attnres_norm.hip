// attnres_norm.hip - layer norm, forward and backward, for gfx950.
//
// A row x of width D:  m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps),
// h = (x - m) r, out = h w + b.  With g = dO w:
//   dx = r (g - mean(g) - h mean(g h)),  dw = sum_rows dO h,  db = sum_rows dO.
//
// Memory bound: the forward reads x and writes out, the backward reads x and dO
// and writes dx, with about one FP32 operation per byte.  A row stays in the
// registers of its lanes between its sums and its output, so each is read once.  32768 x 4096 BF16: forward
// 98 us (5.5 TB/s), backward 154 us (5.2), its column sums 5.
// Statistics are FP32, the variance a second sum over the centred row in
// registers (no difference of squares).

#include "attnres_layers.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

// Workgroups of the forward and, of twice the threads, of the backward; each walks over rows, the next row's
// loads under way while one is worked on, with the weight and the bias in registers.
constexpr int kFwdBlocks = 2048;
constexpr int kNormBlocks = 512;  // each writes one partial row of dw and of db

// Mean and sum of squared deviations of a row, of which each lane holds v (zeros past the row's end).
// Within a wavefront the deviations are taken from its own mean; four wavefronts of a row join
// theirs by the distances of their means, in one exchange through LDS.  `scratch`
// alternates between calls.
template <int LANES, int CH>
__device__ __forceinline__ void row_moments(const float (&v)[CH][kVec], int lane, int width, float (*scratch)[2], float* mean,
                                            float* square) {
  constexpr int kSpan = LANES < 64 ? LANES : 64;  // lanes that add up directly
  const int first = LANES <= 64 ? 0 : __builtin_amdgcn_readfirstlane(lane / 64) * 64;  // of this wavefront
  int count = 0;  // elements of the row in these lanes
#pragma unroll
  for (int k = 0; k < CH; ++k) count += min(max(width - (k * LANES + first) * kVec, 0), kSpan * kVec);
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum += v[k][e];
  }
  const float own = count > 0 ? group_sum<kSpan>(sum) / static_cast<float>(count) : 0.0f;
  float m2 = 0.0f;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float c = v[k][e] - own;
      m2 += (k * LANES + lane) * kVec + e < width ? c * c : 0.0f;
    }
  }
  m2 = group_sum<kSpan>(m2);
  if constexpr (LANES <= 64) {
    *mean = own;
    *square = m2;
  } else {
    constexpr int kWaves = LANES / 64;
    const int base = threadIdx.x / LANES * kWaves;
    if (lane % 64 == 0) {
      scratch[base + lane / 64][0] = own;
      scratch[base + lane / 64][1] = m2;
    }
    __syncthreads();
    float counts[kWaves], all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      int c = 0;
#pragma unroll
      for (int k = 0; k < CH; ++k) c += min(max(width - (k * LANES + w * 64) * kVec, 0), 64 * kVec);
      counts[w] = static_cast<float>(c) / static_cast<float>(width);
      all += counts[w] * scratch[base + w][0];
    }
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float d = scratch[base + w][0] - all;
      total += scratch[base + w][1] + counts[w] * static_cast<float>(width) * d * d;
    }
    *mean = all;
    *square = total;
  }
}

template <int LANES, int CH, class P>
__device__ __forceinline__ void load_row(const P* row, int lane, int width, float missing, float (&x)[CH][kVec]) {
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    if (row != nullptr) {
      load_chunk(row, (k * LANES + lane) * kVec, width, x[k]);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[k][e] = missing;
    }
  }
}

template <int LANES, int CH, class X, class P, bool PAST>
__global__ void __launch_bounds__(kBlock) attnres_norm_fwd_kernel(const X* __restrict__ x, int64_t x_stride, int64_t rows, int width,
                                                                  const P* __restrict__ weight, const P* __restrict__ bias,
                                                                  float eps, X* __restrict__ out, float* __restrict__ stats) {
  constexpr int kGroups = kBlock / LANES;
  __shared__ float scratch[2][kBlock / 64][2];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups;
  // groups of more than a wavefront share row_moments' barrier: as many trips for each, the last one idle for some
  constexpr bool kShared = LANES > 64 && kGroups > 1;
  const int64_t until = kShared ? rows : rows - group;
  if (base >= until) return;
  Chunk<X> next[CH];
  const auto fetch = [&](int64_t from) {
    const int64_t at = !kShared || from + group < rows ? from + group : rows - 1;
#pragma unroll
    for (int k = 0; k < CH; ++k) next[k].load(x + at * x_stride, (k * LANES + lane) * kVec, width);
  };
  fetch(base);
  float w[CH][kVec], b[CH][kVec];
  load_row<LANES>(weight, lane, width, 1.0f, w);
  load_row<LANES>(bias, lane, width, 0.0f, b);
  for (int parity = 0; base < until; base += step, parity ^= 1) {
    const int64_t row = base + group;
    float v[CH][kVec];
#pragma unroll
    for (int k = 0; k < CH; ++k) next[k].unpack(v[k]);
    if (base + step < until) fetch(base + step);
    float mean, square;
    row_moments<LANES>(v, lane, width, scratch[parity], &mean, &square);
    const float rstd = 1.0f / sqrtf(square / static_cast<float>(width) + eps);
    if (kShared && row >= rows) continue;
    if (stats != nullptr && lane == 0) {
      stats[row] = mean;
      stats[rows + row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * LANES + lane) * kVec;
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[k][e] = (v[k][e] - mean) * rstd * w[k][e] + b[k][e];
      if (c < width) store_chunk(out + row * width, c, width, v[k], PAST);
    }
  }
}

// Sums over a row's lanes of two values; `scratch` alternates between calls.
template <int LANES>
__device__ __forceinline__ void row_sums(float& x, float& y, float (*scratch)[2]) {
  constexpr int kSpan = LANES < 64 ? LANES : 64;
  x = group_sum<kSpan>(x);
  y = group_sum<kSpan>(y);
  if constexpr (LANES > 64) {
    constexpr int kWaves = LANES / 64;
    if (threadIdx.x % 64 == 0) {
      scratch[threadIdx.x / 64][0] = x;
      scratch[threadIdx.x / 64][1] = y;
    }
    __syncthreads();
    const int first = threadIdx.x / LANES * kWaves;
    x = y = 0.0f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      x += scratch[first + k][0];
      y += scratch[first + k][1];
    }
  }
}

// The backward: each group of lanes walks over rows, adding up dw and db of its
// own columns in registers; the groups of a workgroup meet in LDS once, at the end,
// and the workgroup writes one partial row of each.  512 workgroups of 512 threads: with 768 or 1024 of them the partial
// rows cost more than the walk gains.
constexpr int kBwdBlock = 512;

template <int LANES, int CH, class X, class P, bool PARAMS, bool PAST>
__global__ void __launch_bounds__(kBwdBlock) attnres_norm_bwd_kernel(
    const X* __restrict__ grad_out, const X* __restrict__ x, int64_t x_stride, int64_t rows, int width,
    const P* __restrict__ weight, const float* __restrict__ stats, X* __restrict__ grad_x, float* __restrict__ partial) {
  constexpr int kGroups = kBwdBlock / LANES;
  __shared__ float scratch[2][kBwdBlock / 64][2];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  float w[CH][kVec], dw[CH][kVec], db[CH][kVec];
  load_row<LANES>(weight, lane, width, 1.0f, w);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) dw[k][e] = db[k][e] = 0.0f;
  }
  const float inv = 1.0f / static_cast<float>(width);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kGroups;
  int64_t base = static_cast<int64_t>(blockIdx.x) * kGroups;
  Chunk<X> next_x[CH], next_g[CH];
  float next_mean, next_rstd;
  const auto fetch = [&](int64_t from) {
    const int64_t at = from + group < rows ? from + group : rows - 1;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      next_x[k].load(x + at * x_stride, (k * LANES + lane) * kVec, width);
      next_g[k].load(grad_out + at * width, (k * LANES + lane) * kVec, width);
    }
    next_mean = stats[at];
    next_rstd = stats[rows + at];
  };
  fetch(base);
  // the same number of trips in every group of the workgroup: row_sums may hold a barrier
  for (int parity = 0; base < rows; base += step, parity ^= 1) {
    const int64_t row = base + group;
    const bool live = row < rows;
    const float mean = next_mean, rstd = next_rstd;
    float h[CH][kVec], g[CH][kVec];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      next_x[k].unpack(h[k]);
      next_g[k].unpack(g[k]);
    }
    if (base + step < rows) fetch(base + step);
    float s1 = 0.0f, s2 = 0.0f;
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
    row_sums<LANES>(s1, s2, scratch[parity]);
    s1 *= inv;
    s2 *= inv;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * LANES + lane) * kVec;
      float d[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) d[e] = rstd * (g[k][e] - s1 - h[k][e] * s2);
      if (c < width) store_chunk(grad_x + row * width, c, width, d, PAST);
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
#pragma unroll
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

// Measured with 268 MB (32768 x 4096 BF16): forward 99.5 -> 95.7 us, backward 155.9 -> 143.9.
template <class X>
bool past_caches(int64_t rows, int64_t width) {
  return rows * width * static_cast<int64_t>(sizeof(X)) >= kPastCaches;
}

// Rows of up to 128 elements take 16 lanes, up to 1024 a wavefront, wider ones 256 lanes; in the backward 512
// from 2049 elements on, as it holds dw and db beside two rows; in the forward of 16-bit rows a wavefront up to 2560 and
// two up to 4096, so that fewer lanes idle past the row's end and fewer rows wait at barriers.  Forward, BF16,
// 256 lanes -> as here, us: 32768 x 1536 42.4 -> 32.7, 65536 x 2048 111 -> 103, 32768 x 2560 85.2 -> 67.5, x
// 4096 110 -> 102; FP32 rows of twice the registers: 8192 x 2048 21.8 -> 23.4, so they keep 256 lanes.
template <int LANES, int CH, class X, class P>
void launch_fwd(const X* x, int64_t x_stride, int64_t rows, int width, const P* weight, const P* bias, float eps, X* out,
                float* stats, hipStream_t stream) {
  constexpr int kRows = kBlock / LANES;
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>((rows + kRows - 1) / kRows, kFwdBlocks)));
  const auto kernel = past_caches<X>(rows, width) ? attnres_norm_fwd_kernel<LANES, CH, X, P, true>
                                                  : attnres_norm_fwd_kernel<LANES, CH, X, P, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, stream, x, x_stride, rows, width, weight, bias, eps, out, stats);
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
  if constexpr (sizeof(X) == 2) {
    if (width <= 1536) return call(launch_fwd<64, 3, X, P>);
    if (width <= 2048) return call(launch_fwd<64, 4, X, P>);
    if (width <= 2560) return call(launch_fwd<64, 5, X, P>);
    if (width <= 4096) return call(launch_fwd<128, 4, X, P>);
  }
  if (width <= 2048) return call(launch_fwd<256, 1, X, P>);
  if (width <= 4096) return call(launch_fwd<256, 2, X, P>);
  if (width <= 6144) return call(launch_fwd<256, 3, X, P>);
  return call(launch_fwd<256, 4, X, P>);
}

int64_t bwd_blocks(int64_t rows, int64_t width) {
  const int groups = kBwdBlock / (width <= 128 ? 16 : width <= 1024 ? 64 : width <= 2048 ? 256 : 512);
  return std::min<int64_t>((rows + groups - 1) / groups, kNormBlocks);
}

template <int LANES, int CH, class X, class P>
void launch_bwd(const X* grad_out, const X* x, int64_t x_stride, int64_t rows, int width, const P* weight, const float* stats,
                X* grad_x, float* partial, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(bwd_blocks(rows, width)));
  const bool past = past_caches<X>(rows, width);
  const auto kernel = partial == nullptr ? attnres_norm_bwd_kernel<LANES, CH, X, P, false, false>
                      : past             ? attnres_norm_bwd_kernel<LANES, CH, X, P, true, true>
                                         : attnres_norm_bwd_kernel<LANES, CH, X, P, true, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kBwdBlock), 0, stream, grad_out, x, x_stride, rows, width, weight, stats, grad_x, partial);
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
    else if (width <= 4096) call(launch_bwd<512, 1, X, P>);
    else call(launch_bwd<512, 2, X, P>);
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
