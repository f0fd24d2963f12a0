// attnres_adamw.hip - an AdamW step over many tensors, for gfx950.
//
//   g = grad * scale,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: FP32 weights and states 28 bytes per element (w, m and v read and written, g read), 8-bit states 16.06.
// A launch takes up to kTensors tensors, whose addresses are kernel arguments, so a step needs no table on the
// device and can be captured; its workgroups find their tensor by a ballot over the tensors' first workgroups.
// A wavefront takes up to 4 times 256 elements, 4 per lane and access, and has all its loads under way
// before it uses the first.  Steps that are larger than the caches go past them in both directions.
// Measured, 377 M elements: FP32 1.74 ms (6.1 TB/s; through the caches 1.97), with 8-bit states 0.98 ms (6.2 TB/s; 1.15), BF16 with
// masters 1.77 ms (6.4 TB/s; 1.96).  torch's copy of 4 GiB reaches 4.8 TB/s on this card.
//
// 8-bit states: the 256 elements of a wavefront's turn are a block with a scale of its own, so a block's largest magnitude
// is a maximum over the wavefront's registers.  Numbers are E4M3 relative to it: 3 bits of mantissa down to
// 2^-15 of it, and the least at 2^-18.  v is held by its root, which has half the exponents to span, and a root above
// zero is never rounded to zero, since the update divides by it.

#include "attnres_layers.h"
#include "attnres_optim_hip.h"

#include <algorithm>
#include <cmath>

namespace attnres_hip {
namespace layers {
namespace {

constexpr int kTensors = 56;  // of a launch: their table stays within the 4 KB of kernel arguments
constexpr int kLane = 4;      // elements per lane and turn
constexpr int kTurn = 64 * kLane;
constexpr int kTurns = 4;     // of a wavefront, or 1 where that leaves compute units without work
constexpr int64_t kFewElements = int64_t{256} * 4096;  // 26 tensors, 0.6 M elements: 4.7 us; 4 turns, factors formed on the device: 7.3
constexpr int64_t kMaxChunks = int64_t{1} << 23;        // of a launch, which takes fewer than 2^32 threads
constexpr float kLargest = 448.0f;                      // of E4M3, and its least number above zero
constexpr float kLeast = 0.001953125f;
constexpr float kLeastScale = 1.17549435e-38f;          // smaller scales' reciprocals leave FP32: the block is zero
static_assert(kTurn == ATTNRES_ADAMW_BLOCK, "a turn is a block");
static_assert(kTensors <= 64, "a tensor per lane");

struct Factors {
  float decay;  // 1 - lr weight_decay
  float rate;   // lr / (1 - beta1^t)
  float unbias; // 1 / sqrt(1 - beta2^t)
};

struct StepArgs {
  attnres_adamw_tensor tensor[kTensors];
  uint32_t first[kTensors];  // workgroup of each; past the last: none
  const float* lr_device;
  const int64_t* step_device;
  const float* grad_scale;
  double lr, beta1, beta2, weight_decay;
  int64_t step;
  Factors factors;  // where neither is on the device
  float keep1, add1, keep2, add2, eps;
};

constexpr int64_t chunk_of(int turns) { return int64_t{turns} * kTurn * (kBlock / 64); }  // elements of a workgroup

__host__ __device__ inline double integer_power(double x, int64_t n) {
  double result = 1.0;
  for (; n > 0; n >>= 1) {
    if (n & 1) result *= x;
    x *= x;
  }
  return result;
}

__host__ __device__ inline Factors factors_of(const StepArgs& g, double lr, int64_t step) {
  return {static_cast<float>(1.0 - lr * g.weight_decay), static_cast<float>(lr / (1.0 - integer_power(g.beta1, step))),
          static_cast<float>(1.0 / sqrt(1.0 - integer_power(g.beta2, step)))};
}

// Four elements as they lie, at element alignment.
template <int BYTES>
struct Words;
template <>
struct Words<4> { using Type = f32x4; };
template <>
struct Words<2> { using Type = uint64_t; };
template <>
struct Words<1> { using Type = uint32_t; };
template <int BYTES>
struct __attribute__((packed, aligned(BYTES))) RawWords { typename Words<BYTES>::Type v; };

struct E4m3 { uint8_t bits; };

template <class T, bool PAST>
struct Four {
  typename Words<sizeof(T)>::Type w;
  // `left` elements count; the others read as zeros and are not written.
  __device__ __forceinline__ void load(const T* from, int64_t left) {
    if (left >= kLane) {
      const auto* words = reinterpret_cast<const RawWords<sizeof(T)>*>(from);
      w = PAST ? __builtin_nontemporal_load(&words->v) : words->v;
    } else {
      T x[kLane] = {};
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        if (e < left) x[e] = from[e];
      }
      __builtin_memcpy(&w, x, sizeof(w));
    }
  }
  __device__ __forceinline__ void store(T* to, int64_t left) const {
    if (left >= kLane) {
      auto* words = reinterpret_cast<RawWords<sizeof(T)>*>(to);
      if (PAST) {
        __builtin_nontemporal_store(w, &words->v);
      } else {
        words->v = w;
      }
    } else {
      T x[kLane];
      __builtin_memcpy(x, &w, sizeof(w));
#pragma unroll
      for (int e = 0; e < kLane; ++e) {
        if (e < left) to[e] = x[e];
      }
    }
  }
  __device__ __forceinline__ f32x4 values() const {
    if constexpr (std::is_same_v<T, float>) {
      return w;
    } else if constexpr (std::is_same_v<T, E4m3>) {
      const int bits = static_cast<int>(w);
      return f32x4{__builtin_amdgcn_cvt_f32_fp8(bits, 0), __builtin_amdgcn_cvt_f32_fp8(bits, 1), __builtin_amdgcn_cvt_f32_fp8(bits, 2),
                   __builtin_amdgcn_cvt_f32_fp8(bits, 3)};
    } else {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < kLane; ++e) x[e] = to_f32(T{static_cast<uint16_t>(w >> (16 * e))});
      return x;
    }
  }
  __device__ __forceinline__ void set(f32x4 x) {
    if constexpr (std::is_same_v<T, float>) {
      w = x;
    } else if constexpr (std::is_same_v<T, E4m3>) {
      const int low = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
      w = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], low, true));
    } else {
      w = static_cast<uint64_t>(pack2<T>(x[2], x[3])) << 32 | pack2<T>(x[0], x[1]);
    }
  }
};

// The largest magnitude of a wavefront's values; NaN where one of them is.
__device__ __forceinline__ float largest_magnitude(f32x4 x) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < kLane; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
  const auto step = [&](float other) { top = max(top, __float_as_uint(other)); };
  step(dpp<0xb1>(__uint_as_float(top)));
  step(dpp<0x4e>(__uint_as_float(top)));
  step(dpp<0x141>(__uint_as_float(top)));
  step(dpp<0x140>(__uint_as_float(top)));
  uint32_t all = 0;
#pragma unroll
  for (int row = 0; row < 4; ++row) all = max(all, __float_as_uint(lane_value(__uint_as_float(top), row * 16)));
  return __uint_as_float(all);
}

// Values to E4M3 numbers and their scale.
template <bool ROOT, bool PAST>
__device__ __forceinline__ float to_numbers(f32x4 x, Four<E4m3, PAST>* numbers) {
  float scale = largest_magnitude(x) * (1.0f / kLargest);
  if (scale < kLeastScale) scale = 0.0f;
  if (!(scale < __builtin_inff())) scale = __builtin_nanf("");  // the whole block
  const float by = scale > 0.0f ? 1.0f / scale : 0.0f;
  f32x4 number = x * by;
  if (ROOT) {
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      if (x[e] > 0.0f && number[e] < kLeast) number[e] = kLeast;
    }
  }
  numbers->set(number);
  return scale;
}

struct Moments {
  float m, v;
};

// Every operation rounded by itself: the numbers that a state is rounded to then do not depend on how a compiler joins operations,
// and any FP32 arithmetic in this order finds the same ones.
__device__ __forceinline__ Moments next_moments(float m, float v, float d, float keep1, float add1, float keep2, float add2) {
#pragma clang fp contract(off)
  return {keep1 * m + add1 * d, keep2 * v + add2 * d * d};
}

// PAST: past the caches.
template <class P, class G, int BITS, int TURNS, bool PAST>
__global__ void __launch_bounds__(kBlock) attnres_adamw_kernel(StepArgs g) {
  using S = std::conditional_t<BITS == 8, E4m3, float>;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
  const uint64_t before = __ballot(lane < kTensors && g.first[min(lane, kTensors - 1)] <= blockIdx.x);
  const int which = __builtin_amdgcn_readfirstlane(__popcll(before) - 1);
  const attnres_adamw_tensor t = g.tensor[which];
  const int64_t at0 = static_cast<int64_t>(blockIdx.x - g.first[which]) * chunk_of(TURNS) + wave * (TURNS * kTurn);
  if (at0 >= t.elements) return;
  P* param = static_cast<P*>(t.param);
  const G* grad = static_cast<const G*>(t.grad);
  S* exp_avg = static_cast<S*>(t.exp_avg);
  S* exp_avg_sq = static_cast<S*>(t.exp_avg_sq);
  const bool has_master = !std::is_same_v<P, float> && t.master != nullptr;
  Four<P, PAST> p[TURNS];
  Four<float, PAST> master[TURNS];
  Four<G, PAST> gradient[TURNS];
  Four<S, PAST> mean[TURNS], square[TURNS];
  float mean_scale[TURNS], square_scale[TURNS];
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int64_t at = at0 + k * kTurn + lane * kLane, left = t.elements - at;
    gradient[k].load(grad + at, left);
    mean[k].load(exp_avg + at, left);
    square[k].load(exp_avg_sq + at, left);
    if (has_master) master[k].load(t.master + at, left);
    else p[k].load(param + at, left);
    if constexpr (BITS == 8) {
      const int64_t block = at0 / kTurn + k;
      const bool any = block * kTurn < t.elements;
      mean_scale[k] = any ? t.exp_avg_scale[block] : 0.0f;
      square_scale[k] = any ? t.exp_avg_sq_scale[block] : 0.0f;
    }
  }
  Factors f = g.factors;
  if (g.lr_device != nullptr || g.step_device != nullptr) {
    f = factors_of(g, g.lr_device != nullptr ? static_cast<double>(*g.lr_device) : g.lr, g.step_device != nullptr ? *g.step_device : g.step);
  }
  const float by = g.grad_scale != nullptr ? *g.grad_scale : 1.0f;
#pragma unroll
  for (int k = 0; k < TURNS; ++k) {
    const int64_t at = at0 + k * kTurn + lane * kLane, left = t.elements - at;
    const f32x4 d = gradient[k].values() * by;
    f32x4 m = mean[k].values(), v = square[k].values(), w = has_master ? master[k].values() : p[k].values();
    if constexpr (BITS == 8) {
      m *= mean_scale[k];
      v *= square_scale[k];
      v *= v;
    }
    f32x4 root;
#pragma unroll
    for (int e = 0; e < kLane; ++e) {
      const Moments next = next_moments(m[e], v[e], d[e], g.keep1, g.add1, g.keep2, g.add2);
      m[e] = next.m;
      v[e] = next.v;
      root[e] = sqrtf(v[e]);
      w[e] = f.decay * w[e] - f.rate * (m[e] / (root[e] * f.unbias + g.eps));
    }
    if (has_master) {
      master[k].set(w);
      master[k].store(t.master + at, left);
    }
    p[k].set(w);
    p[k].store(param + at, left);
    if constexpr (BITS == 8) {
      // elements past the end are zeros and stay so
      const float scale = to_numbers<false>(m, &mean[k]), root_scale = to_numbers<true>(root, &square[k]);
      const int64_t block = at0 / kTurn + k;
      if (lane == 0 && block * kTurn < t.elements) {
        t.exp_avg_scale[block] = scale;
        t.exp_avg_sq_scale[block] = root_scale;
      }
    } else {
      mean[k].set(m);
      square[k].set(v);
    }
    mean[k].store(exp_avg + at, left);
    square[k].store(exp_avg_sq + at, left);
  }
}

// ---------------------------------------------------------------------- host

struct Kind {
  int param_dtype, grad_dtype, bits, turns;
  bool past;
};

template <class P, class G, int BITS>
void launch_step(const StepArgs& g, const Kind& kind, uint32_t chunks, hipStream_t stream) {
  const auto kernel = kind.turns == 1 ? attnres_adamw_kernel<P, G, BITS, 1, false>
                      : kind.past     ? attnres_adamw_kernel<P, G, BITS, kTurns, true>
                                      : attnres_adamw_kernel<P, G, BITS, kTurns, false>;
  hipLaunchKernelGGL(kernel, dim3(chunks), dim3(kBlock), 0, stream, g);
}

template <class P, class G>
void launch_step(const StepArgs& g, const Kind& kind, uint32_t chunks, hipStream_t stream) {
  return kind.bits == 8 ? launch_step<P, G, 8>(g, kind, chunks, stream) : launch_step<P, G, 32>(g, kind, chunks, stream);
}

void launch_step(const StepArgs& g, const Kind& kind, uint32_t chunks, hipStream_t stream) {
  const bool wide = kind.grad_dtype == ATTNRES_F32;
  if (kind.param_dtype == ATTNRES_F32) return launch_step<float, float>(g, kind, chunks, stream);
  if (kind.param_dtype == ATTNRES_BF16) {
    return wide ? launch_step<Bf16, float>(g, kind, chunks, stream) : launch_step<Bf16, Bf16>(g, kind, chunks, stream);
  }
  return wide ? launch_step<F16, float>(g, kind, chunks, stream) : launch_step<F16, F16>(g, kind, chunks, stream);
}

bool aligned(const void* p, int64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int check_tensor(const attnres_adamw_tensor& t, int64_t index, int param_dtype, int grad_dtype, int bits) {
  const long long i = index;
  if (t.elements < 0) return layer_error(ATTNRES_ERR_SHAPE, "tensor %lld: %lld elements", i, (long long)t.elements);
  if (t.elements == 0) return ATTNRES_OK;
  if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "tensor %lld: param, grad, exp_avg or exp_avg_sq is NULL", i);
  }
  if (bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr)) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "tensor %lld: 8-bit states need their scales", i);
  }
  if (t.master != nullptr && param_dtype == ATTNRES_F32) {
    return layer_error(ATTNRES_ERR_SHAPE, "tensor %lld: FP32 parameters have no masters", i);
  }
  const int64_t state = bits == 8 ? 1 : 4;
  if (!aligned(t.param, dtype_size(param_dtype)) || !aligned(t.grad, dtype_size(grad_dtype)) || !aligned(t.exp_avg, state) ||
      !aligned(t.exp_avg_sq, state) || !aligned(t.exp_avg_scale, 4) || !aligned(t.exp_avg_sq_scale, 4) || !aligned(t.master, 4)) {
    return layer_error(ATTNRES_ERR_STRIDE, "tensor %lld: not at its type's alignment", i);
  }
  return ATTNRES_OK;
}

}  // namespace
}  // namespace layers
}  // namespace attnres_hip

using namespace attnres_hip;
using namespace attnres_hip::layers;

extern "C" {

int attnres_hip_adamw(const attnres_adamw_tensor* tensors, int64_t count, int param_dtype, int grad_dtype, int state_bits, double lr,
                      const float* lr_device, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                      const int64_t* step_device, const float* grad_scale, void* stream) {
  if (count < 0) return layer_error(ATTNRES_ERR_SHAPE, "%lld tensors", (long long)count);
  if (!dtype_known(param_dtype)) return layer_error(ATTNRES_ERR_SHAPE, "unknown dtype %d", param_dtype);
  if (grad_dtype != param_dtype && grad_dtype != ATTNRES_F32) {
    return layer_error(ATTNRES_ERR_SHAPE, "gradients of dtype %d for parameters of %d", grad_dtype, param_dtype);
  }
  if (state_bits != 8 && state_bits != 32) return layer_error(ATTNRES_ERR_SCALAR, "states of %d bits: 8 or 32 are known", state_bits);
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return layer_error(ATTNRES_ERR_SCALAR, "betas outside [0, 1)");
  if (!(eps >= 0.0 && std::isfinite(eps) && weight_decay >= 0.0 && std::isfinite(weight_decay))) {
    return layer_error(ATTNRES_ERR_SCALAR, "eps and weight_decay must be finite and not negative");
  }
  if (lr_device == nullptr && !(lr >= 0.0 && std::isfinite(lr))) {
    return layer_error(ATTNRES_ERR_SCALAR, "lr must be finite and not negative");
  }
  if (step_device == nullptr && step < 1) return layer_error(ATTNRES_ERR_SCALAR, "step=%lld: steps count from 1", (long long)step);
  if (count > 0 && tensors == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "tensors is NULL");
  const int64_t param_size = dtype_size(param_dtype), grad_size = dtype_size(grad_dtype), state_size = state_bits == 8 ? 1 : 4;
  int64_t all = 0, written = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (const int status = check_tensor(tensors[i], i, param_dtype, grad_dtype, state_bits)) return status;
    all += tensors[i].elements;
    written += tensors[i].elements * (param_size + 2 * state_size + (tensors[i].master != nullptr ? 4 : 0));
  }
  const Kind kind{param_dtype, grad_dtype, state_bits, all <= kFewElements ? 1 : kTurns, written >= kPastCaches};
  const int64_t chunk = chunk_of(kind.turns);
  StepArgs g{};
  g.lr_device = lr_device;
  g.step_device = step_device;
  g.grad_scale = grad_scale;
  g.lr = lr;
  g.beta1 = beta1;
  g.beta2 = beta2;
  g.weight_decay = weight_decay;
  g.step = step;
  g.eps = static_cast<float>(eps);
  g.keep1 = static_cast<float>(beta1);
  g.add1 = static_cast<float>(1.0 - beta1);
  g.keep2 = static_cast<float>(beta2);
  g.add2 = static_cast<float>(1.0 - beta2);
  if (lr_device == nullptr && step_device == nullptr) g.factors = factors_of(g, lr, step);
  int held = 0;
  int64_t chunks = 0;
  bool launched = false;
  const auto launch = [&] {
    if (held == 0) return;
    launched = true;
    for (int k = held; k < kTensors; ++k) g.first[k] = UINT32_MAX;
    launch_step(g, kind, static_cast<uint32_t>(chunks), static_cast<hipStream_t>(stream));
    held = 0;
    chunks = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    const attnres_adamw_tensor& t = tensors[i];
    for (int64_t from = 0; from < t.elements; from += kMaxChunks * chunk) {  // a launch's share of it
      const int64_t elements = std::min(t.elements - from, kMaxChunks * chunk), need = (elements + chunk - 1) / chunk;
      if (held == kTensors || chunks + need > kMaxChunks) launch();
      const int64_t block = from / kTurn;
      g.tensor[held] = {static_cast<char*>(t.param) + from * param_size,
                        static_cast<const char*>(t.grad) + from * grad_size,
                        static_cast<char*>(t.exp_avg) + from * state_size,
                        static_cast<char*>(t.exp_avg_sq) + from * state_size,
                        t.exp_avg_scale != nullptr ? t.exp_avg_scale + block : nullptr,
                        t.exp_avg_sq_scale != nullptr ? t.exp_avg_sq_scale + block : nullptr,
                        t.master != nullptr ? t.master + from : nullptr,
                        elements};
      g.first[held++] = static_cast<uint32_t>(chunks);
      chunks += need;
    }
  }
  launch();
  return launched ? layer_launch_status("AdamW step") : ATTNRES_OK;
}

}  // extern "C"
