// attnres_ffn.hip - the gated feed-forward block, forward and backward, for gfx950.
//
//   g = X Wg^T,  u = X Wu^T,  a = act(g) u,  Y = a Wd^T            (act: silu or gelu)
//   da = dY Wd,  du = da act(g),  dg = da u act'(g)
//   dWd = dY^T a,  dX = [dg du] W,  dW = [dg du]^T X,              W = [Wg; Wu]
//
// Bound by the matrix cores: 6 N D F operations forward (N rows, D wide, F hidden), 12 backward, against O(N F + D F)
// bytes.  Launches of tiles (attnres_product.h): g and u in one, a gate's and an up's entry in the same lane, so that a is
// formed from the FP32 sums; Y; da, from which dg, du and a again are formed; and dX, dW and dWd in one, or where they are large
// in one each (kTogether).  Tiles are of 256, 128 or 64 by a model of when the chip's last unit is done (choose_cut); products whose
// tiles do not fill the chip are cut along their depth, and the parts' FP32 sums added up in order.
// 16384 x 4096 x 11264, BF16: forward 3.7 ms (1.22 PFLOP/s), backward 7.9 (1.15); power sets the clock there, and the library's
// products of these sizes reach 1.40.  2048 x 1024 x 2816 in 160 us of kernels, 0.66.
//
// What goes from the forward to the backward is g and u, in the order in which a lane holds them, so both sides
// move them 16 bytes per lane with no detour over LDS: FP32 for FP32 inputs, else FP32 cut to 24 bits (2^-17).  Rounded to
// BF16, g and u would each bring an error of the size of the gradients' own rounding (0.0017, root mean square); as it is the gradients
// are off by 0.0024.  With `saved` NULL the backward forms them again, which adds a third to its products.
//
// 16-bit operands are multiplied as they are; a, dg and du are rounded to their type, dg and du of FP16 at a power of two (scale_of).  FP32 values of larger calls (kSingleRows) are written
// as the sum of three BF16 numbers, 24 bits over FP32's whole range, and a product is the six products of parts that are
// not below 2^-26 of it: FP32 matrix instructions run at a sixteenth of the BF16 rate.  Smaller calls (Single) take those, and pack nothing.

#include "attnres_product.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

constexpr int kSub = 16;              // rows and columns of a subtile of saved g and u

template <class X>
constexpr int kParts = std::is_same_v<X, float> ? 3 : 1;
template <class X>
constexpr int kSegments = std::is_same_v<X, float> ? 6 : 1;
// FP32 inputs of fewer rows, as they are, by FP32 matrix instructions.
struct Single {};
template <class X>
using Value = std::conditional_t<std::is_same_v<X, Single>, float, X>;  // of the tensors
template <class X>
constexpr bool kFp32 = std::is_same_v<Value<X>, float>;
template <class X>
using Part = std::conditional_t<std::is_same_v<X, float>, Bf16, Value<X>>;  // of the products
template <class X>
constexpr int kHalves = sizeof(Part<X>) / 2;

// ---------------------------------------------------------------- activation

// FP32 inputs: the library's exponential.  16-bit ones: the instruction's, whose argument's rounding is 2^-24 |x| relative.
template <class X>
__device__ __forceinline__ float exponential(float x) {
  if constexpr (kFp32<X>) return expf(x);
  return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
template <class X>
__device__ __forceinline__ float reciprocal(float x) {
  if constexpr (kFp32<X>) return 1.0f / x;
  return __builtin_amdgcn_rcpf(x);
}

struct Activated {
  float value, slope;
};

// gelu of 16-bit inputs: Abramowitz and Stegun's 7.1.26, the error function's complement as a polynomial of 1 / (1 + p x) times
// e^(-x^2), which the slope needs too.  Phi is within 3e-7, g Phi within 5e-7 (by the library's function, which takes two
// branches, too), and the tail keeps relative bits that 1 + erf loses: 2^-9 of Phi(-5) instead of 2^-4.  16384 x 4096 x 11264, by the
// library's function in brackets: g and u 2.42 (2.54) ms, da 1.54 (1.66).

template <class X, int ACTIVATION, bool SLOPE>
__device__ __forceinline__ Activated activate(float g) {
  if constexpr (ACTIVATION == ATTNRES_SILU) {
    const float s = reciprocal<X>(1.0f + exponential<X>(-g));
    return {g * s, SLOPE ? s * (1.0f + g * (1.0f - s)) : 0.0f};
  }
  float phi, bell = 0.0f;  // the normal distribution's integral, and e^(-g^2 / 2)
  if constexpr (kFp32<X>) {
    phi = 0.5f * (1.0f + erff(g * 0.707106781f));
    if (SLOPE) bell = expf(-0.5f * g * g);
  } else {
    bell = __builtin_amdgcn_exp2f(g * g * -0.721347520f);
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.231641888f * fabsf(g));
    const float tail = t * (0.127414796f + t * (-0.142248368f + t * (0.710706871f + t * (-0.726576014f + t * 0.530702714f)))) * bell;
    phi = g < 0.0f ? tail : 1.0f - tail;
  }
  return {g * phi, SLOPE ? phi + g * 0.398942280f * bell : 0.0f};
}

// f with the activation as a constant: a branch around a few entries, so that theirs are formed side by side: da of
// 2048 x 1024 x 2816 32 us, 34 with a branch around each.
template <class F>
__device__ __forceinline__ void with_activation(int activation, F f) {
  if (activation == ATTNRES_SILU) f(std::integral_constant<int, ATTNRES_SILU>{});
  else f(std::integral_constant<int, ATTNRES_GELU>{});
}

// --------------------------------------------------------------- saved g and u

// A subtile of 16 rows by 16 hidden entries: lane l holds row l % 16 and entries 4 (l / 16) + 0..3.
template <class X>
constexpr int kSubBytes = kFp32<X> ? 2048 : 1536;

template <class X>
__device__ __forceinline__ void save_pair(char* to, int lane, f32x4 g, f32x4 u) {
  if constexpr (kFp32<X>) {
    *reinterpret_cast<f32x4*>(to + lane * 16) = g;
    *reinterpret_cast<f32x4*>(to + 1024 + lane * 16) = u;
  } else {
    // to nearest 24 bits, ties away from zero; NaN of products of 16-bit numbers has zeros there, so it stays NaN
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = __float_as_uint(g[e]);
      w[4 + e] = __float_as_uint(u[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] += 0x80u;
    u32x4 high;
#pragma unroll
    for (int e = 0; e < 4; ++e) high[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302u);
    uint32_t low[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t x = __builtin_amdgcn_perm(w[4 * e + 1], w[4 * e], 0x0c0c0501u);
      const uint32_t y = __builtin_amdgcn_perm(w[4 * e + 3], w[4 * e + 2], 0x0c0c0501u);
      low[e] = y << 16 | x;
    }
    *reinterpret_cast<u32x4*>(to + lane * 16) = high;
    *reinterpret_cast<uint64_t*>(to + 1024 + lane * 8) = static_cast<uint64_t>(low[1]) << 32 | low[0];
  }
}

template <class X>
struct Pair {
  u32x4 high;
  u32x4 rest;  // 16-bit inputs: two words
  __device__ __forceinline__ void load(const char* from, int lane) {
    high = *reinterpret_cast<const u32x4*>(from + lane * 16);
    if constexpr (kFp32<X>) {
      rest = *reinterpret_cast<const u32x4*>(from + 1024 + lane * 16);
    } else {
      const uint64_t low = *reinterpret_cast<const uint64_t*>(from + 1024 + lane * 8);
      rest = u32x4{static_cast<uint32_t>(low), static_cast<uint32_t>(low >> 32), 0, 0};
    }
  }
  __device__ __forceinline__ float word(int e) const {  // g: 0..3, u: 4..7
    // bytes: 0, the low one, the two high ones
    const uint32_t select = (e % 2 == 0 ? 0x0504000cu : 0x0706000cu) | static_cast<uint32_t>(e % 4) << 8;
    return __uint_as_float(__builtin_amdgcn_perm(high[e / 2], rest[e / 4], select));
  }
  __device__ __forceinline__ float gate(int e) const {
    if constexpr (kFp32<X>) return __uint_as_float(high[e]);
    return word(e);
  }
  __device__ __forceinline__ float up(int e) const {
    if constexpr (kFp32<X>) return __uint_as_float(rest[e]);
    return word(4 + e);
  }
};

// What is left of x's for the next part, once `packed` has their leading one.
template <class T>
__device__ __forceinline__ void take_part(float* x, const uint32_t* packed, int count) {
  if constexpr (!std::is_same_v<T, float>) {
#pragma unroll
    for (int e = 0; e < count; ++e) x[e] -= to_f32(T{static_cast<uint16_t>(packed[e / 2] >> (16 * (e % 2)))});
  }
}

// ------------------------------------------------------------------ g, u and a
// 16384 x 4096 x 11264, BF16, 2.40-2.43 ms with g and u saved (1.25 PFLOP/s); 4096 x 2048 x 8192, FP16, 0.25-0.28 without, of
// which about 8 us for each of a unit's four tiles go to filling the ring and to the epilogue; 48 x 2048 x 5632 14 us, reading W at 3.3 TB/s.

struct GateArgs {
  Product product;  // A: gate's and up's rows, paired; B: X
  int64_t rows, hidden, hidden_pad;
  int activation;
  char* saved;      // or nullptr
  uint16_t* out[3]; // a [rows][hidden_pad], zeros past hidden; or nullptr
};

template <class X, int SHAPE>
__global__ void __launch_bounds__(Shape<SHAPE>::kAllThreads, Shape<SHAPE>::kGroupsOf) attnres_ffn_gate_kernel(GateArgs g) {
  using T = Part<X>;
  using S = Shape<SHAPE>;
  constexpr int TILE = S::kTileOf, kDown = S::kDownOf, kAcross = S::kAcrossOf;
  __shared__ __align__(16) uint16_t lds[S::kLds];
  TileAt tile;
  if (!tile_at(g.product, g.product.tiles_b, &tile)) return;
  typename S::Sums acc;
  if (!multiply_tile<SHAPE, T, kSegments<X>, true, true, true>(g.product, tile, stages_of(g.product, 0), lds, acc)) return;
  const int wave = wave_index(), lane = threadIdx.x % 64;
  const int f0 = tile.a * (TILE / 2);
  const int64_t n0 = static_cast<int64_t>(tile.b) * TILE;
  const int sub_f = static_cast<int>(g.hidden_pad) / kSub, sub_n = static_cast<int>((g.rows + kSub - 1) / kSub);
  const int at_f = f0 / kSub + (wave % 2) * (kDown / 2), at_n = static_cast<int>(n0) / kSub + (wave / 2) * kAcross;
  const int inside = static_cast<int>(g.hidden) - at_f * kSub - 4 * (lane / 16);  // this lane's entries that count, 16 to a subtile
  char* const saved = g.saved + (static_cast<int64_t>(at_n) * sub_f + at_f) * kSubBytes<X>;
#pragma unroll
  for (int j = 0; j < kAcross; ++j) {
#pragma unroll
    for (int i = 0; i < kDown / 2; ++i) {
      const f32x4 gate = acc[i][j], up = acc[i + kDown / 2][j];
      if (g.saved != nullptr && at_n + j < sub_n && at_f + i < sub_f) {
        save_pair<X>(saved + (static_cast<int64_t>(j) * sub_f + i) * kSubBytes<X>, lane, gate, up);
      }
      with_activation(g.activation, [&](auto activation) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = activate<X, decltype(activation)::value, false>(gate[e]).value * up[e];
          acc[i][j][e] = i * kSub + e < inside ? x : 0.0f;
        }
      });
      __builtin_amdgcn_sched_barrier(0);  // a few outputs at a time: no registers to spill
    }
  }
  if (g.out[0] == nullptr) return;
  constexpr int kChunks = TILE / 16 * kHalves<X>;  // of 16 bytes, of a row in LDS
#pragma unroll
  for (int part = 0; part < kParts<X>; ++part) {
#pragma unroll
    for (int j = 0; j < kAcross; ++j) {
      const int row = (wave / 2) * (16 * kAcross) + j * 16 + lane % 16;
#pragma unroll
      for (int i = 0; i < kDown / 2; ++i) {
        if constexpr (kHalves<X> == 2) {
          const int chunk = (wave % 2) * (2 * kDown) + i * 4 + lane / 16;
          *reinterpret_cast<f32x4*>(lds + staged<kChunks>(row, chunk) * 8) = acc[i][j];
          continue;
        }
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[i][j][e];
        const uint32_t packed[2] = {pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
        if (part + 1 < kParts<X>) {
          take_part<T>(x, packed, 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = x[e];
        }
        const int chunk = (wave % 2) * kDown + i * 2 + lane / 32;
        *reinterpret_cast<uint64_t*>(lds + staged<kChunks>(row, chunk) * 8 + (lane / 16 % 2) * 4) =
            static_cast<uint64_t>(packed[1]) << 32 | packed[0];
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < TILE * kChunks; k += S::kThreadsOf) {
      const int row = k / kChunks, chunk = k % kChunks;
      const int f = f0 + chunk * (8 / kHalves<X>);
      if (n0 + row < g.rows && f < g.hidden_pad) {
        *reinterpret_cast<u32x4*>(g.out[part] + ((n0 + row) * g.hidden_pad + f) * kHalves<X>) =
            *reinterpret_cast<const u32x4*>(lds + staged<kChunks>(row, chunk) * 8);
      }
    }
    if (part + 1 < kParts<X>) __syncthreads();
  }
}

// --------------------------------------------------- FP16 gradients' power of two
// FP16's step is fixed below 2^-14, and upstream gradients of a mean over many tokens lie there: with dg and du rounded as they come
// gate_up's gradient is off by 0.0024, root mean square, at upstream gradients of 1e-5 (512 x 1024 x 704), scaled by 0.0003, as at 1.
// So where the largest finite one is below 1/4 they are held times the power of two that takes it to between 1/4 and 1/2: dg and du have
// 2^17 of it of room upwards, and normal numbers down to 2^-12 of it.  Larger ones are held as they come.  Finding it reads dY once
// more: 4095 x 1537 4.8 us (2.6 TB/s), 390 -> 396 us in all.

template <class X>
constexpr bool kScaled = std::is_same_v<X, F16>;
constexpr int kSlots = 512;           // workgroups that look for the largest, and what each finds
constexpr uint32_t kScaledTo = 125;   // FP32's exponent of 1/4

struct LargestArgs {
  const F16* x;
  int64_t count;
  uint32_t* slots;
};

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
  for (int mask = 1; mask < 64; mask *= 2) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), mask)));
  return x;
}

__global__ void __launch_bounds__(kBlock) attnres_ffn_largest_kernel(LargestArgs g) {
  __shared__ uint32_t tops[kBlock / 64];
  uint32_t top = 0;
  const auto take = [&](uint32_t bits) {
    bits &= 0x7fffu;
    top = bits < 0x7c00u ? max(top, bits) : top;
  };
  const int64_t chunks = g.count / kVec;
#pragma unroll 4
  for (int64_t k = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; k < chunks; k += kSlots * kBlock) {
    const u32x4 w = reinterpret_cast<const Raw16*>(g.x + k * kVec)->v;
#pragma unroll
    for (int e = 0; e < 4; ++e) take(w[e]), take(w[e] >> 16);
  }
  if (blockIdx.x == 0 && threadIdx.x < g.count % kVec) take(g.x[chunks * kVec + threadIdx.x].bits);
  top = wave_max(top);
  if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (const uint32_t other : tops) top = max(top, other);
    g.slots[blockIdx.x] = top;
  }
}

// What dg and du are multiplied by.
__device__ __forceinline__ float scale_of(const uint32_t* slots) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kSlots / 256; ++k) {
    const u32x4 w = reinterpret_cast<const u32x4*>(slots)[k * 64 + threadIdx.x % 64];
    top = max(top, max(max(w[0], w[1]), max(w[2], w[3])));
  }
  top = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(wave_max(top))));
  const uint32_t exponent = __float_as_uint(to_f32(F16{static_cast<uint16_t>(top)})) >> 23;
  return top == 0 || exponent >= kScaledTo ? 1.0f : __uint_as_float((kScaledTo + 127 - exponent) << 23);
}

// ------------------------------------------------------------- da, dg, du and a
// The product, and in its epilogue 12 bytes per entry and row, 6 read and 6 written (FP32: 8 and 18): 16384 x 4096 x 11264, BF16, 1.52 ms
// (0.99 PFLOP/s), 2048 x 1024 x 2816 on tiles of 128 32 us (0.37); FP32, 16384 x 1024 x 2816, 0.76 ms.

struct SlopeArgs {
  Product product;  // A: Wd by columns, B: dY by rows
  int64_t rows, rows_pad, hidden, hidden_pad;
  int activation;
  const char* saved;
  uint16_t* both[3];  // [rows_pad][2 hidden_pad]: dg, du; zeros past rows and hidden
  uint16_t* out[3];   // a [rows_pad][hidden_pad], likewise
  const uint32_t* largest;  // FP16: for scale_of, or nullptr
};

template <class X, int SHAPE>
__global__ void __launch_bounds__(Shape<SHAPE>::kAllThreads, Shape<SHAPE>::kGroupsOf) attnres_ffn_slope_kernel(SlopeArgs g) {
  using T = Part<X>;
  using S = Shape<SHAPE>;
  constexpr int TILE = S::kTileOf, kDown = S::kDownOf, kAcross = S::kAcrossOf;
  __shared__ __align__(16) uint16_t lds[S::kLds];
  TileAt tile;
  if (!tile_at(g.product, g.product.tiles_b, &tile)) return;
  typename S::Sums acc;
  if (!multiply_tile<SHAPE, T, kSegments<X>, false, true>(g.product, tile, stages_of(g.product, 0), lds, acc)) return;
  const int wave = wave_index(), lane = threadIdx.x % 64;
  const int f0 = tile.a * TILE;
  const int64_t n0 = static_cast<int64_t>(tile.b) * TILE;
  const int sub_f = static_cast<int>(g.hidden_pad) / kSub, sub_n = static_cast<int>((g.rows + kSub - 1) / kSub);
  const int at_f = f0 / kSub + (wave % 2) * kDown, at_n = static_cast<int>(n0) / kSub + (wave / 2) * kAcross;
  const int inside_f = static_cast<int>(g.hidden) - at_f * kSub - 4 * (lane / 16);  // this lane's entries that count, 16 to a subtile
  const int inside_n = static_cast<int>(g.rows) - at_n * kSub - lane % 16;
  const bool whole = f0 + TILE <= g.hidden && n0 + TILE <= g.rows;
  // The saved pairs of a round; the next one's are loaded while a round is stored.
  Pair<X> pairs[kDown];
  const auto load_pairs = [&](int j) {
    // past the last subtile: the last one's, which are left out
    const char* from = g.saved + static_cast<int64_t>(min(at_n + j, sub_n - 1)) * sub_f * kSubBytes<X>;
#pragma unroll
    for (int i = 0; i < kDown; ++i) pairs[i].load(from + static_cast<int64_t>(min(at_f + i, sub_f - 1)) * kSubBytes<X>, lane);
  };
  load_pairs(0);
  float scale = 1.0f;
  if constexpr (kScaled<X>) {
    if (g.largest != nullptr) scale = scale_of(g.largest);
  }
  // A round: 16 rows of every wavefront, of three planes in LDS: dg, du and a; of FP32 one of them in its three parts.
  constexpr int kRows = 16 * (S::kWavesOf / 2), kChunks = TILE / 8 * kHalves<X>;
  constexpr int kPlane = kRows * TILE * kHalves<X>;
  static_assert(3 * kPlane <= S::kLds, "three planes");
  constexpr int kTurns = kParts<X>;
  const auto round = [&](auto number, auto turn_number) {
    constexpr int j = decltype(number)::value, turn = decltype(turn_number)::value;
    const int row = (wave / 2) * 16 + lane % 16;
    if (j + turn > 0) __syncthreads();
    const auto form = [&](auto all) {  // all: every entry counts
#pragma unroll
      for (int i = 0; i < kDown; ++i) {
        Pair<X>& pair = pairs[i];
        float x[3][4];
        if constexpr (turn == 0) {
          Activated formed[4];
          with_activation(g.activation, [&](auto activation) {
#pragma unroll
            for (int e = 0; e < 4; ++e) formed[e] = activate<X, decltype(activation)::value, true>(pair.gate(e));
          });
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const Activated act = formed[e];
            float da = acc[i][j][e];
            if constexpr (kScaled<X>) da *= scale;
            const float up = pair.up(e);
            x[0][e] = da * up * act.slope;
            x[1][e] = da * act.value;
            x[2][e] = act.value * up;
            if constexpr (!decltype(all)::value) {
              const bool inside = j * kSub < inside_n && i * kSub + e < inside_f;
#pragma unroll
              for (int plane = 0; plane < 3; ++plane) x[plane][e] = inside ? x[plane][e] : 0.0f;
            }
            if constexpr (kTurns == 3) {  // the two other turns' values in place of g and u
              pair.high[e] = __float_as_uint(x[1][e]);
              pair.rest[e] = __float_as_uint(x[2][e]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[turn][e] = __uint_as_float(turn == 1 ? pair.high[e] : pair.rest[e]);
        }
        const int chunk = kHalves<X> == 2 ? (wave % 2) * (4 * kDown) + i * 4 + lane / 16 : (wave % 2) * (2 * kDown) + i * 2 + lane / 32;
        uint16_t* to = lds + staged<kChunks>(row, chunk) * 8 + (kHalves<X> == 2 ? 0 : lane / 16 % 2 * 4);
#pragma unroll
        for (int plane = 0; plane < 3; ++plane) {
          if constexpr (kHalves<X> == 2) {
            *reinterpret_cast<f32x4*>(to + plane * kPlane) = f32x4{x[plane][0], x[plane][1], x[plane][2], x[plane][3]};
            continue;
          }
          float* value = x[kTurns == 1 ? plane : turn];
          const uint32_t packed[2] = {pack2<T>(value[0], value[1]), pack2<T>(value[2], value[3])};
          *reinterpret_cast<uint64_t*>(to + plane * kPlane) = static_cast<uint64_t>(packed[1]) << 32 | packed[0];
          if constexpr (kTurns > 1) take_part<T>(value, packed, 4);
        }
        if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (whole) form(std::true_type{});
    else form(std::false_type{});
    if constexpr (turn + 1 == kTurns && j + 1 < kAcross) load_pairs(j + 1);
    __syncthreads();
#pragma unroll
    for (int plane = 0; plane < 3; ++plane) {
      const int what = kTurns == 1 ? plane : turn, part = kTurns == 1 ? 0 : plane;
      uint16_t* out = what == 2 ? g.out[part] : g.both[part];
      if (out == nullptr) continue;
      const int64_t ld = what == 2 ? g.hidden_pad : 2 * g.hidden_pad;
      const int64_t first = what == 1 ? g.hidden_pad : 0;
      for (int k = threadIdx.x; k < kRows * kChunks; k += S::kThreadsOf) {
        const int r = k / kChunks, chunk = k % kChunks;
        const int64_t n = n0 + r / 16 * (16 * kAcross) + j * 16 + r % 16;
        const int f = f0 + chunk * (8 / kHalves<X>);
        if (n < g.rows_pad && f < g.hidden_pad) {
          *reinterpret_cast<u32x4*>(out + (n * ld + first + f) * kHalves<X>) =
              *reinterpret_cast<const u32x4*>(lds + plane * kPlane + staged<kChunks>(r, chunk) * 8);
        }
      }
    }
  };
  const auto turns = [&](auto number) {
    round(number, std::integral_constant<int, 0>{});
    if constexpr (kTurns == 3) {
      round(number, std::integral_constant<int, 1>{});
      round(number, std::integral_constant<int, 2>{});
    }
  };
  turns(std::integral_constant<int, 0>{});
  turns(std::integral_constant<int, 1>{});
  if constexpr (kAcross == 4) {
    turns(std::integral_constant<int, 2>{});
    turns(std::integral_constant<int, 3>{});
  }
}

// --------------------------------------------------------------- Y and gradients

struct OutArgs {
  Product product;
  void* out;            // [splits][rows of B][ld]
  int64_t ld, split_stride;
  int64_t entries_a;    // valid contiguous entries
  int64_t half, half_pad;  // entries of B: halves of `half` that count of `half_pad`, in the output one after the other
  int64_t entries_b;
};

// A tile's sums, rounded once or as a part's FP32 sums.
template <class OUT, int SHAPE>
__device__ __forceinline__ void store_tile(const OutArgs& g, const TileAt& tile, const typename Shape<SHAPE>::Sums& acc, uint16_t* lds) {
  using S = Shape<SHAPE>;
  constexpr int TILE = S::kTileOf;
  const int wave = wave_index(), lane = threadIdx.x % 64;
  OUT* out = static_cast<OUT*>(g.out) + tile.split * g.split_stride;
  const int64_t a0 = static_cast<int64_t>(tile.a) * TILE, b0 = static_cast<int64_t>(tile.b) * TILE;
  constexpr bool kWide = std::is_same_v<OUT, float>;
  constexpr int kRounds = kWide ? 2 : 1;  // rows of 2 TILE bytes in LDS: half of the FP32 outputs, or all 16-bit ones
  constexpr int kChunks = TILE / 8;
  constexpr int kChunk = kWide ? 4 : 8;   // outputs per 16 bytes
#pragma unroll
  for (int round = 0; round < kRounds; ++round) {
    if (!kWide || wave % 2 == round) {
#pragma unroll
      for (int j = 0; j < S::kAcrossOf; ++j) {
        const int column = (wave / 2) * (16 * S::kAcrossOf) + j * 16 + lane % 16;
#pragma unroll
        for (int i = 0; i < S::kDownOf; ++i) {
          const f32x4 x = acc[i][j];
          if constexpr (kWide) {
            *reinterpret_cast<f32x4*>(lds + staged<kChunks>(column, i * 4 + lane / 16) * 8) = x;
          } else {
            const int chunk = (wave % 2) * (2 * S::kDownOf) + i * 2 + lane / 32;
            *reinterpret_cast<uint64_t*>(lds + staged<kChunks>(column, chunk) * 8 + (lane / 16 % 2) * 4) =
                static_cast<uint64_t>(pack2<OUT>(x[2], x[3])) << 32 | pack2<OUT>(x[0], x[1]);
          }
          if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // a few outputs at a time: no registers to spill
        }
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < TILE * kChunks; k += S::kThreadsOf) {
      const int column = k / kChunks, chunk = k % kChunks;
      const int64_t a = a0 + round * (TILE / 2) + chunk * kChunk, b = b0 + column;
      const int64_t second = b >= g.half_pad ? 1 : 0, within = b - second * g.half_pad;
      if (b >= g.entries_b || within >= g.half || a >= g.entries_a) continue;
      OUT* to = out + (second * g.half + within) * g.ld + a;
      const uint16_t* from = lds + staged<kChunks>(column, chunk) * 8;
      if constexpr (kWide) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(from);
        if (a + kChunk <= g.entries_a) {
          reinterpret_cast<Raw32*>(to)->v = x;
        } else {
          for (int e = 0; a + e < g.entries_a; ++e) to[e] = x[e];
        }
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(from);
        if (a + kChunk <= g.entries_a) {
          reinterpret_cast<Raw16*>(to)->v = x;
        } else {
          for (int e = 0; a + e < g.entries_a; ++e) to[e].bits = from[e];
        }
      }
    }
    if (round + 1 < kRounds) __syncthreads();
  }
}

// Y (A: Wd by rows, B: a by rows).  16384 x 4096 x 11264, BF16, 1.25-1.33 ms (1.1-1.2 PFLOP/s); 48 x 2048 x 5632 in 8 parts 9.2 us, reading
// Wd at 2.5 TB/s.
template <class X, class OUT, int SHAPE>
__global__ void __launch_bounds__(Shape<SHAPE>::kAllThreads, Shape<SHAPE>::kGroupsOf) attnres_ffn_out_kernel(OutArgs g) {
  using S = Shape<SHAPE>;
  __shared__ __align__(16) uint16_t lds[S::kLds];
  TileAt tile;
  if (!tile_at(g.product, g.product.tiles_b, &tile)) return;
  typename S::Sums acc;
  if (!multiply_tile<SHAPE, Part<X>, kSegments<X>, true, true>(g.product, tile, stages_of(g.product, tile.split), lds, acc)) return;
  store_tile<OUT, SHAPE>(g, tile, acc, lds);
}

// dX (A: W by columns, B: [dg du] by rows), dW (A: X, B: [dg du], both by columns) and dWd (A: a, B: dY, both by columns) in one
// launch, the tiles that take longest first, so that the three fill the chip together: 2048 x 1024 x 2816, BF16, 63 us (0.94 PFLOP/s);
// 16384 x 4096 x 11264 in three launches 6.2-6.5 ms (1.17-1.23 PFLOP/s).
struct GradientsArgs {
  OutArgs of[3];
  uint32_t first[3];  // workgroup of each; past the last: none
  int b_rows[3], wide[3], scaled[3];
  const uint32_t* largest;  // FP16, where any is scaled
};

template <class X, int SHAPE>
__global__ void __launch_bounds__(Shape<SHAPE>::kAllThreads, Shape<SHAPE>::kGroupsOf) attnres_ffn_gradients_kernel(GradientsArgs args) {
  using S = Shape<SHAPE>;
  __shared__ __align__(16) uint16_t lds[S::kLds];
  const int which = (blockIdx.x >= args.first[1] ? 1 : 0) + (blockIdx.x >= args.first[2] ? 1 : 0);
  const OutArgs& g = args.of[which];
  TileAt tile;
  if (!tile_at(g.product, g.product.tiles_b, static_cast<int>(blockIdx.x - args.first[which]), &tile)) return;
  const Stages stages = stages_of(g.product, tile.split);
  typename S::Sums acc;
  if (args.b_rows[which]) {
    if (!multiply_tile<SHAPE, Part<X>, kSegments<X>, false, true>(g.product, tile, stages, lds, acc)) return;
  } else {
    if (!multiply_tile<SHAPE, Part<X>, kSegments<X>, false, false>(g.product, tile, stages, lds, acc)) return;
  }
  if constexpr (kScaled<X>) {
    if (args.scaled[which]) {
      const float by = 1.0f / scale_of(args.largest);
#pragma unroll
      for (int i = 0; i < S::kDownOf; ++i) {
#pragma unroll
        for (int j = 0; j < S::kAcrossOf; ++j) acc[i][j] *= by;
      }
    }
  }
  if (kFp32<X> || args.wide[which]) store_tile<float, SHAPE>(g, tile, acc, lds);
  else store_tile<Value<X>, SHAPE>(g, tile, acc, lds);
}

// Passes over rows of chunks of kVec, several tensors in one launch: a workgroup takes whole rows, kChunksOfGroup chunks or one row,
// and of a tensor of more than kMaxGroups times that the next ones in turn.
constexpr int kChunksOfGroup = kBlock;
constexpr int64_t kMaxGroups = int64_t{1} << 20;  // a launch of four tensors takes 2^30 threads

struct Rows {
  int64_t rows;
  int chunks;       // of a row
  uint32_t first;   // workgroup; UINT32_MAX: not there
  uint32_t groups;
  __host__ __device__ int of_group() const { return chunks >= kChunksOfGroup ? 1 : kChunksOfGroup / chunks; }
};
Rows rows_of(int64_t rows, int64_t chunks, uint32_t first) {
  Rows r{rows, static_cast<int>(chunks), first, 0};
  r.groups = static_cast<uint32_t>(std::min((rows + r.of_group() - 1) / r.of_group(), kMaxGroups));
  return r;
}

// f(row, chunk) for the workgroup's rows.
template <class F>
__device__ __forceinline__ void for_chunks(const Rows& r, F f) {
  const int of_group = r.of_group();
  const int64_t step = static_cast<int64_t>(r.groups) * of_group;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x - r.first) * of_group; row0 < r.rows; row0 += step) {
    const int here = static_cast<int>(min(static_cast<int64_t>(of_group), r.rows - row0)) * r.chunks;
    for (int i = threadIdx.x; i < here; i += kBlock) f(row0 + i / r.chunks, i % r.chunks);
  }
}

// out[r] = the sum of the parts' rows, in order.  Bound by memory: 4096 x 2048 of two parts 13.7 us (6.1 TB/s).
template <class X>
struct JoinArgs {
  Rows rows[3];
  const float* partial[3];
  int splits[3], width[3];
  int64_t split_stride[3];
  X* out[3];
};

template <class X>
__global__ void __launch_bounds__(kBlock) attnres_ffn_join_kernel(JoinArgs<X> g) {
  const int which = (blockIdx.x >= g.rows[1].first ? 1 : 0) + (blockIdx.x >= g.rows[2].first ? 1 : 0);
  const int splits = g.splits[which], width = g.width[which];
  const int64_t stride = g.split_stride[which];
  const float* partial = g.partial[which];
  X* out = g.out[which];
  const int64_t ld = static_cast<int64_t>(g.rows[which].chunks) * kVec;  // rows are padded to whole chunks
  for_chunks(g.rows[which], [&](int64_t r, int chunk) {
    const float* from = partial + r * ld + chunk * kVec;
    float sum[kVec] = {};
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      float x[kVec];
      load8(from + k * stride, x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] += x[e];
    }
    store_chunk(out + r * width, chunk * kVec, width, sum);
  });
}

// Rows to operands: [2 or 1 halves of half_pad][width_pad], zero-padded, of rows in halves of `half`.  Bound by memory: x, W and Wd of
// 16384 x 1024 x 2816, FP32, 40 us (6.4 TB/s), of 4095 x 1537 x 2051, FP16, 15 (4.2).
template <class X>
struct PackArgs {
  Rows rows;  // of the operand
  const Value<X>* x;
  int64_t stride, half, half_pad;
  int width;
  uint16_t* to[3];
};

template <class X>
struct PacksArgs {
  PackArgs<X> of[4];
};

template <class X>
__global__ void __launch_bounds__(kBlock) attnres_ffn_pack_kernel(PacksArgs<X> args) {
  using T = Part<X>;
  int which = 0;
#pragma unroll
  for (int k = 1; k < 4; ++k) which += blockIdx.x >= args.of[k].rows.first ? 1 : 0;
  const PackArgs<X>& g = args.of[which];
  for_chunks(g.rows, [&](int64_t r, int chunk) {
    const int c = chunk * kVec;
    const int64_t second = r >= g.half_pad ? 1 : 0, within = r - second * g.half_pad;
    float v[kVec] = {};
    if (within < g.half && c < g.width) load_chunk(g.x + (second * g.half + within) * g.stride, c, g.width, v);
    const int64_t at = (r * g.rows.chunks + chunk) * kVec;
#pragma unroll
    for (int part = 0; part < kParts<X>; ++part) {
      if constexpr (kHalves<X> == 2) {
        auto* to = reinterpret_cast<f32x4*>(g.to[0] + at * 2);
        to[0] = f32x4{v[0], v[1], v[2], v[3]};
        to[1] = f32x4{v[4], v[5], v[6], v[7]};
        continue;
      }
      uint32_t packed[kVec / 2];
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) packed[e] = pack2<T>(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<u32x4*>(g.to[part] + at) = u32x4{packed[0], packed[1], packed[2], packed[3]};
      if (part + 1 < kParts<X>) take_part<T>(v, packed, kVec);
    }
  });
}

// ------------------------------------------------------------------- few rows
// The forward of up to 16 rows, 32 of FP32, or kFewRows where tiles need packed weights, reads the weights once and is bound by that:
// wavefronts share the depth of 16 entries of A (of a gate's 8 and the up projection's 8 that belong to them), so that all of a workgroup's weights
// are asked for at once, and nothing is packed.  FP32 inputs by FP32 matrix instructions, which so few rows have time for.
// A lane's 16 bytes are of a row of its own, which the caches serve slowly: BF16, 2048 x 5632, by tiles in brackets, 1 row 19.2 (31) us, 16
// 26.2 (25.8), 48 46.6 (26.8); 1024 x 2816, 1 row 10.7 (20), 32 15.9 (18.4); FP32, 4096 x 11264, 17 rows 184 (241), 32 211 (229);
// packed, 4001 x 4000, 64 rows 117 (157).
constexpr int64_t kFewRows = 64;

// The wavefronts' sums over their shares of the depth, in LDS; ROWS of a's tiles by TILES of the rows'.
template <class X, int WAVES, int ATILES, int TILES>
__device__ __forceinline__ void few_product(const X* const (&a)[ATILES], const X* const (&b)[TILES], int depth,
                                            f32x4 (*parts)[ATILES][TILES][64]) {
  const int wave = wave_index(), lane = threadIdx.x % 64, group = lane / 16;
  constexpr int kSteps = sizeof(X) == 4 || ATILES * TILES > 2 ? 1 : 2;  // of 64 k's under way together
  constexpr int kSpan = kSteps * 64;
  FewChunk<X> next[kSteps][ATILES];
  const auto fetch = [&](int k0) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < ATILES; ++i) next[s][i].load(a[i], k0 + s * 64, group, depth);
    }
  };
  f32x4 acc[ATILES][TILES] = {};
  if (wave * kSpan < depth) fetch(wave * kSpan);
  for (int k0 = wave * kSpan; k0 < depth; k0 += WAVES * kSpan) {
    FewChunk<X> now[kSteps][ATILES];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < ATILES; ++i) now[s][i] = next[s][i];
    }
    if (k0 + WAVES * kSpan < depth) fetch(k0 + WAVES * kSpan);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        FewChunk<X> x;  // the few rows stay in the caches
        x.load(b[t], k0 + s * 64, group, depth);
#pragma unroll
        for (int i = 0; i < ATILES; ++i) acc[i][t] = few_mfma<X>(now[s][i], x, acc[i][t]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ATILES; ++i) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) parts[wave][i][t][lane] = acc[i][t];
  }
  __syncthreads();
}

template <class X, int WAVES, int ATILES, int TILES>
__device__ __forceinline__ f32x4 few_sum(const f32x4 (*parts)[ATILES][TILES][64], int i, int t, int lane) {
  f32x4 sum = parts[0][i][t][lane];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) sum += parts[w][i][t][lane];
  return sum;
}

template <class X>
struct FewGateArgs {
  const X* x;
  const X* gate_up;
  int64_t x_stride, gate_up_stride;
  int rows, width, hidden, hidden_pad, activation;
  char* saved;  // or nullptr
  X* out;       // a [rows][hidden_pad], or nullptr
};

template <class T>
__device__ __forceinline__ void store_quad(T* to, int left, const float* x) {
  T v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = from_f32<T>(x[e]);
  if (left >= 4) {
    __builtin_memcpy(to, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < left) to[e] = v[e];
    }
  }
}

template <class X, int WAVES, int ATILES, int TILES>
__global__ void __launch_bounds__(64 * WAVES) attnres_ffn_few_gate_kernel(FewGateArgs<X> g) {
  __shared__ f32x4 parts[WAVES][ATILES][TILES][64];
  const int entry = threadIdx.x % 16;
  const int f0 = static_cast<int>(blockIdx.x) * (8 * ATILES);
  const X* a[ATILES];
  const X* b[TILES];
#pragma unroll
  for (int i = 0; i < ATILES; ++i) {
    const int64_t f = min(f0 + i * 8 + entry % 8, g.hidden - 1);
    a[i] = g.gate_up + (f + (entry < 8 ? 0 : g.hidden)) * g.gate_up_stride;
  }
#pragma unroll
  for (int t = 0; t < TILES; ++t) b[t] = g.x + min(t * 16 + entry, g.rows - 1) * g.x_stride;
  few_product<X, WAVES, ATILES, TILES>(a, b, g.width, parts);
  // a thread per row and four hidden entries: lanes 0..31 hold a tile's gates, 32..63 what belongs to them
  for (int k = threadIdx.x; k < ATILES * TILES * 32; k += 64 * WAVES) {
    const int i = k / (TILES * 32), t = k / 32 % TILES, lane = k % 32;
    const int row = t * 16 + lane % 16, f = f0 + i * 8 + lane / 16 * 4;
    if (row >= g.rows || f >= g.hidden) continue;
    const f32x4 gate = few_sum<X, WAVES, ATILES, TILES>(parts, i, t, lane), up = few_sum<X, WAVES, ATILES, TILES>(parts, i, t, lane + 32);
    if (g.saved != nullptr) {
      const int64_t sub = static_cast<int64_t>(row / kSub) * (g.hidden_pad / kSub) + f / kSub;
      save_pair<X>(g.saved + sub * kSubBytes<X>, f % kSub / 4 * 16 + row % kSub, gate, up);
    }
    if (g.out != nullptr) {
      float x[4];
      with_activation(g.activation, [&](auto activation) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = activate<X, decltype(activation)::value, false>(gate[e]).value * up[e];
      });
      store_quad(g.out + static_cast<int64_t>(row) * g.hidden_pad + f, g.hidden - f, x);
    }
  }
}

template <class X>
struct FewOutArgs {
  const X* a;
  const X* down;
  int64_t a_stride, down_stride;
  int rows, hidden, out_width;
  X* out;
};

template <class X, int WAVES, int TILES>
__global__ void __launch_bounds__(64 * WAVES) attnres_ffn_few_out_kernel(FewOutArgs<X> g) {
  __shared__ f32x4 parts[WAVES][1][TILES][64];
  const int entry = threadIdx.x % 16;
  const int e0 = static_cast<int>(blockIdx.x) * 16;
  const X* const a[1] = {g.down + min(e0 + entry, g.out_width - 1) * g.down_stride};
  const X* b[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) b[t] = g.a + min(t * 16 + entry, g.rows - 1) * g.a_stride;
  few_product<X, WAVES, 1, TILES>(a, b, g.hidden, parts);
  for (int k = threadIdx.x; k < TILES * 64; k += 64 * WAVES) {
    const int t = k / 64, lane = k % 64;
    const int row = t * 16 + lane % 16, e = e0 + lane / 16 * 4;
    if (row >= g.rows || e >= g.out_width) continue;
    const f32x4 sum = few_sum<X, WAVES, 1, TILES>(parts, 0, t, lane);
    const float x[4] = {sum[0], sum[1], sum[2], sum[3]};
    store_quad(g.out + static_cast<int64_t>(row) * g.out_width + e, g.out_width - e, x);
  }
}

// ---------------------------------------------------------------------- host

constexpr int64_t kMaxRows = int64_t{1} << 24;
constexpr int64_t kMaxHidden = int64_t{1} << 16;
constexpr int64_t kMaxStride = int64_t{1} << 22;  // of operands multiplied in place: 256 rows stay within 32-bit offsets
constexpr int64_t kMaxSecond = int64_t{1} << 30;  // from the gate's rows to the up's, of 16 bits
constexpr int64_t kMaxTiles = int64_t{1} << 22;   // a launch takes fewer than 2^32 threads
// Rounds of the chip up to which the gradients' products go in one launch of tiles of 256 (smaller ones always do): one product's last
// round is filled by the next one's first, which counts less the more rounds there are, and each then finds less of its operands in the
// caches.  Three launches against one, rows x width x hidden, BF16: 4096 x 1024 x 2816 0.309 ms to 0.144, 4096 x 2048 x 5632
// 0.603 to 0.496, 8192 x 2048 x 5632 0.990 to 0.943; 4096 x 4096 x 8192 1.21 to 1.20; 16384 x 4096 x 11264 6.17 to 6.23.  Tiles of 128,
// 2048 x 2048 x 5632: 0.374 to 0.327; FP32 on tiles of 64, 200 x 4096 x 11264: 1.24 to 1.09.
constexpr uint32_t kTogether = 8;
inline bool together(int tile, int64_t workgroups) { return tile < 256 || workgroups <= kTogether * kUnits; }
// Rows, and rows times widths, up to which FP32 inputs are multiplied as they are: FP32 instructions reach 100-115 TFLOP/s, the six products
// of parts 170 once their operands are packed (22 bytes moved per element of a weight and tile of rows, not 4).  Forward and
// backward in kernels, by parts in brackets: 512 x 2048 x 4096 0.66 (0.84) ms, 1024 x 1024 x 2816 0.58 (0.62), 2048 x 512 x 512
// 0.13 (0.19), 4000 x 256 x 1024 0.23 (0.26), 1024 x 4096 x 4096 2.52 (2.52); 1500 x 1024 x 2816 0.82 (0.74).
constexpr int64_t kSingleRows = 1024;
constexpr int64_t kSingleProducts = int64_t{1} << 31;

enum Pass { kForward = 0, kBackward = 1, kBackwardAgain = 2 };  // the last: without saved g and u

struct Sizes {
  int64_t rows, width, hidden, out_width;
  int dtype;
};

// How products are shared out: the tiles' size, and the parts that the depth of each is cut into.
struct Cut {
  int tile, splits[3];
  int shared;  // the depth of tiles of 64, by two (1) or four (2) times as many wavefronts
  int shape() const { return tile + shared; }
};
struct Outputs {
  int64_t a, b, depth;  // entries; 0: not asked for
};

struct FfnPlan {
  int parts, segments;
  bool few, single;  // FP32 by matrix instructions of its own
  int halves;         // of a product's element
  int64_t rows_pad, width_pad, hidden_pad, out_pad;
  bool pack_x, pack_gate_up, pack_down, pack_grad;
  int64_t x[3], gate_up[3], down[3], grad[3], a[3], both[3];  // offsets
  int64_t saved, largest, partial;
  Cut gate, slope, out, gradients;
  int64_t partials[3];
  int64_t bytes, saved_bytes;
};

int64_t tiles_of(int64_t n, int64_t tile) { return (n + tile - 1) / tile; }

// When the last unit is done, if each takes the next tile as soon as it is free: `count` tiles that take `each`, longest first.
class Schedule {
 public:
  void add(int64_t count, double each) {
    const int64_t whole = std::max<int64_t>(count / kUnits - 1, 0);  // rounds of all units
    for (int i = 0; i < size_; ++i) level_[i].time += static_cast<double>(whole) * each;
    for (count -= whole * kUnits; count > 0;) {
      int first = 0;
      for (int i = 1; i < size_; ++i) {
        if (level_[i].time < level_[first].time) first = i;
      }
      Level& level = level_[first];
      if (count >= level.units || size_ == kLevels) {
        level.time += each;
        count -= level.units;
      } else {
        level_[size_++] = {level.time + each, static_cast<int>(count)};
        level.units -= static_cast<int>(count);
        count = 0;
      }
    }
  }
  double end() const {
    double last = 0.0;
    for (int i = 0; i < size_; ++i) last = std::max(last, level_[i].time);
    return last;
  }

 private:
  static constexpr int kLevels = 8;  // one more per product at most
  struct Level {
    double time;
    int units;
  };
  Level level_[kLevels] = {{0.0, kUnits}};
  int size_ = 1;
};

// The cut that takes the least time: the schedule of all tiles at a unit's rate for them, and the partial sums' way to memory and
// back.  Rates as measured on a full chip.
Cut choose_cut(const Outputs* outputs, int count, const FfnPlan& plan, bool whole) {
  const int segments = plan.segments;
  Cut best{256, {1, 1, 1}, 0};
  double least = 0.0;
  for (const int tile : {256, 128, 64}) {
    if (plan.single && tile > 128) continue;
    // a workgroup alone on a unit that has room for more reaches two thirds of its rate
    const double alone = tile == 256 ? 1.0 : 1.5;
    // FP32 operands: their depth counts twice
    const double rate = (plan.single ? (tile == 128 ? 0.23e15 : 0.2e15) : tile == 256 ? 1.25e15 : tile == 128 ? 0.87e15 : 0.6e15) / kUnits;
    const double ends = tile == 256 ? 5e-6 : tile == 128 ? 2e-6 : 1e-6;  // of a tile: its first loads and its epilogue
    int64_t tiles[3] = {};
    bool fits = true;
    for (int i = 0; i < count; ++i) {
      tiles[i] = tiles_of(outputs[i].a, tile) * tiles_of(outputs[i].b, tile);
      fits = fits && (tile == 256 || tiles[i] <= kMaxTiles);
    }
    if (!fits) continue;
    Cut cut{tile, {1, 1, 1}, false};
    int worse = 0;  // cuts since the best one of this size
    double nearest = 1e9;
    for (;;) {
      double each[3], partial = 0.0;
      int order[3] = {0, 1, 2};
      int64_t workgroups = 0, least_depth = int64_t{1} << 40;
      for (int i = 0; i < count; ++i) {
        workgroups += tiles[i] * cut.splits[i];
        if (tiles[i] > 0) least_depth = std::min(least_depth, outputs[i].depth / cut.splits[i]);
        each[i] = 2.0 * tile * tile * static_cast<double>(outputs[i].depth) * segments / cut.splits[i] / rate + ends;
        if (cut.splits[i] > 1) partial += 4e-6 + 8.0 * static_cast<double>(outputs[i].a * outputs[i].b) * cut.splits[i] / 4.5e12;
      }
      std::sort(order, order + count, [&](int i, int j) { return each[i] > each[j]; });
      Schedule schedule;
      for (int i = 0; i < count; ++i) schedule.add(tiles[order[i]] * cut.splits[order[i]], each[order[i]]);
      const int longest = order[0];
      const double time = std::max(schedule.end(), alone * each[longest]) + partial;
      worse = time < nearest ? 0 : worse + 1;
      nearest = std::min(nearest, time);
      if (least == 0.0 || time < least) {
        least = time;
        best = cut;
        const int64_t steps = least_depth / kDepth;
        best.shared = 0;
        if (tile == 64 && workgroups <= kUnits && steps >= 16) best.shared = 2;
        else if (tile == 64 && workgroups > kUnits && workgroups <= 2 * kUnits && steps >= 32) best.shared = 1;
      }
      if (whole || worse == 4 || cut.splits[longest] >= 32 || outputs[longest].depth / kDepth / (cut.splits[longest] + 1) < 4) break;
      ++cut.splits[longest];
    }
  }
  return best;
}

int64_t saved_bytes(const Sizes& s) {
  return tiles_of(s.rows, kSub) * (round_up(s.hidden, kDepth) / kSub) * (s.dtype == ATTNRES_F32 ? kSubBytes<float> : kSubBytes<Bf16>);
}

FfnPlan make_plan(const Sizes& s, int pass) {
  FfnPlan p{};
  p.rows_pad = round_up(s.rows, kDepth);
  p.width_pad = round_up(s.width, kDepth);
  p.hidden_pad = round_up(s.hidden, kDepth);
  p.out_pad = round_up(s.out_width, kDepth);
  p.single = s.dtype == ATTNRES_F32 &&
             (s.rows <= kSingleRows || p.rows_pad * std::max(p.width_pad, p.out_pad) * p.hidden_pad <= kSingleProducts);
  const bool split = s.dtype == ATTNRES_F32 && !p.single, backward = pass != kForward;
  p.parts = split ? 3 : 1;
  p.segments = split ? 6 : 1;
  p.halves = p.single ? 2 : 1;
  const int64_t size = 2 * p.halves;
  // the depth of a product is a whole number of stages, the rest of the last one zeros
  p.few = s.rows <= (s.width != p.width_pad || s.hidden != p.hidden_pad ? kFewRows : p.single ? kFewRows / 2 : kFewRows / 4);
  const bool tiles = backward || !p.few;
  p.pack_x = tiles && (split || s.width != p.width_pad || (backward && s.rows != p.rows_pad));
  p.pack_gate_up = tiles && (split || s.width != p.width_pad || s.hidden != p.hidden_pad);
  p.pack_down = tiles && (split || s.hidden != p.hidden_pad || (backward && s.out_width != p.out_pad));
  p.pack_grad = backward && (split || s.out_width != p.out_pad || s.rows != p.rows_pad);
  p.saved_bytes = saved_bytes(s);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += round_up(bytes, 256);
    return from;
  };
  for (int k = 0; k < p.parts; ++k) {
    if (p.pack_x) p.x[k] = take(size * p.rows_pad * p.width_pad);
    if (p.pack_gate_up) p.gate_up[k] = take(2 * size * p.hidden_pad * p.width_pad);
    if (p.pack_down) p.down[k] = take(size * p.out_pad * p.hidden_pad);
    if (p.pack_grad) p.grad[k] = take(size * p.rows_pad * p.out_pad);
    if (tiles) p.a[k] = take(size * p.rows_pad * p.hidden_pad);
    if (backward) p.both[k] = take(2 * size * p.rows_pad * p.hidden_pad);
  }
  if (!tiles) p.a[0] = take(s.rows * p.hidden_pad * dtype_size(s.dtype));
  if (pass == kBackwardAgain) p.saved = take(p.saved_bytes);
  if (backward && s.dtype == ATTNRES_F16) p.largest = take(4 * kSlots);
  int64_t partial = 0;
  // what the sums of g, u and da go into needs them whole
  const auto one = [&](int64_t a, int64_t b, int64_t depth, bool whole) {
    const Outputs o{a, b, depth * p.halves};
    return choose_cut(&o, 1, p, whole);
  };
  if (tiles) p.gate = one(2 * p.hidden_pad, s.rows, p.width_pad, true);
  if (!backward && tiles) {
    p.out = one(s.out_width, s.rows, p.hidden_pad, false);
    if (p.out.splits[0] > 1) partial = 4 * p.out.splits[0] * s.rows * round_up(s.out_width, kVec);
  }
  if (backward) {
    p.slope = one(p.hidden_pad, p.rows_pad, p.out_pad, true);
    const Outputs o[3] = {{s.width, s.rows, 2 * p.hidden_pad * p.halves},
                          {s.width, 2 * p.hidden_pad, p.rows_pad * p.halves},
                          {s.hidden, s.out_width, p.rows_pad * p.halves}};
    p.gradients = choose_cut(o, 3, p, false);
    for (int i = 0; i < 3; ++i) {
      p.partials[i] = partial;
      if (p.gradients.splits[i] > 1) partial += round_up(4 * p.gradients.splits[i] * o[i].b * round_up(o[i].a, kVec), 256);
    }
  }
  p.partial = take(partial);
  p.bytes = at;
  return p;
}

// The plan of these sizes; a call asks for it up to three times, and a program for the same few.
const FfnPlan& ffn_plan(const Sizes& s, int pass) {
  struct Known {
    Sizes s{-1, 0, 0, 0, 0};
    int pass = 0;
    FfnPlan plan{};
  };
  thread_local Known known[8];
  thread_local int oldest = 0;
  for (const Known& k : known) {
    if (k.pass == pass && k.s.rows == s.rows && k.s.width == s.width && k.s.hidden == s.hidden && k.s.out_width == s.out_width &&
        k.s.dtype == s.dtype) {
      return k.plan;
    }
  }
  Known& k = known[oldest];
  oldest = (oldest + 1) % 8;
  k = {s, pass, make_plan(s, pass)};
  return k.plan;
}

struct Call {
  Sizes s;
  const void* x;
  int64_t x_stride;
  const void* gate_up;
  int64_t gate_up_stride;
  const void* down;
  int64_t down_stride;
  int activation;
  FfnPlan plan;
  char* workspace;
  hipStream_t stream;
  uint16_t* operand(int64_t offset) const { return reinterpret_cast<uint16_t*>(workspace + offset); }
};

template <class X, class F>
void with_shape(const Cut& cut, F f) {
  if constexpr (!std::is_same_v<X, Single>) {
    if (cut.tile == 256) return f(std::integral_constant<int, 256>{});
  }
  if (cut.tile == 128) return f(std::integral_constant<int, 128>{});
  switch (cut.shape()) {
    case 65: return f(std::integral_constant<int, 65>{});
    case 66: return f(std::integral_constant<int, 66>{});
    default: return f(std::integral_constant<int, 64>{});
  }
}

// Operands where they lie, or packed into the workspace, all by one launch.
template <class X>
class Operands {
 public:
  explicit Operands(const Call& c) : c_(c) {
    for (auto& p : args_.of) p.rows.first = UINT32_MAX;
  }
  Operand x() { return place(c_.plan.pack_x, c_.plan.x, c_.x, c_.x_stride, c_.s.rows, c_.plan.rows_pad, 1, c_.s.width, c_.plan.width_pad); }
  Operand gate_up() {
    return place(c_.plan.pack_gate_up, c_.plan.gate_up, c_.gate_up, c_.gate_up_stride, c_.s.hidden, c_.plan.hidden_pad, 2, c_.s.width,
                 c_.plan.width_pad);
  }
  Operand down() {
    return place(c_.plan.pack_down, c_.plan.down, c_.down, c_.down_stride, c_.s.out_width, c_.plan.out_pad, 1, c_.s.hidden,
                 c_.plan.hidden_pad);
  }
  Operand grad(const void* grad) {
    return place(c_.plan.pack_grad, c_.plan.grad, grad, c_.s.out_width, c_.s.rows, c_.plan.rows_pad, 1, c_.s.out_width, c_.plan.out_pad);
  }
  void pack() {
    if (count_ > 0) hipLaunchKernelGGL((attnres_ffn_pack_kernel<X>), dim3(groups_), dim3(kBlock), 0, c_.stream, args_);
  }

 private:
  Operand place(bool pack, const int64_t* offsets, const void* x, int64_t stride, int64_t half, int64_t half_pad, int halves, int64_t width,
                int64_t width_pad) {
    if (!pack) return {{static_cast<const uint16_t*>(x), nullptr, nullptr}, stride, 0, 0, 0};
    PackArgs<X>& g = args_.of[count_++];
    g = {rows_of(halves * half_pad, width_pad / kVec, groups_), static_cast<const Value<X>*>(x), stride, half, half_pad,
         static_cast<int>(width), {}};
    groups_ += g.rows.groups;
    Operand o{{nullptr, nullptr, nullptr}, width_pad, 0, 0, 0};
    for (int k = 0; k < kParts<X>; ++k) o.part[k] = g.to[k] = c_.operand(offsets[k]);
    return o;
  }
  const Call& c_;
  PacksArgs<X> args_{};
  int count_ = 0;
  uint32_t groups_ = 0;
};

// g and u, and a from them.
template <class X>
void launch_gate(const Call& c, const Operand& x, const Operand& gate_up, char* saved, const int64_t* a) {
  const FfnPlan& p = c.plan;
  GateArgs g{};
  Operand w = gate_up, rows = x;
  w.entries = p.pack_gate_up ? p.hidden_pad : c.s.hidden;
  w.second = w.entries * w.ld;
  rows.entries = c.s.rows;
  const int tile = p.gate.tile;
  g.product = {w, rows, nullptr, p.width_pad * p.halves, 0, static_cast<int>(tiles_of(p.hidden_pad, tile / 2)),
               static_cast<int>(tiles_of(c.s.rows, tile)), 1};
  g.rows = c.s.rows;
  g.hidden = c.s.hidden;
  g.hidden_pad = p.hidden_pad;
  g.activation = c.activation;
  g.saved = saved;
  for (int k = 0; a != nullptr && k < kParts<X>; ++k) g.out[k] = c.operand(a[k]);
  with_shape<X>(p.gate, [&](auto size) {
    constexpr int SHAPE = decltype(size)::value;
    hipLaunchKernelGGL((attnres_ffn_gate_kernel<X, SHAPE>), dim3(g.product.tiles_a * g.product.tiles_b), dim3(Shape<SHAPE>::kAllThreads), 0,
                       c.stream, g);
  });
}

// Of few rows: g and u, and a from them.
template <class X>
void launch_few_gate(const Call& c, char* saved, X* a) {
  const FewGateArgs<X> g{static_cast<const X*>(c.x), static_cast<const X*>(c.gate_up), c.x_stride, c.gate_up_stride,
                         static_cast<int>(c.s.rows), static_cast<int>(c.s.width), static_cast<int>(c.s.hidden),
                         static_cast<int>(c.plan.hidden_pad), c.activation, saved, a};
  const auto launch = [&](auto kernel, int waves, int tiles) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles_of(c.s.hidden, 8 * tiles))), dim3(64 * waves), 0, c.stream, g);
  };
  if (c.s.rows <= 16) launch(attnres_ffn_few_gate_kernel<X, 8, 1, 1>, 8, 1);
  else if (c.s.rows <= 32) launch(attnres_ffn_few_gate_kernel<X, 8, 2, 2>, 8, 2);
  else launch(attnres_ffn_few_gate_kernel<X, 8, 2, 4>, 8, 2);
}

template <class X>
void few_forward(const Call& c, void* out, char* saved) {
  X* a = reinterpret_cast<X*>(c.workspace + c.plan.a[0]);
  launch_few_gate<X>(c, saved, a);
  const FewOutArgs<X> g{a, static_cast<const X*>(c.down), c.plan.hidden_pad, c.down_stride, static_cast<int>(c.s.rows),
                        static_cast<int>(c.s.hidden), static_cast<int>(c.s.out_width), static_cast<X*>(out)};
  const auto kernel = c.s.rows <= 16   ? attnres_ffn_few_out_kernel<X, 16, 1>
                      : c.s.rows <= 32 ? attnres_ffn_few_out_kernel<X, 16, 2>
                                       : attnres_ffn_few_out_kernel<X, 16, 4>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles_of(c.s.out_width, 16))), dim3(1024), 0, c.stream, g);
}

// A product into out[b][a], by halves of B's entries, or its parts into the workspace.
OutArgs out_args(const Call& c, const Operand& a, const Operand& b, int64_t depth, int64_t entries_a, int64_t half, int64_t half_pad,
                 int64_t entries_b, int tile, int splits, int64_t partial, void* out) {
  OutArgs g{};
  g.product = {a, b, nullptr, depth * c.plan.halves, 0, static_cast<int>(tiles_of(entries_a, tile)),
               static_cast<int>(tiles_of(entries_b, tile)), splits};
  g.entries_a = entries_a;
  g.half = half;
  g.half_pad = half_pad;
  g.entries_b = entries_b;
  g.out = out;
  g.ld = entries_a;
  if (splits > 1) {
    g.out = c.workspace + c.plan.partial + partial;
    g.ld = round_up(entries_a, kVec);
    g.split_stride = entries_b / half_pad * half * g.ld;
  }
  return g;
}

unsigned workgroups(const OutArgs& g) { return static_cast<unsigned>(g.product.tiles_a) * g.product.tiles_b * g.product.splits; }

// The sums of the parts of those of three products that are cut.
template <class X>
void join_parts(const Call& c, const OutArgs (&of)[3], void* const (&results)[3]) {
  JoinArgs<X> g{};
  int count = 0;
  uint32_t groups = 0;
  for (int i = 0; i < 3; ++i) {
    if (results[i] == nullptr || of[i].product.splits == 1) continue;
    g.rows[count] = rows_of(of[i].split_stride / of[i].ld, of[i].ld / kVec, groups);
    g.partial[count] = static_cast<const float*>(of[i].out);
    g.splits[count] = of[i].product.splits;
    g.width[count] = static_cast<int>(of[i].entries_a);
    g.split_stride[count] = of[i].split_stride;
    g.out[count] = static_cast<X*>(results[i]);
    groups += g.rows[count++].groups;
  }
  for (int k = count; k < 3; ++k) g.rows[k].first = UINT32_MAX;
  if (count > 0) hipLaunchKernelGGL((attnres_ffn_join_kernel<X>), dim3(groups), dim3(kBlock), 0, c.stream, g);
}

template <class X>
void ffn_forward(const Call& c, void* out, char* saved) {
  const FfnPlan& p = c.plan;
  if (p.few) return few_forward<Value<X>>(c, out, saved);
  Operands<X> operands(c);
  const Operand x = operands.x(), gate_up = operands.gate_up();
  Operand down = operands.down(), a{};
  operands.pack();
  launch_gate<X>(c, x, gate_up, saved, p.a);
  down.entries = c.s.out_width;
  for (int k = 0; k < kParts<X>; ++k) a.part[k] = c.operand(p.a[k]);
  a.ld = p.hidden_pad;
  a.entries = c.s.rows;
  const int splits = p.out.splits[0];
  const OutArgs g = out_args(c, down, a, p.hidden_pad, c.s.out_width, c.s.rows, c.s.rows, c.s.rows, p.out.tile, splits, 0, out);
  with_shape<X>(p.out, [&](auto size) {
    constexpr int SHAPE = decltype(size)::value;
    const auto kernel = splits > 1 ? attnres_ffn_out_kernel<X, float, SHAPE> : attnres_ffn_out_kernel<X, Value<X>, SHAPE>;
    hipLaunchKernelGGL(kernel, dim3(workgroups(g)), dim3(Shape<SHAPE>::kAllThreads), 0, c.stream, g);
  });
  join_parts<Value<X>>(c, {g, OutArgs{}, OutArgs{}}, {out, nullptr, nullptr});
}

template <class X>
void ffn_backward(const Call& c, const void* grad_out, const char* saved, void* grad_x, void* grad_gate_up, void* grad_down) {
  const FfnPlan& p = c.plan;
  Operands<X> operands(c);
  Operand x{}, gate_up{};
  const bool again = saved == nullptr && !p.few;
  if (again || grad_gate_up != nullptr) x = operands.x();
  if (again || grad_x != nullptr) gate_up = operands.gate_up();
  Operand down = operands.down();
  const Operand grad = operands.grad(grad_out);
  operands.pack();
  if (saved == nullptr) {
    char* formed = c.workspace + p.saved;
    if (p.few) launch_few_gate<Value<X>>(c, formed, nullptr);
    else launch_gate<X>(c, x, gate_up, formed, nullptr);
    saved = formed;
  }
  const uint32_t* largest = nullptr;
  if constexpr (kScaled<X>) {
    if (grad_x != nullptr || grad_gate_up != nullptr) {
      const LargestArgs g{static_cast<const F16*>(grad_out), c.s.rows * c.s.out_width, reinterpret_cast<uint32_t*>(c.workspace + p.largest)};
      hipLaunchKernelGGL(attnres_ffn_largest_kernel, dim3(kSlots), dim3(kBlock), 0, c.stream, g);
      largest = g.slots;
    }
  }
  {
    SlopeArgs g{};
    g.largest = largest;
    Operand rows = grad;
    down.entries = p.hidden_pad;
    down.depth = p.out_pad;
    rows.entries = c.s.rows;
    const int tile = p.slope.tile;
    g.product = {down, rows, nullptr, p.out_pad * p.halves, 0, static_cast<int>(tiles_of(p.hidden_pad, tile)),
                 static_cast<int>(tiles_of(p.rows_pad, tile)), 1};
    g.rows = c.s.rows;
    g.rows_pad = p.rows_pad;
    g.hidden = c.s.hidden;
    g.hidden_pad = p.hidden_pad;
    g.activation = c.activation;
    g.saved = saved;
    for (int k = 0; k < kParts<X>; ++k) {
      if (grad_x != nullptr || grad_gate_up != nullptr) g.both[k] = c.operand(p.both[k]);
      if (grad_down != nullptr) g.out[k] = c.operand(p.a[k]);
    }
    with_shape<X>(p.slope, [&](auto size) {
      constexpr int SHAPE = decltype(size)::value;
      hipLaunchKernelGGL((attnres_ffn_slope_kernel<X, SHAPE>), dim3(g.product.tiles_a * g.product.tiles_b), dim3(Shape<SHAPE>::kAllThreads), 0,
                         c.stream, g);
    });
  }
  Operand both{}, a{};
  for (int k = 0; k < kParts<X>; ++k) {
    both.part[k] = c.operand(p.both[k]);
    a.part[k] = c.operand(p.a[k]);
  }
  both.ld = 2 * p.hidden_pad;
  a.ld = p.hidden_pad;
  both.depth = a.depth = p.rows_pad;
  // in the order of the plan's cut
  OutArgs of[3] = {};
  const int tile = p.gradients.tile;
  const int* splits = p.gradients.splits;
  void* const results[3] = {grad_x, grad_gate_up, grad_down};
  if (grad_x != nullptr) {
    gate_up.entries = p.pack_gate_up ? p.width_pad : c.s.width;
    gate_up.depth = 2 * p.hidden_pad;
    both.entries = c.s.rows;
    of[0] = out_args(c, gate_up, both, 2 * p.hidden_pad, c.s.width, c.s.rows, c.s.rows, c.s.rows, tile, splits[0], p.partials[0], grad_x);
  }
  if (grad_gate_up != nullptr) {
    x.entries = p.pack_x ? p.width_pad : c.s.width;
    x.depth = p.rows_pad;
    both.entries = 2 * p.hidden_pad;
    of[1] = out_args(c, x, both, p.rows_pad, c.s.width, c.s.hidden, p.hidden_pad, 2 * p.hidden_pad, tile, splits[1], p.partials[1],
                     grad_gate_up);
  }
  if (grad_down != nullptr) {
    Operand rows = grad;
    rows.entries = p.pack_grad ? p.out_pad : c.s.out_width;
    rows.depth = p.rows_pad;
    a.entries = p.hidden_pad;
    of[2] = out_args(c, a, rows, p.rows_pad, c.s.hidden, c.s.out_width, c.s.out_width, c.s.out_width, tile, splits[2], p.partials[2],
                     grad_down);
  }
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int i, int j) { return of[i].product.depth * splits[j] > of[j].product.depth * splits[i]; });
  uint32_t all = 0;
  for (const int i : order) all += results[i] != nullptr ? workgroups(of[i]) : 0;
  const bool one_launch = together(tile, all);
  GradientsArgs g{};
  g.largest = largest;
  int count = 0;
  uint32_t grid = 0;
  const auto launch = [&] {
    if (count == 0) return;
    for (int k = count; k < 3; ++k) g.first[k] = UINT32_MAX;
    with_shape<X>(p.gradients, [&](auto size) {
      constexpr int SHAPE = decltype(size)::value;
      hipLaunchKernelGGL((attnres_ffn_gradients_kernel<X, SHAPE>), dim3(grid), dim3(Shape<SHAPE>::kAllThreads), 0, c.stream, g);
    });
    count = 0;
    grid = 0;
  };
  for (const int i : order) {
    if (results[i] == nullptr) continue;
    g.of[count] = of[i];
    g.b_rows[count] = i == 0;
    g.wide[count] = splits[i] > 1;
    g.scaled[count] = i != 2;
    g.first[count++] = grid;
    grid += static_cast<uint32_t>(round_up(workgroups(of[i]), 8));  // whole rounds of the XCDs
    if (!one_launch) launch();
  }
  launch();
  join_parts<Value<X>>(c, of, results);
}

// What attnres_hip_gated_ffn_plan tells, every gradient being wanted.
int64_t plan_entry(const Sizes& s, const FfnPlan& p, int pass, int entry) {
  const bool backward = pass != kForward;
  const int64_t outputs[3][2] = {{s.width, s.rows}, {s.width, 2 * p.hidden_pad}, {s.hidden, s.out_width}};
  const Cut& cut = backward ? p.gradients : p.out;
  const int shape = cut.shape();
  int64_t products[3] = {}, all = 0, joined = 0;  // workgroups
  const int count = backward ? 3 : p.few ? 0 : 1;
  for (int i = 0; i < count; ++i) {
    const int64_t a = backward ? outputs[i][0] : s.out_width, b = backward ? outputs[i][1] : s.rows;
    products[i] = tiles_of(a, cut.tile) * tiles_of(b, cut.tile) * cut.splits[i];
    all += products[i];
    if (cut.splits[i] > 1) joined += rows_of(backward && i == 1 ? 2 * s.hidden : b, tiles_of(a, kVec), 0).groups;
  }
  const bool one_launch = count == 1 || together(cut.tile, all);
  switch (entry) {
    case ATTNRES_FFN_GATE_TILE: return p.few || pass == kBackward ? 0 : p.gate.shape();
    case ATTNRES_FFN_SLOPE_TILE: return backward ? p.slope.shape() : 0;
    case ATTNRES_FFN_PRODUCT_TILE: return count == 0 ? 0 : shape;
    case ATTNRES_FFN_PRODUCT_LAUNCHES: return count == 0 ? 0 : one_launch ? 1 : 3;
    case ATTNRES_FFN_PRODUCT_PARTS: return count == 0 ? 0 : *std::max_element(cut.splits, cut.splits + count);
    case ATTNRES_FFN_OPERAND_PARTS: return p.single ? 0 : p.parts;
    default: break;
  }
  const auto threads = [](const Cut& of) {
    const auto shape_threads = [](auto known) { return static_cast<int64_t>(Shape<decltype(known)::value>::kAllThreads); };
    int64_t result = 0;
    if (of.tile == 256) return shape_threads(std::integral_constant<int, 256>{});
    with_shape<Single>(of, [&](auto known) { result = shape_threads(known); });
    return result;
  };
  int64_t packed = 0;
  const auto pack = [&](bool needed, int64_t rows, int64_t width) {
    if (needed) packed += rows_of(rows, width / kVec, 0).groups;
  };
  pack(p.pack_x, p.rows_pad, p.width_pad);
  pack(p.pack_gate_up, 2 * p.hidden_pad, p.width_pad);
  pack(p.pack_down, p.out_pad, p.hidden_pad);
  pack(p.pack_grad, p.rows_pad, p.out_pad);
  int64_t most = std::max(packed, joined) * kBlock;
  const auto product = [&](const Cut& of, int64_t workgroups) { most = std::max(most, workgroups * threads(of)); };
  if (!p.few && pass != kBackward) product(p.gate, tiles_of(p.hidden_pad, p.gate.tile / 2) * tiles_of(s.rows, p.gate.tile));
  if (backward) product(p.slope, tiles_of(p.hidden_pad, p.slope.tile) * tiles_of(p.rows_pad, p.slope.tile));
  for (int i = 0; i < count; ++i) product(cut, one_launch ? all + 3 * 8 : products[i] + 8);
  return most;
}

bool known_sizes(const Sizes& s) {
  return s.rows >= 0 && s.rows <= kMaxRows && s.width >= 1 && s.width <= ATTNRES_MAX_WIDTH && s.hidden >= 1 && s.hidden <= kMaxHidden &&
         s.out_width >= 1 && s.out_width <= ATTNRES_MAX_WIDTH && dtype_known(s.dtype) &&
         tiles_of(s.rows, kTile) * tiles_of(s.hidden, kTile / 2) <= kMaxTiles;
}

int check_sizes(const Sizes& s, int activation) {
  if (s.rows < 0 || s.rows > kMaxRows) return layer_error(ATTNRES_ERR_SHAPE, "rows=%lld outside 0..2^24", (long long)s.rows);
  if (s.width < 1 || s.width > ATTNRES_MAX_WIDTH || s.out_width < 1 || s.out_width > ATTNRES_MAX_WIDTH) {
    return layer_error(ATTNRES_ERR_SHAPE, "width=%lld or out_width=%lld outside 1..%d", (long long)s.width, (long long)s.out_width,
                       ATTNRES_MAX_WIDTH);
  }
  if (s.hidden < 1 || s.hidden > kMaxHidden) return layer_error(ATTNRES_ERR_SHAPE, "hidden=%lld outside 1..2^16", (long long)s.hidden);
  if (!dtype_known(s.dtype)) return layer_error(ATTNRES_ERR_SHAPE, "unknown dtype %d", s.dtype);
  if (!known_sizes(s)) return layer_error(ATTNRES_ERR_SHAPE, "rows x hidden outside 2^22 tiles of 256 x 128");
  if (activation != ATTNRES_SILU && activation != ATTNRES_GELU) return layer_error(ATTNRES_ERR_SCALAR, "unknown activation %d", activation);
  return ATTNRES_OK;
}

// Operands that are multiplied where they lie: whole 16-byte loads, 32-bit offsets.
int check_rows(const char* name, const void* x, int64_t stride, bool in_place, int64_t least, int64_t most) {
  if (x == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "%s is NULL", name);
  if (stride < 0) return layer_error(ATTNRES_ERR_STRIDE, "negative row stride of %s", name);
  if (in_place && ((reinterpret_cast<uintptr_t>(x) & 15u) != 0 || stride % 8 != 0 || stride < least || stride > most)) {
    return layer_error(ATTNRES_ERR_STRIDE, "rows of %s must start at multiples of 16 bytes, at most %lld elements apart", name,
                       (long long)most);
  }
  return ATTNRES_OK;
}

int check_call(const Call& c, const void* saved, int64_t workspace_bytes) {
  const FfnPlan& p = c.plan;
  const bool even = c.s.hidden == p.hidden_pad, wide = c.s.width == p.width_pad;
  if (const int status = check_rows("x", c.x, c.x_stride, wide, 0, kMaxStride)) return status;
  if (const int status = check_rows("gate_up", c.gate_up, c.gate_up_stride, wide && even, c.s.width,
                                    std::min(kMaxStride, kMaxSecond * 2 / dtype_size(c.s.dtype) / c.s.hidden))) {
    return status;
  }
  if (const int status = check_rows("down", c.down, c.down_stride, even, c.s.hidden, kMaxStride)) return status;
  if (c.workspace == nullptr || workspace_bytes < p.bytes) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.bytes);
  }
  if (((reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(c.workspace)) & 15u) != 0) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "saved and workspace must start at multiples of 16 bytes");
  }
  return ATTNRES_OK;
}

}  // namespace
}  // namespace layers
}  // namespace attnres_hip

using namespace attnres_hip;
using namespace attnres_hip::layers;

extern "C" {

int64_t attnres_hip_gated_ffn_saved_bytes(int64_t rows, int64_t width, int64_t hidden, int64_t out_width, int dtype) {
  const Sizes s{rows, width, hidden, out_width, dtype};
  return known_sizes(s) ? saved_bytes(s) : -1;
}

int64_t attnres_hip_gated_ffn_workspace_bytes(int64_t rows, int64_t width, int64_t hidden, int64_t out_width, int dtype, int backward) {
  const Sizes s{rows, width, hidden, out_width, dtype};
  return known_sizes(s) && backward >= kForward && backward <= kBackwardAgain ? ffn_plan(s, backward).bytes : -1;
}

int64_t attnres_hip_gated_ffn_plan(int64_t rows, int64_t width, int64_t hidden, int64_t out_width, int dtype, int backward, int entry) {
  const Sizes s{rows, width, hidden, out_width, dtype};
  if (!known_sizes(s) || rows == 0 || backward < kForward || backward > kBackwardAgain || entry < 0 || entry > ATTNRES_FFN_THREADS) return -1;
  return plan_entry(s, ffn_plan(s, backward), backward, entry);
}

int attnres_hip_gated_ffn_forward(const void* x, int64_t x_stride, const void* gate_up, int64_t gate_up_stride, const void* down,
                                  int64_t down_stride, int64_t rows, int64_t width, int64_t hidden, int64_t out_width, int dtype,
                                  int activation, void* out, void* saved, void* workspace, int64_t workspace_bytes, void* stream) {
  const Sizes s{rows, width, hidden, out_width, dtype};
  if (const int status = check_sizes(s, activation)) return status;
  if (rows == 0) return ATTNRES_OK;
  const Call c{s, x, x_stride, gate_up, gate_up_stride, down, down_stride, activation, ffn_plan(s, kForward),
               static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
  if (const int status = check_call(c, saved, workspace_bytes)) return status;
  if (out == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "out is NULL");
  if (dtype == ATTNRES_BF16) ffn_forward<Bf16>(c, out, static_cast<char*>(saved));
  else if (dtype == ATTNRES_F16) ffn_forward<F16>(c, out, static_cast<char*>(saved));
  else if (c.plan.single) ffn_forward<Single>(c, out, static_cast<char*>(saved));
  else ffn_forward<float>(c, out, static_cast<char*>(saved));
  return layer_launch_status("gated feed-forward forward");
}

int attnres_hip_gated_ffn_backward(const void* grad_out, const void* x, int64_t x_stride, const void* gate_up, int64_t gate_up_stride,
                                   const void* down, int64_t down_stride, int64_t rows, int64_t width, int64_t hidden,
                                   int64_t out_width, int dtype, int activation, const void* saved, void* grad_x, void* grad_gate_up,
                                   void* grad_down, void* workspace, int64_t workspace_bytes, void* stream) {
  const Sizes s{rows, width, hidden, out_width, dtype};
  if (const int status = check_sizes(s, activation)) return status;
  if (rows == 0) return layer_error(ATTNRES_ERR_SHAPE, "no rows: the weights' gradients are zeros, which the caller writes");
  const Call c{s, x, x_stride, gate_up, gate_up_stride, down, down_stride, activation,
               ffn_plan(s, saved != nullptr ? kBackward : kBackwardAgain), static_cast<char*>(workspace),
               static_cast<hipStream_t>(stream)};
  if (const int status = check_call(c, saved, workspace_bytes)) return status;
  if (const int status = check_rows("grad_out", grad_out, out_width, !c.plan.pack_grad, 0, kMaxStride)) return status;
  if (grad_x == nullptr && grad_gate_up == nullptr && grad_down == nullptr) return ATTNRES_OK;
  const char* kept = static_cast<const char*>(saved);
  if (dtype == ATTNRES_BF16) ffn_backward<Bf16>(c, grad_out, kept, grad_x, grad_gate_up, grad_down);
  else if (dtype == ATTNRES_F16) ffn_backward<F16>(c, grad_out, kept, grad_x, grad_gate_up, grad_down);
  else if (c.plan.single) ffn_backward<Single>(c, grad_out, kept, grad_x, grad_gate_up, grad_down);
  else ffn_backward<float>(c, grad_out, kept, grad_x, grad_gate_up, grad_down);
  return layer_launch_status("gated feed-forward backward");
}

}  // extern "C"
