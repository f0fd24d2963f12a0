// attnres_loss.hip - softmax cross entropy of logits = H W^T over a vocabulary, for gfx950.
//
//   l[n, v] = <H_n, W_v>,  lse_n = log sum_v exp(l[n, v]),  loss_n = lse_n - l[n, t_n]
//   P[n, v] = g_n (exp(l[n, v] - lse_n) - [v = t_n]),  dH = P W,  dW = P^T H
//
// Bound by the matrix cores: three products of 2 N V D operations (the logits and two gradient products) against
// O(V D + N D) bytes.  The forward reduces the logits, per row and 128 columns, to a
// reference and a sum of powers above it, and keeps the powers for the backward (2 or 4 bytes each, up to
// kKeepBytes; of few rows the FP32 logits themselves), which makes P of them in one pass, for one piece of the vocabulary at a time.
// Without kept powers the backward multiplies again, four products in all.  Forward and backward, kept / again: 16384 x 131072 x 2048 BF16
// 22.5 / 27.9 ms, 2048 x 32768 x 1024 BF16 0.45 / 0.54, 4096 x 32768 x 1024 FP32 2.45 / 3.04.
//
// Rows whose target is ignored are left out before anything is multiplied: the rows that count are
// packed together (in order, the row length padded with zeros to whole stages), so ignored
// rows cost nothing and what they hold (NaN, infinities) reaches nothing.
//
// Operands are 16 bits wide.  BF16 and FP16 inputs are multiplied as they are.  FP32
// inputs are scaled by a power of two to just under 2^15 and written as the sum of two FP16 numbers, hi +
// lo, and a product is hi hi + hi lo + lo hi.  The pair has 24 bits for all within 2^-16 of the largest; it ends at 2^-40 of
// that, so smaller numbers have a bit less for every further power of two (15 at 2^-25).  What is left out, lo lo, is below 2^-24 of the product, like FP32's own
// rounding.  Three FP16 products take 0.78 ms (16384 x 8192 x 1024, logits) where FP32 matrix instructions, at a
// sixteenth of the FP16 rate, take 1.8 at the rate of a large library product.
// P is rounded to the operands' type (BF16), or, for FP16 and FP32 inputs, without its row's power of two (RowPowers) scaled by
// 2^14 and written as one or two FP16 numbers, so that probabilities down to 2^-28 are normal numbers.  For BF16
// inputs this is the gradients' largest error beside their own rounding: 0.0019 to 0.0026 relative, root mean square, for both
// together, 0.0017 for the outputs' rounding alone.  P in FP16 would need W in FP16 as well, another copy of it.

#include "attnres_layers.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

constexpr int kTile = 256;     // rows and columns of a workgroup's tile
constexpr int kWaves = 8;      // of 128 x 64 outputs, two per SIMD
constexpr int kThreads = 64 * kWaves;
constexpr int kDown = 8;       // 16 x 16 tiles of a wavefront: down (A) and across (B)
constexpr int kAcross = 4;
constexpr int kDepth = 32;     // of a stage of a tile's operands in LDS
constexpr int kStages = 4;     // in LDS: one that is multiplied, three on their way
constexpr int kLoads = 2;      // per wavefront, operand and stage: 1 KB each
constexpr int kOperand = kTile * kDepth;  // elements of one operand's stage
constexpr float kProbabilityScale = 16384.0f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define ATTNRES_LDS __attribute__((address_space(3)))
#define ATTNRES_GLOBAL __attribute__((address_space(1)))

__host__ __device__ inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// What the forward leaves for the backward: a header, then per packed row the (reference,
// 1 / sum of powers above it) of its logits, its source row and its target, and per
// source row its packed one (or -1).
struct Header {
  int32_t count;      // packed rows
  float scale[2];     // of H and W (FP32 inputs; else 1)
  uint32_t amax[2];   // their largest finite magnitudes, as bits
};

// With `keep` also the (reference, sum) of every row and 128 columns, the powers themselves and, where those are rounded to
// FP16, the target's logit of every packed row.
struct Saved {
  Header* header;
  f32x2* stats;
  int32_t* index;
  int32_t* packed;
  int32_t* target;
  f32x2* sums;  // [columns / 128][row_tiles]
  float* target_logit;  // [row_tiles]
  void* powers; // [row_tiles][vocabulary, padded]
};

constexpr int64_t kHeaderBytes = 256;

// ------------------------------------------------------------- matrix product
// out[b][a] = sum_k A[a][k] B[b][k] over a tile of 256 x 256: A's index is the contiguous
// one of the output.  An operand lies either as rows of k (ROWS: the row is contiguous in k) or as
// columns (row k holds all of the operand's entries).  Both go to LDS as they lie, 16 bytes
// per lane straight from memory; a column operand's fragments are transposed on the way
// from LDS (ds_read_b64_tr_b16).  16-byte slots are permuted within an LDS row so that the lanes which
// LDS serves together meet every bank once: slot = chunk ^ (-(row / 4) % 4) for rows of k (64 bytes; lanes 0-3,
// 12-15, 20-23 and 24-27 go together), chunk ^ (4 (k % 4) + 2 (k / 8 % 2)) for columns (512 bytes).
// 16 x 16 x 32 matrix instructions: the chip is limited by power here (1.7 of 2.4 GHz), and on registers alone
// these reach 2.2 PFLOP/s, 32 x 32 x 16 ones 2.0.  Measured, 16384 x 16384 x 2048: dW (both operands transposed) 785-836 us (1.36
// PFLOP/s), dH with its FP32 sums over the pieces 830-907 (1.25), logits 1.13-1.25 with their reduction.  Five LDS stages, other depths and orders of loads, and
// wave priorities were no faster.

struct Operand {
  const uint16_t* part[2];  // hi, lo
  int64_t ld;
  int64_t entries;          // readable entries (rows: clamped row; columns: multiple of 8)
  int64_t depth;            // readable k of a column operand
};

struct Product {
  Operand a, b;
  const int32_t* count;  // live packed rows
  int64_t depth;         // k of the whole product, of all splits; operands hold zeros up to a whole stage
  int depth_is_count;    // depth: the packed rows
  int tiles_a, tiles_b, splits;
};

__device__ __forceinline__ int row_swizzle(int row) { return -(row >> 2) & 3; }
__device__ __forceinline__ int column_swizzle(int k) { return (k & 3) << 2 | (k >> 3 & 1) << 1; }

template <bool ROWS>
struct Loader {
  uint32_t offset[kLoads];  // bytes from the stage's origin; columns: of the chunk alone
  int row;                  // columns: k of the first load
  __device__ __forceinline__ void init(const Operand& o, int64_t entry0, int wave, int lane) {
    row = wave * kLoads * 2 + lane / 32;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if constexpr (ROWS) {
        const int r = (wave * kLoads + j) * 16 + lane / 4;
        const int64_t left = o.entries - 1 - entry0;
        const int64_t at = r < left ? r : left;
        offset[j] = static_cast<uint32_t>((at * o.ld + ((lane % 4) ^ row_swizzle(r)) * 8) * 2);
      } else {
        const int chunk = (lane % 32) ^ column_swizzle(row + j * 2);
        const int64_t left = o.entries - 8 - entry0;
        const int64_t at = chunk * 8 < left ? chunk * 8 : left;
        offset[j] = static_cast<uint32_t>(at * 2);
      }
    }
  }
  // Offsets of a stage; left: k's of it that a column operand holds, less one.
  __device__ __forceinline__ void offsets(const Operand& o, int left, uint32_t (&at)[kLoads]) const {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      at[j] = offset[j];
      if constexpr (!ROWS) at[j] += static_cast<uint32_t>(min(row + j * 2, left)) * static_cast<uint32_t>(o.ld * 2);
    }
  }
};

// A 1-KB load into LDS byte `lds` from `base` (scalar) and `at` bytes on, 16 bytes per lane.  Written out,
// since the compiler makes transposing LDS reads wait for every load into LDS that it knows of; what has to
// have landed is waited for in landed().  The address registers are read when the load is issued, and
// nothing comes back in registers.
__device__ __forceinline__ void load_lds(const char* base, uint32_t at, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(at), "s"(base) : "m0");
}

// The LDS byte of a pointer into LDS.
__device__ __forceinline__ uint32_t lds_byte(const uint16_t* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const ATTNRES_LDS uint16_t*)p));
}

// Fragments of 16 entries and a stage's 32 k's: lane l holds entry l % 16, k = 8 (l / 16) + 0..7.
template <bool ROWS>
struct Reader {
  uint32_t at;      // the lane's byte of a stage; columns: of its row of k
  uint32_t column;  // columns: the lane's byte in that row, before the fragment's number is permuted in
  __device__ __forceinline__ void init(int entry, int lane) {
    const int group = lane / 16, j = lane % 16;
    if constexpr (ROWS) {
      at = static_cast<uint32_t>((entry + j) * kDepth + (group ^ row_swizzle(j)) * 8) * 2;
      column = 0;
    } else {
      // 16 lanes read 4 k's of 16 entries and get one entry's 4 k's each
      const int k = group * 8 + j / 4;
      const int chunk = entry / 8 + j % 4 / 2;  // the fragment's number is a part of its low four bits
      at = static_cast<uint32_t>(k * kTile + chunk / 16 * 128) * 2;
      column = static_cast<uint32_t>((chunk % 16 ^ column_swizzle(k)) * 8 + j % 2 * 4) * 2;
    }
  }
  __device__ __forceinline__ s16x8 read(uint32_t stage, int f) const {
    if constexpr (ROWS) {
      return *(ATTNRES_LDS const s16x8*)(stage + at + f * 16 * kDepth * 2);
    } else {
      const uint32_t from = stage + at + (column ^ (f * 32u));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTNRES_LDS s16x4*)(from));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTNRES_LDS s16x4*)(from + 4 * kTile * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

template <class T>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (std::is_same_v<T, Bf16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64)); }

struct TileAt {
  int a, b, split;
};

// Workgroup to tile: workgroups go round the 8 XCDs in turn, so each XCD takes one contiguous part of
// the tiles' order, in which 4 tiles of B by all of A's follow each other: the 32 tiles that run on an
// XCD at a time share 4 + 8 operand stripes in its L2.  tiles_b: those with rows that count, so that the XCDs
// get equal shares of them; false for the workgroups past the last tile.
__device__ __forceinline__ bool tile_at(const Product& p, int tiles_b, TileAt* tile) {
  const int total = p.tiles_a * tiles_b * p.splits;
  const int id = blockIdx.x;
  if (id >= total) return false;
  const int q = total / 8, r = total % 8, xcd = id % 8, i = id / 8;
  int at = xcd < r ? xcd * (q + 1) + i : r * (q + 1) + (xcd - r) * q + i;
  const int split = at / (p.tiles_a * tiles_b);
  at -= split * p.tiles_a * tiles_b;
  constexpr int kGroup = 4;
  const int group = at / (kGroup * p.tiles_a);
  const int size = min(kGroup, tiles_b - group * kGroup);
  at -= group * kGroup * p.tiles_a;
  *tile = {at / size, group * kGroup + at % size, split};
  return true;
}

// [16 entries of A][16 entries of B]; lane l, register e: entry 4 (l / 16) + e of A, l % 16 of B.
using Accumulators = f32x4[kDown][kAcross];

// A pointer that every lane holds, in scalar registers, and opaque from here on.
__device__ __forceinline__ const char* scalar(const char* p) {
  const uint64_t bits = reinterpret_cast<uint64_t>(p);
  uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bits)));
  uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bits >> 32)));
  asm volatile("" : "+s"(lo), "+s"(hi));
  return reinterpret_cast<const char*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// This wavefront's reads from LDS are done and its loads of the next stage have landed, and so it is for every
// wavefront (a barrier alone waits for neither).  Loads arrive in order: with `more`, those of
// the stages after the next one may still be on their way.
__device__ __forceinline__ void landed(bool more) {
  if (more) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"((kStages - 2) * 2 * kLoads) : "memory");
  } else {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The stages of a tile's split; none where there are fewer stages than splits.
struct Stages {
  int first, count;
};
__device__ __forceinline__ Stages stages_of(const Product& p, int split) {
  const int64_t depth = p.depth_is_count ? *p.count : p.depth;
  const int64_t all = (depth + kDepth - 1) / kDepth;
  const int first = static_cast<int>(all * split / p.splits);
  return {__builtin_amdgcn_readfirstlane(first),
          __builtin_amdgcn_readfirstlane(static_cast<int>(all * (split + 1) / p.splits) - first)};
}

// The sum of a tile over its split's k's (at least one stage); SEGMENTS 3: hi hi + hi lo + lo hi.
template <class T, int SEGMENTS, bool A_ROWS, bool B_ROWS>
__device__ __forceinline__ void multiply(const Product& p, const TileAt& tile, const Stages& range, uint16_t* lds, Accumulators& acc) {
  const int wave = wave_index(), lane = threadIdx.x % 64;
#pragma unroll
  for (int i = 0; i < kDown; ++i) {
#pragma unroll
    for (int j = 0; j < kAcross; ++j) acc[i][j] = f32x4{};
  }
  const int first = range.first, stages = range.count;
  const int64_t a0 = static_cast<int64_t>(tile.a) * kTile, b0 = static_cast<int64_t>(tile.b) * kTile;
  Loader<A_ROWS> load_a;
  Loader<B_ROWS> load_b;
  load_a.init(p.a, a0, wave, lane);
  load_b.init(p.b, b0, wave, lane);
  // bytes from the operand's start to the tile, and from a stage to the next
  const int64_t origin_a = (A_ROWS ? a0 * p.a.ld : a0) * 2, origin_b = (B_ROWS ? b0 * p.b.ld : b0) * 2;
  const int64_t next_a = (A_ROWS ? 1 : p.a.ld) * kDepth * 2, next_b = (B_ROWS ? 1 : p.b.ld) * kDepth * 2;
  int segment = 0, stage = 0;  // of the next load
  // one scalar base per half stage and 32-bit offsets
  const auto base_a = [&] {
    return scalar(reinterpret_cast<const char*>(p.a.part[SEGMENTS == 3 && segment == 2]) + origin_a + (first + stage) * next_a);
  };
  const auto base_b = [&] {
    return scalar(reinterpret_cast<const char*>(p.b.part[SEGMENTS == 3 && segment == 1]) + origin_b + (first + stage) * next_b);
  };
  // k's left in a column operand from this stage on, less one
  const auto left = [&](const Operand& o) {
    return __builtin_amdgcn_readfirstlane(static_cast<int>(o.depth - 1 - static_cast<int64_t>(first + stage) * kDepth));
  };
  const auto loaded = [&] {
    if (++stage == stages) stage = 0, ++segment;
  };
  const uint32_t lds0 = lds_byte(lds);
  const auto buffer = [&](int s) { return lds0 + (s % kStages) * (2 * kOperand * 2); };
  constexpr uint32_t kB = kOperand * 2;  // B's operand in a stage, bytes
  const uint32_t slot = wave * (kLoads * 1024);
  Reader<A_ROWS> read_a;
  Reader<B_ROWS> read_b;
  read_a.init((wave % 2) * 128, lane);
  read_b.init((wave / 2) * (16 * kAcross), lane);
  // A stage in two steps, the upper and the lower half of A's fragments, with all of B's.
  constexpr int kHalf = kDown / 2;
  using FragmentsA = s16x8[kHalf];
  using FragmentsB = s16x8[kAcross];
  // One step: the matrix instructions on (a, b), between them the reads of the next step's fragments, in the
  // order of their use, and the loads.
  const auto step = [&](auto lower, const FragmentsA& a, const FragmentsB& b, auto read, auto load) {
    constexpr int kFirst = decltype(lower)::value ? kHalf : 0;
#pragma unroll
    for (int m = 0; m < kHalf * kAcross; ++m) {
      f32x4& c = acc[kFirst + m / kAcross][m % kAcross];
      c = mfma<T>(a[m / kAcross], b[m % kAcross], c);
      if (m % 2 == 0) read(m / 2);
      if (m % 8 == 1) load(m / 8);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  FragmentsA upper, lower;
  FragmentsB b_even, b_odd;  // of even and odd stages
  // Reads of a step, eight at most: the lower half of the stage, or the next stage's upper half and B.
  const auto read_lower = [&](uint32_t from) {
    return [&, from](int r) {
      if (r < kHalf) lower[r] = read_a.read(from, kHalf + r);
    };
  };
  const auto read_next = [&](uint32_t from, FragmentsB& b) {
    return [&, from](int r) {
      if (r == 0) upper[0] = read_a.read(from, 0);
      else if (r <= kAcross) b[r - 1] = read_b.read(from + kB, r - 1);
      else upper[r - kAcross] = read_a.read(from, r - kAcross);
    };
  };
  static_assert(kHalf + kAcross == 8 && kHalf * kAcross == 16, "eight reads, one per two matrix instructions");
  const auto nothing = [](int) {};
  const int total = stages * SEGMENTS;
  uint32_t at[kLoads];
  for (int s = 0; s < kStages && s < total; ++s) {
    const char *a = base_a(), *b = base_b();
    load_a.offsets(p.a, left(p.a), at);
    for (int j = 0; j < kLoads; ++j) load_lds(a, at[j], buffer(s) + slot + j * 1024);
    load_b.offsets(p.b, left(p.b), at);
    for (int j = 0; j < kLoads; ++j) load_lds(b, at[j], buffer(s) + kB + slot + j * 1024);
    loaded();
  }
  landed(total >= kStages);
  const auto read_first = read_next(lds0, b_even);
#pragma unroll
  for (int r = 0; r < 8; ++r) read_first(r);
  step(std::false_type{}, upper, b_even, read_lower(lds0), nothing);
  landed(total >= kStages);
  // A stage's lower step and the next one's upper step make a trip.  Loads go to the buffer whose stage is
  // finished but for fragments in registers: every wavefront has passed landed() since it read them.
  int s = 1;
  const auto trip = [&](FragmentsB& now, FragmentsB& next) {
    const uint32_t to = buffer(s + kStages - 1) + slot;
    const char* a = base_a();
    load_a.offsets(p.a, left(p.a), at);
    step(std::true_type{}, lower, now, read_next(buffer(s), next), [&](int j) { load_lds(a, at[j], to + j * 1024); });
    const char* b = base_b();
    load_b.offsets(p.b, left(p.b), at);
    step(std::false_type{}, upper, next, read_lower(buffer(s)), [&](int j) { load_lds(b, at[j], to + kB + j * 1024); });
    loaded();
    landed(true);
    ++s;
  };
  const auto last_trip = [&](FragmentsB& now, FragmentsB& next) {  // nothing more to load
    step(std::true_type{}, lower, now, read_next(buffer(s), next), nothing);
    step(std::false_type{}, upper, next, read_lower(buffer(s)), nothing);
    landed(false);
    ++s;
  };
  while (s + kStages < total) {
    trip(b_even, b_odd);
    trip(b_odd, b_even);
  }
  // fewer than two trips with loads are left, then those without; after an odd number B's fragments change
  // their registers
  const auto swap = [&] {
#pragma unroll
    for (int j = 0; j < kAcross; ++j) b_even[j] = b_odd[j];
  };
  if (s + kStages - 1 < total) {
    trip(b_even, b_odd);
    swap();
  }
  while (s < total) {
    last_trip(b_even, b_odd);
    swap();
  }
  step(std::true_type{}, lower, b_even, nothing, nothing);
  __syncthreads();  // LDS is free for the epilogue
}

// -------------------------------------------------------------------- logits

// Exponentials are powers of two above a reference c, an integer near the largest logit over ln 2, so that joining sums
// of different c's rounds nothing.  A logit over ln 2 is rounded before c is taken from it, the same wherever it is
// formed: of logits so large that c's neighbours are far apart, the largest is still c itself.
constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;

__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }

// A product that is rounded, not fused with what follows.
__device__ __forceinline__ float over_ln2(float x, float by = kLog2e) {
#pragma clang fp contract(off)
  return x * by;
}

// Joins two (reference, sum of powers above it).  A side without entries is (-inf, 0);
// a NaN sum stays NaN.
__device__ __forceinline__ f32x2 join(f32x2 x, f32x2 y) {
  const float top = fmaxf(x.x, y.x);
  if (top == -__builtin_inff()) return f32x2{top, x.y + y.y};
  return f32x2{top, x.y * power(x.x - top) + y.y * power(y.x - top)};
}

// Logits from the product of scaled operands: by the two powers of two in turn, the smaller
// first, so that neither step leaves FP32 where the logit itself does not.
struct Logit {
  float first = 1.0f, second = 1.0f;
  bool any;
  __device__ __forceinline__ explicit Logit(const Header* header) : any(header != nullptr) {
    if (!any) return;
    const float h = 1.0f / header->scale[0], w = 1.0f / header->scale[1];
    first = fminf(h, w);
    second = fmaxf(h, w);
  }
  __device__ __forceinline__ float operator()(float x) const { return any ? x * first * second : x; }
  __device__ __forceinline__ float above(float x, float c) const {  // log2 of the power
    return over_ln2(any ? x * first : x, second * kLog2e) - c;
  }
};

// What powers are kept in for the backward.  BF16 operands: FP16, whose rounding of 2^-11 adds an eighth to
// that of the probabilities to BF16.  At the target that would be 2^-11 of p where P is p - 1, far more than P itself for a
// token that is all but certain, so there the backward takes the power from the target's own logit, kept in FP32.
// Others: FP32, as FP16 would double the rounding of the probabilities to FP16.
template <class T>
using Power = std::conditional_t<std::is_same_v<T, Bf16>, F16, float>;

// The reference for logits of at most `top`.  Powers that are kept in FP16 are shifted up by 15, so that those down
// to 2^-29 of the largest are normal numbers; not where the reference is no exact integer any more.
constexpr float kShift = 15.0f;
template <class T>
__device__ __forceinline__ float reference(float top) {
  const float c = rintf(over_ln2(top));
  return std::is_same_v<Power<T>, F16> && fabsf(c) < 8388608.0f ? c - kShift : c;
}

struct LogitArgs {
  Product product;  // A: W (vocabulary), B: H (packed rows)
  const Header* header;
  const int32_t* target;
  int64_t vocab;
  int64_t first;      // of the piece's columns
  int64_t row_tiles;  // packed rows, padded
  // forward
  f32x2* sums;          // [columns / 128][row_tiles] (reference, sum of powers above it)
  float* target_logit;  // [row_tiles]; in the backward where the powers are FP16
  void* powers;         // [row_tiles][powers_ld], or nullptr: not kept
  int64_t powers_ld;
  // backward
  const f32x2* stats;
  const float* row_scale;  // [row_tiles] upstream gradient per packed row, scaled; 0 past the last
  uint16_t* p[2];          // [row_tiles][p_ld]
  int64_t p_ld;
};

// 16-byte slot of a staged output row of 512 bytes: a permutation per row, so that 32 lanes
// writing one chunk of 32 rows meet 32 different slots.
__device__ __forceinline__ int staged(int row, int chunk) { return row * 32 + (chunk ^ (row & 31)); }

// Forward: (reference, sum) of a tile's two times 128 logits per row, and the target's logit.  KEEP: the powers too, staged
// in LDS and stored 512 bytes of a row at a time (256 where they are FP32, in two rounds).  The reduction is vector
// work that the next tile's products do not cover: 16384 x 131072 x 2048 BF16 6.9 ms, with kept powers 7.8.
template <class T, int SEGMENTS, bool KEEP>
__global__ void __launch_bounds__(kThreads) attnres_loss_logits_kernel(LogitArgs g) {
  __shared__ __align__(16) uint16_t lds[kStages * 2 * kOperand];
  const int count = __builtin_amdgcn_readfirstlane(*g.product.count);
  TileAt tile;
  if (!tile_at(g.product, (count + kTile - 1) / kTile, &tile)) return;
  Accumulators acc;
  multiply<T, SEGMENTS, true, true>(g.product, tile, stages_of(g.product, 0), lds, acc);
  const int wave = wave_index(), lane = threadIdx.x % 64;
  const Logit logit(SEGMENTS == 3 ? g.header : nullptr);
  const int64_t v0 = static_cast<int64_t>(tile.a) * kTile + (wave % 2) * 128;
  const int limit = __builtin_amdgcn_readfirstlane(static_cast<int>(g.vocab - v0 < 128 ? g.vocab - v0 : 128));
  float tops[kAcross], sums[kAcross];  // from a round to the next
  // The powers of 16 kDown / kRounds entries at a time, as many as LDS holds.
  using E = Power<T>;
  constexpr int kRounds = KEEP ? sizeof(E) / 2 : 1;
  constexpr int kPart = kDown / kRounds;
  // ENDS: the vocabulary ends in this half of the tile
  const auto reduce = [&](auto ends, auto at) {
    constexpr bool ENDS = decltype(ends)::value;
    constexpr int round = decltype(at)::value;
    const int last = limit - 4 * (lane / 16);  // entries below it count
#pragma unroll
    for (int j = 0; j < kAcross; ++j) {
      const int column = (wave / 2) * (16 * kAcross) + j * 16 + lane % 16;
      float top, sum = 0.0f;
      if constexpr (round == 0) {
        const int row = tile.b * kTile + column;
        const int64_t from_v0 = g.target[min(row, count - 1)] - v0;
        const int rel = row < count && from_v0 >= 0 && from_v0 < 128 ? static_cast<int>(from_v0) : -1;
        float x = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < kDown; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x = fmaxf(x, !ENDS || i * 16 + e < last ? acc[i][j][e] : -__builtin_inff());
        }
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        top = reference<T>(logit(fmaxf(x, __shfl_xor(x, 32, 64))));
        if (__any(rel >= 0)) {
          float own = 0.0f;
#pragma unroll
          for (int i = 0; i < kDown; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e) own = i * 16 + e == rel - 4 * (lane / 16) ? acc[i][j][e] : own;
          }
          if (rel >= 0 && (rel >> 2 & 3) == lane / 16) g.target_logit[row] = logit(own);
        }
      } else {
        top = tops[j];
        sum = sums[j];
      }
      const float from = top == -__builtin_inff() ? 0.0f : top;  // nothing but NaN, or nothing at all
#pragma unroll
      for (int i = 0; i < kPart; ++i) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = power(logit.above(acc[round * kPart + i][j][e], from));
          if (ENDS) x[e] = (round * kPart + i) * 16 + e < last ? x[e] : 0.0f;
          sum += x[e];
        }
        if constexpr (KEEP && std::is_same_v<E, F16>) {
          const int chunk = (wave % 2) * 16 + i * 2 + lane / 32;
          *reinterpret_cast<uint64_t*>(lds + staged(column, chunk) * 8 + (lane / 16 % 2) * 4) =
              static_cast<uint64_t>(pack2<F16>(x[2], x[3])) << 32 | pack2<F16>(x[0], x[1]);
        } else if constexpr (KEEP) {
          *reinterpret_cast<f32x4*>(lds + staged(column, (wave % 2) * 16 + i * 4 + lane / 16) * 8) = f32x4{x[0], x[1], x[2], x[3]};
        }
        if (KEEP && i % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // a few outputs at a time: no registers to spill
      }
      if constexpr (round < kRounds - 1) {
        tops[j] = top;
        sums[j] = sum;
      } else {
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lane < 16) {
          g.sums[(static_cast<int64_t>(tile.a) * 2 + wave % 2) * g.row_tiles + tile.b * kTile + column] = f32x2{top, sum};
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto pass = [&](auto at) {
    constexpr int round = decltype(at)::value;
    if (limit < 128) {
      reduce(std::true_type{}, at);
    } else {
      reduce(std::false_type{}, at);
    }
    if constexpr (KEEP) {
      __syncthreads();
      constexpr int kChunk = 16 / sizeof(E);
      for (int k = threadIdx.x; k < kTile * 32; k += kThreads) {
        const int column = k / 32, chunk = k % 32;
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds + staged(column, chunk) * 8);
        const int entry = chunk / 16 * 128 + round * 16 * kPart + chunk % 16 * kChunk;
        E* to = static_cast<E*>(g.powers) + (static_cast<int64_t>(tile.b) * kTile + column) * g.powers_ld +
                static_cast<int64_t>(tile.a) * kTile + entry;
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to));
      }
    }
  };
  pass(std::integral_constant<int, 0>{});
  if constexpr (kRounds == 2) {
    __syncthreads();
    pass(std::integral_constant<int, 1>{});
  }
}

// Backward of kept powers: P of a piece's columns, read from the powers and written as operands, both past the caches.
// 16 rows of 512 columns per workgroup, 8 columns per thread and row.  Memory bound: 16384 x 16384 of FP16 to BF16 (1.07
// GB) 160 us, 6.7 TB/s.
constexpr int kScaleRows = 16, kScaleColumns = 64 * kVec;

template <class E, class T, int PARTS>
__global__ void __launch_bounds__(kBlock) attnres_loss_rescale_kernel(LogitArgs g, int64_t columns, int column_blocks) {
  const int count = *g.product.count;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / column_blocks) * kScaleRows + threadIdx.x / 64;
  const int64_t column = static_cast<int64_t>(blockIdx.x % column_blocks) * kScaleColumns + threadIdx.x % 64 * kVec;
  if (row0 >= round_up(count, kTile) || column >= columns) return;
  constexpr int kRounds = kScaleRows / (kBlock / 64);
  const int64_t v = g.first + column;
  const E* powers = static_cast<const E*>(g.powers);
  Chunk<E> chunk[kRounds];
  float factor[kRounds], by[kRounds], own[kRounds];
  int64_t rel[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t row = row0 + k * (kBlock / 64);
    chunk[k].load_past(powers + row * g.powers_ld + v);
    const int64_t at = row < count ? row : count - 1;
    const f32x2 sum = g.sums[v / 128 * g.row_tiles + row], stats = g.stats[at];
    by[k] = g.row_scale[row];
    factor[k] = row < count ? power(sum.x - stats.x) * stats.y * by[k] : 0.0f;
    rel[k] = g.target[at] - v;
    // the target's entry of FP16 powers, from its logit as in the recomputed probabilities; 0 past the last row
    own[k] = 0.0f;
    if (std::is_same_v<E, F16> && row < count && rel[k] >= 0 && rel[k] < kVec) {
      own[k] = power(over_ln2(g.target_logit[row]) - stats.x) * (stats.y * by[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int64_t row = row0 + k * (kBlock / 64);
    float x[kVec];
    chunk[k].unpack(x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      x[e] = row < count ? x[e] * factor[k] : 0.0f;
      if (rel[k] == e) x[e] = (std::is_same_v<E, F16> ? own[k] : x[e]) - by[k];  // by: 0 past the last row
      if (PARTS == 2) asm("" : "+v"(x[e]));  // one rounding to hi, as in the recomputed probabilities
    }
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      u32x4 packed;
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) {
        packed[e] = pack2<T>(x[2 * e], x[2 * e + 1]);
        x[2 * e] -= to_f32(T{static_cast<uint16_t>(packed[e] & 0xffffu)});  // lo
        x[2 * e + 1] -= to_f32(T{static_cast<uint16_t>(packed[e] >> 16)});
      }
      __builtin_nontemporal_store(packed, reinterpret_cast<u32x4*>(g.p[part] + row * g.p_ld + column));
    }
  }
}

// Backward without kept powers: P of a tile, rounded to the operands' type; 893 us for 16384 x 16384 x 2048 BF16.
template <class T, int SEGMENTS>
__global__ void __launch_bounds__(kThreads) attnres_loss_probability_kernel(LogitArgs g) {
  __shared__ __align__(16) uint16_t lds[kStages * 2 * kOperand];
  const int count = __builtin_amdgcn_readfirstlane(*g.product.count);
  TileAt tile;
  if (!tile_at(g.product, (count + kTile - 1) / kTile, &tile)) return;
  Accumulators acc;
  multiply<T, SEGMENTS, true, true>(g.product, tile, stages_of(g.product, 0), lds, acc);
  const int wave = wave_index(), lane = threadIdx.x % 64;
  const Logit logit(SEGMENTS == 3 ? g.header : nullptr);
  const int64_t v0 = g.first + static_cast<int64_t>(tile.a) * kTile + (wave % 2) * 128;
  const int limit = __builtin_amdgcn_readfirstlane(static_cast<int>(g.vocab - v0 < 128 ? g.vocab - v0 : 128));
  constexpr int kParts = SEGMENTS == 3 ? 2 : 1;
  // With two parts, the columns of four wavefronts at a time: hi and lo of 128 rows are staged together.
  constexpr int kColumns = kTile / kParts;
  // SPECIAL: the vocabulary ends in these columns, or the target of one of the 16 rows is among them
  const auto stage = [&](auto special, int j, int base) {
    constexpr bool SPECIAL = decltype(special)::value;
    const int last = limit - 4 * (lane / 16);
    const int column = (wave / 2) * (16 * kAcross) + j * 16 + lane % 16;
    const int row = tile.b * kTile + column;
    const int at = min(row, count - 1);
    const int64_t from_v0 = g.target[at] - v0;
    const int rel = from_v0 >= 0 && from_v0 < 128 ? static_cast<int>(from_v0) - 4 * (lane / 16) : -128;
    // a row past the last one has zeros in H, so logits of 0, and a factor of 0
    const float c = row < count ? g.stats[at].x : 0.0f;
    const float by = g.row_scale[row], factor = row < count ? g.stats[at].y * by : 0.0f;
#pragma unroll
    for (int i = 0; i < kDown; ++i) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = power(logit.above(acc[i][j][e], c)) * factor;
        if (SPECIAL) {
          if (i * 16 + e == rel) x[e] -= by;
          if (i * 16 + e >= last) x[e] = 0.0f;
        }
        // the FP32 value itself: hi has to be the same number where it is stored and where lo
        // is what it leaves, and a product folded into one of the conversions rounds apart
        if (kParts == 2) asm("" : "+v"(x[e]));
      }
      const int chunk = (wave % 2) * 16 + i * 2 + lane / 32;
      uint16_t* to = lds + staged(column - base, chunk) * 8 + (lane / 16 % 2) * 4;
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
        const uint32_t packed[2] = {pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
        *reinterpret_cast<uint64_t*>(to + part * kColumns * kTile) = static_cast<uint64_t>(packed[1]) << 32 | packed[0];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] -= to_f32(T{static_cast<uint16_t>(packed[e / 2] >> (16 * (e % 2)))});  // lo
      }
      if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // a few outputs at a time: no registers to spill
    }
  };
  for (int base = 0; base < kTile; base += kColumns) {
    if (kParts == 1 || (wave / 2) * (16 * kAcross) / kColumns == base / kColumns) {
#pragma unroll
      for (int j = 0; j < kAcross; ++j) {
        const int64_t from_v0 = g.target[min(tile.b * kTile + (wave / 2) * (16 * kAcross) + j * 16 + lane % 16, count - 1)] - v0;
        if (limit < 128 || __any(from_v0 >= 0 && from_v0 < 128)) {
          stage(std::true_type{}, j, base);
        } else {
          stage(std::false_type{}, j, base);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int part = 0; part < kParts; ++part) {
      for (int k = threadIdx.x; k < kColumns * 32; k += kThreads) {
        const int column = k / 32, chunk = k % 32;
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds + part * kColumns * kTile + staged(column, chunk) * 8);
        // past the caches, where the operands of the tiles to come stay: 992 -> 910 us for 512 MB of P
        uint16_t* to = g.p[part] + (static_cast<int64_t>(tile.b) * kTile + base + column) * g.p_ld + tile.a * kTile + chunk * 8;
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(to));
      }
    }
    if (base + kColumns < kTile) __syncthreads();
  }
}

// ----------------------------------------------------------- gradient products

struct GradientArgs {
  Product product;
  const float* alpha;  // two factors of the output; nullptr: 1
  void* out;           // [splits][columns][ld]
  int64_t ld;
  int64_t split_stride;
  int64_t entries_a;   // valid contiguous entries
  int64_t entries_b;
  int add;             // FP32: add to what is there
  int live_only;       // entries of B past the packed rows are not needed
};

// A tile's outputs where there is nothing to multiply.
template <class OUT>
__device__ __forceinline__ void zero_tile(const GradientArgs& g, const TileAt& tile, OUT* out) {
  if (g.add) return;
  out += tile.split * g.split_stride;
  const int64_t a = static_cast<int64_t>(tile.a) * kTile + threadIdx.x, b0 = static_cast<int64_t>(tile.b) * kTile;
  if (a >= g.entries_a) return;
  for (int64_t b = b0; b < b0 + kTile && b < g.entries_b; ++b) out[b * g.ld + a] = from_f32<OUT>(0.0f);
}

// dH (A: W by columns, B: P by rows) and dW (A: H by columns, B: P by columns).  OUT float:
// FP32 partial sums or an FP32 gradient; else the 16-bit gradient itself.  dH is summed over the pieces in FP32, in order.
template <class T, class OUT, int SEGMENTS, bool B_ROWS>
__global__ void __launch_bounds__(kThreads) attnres_loss_gradient_kernel(GradientArgs g) {
  __shared__ __align__(16) uint16_t lds[kStages * 2 * kOperand];
  const int live = (__builtin_amdgcn_readfirstlane(*g.product.count) + kTile - 1) / kTile;
  TileAt tile;
  if (!tile_at(g.product, g.live_only ? live : g.product.tiles_b, &tile)) return;
  const Stages stages = stages_of(g.product, tile.split);
  if (stages.count == 0) return zero_tile(g, tile, static_cast<OUT*>(g.out));
  Accumulators acc;
  multiply<T, SEGMENTS, false, B_ROWS>(g.product, tile, stages, lds, acc);
  const int wave = wave_index(), lane = threadIdx.x % 64;
  const float by = g.alpha != nullptr ? g.alpha[0] : 1.0f, unscale = g.alpha != nullptr ? g.alpha[1] : 1.0f;
  OUT* out = static_cast<OUT*>(g.out) + tile.split * g.split_stride;
  const int64_t a0 = static_cast<int64_t>(tile.a) * kTile, b0 = static_cast<int64_t>(tile.b) * kTile;
  constexpr bool kWide = std::is_same_v<OUT, float>;
  constexpr int kRounds = kWide ? 2 : 1;    // 512-byte rows: 128 FP32 or 256 16-bit outputs
  constexpr int kChunk = kWide ? 4 : 8;     // outputs per 16 bytes
#pragma unroll
  for (int round = 0; round < kRounds; ++round) {
    if (!kWide || wave % 2 == round) {
#pragma unroll
      for (int j = 0; j < kAcross; ++j) {
        const int column = (wave / 2) * (16 * kAcross) + j * 16 + lane % 16;
#pragma unroll
        for (int i = 0; i < kDown; ++i) {
          const f32x4 x = acc[i][j] * by * unscale;
          if constexpr (kWide) {
            *reinterpret_cast<f32x4*>(lds + staged(column, i * 4 + lane / 16) * 8) = x;
          } else {
            const int chunk = (wave % 2) * 16 + i * 2 + lane / 32;
            *reinterpret_cast<uint64_t*>(lds + staged(column, chunk) * 8 + (lane / 16 % 2) * 4) =
                static_cast<uint64_t>(pack2<OUT>(x[2], x[3])) << 32 | pack2<OUT>(x[0], x[1]);
          }
          if (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // a few outputs at a time: no registers to spill
        }
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < kTile * 32; k += kThreads) {
      const int column = k / 32, chunk = k % 32;
      const int64_t a = a0 + round * 128 + chunk * kChunk, b = b0 + column;
      if (b >= g.entries_b || a >= g.entries_a) continue;
      OUT* to = out + b * g.ld + a;
      const uint16_t* from = lds + staged(column, chunk) * 8;
      if constexpr (kWide) {
        f32x4 x = *reinterpret_cast<const f32x4*>(from);
        if (a + kChunk <= g.entries_a) {
          if (g.add) x += reinterpret_cast<const Raw32*>(to)->v;
          reinterpret_cast<Raw32*>(to)->v = x;
        } else {
          for (int e = 0; a + e < g.entries_a; ++e) to[e] = g.add ? to[e] + x[e] : x[e];
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

// ------------------------------------------------------------------ small passes

// One workgroup: the rows whose target counts, in order, eight rounds of 1024 rows at a time.  A target outside
// the vocabulary is marked -1 (the row's loss and gradients become NaN).
constexpr int kScanThreads = 1024;
constexpr int kScanRounds = 8;
constexpr int kScanWaves = kScanThreads / 64;

__global__ void __launch_bounds__(kScanThreads) attnres_loss_rows_kernel(const void* targets, int target_bytes, int64_t rows, int64_t vocab,
                                                                         int64_t ignore_index, Saved s) {
  __shared__ int before[kScanRounds * kScanWaves + 1];  // rows that count before a round's wavefront
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  int base = 0;
  for (int64_t r0 = 0; r0 < rows; r0 += kScanThreads * kScanRounds) {
    int64_t target[kScanRounds];
#pragma unroll
    for (int k = 0; k < kScanRounds; ++k) {
      const int64_t row = min(r0 + k * kScanThreads + threadIdx.x, rows - 1);
      target[k] = target_bytes == 8 ? static_cast<const int64_t*>(targets)[row] : static_cast<const int32_t*>(targets)[row];
    }
    uint64_t counts[kScanRounds];
#pragma unroll
    for (int k = 0; k < kScanRounds; ++k) {
      counts[k] = __ballot(r0 + k * kScanThreads + threadIdx.x < rows && target[k] != ignore_index);
      if (lane == 0) before[k * kScanWaves + wave] = __popcll(counts[k]);
    }
    __syncthreads();
    if (wave == 0) {  // two entries per lane
      static_assert(kScanRounds * kScanWaves == 128, "two counts per lane");
      const int x = before[2 * lane], y = before[2 * lane + 1];
      int scan = x + y;
#pragma unroll
      for (int step = 1; step < 64; step <<= 1) {
        const int other = __shfl_up(scan, step, 64);
        scan += lane >= step ? other : 0;
      }
      before[2 * lane] = scan - x - y;
      before[2 * lane + 1] = scan - y;
      if (lane == 63) before[128] = scan;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kScanRounds; ++k) {
      const int64_t row = r0 + k * kScanThreads + threadIdx.x;
      const bool live = counts[k] >> lane & 1;
      const int at = base + before[k * kScanWaves + wave] + __popcll(counts[k] & ((uint64_t{1} << lane) - 1));
      if (row < rows) s.packed[row] = live ? at : -1;
      if (live) {
        s.index[at] = static_cast<int32_t>(row);
        s.target[at] = target[k] >= 0 && target[k] < vocab ? static_cast<int32_t>(target[k]) : -1;
      }
    }
    base += before[128];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    s.header->count = base;
    s.header->scale[0] = s.header->scale[1] = 1.0f;
    s.header->amax[0] = s.header->amax[1] = 0;
  }
}

// ------------------------------------------------------------------- few rows
// The forward of few rows (few_rows()) reads W once and is bound by that.  A workgroup takes 128 words, 32 to four
// wavefronts, which share the k's (so that all of W is asked for at once); where that would leave half of the units
// without work, 32 words to sixteen (3 rows of 3840 x 3510 FP16 32 -> 14 us; of 32767 x 1024 BF16 23 -> 32, as H is read
// oftener); W and H go straight to registers as
// they lie (any width and alignment; FP32 inputs by FP32 matrix instructions, which the few rows have time for),
// no packing: a row's logits are its own, so ignored rows are worked on and left out afterwards.  A
// lane holds 16 bytes of every 64 of its word or row; the order of the k's in a matrix instruction is of no
// account, as both operands share it.  16 rows of a 32768 x 1024 BF16 vocabulary (67 MB): 17.6 us, 3.8 TB/s (by 256 x
// 256 tiles 27 us and 8 for packing).
constexpr int kFewRows = 64;
constexpr int kFewBlock = 1024;
constexpr int kFewWords = 128;  // of a workgroup, at most

template <class X>
struct FewChunk {  // a lane's 16 of 64 k's, as they lie: 16 bytes of every 64
  static constexpr int kPieces = sizeof(X);
  static constexpr int kPiece = 16 / sizeof(X);
  u32x4 w[kPieces];
  __device__ __forceinline__ void load(const X* row, int k0, int group, int width) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int k = k0 + (i * 4 + group) * kPiece;
      if (k + kPiece <= width) {
        w[i] = reinterpret_cast<const Raw16*>(row + k)->v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (std::is_same_v<X, float>) {
            w[i][e] = k + e < width ? __float_as_uint(row[k + e]) : 0;
          } else {
            const uint32_t lo = k + 2 * e < width ? row[k + 2 * e].bits : 0;
            const uint32_t hi = k + 2 * e + 1 < width ? row[k + 2 * e + 1].bits : 0;
            w[i][e] = hi << 16 | lo;
          }
        }
      }
    }
  }
};

template <class X>
__device__ __forceinline__ f32x4 few_mfma(const FewChunk<X>& a, const FewChunk<X>& b, f32x4 c) {
  if constexpr (std::is_same_v<X, float>) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w[i][e]), __uint_as_float(b.w[i][e]), c, 0, 0, 0);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) c = mfma<X>(__builtin_bit_cast(s16x8, a.w[i]), __builtin_bit_cast(s16x8, b.w[i]), c);
  }
  return c;
}

template <class X>
struct FewArgs {
  const X* hidden;
  const X* weight;
  int64_t hidden_stride, weight_stride, vocab;
  int width, rows;
  const void* targets;
  int target_bytes;
  int64_t ignore_index;
  Saved saved;
  f32x2* sums;          // [workgroups][kFewRows]
  float* target_logit;  // [kFewRows]
  float* logits;        // [16 TILES][logits_ld], or nullptr: not kept
  int64_t logits_ld;
};

template <class X, int TILES, int WORDS>  // TILES of 16 rows
__global__ void __launch_bounds__(kFewBlock) attnres_loss_few_kernel(FewArgs<X> g) {
  constexpr int kGroups = WORDS / 32, kFewParts = kFewBlock / 64 / kGroups;
  __shared__ int target[kFewRows];  // -1: not known or ignored
  __shared__ f32x4 parts[kFewBlock / 64][64];
  __shared__ f32x2 meet[kGroups][TILES * 16];
  const int wave = wave_index(), lane = threadIdx.x % 64, group = lane / 16, entry = lane % 16;
  const int part = wave % kFewParts, words = wave / kFewParts;
  const int64_t v0 = static_cast<int64_t>(blockIdx.x) * WORDS + words * 32;
  const X* w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = g.weight + min(v0 + i * 16 + entry, g.vocab - 1) * g.weight_stride;
  constexpr int kSteps = sizeof(X) == 4 || TILES == 4 || WORDS == 32 ? 1 : 2;  // of 64 k's under way together
  constexpr int kSpan = kSteps * 64;
  FewChunk<X> next[kSteps][2];
  const auto fetch = [&](int k0) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) next[s][i].load(w[i], k0 + s * 64, group, g.width);
    }
  };
  fetch(part * kSpan);
  const X* h[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) h[t] = g.hidden + min(t * 16 + entry, g.rows - 1) * g.hidden_stride;
  if (g.targets == nullptr) {
    if (wave == 0) target[lane] = -1;
  } else if (wave == 0) {
    const int row = min(lane, g.rows - 1);
    const int64_t t = g.target_bytes == 8 ? static_cast<const int64_t*>(g.targets)[row] : static_cast<const int32_t*>(g.targets)[row];
    const bool counts = lane < g.rows && t != g.ignore_index;
    const int known = counts && t >= 0 && t < g.vocab ? static_cast<int>(t) : -1;
    target[lane] = known;
    if (blockIdx.x == 0) {
      const uint64_t all = __ballot(counts);
      const int at = __popcll(all & ((uint64_t{1} << lane) - 1));
      if (lane < g.rows) g.saved.packed[lane] = counts ? at : -1;
      if (counts) g.saved.index[at] = lane, g.saved.target[at] = known;
      if (lane == 0) *g.saved.header = Header{static_cast<int32_t>(__popcll(all)), {1.0f, 1.0f}, {0, 0}};
    }
  }
  f32x4 acc[2][TILES] = {};
  for (int k0 = part * kSpan; k0 < g.width; k0 += kFewParts * kSpan) {
    FewChunk<X> now[kSteps][2];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int i = 0; i < 2; ++i) now[s][i] = next[s][i];
    }
    if (k0 + kFewParts * kSpan < g.width) fetch(k0 + kFewParts * kSpan);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        FewChunk<X> b;  // the few rows stay in the caches
        b.load(h[t], k0 + s * 64, group, g.width);
#pragma unroll
        for (int i = 0; i < 2; ++i) acc[i][t] = few_mfma<X>(now[s][i], b, acc[i][t]);
      }
    }
  }
  // the parts in order, then the words' (maximum, sum) per row
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
      parts[wave][lane] = acc[i][t];
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int p = 1; p < kFewParts; ++p) acc[i][t] += parts[wave + p][lane];
      }
    }
    if (part != 0) continue;
    const int row = t * 16 + entry;
    if (g.logits != nullptr) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<f32x4*>(g.logits + row * g.logits_ld + v0 + i * 16 + 4 * group) = acc[i][t];
      }
    }
    const int64_t from_v0 = target[row] - v0;  // -1 is before every word
    float top = -__builtin_inff(), sum = 0.0f;
    bool counts[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int v = i * 16 + 4 * group + e;
        counts[i][e] = v0 + v < g.vocab;
        top = fmaxf(top, counts[i][e] ? acc[i][t][e] : -__builtin_inff());
        if (from_v0 == v) g.target_logit[row] = acc[i][t][e];
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    top = reference<float>(top);
    const float from = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += counts[i][e] ? power(over_ln2(acc[i][t][e]) - from) : 0.0f;
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 16) meet[words][row] = f32x2{top, sum};
  }
  __syncthreads();
  if (threadIdx.x < TILES * 16) {
    f32x2 sum = meet[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kGroups; ++k) sum = join(sum, meet[k][threadIdx.x]);
    g.sums[static_cast<int64_t>(blockIdx.x) * kFewRows + threadIdx.x] = sum;
  }
}

// The backward of few rows reads W and writes dW once.  A workgroup takes 256 columns, 64 to a wavefront, and every
// parts'th block of 32 words: it forms the block's P (FP32, from the kept logits) in LDS, adds P W to its sums of dH and
// writes P^T H.  FP32 matrix instructions for all types: P is not rounded, and with so few rows they have the time.
// Column n of an instruction stands for columns 4 n .. 4 n + 3 of four of them, so a lane loads and stores 4 columns
// together.  The parts' sums of dH are added up in order after.  With the sums, 16 rows: 32768 x 1024 BF16 (134 MB of W and dW)
// 46 us, FP32 60; more workgroups (768 to 2048) change that by less than their partial sums cost.
constexpr int kBackWords = 32;
constexpr int kBackColumns = 256;
constexpr int kBackSteps = kBackWords / 4;
constexpr int kBackStride = kBackWords + 4;  // of P's rows in LDS: 16 rows by 4 words meet 64 banks
constexpr int kBackGroups = 512;             // workgroups

template <class X>
struct Quad {  // four columns as they lie
  uint32_t w[sizeof(X)];
  __device__ __forceinline__ void load(const X* row, int c, int width) {
    if (c + 4 <= width) {
      __builtin_memcpy(w, row + c, sizeof(w));
    } else {
      X x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = c + e < width ? row[c + e] : from_f32<X>(0.0f);
      __builtin_memcpy(w, x, sizeof(w));
    }
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (std::is_same_v<X, float>) {
      return __uint_as_float(w[e]);
    } else {
      return to_f32(X{static_cast<uint16_t>(w[e / 2] >> (16 * (e % 2)))});
    }
  }
};

template <class X>
struct FewBackArgs {
  const X* hidden;
  const X* weight;
  int64_t hidden_stride, weight_stride, vocab;
  int width, rows;
  Saved saved;
  const float* logits;
  int64_t logits_ld;
  const float* grad_loss;
  int reduction;
  X* grad_weight;  // or nullptr
  float* partial;  // [parts][16 TILES][ld], or nullptr: dH is not wanted
  int64_t ld;
  int parts;
};

template <class X, int TILES>
__global__ void __launch_bounds__(kBlock) attnres_loss_few_backward_kernel(FewBackArgs<X> g) {
  constexpr int kRows = TILES * 16;
  struct Row {
    float c, factor, by;
    int target;  // -2: ignored, or no row at all
  };
  __shared__ Row info[kRows];
  __shared__ float lds[2][kRows][kBackStride];
  const int lane = threadIdx.x % 64, group = lane / 16, entry = lane % 16;
  const int column = static_cast<int>(blockIdx.y) * kBackColumns + wave_index() * 64 + entry * 4;
  if (threadIdx.x < kRows) {
    const int row = threadIdx.x;
    Row r{0.0f, 0.0f, 0.0f, -2};
    const int at = row < g.rows ? g.saved.packed[row] : -1;
    if (at >= 0) {
      r.by = g.reduction == ATTNRES_REDUCE_NONE ? g.grad_loss[row] : g.grad_loss[0];
      if (g.reduction == ATTNRES_REDUCE_MEAN) r.by /= static_cast<float>(g.saved.header->count);
      r.c = g.saved.stats[at].x;
      r.factor = g.saved.stats[at].y * r.by;
      r.target = g.saved.target[at];
    }
    info[row] = r;
  }
  __syncthreads();
  // H: row 4 k + group; what an ignored row holds is not looked at
  float h[kRows / 4][4];
#pragma unroll
  for (int k = 0; k < kRows / 4; ++k) {
    const int row = k * 4 + group;
    Quad<X> x;
    x.load(g.hidden + min(row, g.rows - 1) * g.hidden_stride, column, g.width);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[k][e] = info[row].target == -2 ? 0.0f : x.at(e);
  }
  const int64_t blocks = (g.vocab + kBackWords - 1) / kBackWords;
  Quad<X> next_w[kBackSteps];
  float next_logit[TILES * 2];
  const auto fetch = [&](int64_t block) {
    const int64_t v0 = block * kBackWords;
#pragma unroll
    for (int s = 0; s < kBackSteps; ++s) {
      next_w[s].load(g.weight + min(v0 + s * 4 + group, g.vocab - 1) * g.weight_stride, column, g.width);
    }
#pragma unroll
    for (int i = 0; i < TILES * 2; ++i) {
      next_logit[i] = g.logits[(threadIdx.x / kBackWords + i * 8) * g.logits_ld + v0 + threadIdx.x % kBackWords];
    }
  };
  f32x4 dh[TILES][4] = {};
  fetch(blockIdx.x);
  int buffer = 0;
  for (int64_t block = blockIdx.x; block < blocks; block += g.parts, buffer ^= 1) {
    const int64_t v0 = block * kBackWords;
#pragma unroll
    for (int i = 0; i < TILES * 2; ++i) {
      const int row = threadIdx.x / kBackWords + i * 8, word = threadIdx.x % kBackWords;
      const Row r = info[row];
      float x = power(over_ln2(next_logit[i]) - r.c) * r.factor;
      if (r.target == v0 + word) x -= r.by;
      lds[buffer][row][word] = r.target == -2 || v0 + word >= g.vocab ? 0.0f : x;
    }
    Quad<X> w[kBackSteps];
#pragma unroll
    for (int s = 0; s < kBackSteps; ++s) w[s] = next_w[s];
    if (block + g.parts < blocks) fetch(block + g.parts);
    __syncthreads();
    if (g.partial != nullptr) {
#pragma unroll
      for (int s = 0; s < kBackSteps; ++s) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          const float a = lds[buffer][t * 16 + entry][s * 4 + group];
#pragma unroll
          for (int e = 0; e < 4; ++e) dh[t][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, w[s].at(e), dh[t][e], 0, 0, 0);
        }
      }
    }
    if (g.grad_weight != nullptr) {
#pragma unroll
      for (int m = 0; m < kBackWords / 16; ++m) {
        f32x4 dw[4] = {};
#pragma unroll
        for (int k = 0; k < kRows / 4; ++k) {
          const float a = lds[buffer][k * 4 + group][m * 16 + entry];
#pragma unroll
          for (int e = 0; e < 4; ++e) dw[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, h[k][e], dw[e], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t v = v0 + m * 16 + group * 4 + r;
          if (v >= g.vocab) continue;
          X x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = from_f32<X>(dw[e][r]);
          X* to = g.grad_weight + v * g.width + column;
          if (column + 4 <= g.width) {
            __builtin_memcpy(to, x, sizeof(x));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (column + e < g.width) to[e] = x[e];
            }
          }
        }
      }
    }
  }
  if (g.partial == nullptr) return;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (column >= g.ld) continue;
      float* to = g.partial + (static_cast<int64_t>(blockIdx.x) * kRows + t * 16 + group * 4 + r) * g.ld + column;
      *reinterpret_cast<f32x4*>(to) = f32x4{dh[t][0][r], dh[t][1][r], dh[t][2][r], dh[t][3][r]};
    }
  }
}

// dH from the parts' sums: a row and 64 columns per workgroup, 16 groups that add up every 16th part each.
constexpr int kFewJoinColumns = 64, kFewJoinGroups = kBlock / (kFewJoinColumns / 4);

template <class X>
__global__ void __launch_bounds__(kBlock) attnres_loss_few_join_kernel(const float* __restrict__ partial, int parts, int padded, int64_t ld,
                                                                       const int32_t* packed, int width, X* __restrict__ out) {
  __shared__ f32x4 sums[kFewJoinGroups][kFewJoinColumns / 4];
  const int group = threadIdx.x / (kFewJoinColumns / 4), member = threadIdx.x % (kFewJoinColumns / 4);
  const int64_t row = blockIdx.y;
  const int column = static_cast<int>(blockIdx.x) * kFewJoinColumns + member * 4;
  const int64_t from = min(static_cast<int64_t>(column), ld - 4);
  f32x4 sum = {};
#pragma unroll 8
  for (int k = group; k < parts; k += kFewJoinGroups) {
    sum += *reinterpret_cast<const f32x4*>(partial + (static_cast<int64_t>(k) * padded + row) * ld + from);
  }
  sums[group][member] = sum;
  __syncthreads();
  if (group != 0) return;
  for (int k = 1; k < kFewJoinGroups; ++k) sum += sums[k][member];
  const bool counts = packed[row] >= 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (column + e < width) out[row * width + column + e] = from_f32<X>(counts ? sum[e] : 0.0f);
  }
}

// Upstream gradients of rows that differ (no reduction), for operands of FP16, which has no exponents for them: P is of a
// gradient in [1/2, 1), and the rest, a power of two per row, multiplies the row of dH after its product and the row of H before
// that of dW, in a copy of H of its own (P with the largest row's power would hold a row of weight w of it to 2^-39 / w).  What a row
// adds to dW is held to 2^-39 of the largest product of H and its row's power.
struct RowPowers {
  const float* power;  // per packed row; nullptr: none
  float* alpha;        // dW's two factors, the largest magnitude of H times its row's power over the largest power (as bits), that power
  __device__ __forceinline__ float of(int64_t row) const { return power[row] / alpha[3]; }
};

// Largest finite magnitude of the rows (an integer maximum of the bits: the same in any order).
template <class X>
__global__ void __launch_bounds__(kBlock) attnres_loss_amax_kernel(const X* __restrict__ x, int64_t stride, int64_t rows, int width,
                                                                   const int32_t* index, const int32_t* count, RowPowers powers,
                                                                   uint32_t* amax) {
  __shared__ uint32_t waves[kBlock / 64];
  const int64_t live = count != nullptr ? *count : rows;
  uint32_t top = 0;
  for (int64_t r = blockIdx.x; r < live; r += gridDim.x) {
    const X* row = x + (index != nullptr ? index[r] : r) * stride;
    const float by = powers.power != nullptr ? powers.of(r) : 1.0f;
    for (int c = threadIdx.x * kVec; c < width; c += kBlock * kVec) {
      float v[kVec];
      load_chunk(row, c, width, v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const uint32_t bits = __float_as_uint(v[e] * by) & 0x7fffffffu;
        if (bits < 0x7f800000u && bits > top) top = bits;
      }
    }
  }
#pragma unroll
  for (int step = 32; step > 0; step >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), step, 64)));
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kBlock / 64; ++w) top = max(top, waves[w]);
    atomicMax(amax, top);
  }
}

// Of a power of two that is a normal number.
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }

// The power of two that takes the largest magnitude into [2^14, 2^15), within 2^-110..2^110.
__device__ __forceinline__ float split_scale(uint32_t amax) {
  if (amax == 0) return 1.0f;
  const int exponent = static_cast<int>(amax >> 23) - 127;
  const int shift = min(110, max(-110, 14 - exponent));
  return __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
}

// Rows to operands: [rows_out][width_out] zero-padded, as they are (X 16 bits) or as hi and
// lo (X float).  index/count: the rows that count.  WEIGHED: times their rows' powers, scaled as FP32 rows are.
template <class X, bool WEIGHED>
__global__ void __launch_bounds__(kBlock) attnres_loss_pack_kernel(const X* __restrict__ x, int64_t stride, int64_t rows, int width,
                                                                   const int32_t* index, const int32_t* count, int64_t rows_out,
                                                                   int width_out, Header* header, int which, bool keep_scale,
                                                                   RowPowers powers, uint16_t* __restrict__ hi,
                                                                   uint16_t* __restrict__ lo) {
  const int64_t live = count != nullptr ? *count : rows;
  float scale = 1.0f;
  if constexpr (WEIGHED) {
    scale = split_scale(__float_as_uint(powers.alpha[2]));
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      // of dW: the largest power over the scales of P and of this copy, in two factors where one does not hold it
      const int exponent = exponent_of(powers.alpha[3]) - exponent_of(kProbabilityScale) - exponent_of(scale);
      const int first = min(127, max(-126, exponent));
      powers.alpha[0] = ldexpf(1.0f, first);
      powers.alpha[1] = ldexpf(1.0f, exponent - first);
    }
  } else if constexpr (std::is_same_v<X, float>) {
    scale = split_scale(header->amax[which]);
    if (keep_scale && blockIdx.x == 0 && threadIdx.x == 0) header->scale[which] = scale;
  }
  const int chunks = width_out / kVec;
  const int64_t all = rows_out * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / chunks;
    const int c = static_cast<int>(i - r * chunks) * kVec;
    u32x4 h = {0, 0, 0, 0}, l = {0, 0, 0, 0};
    if (r < live && c < width) {
      const X* row = x + (index != nullptr ? index[r] : r) * stride;
      float v[kVec];
      load_chunk(row, c, width, v);
      const float by = WEIGHED ? powers.of(r) * scale : scale;
      if constexpr (std::is_same_v<X, float>) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float a = v[2 * e] * by, b = v[2 * e + 1] * by;
          asm("" : "+v"(a), "+v"(b));  // one rounding to hi, as in the probabilities
          h[e] = pack2<F16>(a, b);
          l[e] = pack2<F16>(a - to_f32(F16{static_cast<uint16_t>(h[e] & 0xffffu)}),
                            b - to_f32(F16{static_cast<uint16_t>(h[e] >> 16)}));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = WEIGHED ? pack2<X>(v[2 * e] * by, v[2 * e + 1] * by) : pack2<X>(v[2 * e], v[2 * e + 1]);
      }
    }
    *reinterpret_cast<u32x4*>(hi + i * kVec) = h;
    if constexpr (std::is_same_v<X, float>) *reinterpret_cast<u32x4*>(lo + i * kVec) = l;
  }
}

// Per row of the input: its log-sum from the tiles' sums (by packed row, or by row), and its loss.  ROWS rows
// by kBlock / ROWS parts of the tiles per workgroup: 16, which read whole lines, or 4 where that would leave units without work:
// with few rows the tiles' sums are long chains, and their latency is all there is.
template <int ROWS>
__global__ void __launch_bounds__(kBlock) attnres_loss_reduce_kernel(const f32x2* __restrict__ sums, int tiles, int64_t row_tiles,
                                                                     const float* __restrict__ target_logit, int64_t rows, bool packed,
                                                                     Saved s, float* __restrict__ loss) {
  __shared__ f32x2 part[kBlock / 64][ROWS];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x % ROWS;
  const int which = threadIdx.x / ROWS;
  const int at = row < rows ? s.packed[row] : -1;
  const int64_t column = packed ? at : row;  // of the sums
  f32x2 total = {-__builtin_inff(), 0.0f};
  if (at >= 0) {
#pragma unroll 8
    for (int t = which; t < tiles; t += (kBlock / ROWS)) total = join(total, sums[static_cast<int64_t>(t) * row_tiles + column]);
  }
#pragma unroll
  for (int step = ROWS; step < 64; step <<= 1) {
    total = join(total, f32x2{__shfl_xor(total.x, step, 64), __shfl_xor(total.y, step, 64)});
  }
  if (threadIdx.x % 64 < ROWS) part[threadIdx.x / 64][threadIdx.x % 64] = total;
  __syncthreads();
  if (which != 0 || row >= rows) return;
  if (at < 0) {
    loss[row] = 0.0f;
    return;
  }
  for (int k = 1; k < kBlock / 64; ++k) total = join(total, part[k][threadIdx.x]);
  const bool known = s.target[at] >= 0;
  s.stats[at] = f32x2{total.x, known ? 1.0f / total.y : __builtin_nanf("")};
  // both terms are small where the target's probability is near one, and the loss is not below zero
  const int up = fabsf(total.x) < 4194304.0f ? __builtin_amdgcn_frexp_expf(total.y) : 0;  // total.x + up: exact
  const float rest = over_ln2(target_logit[column]) - (total.x + static_cast<float>(up));
  const float value = kLn2 * (log2f(ldexpf(total.y, -up)) - rest);
  loss[row] = !known ? __builtin_nanf("") : value < 0.0f ? 0.0f : value;
}

__global__ void __launch_bounds__(kScanThreads) attnres_loss_total_kernel(const float* __restrict__ loss, int64_t rows, const Header* header,
                                                                          int mean, float* __restrict__ out) {
  __shared__ float waves[kScanThreads / 64];
  float sum = 0.0f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < rows; r += kScanThreads) sum += loss[r];
  sum = group_sum<64>(sum);
  if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0.0f;
  for (int w = 0; w < kScanThreads / 64; ++w) sum += waves[w];
  out[0] = mean ? sum / static_cast<float>(header->count) : sum;
}

// Factors of the backward: per packed row its upstream gradient over a power of two, its own (row_power) or the
// largest one's (one row's factor is at most 1), times the scale of P; and what the outputs are multiplied by.
__global__ void __launch_bounds__(kScanThreads) attnres_loss_factors_kernel(const float* __restrict__ grad_loss, int reduction, Saved s,
                                                                            int64_t row_tiles, float p_scale, float* row_scale,
                                                                            float* row_power, float* alpha) {
  __shared__ uint32_t waves[kScanThreads / 64];
  const int count = s.header->count;
  float outer = count > 0 || row_power != nullptr ? 1.0f : 0.0f;  // nothing counts: zero gradients
  // the power of two above a magnitude, from 2^(least - 127) to 2^(most - 127)
  const auto above = [](uint32_t bits, int least, int most) {
    return __uint_as_float(static_cast<uint32_t>(min(most, max(least, static_cast<int>(bits >> 23) + 1))) << 23);
  };
  if (count > 0 && reduction == ATTNRES_REDUCE_NONE) {
    uint32_t top = 0;
    for (int r = threadIdx.x; r < count; r += kScanThreads) {
      const uint32_t bits = __float_as_uint(grad_loss[s.index[r]]) & 0x7fffffffu;
      if (bits < 0x7f800000u && bits > top) top = bits;
    }
#pragma unroll
    for (int step = 32; step > 0; step >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), step, 64)));
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = top;
    __syncthreads();
    top = 0;
    for (int w = 0; w < kScanThreads / 64; ++w) top = max(top, waves[w]);
    if (top != 0) outer = row_power != nullptr ? above(top, 1, 254) : above(top, 27, 227);
  } else if (count > 0) {
    outer = reduction == ATTNRES_REDUCE_MEAN ? grad_loss[0] / static_cast<float>(count) : grad_loss[0];
  }
  for (int64_t r = threadIdx.x; r < row_tiles; r += kScanThreads) {
    float by = 0.0f;
    if (r < count && reduction == ATTNRES_REDUCE_NONE) {
      const float grad = grad_loss[s.index[r]];
      float over = outer;
      if (row_power != nullptr) {
        const uint32_t bits = __float_as_uint(grad) & 0x7fffffffu;
        if (bits < 0x7f800000u) over = above(bits, 1, 254);
        row_power[r] = over;
      }
      by = grad / over * p_scale;
    } else if (r < count) {
      by = p_scale;
    }
    row_scale[r] = by;
  }
  if (threadIdx.x == 0) {
    // of dH = P W and dW = P^T H; two factors each, as their product may leave FP32 where the gradient does not
    alpha[0] = (row_power != nullptr ? 1.0f : outer) / p_scale;
    alpha[1] = 1.0f / s.header->scale[1];
    alpha[2] = outer / p_scale;
    alpha[3] = 1.0f / s.header->scale[0];
    alpha[4] = 0.0f;  // the rest for row_power
    alpha[5] = outer;
  }
}

// out[r] = both alpha's (and the row's power) times the sum of the splits' partial rows; packed: of the row's packed one,
// zeros where it has none.
template <class OUT>
__global__ void __launch_bounds__(kBlock) attnres_loss_join_kernel(const float* __restrict__ partial, int splits, int64_t split_stride,
                                                                   int64_t ld, const int32_t* packed, int64_t rows, int width,
                                                                   const float* __restrict__ alpha, const float* __restrict__ row_power,
                                                                   OUT* __restrict__ out) {
  const float by = alpha[0], unscale = alpha[1];
  const int chunks = (width + kVec - 1) / kVec;
  const int64_t all = rows * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * kBlock) {
    const int64_t r = i / chunks;
    const int c = static_cast<int>(i - r * chunks) * kVec;
    const int64_t at = packed != nullptr ? packed[r] : r;
    float sum[kVec] = {};
    if (at >= 0) {
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        float x[kVec];
        load8(partial + k * split_stride + at * ld + c, x);  // rows are padded to whole chunks
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum[e] += x[e];
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        // powers of two all three: their exponents' sum leaves FP32 only where the gradient does
        sum[e] = row_power != nullptr ? ldexpf(sum[e], exponent_of(by) + exponent_of(unscale) + exponent_of(row_power[at]))
                                      : sum[e] * by * unscale;
      }
    }
    store_chunk(out + r * width, c, width, sum);
  }
}

// ---------------------------------------------------------------------- host

constexpr int64_t kMaxRows = int64_t{1} << 24;
constexpr int64_t kMaxVocab = int64_t{1} << 24;
constexpr int64_t kMaxStride = int64_t{1} << 22;  // of W multiplied in place: 256 rows stay within 32-bit offsets
constexpr int64_t kPieceBytes = int64_t{512} << 20;  // of P at a time
constexpr int64_t kKeepBytes = int64_t{8} << 30;     // of powers kept for the backward
constexpr int kUnits = 256;                          // compute units, one workgroup each

// How many parts the depth of a gradient product is cut into, so that its workgroups fill the chip: what takes the
// least time at 1.1 PFLOP/s for full rounds of workgroups and 4.5 TB/s for the FP32 partial sums that are
// written and read again (both as measured).  `direct`: one part needs no partial sums.  A part keeps at least 8 stages.
int choose_splits(int64_t tiles, int64_t depth, int segments, bool direct) {
  int best = 1;
  double best_time = 0.0;
  for (int s = 1; s <= 32; ++s) {
    if (s > 1 && depth / kDepth / s < 8) break;
    const int64_t rounds = (tiles * s + kUnits - 1) / kUnits;
    const double tile = 2.0 * kTile * kTile * static_cast<double>(depth) * segments / s / (1.1e15 / kUnits);
    const double partial = s == 1 && direct ? 0.0 : 8.0 * kTile * kTile * static_cast<double>(tiles) * s / 4.5e12;
    const double time = static_cast<double>(rounds) * tile + partial;
    if (s == 1 || time < best_time) best = s, best_time = time;
  }
  return best;
}

// Rows that go the way of few rows.  Forward, us, its way -> by tiles, 16 / 32 / 64 rows: BF16, 32768 x 1024
// 20.8 / 26.4 / 34.6 -> 37, 131072 x 2048 126 / 157 / 212 -> 156; where W has to be packed for the tiles, FP16, 50021 x 1000
// 31 / 38 / 50 -> 71, FP32, 32768 x 1024 34 / 48 / 80 -> 166.  Backward: BF16, 32768 x 1024 46 / 63 / - -> 74, 131072 x 2048
// 308 / 413 / - -> 338; FP16, 50021 x 1000 93 / - / 205 -> 154; FP32, 32768 x 1024 60 / 71 / 121 -> 216.
int64_t few_rows(bool pack_weight) { return pack_weight ? kFewRows : kFewRows / 2; }

struct LossPlan {
  bool split, pack_weight, few, keep;
  int64_t rows_pad, width_pad, vocab_pad, piece;
  int64_t hidden[2], weight[2], sums, target_logit, losses;  // offsets
  int64_t row_scale, row_power, alpha, weighed[2], p[2], dh, dw, logits, logits_ld;
  int few_tiles, few_words, parts;
  int splits_h, splits_w;
  int64_t bytes;
  int64_t saved_sums, saved_target, saved_powers, saved_bytes;
};

enum Pass { kForward = 0, kBackward = 1, kBackwardOfTotal = 2 };  // the last: of a sum or mean, which has one upstream gradient

LossPlan loss_plan(int64_t rows, int64_t vocab, int64_t width, int dtype, bool keep, int pass) {
  const bool backward = pass != kForward;
  LossPlan p{};
  p.split = dtype == ATTNRES_F32;
  p.pack_weight = p.split || width % kDepth != 0;
  p.rows_pad = round_up(std::max<int64_t>(rows, 1), kTile);
  p.width_pad = round_up(width, kDepth);
  p.vocab_pad = round_up(vocab, kTile);
  const int parts = p.split ? 2 : 1;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += round_up(bytes, 256);
    return from;
  };
  p.few = rows > 0 && rows <= few_rows(p.pack_weight);
  p.few_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  p.few_words = vocab > kFewWords / 2 * kUnits ? kFewWords : 32;
  p.logits_ld = round_up(vocab, kFewWords);
  const int64_t logits = 4 * 16 * p.few_tiles * p.logits_ld;
  const int64_t powers = p.few ? logits : (dtype == ATTNRES_BF16 ? 2 : 4) * p.rows_pad * p.vocab_pad;
  p.keep = keep && rows > 0 && powers <= kKeepBytes;
  p.saved_bytes = kHeaderBytes + 20 * rows;
  if (p.keep) {
    p.saved_sums = round_up(p.saved_bytes, 256);
    p.saved_target = p.saved_sums + (p.few ? 0 : 8 * (p.vocab_pad / 128) * p.rows_pad);
    p.saved_powers = p.saved_target + (!p.few && dtype == ATTNRES_BF16 ? 4 * p.rows_pad : 0);
    p.saved_bytes = p.saved_powers + powers;
  }
  const bool scores = !backward || (p.few && !p.keep);  // the forward's kernels run
  if (!p.few) {  // packed operands: kept beside the powers
    const auto place = [&](int64_t bytes) {
      if (!p.keep) return take(bytes);
      const int64_t from = p.saved_bytes;
      p.saved_bytes += round_up(bytes, 256);
      return from;
    };
    for (int k = 0; k < parts; ++k) p.hidden[k] = place(2 * p.rows_pad * p.width_pad);
    for (int k = 0; p.pack_weight && k < parts; ++k) p.weight[k] = place(2 * vocab * p.width_pad);
  }
  if (scores) {
    if (p.few) p.sums = take(8 * (p.logits_ld / p.few_words) * kFewRows);
    else if (!p.keep) p.sums = take(8 * (p.vocab_pad / 128) * p.rows_pad);
    p.target_logit = take(4 * p.rows_pad);
  }
  if (!backward) {
    p.losses = take(4 * rows);
  } else if (p.few) {
    if (!p.keep) p.logits = take(logits);
    const int64_t slabs = (width + kBackColumns - 1) / kBackColumns;
    p.parts = static_cast<int>(std::min<int64_t>((vocab + kBackWords - 1) / kBackWords, std::max<int64_t>(kBackGroups / slabs, 1)));
    p.dh = take(4 * p.parts * 16 * p.few_tiles * p.width_pad);
  } else {
    p.row_scale = take(4 * p.rows_pad);
    p.alpha = take(32);
    if (pass != kBackwardOfTotal && dtype != ATTNRES_BF16) {
      p.row_power = take(4 * p.rows_pad);
      for (int k = 0; k < parts; ++k) p.weighed[k] = take(2 * p.rows_pad * p.width_pad);
    }
    p.piece = std::min(p.vocab_pad, std::max<int64_t>(kPieceBytes / (2 * parts * p.rows_pad) / kTile, 1) * kTile);
    const int64_t pieces = (p.vocab_pad + p.piece - 1) / p.piece;
    p.piece = round_up((p.vocab_pad + pieces - 1) / pieces, kTile);
    for (int k = 0; k < parts; ++k) p.p[k] = take(2 * p.rows_pad * p.piece);
    const int64_t tiles_d = (width + kTile - 1) / kTile;
    p.splits_h = choose_splits(tiles_d * (p.rows_pad / kTile), p.piece, p.split ? 3 : 1, false);
    p.dh = take(4 * p.splits_h * p.rows_pad * p.width_pad);
    p.splits_w = choose_splits(tiles_d * (p.piece / kTile), p.rows_pad, p.split ? 3 : 1, true);
    if (p.splits_w > 1) p.dw = take(4 * p.splits_w * p.piece * p.width_pad);
  }
  p.bytes = at;
  return p;
}

Saved saved_views(void* base, int64_t rows, const LossPlan& p) {
  char* from = static_cast<char*>(base);
  char* at = from + kHeaderBytes;
  return {reinterpret_cast<Header*>(from), reinterpret_cast<f32x2*>(at), reinterpret_cast<int32_t*>(at + 8 * rows),
          reinterpret_cast<int32_t*>(at + 12 * rows), reinterpret_cast<int32_t*>(at + 16 * rows),
          p.keep ? reinterpret_cast<f32x2*>(from + p.saved_sums) : nullptr,
          p.saved_powers > p.saved_target ? reinterpret_cast<float*>(from + p.saved_target) : nullptr,
          p.keep ? from + p.saved_powers : nullptr};
}

unsigned stride_grid(int64_t items) { return static_cast<unsigned>(std::min<int64_t>((items + kBlock - 1) / kBlock, 8192)); }

struct Call {
  const void* hidden;
  int64_t hidden_stride;
  const void* weight;
  int64_t weight_stride;
  int64_t rows, vocab, width;
  LossPlan plan;
  Saved saved;
  char* workspace;
  hipStream_t stream;
  template <class X>
  X* at(int64_t offset) const { return reinterpret_cast<X*>(workspace + offset); }
  uint16_t* operand(int64_t offset) const {
    return reinterpret_cast<uint16_t*>((plan.keep ? reinterpret_cast<char*>(saved.header) : workspace) + offset);
  }
};

// The operands of both directions: H's rows that count, packed, and W as it is or packed.  The backward finds
// them packed where powers are kept.
template <class X>
void prepare_operands(const Call& c, bool forward, Operand* h, Operand* w) {
  const LossPlan& p = c.plan;
  constexpr bool kSplit = std::is_same_v<X, float>;
  const X* hidden = static_cast<const X*>(c.hidden);
  const X* weight = static_cast<const X*>(c.weight);
  Header* header = c.saved.header;
  if constexpr (kSplit) {
    if (forward) {
      const unsigned grid_h = static_cast<unsigned>(std::min<int64_t>(c.rows, 1024));
      hipLaunchKernelGGL(attnres_loss_amax_kernel<float>, dim3(grid_h), dim3(kBlock), 0, c.stream, hidden, c.hidden_stride, c.rows,
                         static_cast<int>(c.width), c.saved.index, &header->count, RowPowers{}, &header->amax[0]);
      const unsigned grid_w = static_cast<unsigned>(std::min<int64_t>(c.vocab, 2048));
      hipLaunchKernelGGL(attnres_loss_amax_kernel<float>, dim3(grid_w), dim3(kBlock), 0, c.stream, weight, c.weight_stride, c.vocab,
                         static_cast<int>(c.width), static_cast<const int32_t*>(nullptr), static_cast<const int32_t*>(nullptr),
                         RowPowers{}, &header->amax[1]);
    }
  }
  const bool pack = forward || !p.keep;
  uint16_t* packed[2] = {c.operand(p.hidden[0]), kSplit ? c.operand(p.hidden[1]) : nullptr};
  if (pack) {
    hipLaunchKernelGGL((attnres_loss_pack_kernel<X, false>), dim3(stride_grid(p.rows_pad * p.width_pad / kVec)), dim3(kBlock), 0, c.stream,
                       hidden, c.hidden_stride, c.rows, static_cast<int>(c.width), c.saved.index, &header->count, p.rows_pad,
                       static_cast<int>(p.width_pad), header, 0, forward, RowPowers{}, packed[0], packed[1]);
  }
  *h = {{packed[0], packed[1]}, p.width_pad, p.rows_pad, 0};
  if (p.pack_weight) {
    uint16_t* to[2] = {c.operand(p.weight[0]), kSplit ? c.operand(p.weight[1]) : nullptr};
    if (pack) {
      hipLaunchKernelGGL((attnres_loss_pack_kernel<X, false>), dim3(stride_grid(c.vocab * p.width_pad / kVec)), dim3(kBlock), 0, c.stream,
                         weight, c.weight_stride, c.vocab, static_cast<int>(c.width), static_cast<const int32_t*>(nullptr),
                         static_cast<const int32_t*>(nullptr), c.vocab, static_cast<int>(p.width_pad), header, 1, forward, RowPowers{}, to[0],
                         to[1]);
    }
    *w = {{to[0], to[1]}, p.width_pad, c.vocab, 0};
  } else {
    *w = {{reinterpret_cast<const uint16_t*>(weight), nullptr}, c.weight_stride, c.vocab, 0};
  }
}

// H times its rows' powers, for dW.
template <class X>
Operand weigh_rows(const Call& c, const RowPowers& powers) {
  const LossPlan& p = c.plan;
  const X* hidden = static_cast<const X*>(c.hidden);
  Header* header = c.saved.header;
  hipLaunchKernelGGL((attnres_loss_amax_kernel<X>), dim3(static_cast<unsigned>(std::min<int64_t>(c.rows, 1024))), dim3(kBlock), 0,
                     c.stream, hidden, c.hidden_stride, c.rows, static_cast<int>(c.width), c.saved.index, &header->count, powers,
                     reinterpret_cast<uint32_t*>(powers.alpha + 2));
  uint16_t* to[2] = {c.at<uint16_t>(p.weighed[0]), std::is_same_v<X, float> ? c.at<uint16_t>(p.weighed[1]) : nullptr};
  hipLaunchKernelGGL((attnres_loss_pack_kernel<X, true>), dim3(stride_grid(p.rows_pad * p.width_pad / kVec)), dim3(kBlock), 0, c.stream,
                     hidden, c.hidden_stride, c.rows, static_cast<int>(c.width), c.saved.index, &header->count, p.rows_pad,
                     static_cast<int>(p.width_pad), header, 0, false, powers, to[0], to[1]);
  return {{to[0], to[1]}, p.width_pad, p.rows_pad, 0};
}

// The logits of few rows; logits: where they are kept, or nullptr.  targets: nullptr in the backward, where
// saved and ignored rows are known.
template <class X>
void launch_few(const Call& c, const void* targets, int target_bytes, int64_t ignore_index, float* logits) {
  const LossPlan& p = c.plan;
  const FewArgs<X> g{static_cast<const X*>(c.hidden), static_cast<const X*>(c.weight), c.hidden_stride, c.weight_stride, c.vocab,
                     static_cast<int>(c.width), static_cast<int>(c.rows), targets, target_bytes, ignore_index, c.saved,
                     c.at<f32x2>(p.sums), c.at<float>(p.target_logit), logits, p.logits_ld};
  const auto launch = [&](auto words) {
    constexpr int WORDS = decltype(words)::value;
    const auto kernel = p.few_tiles == 1   ? attnres_loss_few_kernel<X, 1, WORDS>
                        : p.few_tiles == 2 ? attnres_loss_few_kernel<X, 2, WORDS>
                                           : attnres_loss_few_kernel<X, 4, WORDS>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(p.logits_ld / WORDS)), dim3(kFewBlock), 0, c.stream, g);
  };
  if (p.few_words == 32) {
    launch(std::integral_constant<int, 32>{});
  } else {
    launch(std::integral_constant<int, kFewWords>{});
  }
}

template <class X>
void few_backward(const Call& c, int reduction, const float* grad_loss, void* grad_hidden, void* grad_weight) {
  const LossPlan& p = c.plan;
  const float* logits = static_cast<const float*>(c.saved.powers);
  if (!p.keep) {
    float* again = c.at<float>(p.logits);
    launch_few<X>(c, nullptr, 8, 0, again);
    logits = again;
  }
  const FewBackArgs<X> g{static_cast<const X*>(c.hidden), static_cast<const X*>(c.weight), c.hidden_stride, c.weight_stride, c.vocab,
                         static_cast<int>(c.width), static_cast<int>(c.rows), c.saved, logits, p.logits_ld, grad_loss, reduction,
                         static_cast<X*>(grad_weight), grad_hidden != nullptr ? c.at<float>(p.dh) : nullptr, p.width_pad, p.parts};
  const auto kernel = p.few_tiles == 1   ? attnres_loss_few_backward_kernel<X, 1>
                      : p.few_tiles == 2 ? attnres_loss_few_backward_kernel<X, 2>
                                         : attnres_loss_few_backward_kernel<X, 4>;
  const unsigned slabs = static_cast<unsigned>((c.width + kBackColumns - 1) / kBackColumns);
  hipLaunchKernelGGL(kernel, dim3(p.parts, slabs), dim3(kBlock), 0, c.stream, g);
  if (grad_hidden != nullptr) {
    const dim3 grid(static_cast<unsigned>((c.width + kFewJoinColumns - 1) / kFewJoinColumns), static_cast<unsigned>(c.rows));
    hipLaunchKernelGGL((attnres_loss_few_join_kernel<X>), grid, dim3(kBlock), 0, c.stream, c.at<const float>(p.dh), p.parts,
                       16 * p.few_tiles, p.width_pad, c.saved.packed, static_cast<int>(c.width), static_cast<X*>(grad_hidden));
  }
}

// X: the inputs' type; T: the operands'.
template <class X, class T, int SEGMENTS>
void loss_forward(const Call& c, const void* targets, int target_bytes, int64_t ignore_index, int reduction, float* loss) {
  const LossPlan& p = c.plan;
  if (!p.few) {
    hipLaunchKernelGGL(attnres_loss_rows_kernel, dim3(1), dim3(kScanThreads), 0, c.stream, targets, target_bytes, c.rows, c.vocab,
                       ignore_index, c.saved);
  }
  if (c.rows > 0) {
    f32x2* sums = p.keep && !p.few ? c.saved.sums : c.at<f32x2>(p.sums);
    float* target_logit = c.saved.target_logit != nullptr ? c.saved.target_logit : c.at<float>(p.target_logit);
    int tiles;
    int64_t row_tiles;
    if (p.few) {
      tiles = static_cast<int>(p.logits_ld / p.few_words);
      row_tiles = kFewRows;
      launch_few<X>(c, targets, target_bytes, ignore_index, static_cast<float*>(c.saved.powers));
    } else {
      LogitArgs g{};
      prepare_operands<X>(c, true, &g.product.b, &g.product.a);
      g.product.count = &c.saved.header->count;
      g.product.depth = p.width_pad;
      g.product.tiles_a = static_cast<int>(p.vocab_pad / kTile);
      tiles = 2 * g.product.tiles_a;
      g.product.tiles_b = static_cast<int>(p.rows_pad / kTile);
      g.product.splits = 1;
      g.header = c.saved.header;
      g.target = c.saved.target;
      g.vocab = c.vocab;
      g.row_tiles = row_tiles = p.rows_pad;
      g.sums = sums;
      g.target_logit = target_logit;
      g.powers = c.saved.powers;
      g.powers_ld = p.vocab_pad;
      const auto kernel = p.keep ? attnres_loss_logits_kernel<T, SEGMENTS, true> : attnres_loss_logits_kernel<T, SEGMENTS, false>;
      hipLaunchKernelGGL(kernel, dim3(g.product.tiles_a * g.product.tiles_b), dim3(kThreads), 0,
                         c.stream, g);
    }
    float* losses = reduction == ATTNRES_REDUCE_NONE ? loss : c.at<float>(p.losses);
    const bool many = c.rows >= 16 * kUnits;
    const auto reduce = many ? attnres_loss_reduce_kernel<16> : attnres_loss_reduce_kernel<4>;
    hipLaunchKernelGGL(reduce, dim3(static_cast<unsigned>((c.rows + (many ? 15 : 3)) / (many ? 16 : 4))), dim3(kBlock), 0, c.stream,
                       sums, tiles, row_tiles, target_logit, c.rows, !p.few, c.saved, losses);
  }
  if (reduction != ATTNRES_REDUCE_NONE) {
    hipLaunchKernelGGL(attnres_loss_total_kernel, dim3(1), dim3(kScanThreads), 0, c.stream, c.at<const float>(p.losses), c.rows,
                       c.saved.header, reduction == ATTNRES_REDUCE_MEAN ? 1 : 0, loss);
  }
}

template <class X, class T, int SEGMENTS>
void loss_backward(const Call& c, int reduction, const float* grad_loss, void* grad_hidden, void* grad_weight) {
  const LossPlan& p = c.plan;
  constexpr int kParts = SEGMENTS == 3 ? 2 : 1;
  if (p.few) return few_backward<X>(c, reduction, grad_loss, grad_hidden, grad_weight);
  Operand h{}, w{};
  prepare_operands<X>(c, false, &h, &w);
  const float p_scale = std::is_same_v<T, Bf16> ? 1.0f : kProbabilityScale;
  float* alpha = c.at<float>(p.alpha);
  float* row_scale = c.at<float>(p.row_scale);
  float* row_power = !std::is_same_v<T, Bf16> && reduction == ATTNRES_REDUCE_NONE ? c.at<float>(p.row_power) : nullptr;
  hipLaunchKernelGGL(attnres_loss_factors_kernel, dim3(1), dim3(kScanThreads), 0, c.stream, grad_loss, reduction, c.saved,
                     p.rows_pad, p_scale, row_scale, row_power, alpha);
  Operand rows = h;  // of dW
  if constexpr (!std::is_same_v<T, Bf16>) {
    if (row_power != nullptr && grad_weight != nullptr && c.rows > 0) {
      // from alpha + 2 on: the factors that go with these rows, and what they are made from
      rows = weigh_rows<X>(c, RowPowers{row_power, alpha + 2});
    }
  }
  const int32_t* count = &c.saved.header->count;
  const int tiles_d = static_cast<int>((c.width + kTile - 1) / kTile), tiles_n = static_cast<int>(p.rows_pad / kTile);
  Operand probability{{c.at<const uint16_t>(p.p[0]), kParts == 2 ? c.at<const uint16_t>(p.p[1]) : nullptr}, p.piece, 0, 0};
  for (int64_t v0 = 0; v0 < c.vocab; v0 += p.piece) {
    const int64_t columns = std::min(p.piece, c.vocab - v0);
    const int tiles_v = static_cast<int>((columns + kTile - 1) / kTile);
    Operand piece = w;
    for (int k = 0; k < kParts; ++k) piece.part[k] = w.part[k] + v0 * w.ld;
    piece.entries = columns;
    LogitArgs g{};
    g.product = {piece, h, count, p.width_pad, 0, tiles_v, tiles_n, 1};
    g.header = c.saved.header;
    g.target = c.saved.target;
    g.vocab = c.vocab;
    g.first = v0;
    g.row_tiles = p.rows_pad;
    g.stats = c.saved.stats;
    g.row_scale = row_scale;
    for (int k = 0; k < kParts; ++k) g.p[k] = c.at<uint16_t>(p.p[k]);
    g.p_ld = p.piece;
    if (p.keep) {
      using E = Power<T>;
      g.sums = c.saved.sums;
      g.target_logit = c.saved.target_logit;
      g.powers = c.saved.powers;
      g.powers_ld = p.vocab_pad;
      const int64_t wide = static_cast<int64_t>(tiles_v) * kTile;
      const int blocks = static_cast<int>((wide + kScaleColumns - 1) / kScaleColumns);
      hipLaunchKernelGGL((attnres_loss_rescale_kernel<E, T, kParts>), dim3(static_cast<unsigned>(p.rows_pad / kScaleRows * blocks)),
                         dim3(kBlock), 0, c.stream, g, wide, blocks);
    } else {
      hipLaunchKernelGGL((attnres_loss_probability_kernel<T, SEGMENTS>), dim3(tiles_v * tiles_n), dim3(kThreads), 0, c.stream, g);
    }
    if (grad_weight != nullptr) {
      Operand a = rows, b = probability;
      a.entries = p.width_pad;
      a.depth = b.depth = p.rows_pad;
      b.entries = p.piece;
      GradientArgs e{};
      e.product = {a, b, count, 0, 1, tiles_d, tiles_v, p.splits_w};
      e.entries_a = c.width;
      e.entries_b = columns;
      const dim3 grid(tiles_d * tiles_v * p.splits_w);
      X* out = static_cast<X*>(grad_weight) + v0 * c.width;
      if (p.splits_w == 1) {
        e.alpha = alpha + 2;
        e.out = out;
        e.ld = c.width;
        hipLaunchKernelGGL((attnres_loss_gradient_kernel<T, X, SEGMENTS, false>), grid, dim3(kThreads), 0, c.stream, e);
      } else {
        e.out = c.at<float>(p.dw);
        e.ld = p.width_pad;
        e.entries_a = p.width_pad;
        e.split_stride = p.piece * p.width_pad;
        hipLaunchKernelGGL((attnres_loss_gradient_kernel<T, float, SEGMENTS, false>), grid, dim3(kThreads), 0, c.stream, e);
        hipLaunchKernelGGL((attnres_loss_join_kernel<X>), dim3(stride_grid(columns * ((c.width + kVec - 1) / kVec))), dim3(kBlock), 0,
                           c.stream, c.at<const float>(p.dw), p.splits_w, e.split_stride, p.width_pad,
                           static_cast<const int32_t*>(nullptr), columns, static_cast<int>(c.width), alpha + 2,
                           static_cast<const float*>(nullptr), out);
      }
    }
    if (grad_hidden != nullptr) {
      Operand a = piece, b = probability;
      a.entries = p.pack_weight ? p.width_pad : c.width;
      a.depth = columns;
      b.entries = p.rows_pad;
      GradientArgs e{};
      e.product = {a, b, count, round_up(columns, kDepth), 0, tiles_d, tiles_n, p.splits_h};
      e.out = c.at<float>(p.dh);
      e.ld = p.width_pad;
      e.split_stride = p.rows_pad * p.width_pad;
      e.entries_a = p.width_pad;
      e.entries_b = p.rows_pad;
      e.add = v0 > 0 ? 1 : 0;
      e.live_only = 1;
      hipLaunchKernelGGL((attnres_loss_gradient_kernel<T, float, SEGMENTS, true>), dim3(tiles_d * tiles_n * p.splits_h),
                         dim3(kThreads), 0, c.stream, e);
    }
  }
  if (grad_hidden != nullptr && c.rows > 0) {
    hipLaunchKernelGGL((attnres_loss_join_kernel<X>), dim3(stride_grid(c.rows * ((c.width + kVec - 1) / kVec))), dim3(kBlock), 0,
                       c.stream, c.at<const float>(p.dh), p.splits_h, p.rows_pad * p.width_pad, p.width_pad, c.saved.packed, c.rows,
                       static_cast<int>(c.width), alpha, row_power, static_cast<X*>(grad_hidden));
  }
}

// A launch takes fewer than 2^32 threads: 2^23 workgroups of a tile each are too many.
constexpr int64_t kMaxTiles = int64_t{1} << 22;
bool fits_grid(int64_t rows, int64_t vocab) {
  return (rows + kTile - 1) / kTile * ((vocab + kTile - 1) / kTile) <= kMaxTiles;
}

bool known_shape(int64_t rows, int64_t vocab, int64_t width, int dtype) {
  return rows >= 0 && rows <= kMaxRows && vocab >= 1 && vocab <= kMaxVocab && width >= 1 && width <= ATTNRES_MAX_WIDTH &&
         dtype_known(dtype) && fits_grid(rows, vocab);
}

// Offsets into both are multiples of 16 bytes, which the products' loads into LDS need.
int check_places(const void* saved, const void* workspace, int64_t workspace_bytes, int64_t need) {
  if (workspace == nullptr || workspace_bytes < need) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  }
  if (((reinterpret_cast<uintptr_t>(saved) | reinterpret_cast<uintptr_t>(workspace)) & 15u) != 0) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "saved and workspace must start at multiples of 16 bytes");
  }
  return ATTNRES_OK;
}

int check_loss(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride, int64_t rows, int64_t vocab,
               int64_t width, int dtype, int reduction) {
  if (rows < 0 || rows > kMaxRows) return layer_error(ATTNRES_ERR_SHAPE, "rows=%lld outside 0..2^24", (long long)rows);
  if (vocab < 1 || vocab > kMaxVocab) return layer_error(ATTNRES_ERR_SHAPE, "vocab=%lld outside 1..2^24", (long long)vocab);
  if (width < 1 || width > ATTNRES_MAX_WIDTH) {
    return layer_error(ATTNRES_ERR_SHAPE, "width=%lld outside 1..%d", (long long)width, ATTNRES_MAX_WIDTH);
  }
  if (!dtype_known(dtype)) return layer_error(ATTNRES_ERR_SHAPE, "unknown dtype %d", dtype);
  if (reduction < ATTNRES_REDUCE_NONE || reduction > ATTNRES_REDUCE_MEAN) {
    return layer_error(ATTNRES_ERR_SCALAR, "unknown reduction %d", reduction);
  }
  if (!fits_grid(rows, vocab)) return layer_error(ATTNRES_ERR_SHAPE, "rows x vocab outside 2^22 tiles of 256 x 256");
  if (hidden_stride < 0 || weight_stride < 0) return layer_error(ATTNRES_ERR_STRIDE, "negative row stride");
  if ((rows > 0 && hidden == nullptr) || weight == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "hidden or weight is NULL");
  if (dtype != ATTNRES_F32 && width % kDepth == 0 &&
      ((reinterpret_cast<uintptr_t>(weight) & 15u) != 0 || weight_stride % 8 != 0 || weight_stride < width ||
       weight_stride > kMaxStride)) {
    return layer_error(ATTNRES_ERR_STRIDE, "weight rows must start at multiples of 16 bytes, at most %lld elements apart",
                       (long long)kMaxStride);
  }
  return ATTNRES_OK;
}

}  // namespace
}  // namespace layers
}  // namespace attnres_hip

using namespace attnres_hip;
using namespace attnres_hip::layers;

extern "C" {

int64_t attnres_hip_loss_saved_bytes(int64_t rows, int64_t vocab, int64_t width, int dtype, int keep) {
  return known_shape(rows, vocab, width, dtype) ? loss_plan(rows, vocab, width, dtype, keep != 0, kForward).saved_bytes : -1;
}

int64_t attnres_hip_loss_workspace_bytes(int64_t rows, int64_t vocab, int64_t width, int dtype, int keep, int backward) {
  return known_shape(rows, vocab, width, dtype) ? loss_plan(rows, vocab, width, dtype, keep != 0, backward).bytes : -1;
}

int attnres_hip_loss_forward(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride,
                             const void* targets, int target_bytes, int64_t rows, int64_t vocab, int64_t width, int dtype,
                             int64_t ignore_index, int reduction, int keep, float* loss, void* saved, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  if (const int status = check_loss(hidden, hidden_stride, weight, weight_stride, rows, vocab, width, dtype, reduction)) return status;
  if (target_bytes != 4 && target_bytes != 8) return layer_error(ATTNRES_ERR_SHAPE, "targets must be int32 or int64");
  if (loss == nullptr || saved == nullptr || (rows > 0 && targets == nullptr)) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "targets, loss or saved is NULL");
  }
  const LossPlan plan = loss_plan(rows, vocab, width, dtype, keep != 0, kForward);
  const Call c{hidden, hidden_stride, weight, weight_stride, rows, vocab, width, plan, saved_views(saved, rows, plan),
               static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
  if (const int status = check_places(saved, workspace, workspace_bytes, c.plan.bytes)) return status;
  if (dtype == ATTNRES_BF16) loss_forward<Bf16, Bf16, 1>(c, targets, target_bytes, ignore_index, reduction, loss);
  else if (dtype == ATTNRES_F16) loss_forward<F16, F16, 1>(c, targets, target_bytes, ignore_index, reduction, loss);
  else loss_forward<float, F16, 3>(c, targets, target_bytes, ignore_index, reduction, loss);
  return layer_launch_status("loss forward");
}

int attnres_hip_loss_backward(const void* hidden, int64_t hidden_stride, const void* weight, int64_t weight_stride, int64_t rows,
                              int64_t vocab, int64_t width, int dtype, int reduction, int keep, const void* saved,
                              const float* grad_loss, void* grad_hidden, void* grad_weight, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  if (const int status = check_loss(hidden, hidden_stride, weight, weight_stride, rows, vocab, width, dtype, reduction)) return status;
  if (saved == nullptr || grad_loss == nullptr) return layer_error(ATTNRES_ERR_NULL_POINTER, "saved or grad_loss is NULL");
  const LossPlan plan = loss_plan(rows, vocab, width, dtype, keep != 0,
                                  reduction == ATTNRES_REDUCE_NONE ? kBackward : kBackwardOfTotal);
  const Call c{hidden, hidden_stride, weight, weight_stride, rows, vocab, width, plan,
               saved_views(const_cast<void*>(saved), rows, plan),  // read only
               static_cast<char*>(workspace), static_cast<hipStream_t>(stream)};
  if (const int status = check_places(saved, workspace, workspace_bytes, c.plan.bytes)) return status;
  if (grad_hidden == nullptr && grad_weight == nullptr) return ATTNRES_OK;
  if (dtype == ATTNRES_BF16) loss_backward<Bf16, Bf16, 1>(c, reduction, grad_loss, grad_hidden, grad_weight);
  else if (dtype == ATTNRES_F16) loss_backward<F16, F16, 1>(c, reduction, grad_loss, grad_hidden, grad_weight);
  else loss_backward<float, F16, 3>(c, reduction, grad_loss, grad_hidden, grad_weight);
  return layer_launch_status("loss backward");
}

}  // extern "C"
