// attnres_product.h - the matrix product of the layers: tiles of 256 x 256, 128 x 128 or 64 x 64 outputs of 16-bit
// operands on the matrix cores, summed in FP32 (attnres_loss.hip, attnres_ffn.hip).
#ifndef ATTNRES_PRODUCT_H
#define ATTNRES_PRODUCT_H

#include "attnres_layers.h"

namespace attnres_hip {
namespace layers {

constexpr int kTile = 256;     // rows and columns of a workgroup's tile
constexpr int kWaves = 8;      // of 128 x 64 outputs, two per SIMD
constexpr int kThreads = 64 * kWaves;
constexpr int kDown = 8;       // 16 x 16 tiles of a wavefront: down (A) and across (B)
constexpr int kAcross = 4;
constexpr int kDepth = 32;     // of a stage of a tile's operands in LDS
constexpr int kStages = 4;     // in LDS: one that is multiplied, three on their way
constexpr int kLoads = 2;      // per wavefront, operand and stage: 1 KB each
constexpr int kOperand = kTile * kDepth;  // elements of one operand's stage

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define ATTNRES_LDS __attribute__((address_space(3)))
#define ATTNRES_GLOBAL __attribute__((address_space(1)))

__host__ __device__ inline int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

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
  const uint16_t* part[3];  // hi, lo; or the three parts of FP32 values
  int64_t ld;
  int64_t entries;          // readable entries (rows: clamped row; columns: multiple of 8)
  int64_t depth;            // readable k of a column operand
  int64_t second;           // PAIRED rows: elements from the first half's start to the second's
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

// PAIRED rows: a tile holds 128 entries of each of two operands of one shape, so that a wavefront's accumulators
// i and i + kDown / 2 are entry e of the one and of the other: 64 of the first, 64 of the second, in turn.
constexpr int kPaired = 64;

template <bool ROWS, bool PAIRED = false>
struct Loader {
  uint32_t offset[kLoads];  // bytes from the stage's origin; columns: of the chunk alone
  int row;                  // columns: k of the first load
  __device__ __forceinline__ void init(const Operand& o, int64_t entry0, int wave, int lane) {
    row = wave * kLoads * 2 + lane / 32;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if constexpr (ROWS) {
        const int r = (wave * kLoads + j) * 16 + lane / 4;
        const int entry = PAIRED ? r / (2 * kPaired) * kPaired + r % kPaired : r;
        const int64_t left = o.entries - 1 - entry0;
        const int64_t at = entry < left ? entry : left;
        const int64_t from = at * o.ld + (PAIRED && r / kPaired % 2 == 1 ? o.second : 0);
        offset[j] = static_cast<uint32_t>((from + ((lane % 4) ^ row_swizzle(r)) * 8) * 2);
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

// FP32: 16 bytes are 4 k's, and the order of the k's is of no account, as both operands share it.
template <class T>
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
  if constexpr (std::is_same_v<T, float>) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same_v<T, Bf16>) {
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
__device__ __forceinline__ bool tile_at(const Product& p, int tiles_b, int id, TileAt* tile) {
  const int total = p.tiles_a * tiles_b * p.splits;
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
__device__ __forceinline__ bool tile_at(const Product& p, int tiles_b, TileAt* tile) {
  return tile_at(p, tiles_b, static_cast<int>(blockIdx.x), tile);
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

// The parts that a segment multiplies.  3: hi hi + hi lo + lo hi; 6: of three parts each those products that are not
// below 2^-26 of the whole.
template <int SEGMENTS>
__device__ __forceinline__ int part_of_a(int segment) {
  if constexpr (SEGMENTS == 3) return segment == 2;
  if constexpr (SEGMENTS == 6) return segment == 5 ? 2 : segment / 2 % 2;  // 0 0 1 1 0 2
  return 0;
}
template <int SEGMENTS>
__device__ __forceinline__ int part_of_b(int segment) {
  if constexpr (SEGMENTS == 3) return segment == 1;
  if constexpr (SEGMENTS == 6) return segment == 4 ? 2 : segment == 5 ? 0 : segment % 2;  // 0 1 0 1 2 0
  return 0;
}

// The sum of a tile over its split's k's (at least one stage).  PAIRED: tile.a counts tiles of 128 entries.
template <class T, int SEGMENTS, bool A_ROWS, bool B_ROWS, bool PAIRED = false>
__device__ __forceinline__ void multiply(const Product& p, const TileAt& tile, const Stages& range, uint16_t* lds, Accumulators& acc) {
  const int wave = wave_index(), lane = threadIdx.x % 64;
#pragma unroll
  for (int i = 0; i < kDown; ++i) {
#pragma unroll
    for (int j = 0; j < kAcross; ++j) acc[i][j] = f32x4{};
  }
  const int first = range.first, stages = range.count;
  const int64_t a0 = static_cast<int64_t>(tile.a) * (PAIRED ? kTile / 2 : kTile), b0 = static_cast<int64_t>(tile.b) * kTile;
  Loader<A_ROWS, PAIRED> load_a;
  Loader<B_ROWS> load_b;
  load_a.init(p.a, a0, wave, lane);
  load_b.init(p.b, b0, wave, lane);
  // bytes from the operand's start to the tile, and from a stage to the next
  const int64_t origin_a = (A_ROWS ? a0 * p.a.ld : a0) * 2, origin_b = (B_ROWS ? b0 * p.b.ld : b0) * 2;
  const int64_t next_a = (A_ROWS ? 1 : p.a.ld) * kDepth * 2, next_b = (B_ROWS ? 1 : p.b.ld) * kDepth * 2;
  int segment = 0, stage = 0;  // of the next load
  // one scalar base per half stage and 32-bit offsets
  const auto base_a = [&] {
    return scalar(reinterpret_cast<const char*>(p.a.part[part_of_a<SEGMENTS>(segment)]) + origin_a + (first + stage) * next_a);
  };
  const auto base_b = [&] {
    return scalar(reinterpret_cast<const char*>(p.b.part[part_of_b<SEGMENTS>(segment)]) + origin_b + (first + stage) * next_b);
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

// -------------------------------------------------------------- smaller tiles
// The same product in tiles of 128 x 128 or 64 x 64, four wavefronts each, two by two, and two or four workgroups on a
// unit: for outputs that tiles of 256 do not share out evenly.  Where an operand lies as rows of k a stage is 64 k's, so that
// they are read by whole lines of 128 bytes (4096 x 16384 x 4096, both as rows, tiles of 128: 710 -> 614 us), else 32, twice as many stages ahead
// (both as columns: 610 -> 592; tiles of 64 are faster with 64, 55 -> 47 us for 1024 x 5632 x 2048).  A step is 32 k's, and the next
// one's fragments are read meanwhile.
// SHAPE: the tile's size, or 65 and 66: tiles of 64 by two and by four times as many wavefronts, which share the depth and have a ring
// of stages each.  For launches of two workgroups or one to a unit, which has nothing else to do while a step's reads and the barrier
// are waited for (four times: 64 x 11264 x 2048 19.6 -> 13.0 us, 1024 x 1024 x 2816 24.6 -> 16.4, more stages ahead change nothing;
// twice: 32 x 22528 x 4096 51 -> 37 us, 128 x 11264 x 2048 19.6 -> 18.1; but 300 x 4096 x 768 10.6 -> 11.8, so from a depth of 1024 on).
template <int SHAPE>
struct Shape {
  static constexpr int kTileOf = SHAPE - SHAPE % 4, TILE = kTileOf;
  static constexpr int kWavesOf = TILE == 256 ? kWaves : 4;  // of a sharer: two along A, the others along B
  static constexpr int kSharers = 1 << SHAPE % 4;
  static constexpr int kThreadsOf = 64 * kWavesOf;           // of the epilogue
  static constexpr int kAllThreads = kThreadsOf * kSharers;
  static constexpr int kGroupsOf = TILE == 64 ? 4 : 2;       // wavefronts per SIMD
  static constexpr int kDownOf = TILE / 32;
  static constexpr int kAcrossOf = TILE == 256 ? kAcross : TILE / 32;
  static constexpr int kPairedOf = kDownOf * 8;  // PAIRED rows: entries of a wavefront's half
  static constexpr int kRing = kStages * 2 * TILE * kDepth;  // 16-bit elements: 4 stages of 32 k's, or 2 of 64
  static constexpr int kLds = kRing * kSharers;
  using Sums = f32x4[kDownOf][kAcrossOf];
};
static_assert(Shape<256>::kDownOf == kDown && Shape<256>::kPairedOf == kPaired, "one shape");

// 16-byte slots within an LDS row.  Rows of k (128 bytes) and columns of 64 alternate between the banks' halves by themselves.
__device__ __forceinline__ int small_row_swizzle(int row) { return row >> 1 & 7; }
template <int TILE, int HALVES>
__device__ __forceinline__ int small_column_swizzle(int k) {
  if constexpr (HALVES == 2) return (k >> 2 & 3) << 2;  // four k's to a lane: each group of lanes has its 64 of 256 bytes
  return TILE == 64 ? (k >> 1 & 1) << 1 | (k >> 3 & 1) << 2 : column_swizzle(k);
}

// HALVES: of an element, 2 for FP32.  Depths here and in a Product, but not an operand's own, count halves.
template <int TILE, int DEPTH, bool ROWS, bool PAIRED, int HALVES>
struct SmallLoader {
  using S = Shape<TILE>;  // its tile and wavefronts are all that is used
  static constexpr int kLoadsOf = TILE * DEPTH / 512 / S::kWavesOf;  // of 1 KB per wavefront and stage
  static constexpr int kRowsOfLoad = ROWS ? 8 : 512 / TILE / HALVES, kLanesOfRow = 64 / kRowsOfLoad;
  uint32_t offset[kLoadsOf];  // bytes from the stage's origin; columns: of the chunk alone
  int row;                    // of the first load
  __device__ __forceinline__ void init(const Operand& o, int64_t entry0, int wave, int lane) {
    row = wave * kLoadsOf * kRowsOfLoad + lane / kLanesOfRow;
#pragma unroll
    for (int j = 0; j < kLoadsOf; ++j) {
      const int r = row + j * kRowsOfLoad;
      if constexpr (ROWS) {
        const int entry = PAIRED ? r / (2 * S::kPairedOf) * S::kPairedOf + r % S::kPairedOf : r;
        const int64_t left = o.entries - 1 - entry0;
        const int64_t at = entry < left ? entry : left;
        const int64_t from = at * o.ld + (PAIRED && r / S::kPairedOf % 2 == 1 ? o.second : 0);
        offset[j] = static_cast<uint32_t>((from * HALVES + ((lane % 8) ^ small_row_swizzle(r)) * 8) * 2);
      } else {
        constexpr int kChunk = 8 / HALVES;  // entries of 16 bytes
        const int chunk = (lane % kLanesOfRow) ^ small_column_swizzle<TILE, HALVES>(r);
        const int64_t left = o.entries - kChunk - entry0;
        const int64_t at = chunk * kChunk < left ? chunk * kChunk : left;
        offset[j] = static_cast<uint32_t>(at * 2 * HALVES);
      }
    }
  }
  // Of load j of a stage; left: k's of it that the operand holds, less one.  Of a stage of 32 k's rows load them twice.
  __device__ __forceinline__ uint32_t at(const Operand& o, int left, bool half, int lane, int j) const {
    if constexpr (ROWS) {
      const bool upper = (((lane % 8) ^ small_row_swizzle(row + j * kRowsOfLoad)) & 4) != 0;
      return half && upper ? offset[j] - 64 : offset[j];
    } else {
      return offset[j] + static_cast<uint32_t>(min(row + j * kRowsOfLoad, left)) * static_cast<uint32_t>(o.ld * 2 * HALVES);
    }
  }
};

// Fragments of 16 entries and a step's 32 k's (FP32: 16), as Reader's.
template <int TILE, bool ROWS, int HALVES>
struct SmallReader {
  uint32_t at, column;
  __device__ __forceinline__ void init(int entry, int lane) {
    const int group = lane / 16, j = lane % 16;
    if constexpr (ROWS) {
      at = static_cast<uint32_t>((entry + j) * 128);
      column = static_cast<uint32_t>((group ^ small_row_swizzle(j)) * 16);
    } else if constexpr (HALVES == 2) {
      at = static_cast<uint32_t>(group * 4 * TILE + j % 4) * 4;
      column = static_cast<uint32_t>(((entry + j) / 4) ^ small_column_swizzle<TILE, HALVES>(group * 4)) * 16;
    } else {
      const int k = group * 8 + j / 4;
      at = static_cast<uint32_t>(k * TILE) * 2;
      column = static_cast<uint32_t>(((entry / 8 + j % 4 / 2) ^ small_column_swizzle<TILE, HALVES>(k)) * 8 + j % 2 * 4) * 2;
    }
  }
  __device__ __forceinline__ s16x8 read(uint32_t stage, int step, int f) const {
    if constexpr (ROWS) {
      return *(ATTNRES_LDS const s16x8*)(stage + at + (column ^ (step * 64u)) + f * 16 * 128);
    } else if constexpr (HALVES == 2) {
      const uint32_t from = stage + step * 32 * TILE * 2 + at + (column ^ (f * 64u));
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = *(ATTNRES_LDS const float*)(from + e * TILE * 4);
      return __builtin_bit_cast(s16x8, x);
    } else {
      const uint32_t from = stage + step * 32 * TILE * 2 + at + (column ^ (f * 32u));
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTNRES_LDS s16x4*)(from));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ATTNRES_LDS s16x4*)(from + 4 * TILE * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// As multiply(): the sum of a tile over its split's k's (at least one stage of 32 for each sharer).  False for the wavefronts that
// have no part in the epilogue: they end, and barriers are then met by the others alone.
template <int SHAPE, class T, int SEGMENTS, bool A_ROWS, bool B_ROWS, bool PAIRED>
__device__ __forceinline__ bool small_multiply(const Product& p, const TileAt& tile, const Stages& whole, uint16_t* lds,
                                               typename Shape<SHAPE>::Sums& acc) {
  using S = Shape<SHAPE>;
  constexpr int TILE = S::kTileOf, kDownOf = S::kDownOf, kAcrossOf = S::kAcrossOf, kSharers = S::kSharers;
  constexpr int kHalves = sizeof(T) / 2;
  constexpr int kSteps = A_ROWS || B_ROWS || TILE == 64 ? 2 : 1, kDepthOf = kSteps * kDepth, kStagesOf = kStages / kSteps;
  const int wave = wave_index() % S::kWavesOf, sharer = wave_index() / S::kWavesOf, lane = threadIdx.x % 64;
  // a sharer's stages, at least one; by pairs of 32 k's, so that lines stay whole
  const auto share = [&](int which) {
    const int pairs = (whole.count + 1) / 2, from = pairs * which / kSharers, to = pairs * (which + 1) / kSharers;
    return Stages{whole.first + 2 * from, min(2 * (to - from), whole.count - 2 * from)};
  };
  const Stages range = kSharers == 1 ? whole : share(sharer);
#pragma unroll
  for (int i = 0; i < kDownOf; ++i) {
#pragma unroll
    for (int j = 0; j < kAcrossOf; ++j) acc[i][j] = f32x4{};
  }
  const int first = range.first, stages = (range.count + kSteps - 1) / kSteps, total = stages * SEGMENTS;
  const bool odd = range.count % kSteps != 0;  // the last stage is one step
  const int64_t a0 = static_cast<int64_t>(tile.a) * (PAIRED ? TILE / 2 : TILE), b0 = static_cast<int64_t>(tile.b) * TILE;
  SmallLoader<TILE, kDepthOf, A_ROWS, PAIRED, kHalves> load_a;
  SmallLoader<TILE, kDepthOf, B_ROWS, false, kHalves> load_b;
  constexpr int kLoadsOf = decltype(load_a)::kLoadsOf;
  load_a.init(p.a, a0, wave, lane);
  load_b.init(p.b, b0, wave, lane);
  const int64_t origin_a = (A_ROWS ? a0 * p.a.ld : a0) * 2 * kHalves, origin_b = (B_ROWS ? b0 * p.b.ld : b0) * 2 * kHalves;
  const int64_t next_a = (A_ROWS ? 1 : p.a.ld) * kDepthOf * 2, next_b = (B_ROWS ? 1 : p.b.ld) * kDepthOf * 2;
  const int64_t from_a = origin_a + first * (next_a / kSteps), from_b = origin_b + first * (next_b / kSteps);
  const uint32_t lds0 = lds_byte(lds + sharer * S::kRing);
  constexpr uint32_t kB = TILE * kDepthOf * 2, kStageBytes = 2 * kB;
  const uint32_t slot = wave * (kLoadsOf * 1024);
  int segment = 0, stage = 0;  // of the next load
  const auto load = [&](uint32_t buffer) {
    const char* a = scalar(reinterpret_cast<const char*>(p.a.part[part_of_a<SEGMENTS>(segment)]) + from_a + stage * next_a);
    const char* b = scalar(reinterpret_cast<const char*>(p.b.part[part_of_b<SEGMENTS>(segment)]) + from_b + stage * next_b);
    const int64_t k = (first + static_cast<int64_t>(stage) * kSteps) * (kDepth / kHalves);
    const int left_a = __builtin_amdgcn_readfirstlane(static_cast<int>(p.a.depth - 1 - k));
    const int left_b = __builtin_amdgcn_readfirstlane(static_cast<int>(p.b.depth - 1 - k));
    const bool half = odd && stage + 1 == stages;
#pragma unroll
    for (int j = 0; j < kLoadsOf; ++j) load_lds(a, load_a.at(p.a, left_a, half, lane, j), buffer + slot + j * 1024);
#pragma unroll
    for (int j = 0; j < kLoadsOf; ++j) load_lds(b, load_b.at(p.b, left_b, half, lane, j), buffer + kB + slot + j * 1024);
    if (++stage == stages) stage = 0, ++segment;
  };
  SmallReader<TILE, A_ROWS, kHalves> read_a;
  SmallReader<TILE, B_ROWS, kHalves> read_b;
  read_a.init((wave % 2) * (16 * kDownOf), lane);
  read_b.init((wave / 2) * (16 * kAcrossOf), lane);
  struct Fragments {
    s16x8 a[kDownOf], b[kAcrossOf];
  };
  constexpr int kReads = kDownOf + kAcrossOf, kProducts = kDownOf * kAcrossOf;
  static_assert(kReads <= kProducts, "a read between two products at most");
  const auto read = [&](uint32_t buffer, int step, Fragments& f, int r) {
    if (r < kAcrossOf) f.b[r] = read_b.read(buffer + kB, step, r);
    else f.a[r - kAcrossOf] = read_a.read(buffer, step, r - kAcrossOf);
  };
  const auto read_all = [&](uint32_t buffer, Fragments& f) {
#pragma unroll
    for (int r = 0; r < kReads; ++r) read(buffer, 0, f, r);
  };
  // Every wavefront's reads from LDS are done and its loads have landed but for those of `ahead` stages.
  static_assert((kStagesOf - 1) * 2 * kLoadsOf < 64, "the counter has six bits");
  const auto arrived = [&](auto ahead) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(decltype(ahead)::value * 2 * kLoadsOf) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  const auto next = [&](int& at) {  // a stage's buffer
    const uint32_t buffer = lds0 + at;
    at = at + kStageBytes == kStagesOf * kStageBytes ? 0 : at + kStageBytes;
    return buffer;
  };
  const auto products = [&](Fragments& now, auto meanwhile) {
#pragma unroll
    for (int m = 0; m < kProducts; ++m) {
      f32x4& c = acc[m / kAcrossOf][m % kAcrossOf];
      c = mfma<T>(now.a[m / kAcrossOf], now.b[m % kAcrossOf], c);
      if (m * kReads / kProducts != (m + 1) * kReads / kProducts) meanwhile(m * kReads / kProducts);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const auto nothing = [](int) {};
  int loading = 0, reading = 0;  // LDS bytes of the next buffer
  for (int s = 0; s < kStagesOf && s < total; ++s) load(next(loading));
  if (total >= kStagesOf) arrived(std::integral_constant<int, kStagesOf - 1>{});
  else arrived(std::integral_constant<int, 0>{});
  Fragments lower, upper;
  uint32_t buffer = next(reading);
  read_all(buffer, lower);
  // From stage s to the next one, all of s in registers: its buffer gets the loads of a stage to come.
  const auto cross = [&](int s) {
    if (s + kStagesOf - 1 < total) arrived(std::integral_constant<int, kStagesOf - 2>{});
    else arrived(std::integral_constant<int, 0>{});
    if (s + kStagesOf < total) load(next(loading));
    buffer = next(reading);
  };
  if constexpr (kSteps == 2) {
    int within = 0;  // the stage's number in its segment
    for (int s = 0; s < total; ++s) {
      products(lower, [&](int r) { read(buffer, 1, upper, r); });
      const bool half = odd && within + 1 == stages;
      within = within + 1 == stages ? 0 : within + 1;
      if (s + 1 == total) {
        if (!half) products(upper, nothing);
        break;
      }
      cross(s);
      if (half) read_all(buffer, lower);
      else products(upper, [&](int r) { read(buffer, 0, lower, r); });
    }
  } else {
    int s = 0;
    for (; s + 2 < total; s += 2) {
      cross(s);
      products(lower, [&](int r) { read(buffer, 0, upper, r); });
      cross(s + 1);
      products(upper, [&](int r) { read(buffer, 0, lower, r); });
    }
    if (s + 1 < total) {
      cross(s);
      products(lower, [&](int r) { read(buffer, 0, upper, r); });
      products(upper, nothing);
    } else {
      products(lower, nothing);
    }
  }
  if constexpr (kSharers > 1) {
    // as many barriers as the sharer with the most stages has met
    int most = 0;
    for (int which = 0; which < kSharers; ++which) most = max(most, (share(which).count + kSteps - 1) / kSteps * SEGMENTS);
    for (int extra = total; extra < most; ++extra) __builtin_amdgcn_s_barrier();
    __syncthreads();
    // the first sharer adds up the sums, in order; the others are done
    f32x4* sums = reinterpret_cast<f32x4*>(lds);
    const auto place = [&](int which, int m) { return (((which - 1) * S::kWavesOf + wave) * kProducts + m) * 64 + lane; };
    if (sharer > 0) {
#pragma unroll
      for (int m = 0; m < kProducts; ++m) sums[place(sharer, m)] = acc[m / kAcrossOf][m % kAcrossOf];
    }
    __syncthreads();
    if (sharer > 0) return false;
#pragma unroll
    for (int which = 1; which < kSharers; ++which) {
#pragma unroll
      for (int m = 0; m < kProducts; ++m) acc[m / kAcrossOf][m % kAcrossOf] += sums[place(which, m)];
    }
  }
  __syncthreads();  // LDS is free for the epilogue
  return true;
}

template <int SHAPE, class T, int SEGMENTS, bool A_ROWS, bool B_ROWS, bool PAIRED = false>
__device__ __forceinline__ bool multiply_tile(const Product& p, const TileAt& tile, const Stages& range, uint16_t* lds,
                                              typename Shape<SHAPE>::Sums& acc) {
  if constexpr (SHAPE == 256) {
    multiply<T, SEGMENTS, A_ROWS, B_ROWS, PAIRED>(p, tile, range, lds, acc);
    return true;
  } else {
    return small_multiply<SHAPE, T, SEGMENTS, A_ROWS, B_ROWS, PAIRED>(p, tile, range, lds, acc);
  }
}

// ------------------------------------------------------------- few rows
// Operands that go straight to registers as they lie (any width and alignment): a lane holds 16 bytes of every 64 of its
// row; the order of the k's in a matrix instruction is of no account, as both operands share it.

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

// 16-byte slot of a staged output row of 512 bytes (CHUNKS of 16): a permutation per row, so that 32 lanes
// writing one chunk of 32 rows meet 32 different slots.
template <int CHUNKS = 32>
__device__ __forceinline__ int staged(int row, int chunk) { return row * CHUNKS + (chunk ^ (row & (CHUNKS - 1))); }

constexpr int kUnits = 256;  // compute units, one workgroup each

// How many parts the depth of a gradient product is cut into, so that its workgroups fill the chip: what takes the
// least time at 1.1 PFLOP/s for full rounds of workgroups and 4.5 TB/s for the FP32 partial sums that are
// written and read again (both as measured).  `direct`: one part needs no partial sums.  A part keeps at least 8 stages.
inline int choose_splits(int64_t tiles, int64_t depth, int segments, bool direct) {
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

}  // namespace layers
}  // namespace attnres_hip

#endif  // ATTNRES_PRODUCT_H
