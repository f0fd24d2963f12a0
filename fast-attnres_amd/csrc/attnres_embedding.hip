// attnres_embedding.hip - embedding lookup and its gradient by sorted tokens, for gfx950.
//
//   out[b, t] = scale W[tok[b, t]] + pos[t]
//   dW[v] = scale sum_{i: tok_i = v} dO_i,   dpos[t] = sum_b dO[b, t]
//
// Memory bound: the lookup reads one table row and writes one output row per token (32768 x 2048 BF16 of 131072 rows: 51
// us); the gradient reads dO once and writes the whole table (there 537 MB: 175 us, half of it the sort's four launches,
// which clear the table meanwhile at 5.7 TB/s).  The tokens are sorted (stable, least
// significant digit first), so every table row's sum is a run of the sorted list, added up in
// FP32 in the order of the tokens: no atomics on values, the same bits every time.

#include "attnres_layers.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

// Launches take fewer than 2^32 threads, 2^24 workgroups: one for 64 tokens in the sums and in the joins, which share their
// launch with the positions' workgroups.
constexpr int64_t kMaxTokens = int64_t{1} << 29;
constexpr int64_t kMaxPlaces = int64_t{1} << 26;
constexpr int64_t kMaxVocab = int64_t{1} << 30;
constexpr int64_t kMaxFwdBlocks = int64_t{1} << 23;
constexpr int64_t kMaxPlaceBlocks = int64_t{1} << 22;

__device__ __forceinline__ int64_t token_at(const void* tokens, int bytes, int64_t i) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[i] : static_cast<const int32_t*>(tokens)[i];
}

// Threads that share a row: the power of two that covers its chunks, 8..256.
int row_threads(int64_t width) {
  int threads = 8;
  while (threads < kBlock && threads * kVec < width) threads *= 2;
  return threads;
}

template <class W, class O>
__global__ void __launch_bounds__(kBlock) attnres_embedding_fwd_kernel(const void* __restrict__ tokens, int token_bytes, int64_t rows,
                                                                       int64_t length, const W* __restrict__ weight, int64_t vocab,
                                                                       int width, const W* __restrict__ positions, float scale,
                                                                       O* __restrict__ out, int threads,
                                                                       bool past) {
  const int per_block = kBlock / threads;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / threads; row < rows;
       row += static_cast<int64_t>(gridDim.x) * per_block) {
    const int64_t token = token_at(tokens, token_bytes, row);
    const bool known = token >= 0 && token < vocab;
    const W* from = weight + (known ? token : 0) * width;
    const W* place = positions != nullptr ? positions + row % length * width : nullptr;
    for (int c = (threadIdx.x % threads) * kVec; c < width; c += threads * kVec) {
      float x[kVec], p[kVec];
      load_chunk(from, c, width, x);
      if (place != nullptr) load_chunk(place, c, width, p);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        x[e] *= scale;
        if (place != nullptr) x[e] += p[e];
        if (!known) x[e] = __builtin_nanf("");
      }
      store_chunk(out + row * width, c, width, x, past);
    }
  }
}

// ------------------------------------------------------------------- sorting
// Keys are tokens (vocab for one outside the table, so those come last), values their
// positions.  A pass takes tiles of kTile entries, a wavefront each quarter of a tile: counts
// per digit, then a place for each entry -- the entries of smaller digits, of earlier tiles and
// of earlier wavefronts, then the order within the wavefront (ballots of the digit's bits).

constexpr int kTile = 1024;
constexpr int kWaves = kBlock / 64;
constexpr int kMaxDigits = 1024;

struct SortPass {
  const void* tokens;  // first pass: the tokens themselves
  int token_bytes;
  const uint32_t* keys_in;
  const uint32_t* values_in;
  uint32_t* keys_out;
  uint32_t* values_out;
  uint32_t* counts;  // [tiles][digits]
  uint32_t* totals;  // [digits] where a launch of its own scans the counts, else nullptr
  int64_t n;
  int64_t vocab;
  int shift, bits, tiles;
};

__device__ __forceinline__ uint32_t sort_key(const SortPass& p, int64_t i) {
  if (p.tokens == nullptr) return p.keys_in[i];
  const int64_t token = token_at(p.tokens, p.token_bytes, i);
  return static_cast<uint32_t>(token >= 0 && token < p.vocab ? token : p.vocab);
}

// Elements first .. end-1 of the table's gradient, to clear.
template <class W>
struct ZeroFill {
  W* to;
  int64_t first, end;
  bool past;  // the caches
};

template <class W>
__device__ __forceinline__ void zero_fill(const ZeroFill<W>& z, int64_t block, int64_t blocks) {
  float zero[kVec] = {};
  // each block a contiguous part: the gradient of 32768 tokens, 131072 x 2048 BF16, 181 -> 175 us against parts that lie
  // a grid apart, of 8192 tokens, 262144 x 2048, 270 -> 229
  const int64_t chunk = static_cast<int64_t>(blockDim.x) * kVec;
  const int64_t part = ((z.end - z.first + chunk - 1) / chunk + blocks - 1) / blocks * chunk;
  const int64_t from = z.first + block * part, end = min(from + part, z.end);
  for (int64_t i = from + threadIdx.x * kVec; i < end; i += chunk) {
    if (i + kVec <= end) {
      store8(z.to + i, zero, z.past);
    } else {
      for (int64_t e = i; e < end; ++e) z.to[e] = from_f32<W>(0.0f);
    }
  }
}

// Blocks 0 .. tiles-1 count their tile's digits, or place its entries; the others clear a part of the
// table's gradient meanwhile.
template <class W>
__global__ void __launch_bounds__(kBlock) attnres_sort_count_kernel(SortPass p, ZeroFill<W> zero) {
  const int tile = blockIdx.x;
  if (tile >= p.tiles) return zero_fill(zero, tile - p.tiles, gridDim.x - p.tiles);
  __shared__ uint32_t count[kMaxDigits];
  const int digits = 1 << p.bits;
  for (int d = threadIdx.x; d < digits; d += kBlock) count[d] = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(tile) * kTile;
  for (int k = threadIdx.x; k < kTile; k += kBlock) {
    if (first + k < p.n) atomicAdd(&count[sort_key(p, first + k) >> p.shift & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kBlock) p.counts[static_cast<int64_t>(tile) * digits + d] = count[d];
}

// Many tiles: counts to the sums of the tiles before, and all tiles' totals.  64 digits per workgroup, a
// sixteenth of the tiles per wavefront.  Up to kDirectTiles every tile makes these sums for itself, which
// saves the launches but grows with the square of the tiles.  Whole gradient of a 131072 x 1024 BF16 table, us,
// direct / with this launch: 16384 tokens 81 / 87, 32768 98 / 100, 65536 128 / 125, 262144 312 / 288, 1048576 1221 / 816.
constexpr int kScanBlock = 1024;
constexpr int kDirectTiles = 48;

__global__ void __launch_bounds__(kScanBlock) attnres_sort_scan_kernel(SortPass p) {
  constexpr int kParts = kScanBlock / 64;
  __shared__ uint32_t sums[kParts][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int digits = 1 << p.bits, d = blockIdx.x * 64 + lane;
  const int share = (p.tiles + kParts - 1) / kParts;
  const int first = min(wave * share, p.tiles), end = d < digits ? min(first + share, p.tiles) : first;
  uint32_t* counts = p.counts + d;
  uint32_t sum = 0;
#pragma unroll 16
  for (int t = first; t < end; ++t) sum += counts[static_cast<int64_t>(t) * digits];
  sums[wave][lane] = sum;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kParts; ++w) {
    before += w < wave ? sums[w][lane] : 0;
    total += sums[w][lane];
  }
#pragma unroll 16
  for (int t = first; t < end; ++t) {
    const uint32_t c = counts[static_cast<int64_t>(t) * digits];
    counts[static_cast<int64_t>(t) * digits] = before;
    before += c;
  }
  if (wave == 0 && d < digits) p.totals[d] = total;
}

template <class W>
__global__ void __launch_bounds__(kBlock) attnres_sort_place_kernel(SortPass p, ZeroFill<W> zero) {
  if (static_cast<int>(blockIdx.x) >= p.tiles) return zero_fill(zero, blockIdx.x - p.tiles, gridDim.x - p.tiles);
  __shared__ uint32_t place[kWaves][kMaxDigits];  // next place of the wavefront's entries of a digit
  __shared__ uint32_t block_sums[kWaves];
  const int tile = blockIdx.x, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int digits = 1 << p.bits, mask = digits - 1;
  constexpr int kQuarter = kTile / kWaves;
  for (int d = threadIdx.x; d < digits; d += kBlock) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) place[w][d] = 0;
  }
  __syncthreads();
  const int64_t first = static_cast<int64_t>(tile) * kTile + wave * kQuarter;
  uint32_t keys[kQuarter / 64];
#pragma unroll
  for (int k = 0; k < kQuarter / 64; ++k) {
    const int64_t i = first + k * 64 + lane;
    keys[k] = 0;
    if (i < p.n) {
      keys[k] = sort_key(p, i);
      atomicAdd(&place[wave][keys[k] >> p.shift & mask], 1u);
    }
  }
  __syncthreads();
  // thread t scans the digits [t * per, (t + 1) * per): totals over all tiles, then the
  // block's scan of the threads' sums
  const int per = (digits + kBlock - 1) / kBlock;
  uint32_t total[kMaxDigits / kBlock], before[kMaxDigits / kBlock];
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < kMaxDigits / kBlock; ++j) {
    total[j] = before[j] = 0;
    const int d = threadIdx.x * per + j;
    if (j < per && d < digits) {
      if (p.totals != nullptr) {
        before[j] = p.counts[static_cast<int64_t>(tile) * digits + d];
        total[j] = p.totals[d];
      } else {
#pragma unroll 8
        for (int t = 0; t < p.tiles; ++t) {
          const uint32_t c = p.counts[static_cast<int64_t>(t) * digits + d];
          total[j] += c;
          before[j] += t < tile ? c : 0;
        }
      }
      mine += total[j];
    }
  }
  uint32_t scan = mine;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const uint32_t other = __shfl_up(scan, step, 64);
    scan += lane >= step ? other : 0;
  }
  if (lane == 63) block_sums[wave] = scan;
  __syncthreads();
  uint32_t base = scan - mine;
  for (int w = 0; w < wave; ++w) base += block_sums[w];
#pragma unroll
  for (int j = 0; j < kMaxDigits / kBlock; ++j) {
    const int d = threadIdx.x * per + j;
    if (j < per && d < digits) {
      uint32_t next = base + before[j];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t c = place[w][d];
        place[w][d] = next;
        next += c;
      }
      base += total[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kQuarter / 64; ++k) {
    const int64_t i = first + k * 64 + lane;
    const bool live = i < p.n;
    const int digit = keys[k] >> p.shift & mask;
    uint64_t same = __ballot(live);
    for (int b = 0; b < p.bits; ++b) {
      const uint64_t set = __ballot(live && (digit >> b & 1));
      same &= digit >> b & 1 ? set : ~set;
    }
    const uint64_t below = same & ((uint64_t{1} << lane) - 1);
    uint32_t at = 0;
    if (live) at = place[wave][digit] + __popcll(below);
    __builtin_amdgcn_wave_barrier();  // every lane has read its place before one of them moves it
    if (live && below == 0) place[wave][digit] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (live) {
      p.keys_out[at] = keys[k];
      p.values_out[at] = p.tokens != nullptr ? static_cast<uint32_t>(i) : p.values_in[i];
    }
  }
}

// Up to kSmall tokens: one workgroup sorts them, pass after pass, and the others clear the table's gradient
// meanwhile: one launch for all of it (2048 tokens of a 32768 x 1024 FP32 table: 26 us, the time of its 134 MB; four
// launches 46).  Its 16 wavefronts take a sixteenth of the list each; between the passes the list lies in
// memory, which a barrier of the workgroup orders.  It sorts 1024 tokens in about 5.5 us.
constexpr int kSmall = 4096;
constexpr int kSmallBlock = 1024;
constexpr int kSmallWaves = kSmallBlock / 64;

__device__ __forceinline__ void sort_pass_small(const SortPass& p, uint32_t (*place)[kMaxDigits], uint32_t* block_sums) {
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int digits = 1 << p.bits, mask = digits - 1;
  for (int d = threadIdx.x; d < digits * kSmallWaves; d += kSmallBlock) place[d / digits][d % digits] = 0;
  __syncthreads();
  const int n = static_cast<int>(p.n);
  const int share = (n + kSmallBlock - 1) / kSmallBlock * 64;
  const int first = wave * share, end = min(first + share, n);
#pragma unroll 4
  for (int i = first + lane; i < end; i += 64) atomicAdd(&place[wave][sort_key(p, i) >> p.shift & mask], 1u);
  __syncthreads();
  const int d = threadIdx.x;  // at most as many digits as threads
  uint32_t mine = 0;
  if (d < digits) {
    for (int w = 0; w < kSmallWaves; ++w) mine += place[w][d];
  }
  uint32_t scan = mine;
#pragma unroll
  for (int step = 1; step < 64; step <<= 1) {
    const uint32_t other = __shfl_up(scan, step, 64);
    scan += lane >= step ? other : 0;
  }
  if (lane == 63) block_sums[wave] = scan;
  __syncthreads();
  if (d < digits) {
    uint32_t next = scan - mine;
    for (int w = 0; w < wave; ++w) next += block_sums[w];
    for (int w = 0; w < kSmallWaves; ++w) {
      const uint32_t c = place[w][d];
      place[w][d] = next;
      next += c;
    }
  }
  __syncthreads();
  constexpr int kRounds = 4;  // whose loads are under way together
  for (int i0 = first; i0 < end; i0 += 64 * kRounds) {
    uint32_t keys[kRounds], values[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int i = min(i0 + k * 64 + lane, n - 1);
      keys[k] = sort_key(p, i);
      values[k] = p.tokens != nullptr ? static_cast<uint32_t>(i) : p.values_in[i];
    }
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const bool live = i0 + k * 64 + lane < end;
      const int digit = keys[k] >> p.shift & mask;
      uint64_t same = __ballot(live);
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t set = __ballot(live && (digit >> b & 1));
        same &= digit >> b & 1 ? set : ~set;
      }
      const uint64_t below = same & ((uint64_t{1} << lane) - 1);
      uint32_t at = 0;
      if (live) at = place[wave][digit] + __popcll(below);
      __builtin_amdgcn_wave_barrier();  // every lane has read its place before one of them moves it
      if (live && below == 0) place[wave][digit] += __popcll(same);
      __builtin_amdgcn_wave_barrier();
      if (live) {
        p.keys_out[at] = keys[k];
        p.values_out[at] = values[k];
      }
    }
  }
  __syncthreads();
}

template <class W>
__global__ void __launch_bounds__(kSmallBlock) attnres_sort_small_kernel(SortPass p, int passes, uint32_t* keys0, uint32_t* values0,
                                                                         uint32_t* keys1, uint32_t* values1, ZeroFill<W> zero) {
  __shared__ uint32_t place[kSmallWaves][kMaxDigits];
  __shared__ uint32_t block_sums[kSmallWaves];
  if (blockIdx.x > 0) return zero_fill(zero, blockIdx.x - 1, gridDim.x - 1);
  for (int pass = 0; pass < passes; ++pass) {
    p.keys_out = pass % 2 ? keys1 : keys0;
    p.values_out = pass % 2 ? values1 : values0;
    sort_pass_small(p, place, block_sums);
    p.tokens = nullptr;
    p.keys_in = p.keys_out;
    p.values_in = p.values_out;
    p.shift += p.bits;
  }
}

// --------------------------------------------------------------------- sums
// The sorted list in pieces: a run of one token inside a piece is its table row's
// gradient; what crosses a piece's border goes to the piece's partial rows
// (0: began before the piece, 1: began in it and goes on) and is joined after.  About a thousand pieces: with twice as
// many the partial rows cost more than the shorter walks gain.  32768 x 2048 BF16 65 us, joined in 16.

struct Runs {
  const uint32_t* keys;
  const uint32_t* values;
  int64_t n;
  int64_t vocab;
  int piece;
  float* partial;  // [pieces][2][width]
};

constexpr int kAhead = 8;       // rows in flight per thread
constexpr int kMaxPiece = 64;

template <class O, class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_sum_kernel(Runs r, const O* __restrict__ grad_out, int width, float scale,
                                                                       W* __restrict__ grad_weight, int threads) {
  __shared__ uint32_t all_keys[kBlock / 8 * (kMaxPiece + 1)], all_values[kBlock / 8 * kMaxPiece];
  const int per_block = kBlock / threads, group = threadIdx.x / threads, member = threadIdx.x % threads;
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * per_block + group;
  const int64_t first = piece * r.piece;
  const int count = static_cast<int>(max(min(r.n - first, static_cast<int64_t>(r.piece)), int64_t{0}));
  uint32_t* keys = all_keys + group * (r.piece + 1);
  uint32_t* values = all_values + group * r.piece;
  for (int i = member; i < count; i += threads) {
    keys[i] = r.keys[first + i];
    values[i] = r.values[first + i];
  }
  if (member == 0 && count > 0) keys[count] = first + count < r.n ? r.keys[first + count] : ~0u;
  __syncthreads();
  const int c = (static_cast<int>(blockIdx.y) * threads + member) * kVec;
  if (count == 0 || c >= width) return;
  uint32_t key = keys[0];
  bool from_left = first > 0 && r.keys[first - 1] == key;
  float sum[kVec] = {};
  for (int i0 = 0; i0 < count; i0 += kAhead) {
    Chunk<O> rows[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      rows[j].load(grad_out + static_cast<int64_t>(values[min(i0 + j, count - 1)]) * width, c, width);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j >= count) break;
      if (key >= r.vocab) return;  // tokens outside the table: the rest of the list
      float x[kVec];
      rows[j].unpack(x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] += x[e];
      const uint32_t next = keys[i0 + j + 1];
      const bool goes_on = next == key;
      if (goes_on && i0 + j + 1 < count) continue;
      if (from_left || goes_on) {
        store_chunk(r.partial + (piece * 2 + (from_left ? 0 : 1)) * width, c, width, sum);
      } else {
        float y[kVec];
#pragma unroll
        for (int e = 0; e < kVec; ++e) y[e] = sum[e] * scale;
        store_chunk(grad_weight + static_cast<int64_t>(key) * width, c, width, y);
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] = 0.0f;
      from_left = false;
      key = next;
    }
  }
}

// The runs that cross pieces: for the piece where one begins, kJoinCols chunks of columns by kJoinGroups; a
// group adds up every kJoinGroups-th partial row of the run, the groups' sums are added in order.
constexpr int kJoinGroups = 8;
constexpr int kJoinCols = kBlock / kJoinGroups;

template <class W>
__device__ __forceinline__ void join_runs(const Runs& r, int64_t piece, int width, float scale, W* grad_weight,
                                          float (*sums)[kJoinCols * kVec]) {
  const int64_t first = piece * r.piece, end = first + r.piece;
  if (end >= r.n) return;
  const uint32_t key = r.keys[end - 1];
  if (key >= r.vocab || r.keys[end] != key) return;
  if (r.keys[first] == key && first > 0 && r.keys[first - 1] == key) return;  // began before this piece
  const int group = threadIdx.x / kJoinCols, member = threadIdx.x % kJoinCols;
  const int c = (static_cast<int>(blockIdx.y) * kJoinCols + member) * kVec;
  const int64_t pieces = (r.n + r.piece - 1) / r.piece;
  float sum[kVec] = {};
  if (group == 0) load_chunk(r.partial + (piece * 2 + 1) * width, c, width, sum);
  bool on = true;
  for (int64_t p = piece + 1 + group; on; p += kJoinGroups * 4) {
    float x[4][kVec];
    bool same[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = p + j * kJoinGroups < pieces ? p + j * kJoinGroups : pieces - 1;
      same[j] = p + j * kJoinGroups < pieces && r.keys[at * r.piece] == key;
      load_chunk(r.partial + at * 2 * width, c, width, x[j]);  // stale where the run has ended: not added
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      on = on && same[j];
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] = on ? sum[e] + x[j][e] : sum[e];
    }
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) sums[group][member * kVec + e] = sum[e];
  __syncthreads();
  if (group > 0 || c >= width) return;
  for (int g = 1; g < kJoinGroups; ++g) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] += sums[g][member * kVec + e];
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) sum[e] *= scale;
  store_chunk(grad_weight + static_cast<int64_t>(key) * width, c, width, sum);
}

// The positions' gradient is a sum over the batch for each of `length` rows: up to kInner sequences, beside the joins.
constexpr int64_t kInner = 64;

template <class O, class W>
struct Places {
  const O* grad_out;
  int64_t batch, length;
  W* grad_positions;
  int64_t rows;
};

// Blocks 0 .. join-1 join a piece's run, the others sum the positions' gradient over the batch.
template <class O, class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_join_kernel(Runs r, int width, float scale, W* __restrict__ grad_weight,
                                                                        int join, Places<O, W> place) {
  __shared__ float sums[kJoinGroups][kJoinCols * kVec];
  if (static_cast<int>(blockIdx.x) < join) return join_runs(r, blockIdx.x, width, scale, grad_weight, sums);
  const int c = (static_cast<int>(blockIdx.y) * kJoinCols + threadIdx.x % kJoinCols) * kVec;
  if (c >= width) return;
  const int64_t step = static_cast<int64_t>(gridDim.x - join) * kJoinGroups;
  for (int64_t t = static_cast<int64_t>(blockIdx.x - join) * kJoinGroups + threadIdx.x / kJoinCols; t < place.rows; t += step) {
    float sum[kVec] = {};
    if (t < place.length) {
#pragma unroll 4
      for (int64_t b = 0; b < place.batch; ++b) {
        float x[kVec];
        load_chunk(place.grad_out + (b * place.length + t) * width, c, width, x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum[e] += x[e];
      }
    }
    store_chunk(place.grad_positions + t * width, c, width, sum);
  }
}

// Larger batches: a lane adds up kInner sequences and then these sums, as one FP32 sum of a large batch loses what it counts (a
// million equal values: 1e-2 relative; ones end at 2^24).  Where the rows are too few for the chip the batch goes in parts, whose sums
// (FP32) a second launch adds up in order: BF16, us, one sum / parts, 512 sequences of 128 at 1024 columns 166 / 31, 4096 of
// 16 at 256 1227 / 26, 65536 of 1 at 64 18600 / 68.  A launch of its own, for the registers of the joins.
struct PlacePlan {
  int64_t share;  // sequences of a part
  int parts;
  int64_t bytes;
};
constexpr int64_t kPlaceRows = 4096;  // of 256 columns, eight to a workgroup: two workgroups per CU

template <class O, class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_batch_kernel(Places<O, W> place, PlacePlan plan, int width,
                                                                         float* __restrict__ partial) {
  const int c = (static_cast<int>(blockIdx.y) * kJoinCols + threadIdx.x % kJoinCols) * kVec;
  if (c >= width) return;
  // parts times length rows of sums, then the rows past length
  const int64_t sums_end = plan.parts * place.length, all = sums_end + place.rows - place.length;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kJoinGroups;
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * kJoinGroups + threadIdx.x / kJoinCols; r < all; r += step) {
    float sum[kVec] = {};
    if (r >= sums_end) {
      store_chunk(place.grad_positions + (place.length + r - sums_end) * width, c, width, sum);
      continue;
    }
    const int64_t part = plan.parts == 1 ? 0 : r / place.length, t = r - part * place.length;
    const int64_t first = part * plan.share, end = min(first + plan.share, place.batch);
    for (int64_t b0 = first; b0 < end; b0 += kInner) {
      float inner[kVec] = {};
      const int64_t b1 = min(b0 + kInner, end);
#pragma unroll 4
      for (int64_t b = b0; b < b1; ++b) {
        float x[kVec];
        load_chunk(place.grad_out + (b * place.length + t) * width, c, width, x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) inner[e] += x[e];
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] += inner[e];
    }
    if (plan.parts == 1) {
      store_chunk(place.grad_positions + t * width, c, width, sum);
    } else {
      store_chunk(partial + r * width, c, width, sum);
    }
  }
}

// The parts' sums of one row: kJoinGroups groups that add up every kJoinGroups-th part, then the groups in order.
template <class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_places_kernel(const float* __restrict__ partial, int parts, int64_t length,
                                                                          int width, W* __restrict__ grad_positions) {
  __shared__ float sums[kJoinGroups][kJoinCols * kVec];
  const int group = threadIdx.x / kJoinCols, member = threadIdx.x % kJoinCols;
  const int64_t t = blockIdx.x;
  const int c = (static_cast<int>(blockIdx.y) * kJoinCols + member) * kVec;
  float sum[kVec] = {};
#pragma unroll 4
  for (int p = group; p < parts; p += kJoinGroups) {
    float x[kVec];
    load_chunk(partial + (p * length + t) * width, c, width, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] += x[e];
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) sums[group][member * kVec + e] = sum[e];
  __syncthreads();
  if (group > 0 || c >= width) return;
  for (int g = 1; g < kJoinGroups; ++g) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] += sums[g][member * kVec + e];
  }
  store_chunk(grad_positions + t * width, c, width, sum);
}

// ---------------------------------------------------------------------- host

PlacePlan place_plan(int64_t batch, int64_t length, int64_t width) {
  const int64_t rows = length * ((width + kJoinCols * kVec - 1) / (kJoinCols * kVec));
  const int64_t most = (batch + kInner - 1) / kInner;  // whole inner sums
  const int64_t parts = rows > 0 ? std::max<int64_t>(std::min(kPlaceRows / rows, most), 1) : 1;
  PlacePlan p{};
  p.share = (batch + parts - 1) / parts;
  p.parts = static_cast<int>(p.share > 0 ? (batch + p.share - 1) / p.share : 1);
  p.bytes = p.parts > 1 ? (4 * p.parts * length * width + 255) / 256 * 256 : 0;
  return p;
}

struct Plan {
  int tiles, bits, passes, piece;
  int64_t pieces, keys[2], values[2], counts, totals, partial, bytes;
};

// The workspace: the positions' sums, then the table's part.
Plan plan(int64_t batch, int64_t length, int64_t vocab, int64_t width) {
  const int64_t n = batch * length;
  Plan p{};
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
  p.passes = (bits + 9) / 10;           // digits of at most 10 bits
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tiles = static_cast<int>((n + kTile - 1) / kTile);
  // pieces of 8 to 64 entries, about a thousand of them
  p.piece = 8;
  while (p.piece < kMaxPiece && p.piece * 1024 < n) p.piece *= 2;
  p.pieces = (n + p.piece - 1) / p.piece;
  int64_t at = place_plan(batch, length, width).bytes;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  for (int k = 0; k < 2; ++k) p.keys[k] = take(4 * n), p.values[k] = take(4 * n);
  p.counts = take(4 * (int64_t{1} << p.bits) * p.tiles);
  p.totals = take(4 * (int64_t{1} << p.bits));
  p.partial = take(4 * p.pieces * 2 * width);
  p.bytes = at;
  return p;
}

template <class O, class W>
void embedding_backward(const void* grad_out, const void* tokens, int token_bytes, int64_t batch, int64_t length, int64_t vocab,
                        int64_t width, float scale, void* grad_weight, void* grad_positions, int64_t position_rows,
                        char* workspace, hipStream_t stream) {
  const int64_t n = batch * length;
  const int threads = row_threads(width), per_block = kBlock / threads;
  const unsigned slabs = static_cast<unsigned>((width + threads * kVec - 1) / (threads * kVec));
  Runs runs{};
  int join = 0;
  if (grad_weight != nullptr) {
    const Plan p = plan(batch, length, vocab, width);
    const int64_t elements = vocab * width;
    ZeroFill<W> zero{static_cast<W*>(grad_weight), 0, elements, elements * static_cast<int64_t>(sizeof(W)) >= kPastCaches};
    uint32_t* keys[2];
    uint32_t* values[2];
    for (int k = 0; k < 2; ++k) {
      keys[k] = reinterpret_cast<uint32_t*>(workspace + p.keys[k]);
      values[k] = reinterpret_cast<uint32_t*>(workspace + p.values[k]);
    }
    SortPass s{};
    s.token_bytes = token_bytes;
    s.counts = reinterpret_cast<uint32_t*>(workspace + p.counts);
    if (p.tiles > kDirectTiles) s.totals = reinterpret_cast<uint32_t*>(workspace + p.totals);
    s.n = n;
    s.vocab = vocab;
    s.bits = p.bits;
    s.tiles = p.tiles;
    const int last = (p.passes - 1) % 2;
    if (n <= kSmall) {
      s.tokens = tokens;
      const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((elements + 8191) / 8192, 512));
      hipLaunchKernelGGL((attnres_sort_small_kernel<W>), dim3(1 + blocks), dim3(kSmallBlock), 0, stream, s, n > 0 ? p.passes : 0,
                         keys[0], values[0], keys[1], values[1], zero);
    } else {
      // every launch of the sort, which leaves most of the chip idle, clears its share of the table's gradient
      const int64_t share = (elements / (2 * p.passes) + 255) / 256 * 256;
      const unsigned fill = static_cast<unsigned>(std::min<int64_t>(share / (kBlock * kVec) + 1, 2048));
      for (int pass = 0; pass < p.passes; ++pass) {
        s.tokens = pass == 0 ? tokens : nullptr;
        s.keys_in = keys[(pass + 1) % 2];
        s.values_in = values[(pass + 1) % 2];
        s.keys_out = keys[pass % 2];
        s.values_out = values[pass % 2];
        s.shift = pass * p.bits;
        const auto next_share = [&](bool rest) {
          zero.first = pass == 0 && !rest ? 0 : zero.end;
          zero.end = rest && pass == p.passes - 1 ? elements : std::min(zero.first + share, elements);
        };
        next_share(false);
        hipLaunchKernelGGL((attnres_sort_count_kernel<W>), dim3(p.tiles + fill), dim3(kBlock), 0, stream, s, zero);
        if (s.totals != nullptr) {
          hipLaunchKernelGGL(attnres_sort_scan_kernel, dim3(((1 << s.bits) + 63) / 64), dim3(kScanBlock), 0, stream, s);
        }
        next_share(true);
        hipLaunchKernelGGL((attnres_sort_place_kernel<W>), dim3(p.tiles + fill), dim3(kBlock), 0, stream, s, zero);
      }
    }
    runs = Runs{keys[last], values[last], n, vocab, p.piece, reinterpret_cast<float*>(workspace + p.partial)};
    if (n > 0) {
      join = static_cast<int>(p.pieces);
      hipLaunchKernelGGL((attnres_embedding_sum_kernel<O, W>), dim3((join + per_block - 1) / per_block, slabs), dim3(kBlock), 0, stream, runs,
                         static_cast<const O*>(grad_out), static_cast<int>(width), scale, static_cast<W*>(grad_weight), threads);
    }
  }
  const Places<O, W> place{static_cast<const O*>(grad_out), batch, length, static_cast<W*>(grad_positions),
                           grad_positions != nullptr ? position_rows : 0};
  const bool large = place.rows > 0 && batch > kInner;
  const unsigned columns = static_cast<unsigned>((width + kJoinCols * kVec - 1) / (kJoinCols * kVec));
  const auto blocks_of = [](int64_t rows) { return std::min((rows + kJoinGroups - 1) / kJoinGroups, kMaxPlaceBlocks); };
  const int64_t blocks = join + (large ? 0 : blocks_of(place.rows));
  if (blocks > 0) {
    hipLaunchKernelGGL((attnres_embedding_join_kernel<O, W>), dim3(static_cast<unsigned>(blocks), columns), dim3(kBlock), 0, stream,
                       runs, static_cast<int>(width), scale, static_cast<W*>(grad_weight), join, place);
  }
  if (large) {
    const PlacePlan p = workspace != nullptr ? place_plan(batch, length, width) : PlacePlan{batch, 1, 0};
    float* partial = reinterpret_cast<float*>(workspace);
    hipLaunchKernelGGL((attnres_embedding_batch_kernel<O, W>),
                       dim3(static_cast<unsigned>(blocks_of(p.parts * length + position_rows - length)), columns), dim3(kBlock), 0, stream,
                       place, p, static_cast<int>(width), partial);
    if (p.parts > 1) {
      hipLaunchKernelGGL((attnres_embedding_places_kernel<W>), dim3(static_cast<unsigned>(length), columns), dim3(kBlock), 0, stream,
                         partial, p.parts, length, static_cast<int>(width), static_cast<W*>(grad_positions));
    }
  }
}

int check_embedding(int64_t batch, int64_t length, int64_t vocab, int64_t width, int weight_dtype, int out_dtype,
                    int token_bytes) {
  if (batch < 0 || length < 0 || (length > 0 && batch > kMaxTokens / length)) {
    return layer_error(ATTNRES_ERR_SHAPE, "batch=%lld x length=%lld outside 0..2^29 tokens", (long long)batch, (long long)length);
  }
  if (vocab < 1 || vocab > kMaxVocab) return layer_error(ATTNRES_ERR_SHAPE, "vocab=%lld outside 1..2^30", (long long)vocab);
  if (width < 1 || width > ATTNRES_MAX_WIDTH) {
    return layer_error(ATTNRES_ERR_SHAPE, "width=%lld outside 1..%d", (long long)width, ATTNRES_MAX_WIDTH);
  }
  if (!dtype_known(weight_dtype) || !dtype_known(out_dtype)) return layer_error(ATTNRES_ERR_SHAPE, "unknown dtype");
  if (token_bytes != 4 && token_bytes != 8) return layer_error(ATTNRES_ERR_SHAPE, "tokens must be int32 or int64");
  return ATTNRES_OK;
}

// W: the table's type, O: the output's; every pair is a use (a table in FP32 and a
// stream in 16 bits under autocast, or a 16-bit table read into an FP32 stream).
template <class F>
void with_types(int weight_dtype, int out_dtype, F f) {
  const auto second = [&](auto w) {
    if (out_dtype == ATTNRES_F32) return f(w, float{});
    if (out_dtype == ATTNRES_BF16) return f(w, Bf16{});
    return f(w, F16{});
  };
  if (weight_dtype == ATTNRES_F32) return second(float{});
  if (weight_dtype == ATTNRES_BF16) return second(Bf16{});
  return second(F16{});
}

}  // namespace
}  // namespace layers
}  // namespace attnres_hip

using namespace attnres_hip;
using namespace attnres_hip::layers;

extern "C" {

int attnres_hip_embedding_forward(const void* tokens, int token_bytes, int64_t batch, int64_t length, const void* weight,
                                  int64_t vocab, int64_t width, int weight_dtype, const void* positions, float scale,
                                  void* out, int out_dtype, void* stream) {
  if (const int status = check_embedding(batch, length, vocab, width, weight_dtype, out_dtype, token_bytes)) return status;
  const int64_t rows = batch * length;
  if (rows == 0) return ATTNRES_OK;
  if (tokens == nullptr || weight == nullptr || out == nullptr) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "tokens, weight or out is NULL");
  }
  const int threads = row_threads(width), per_block = kBlock / threads;
  with_types(weight_dtype, out_dtype, [&](auto w, auto o) {
    using W = decltype(w);
    using O = decltype(o);
    const int64_t blocks = std::min((rows + per_block - 1) / per_block, kMaxFwdBlocks);
    hipLaunchKernelGGL((attnres_embedding_fwd_kernel<W, O>), dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0,
                       static_cast<hipStream_t>(stream), tokens, token_bytes, rows, length, static_cast<const W*>(weight), vocab,
                       static_cast<int>(width), static_cast<const W*>(positions), scale, static_cast<O*>(out), threads,
                       rows * width * static_cast<int64_t>(sizeof(O)) >= kPastCaches);
  });
  return layer_launch_status("embedding forward");
}

int64_t attnres_hip_embedding_workspace_bytes(int64_t batch, int64_t length, int64_t vocab, int64_t width) {
  if (batch < 0 || length < 0 || (length > 0 && batch > kMaxTokens / length) || vocab < 1 || vocab > kMaxVocab || width < 1 ||
      width > ATTNRES_MAX_WIDTH) {
    return -1;
  }
  return plan(batch, length, vocab, width).bytes;
}

int64_t attnres_hip_embedding_positions_workspace_bytes(int64_t batch, int64_t length, int64_t width) {
  if (batch < 0 || length < 0 || (length > 0 && batch > kMaxTokens / length) || width < 1 || width > ATTNRES_MAX_WIDTH) return -1;
  return place_plan(batch, length, width).bytes;
}

int attnres_hip_embedding_backward(const void* grad_out, int out_dtype, const void* tokens, int token_bytes, int64_t batch,
                                   int64_t length, int64_t vocab, int64_t width, int weight_dtype, float scale,
                                   void* grad_weight, void* grad_positions, int64_t position_rows, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (const int status = check_embedding(batch, length, vocab, width, weight_dtype, out_dtype, token_bytes)) return status;
  if (batch * length > 0 && (grad_out == nullptr || tokens == nullptr)) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "grad_out or tokens is NULL");
  }
  if (grad_positions != nullptr && (position_rows < length || position_rows > kMaxPlaces)) {
    return layer_error(ATTNRES_ERR_SHAPE, "position_rows=%lld outside length=%lld..2^26", (long long)position_rows,
                       (long long)length);
  }
  const int64_t need = attnres_hip_embedding_workspace_bytes(batch, length, vocab, width);
  if (grad_weight != nullptr && need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                       (long long)need);
  }
  if (grad_weight == nullptr && workspace != nullptr &&
      workspace_bytes < attnres_hip_embedding_positions_workspace_bytes(batch, length, width)) {
    workspace = nullptr;  // as without one
  }
  with_types(weight_dtype, out_dtype, [&](auto w, auto o) {
    embedding_backward<decltype(o), decltype(w)>(grad_out, tokens, token_bytes, batch, length, vocab, width, scale,
                                                 grad_weight, grad_positions, position_rows, static_cast<char*>(workspace),
                                                 static_cast<hipStream_t>(stream));
  });
  return layer_launch_status("embedding backward");
}

}  // extern "C"
