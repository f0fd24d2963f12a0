// attnres_embedding.hip - embedding lookup and its gradient by sorted tokens, for gfx950.
//
//   out[b, t] = scale W[tok[b, t]] + pos[t]
//   dW[v] = scale sum_{i: tok_i = v} dO_i,   dpos[t] = sum_b dO[b, t]
//
// Memory bound: the lookup reads one table row and writes one output row per token; the
// gradient reads dO once and writes the whole table.  The tokens are sorted (stable, least
// significant digit first), so every table row's sum is a run of the sorted list, added up in
// FP32 in the order of the tokens: no atomics on values, the same bits every time.

#include "attnres_layers.h"

#include <algorithm>

namespace attnres_hip {
namespace layers {
namespace {

constexpr int64_t kMaxTokens = int64_t{1} << 30;  // positions are sorted as 32-bit numbers
constexpr int64_t kMaxVocab = int64_t{1} << 30;

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
                                                                       O* __restrict__ out, int threads) {
  const int per_block = kBlock / threads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / threads;
  if (row >= rows) return;
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
    store_chunk(out + row * width, c, width, x);
  }
}

// ------------------------------------------------------------------- sorting
// Keys are tokens (vocab for one outside the table, so those come last), values their
// positions.  A pass takes tiles of kTile entries, a wavefront each quarter of a tile: counts
// per digit, then a place for each entry -- the entries of smaller digits, of earlier tiles and
// of earlier wavefronts, then the order within the wavefront (ballots of the digit's bits).

constexpr int kTile = 2048;
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
  int64_t n;
  int64_t vocab;
  int shift, bits, tiles;
};

__device__ __forceinline__ uint32_t sort_key(const SortPass& p, int64_t i) {
  if (p.tokens == nullptr) return p.keys_in[i];
  const int64_t token = token_at(p.tokens, p.token_bytes, i);
  return static_cast<uint32_t>(token >= 0 && token < p.vocab ? token : p.vocab);
}

template <class W>
struct ZeroFill {
  W* to;
  int64_t elements;
};

template <class W>
__device__ __forceinline__ void zero_fill(const ZeroFill<W>& z, int64_t block, int64_t blocks) {
  float zero[kVec] = {};
  const int64_t step = blocks * kBlock * kVec;
  for (int64_t i = (block * kBlock + threadIdx.x) * kVec; i < z.elements; i += step) {
    if (i + kVec <= z.elements) {
      store8(z.to + i, zero);
    } else {
      for (int64_t e = i; e < z.elements; ++e) z.to[e] = from_f32<W>(0.0f);
    }
  }
}

// Blocks 0 .. tiles-1 count their tile's digits; in the first pass the others
// clear the table's gradient meanwhile.
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

__global__ void __launch_bounds__(kBlock) attnres_sort_place_kernel(SortPass p) {
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
#pragma unroll 8
      for (int t = 0; t < p.tiles; ++t) {
        const uint32_t c = p.counts[static_cast<int64_t>(t) * digits + d];
        total[j] += c;
        before[j] += t < tile ? c : 0;
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

// --------------------------------------------------------------------- sums
// The sorted list in pieces: a run of one token inside a piece is its table row's
// gradient; what crosses a piece's border goes to the piece's partial rows
// (0: began before the piece, 1: began in it and goes on) and is joined after.

struct Runs {
  const uint32_t* keys;
  const uint32_t* values;
  int64_t n;
  int64_t vocab;
  int piece;
  float* partial;  // [pieces][2][width]
};

constexpr int kAhead = 4;  // rows in flight per thread

template <class O, class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_sum_kernel(Runs r, const O* __restrict__ grad_out, int width, float scale,
                                                                       W* __restrict__ grad_weight, int threads) {
  const int per_block = kBlock / threads;
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / threads;
  const int64_t first = piece * r.piece;
  const int c = (static_cast<int>(blockIdx.y) * threads + threadIdx.x % threads) * kVec;
  if (first >= r.n || c >= width) return;
  const int count = static_cast<int>(r.n - first < r.piece ? r.n - first : r.piece);
  bool from_left = first > 0 && r.keys[first - 1] == r.keys[first];
  float sum[kVec] = {};
  uint32_t key = r.keys[first];
  for (int i0 = 0; i0 < count; i0 += kAhead) {
    float x[kAhead][kVec];
    uint32_t next[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = first + (i0 + j < count ? i0 + j : count - 1);
      load_chunk(grad_out + static_cast<int64_t>(r.values[i]) * width, c, width, x[j]);
      next[j] = i + 1 < r.n ? r.keys[i + 1] : ~0u;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j >= count) break;
      if (key >= r.vocab) return;  // tokens outside the table: the rest of the list
#pragma unroll
      for (int e = 0; e < kVec; ++e) sum[e] += x[j][e];
      const bool goes_on = next[j] == key;
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
      key = next[j];
    }
  }
}

// The runs that cross pieces: the piece where one begins adds up the others' partial rows.
template <class W>
__global__ void __launch_bounds__(kBlock) attnres_embedding_join_kernel(Runs r, int width, float scale, W* __restrict__ grad_weight,
                                                                        int threads) {
  const int per_block = kBlock / threads;
  const int64_t piece = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / threads;
  const int64_t first = piece * r.piece, end = first + r.piece;
  const int c = (static_cast<int>(blockIdx.y) * threads + threadIdx.x % threads) * kVec;
  if (end >= r.n || c >= width) return;
  const uint32_t key = r.keys[end - 1];
  if (key >= r.vocab || r.keys[end] != key) return;
  if (r.keys[first] == key && first > 0 && r.keys[first - 1] == key) return;  // began before this piece
  float sum[kVec];
  load_chunk(r.partial + (piece * 2 + 1) * width, c, width, sum);
  for (int64_t p = piece + 1; p * r.piece < r.n && r.keys[p * r.piece] == key; ++p) {
    float x[kVec];
    load_chunk(r.partial + p * 2 * width, c, width, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) sum[e] += x[e];
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) sum[e] *= scale;
  store_chunk(grad_weight + static_cast<int64_t>(key) * width, c, width, sum);
}

template <class O, class W>
__global__ void __launch_bounds__(kBlock) attnres_positions_kernel(const O* __restrict__ grad_out, int64_t batch, int64_t length,
                                                                   int width, W* __restrict__ grad_positions, int64_t position_rows,
                                                                   int threads) {
  const int per_block = kBlock / threads;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * per_block + threadIdx.x / threads;
  if (t >= position_rows) return;
  for (int c = (threadIdx.x % threads) * kVec; c < width; c += threads * kVec) {
    float sum[kVec] = {};
    if (t < length) {
#pragma unroll 4
      for (int64_t b = 0; b < batch; ++b) {
        float x[kVec];
        load_chunk(grad_out + (b * length + t) * width, c, width, x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) sum[e] += x[e];
      }
    }
    store_chunk(grad_positions + t * width, c, width, sum);
  }
}

// ---------------------------------------------------------------------- host

struct Plan {
  int tiles, bits, passes, piece;
  int64_t pieces, keys[2], values[2], counts, partial, bytes;
};

Plan plan(int64_t n, int64_t vocab, int64_t width) {
  Plan p{};
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;  // keys 0 .. vocab
  p.passes = (bits + 9) / 10;           // digits of at most 10 bits
  p.bits = (bits + p.passes - 1) / p.passes;
  p.tiles = static_cast<int>((n + kTile - 1) / kTile);
  // pieces of 4 to 64 entries, about a thousand of them
  p.piece = 4;
  while (p.piece < 64 && p.piece * 1024 < n) p.piece *= 2;
  p.pieces = (n + p.piece - 1) / p.piece;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  for (int k = 0; k < 2; ++k) p.keys[k] = take(4 * n), p.values[k] = take(4 * n);
  p.counts = take(4 * (int64_t{1} << p.bits) * p.tiles);
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
  if (grad_weight != nullptr) {
    const Plan p = plan(n, vocab, width);
    const ZeroFill<W> zero{static_cast<W*>(grad_weight), vocab * width};
    const int64_t fill = std::min<int64_t>((zero.elements + kBlock * kVec - 1) / (kBlock * kVec), 2048);
    uint32_t* keys[2];
    uint32_t* values[2];
    for (int k = 0; k < 2; ++k) {
      keys[k] = reinterpret_cast<uint32_t*>(workspace + p.keys[k]);
      values[k] = reinterpret_cast<uint32_t*>(workspace + p.values[k]);
    }
    SortPass s{};
    s.token_bytes = token_bytes;
    s.counts = reinterpret_cast<uint32_t*>(workspace + p.counts);
    s.n = n;
    s.vocab = vocab;
    s.bits = p.bits;
    s.tiles = p.tiles;
    for (int pass = 0; pass < p.passes; ++pass) {
      s.tokens = pass == 0 ? tokens : nullptr;
      s.keys_in = keys[(pass + 1) % 2];
      s.values_in = values[(pass + 1) % 2];
      s.keys_out = keys[pass % 2];
      s.values_out = values[pass % 2];
      s.shift = pass * p.bits;
      const unsigned grid = static_cast<unsigned>(p.tiles + (pass == 0 ? fill : 0));
      if (grid > 0) hipLaunchKernelGGL((attnres_sort_count_kernel<W>), dim3(grid), dim3(kBlock), 0, stream, s, zero);
      if (n > 0) hipLaunchKernelGGL(attnres_sort_place_kernel, dim3(p.tiles), dim3(kBlock), 0, stream, s);
    }
    if (n > 0) {
      const Runs r{s.keys_out, s.values_out, n, vocab, p.piece, reinterpret_cast<float*>(workspace + p.partial)};
      const dim3 grid(static_cast<unsigned>((p.pieces + per_block - 1) / per_block),
                      static_cast<unsigned>((width + threads * kVec - 1) / (threads * kVec)));
      hipLaunchKernelGGL((attnres_embedding_sum_kernel<O, W>), grid, dim3(kBlock), 0, stream, r,
                         static_cast<const O*>(grad_out), static_cast<int>(width), scale, static_cast<W*>(grad_weight), threads);
      hipLaunchKernelGGL((attnres_embedding_join_kernel<W>), grid, dim3(kBlock), 0, stream, r, static_cast<int>(width), scale,
                         static_cast<W*>(grad_weight), threads);
    }
  }
  if (grad_positions != nullptr && position_rows > 0) {
    hipLaunchKernelGGL((attnres_positions_kernel<O, W>), dim3(static_cast<unsigned>((position_rows + per_block - 1) / per_block)),
                       dim3(kBlock), 0, stream, static_cast<const O*>(grad_out), batch, length, static_cast<int>(width),
                       static_cast<W*>(grad_positions), position_rows, threads);
  }
}

int check_embedding(int64_t batch, int64_t length, int64_t vocab, int64_t width, int weight_dtype, int out_dtype,
                    int token_bytes) {
  if (batch < 0 || length < 0 || (length > 0 && batch > kMaxTokens / length)) {
    return layer_error(ATTNRES_ERR_SHAPE, "batch=%lld x length=%lld outside 0..2^30 tokens", (long long)batch, (long long)length);
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
    hipLaunchKernelGGL((attnres_embedding_fwd_kernel<W, O>), dim3(static_cast<unsigned>((rows + per_block - 1) / per_block)),
                       dim3(kBlock), 0, static_cast<hipStream_t>(stream), tokens, token_bytes, rows, length,
                       static_cast<const W*>(weight), vocab, static_cast<int>(width), static_cast<const W*>(positions), scale,
                       static_cast<O*>(out), threads);
  });
  return layer_launch_status("embedding forward");
}

int64_t attnres_hip_embedding_workspace_bytes(int64_t batch, int64_t length, int64_t vocab, int64_t width) {
  if (batch < 0 || length < 0 || (length > 0 && batch > kMaxTokens / length) || vocab < 1 || vocab > kMaxVocab || width < 1 ||
      width > ATTNRES_MAX_WIDTH) {
    return -1;
  }
  return plan(batch * length, vocab, width).bytes;
}

int attnres_hip_embedding_backward(const void* grad_out, int out_dtype, const void* tokens, int token_bytes, int64_t batch,
                                   int64_t length, int64_t vocab, int64_t width, int weight_dtype, float scale,
                                   void* grad_weight, void* grad_positions, int64_t position_rows, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (const int status = check_embedding(batch, length, vocab, width, weight_dtype, out_dtype, token_bytes)) return status;
  if (batch * length > 0 && (grad_out == nullptr || tokens == nullptr)) {
    return layer_error(ATTNRES_ERR_NULL_POINTER, "grad_out or tokens is NULL");
  }
  if (grad_positions != nullptr && (position_rows < length || position_rows > kMaxTokens)) {
    return layer_error(ATTNRES_ERR_SHAPE, "position_rows=%lld outside length=%lld..2^30", (long long)position_rows,
                       (long long)length);
  }
  const int64_t need = attnres_hip_embedding_workspace_bytes(batch, length, vocab, width);
  if (grad_weight != nullptr && need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    return layer_error(ATTNRES_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                       (long long)need);
  }
  with_types(weight_dtype, out_dtype, [&](auto w, auto o) {
    embedding_backward<decltype(o), decltype(w)>(grad_out, tokens, token_bytes, batch, length, vocab, width, scale,
                                                 grad_weight, grad_positions, position_rows, static_cast<char*>(workspace),
                                                 static_cast<hipStream_t>(stream));
  });
  return layer_launch_status("embedding backward");
}

}  // extern "C"
