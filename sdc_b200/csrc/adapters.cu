// Low-rank adapters of many requests beside a shared projection, and their
// gradients. A token t of adapter g = g(t) adds
//
//   y_t = base_t + B_g s_t,   s_t = scale_g A_g x_t,   A_g [r, K], B_g [N, r]
//
// and with d_t = scale_g B_g^T dy_t
//
//   dx_t = A_g^T d_t,   dA_g = sum_t d_t (x_t)^T,   dB_g = sum_t dy_t (s_t)^T
//   (s_t and d_t both carry the scale once).
//
// Three kernels serve both directions:
//   shrink  low[t, :] = scale_g * rows of a streamed [T, width] matrix times
//           the adapter's weight (x by A, dy by B)
//   expand  out[t, :] = base[t, :] + low[t, :] times the other weight
//   outer   dW_g = sum over g's tokens of streamed row x low row
//
// A rank r of a few dozen against widths of thousands leaves about r flops a
// byte of the streamed matrix: all three are bound by reading x, base and dy
// and writing y and dx once, not by the tensor cores. Tokens of one adapter
// are gathered into tiles of 64 rows (16 when adapters have few tokens, as in
// decoding, where the weights are the traffic); low ranks are summed over the
// width in fp32, across the blocks of a cluster through distributed shared
// memory, so nothing is added in an order that changes.
//
// `low` is kept as two 16-bit planes, hi = round(v) and lo = round(v - hi):
// the tensor cores take 16-bit operands, and the second product then loses
// 2^-17 of v (2^-22 in fp16) rather than 2^-9, for one more multiply on pipes
// that wait for memory anyway.
#include <algorithm>
#include <atomic>
#include <climits>

#include "mma.cuh"

namespace sdc {
namespace {

constexpr int kAdapterThreads = 128;
constexpr int kMaxRank = 256;
constexpr int kMaxSplit = 8;

struct Tile {
  int32_t start, count, adapter;
};

struct AdapterParams {
  const void* rows_in;       // streamed matrix [tokens, width]
  int64_t row_stride;
  int64_t tokens;
  const int32_t* rows;       // token of each slot
  const Tile* tiles;
  const int32_t* group_offsets;  // outer: slots of adapter g are [g, g + 1)
  int adapters;
  const void* weight;
  int rank, rank_pad;        // rank_pad: multiple of 16
  int64_t width;
  const float* scale;        // nullable: 1
  void* low;                 // planes [2][slots][rank_pad]
  int64_t slots;
  bool vector_rows, vector_weight, vector_out;
  const void* base;          // expand, nullable: 0
  int64_t base_stride;
  void* out;
  int64_t out_stride;        // expand: row; outer: column
  int64_t out_rank_stride;   // outer
  int chunks_per_split;
  int tile_count, tiles_per_block;  // expand
  int piece_bits;            // expand: 2^piece_bits >= rank_pad / 8 threads copy a row
};

__device__ __forceinline__ int64_t token_of(const AdapterParams& p, int64_t slot) {
  const int32_t token = p.rows[slot];
  return token >= 0 && token < p.tokens ? token : -1;
}

// ------------------------------------------------------------------ shrink ----

// ROWS 64: four warps of 16 rows; ROWS 16: four warps share the rows and take
// a quarter of each chunk of the width. RANK: columns of `low` per block.
template <int ROWS, int RANK, bool TRANS>
struct ShrinkShape {
  static constexpr int kChunk = ROWS == 64 ? 64 : 256;
  static constexpr int kStages = 4;
  static constexpr int kRowPitch = kChunk + 8;
  static constexpr int kWeightRows = TRANS ? kChunk : RANK;
  static constexpr int kWeightCols = TRANS ? RANK : kChunk;
  static constexpr int kWeightPitch = kWeightCols + 8;
  static constexpr int kStageElements = ROWS * kRowPitch + kWeightRows * kWeightPitch;
  static constexpr int kPartRows = ROWS == 64 ? 64 : 4 * 16;
  static constexpr int kPartBytes = kPartRows * RANK * 4;
  static constexpr int kBytes = kStages * kStageElements * 2 > kPartBytes ? kStages * kStageElements * 2 : kPartBytes;
};

template <typename T, int ROWS, int RANK, bool TRANS>
__global__ void __launch_bounds__(kAdapterThreads) adapter_shrink(AdapterParams p) {
  using S = ShrinkShape<ROWS, RANK, TRANS>;
  extern __shared__ __align__(16) uint8_t shared[];
  T* stages = reinterpret_cast<T*>(shared);
  griddep_launch_dependents();
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = cluster_ctarank();
  const Tile tile = p.tiles[blockIdx.x / splits];
  const int rank0 = blockIdx.y * RANK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool valid = tile.adapter >= 0 && tile.adapter < p.adapters;
  const int count = valid ? tile.count : 0;
  const T* x = static_cast<const T*>(p.rows_in);
  const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(valid ? tile.adapter : 0) * p.rank * p.width;

  const int chunks = static_cast<int>((p.width + S::kChunk - 1) / S::kChunk);
  const int first = min(static_cast<int>(split) * p.chunks_per_split, chunks);
  const int last = min(first + p.chunks_per_split, chunks);

  // Rows beyond the tile and ranks beyond the adapter stay zero throughout.
  for (int i = tid; i < S::kStages * S::kStageElements / 8; i += kAdapterThreads) {
    reinterpret_cast<uint4*>(shared)[i] = make_uint4(0, 0, 0, 0);
  }
  constexpr int kPieces = S::kChunk / 8;            // 16-byte pieces of a row
  constexpr int kRowStep = kAdapterThreads / kPieces;
  constexpr int kPasses = ROWS / kRowStep;
  const int piece = tid % kPieces;
  const T* source[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int row = tid / kPieces + i * kRowStep;
    const int64_t token = row < count ? token_of(p, tile.start + row) : -1;
    source[i] = token >= 0 ? x + token * p.row_stride + piece * 8 : nullptr;
  }
  __syncthreads();

  auto load = [&](int chunk) {
    T* rows = stages + ((chunk - first) % S::kStages) * S::kStageElements;
    T* w = rows + ROWS * S::kRowPitch;
    const int64_t k0 = static_cast<int64_t>(chunk) * S::kChunk;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      if (source[i] == nullptr) continue;
      const int row = tid / kPieces + i * kRowStep;
      copy8(rows + row * S::kRowPitch + piece * 8, source[i] + k0, p.width - (k0 + piece * 8), p.vector_rows);
    }
    if constexpr (!TRANS) {  // weight [rank, width]
      for (int i = tid; i < RANK * kPieces; i += kAdapterThreads) {
        const int r = i / kPieces, c = i % kPieces * 8;
        if (rank0 + r < p.rank) {
          copy8(w + r * S::kWeightPitch + c, weight + (rank0 + r) * p.width + k0 + c, p.width - (k0 + c),
                p.vector_weight);
        }
      }
    } else {  // weight [width, rank]
      for (int i = tid; i < S::kChunk * (RANK / 8); i += kAdapterThreads) {
        const int k = i / (RANK / 8), c = i % (RANK / 8) * 8;
        copy8(w + k * S::kWeightPitch + c, weight + (k0 + k) * p.rank + rank0 + c,
              k0 + k < p.width ? p.rank - (rank0 + c) : 0, p.vector_weight);
      }
    }
  };

  float acc[RANK / 8][4];
#pragma unroll
  for (int i = 0; i < RANK / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (first + i < last) load(first + i);
    cp_async_commit();
  }
  const int row0 = ROWS == 64 ? warp * 16 : 0;
  for (int chunk = first; chunk < last; ++chunk) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();
    if (chunk + S::kStages - 1 < last) load(chunk + S::kStages - 1);
    cp_async_commit();
    const T* rows = stages + ((chunk - first) % S::kStages) * S::kStageElements;
    const T* w = rows + ROWS * S::kRowPitch;
    constexpr int kSteps = ROWS == 64 ? S::kChunk / 16 : S::kChunk / 64;
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      const int k = (ROWS == 64 ? 0 : warp * (S::kChunk / 4)) + step * 16;
      uint32_t a[4];
      ldmatrix_x4(a, rows + (row0 + (lane & 15)) * S::kRowPitch + k + (lane >> 4) * 8);
#pragma unroll
      for (int n = 0; n < RANK / 16; ++n) {
        uint32_t b[4];
        if constexpr (!TRANS) {
          ldmatrix_x4(b, w + (n * 16 + (lane >> 4) * 8 + (lane & 7)) * S::kWeightPitch + k + ((lane >> 3) & 1) * 8);
        } else {
          ldmatrix_x4_trans(b, w + (k + ((lane >> 3) & 1) * 8 + (lane & 7)) * S::kWeightPitch + n * 16 + (lane >> 4) * 8);
        }
        mma_16816<T>(acc[2 * n], a, b);
        mma_16816<T>(acc[2 * n + 1], a, b + 2);
      }
    }
  }

  // Sum over the warps that shared the rows and over the cluster, in order.
  cp_async_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(shared);
  const int part_row = warp * 16 + (lane >> 2);
#pragma unroll
  for (int i = 0; i < RANK / 8; ++i) {
    const int c = i * 8 + (lane & 3) * 2;
    part[part_row * RANK + c] = acc[i][0];
    part[part_row * RANK + c + 1] = acc[i][1];
    part[(part_row + 8) * RANK + c] = acc[i][2];
    part[(part_row + 8) * RANK + c + 1] = acc[i][3];
  }
  cluster_sync();
  const float scale = p.scale != nullptr && valid ? p.scale[tile.adapter] : 1.f;
  T* high = static_cast<T*>(p.low);
  T* low = high + p.slots * p.rank_pad;
  for (int e = static_cast<int>(split) * kAdapterThreads + tid; e < count * RANK;
       e += static_cast<int>(splits) * kAdapterThreads) {
    const int row = e / RANK, c = e % RANK;
    if (rank0 + c >= p.rank_pad) continue;
    float v = 0.f;
    for (uint32_t s = 0; s < splits; ++s) {
      const uint32_t from = mapa_shared(part, s) + e * 4;
      v += load_cluster_f32(from);
      if constexpr (ROWS == 16) {
#pragma unroll
        for (int other = 1; other < 4; ++other) v += load_cluster_f32(from + other * 16 * RANK * 4);
      }
    }
    v *= scale;
    const T hi = from_float<T>(v);
    const float rest = v - to_float(hi);
    const int64_t at = (tile.start + row) * static_cast<int64_t>(p.rank_pad) + rank0 + c;
    high[at] = hi;
    low[at] = from_float<T>(isfinite(rest) ? rest : 0.f);  // an infinite sum stays one
  }
  cluster_sync();  // the others may still be reading this block's sums
}

// ------------------------------------------------------------------ expand ----

// ROWS 64: a warp takes 16 rows of 256 columns; ROWS 16: all 16 rows of 32 of
// 128 columns. A thread's accumulators over four 8-column tiles are made 8
// neighbouring columns by assigning column 8 q + 2 j + b of 32 to element
// 2 q + b of tile j: base and out then move in 16-byte words straight between
// registers and memory.
template <int ROWS>
struct ExpandShape {
  static constexpr int kColumns = ROWS == 64 ? 256 : 128;
  static constexpr int kGroups = ROWS == 64 ? 8 : 1;  // 32-column groups per warp
};

// Shared layout of the weight: !TRANS (weight [width, rank]): column-major
// rows of rank_pad + 8 elements, each run of 8 columns skewed by 32 bytes so
// that the 8 rows of a fragment (columns 0, 1, 8, 9, 16, ... of a group) hit
// different banks. TRANS (weight [rank, width]): rank_pad rows of permuted
// columns.
__host__ __device__ constexpr int expand_group_bytes(int rank_pad) { return 32 * (rank_pad + 8) * 2 + 96; }
__host__ __device__ constexpr int expand_weight_bytes(int columns, int rank_pad, bool trans) {
  return trans ? rank_pad * (columns + 8) * 2 : columns / 32 * expand_group_bytes(rank_pad);
}
// Two tiles' low rows, or one where two do not fit.
__host__ __device__ constexpr int low_buffers(int rank_pad) { return rank_pad <= 128 ? 2 : 1; }
__host__ __device__ constexpr int expand_bytes(int rows, int columns, int rank_pad, bool trans) {
  return expand_weight_bytes(columns, rank_pad, trans) + low_buffers(rank_pad) * 2 * rows * (rank_pad + 8) * 2;
}

// A block keeps 256 columns of one adapter's weight in shared memory and walks
// a run of tiles: the next tile's low rows are copied and its part of base is
// loaded into registers as soon as the current one's has been used, so loads
// never stop. FAST: widths, strides and addresses allow 16-byte accesses to
// base and out throughout.
template <typename T, int ROWS, bool TRANS, bool FAST>
__global__ void __launch_bounds__(kAdapterThreads, 4) adapter_expand(AdapterParams p) {
  using S = ExpandShape<ROWS>;
  extern __shared__ __align__(16) uint8_t shared[];
  const int width = static_cast<int>(p.width);
  const int column_blocks = (width + S::kColumns - 1) / S::kColumns;
  const int run = static_cast<int>(blockIdx.x) / column_blocks;
  const int column0 = (static_cast<int>(blockIdx.x) - run * column_blocks) * S::kColumns;
  const int first = run * p.tiles_per_block, last = min(first + p.tiles_per_block, p.tile_count);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pitch = p.rank_pad + 8, pieces = p.rank_pad / 8;
  uint8_t* weight_shared = shared;
  T* low_shared = reinterpret_cast<T*>(shared + expand_weight_bytes(S::kColumns, p.rank_pad, TRANS));
  const int low_elements = 2 * ROWS * pitch;  // of one tile
  const bool two_buffers = low_buffers(p.rank_pad) == 2;

  auto load_weight = [&](int adapter) {
    const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(adapter) * p.rank * p.width;
    if constexpr (!TRANS) {
      const int piece = (tid & ((1 << p.piece_bits) - 1)), r = piece * 8;
      if (piece < pieces) {
        for (int c = tid >> p.piece_bits; c < S::kColumns; c += kAdapterThreads >> p.piece_bits) {
          T* to = reinterpret_cast<T*>(weight_shared + (c >> 5) * expand_group_bytes(p.rank_pad) +
                                       (c & 31) * pitch * 2 + ((c >> 3) & 3) * 32) + r;
          copy8(to, weight + static_cast<int64_t>(column0 + c) * p.rank + r, column0 + c < width ? p.rank - r : 0,
                p.vector_weight);
        }
      }
    } else {
      constexpr int kPieces = S::kColumns / 8;
      for (int i = tid; i < p.rank_pad * kPieces; i += kAdapterThreads) {
        const int r = i / kPieces, c = i % kPieces * 8;
        const T* from = weight + r * p.width + column0 + c;
        const int left = r < p.rank ? width - (column0 + c) : 0;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (left >= 8 && p.vector_weight) {
          w = *reinterpret_cast<const uint4*>(from);
        } else {
          T* e = reinterpret_cast<T*>(&w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j < left) e[j] = from[j];
          }
        }
        uint32_t* to = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(weight_shared) +
                                                   r * (S::kColumns + 8) + (c & ~31) + ((c >> 3) & 3) * 2);
        to[0] = w.x, to[4] = w.y, to[8] = w.z, to[12] = w.w;
      }
    }
  };
  auto load_low = [&](const Tile& tile, int buffer) {
    T* to_tile = low_shared + buffer * low_elements;
    const T* from = static_cast<const T*>(p.low) + static_cast<int64_t>(tile.start) * p.rank_pad;
    const int piece = tid & ((1 << p.piece_bits) - 1), r = piece * 8;
    if (piece >= pieces) return;
    for (int i = tid >> p.piece_bits; i < 2 * ROWS; i += kAdapterThreads >> p.piece_bits) {
      const int row = i % ROWS;
      T* to = to_tile + i * pitch + r;
      if (row < tile.count) {
        cp_async16(to, from + (i >= ROWS ? p.slots * p.rank_pad : 0) + row * p.rank_pad + r);
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
      }
    }
  };
  auto adapted = [&](const Tile& tile) { return tile.adapter >= 0 && tile.adapter < p.adapters; };

  // This thread's part of base and out: rows lane / 4 and lane / 4 + 8 of its
  // 16, 8 columns of each 32.
  const int row0 = (ROWS == 64 ? warp * 16 : 0) + (lane >> 2);
  const int column = column0 + (ROWS == 64 ? 0 : warp * 32) + (lane & 3) * 8;
  auto look = [&](const Tile& tile, int64_t* token) {
#pragma unroll
    for (int h = 0; h < 2; ++h) token[h] = row0 + 8 * h < tile.count ? token_of(p, tile.start + row0 + 8 * h) : -1;
  };
  const T* base = static_cast<const T*>(p.base);
  auto load_base = [&](int64_t token, int g) {
    Raw8<T> r;
    r.w[0] = make_uint4(0, 0, 0, 0);
    const int left = width - (column + g * 32);
    if (base == nullptr || token < 0 || left <= 0) return r;
    const T* from = base + token * p.base_stride + column + g * 32;
    if constexpr (FAST) {
      r = load8(from);
    } else {
      T* e = reinterpret_cast<T*>(&r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < left) e[j] = from[j];
      }
    }
    return r;
  };

  Tile tile = p.tiles[first];
  int64_t token[2], next_token[2];
  look(tile, token);
  Raw8<T> part[S::kGroups][2];
#pragma unroll
  for (int g = 0; g < S::kGroups; ++g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) part[g][h] = load_base(token[h], g);
  }
  int adapter = -1;  // whose weight is in shared memory
  if (adapted(tile)) load_weight(adapter = tile.adapter);
  griddep_wait();  // `low` from here on
  if (adapted(tile)) load_low(tile, 0);
  cp_async_commit();
  Tile next = first + 1 < last ? p.tiles[first + 1] : Tile{0, 0, -1};
  for (int t = first; t < last; ++t) {
    const int buffer = two_buffers ? (t - first) & 1 : 0;
    const bool more = t + 1 < last;
    const Tile after = t + 2 < last ? p.tiles[t + 2] : Tile{0, 0, -1};
    if (more) look(next, next_token);
    if (two_buffers && more && adapted(next)) load_low(next, buffer ^ 1);
    cp_async_commit();
    if (adapted(tile) && tile.adapter != adapter) {
      __syncthreads();  // the last tile's products are done with the old weight
      load_weight(adapter = tile.adapter);
      cp_async_commit();
      cp_async_wait<0>();
    } else {
      cp_async_wait<1>();
    }
    __syncthreads();
    const T* low = low_shared + buffer * low_elements + ((ROWS == 64 ? warp * 16 : 0) + (lane & 15)) * pitch + (lane >> 4) * 8;
#pragma unroll
    for (int g = 0; g < S::kGroups; ++g) {
      float acc[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
      if (adapted(tile)) {
        const int group = ROWS == 64 ? g : warp;
        for (int k = 0; k < p.rank_pad; k += 16) {
          uint32_t hi[4], lo[4];
          ldmatrix_x4(hi, low + k);
          ldmatrix_x4(lo, low + ROWS * pitch + k);
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            uint32_t b[4];
            if constexpr (!TRANS) {
              const int i = lane & 7, j = 2 * pair + (lane >> 4);
              const int c = (i >> 1) * 8 + j * 2 + (i & 1);
              ldmatrix_x4(b, reinterpret_cast<const T*>(weight_shared + group * expand_group_bytes(p.rank_pad) +
                                                        c * pitch * 2 + (c >> 3) * 32) + k + ((lane >> 3) & 1) * 8);
            } else {
              ldmatrix_x4_trans(b, reinterpret_cast<const T*>(weight_shared) +
                                       (k + ((lane >> 3) & 1) * 8 + (lane & 7)) * (S::kColumns + 8) + group * 32 +
                                       pair * 16 + (lane >> 4) * 8);
            }
            mma_16816<T>(acc[2 * pair], hi, b);
            mma_16816<T>(acc[2 * pair + 1], hi, b + 2);
            mma_16816<T>(acc[2 * pair], lo, b);
            mma_16816<T>(acc[2 * pair + 1], lo, b + 2);
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        unpack8(part[g][h], v);
        if (more) part[g][h] = load_base(next_token[h], g);
        const int left = width - (column + g * 32);
        if (token[h] < 0 || left <= 0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] += acc[j][2 * h];
          v[2 * j + 1] += acc[j][2 * h + 1];
        }
        T* to = static_cast<T*>(p.out) + token[h] * p.out_stride + column + g * 32;
        if constexpr (FAST) {
          store8(to, pack8<T>(v));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j < left) to[j] = from_float<T>(v[j]);
          }
        }
      }
    }
    if (!two_buffers) {
      __syncthreads();
      if (more && adapted(next)) load_low(next, 0);
      cp_async_commit();
      cp_async_wait<0>();
    }
    tile = next;
    next = after;
#pragma unroll
    for (int h = 0; h < 2; ++h) token[h] = next_token[h];
  }
}

// ------------------------------------------------------------------- outer ----

// dW[column, r] = sum over the adapter's slots of row[column] * low[r]. A
// block takes 128 columns and RANK ranks; the blocks of a cluster share the
// adapter's tokens.
template <int RANK>
struct OuterShape {
  static constexpr int kColumns = 128;
  static constexpr int kTokens = 32;
  static constexpr int kStages = 4;
  static constexpr int kLook = 2 * kStages;  // token lists in flight
  static constexpr int kRowPitch = kColumns + 8;
  static constexpr int kLowPitch = RANK + 8;
  static constexpr int kStageElements = kTokens * (kRowPitch + 2 * kLowPitch);
  static constexpr int kPartPitch = RANK + 1;
  static constexpr int kPartBytes = kColumns * kPartPitch * 4;
  static constexpr int kBytes = kStages * kStageElements * 2 > kPartBytes ? kStages * kStageElements * 2 : kPartBytes;
};

template <typename T, int RANK>
__global__ void __launch_bounds__(kAdapterThreads) adapter_outer(AdapterParams p) {
  using S = OuterShape<RANK>;
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ int32_t tokens[S::kLook][S::kTokens];
  T* stages = reinterpret_cast<T*>(shared);
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = cluster_ctarank();
  const int64_t column0 = static_cast<int64_t>(blockIdx.x / splits) * S::kColumns;
  const int adapter = blockIdx.y;
  const int rank0 = blockIdx.z * RANK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t begin = p.group_offsets[adapter], end = p.group_offsets[adapter + 1];
  const int tiles = (end - begin + S::kTokens - 1) / S::kTokens;
  const int per_split = (tiles + static_cast<int>(splits) - 1) / static_cast<int>(splits);
  const int first = min(static_cast<int>(split) * per_split, tiles);
  const int last = min(first + per_split, tiles);

  constexpr int kPieces = S::kColumns / 8;
  constexpr int kRowStep = kAdapterThreads / kPieces;
  constexpr int kPasses = S::kTokens / kRowStep;
  const int piece = tid % kPieces;
  const T* x = static_cast<const T*>(p.rows_in) + column0 + piece * 8;
  const int64_t columns_left = p.width - (column0 + piece * 8);
  const T* low = static_cast<const T*>(p.low);

  // The tokens of a tile are copied kStages - 1 tiles before its rows.
  auto look = [&](int tile) {
    const int64_t slot = begin + static_cast<int64_t>(tile) * S::kTokens + tid;
    if (tid >= S::kTokens || tile >= last) return;
    if (slot < end) cp_async4(&tokens[tile % S::kLook][tid], p.rows + slot);
    else tokens[tile % S::kLook][tid] = -1;
  };
  auto load = [&](int tile) {
    T* rows = stages + ((tile - first) % S::kStages) * S::kStageElements;
    T* lows = rows + S::kTokens * S::kRowPitch;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int row = tid / kPieces + i * kRowStep;
      const int64_t token = tokens[tile % S::kLook][row];
      copy8(rows + row * S::kRowPitch + piece * 8, x + token * p.row_stride,
            token >= 0 && token < p.tokens ? columns_left : 0, p.vector_rows);
    }
    const int64_t slot0 = begin + static_cast<int64_t>(tile) * S::kTokens;
    for (int i = tid; i < 2 * S::kTokens * (RANK / 8); i += kAdapterThreads) {
      const int plane = i / (S::kTokens * (RANK / 8));
      const int row = i / (RANK / 8) % S::kTokens, r = i % (RANK / 8) * 8;
      const bool in = slot0 + row < end && rank0 + r < p.rank_pad;
      copy8(lows + (plane * S::kTokens + row) * S::kLowPitch + r,
            low + (plane * p.slots + slot0 + row) * p.rank_pad + rank0 + r, in ? 8 : 0, true);
    }
  };

  float acc[2][RANK / 8][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int i = 0; i < RANK / 8; ++i) acc[m][i][0] = acc[m][i][1] = acc[m][i][2] = acc[m][i][3] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < 2 * (S::kStages - 1); ++i) look(first + i);
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S::kStages - 1; ++i) {
    if (first + i < last) load(first + i);
    cp_async_commit();
  }
  for (int tile = first; tile < last; ++tile) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();
    if (tile + S::kStages - 1 < last) load(tile + S::kStages - 1);
    look(tile + 2 * (S::kStages - 1));
    cp_async_commit();
    const T* rows = stages + ((tile - first) % S::kStages) * S::kStageElements;
    const T* lows = rows + S::kTokens * S::kRowPitch;
#pragma unroll
    for (int k = 0; k < S::kTokens; k += 16) {
      uint32_t a[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        ldmatrix_x4_trans(a[m], rows + (k + (lane >> 4) * 8 + (lane & 7)) * S::kRowPitch + warp * 32 + m * 16 +
                                    ((lane >> 3) & 1) * 8);
      }
#pragma unroll
      for (int n = 0; n < RANK / 16; ++n) {
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, lows + (plane * S::kTokens + k + ((lane >> 3) & 1) * 8 + (lane & 7)) * S::kLowPitch +
                                   n * 16 + (lane >> 4) * 8);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            mma_16816<T>(acc[m][2 * n], a[m], b);
            mma_16816<T>(acc[m][2 * n + 1], a[m], b + 2);
          }
        }
      }
    }
  }

  cp_async_wait<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(shared);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int c = warp * 32 + m * 16 + (lane >> 2);
#pragma unroll
    for (int i = 0; i < RANK / 8; ++i) {
      const int r = i * 8 + (lane & 3) * 2;
      part[c * S::kPartPitch + r] = acc[m][i][0];
      part[c * S::kPartPitch + r + 1] = acc[m][i][1];
      part[(c + 8) * S::kPartPitch + r] = acc[m][i][2];
      part[(c + 8) * S::kPartPitch + r + 1] = acc[m][i][3];
    }
  }
  cluster_sync();
  T* out = static_cast<T*>(p.out) + static_cast<int64_t>(adapter) * p.rank * p.width;
  const bool columns_fast = p.out_stride == 1;  // neighbouring threads write neighbouring elements
  for (int e = static_cast<int>(split) * kAdapterThreads + tid; e < S::kColumns * RANK;
       e += static_cast<int>(splits) * kAdapterThreads) {
    const int c = columns_fast ? e % S::kColumns : e / RANK;
    const int r = columns_fast ? e / S::kColumns : e % RANK;
    if (column0 + c >= p.width || rank0 + r >= p.rank) continue;
    float v = 0.f;
    for (uint32_t s = 0; s < splits; ++s) v += load_cluster_f32(mapa_shared(part, s) + (c * S::kPartPitch + r) * 4);
    out[(column0 + c) * p.out_stride + (rank0 + r) * p.out_rank_stride] = from_float<T>(v);
  }
  cluster_sync();
}

// -------------------------------------------------------------------- host ----

template <typename Kernel>
int launch_clustered(Kernel kernel, const AdapterParams& p, dim3 grid, int cluster, int shared, bool dependent,
                     cudaStream_t stream) {
  if (shared > 48 * 1024) {
    SDC_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
  }
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(kAdapterThreads);
  config.dynamicSmemBytes = static_cast<size_t>(shared);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  int attrs = 0;
  if (cluster > 0) {
    attribute[attrs].id = cudaLaunchAttributeClusterDimension;
    attribute[attrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attribute[attrs].val.clusterDim.y = 1;
    attribute[attrs].val.clusterDim.z = 1;
    ++attrs;
  }
  if (dependent) {
    attribute[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[attrs].val.programmaticStreamSerializationAllowed = 1;
    ++attrs;
  }
  config.attrs = attribute;
  config.numAttrs = attrs;
  SDC_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, p));
  return SDC_OK;
}

int check_adapters(int dtype, int64_t tokens, int64_t width, int rank, int adapters) {
  SDC_REQUIRE(dtype == kBF16 || dtype == kF16, "low-rank adapters compute BF16 (1) or FP16 (2)");
  SDC_REQUIRE(tokens >= 0 && tokens < INT_MAX - 128, "low-rank adapters take fewer than 2^31 - 128 tokens");
  SDC_REQUIRE(width > 0 && width < INT_MAX - 512, "low-rank adapter widths must be positive and fit padded int32 extents");
  SDC_REQUIRE(rank >= 1 && rank <= kMaxRank, "low-rank adapters take ranks of 1 to 256");
  SDC_REQUIRE(adapters >= 1 && adapters <= 65535, "low-rank adapters take 1 to 65535 adapters");
  return SDC_OK;
}

int pad_rank(int rank) { return (rank + 15) / 16 * 16; }
int rank_tile(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

bool vector_rows(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

// Blocks that share a tile's sum: enough for two blocks on every SM, as long
// as each keeps two chunks.
int split_count(int64_t blocks, int64_t chunks) {
  int split = 1;
  while (split < kMaxSplit && blocks * split < 2 * sm_count() && chunks >= 4 * split) split *= 2;
  return split;
}

template <typename T, int ROWS, int RANK, bool TRANS>
int launch_shrink(AdapterParams p, int64_t tiles, cudaStream_t stream) {
  using S = ShrinkShape<ROWS, RANK, TRANS>;
  const int64_t chunks = ceil_div(p.width, S::kChunk);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int split = split_count(tiles * rank_blocks, chunks);
  p.chunks_per_split = static_cast<int>(ceil_div(chunks, split));
  return launch_clustered(adapter_shrink<T, ROWS, RANK, TRANS>, p,
                          dim3(static_cast<unsigned>(tiles * split), rank_blocks), split, S::kBytes, false, stream);
}

template <typename T, int ROWS, bool TRANS>
int shrink_by_rank(const AdapterParams& p, int64_t tiles, cudaStream_t stream) {
  switch (rank_tile(p.rank)) {
    case 16: return launch_shrink<T, ROWS, 16, TRANS>(p, tiles, stream);
    case 32: return launch_shrink<T, ROWS, 32, TRANS>(p, tiles, stream);
    default: return launch_shrink<T, ROWS, 64, TRANS>(p, tiles, stream);
  }
}

template <typename T>
int shrink_typed(const AdapterParams& p, int tile_rows, bool trans, int64_t tiles, cudaStream_t stream) {
  if (tile_rows == 64) return trans ? shrink_by_rank<T, 64, true>(p, tiles, stream) : shrink_by_rank<T, 64, false>(p, tiles, stream);
  return trans ? shrink_by_rank<T, 16, true>(p, tiles, stream) : shrink_by_rank<T, 16, false>(p, tiles, stream);
}

template <typename T, int ROWS, bool TRANS>
int launch_expand(AdapterParams p, int64_t tiles, bool dependent, cudaStream_t stream) {
  constexpr int kColumns = ExpandShape<ROWS>::kColumns;
  const int64_t column_blocks = ceil_div(p.width, kColumns);
  // Runs of tiles that fill the SMs' four blocks each once; tiles of few rows
  // are bound by the weight, of which each then wants its own.
  p.tile_count = static_cast<int>(tiles);
  const int64_t runs = std::max<int64_t>(1, 4 * sm_count() / column_blocks);
  p.tiles_per_block = ROWS == 64 ? static_cast<int>(ceil_div(tiles, runs)) : 1;
  const int64_t blocks = column_blocks * ceil_div(tiles, p.tiles_per_block);
  SDC_REQUIRE(blocks <= INT_MAX, "low-rank adapters have too many tiles for one launch");
  while ((8 << p.piece_bits) < p.rank_pad) ++p.piece_bits;
  const int shared = expand_bytes(ROWS, kColumns, p.rank_pad, TRANS);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (p.vector_rows && p.vector_out && p.width % 8 == 0) {
    return launch_clustered(adapter_expand<T, ROWS, TRANS, true>, p, grid, 0, shared, dependent, stream);
  }
  return launch_clustered(adapter_expand<T, ROWS, TRANS, false>, p, grid, 0, shared, dependent, stream);
}

template <typename T>
int expand_typed(const AdapterParams& p, int tile_rows, bool trans, int64_t tiles, bool dependent, cudaStream_t stream) {
  if (tile_rows == 64) {
    return trans ? launch_expand<T, 64, true>(p, tiles, dependent, stream)
                 : launch_expand<T, 64, false>(p, tiles, dependent, stream);
  }
  return trans ? launch_expand<T, 16, true>(p, tiles, dependent, stream)
               : launch_expand<T, 16, false>(p, tiles, dependent, stream);
}

template <typename T, int RANK>
int launch_outer(const AdapterParams& p, cudaStream_t stream) {
  using S = OuterShape<RANK>;
  const int64_t columns = ceil_div(p.width, S::kColumns);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int64_t tiles = ceil_div(ceil_div(p.slots, p.adapters), S::kTokens);
  const int split = split_count(columns * p.adapters * rank_blocks, tiles);
  return launch_clustered(adapter_outer<T, RANK>, p,
                          dim3(static_cast<unsigned>(columns * split), static_cast<unsigned>(p.adapters), rank_blocks),
                          split, S::kBytes, false, stream);
}

template <typename T>
int outer_typed(const AdapterParams& p, cudaStream_t stream) {
  switch (rank_tile(p.rank)) {
    case 16: return launch_outer<T, 16>(p, stream);
    case 32: return launch_outer<T, 32>(p, stream);
    default: return launch_outer<T, 64>(p, stream);
  }
}

}  // namespace
}  // namespace sdc

extern "C" {

size_t sdc_adapter_low_bytes(int64_t slots, int rank) {
  if (slots <= 0 || rank <= 0 || rank > sdc::kMaxRank) return 0;
  return static_cast<size_t>(slots) * sdc::pad_rank(rank) * 2 * sizeof(uint16_t);
}

int sdc_adapter_shrink(int dtype, const void* x, int64_t x_stride, int64_t tokens, const int32_t* rows,
                       const int32_t* tiles, int64_t tile_count, int tile_rows, const void* weight, int adapters,
                       int rank, int64_t width, int weight_rank_minor, const float* scale, void* low, int64_t slots,
                       sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_adapters(dtype, tokens, width, rank, adapters);
  if (rc != SDC_OK) return rc;
  SDC_REQUIRE(tile_rows == 16 || tile_rows == 64, "low-rank adapter tiles have 16 or 64 rows");
  SDC_REQUIRE(tile_count >= 0 && tile_count <= INT_MAX / kMaxSplit, "low-rank adapters have too many tiles for one launch");
  if (tile_count == 0) return SDC_OK;
  SDC_REQUIRE(x != nullptr && rows != nullptr && tiles != nullptr && weight != nullptr && low != nullptr && aligned16(low),
              "low-rank adapter pointers must not be null and the low-rank rows must be 16-byte aligned");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  AdapterParams p{};
  p.rows_in = x;
  p.row_stride = x_stride;
  p.tokens = tokens;
  p.rows = rows;
  p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.adapters = adapters;
  p.weight = weight;
  p.rank = rank;
  p.rank_pad = pad_rank(rank);
  p.width = width;
  p.scale = scale;
  p.low = low;
  p.slots = slots;
  p.vector_rows = vector_rows(x, x_stride);
  p.vector_weight = vector_rows(weight, weight_rank_minor ? rank : width);
  return dtype == kBF16 ? shrink_typed<__nv_bfloat16>(p, tile_rows, weight_rank_minor != 0, tile_count, stream)
                        : shrink_typed<__half>(p, tile_rows, weight_rank_minor != 0, tile_count, stream);
}

int sdc_adapter_expand(int dtype, const void* base, int64_t base_stride, int64_t tokens, const int32_t* rows,
                       const int32_t* tiles, int64_t tile_count, int tile_rows, const void* weight, int adapters,
                       int rank, int64_t width, int weight_rank_minor, const void* low, int64_t slots,
                       int after_shrink, void* out, int64_t out_stride, sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_adapters(dtype, tokens, width, rank, adapters);
  if (rc != SDC_OK) return rc;
  SDC_REQUIRE(tile_rows == 16 || tile_rows == 64, "low-rank adapter tiles have 16 or 64 rows");
  SDC_REQUIRE(tile_count >= 0 && tile_count <= INT_MAX, "low-rank adapters have too many tiles for one launch");
  if (tile_count == 0) return SDC_OK;
  SDC_REQUIRE(rows != nullptr && tiles != nullptr && weight != nullptr && (low != nullptr || slots == 0) && out != nullptr &&
                  aligned16(low),
              "low-rank adapter pointers must not be null and the low-rank rows must be 16-byte aligned");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  AdapterParams p{};
  p.tokens = tokens;
  p.rows = rows;
  p.tiles = reinterpret_cast<const Tile*>(tiles);
  p.adapters = adapters;
  p.weight = weight;
  p.rank = rank;
  p.rank_pad = pad_rank(rank);
  p.width = width;
  p.low = const_cast<void*>(low);
  p.slots = slots;
  p.base = base;
  p.base_stride = base_stride;
  p.out = out;
  p.out_stride = out_stride;
  p.vector_rows = vector_rows(base, base_stride);
  p.vector_out = vector_rows(out, out_stride);
  p.vector_weight = vector_rows(weight, weight_rank_minor ? rank : width);
  // In this kernel "transposed" is the weight whose columns are the width.
  return dtype == kBF16
             ? expand_typed<__nv_bfloat16>(p, tile_rows, weight_rank_minor == 0, tile_count, after_shrink != 0, stream)
             : expand_typed<__half>(p, tile_rows, weight_rank_minor == 0, tile_count, after_shrink != 0, stream);
}

int sdc_adapter_outer(int dtype, const void* x, int64_t x_stride, int64_t tokens, const int32_t* rows,
                      const int32_t* group_offsets, int adapters, const void* low, int64_t slots, int rank,
                      int64_t width, int out_rank_minor, void* out, sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_adapters(dtype, tokens, width, rank, adapters);
  if (rc != SDC_OK) return rc;
  SDC_REQUIRE(group_offsets != nullptr && out != nullptr &&
                  (slots == 0 || (x != nullptr && rows != nullptr && low != nullptr && aligned16(low))),
              "low-rank adapter pointers must not be null and the low-rank rows must be 16-byte aligned");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  AdapterParams p{};
  p.rows_in = x;
  p.row_stride = x_stride;
  p.tokens = tokens;
  p.rows = rows;
  p.group_offsets = group_offsets;
  p.adapters = adapters;
  p.rank = rank;
  p.rank_pad = pad_rank(rank);
  p.width = width;
  p.low = const_cast<void*>(low);
  p.slots = slots;
  p.out = out;
  p.out_stride = out_rank_minor ? rank : 1;
  p.out_rank_stride = out_rank_minor ? 1 : width;
  p.vector_rows = vector_rows(x, x_stride);
  return dtype == kBF16 ? outer_typed<__nv_bfloat16>(p, stream) : outer_typed<__half>(p, stream);
}

}  // extern "C"
