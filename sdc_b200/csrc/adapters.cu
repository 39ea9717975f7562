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
// are gathered into tiles of 128 rows (16 when adapters have few tokens, as in
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

constexpr int kWide = 128, kNarrow = 16;  // rows of a tile
constexpr int kMaxWideRank = 128;         // beyond, a wide tile's low rows and weight do not fit together
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

// ROWS kWide: eight warps of 16 rows; ROWS kNarrow: four warps share the rows and take
// a quarter of each chunk of the width. RANK: columns of `low` per block.
template <int ROWS, int RANK, bool TRANS>
struct ShrinkShape {
  static constexpr int kThreads = ROWS == kWide ? 256 : 128;
  static constexpr int kChunk = ROWS == kWide ? 64 : 256;
  static constexpr int kStages = 4;
  static constexpr int kRowBytes = (kChunk + 8) * 2;  // 8 elements of padding: fragment rows on different banks
  static constexpr int kWeightRows = TRANS ? kChunk : RANK;
  static constexpr int kWeightBytes = ((TRANS ? RANK : kChunk) + 8) * 2;
  static constexpr int kStageBytes = ROWS * kRowBytes + kWeightRows * kWeightBytes;
  static constexpr int kPartRows = ROWS == kWide ? ROWS : 4 * ROWS;
  static constexpr int kPartBytes = kPartRows * RANK * 4;
  static constexpr int kBytes = kStages * kStageBytes > kPartBytes ? kStages * kStageBytes : kPartBytes;
};

template <typename T, int ROWS, int RANK, bool TRANS, bool FAST>
__global__ void __launch_bounds__(ShrinkShape<ROWS, RANK, TRANS>::kThreads) adapter_shrink(AdapterParams p) {
  using S = ShrinkShape<ROWS, RANK, TRANS>;
  extern __shared__ __align__(16) uint8_t shared[];
  const uint32_t stages = smem_u32(shared);
  griddep_launch_dependents();
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = cluster_ctarank();
  const Tile tile = p.tiles[blockIdx.x / splits];
  const int rank0 = blockIdx.y * RANK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool valid = tile.adapter >= 0 && tile.adapter < p.adapters;
  const int count = valid ? tile.count : 0;
  const int width = static_cast<int>(p.width);
  const int chunks = (width + S::kChunk - 1) / S::kChunk;
  const int first = min(static_cast<int>(split) * p.chunks_per_split, chunks);
  const int last = min(first + p.chunks_per_split, chunks);

  // What this thread copies of a chunk: pieces of 8 elements of the rows, and
  // of the weight [rank, width], or [width, rank] when TRANS.
  constexpr int kPieces = S::kChunk / 8;
  constexpr int kRowStep = S::kThreads / kPieces, kRowCopies = ROWS / kRowStep;
  constexpr int kWeightPieces = TRANS ? RANK / 8 : kPieces;
  constexpr int kWeightStep = S::kThreads / kWeightPieces;
  constexpr int kWeightCopies = (S::kWeightRows + kWeightStep - 1) / kWeightStep;
  const int piece = tid % kPieces, row_of = tid / kPieces;
  const int weight_piece = tid % kWeightPieces, weight_row = tid / kWeightPieces;
  const T* source[kRowCopies];
  uint32_t present = 0;
#pragma unroll
  for (int i = 0; i < kRowCopies; ++i) {
    const int row = row_of + i * kRowStep;
    const int64_t token = row < count ? token_of(p, tile.start + row) : -1;
    if (token >= 0) present |= 1u << i;
    source[i] = static_cast<const T*>(p.rows_in) + (token >= 0 ? token * p.row_stride : 0) + piece * 8;
  }
  const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(valid ? tile.adapter : 0) * p.rank * p.width;
  weight += TRANS ? static_cast<int64_t>(weight_row) * p.rank + rank0 + weight_piece * 8
                  : static_cast<int64_t>(rank0 + weight_row) * width + weight_piece * 8;
  const uint32_t row_to = stages + row_of * S::kRowBytes + piece * 16;
  const uint32_t weight_to = stages + ROWS * S::kRowBytes + weight_row * S::kWeightBytes + weight_piece * 16;

  auto load = [&](int chunk) {
    const uint32_t stage = static_cast<uint32_t>((chunk - first) % S::kStages) * S::kStageBytes;
    const int k0 = chunk * S::kChunk, left = width - k0 - piece * 8;
#pragma unroll
    for (int i = 0; i < kRowCopies; ++i) {
      copy8<T, FAST>(row_to + stage + i * kRowStep * S::kRowBytes, left > 0 ? source[i] + k0 : source[i],
                     (present >> i & 1) ? left : 0);
    }
#pragma unroll
    for (int i = 0; i < kWeightCopies; ++i) {
      const int at = weight_row + i * kWeightStep;
      if (S::kWeightRows % kWeightStep != 0 && at >= S::kWeightRows) continue;
      const int in = TRANS ? (k0 + at < width ? p.rank - (rank0 + weight_piece * 8) : 0) : (rank0 + at < p.rank ? left : 0);
      const T* from = weight + (TRANS ? static_cast<int64_t>(k0 + i * kWeightStep) * p.rank
                                      : static_cast<int64_t>(i * kWeightStep) * width + k0);
      copy8<T, FAST>(weight_to + stage + i * kWeightStep * S::kWeightBytes, in > 0 ? from : static_cast<const T*>(p.weight), in);
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
  const int k_of = ROWS == kWide ? 0 : warp * (S::kChunk / 4);
  const uint32_t a_from = stages + ((ROWS == kWide ? warp * 16 : 0) + (lane & 15)) * S::kRowBytes + (k_of + (lane >> 4) * 8) * 2;
  const uint32_t b_from =
      stages + ROWS * S::kRowBytes +
      (TRANS ? (k_of + ((lane >> 3) & 1) * 8 + (lane & 7)) * S::kWeightBytes + (lane >> 4) * 16
             : ((lane >> 4) * 8 + (lane & 7)) * S::kWeightBytes + (k_of + ((lane >> 3) & 1) * 8) * 2);
  for (int chunk = first; chunk < last; ++chunk) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();
    if (chunk + S::kStages - 1 < last) load(chunk + S::kStages - 1);
    cp_async_commit();
    const uint32_t stage = static_cast<uint32_t>((chunk - first) % S::kStages) * S::kStageBytes;
    constexpr int kSteps = ROWS == kWide ? S::kChunk / 16 : S::kChunk / 64;
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      uint32_t a[4];
      ldmatrix_x4(a, a_from + stage + step * 32);
#pragma unroll
      for (int n = 0; n < RANK / 16; ++n) {
        uint32_t b[4];
        if constexpr (!TRANS) ldmatrix_x4(b, b_from + stage + n * 16 * S::kWeightBytes + step * 32);
        else ldmatrix_x4_trans(b, b_from + stage + step * 16 * S::kWeightBytes + n * 32);
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
  for (int e = static_cast<int>(split) * S::kThreads + tid; e < count * RANK; e += static_cast<int>(splits) * S::kThreads) {
    const int row = e / RANK, c = e % RANK;
    if (rank0 + c >= p.rank_pad) continue;
    float v = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < splits; ++s) {
      const uint32_t from = mapa_shared(part, s) + e * 4;
      v += load_cluster_f32(from);
      if constexpr (ROWS == kNarrow) {
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

// ROWS kWide: a warp takes 16 rows of 256 columns; ROWS kNarrow: all 16 rows of 32 of
// 128 columns. A thread's accumulators over four 8-column tiles are made 8
// neighbouring columns by assigning column 8 q + 2 j + b of 32 to element
// 2 q + b of tile j: base and out then move in 16-byte words straight between
// registers and memory.
template <int ROWS>
struct ExpandShape {
  static constexpr int kThreads = ROWS == kWide ? 256 : 128;
  static constexpr int kBlocks = ROWS == kWide ? 2 : 4;  // at least, on an SM
  static constexpr int kColumns = ROWS == kWide ? 256 : 128;
  static constexpr int kGroups = ROWS == kWide ? 8 : 1;  // 32-column groups per warp
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
// never stop. FAST: widths, strides and addresses allow 16-byte accesses
// throughout. PAD: rank_pad, or 0 where it is read from the parameters.
template <typename T, int ROWS, bool TRANS, bool FAST, int PAD>
__global__ void __launch_bounds__(ExpandShape<ROWS>::kThreads, ExpandShape<ROWS>::kBlocks) adapter_expand(AdapterParams p) {
  using S = ExpandShape<ROWS>;
  extern __shared__ __align__(16) uint8_t shared[];
  const int pad = PAD > 0 ? PAD : p.rank_pad;
  const int width = static_cast<int>(p.width);
  const int column_blocks = (width + S::kColumns - 1) / S::kColumns;
  const int run = static_cast<int>(blockIdx.x) / column_blocks;
  const int column0 = (static_cast<int>(blockIdx.x) - run * column_blocks) * S::kColumns;
  const int first = run * p.tiles_per_block, last = min(first + p.tiles_per_block, p.tile_count);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pitch = (pad + 8) * 2;  // bytes of a low row, and of a weight row when !TRANS
  const int group_bytes = expand_group_bytes(pad);
  constexpr int kTransPitch = (S::kColumns + 8) * 2;
  const uint32_t weight_shared = smem_u32(shared);
  const uint32_t low_shared = weight_shared + expand_weight_bytes(S::kColumns, pad, TRANS);
  const uint32_t low_bytes = 2 * ROWS * pitch;  // of one tile
  const bool two_buffers = low_buffers(pad) == 2;
  const int piece_bits = PAD > 0 ? (PAD <= 16 ? 1 : PAD <= 32 ? 2 : 3) : p.piece_bits;
  const int piece = tid & ((1 << piece_bits) - 1), piece_row = tid >> piece_bits;
  const int piece_step = S::kThreads >> piece_bits;

  auto load_weight = [&](int adapter) {
    const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(adapter) * p.rank * p.width;
    if constexpr (!TRANS) {
      if (piece * 8 >= pad) return;
      for (int c = piece_row; c < S::kColumns; c += piece_step) {
        const uint32_t to = weight_shared + (c >> 5) * group_bytes + (c & 31) * pitch + ((c >> 3) & 3) * 32 + piece * 16;
        const int in = column0 + c < width ? p.rank - piece * 8 : 0;
        copy8<T, FAST>(to, in > 0 ? weight + static_cast<int64_t>(column0 + c) * p.rank + piece * 8 : weight, in);
      }
    } else {
      constexpr int kPieces = S::kColumns / 8;
      for (int i = tid; i < pad * kPieces; i += S::kThreads) {
        const int r = i / kPieces, c = i % kPieces * 8;
        const T* from = weight + r * p.width + column0 + c;
        const int left = r < p.rank ? width - (column0 + c) : 0;
        uint4 w = make_uint4(0, 0, 0, 0);
        if constexpr (FAST) {
          if (left > 0) w = *reinterpret_cast<const uint4*>(from);
        } else {
          T* e = reinterpret_cast<T*>(&w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (j < left) e[j] = from[j];
          }
        }
        const uint32_t to = weight_shared + r * kTransPitch + (c & ~31) * 2 + ((c >> 3) & 3) * 4;
        asm volatile("st.shared.b32 [%0], %1;\n\tst.shared.b32 [%0 + 16], %2;\n\t"
                     "st.shared.b32 [%0 + 32], %3;\n\tst.shared.b32 [%0 + 48], %4;" ::"r"(to), "r"(w.x), "r"(w.y),
                     "r"(w.z), "r"(w.w)
                     : "memory");
      }
    }
  };
  auto load_low = [&](const Tile& tile, int buffer) {
    if (piece * 8 >= pad) return;
    const T* from = static_cast<const T*>(p.low) + static_cast<int64_t>(tile.start) * pad + piece * 8;
    const uint32_t to = low_shared + buffer * low_bytes + piece * 16;
    for (int i = piece_row; i < 2 * ROWS; i += piece_step) {
      const int row = i % ROWS;
      const bool in = row < tile.count;
      cp_async16(to + i * pitch, in ? from + (i >= ROWS ? p.slots * pad : 0) + row * pad : from, in);
    }
  };
  auto adapted = [&](const Tile& tile) { return tile.adapter >= 0 && tile.adapter < p.adapters; };

  // This thread's part of base and out: rows lane / 4 and lane / 4 + 8 of its
  // 16, 8 columns of each 32.
  const int row0 = (ROWS == kWide ? warp * 16 : 0) + (lane >> 2);
  const int column = column0 + (ROWS == kWide ? 0 : warp * 32) + (lane & 3) * 8;
  const int columns_left = width - column;  // column + 32 g + j lies in the matrix when 32 g + j is less
  struct Rows {
    const T* base[2];
    T* out[2];
    int base_limit[2], out_limit[2];  // columns_left where there is a base and a row, else 0
  };
  auto look = [&](const Tile& tile) {
    Rows r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t token = row0 + 8 * h < tile.count ? token_of(p, tile.start + row0 + 8 * h) : -1;
      r.base[h] = static_cast<const T*>(p.base) + token * p.base_stride + column;
      r.out[h] = static_cast<T*>(p.out) + token * p.out_stride + column;
      r.out_limit[h] = token >= 0 ? columns_left : 0;
      r.base_limit[h] = p.base != nullptr ? r.out_limit[h] : 0;
    }
    return r;
  };
  auto load_base = [&](const Rows& rows, int h, int g) {
    Raw8<T> r;
    r.w[0] = make_uint4(0, 0, 0, 0);
    if constexpr (FAST) {
      if (32 * g < rows.base_limit[h]) r = load8(rows.base[h] + 32 * g);
    } else {
      T* e = reinterpret_cast<T*>(&r);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (32 * g + j < rows.base_limit[h]) e[j] = rows.base[h][32 * g + j];
      }
    }
    return r;
  };

  Tile tile = p.tiles[first];
  Rows rows = look(tile), next_rows{};
  Raw8<T> part[S::kGroups][2];
#pragma unroll
  for (int g = 0; g < S::kGroups; ++g) {
#pragma unroll
    for (int h = 0; h < 2; ++h) part[g][h] = load_base(rows, h, g);
  }
  int adapter = -1;  // whose weight is in shared memory
  if (adapted(tile)) load_weight(adapter = tile.adapter);
  griddep_wait();  // `low` from here on
  if (adapted(tile)) load_low(tile, 0);
  cp_async_commit();
  Tile next = first + 1 < last ? p.tiles[first + 1] : Tile{0, 0, -1};
  // Fragment addresses: low rows, and the weight's columns in the order above.
  const uint32_t low_from = low_shared + ((ROWS == kWide ? warp * 16 : 0) + (lane & 15)) * pitch + (lane >> 4) * 16;
  uint32_t weight_from[2];
#pragma unroll
  for (int pair = 0; pair < 2; ++pair) {
    const int i = lane & 7, j = 2 * pair + (lane >> 4), c = (i >> 1) * 8 + j * 2 + (i & 1);
    weight_from[pair] = weight_shared + (TRANS ? (((lane >> 3) & 1) * 8 + i) * kTransPitch + pair * 32 + (lane >> 4) * 16
                                               : c * pitch + (c >> 3) * 32 + ((lane >> 3) & 1) * 16);
    if (ROWS == kNarrow) weight_from[pair] += warp * (TRANS ? 64 : group_bytes);
  }
  for (int t = first; t < last; ++t) {
    const int buffer = two_buffers ? (t - first) & 1 : 0;
    const bool more = t + 1 < last;
    const Tile after = t + 2 < last ? p.tiles[t + 2] : Tile{0, 0, -1};
    next_rows = look(next);
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
    const uint32_t low = low_from + buffer * low_bytes;
    auto group = [&](int g, bool mine) {
      float acc[4][4];  // base, to which the products are added
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
        unpack8(part[g][h], v);
        part[g][h] = load_base(next_rows, h, g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[j][2 * h] = v[2 * j];
          acc[j][2 * h + 1] = v[2 * j + 1];
        }
      }
      if (mine) {
        auto step = [&](int k) {
          uint32_t hi[4], lo[4];
          ldmatrix_x4(hi, low + k * 2);
          ldmatrix_x4(lo, low + ROWS * pitch + k * 2);
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            uint32_t b[4];
            if constexpr (!TRANS) ldmatrix_x4(b, weight_from[pair] + g * group_bytes + k * 2);
            else ldmatrix_x4_trans(b, weight_from[pair] + g * 64 + k * kTransPitch);
            mma_16816<T>(acc[2 * pair], hi, b);
            mma_16816<T>(acc[2 * pair + 1], hi, b + 2);
            mma_16816<T>(acc[2 * pair], lo, b);
            mma_16816<T>(acc[2 * pair + 1], lo, b + 2);
          }
        };
        if constexpr (PAD > 0) {
#pragma unroll
          for (int k = 0; k < PAD; k += 16) step(k);
        } else {
          for (int k = 0; k < pad; k += 16) step(k);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] = acc[j][2 * h];
          v[2 * j + 1] = acc[j][2 * h + 1];
        }
        T* to = rows.out[h] + 32 * g;
        if constexpr (FAST) {
          if (32 * g < rows.out_limit[h]) store8(to, pack8<T>(v));
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (32 * g + j < rows.out_limit[h]) to[j] = from_float<T>(v[j]);
          }
        }
      }
    };
    if (adapted(tile)) {
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) group(g, true);
    } else {
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) group(g, false);
    }
    if (!two_buffers) {
      __syncthreads();
      if (more && adapted(next)) load_low(next, 0);
      cp_async_commit();
      cp_async_wait<0>();
    }
    tile = next;
    next = after;
    rows = next_rows;
  }
}

// ------------------------------------------------------------------- outer ----

// dW[column, r] = sum over the adapter's slots of row[column] * low[r]. A
// block takes 128 columns and RANK ranks; the blocks of a cluster share the
// adapter's tokens.
template <int RANK>
struct OuterShape {
  static constexpr int kThreads = 256;
  static constexpr int kColumns = 256;
  static constexpr int kTokens = 32;
  static constexpr int kStages = 4;
  static constexpr int kLook = 2 * kStages;  // token lists in flight
  static constexpr int kRowBytes = (kColumns + 8) * 2;
  static constexpr int kLowBytes = (RANK + 8) * 2;
  static constexpr int kStageBytes = kTokens * (kRowBytes + 2 * kLowBytes);
  static constexpr int kPartPitch = RANK + 1;
  static constexpr int kPartBytes = kColumns * kPartPitch * 4;
  static constexpr int kBytes = kStages * kStageBytes > kPartBytes ? kStages * kStageBytes : kPartBytes;
};

template <typename T, int RANK, bool FAST>
__global__ void __launch_bounds__(OuterShape<RANK>::kThreads, 2) adapter_outer(AdapterParams p) {
  using S = OuterShape<RANK>;
  extern __shared__ __align__(16) uint8_t shared[];
  __shared__ int32_t tokens[S::kLook][S::kTokens];
  const uint32_t stages = smem_u32(shared);
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

  constexpr int kPieces = S::kColumns / 8, kRowStep = S::kThreads / kPieces, kRowCopies = S::kTokens / kRowStep;
  constexpr int kLowPieces = RANK / 8, kLowStep = S::kThreads / kLowPieces;
  constexpr int kLowCopies = (2 * S::kTokens + kLowStep - 1) / kLowStep;
  const int piece = tid % kPieces, row_of = tid / kPieces;
  const int low_piece = tid % kLowPieces, low_row = tid / kLowPieces;
  const T* x = static_cast<const T*>(p.rows_in) + column0 + piece * 8;
  const int columns_left = static_cast<int>(p.width - column0) - piece * 8;
  const bool low_in = rank0 + low_piece * 8 < p.rank_pad;
  const T* low = static_cast<const T*>(p.low) + (low_in ? rank0 + low_piece * 8 : 0);
  const uint32_t row_to = stages + row_of * S::kRowBytes + piece * 16;
  const uint32_t low_to = stages + S::kTokens * S::kRowBytes + low_row * S::kLowBytes + low_piece * 16;

  // The tokens of a tile are copied kStages - 1 tiles before its rows.
  auto look = [&](int tile) {
    const int64_t slot = begin + static_cast<int64_t>(tile) * S::kTokens + tid;
    if (tid >= S::kTokens || tile >= last) return;
    if (slot < end) cp_async4(smem_u32(&tokens[tile % S::kLook][tid]), p.rows + slot);
    else tokens[tile % S::kLook][tid] = -1;
  };
  auto load = [&](int tile) {
    const uint32_t stage = static_cast<uint32_t>((tile - first) % S::kStages) * S::kStageBytes;
#pragma unroll
    for (int i = 0; i < kRowCopies; ++i) {
      const int32_t token = tokens[tile % S::kLook][row_of + i * kRowStep];
      const bool in = token >= 0 && token < p.tokens && columns_left > 0;
      copy8<T, FAST>(row_to + stage + i * kRowStep * S::kRowBytes,
                     in ? x + token * p.row_stride : static_cast<const T*>(p.rows_in), in ? columns_left : 0);
    }
    const int slot0 = begin + tile * S::kTokens;
#pragma unroll
    for (int i = 0; i < kLowCopies; ++i) {
      const int at = low_row + i * kLowStep, row = at % S::kTokens;
      if (2 * S::kTokens % kLowStep != 0 && at >= 2 * S::kTokens) continue;
      const bool in = low_in && slot0 + row < end;
      cp_async16(low_to + stage + i * kLowStep * S::kLowBytes,
                 in ? low + (at / S::kTokens * p.slots + slot0 + row) * p.rank_pad : low, in);
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
  const uint32_t a_from = stages + ((lane >> 4) * 8 + (lane & 7)) * S::kRowBytes + (warp * 32 + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t b_from = stages + S::kTokens * S::kRowBytes + (((lane >> 3) & 1) * 8 + (lane & 7)) * S::kLowBytes +
                          (lane >> 4) * 16;
  for (int tile = first; tile < last; ++tile) {
    cp_async_wait<S::kStages - 2>();
    __syncthreads();
    if (tile + S::kStages - 1 < last) load(tile + S::kStages - 1);
    look(tile + 2 * (S::kStages - 1));
    cp_async_commit();
    const uint32_t stage = static_cast<uint32_t>((tile - first) % S::kStages) * S::kStageBytes;
#pragma unroll
    for (int k = 0; k < S::kTokens; k += 16) {
      uint32_t a[2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m) ldmatrix_x4_trans(a[m], a_from + stage + k * S::kRowBytes + m * 32);
#pragma unroll
      for (int n = 0; n < RANK / 16; ++n) {
#pragma unroll
        for (int plane = 0; plane < 2; ++plane) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, b_from + stage + (plane * S::kTokens + k) * S::kLowBytes + n * 32);
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
  for (int e = static_cast<int>(split) * S::kThreads + tid; e < S::kColumns * RANK;
       e += static_cast<int>(splits) * S::kThreads) {
    const int c = columns_fast ? e % S::kColumns : e / RANK;
    const int r = columns_fast ? e / S::kColumns : e % RANK;
    if (column0 + c >= p.width || rank0 + r >= p.rank) continue;
    float v = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < splits; ++s) v += load_cluster_f32(mapa_shared(part, s) + (c * S::kPartPitch + r) * 4);
    out[(column0 + c) * p.out_stride + (rank0 + r) * p.out_rank_stride] = from_float<T>(v);
  }
  cluster_sync();
}

// -------------------------------------------------------------------- host ----

template <typename Kernel>
int launch_clustered(Kernel kernel, const AdapterParams& p, dim3 grid, int threads, int cluster, int shared,
                     bool dependent, cudaStream_t stream) {
  if (shared > 48 * 1024) {
    SDC_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared));
  }
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
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

// Blocks that share a tile's sum: as many as fill the SMs' `resident` blocks
// each once, as long as each keeps two chunks.
int split_count(int64_t blocks, int64_t chunks, int resident) {
  const int64_t wanted = std::min<int64_t>(static_cast<int64_t>(resident) * sm_count() / std::max<int64_t>(blocks, 1), chunks / 2);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(wanted, kMaxSplit)));
}

template <typename T, int ROWS, int RANK, bool TRANS>
int launch_shrink(AdapterParams p, int64_t tiles, cudaStream_t stream) {
  using S = ShrinkShape<ROWS, RANK, TRANS>;
  const int64_t chunks = ceil_div(p.width, S::kChunk);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int split = split_count(tiles * rank_blocks, chunks, ROWS == kWide ? 2 : 4);
  p.chunks_per_split = static_cast<int>(ceil_div(chunks, split));
  const dim3 grid(static_cast<unsigned>(tiles * split), rank_blocks);
  const bool fast = p.vector_rows && p.vector_weight && p.width % 8 == 0 && (!TRANS || p.rank % 8 == 0);
  return fast ? launch_clustered(adapter_shrink<T, ROWS, RANK, TRANS, true>, p, grid, S::kThreads, split, S::kBytes, false, stream)
              : launch_clustered(adapter_shrink<T, ROWS, RANK, TRANS, false>, p, grid, S::kThreads, split, S::kBytes, false, stream);
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
  if (tile_rows == kWide) return trans ? shrink_by_rank<T, kWide, true>(p, tiles, stream) : shrink_by_rank<T, kWide, false>(p, tiles, stream);
  return trans ? shrink_by_rank<T, kNarrow, true>(p, tiles, stream) : shrink_by_rank<T, kNarrow, false>(p, tiles, stream);
}

template <typename T, int ROWS, bool TRANS>
int launch_expand(AdapterParams p, int64_t tiles, bool dependent, cudaStream_t stream) {
  using S = ExpandShape<ROWS>;
  constexpr int kColumns = S::kColumns;
  const int64_t column_blocks = ceil_div(p.width, kColumns);
  // Runs of tiles that fill the SMs' blocks once; tiles of few rows
  // are bound by the weight, of which each then wants its own.
  p.tile_count = static_cast<int>(tiles);
  const int64_t runs = std::max<int64_t>(1, S::kBlocks * sm_count() / column_blocks);
  p.tiles_per_block = ROWS == kWide ? static_cast<int>(ceil_div(tiles, runs)) : 1;
  const int64_t blocks = column_blocks * ceil_div(tiles, p.tiles_per_block);
  SDC_REQUIRE(blocks <= INT_MAX, "low-rank adapters have too many tiles for one launch");
  while ((8 << p.piece_bits) < p.rank_pad) ++p.piece_bits;
  dependent = dependent && ROWS == kNarrow;  // blocks of long runs that start early, where there is room, end late
  const int shared = expand_bytes(ROWS, kColumns, p.rank_pad, TRANS);
  const dim3 grid(static_cast<unsigned>(blocks));
  const bool fast = p.vector_rows && p.vector_out && p.vector_weight && p.width % 8 == 0 && (TRANS || p.rank % 8 == 0);
  if (!fast) return launch_clustered(adapter_expand<T, ROWS, TRANS, false, 0>, p, grid, ExpandShape<ROWS>::kThreads, 0, shared, dependent, stream);
  switch (p.rank_pad) {
    case 16: return launch_clustered(adapter_expand<T, ROWS, TRANS, true, 16>, p, grid, ExpandShape<ROWS>::kThreads, 0, shared, dependent, stream);
    case 32: return launch_clustered(adapter_expand<T, ROWS, TRANS, true, 32>, p, grid, ExpandShape<ROWS>::kThreads, 0, shared, dependent, stream);
    case 64: return launch_clustered(adapter_expand<T, ROWS, TRANS, true, 64>, p, grid, ExpandShape<ROWS>::kThreads, 0, shared, dependent, stream);
    default: return launch_clustered(adapter_expand<T, ROWS, TRANS, true, 0>, p, grid, ExpandShape<ROWS>::kThreads, 0, shared, dependent, stream);
  }
}

template <typename T>
int expand_typed(const AdapterParams& p, int tile_rows, bool trans, int64_t tiles, bool dependent, cudaStream_t stream) {
  if (tile_rows == kWide) {
    return trans ? launch_expand<T, kWide, true>(p, tiles, dependent, stream)
                 : launch_expand<T, kWide, false>(p, tiles, dependent, stream);
  }
  return trans ? launch_expand<T, kNarrow, true>(p, tiles, dependent, stream)
               : launch_expand<T, kNarrow, false>(p, tiles, dependent, stream);
}

template <typename T, int RANK>
int launch_outer(const AdapterParams& p, cudaStream_t stream) {
  using S = OuterShape<RANK>;
  const int64_t columns = ceil_div(p.width, S::kColumns);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int64_t tiles = ceil_div(ceil_div(p.slots, p.adapters), S::kTokens);
  const int split = split_count(columns * p.adapters * rank_blocks, tiles, 2);
  const dim3 grid(static_cast<unsigned>(columns * split), static_cast<unsigned>(p.adapters), rank_blocks);
  return p.vector_rows && p.width % 8 == 0
             ? launch_clustered(adapter_outer<T, RANK, true>, p, grid, S::kThreads, split, S::kBytes, false, stream)
             : launch_clustered(adapter_outer<T, RANK, false>, p, grid, S::kThreads, split, S::kBytes, false, stream);
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
  SDC_REQUIRE(tile_rows == kNarrow || (tile_rows == kWide && rank <= kMaxWideRank),
              "low-rank adapter tiles have 16 rows, or 128 for ranks of up to 128");
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
  SDC_REQUIRE(tile_rows == kNarrow || (tile_rows == kWide && rank <= kMaxWideRank),
              "low-rank adapter tiles have 16 rows, or 128 for ranks of up to 128");
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
