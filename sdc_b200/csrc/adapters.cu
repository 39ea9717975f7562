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
// are gathered into tiles of 128 rows, whose products accumulate in tensor
// memory, or of 16 when adapters have few tokens, as in decoding, where the
// weights are the traffic. Sums over the width or over the tokens are fp32,
// across the blocks of a cluster through distributed shared memory in a fixed
// order, so nothing is added in an order that changes.
//
// Copies are each thread's own (16 bytes, zeros where there is nothing): the
// rows of a tile lie anywhere, and any stride and alignment is taken.
//
// `low` is kept as two 16-bit planes, hi = round(v) and lo = round(v - hi):
// the tensor cores take 16-bit operands, and the second product then loses
// 2^-17 of v (2^-21 in fp16) rather than 2^-9, for one more multiply on pipes
// that wait for memory anyway. bf16 has the range of fp32. fp16 has not: small
// rows (gradients of a mean loss) would lose their second plane and then their
// first, large ones would overflow although the other weight brings them back.
// Its rows are therefore scaled by a power of two that brings the largest finite
// value into [2^14, 2^15), and products are scaled back: by each row's own power
// in expand, so that no token depends on another, in outer by one for the tokens
// that a block adds up. What is 2^-17 of the largest keeps all 21 bits, and 2^-39
// of it is what is lost. The power travels in the row itself, as the lowest bits
// of the first eight values of the second plane.
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "mma.cuh"

namespace sdc {
namespace {

constexpr int kWide = 128, kNarrow = 16;  // rows of a tile
constexpr int kMaxWideRank = 128;         // beyond, a wide tile's low rows and weight do not fit together
constexpr int kMaxRank = 256;
constexpr int kMaxSplit = 16;  // blocks of a cluster
constexpr int kPortableSplit = 8;

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
  int32_t* watchdog;
  uint64_t wait_limit_ns;
  bool expire;               // test hook: a wait that nothing ends
  int tile_count, tiles_per_block;  // expand
  int weights;               // expand of wide tiles: buffers of weights, 1 or 2
  int piece_bits;            // expand: 2^piece_bits >= rank_pad / 8 threads copy a row
};

__device__ __forceinline__ int64_t token_of(const AdapterParams& p, int64_t slot) {
  const int32_t token = p.rows[slot];
  return token >= 0 && token < p.tokens ? token : -1;
}

// ------------------------------------------------------------------ shrink ----

template <typename T>
constexpr bool kScaled = std::is_same_v<T, __half>;  // the rows of `low` are

// N neighbouring values of a row's two planes.
template <typename T, int N>
struct alignas(2 * N) Planes {
  T hi[N];
  alignas(2 * N) T lo[N];
};
template <typename T, int N>
__device__ __forceinline__ Planes<T, N> split(const float (&v)[N]) {
  Planes<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    r.hi[i] = from_float<T>(v[i]);
    const float rest = v[i] - to_float(r.hi[i]);
    r.lo[i] = from_float<T>(isfinite(rest) ? rest : 0.f);  // an infinite sum stays one
  }
  return r;
}

// Scaled rows. `back` is the exponent (biased, as in fp32) of the power of two
// that undoes a row's scale: 1 for rows of zeros, so that the bits that hold it
// vanish from the products as well.
__device__ __forceinline__ float power_of_two(uint32_t exponent) { return __uint_as_float(exponent << 23); }
template <int N>
__device__ __forceinline__ float largest_finite(const float (&v)[N]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(v[i]) < INFINITY ? fabsf(v[i]) : 0.f);
  return most;
}
template <int LANES>
__device__ __forceinline__ float neighbours_max(float v) {
#pragma unroll
  for (int step = 1; step < LANES; step *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, step));
  return v;
}
__device__ __forceinline__ uint32_t back_for(float largest) {
  return static_cast<uint32_t>(max(static_cast<int>(__float_as_uint(largest) >> 23) - 14, 1));
}
// Values of a row from column `c` on, scaled, and the exponent's bits there.
template <typename T, int N>
__device__ __forceinline__ Planes<T, N> split_scaled(const float (&v)[N], uint32_t back, int c) {
  const float scale = power_of_two(254 - back);
  float scaled[N];
#pragma unroll
  for (int i = 0; i < N; ++i) scaled[i] = v[i] * scale;
  Planes<T, N> r = split<T, N>(scaled);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t bits = __half_as_ushort(r.lo[i]);
    if (c < 8) r.lo[i] = __ushort_as_half(static_cast<uint16_t>((bits & 0xfffeu) | (back >> (c + i) & 1u)));
  }
  return r;
}
// The exponent from the first eight values of a row's second plane.
__device__ __forceinline__ uint32_t back_of(const uint4& lo) {
  const uint32_t x = (lo.x & 0x10001u) | (lo.y & 0x10001u) << 2 | (lo.z & 0x10001u) << 4 | (lo.w & 0x10001u) << 6;
  return (x & 0x55u) | (x >> 15 & 0xaau);
}
__device__ __forceinline__ uint4 load_shared4(uint32_t shared) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(shared) : "memory");
  return w;
}

template <typename T, int N>
__device__ __forceinline__ void store_row_planes(const AdapterParams& p, int64_t slot, int c, const Planes<T, N>& r) {
  using Words = std::conditional_t<N == 4, uint2, std::conditional_t<N == 2, uint32_t, uint16_t>>;
  static_assert(sizeof(Words) == 2 * N, "one word a plane");
  T* to = static_cast<T*>(p.low) + slot * p.rank_pad + c;  // c is a multiple of N, rank_pad of 16
  *reinterpret_cast<Words*>(to) = *reinterpret_cast<const Words*>(r.hi);
  *reinterpret_cast<Words*>(to + p.slots * p.rank_pad) = *reinterpret_cast<const Words*>(r.lo);
}
// Where a row's fp32 values from column `c` on stand in the place of its
// planes: the first half in the first.
template <typename T>
__device__ __forceinline__ float* whole_row(const AdapterParams& p, int64_t slot, int c) {
  const int half = p.rank_pad / 2;
  T* plane = static_cast<T*>(p.low) + (slot + (c >= half ? p.slots : 0)) * p.rank_pad;
  return reinterpret_cast<float*>(plane) + (c >= half ? c - half : c);
}

// Writes neighbouring sums of a row, c columns into the rank, `in` where there
// is such a row. Columns that pad the rank are zeros whatever the row: an
// infinity times their missing weights is no sum. All lanes of a warp call it;
// LANES neighbours hold a row's part. Scaled rows in several parts wait as fp32
// for adapter_split.
template <typename T, int LANES, int N>
__device__ __forceinline__ void store_low(const AdapterParams& p, bool in, int64_t slot, int c, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = c + i < p.rank ? v[i] : 0.f;
  in = in && c < p.rank_pad;
  if constexpr (!kScaled<T>) {
    if (in) store_row_planes<T, N>(p, slot, c, split<T, N>(v));
  } else if (gridDim.y > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (in) *whole_row<T>(p, slot, c + i) = v[i];
    }
  } else {
    const uint32_t back = back_for(neighbours_max<LANES>(largest_finite<N>(v)));
    if (in) store_row_planes<T, N>(p, slot, c, split_scaled<T, N>(v, back, c));
  }
}

// Scaled rows of more than 64 ranks, whose parts come from different blocks of
// shrink: fp32 to planes in place, a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) adapter_split(AdapterParams p) {
  const Tile tile = p.tiles[blockIdx.x];
  if (tile.adapter < 0 || tile.adapter >= p.adapters) return;
  const int lane = threadIdx.x & 31;
  for (int row = threadIdx.x / 32; row < tile.count; row += 8) {
    const int64_t slot = static_cast<int64_t>(tile.start) + row;
    constexpr int kQuads = kMaxRank / 4 / 32;
    float v[kQuads][4];
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int c = (lane + 32 * i) * 4;
      const float4 q = c < p.rank_pad ? *reinterpret_cast<const float4*>(whole_row<T>(p, slot, c)) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[i][0] = q.x, v[i][1] = q.y, v[i][2] = q.z, v[i][3] = q.w;
      most = fmaxf(most, largest_finite<4>(v[i]));
    }
    const uint32_t back = back_for(neighbours_max<32>(most));  // the whole row has been read
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const int c = (lane + 32 * i) * 4;
      if (c < p.rank_pad) store_row_planes<T, 4>(p, slot, c, split_scaled<T, 4>(v[i], back, c));
    }
  }
}

// Tiles of 16 rows (decoding): the weight is the traffic, and the tensor
// memory's 128 rows would be empty. Four warps share the rows and take a
// quarter of each chunk of the width. RANK: columns of `low` per block. The
// width is split over a cluster of up to 8 blocks until they fill the SMs,
// and the expand kernel may start behind it (its weight and base do not wait).
// One row, width 3584, rank 16: 5.0 us, the time of a launch with a cluster's
// exchange; 192 rows of 48 adapters: 6.7 us.
template <int RANK, bool TRANS>
struct NarrowShape {
  static constexpr int ROWS = kNarrow;
  static constexpr int kThreads = 128;
  static constexpr int kChunk = 256;
  static constexpr int kStages = 4;
  static constexpr int kRowBytes = (kChunk + 8) * 2;  // 8 elements of padding: fragment rows on different banks
  static constexpr int kWeightRows = TRANS ? kChunk : RANK;
  static constexpr int kWeightBytes = ((TRANS ? RANK : kChunk) + 8) * 2;
  static constexpr int kStageBytes = ROWS * kRowBytes + kWeightRows * kWeightBytes;
  static constexpr int kPartRows = 4 * ROWS;
  static constexpr int kPartBytes = kPartRows * RANK * 4;
  static constexpr int kBytes = kStages * kStageBytes > kPartBytes ? kStages * kStageBytes : kPartBytes;
};

template <typename T, int RANK, bool TRANS, bool FAST>
__global__ void __launch_bounds__(NarrowShape<RANK, TRANS>::kThreads) adapter_shrink(AdapterParams p) {
  using S = NarrowShape<RANK, TRANS>;
  constexpr int ROWS = kNarrow;
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
  const int k_of = warp * (S::kChunk / 4);
  const uint32_t a_from = stages + (lane & 15) * S::kRowBytes + (k_of + (lane >> 4) * 8) * 2;
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
    constexpr int kSteps = S::kChunk / 64;
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
  constexpr int kEach = RANK > 32 ? RANK / 32 : 1, kLanes = RANK / kEach;  // a row's lanes
  for (int at = static_cast<int>(split) * S::kThreads + warp * 32; at < count * kLanes; at += static_cast<int>(splits) * S::kThreads) {
    const int e = at + lane, row = e / kLanes, c = e % kLanes * kEach;
    const bool in = row < count;
    float v[kEach] = {};
    if (in) {
#pragma unroll 4
      for (uint32_t s = 0; s < splits; ++s) {
        const uint32_t from = mapa_shared(part, s) + (row * RANK + c) * 4;
#pragma unroll
        for (int other = 0; other < 4; ++other) {
#pragma unroll
          for (int i = 0; i < kEach; ++i) v[i] += load_cluster_f32(from + (other * ROWS * RANK + i) * 4);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] *= scale;
    store_low<T, kLanes, kEach>(p, in, tile.start + row, rank0 + c, v);
  }
  cluster_sync();  // the others may still be reading this block's sums
}

// ---- tensor memory: shrink of wide tiles, and outer ----

// kind::f16 instruction: fp32 accumulators, both operands T; *_mn: the
// operand's rows (A) or columns (B) are contiguous in memory, not its K.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool a_mn, bool b_mn) {
  const uint32_t type = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// Layouts of the operands in shared memory.
//   swizzled  rows of 128 bytes in groups of 8 (1024 bytes); the 16-byte
//             pieces of row r are permuted by r % 8 (128-byte swizzle). K-major
//             when a row holds K, MN-major when it holds 64 rows of A.
//   panels    (MN-major, no swizzle) the 8 columns n of a panel for 8 values
//             of K are 8 consecutive 16-byte pieces; K groups are 128 bytes
//             apart, panels `stride`.
__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }
__device__ __forceinline__ uint32_t paneled(int k, int panel, int stride) { return panel * stride + k * 16; }

// A ring of stages that eight warps fill and a ninth multiplies from. A
// filling is full when every filling thread's copies have arrived, and its
// stage is free again when the products that read it have completed. Waits
// are bounded: one that runs out is recorded in the watchdog word, the warps
// leave their loops one after the other and meet at the block's next barrier,
// where the block's sums become NaN, so that nothing made of them looks whole.
constexpr int kFillThreads = 256, kTensorThreads = kFillThreads + 32;

template <int STAGES>
struct TensorRing {
  uint64_t full[STAGES], used[STAGES], never;
  uint32_t tensor_memory;
  int32_t abort;

  // One warp; everyone else sees it after the block's next barrier.
  __device__ __forceinline__ void start(int columns) {
    if ((threadIdx.x & 31) == 0) {
      for (int i = 0; i < STAGES; ++i) {
        mbar_init(&full[i], kFillThreads);
        mbar_init(&used[i], 1);
      }
      mbar_init(&never, 1);
      fence_barrier_init();
      abort = 0;
    }
    __syncwarp();
    tmem_alloc(&tensor_memory, static_cast<uint32_t>(columns));
    tmem_relinquish();
  }
  // Until the index-th filling is full, or its products have completed. The
  // same for a whole warp.
  __device__ __forceinline__ bool wait(uint64_t* bars, int index, const AdapterParams& p) {
    return wait_bar(&bars[index % STAGES], static_cast<uint32_t>(index / STAGES) & 1, p);
  }
  __device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, const AdapterParams& p) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, kWaitAdapters, &abort, p.watchdog, p.wait_limit_ns)) != 0;
  }
  // A filling thread's copies of a filling have been issued (FAST: the
  // barrier counts it when they arrive) or made.
  template <bool FAST>
  __device__ __forceinline__ void filled(int index) {
    if constexpr (FAST) {
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[index % STAGES]))
                   : "memory");
    } else {
      cp_async_commit();
      cp_async_wait<0>();
      mbar_arrive(&full[index % STAGES]);
    }
  }
  // After the block's barrier behind the loops.
  __device__ __forceinline__ bool gave_up() const { return abort != 0; }
  __device__ __forceinline__ float instead() const { return gave_up() ? __int_as_float(0x7fffffff) : 0.f; }
  __device__ __forceinline__ void drain(int index) {
    mbar_drain(&used[index % STAGES], static_cast<uint32_t>(index / STAGES) & 1);
  }
  // The ninth warp: products of `count` fillings, issued by one lane.
  template <typename Products>
  __device__ __forceinline__ void multiply(int count, const AdapterParams& p, const Products& products) {
    int done = 0;
    if (p.expire && count > 0 && !wait_bar(&never, 0, p)) return;
    for (; done < count; ++done) {
      if (!wait(full, done, p)) break;
      fence_proxy_async_smem();  // the copies were made by ordinary writes
      tc_fence_after();
      if ((threadIdx.x & 31) == 0) {
        products(done);
        tc_commit(&used[done % STAGES]);
      }
      __syncwarp();
    }
    if (abort != 0 && done > 0 && (threadIdx.x & 31) == 0) drain(done - 1);  // nothing may stay in flight
    __syncwarp();
  }
};

// Sums in shared memory: rows of RANK floats and 16 bytes of padding (the
// lanes of a tensor-memory load write their rows' words to different banks).
// Four neighbouring ones over the blocks of a cluster, in their order.
__device__ __forceinline__ float4 sum_cluster(const float* part, int at, uint32_t splits) {
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (uint32_t s = 0; s < splits; ++s) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(mapa_shared(part, s) + at * 4)
                 : "memory");
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  return sum;
}
// This thread's row of an accumulator, or `instead` where nothing was multiplied;
// PLANES: 2 where RANK further columns hold the second plane's sums.
template <int RANK, int PLANES>
__device__ __forceinline__ void store_part(float* row, uint32_t accumulator, bool any, float instead, float back = 1.f) {
  constexpr int kStep = RANK < 32 ? RANK : 32;
#pragma unroll
  for (int c0 = 0; c0 < RANK; c0 += kStep) {
    uint32_t v[32];
    tmem_ld_32x32b_x32(accumulator + c0, v);
    tmem_ld_wait();
    float f[kStep];
#pragma unroll
    for (int c = 0; c < kStep; ++c) f[c] = __uint_as_float(v[c]);
    if constexpr (PLANES == 2 && 2 * RANK <= 32) {
#pragma unroll
      for (int c = 0; c < kStep; ++c) f[c] += __uint_as_float(v[RANK + c]);
    } else if constexpr (PLANES == 2) {
      tmem_ld_32x32b_x32(accumulator + RANK + c0, v);
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < kStep; ++c) f[c] += __uint_as_float(v[c]);
    }
#pragma unroll
    for (int c = 0; c < kStep; c += 4) {
      *reinterpret_cast<float4*>(row + c0 + c) =
          any ? make_float4(f[c] * back, f[c + 1] * back, f[c + 2] * back, f[c + 3] * back)
              : make_float4(instead, instead, instead, instead);
    }
  }
}

template <int RANK, bool TRANS>
struct WideShape {
  static constexpr int kThreads = kTensorThreads;
  static constexpr int kChunk = 64;  // of the width: one swizzled row of 128 bytes
  static constexpr int kStages = 4;
  static constexpr int kRowBytes = kWide * 128;
  static constexpr int kStageBytes = kRowBytes + kChunk * RANK * 2;
  static constexpr int kTensorColumns = RANK < 32 ? 32 : RANK;
  static constexpr int kPartPitch = RANK + 4;
  static constexpr int kPartBytes = kWide * kPartPitch * 4;
  static constexpr int kBytes = 1024 + (kStages * kStageBytes > kPartBytes ? kStages * kStageBytes : kPartBytes);
};

// Tiles of 128 rows: D [128, RANK] in tensor memory. The rows are A (K-major,
// swizzled); the weight chunk is B, K-major and swizzled ([rank, width]) or in
// panels ([width, rank]). Two blocks an SM keep 128 KB of copies under way.
// 16384 x 3584 bf16, rank 32: 25.7 us (4.6 TB/s), of which about 10 start and
// end the launch: each further 16384 rows take 19.3 (6.1 TB/s, bound by
// memory). Register accumulators and mma.sync took 35. Chunks of 128 columns
// and 3 to 6 stages measured the same.
template <typename T, int RANK, bool TRANS, bool FAST>
__global__ void __launch_bounds__(WideShape<RANK, TRANS>::kThreads, 2) adapter_shrink_wide(AdapterParams p) {
  using S = WideShape<RANK, TRANS>;
  extern __shared__ uint8_t shared_raw[];
  __shared__ TensorRing<S::kStages> ring;
  uint8_t* shared = shared_raw + (-smem_u32(shared_raw) & 1023u);  // the swizzle goes by address bits
  const uint32_t stages = smem_u32(shared);
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = cluster_ctarank();
  const Tile tile = p.tiles[blockIdx.x / splits];
  const int rank0 = blockIdx.y * RANK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 8) ring.start(S::kTensorColumns);
  const bool valid = tile.adapter >= 0 && tile.adapter < p.adapters;
  const int count = valid ? tile.count : 0;
  const int width = static_cast<int>(p.width);
  const int chunks = (width + S::kChunk - 1) / S::kChunk;
  const int first = min(static_cast<int>(split) * p.chunks_per_split, chunks);
  const int last = min(first + p.chunks_per_split, chunks);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t accumulator = ring.tensor_memory;

  if (warp < 8) {
    constexpr int kPieces = 8, kRowStep = kFillThreads / kPieces, kRowCopies = kWide / kRowStep;
    constexpr int kWeightPieces = TRANS ? RANK / 8 : kPieces, kWeightRows = TRANS ? S::kChunk : RANK;
    constexpr int kWeightStep = kFillThreads / kWeightPieces;
    constexpr int kWeightCopies = (kWeightRows + kWeightStep - 1) / kWeightStep;
    const int piece = tid % kPieces, row_of = tid / kPieces;
    const int weight_piece = tid % kWeightPieces, weight_row = tid / kWeightPieces;
    // Sources of the next chunk, and where they may no longer be read from:
    // columns left from this thread's piece on (0 for rows that are not there).
    const T* source[kRowCopies];
    int left[kRowCopies];
    const int skipped = first * S::kChunk;
#pragma unroll
    for (int i = 0; i < kRowCopies; ++i) {
      const int row = row_of + i * kRowStep;
      const int64_t token = row < count ? token_of(p, tile.start + row) : -1;
      source[i] = static_cast<const T*>(p.rows_in) + (token >= 0 ? token * p.row_stride : 0) + piece * 8 + skipped;
      left[i] = token >= 0 ? width - piece * 8 - skipped : 0;
    }
    const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(valid ? tile.adapter : 0) * p.rank * p.width;
    weight += TRANS ? static_cast<int64_t>(skipped + weight_row) * p.rank + rank0 + weight_piece * 8
                    : static_cast<int64_t>(rank0 + weight_row) * width + weight_piece * 8 + skipped;
    const int64_t weight_step = TRANS ? static_cast<int64_t>(kWeightStep) * p.rank : static_cast<int64_t>(kWeightStep) * width;
    const int64_t weight_chunk = TRANS ? static_cast<int64_t>(S::kChunk) * p.rank : S::kChunk;
    const int ranks_left = p.rank - rank0 - (TRANS ? weight_piece * 8 : weight_row);
    int weight_left = TRANS ? width - skipped - weight_row : width - skipped - weight_piece * 8;
    // Row and weight steps are multiples of 8: the swizzle is the same for all of a thread's copies.
    const uint32_t row_to = stages + swizzled(row_of, piece);
    const uint32_t weight_to = stages + S::kRowBytes +
                               (TRANS ? paneled(weight_row, weight_piece, S::kChunk * 16) : swizzled(weight_row, weight_piece));
    constexpr int kWeightStride = kWeightStep * (TRANS ? 16 : 128);
    for (int fill = 0; fill < last - first; ++fill) {
      if (fill >= S::kStages && !ring.wait(ring.used, fill - S::kStages, p)) break;
      const uint32_t stage = static_cast<uint32_t>(fill % S::kStages) * S::kStageBytes;
#pragma unroll
      for (int i = 0; i < kRowCopies; ++i) {
        copy8<T, FAST>(row_to + stage + i * kRowStep * 128, source[i], left[i]);
        source[i] += S::kChunk;
        left[i] -= S::kChunk;
      }
#pragma unroll
      for (int i = 0; i < kWeightCopies; ++i) {
        if (kWeightRows % kWeightStep != 0 && weight_row + i * kWeightStep >= kWeightRows) continue;
        const int in = TRANS ? (weight_left > i * kWeightStep ? ranks_left : 0) : (ranks_left > i * kWeightStep ? weight_left : 0);
        copy8<T, FAST>(weight_to + stage + i * kWeightStride, weight + i * weight_step, in);
      }
      weight += weight_chunk;
      weight_left -= S::kChunk;
      ring.filled<FAST>(fill);
    }
    cp_async_commit();
    cp_async_wait<0>();
  } else {
    constexpr uint32_t kInstruction = idesc_f16<T>(kWide, RANK, false, TRANS);
    const uint64_t a = sw128_desc(stages);
    const uint64_t b = TRANS ? smem_desc(stages + S::kRowBytes, 128, S::kChunk * 16, 0) : sw128_desc(stages + S::kRowBytes);
    ring.multiply(last - first, p, [&](int fill) {
      // Addresses advance in the descriptors' units of 16 bytes.
      const uint64_t stage = static_cast<uint64_t>(fill % S::kStages) * (S::kStageBytes / 16);
#pragma unroll
      for (int k = 0; k < S::kChunk / 16; ++k) {
        mma_bf16(accumulator, a + stage + k * 2, b + stage + k * (TRANS ? 16 : 2), kInstruction, fill > 0 || k > 0);
      }
    });
  }
  float* part = reinterpret_cast<float*>(shared);
  if (first < last) ring.wait(ring.used, last - 1 - first, p);
  tc_fence_after();
  __syncthreads();
  if (warp < 4) {
    store_part<RANK, 1>(part + (warp * 32 + lane) * S::kPartPitch, accumulator + (static_cast<uint32_t>(warp) << 21),
                        first < last && !ring.gave_up(), ring.instead());
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(accumulator, S::kTensorColumns);
  const float scale = p.scale != nullptr && valid ? p.scale[tile.adapter] : 1.f;
  constexpr int kQuads = RANK / 4;
  for (int at = static_cast<int>(split) * S::kThreads + warp * 32; at < count * kQuads; at += static_cast<int>(splits) * S::kThreads) {
    const int e = at + lane, row = e / kQuads, c = e % kQuads * 4;
    const bool in = e < count * kQuads;
    const float4 sum = in ? sum_cluster(part, row * S::kPartPitch + c, splits) : make_float4(0.f, 0.f, 0.f, 0.f);
    float v[4] = {sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale};
    store_low<T, kQuads, 4>(p, in, tile.start + row, rank0 + c, v);
  }
  cluster_sync();  // the others may still be reading this block's sums
}

// ------------------------------------------------------------------ expand ----

// Tiles of 16 rows: bound by the weight, of which each block reads 128 columns
// (with base, before it waits for `low`), and by the launch: one row of 3584
// columns takes 4.9 us, 192 rows of 48 adapters, width 4608, 9.6. Four warps, each all 16 rows of 32
// columns. A thread's accumulators over four 8-column tiles are made 8
// neighbouring columns by assigning column 8 q + 2 j + b of 32 to element
// 2 q + b of tile j: base and out then move in 16-byte words straight between
// registers and memory.
//
// Shared layout of the weight: !TRANS (weight [width, rank]): rows of a column's
// ranks and 8 elements of padding, each run of 8 columns skewed by 32 bytes so
// that the 8 rows of a fragment (columns 0, 1, 8, 9, 16, ... of a group) hit
// different banks. TRANS (weight [rank, width]): rows of permuted columns.
struct NarrowExpand {
  static constexpr int kThreads = 128;
  static constexpr int kColumns = 128;
  static constexpr int kTransPitch = (kColumns + 8) * 2;
  static __host__ __device__ constexpr int group_bytes(int pad) { return 32 * (pad + 8) * 2 + 96; }
  static __host__ __device__ constexpr int weight_bytes(int pad, bool trans) {
    return trans ? pad * kTransPitch : kColumns / 32 * group_bytes(pad);
  }
  static __host__ __device__ constexpr int bytes(int pad, bool trans) {
    return weight_bytes(pad, trans) + 2 * kNarrow * (pad + 8) * 2;
  }
};

// FAST: widths, strides and addresses allow 16-byte accesses throughout. PAD:
// rank_pad, or 0 where it is read from the parameters.
template <typename T, bool TRANS, bool FAST, int PAD>
__global__ void __launch_bounds__(NarrowExpand::kThreads, 4) adapter_expand(AdapterParams p) {
  using S = NarrowExpand;
  extern __shared__ __align__(16) uint8_t shared[];
  const int pad = PAD > 0 ? PAD : p.rank_pad;
  const int width = static_cast<int>(p.width);
  const int column_blocks = (width + S::kColumns - 1) / S::kColumns;
  const Tile tile = p.tiles[blockIdx.x / column_blocks];
  const int column0 = static_cast<int>(blockIdx.x % column_blocks) * S::kColumns;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int pitch = (pad + 8) * 2;  // bytes of a low row, and of a weight row when !TRANS
  const int group_bytes = S::group_bytes(pad);
  const uint32_t weight_shared = smem_u32(shared);
  const uint32_t low_shared = weight_shared + S::weight_bytes(pad, TRANS);
  const int piece_bits = PAD > 0 ? (PAD <= 16 ? 1 : PAD <= 32 ? 2 : 3) : p.piece_bits;
  const int piece = tid & ((1 << piece_bits) - 1), piece_row = tid >> piece_bits;
  const int piece_step = S::kThreads >> piece_bits;
  const bool adapted = tile.adapter >= 0 && tile.adapter < p.adapters;

  if (adapted) {
    const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(tile.adapter) * p.rank * p.width;
    if constexpr (!TRANS) {
      for (int c = piece_row; c < S::kColumns && piece * 8 < pad; c += piece_step) {
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
        const uint32_t to = weight_shared + r * S::kTransPitch + (c & ~31) * 2 + ((c >> 3) & 3) * 4;
        asm volatile("st.shared.b32 [%0], %1;\n\tst.shared.b32 [%0 + 16], %2;\n\t"
                     "st.shared.b32 [%0 + 32], %3;\n\tst.shared.b32 [%0 + 48], %4;" ::"r"(to), "r"(w.x), "r"(w.y),
                     "r"(w.z), "r"(w.w)
                     : "memory");
      }
    }
  }

  // This thread's part of base and out: rows lane / 4 and lane / 4 + 8, 8
  // columns of the warp's 32. The accumulators start from it, or it is added to
  // the products of scaled rows.
  const int column = column0 + warp * 32 + (lane & 3) * 8;
  float acc[4][4];
  Raw8<T> base[2];
  T* out[2];
  int limit[2];  // columns of out; 0 where there is no row
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = (lane >> 2) + 8 * h;
    const int64_t token = row < tile.count ? token_of(p, tile.start + row) : -1;
    limit[h] = token >= 0 ? width - column : 0;
    out[h] = static_cast<T*>(p.out) + token * p.out_stride + column;
    base[h].w[0] = make_uint4(0, 0, 0, 0);
    const T* from = static_cast<const T*>(p.base) + token * p.base_stride + column;
    if (p.base != nullptr) {
      if constexpr (FAST) {
        if (limit[h] > 0) base[h] = load8(from);
      } else {
        T* e = reinterpret_cast<T*>(&base[h]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < limit[h]) e[j] = from[j];
        }
      }
    }
    float v[8];
    unpack8(base[h], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[j][2 * h] = kScaled<T> ? 0.f : v[2 * j];
      acc[j][2 * h + 1] = kScaled<T> ? 0.f : v[2 * j + 1];
    }
  }

  griddep_wait();  // `low` from here on
  if (adapted) {
    const T* from = static_cast<const T*>(p.low) + static_cast<int64_t>(tile.start) * pad + piece * 8;
    for (int i = piece_row; i < 2 * kNarrow && piece * 8 < pad; i += piece_step) {
      const int row = i % kNarrow;
      const bool in = row < tile.count;
      cp_async16(low_shared + i * pitch + piece * 16, in ? from + (i >= kNarrow ? p.slots * pad : 0) + row * pad : from, in);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    const uint32_t low = low_shared + (lane & 15) * pitch + (lane >> 4) * 16;
    auto step = [&](int k) {
      uint32_t hi[4], lo[4];
      ldmatrix_x4(hi, low + k * 2);
      ldmatrix_x4(lo, low + kNarrow * pitch + k * 2);
#pragma unroll
      for (int pair = 0; pair < 2; ++pair) {
        uint32_t b[4];
        const int i = lane & 7, j = 2 * pair + (lane >> 4), c = (i >> 1) * 8 + j * 2 + (i & 1);
        if constexpr (!TRANS) {
          ldmatrix_x4(b, weight_shared + warp * group_bytes + c * pitch + (c >> 3) * 32 + ((lane >> 3) & 1) * 16 + k * 2);
        } else {
          ldmatrix_x4_trans(b, weight_shared + (((lane >> 3) & 1) * 8 + i + k) * S::kTransPitch + warp * 64 + j * 16);
        }
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
    if (kScaled<T> && adapted) {
      const float back = power_of_two(back_of(load_shared4(low_shared + (kNarrow + (lane >> 2) + 8 * h) * pitch)));
      unpack8(base[h], v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = fmaf(acc[j][2 * h], back, v[2 * j]);
        v[2 * j + 1] = fmaf(acc[j][2 * h + 1], back, v[2 * j + 1]);
      }
    } else if constexpr (kScaled<T>) {
      unpack8(base[h], v);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[2 * j] = acc[j][2 * h], v[2 * j + 1] = acc[j][2 * h + 1];
    }
    if constexpr (FAST) {
      if (limit[h] > 0) store8(out[h], pack8<T>(v));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < limit[h]) out[h][j] = from_float<T>(v[j]);
      }
    }
  }
}

// ---- expand of wide tiles ----

// A block keeps 256 columns of one adapter's weight in shared memory and walks
// a run of tiles. D [128 rows, 256 columns] in tensor memory is the product of
// a tile's two low planes (A, K-major panels) with the weight (B); eight warps
// add it to base, 32 columns of 16 rows at a time: a 16x256b load gives a
// thread rows lane / 4 and lane / 4 + 8 and two columns of each 8. The weight's
// columns are permuted within 32 (column 8 q + 2 j + b stands at 8 j + 2 q + b)
// so that these are 8 neighbours, and base and out move in 16-byte words. The
// next tile's part of base is loaded as soon as the current one's has been
// used, its low rows (and weight, if another) while the current tile is worked
// on. Bound by base and out: 16384 x 3584 bf16, rank 32, 49 us (4.8 TB/s; each
// further 16384 rows take 40, 5.8 TB/s), rank 64 63 us (register accumulators
// and mma.sync: 80); 8191 x 18944 fp16 of 23 ragged adapters 122 us (5.0 TB/s).
// Blocks of 128 columns, two or three to an SM, took 58 and 66 us for the
// first; runs half as long, in two waves, 57, though 4 % less where ragged
// adapters leave the runs uneven.
struct ExpandWide {
  static constexpr int kThreads = kFillThreads;
  static constexpr int kColumns = 256;
  static constexpr int kWarps = 8, kHalves = 2, kGroups = 4;  // a warp: 32 rows of 128 columns
  static constexpr int kWeightStep = kColumns * 16, kLowStep = kWide * 16;  // bytes of 8 ranks
  static __host__ __device__ constexpr int weight_bytes(int pad) { return pad / 8 * kWeightStep; }
  static __host__ __device__ constexpr int low_bytes(int pad) { return 2 * (pad / 8) * kLowStep; }  // of one tile
  static __host__ __device__ constexpr int bytes(int pad, int weights) { return weights * weight_bytes(pad) + 2 * low_bytes(pad); }
  static constexpr int kBlockBytes = 110 * 1024;  // of two blocks on an SM
};

// 16 rows of 32 columns: v[4 j ..] are tile j's (row lane / 4: two columns;
// row lane / 4 + 8: the same).
__device__ __forceinline__ void tmem_ld_16x256b_x4(uint32_t address, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(address));
}

template <typename T, bool TRANS, bool FAST>
__global__ void __launch_bounds__(ExpandWide::kThreads, 2) adapter_expand_wide(AdapterParams p) {
  using S = ExpandWide;
  extern __shared__ __align__(128) uint8_t shared[];
  __shared__ uint64_t loaded[2], ready, drained, never;
  __shared__ uint32_t tensor_memory;
  __shared__ int32_t abort;
  const int width = static_cast<int>(p.width), pad = p.rank_pad, pieces = pad / 8;
  const int column_blocks = (width + S::kColumns - 1) / S::kColumns;
  const int run = static_cast<int>(blockIdx.x) / column_blocks;
  const int column0 = (static_cast<int>(blockIdx.x) - run * column_blocks) * S::kColumns;
  const int first = run * p.tiles_per_block, last = min(first + p.tiles_per_block, p.tile_count);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t weights_shared = smem_u32(shared), low_shared = weights_shared + p.weights * S::weight_bytes(pad);
  uint32_t weight_shared = weights_shared;  // the current tile's
  if (warp == 0) {
    if (lane == 0) {
      mbar_init(&loaded[0], kFillThreads);
      mbar_init(&loaded[1], kFillThreads);
      mbar_init(&ready, 1);
      mbar_init(&drained, S::kWarps);
      mbar_init(&never, 1);
      fence_barrier_init();
      abort = 0;
    }
    __syncwarp();
    tmem_alloc(&tensor_memory, S::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t accumulator = tensor_memory;
  // False for the whole warp once a wait of the block has run out: the warps
  // then leave their loops one after the other and meet at the last barrier.
  auto wait = [&](uint64_t* bar, int index) {
    const uint32_t parity = static_cast<uint32_t>(index) & 1;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, kWaitAdapters, &abort, p.watchdog, p.wait_limit_ns)) != 0;
  };
  auto adapted = [&](const Tile& tile) { return tile.adapter >= 0 && tile.adapter < p.adapters; };
  constexpr Tile kNone{0, 0, -1};

  // Warp 0, one lane: a tile's product, once its operands are there and the
  // last one has been read.
  int issued = 0;
  auto multiply = [&](int product) {
    if (p.expire && product == 0 && !wait(&never, 0)) return;
    if (!wait(&loaded[product & 1], product >> 1) || (product > 0 && !wait(&drained, product - 1))) return;
    fence_proxy_async_smem();  // the copies were made by ordinary writes
    tc_fence_after();
    if (lane == 0) {
      constexpr uint32_t kInstruction = idesc_f16<T>(kWide, S::kColumns, false, TRANS);
      // K-major panels: rows of 8 ranks, groups of 8 rows 128 bytes apart; the weight [rank, width] by columns.
      const uint64_t a = smem_desc(low_shared + (product & 1) * S::low_bytes(pad), S::kLowStep, 128, 0);
      const uint64_t b = TRANS ? smem_desc(weight_shared, 128, pad * 16, 0) : smem_desc(weight_shared, S::kWeightStep, 128, 0);
      constexpr int kStep = (TRANS ? 256 : 2 * S::kWeightStep) / 16;
      for (int plane = 0; plane < 2; ++plane) {
        for (int k = 0; k < pad / 16; ++k) {
          mma_bf16(accumulator, a + (plane * pieces + 2 * k) * (S::kLowStep / 16), b + k * kStep, kInstruction,
                   plane > 0 || k > 0);
        }
      }
      tc_commit(&ready);
    }
    issued = product + 1;
    __syncwarp();
  };
  {
    // Copies by these 256 threads; each arrives once for every product.
    auto load_low = [&](const Tile& tile, int product) {
      const T* from = static_cast<const T*>(p.low) + static_cast<int64_t>(tile.start) * pad;
      const uint32_t to = low_shared + (product & 1) * S::low_bytes(pad);
      const int row = tid & 127, plane = tid >> 7;
      const bool in = row < tile.count;
      const T* source = from + (in ? (plane * p.slots + row) * pad : 0);
      for (int i = 0; i < pieces; ++i) {
        cp_async16(to + (plane * pieces + i) * S::kLowStep + row * 16, source + i * 8, in);
      }
    };
    auto load_weight = [&](int adapter, uint32_t weight_shared) {
      const T* weight = static_cast<const T*>(p.weight) + static_cast<int64_t>(adapter) * p.rank * p.width;
      if constexpr (!TRANS) {
        const int c = tid;  // one column a thread
        const int at = (c & ~31) + c % 8 / 2 * 8 + c / 8 % 4 * 2 + (c & 1);
        for (int i = 0; i < pieces; ++i) {
          const int in = column0 + c < width ? p.rank - i * 8 : 0;
          copy8<T, FAST>(weight_shared + i * S::kWeightStep + at * 16,
                         in > 0 ? weight + static_cast<int64_t>(column0 + c) * p.rank + i * 8 : weight, in);
        }
      } else {
        for (int i = tid; i < pad * (S::kColumns / 8); i += kFillThreads) {
          const int r = i / (S::kColumns / 8), c = i % (S::kColumns / 8) * 8;
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
          // Panels of 8 columns: pair j of these 8 goes to panel j of its 32 columns, at 2 (c / 8 % 4).
          const uint32_t to = weight_shared + (c / 32 * 4) * (pad * 16) + r * 16 + c / 8 % 4 * 4;
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(to + j * (pad * 16)), "r"(words[j]) : "memory");
          }
        }
      }
    };
    int adapter = -1;  // whose weight was loaded last, and to where
    uint32_t newest = weights_shared;
    auto load = [&](const Tile& tile, int product) {
      if (!adapted(tile)) return;
      load_low(tile, product);
      if (tile.adapter == adapter) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&loaded[product & 1])) : "memory");
        return;
      }
      if (p.weights == 2 && adapter >= 0) newest = 2 * weights_shared + S::weight_bytes(pad) - newest;  // the other one
      load_weight(adapter = tile.adapter, newest);
      if constexpr (FAST && !TRANS) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&loaded[product & 1])) : "memory");
      } else {  // written by ordinary stores
        cp_async_commit();
        cp_async_wait<0>();
        mbar_arrive(&loaded[product & 1]);
      }
    };

    // This thread's rows of a tile, two of each half of its warp's 32, and columns.
    const int quarter = warp % 4, row0 = quarter * 32 + (lane >> 2);
    const int column = column0 + warp / 4 * 128 + (lane & 3) * 8, columns_left = width - column;
    auto look = [&](const Tile& tile, int32_t (&token)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        token[i] = row0 + 8 * i < tile.count ? p.rows[tile.start + row0 + 8 * i] : -1;
      }
    };
    // Apart from the look, so that its loads stay under way.
    auto check = [&](int32_t (&token)[4]) {
#pragma unroll
      for (int i = 0; i < 4; ++i) token[i] = static_cast<uint32_t>(token[i]) < static_cast<uint32_t>(p.tokens) ? token[i] : -1;
    };
    auto load_base = [&](int32_t token, int g) {
      Raw8<T> r;
      r.w[0] = make_uint4(0, 0, 0, 0);
      const T* from = static_cast<const T*>(p.base) + static_cast<int64_t>(token) * p.base_stride + column + 32 * g;
      const int limit = p.base != nullptr && token >= 0 ? columns_left - 32 * g : 0;
      if constexpr (FAST) {
        if (limit > 0) r = load8(from);
      } else {
        T* e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j < limit) e[j] = from[j];
        }
      }
      return r;
    };
    Tile tile = p.tiles[first], next = first + 1 < last ? p.tiles[first + 1] : kNone;
    int32_t token[4], next_token[4];
    look(tile, token);
    check(token);
    Raw8<T> part[S::kHalves][S::kGroups][2];
#pragma unroll
    for (int half = 0; half < S::kHalves; ++half) {
#pragma unroll
      for (int g = 0; g < S::kGroups; ++g) {
#pragma unroll
        for (int h = 0; h < 2; ++h) part[half][g][h] = load_base(token[2 * half + h], g);
      }
    }
    load(tile, 0);
    int product = 0;  // of the current tile, if it has one
    for (int t = first; t < last; ++t) {
      const bool mine = adapted(tile);
      const int next_product = product + mine;
      // The next tile's low rows go where those of the product before this
      // one were (it has completed), a new weight where the one before this
      // was; with room for one only it waits for this product.
      weight_shared = newest;
      // Scaled rows: their powers are read with the products they belong to.
      if (kScaled<T> && product > 0 && !wait(&drained, product - 1)) break;
      const bool early = !mine || next.adapter == adapter || p.weights == 2;
      if (early) load(next, next_product);
      look(next, next_token);
      if (mine && warp == 0) multiply(product);
      if (mine && !wait(&ready, product)) break;
      if (kScaled<T> && mine && !wait(&loaded[product & 1], product >> 1)) break;  // long there: for the rows' powers
      if (!early) load(next, next_product);
      check(next_token);
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < S::kHalves; ++half) {
        float back[2] = {1.f, 1.f};
        if (kScaled<T> && mine) {
          const uint32_t at = low_shared + (product & 1) * S::low_bytes(pad) + pieces * S::kLowStep;
#pragma unroll
          for (int h = 0; h < 2; ++h) back[h] = power_of_two(back_of(load_shared4(at + (row0 + 16 * half + 8 * h) * 16)));
        }
#pragma unroll
        for (int g = 0; g < S::kGroups; ++g) {
          uint32_t d[16];
          if (mine) {
            tmem_ld_16x256b_x4(accumulator + (static_cast<uint32_t>(quarter * 32 + half * 16) << 16) + warp / 4 * 128 + g * 32, d);
            tmem_ld_wait();
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[8];
            unpack8(part[half][g][h], v);
            part[half][g][h] = load_base(next_token[2 * half + h], g);
            if (mine) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                v[2 * j] = fmaf(__uint_as_float(d[4 * j + 2 * h]), back[h], v[2 * j]);
                v[2 * j + 1] = fmaf(__uint_as_float(d[4 * j + 2 * h + 1]), back[h], v[2 * j + 1]);
              }
            }
            const int32_t row = token[2 * half + h];
            T* to = static_cast<T*>(p.out) + static_cast<int64_t>(row) * p.out_stride + column + 32 * g;
            const int limit = row >= 0 ? columns_left - 32 * g : 0;
            if constexpr (FAST) {
              if (limit > 0) store8(to, pack8<T>(v));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                if (j < limit) to[j] = from_float<T>(v[j]);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (mine && lane == 0) mbar_arrive(&drained);
      tile = next;
      next = t + 2 < last ? p.tiles[t + 2] : kNone;
      product = next_product;
#pragma unroll
      for (int i = 0; i < 4; ++i) token[i] = next_token[i];
    }
    cp_async_commit();
    cp_async_wait<0>();
  }
  if (abort != 0 && tid == 0 && issued > 0) mbar_drain(&ready, static_cast<uint32_t>(issued - 1) & 1);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0) tmem_dealloc(accumulator, S::kColumns);
  if (abort == 0) return;
  const int columns = min(S::kColumns, width - column0);
  for (int t = first; t < last; ++t) {
    const Tile tile = p.tiles[t];
    for (int i = tid; i < tile.count * columns; i += S::kThreads) {
      const int64_t token = token_of(p, tile.start + i / columns);
      T* row = static_cast<T*>(p.out) + token * p.out_stride + column0;
      if (token >= 0) row[i % columns] = from_float<T>(__int_as_float(0x7fffffff));
    }
  }
}

// ------------------------------------------------------------------- outer ----

// dW[column, r] = sum over the adapter's slots of row[column] * low[r]: D
// [128 columns, 2 RANK] twice in tensor memory, K the slots. The rows are A
// (MN-major: 64 columns are a swizzled row of 128 bytes), both planes of `low`
// side by side are B (in panels), so that A, whose reading takes longer than
// the product, is read once; the planes' sums are added at the end. Each block
// takes about 0.43 us for a stage of 16 KB, with one or two blocks on the SM
// and 4 or 5 stages. 16384 x 3584 bf16, rank 32, 4 adapters: 36 us (3.3 TB/s),
// 41 to 47 behind the product that writes dx, whose rows are still leaving L2;
// fp16 38 and up to 51. Each further 16384 rows of bf16 take 24 (4.9 TB/s).
// Register accumulators took 68. A block takes 256 columns and RANK ranks; the
// blocks of a cluster share the adapter's tokens.
// Scaled rows: the pieces of a row are read and written again by neighbouring
// lanes, so the panels stand 128 bytes / panels further apart, on other banks.
template <int RANK, bool SCALED>
struct OuterShape {
  static constexpr int kThreads = kTensorThreads;
  static constexpr int kColumns = 256;
  static constexpr int kTokens = 32;
  static constexpr int kStages = 4;
  static constexpr int kSubBytes = kTokens * 128;  // 64 columns
  static constexpr int kRowBytes = kColumns / 64 * kSubBytes;
  static constexpr int kPanelBytes = kTokens * 16 + (SCALED ? 128 / (RANK / 8) : 0);
  static constexpr int kPlaneBytes = RANK / 8 * kPanelBytes;
  static constexpr int kStageBytes = (kRowBytes + 2 * kPlaneBytes + 1023) / 1024 * 1024;  // the swizzle goes by address bits
  static constexpr int kTensorColumns = 4 * RANK;
  static constexpr int kPartPitch = RANK + 4;
  static constexpr int kPartBytes = kColumns * kPartPitch * 4 * 3 / 2;  // and a cluster's share, at most half
  static constexpr int kBytes = 1024 + (kStages * kStageBytes > kPartBytes ? kStages * kStageBytes : kPartBytes);
};

template <typename T, int RANK, bool FAST>
__global__ void __launch_bounds__(kTensorThreads, 2) adapter_outer(AdapterParams p) {
  using S = OuterShape<RANK, kScaled<T>>;
  extern __shared__ uint8_t shared_raw[];
  __shared__ TensorRing<S::kStages> ring;
  uint8_t* shared = shared_raw + (-smem_u32(shared_raw) & 1023u);  // the swizzle goes by address bits
  const uint32_t stages = smem_u32(shared);
  uint32_t splits;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(splits));
  const uint32_t split = cluster_ctarank();
  const int64_t column0 = static_cast<int64_t>(blockIdx.x / splits) * S::kColumns;
  const int adapter = blockIdx.y;
  const int rank0 = blockIdx.z * RANK;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 8) ring.start(S::kTensorColumns);
  const int32_t begin = p.group_offsets[adapter], end = p.group_offsets[adapter + 1];
  const int tiles = (end - begin + S::kTokens - 1) / S::kTokens;
  const int per_split = (tiles + static_cast<int>(splits) - 1) / static_cast<int>(splits);
  const int first = min(static_cast<int>(split) * per_split, tiles);
  const int last = min(first + per_split, tiles);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t accumulator = ring.tensor_memory;

  uint32_t back = 127;  // scaled rows: the block's, the same for all filling threads
  if (warp < 8) {
    constexpr int kRowCopies = S::kTokens / 8;  // a warp copies rows warp, warp + 8, ...: whole lines
    static_assert(S::kColumns == 32 * 8, "a lane copies one piece of a row");
    constexpr int kLowPieces = RANK / 8, kLowStep = kFillThreads / kLowPieces;
    constexpr int kLowCopies = (2 * S::kTokens + kLowStep - 1) / kLowStep;
    const int columns_left = static_cast<int>(min(p.width - column0, static_cast<int64_t>(S::kColumns))) - lane * 8;
    const T* x = static_cast<const T*>(p.rows_in) + (columns_left > 0 ? column0 + lane * 8 : 0);
    const uint32_t row_to = stages + lane / 8 * S::kSubBytes + swizzled(warp, lane % 8);
    const int low_piece = tid % kLowPieces, low_row = tid / kLowPieces;
    const bool low_in = rank0 + low_piece * 8 < p.rank_pad;
    const T* low = static_cast<const T*>(p.low) + (low_in ? rank0 + low_piece * 8 : 0);
    const uint32_t low_to = stages + S::kRowBytes;
    const int row_of_low = low_row % S::kTokens;  // of all of a thread's pieces of a tile
    static_assert(kLowStep % S::kTokens == 0, "a thread's pieces are of one row");

    // Tokens of the warp's rows of 8 tiles, one a lane, read 8 tiles ahead.
    auto look = [&](int tile) {
      const int slot = begin + (tile + lane / kRowCopies) * S::kTokens + warp + lane % kRowCopies * 8;
      if (slot >= end) return -1;
      const int32_t token = p.rows[slot];
      return token < p.tokens ? token : -1;
    };
    constexpr int kBatch = 32 / kRowCopies;
    int32_t tokens = look(first), next_tokens = look(first + kBatch);
    auto copy_rows = [&](int fill) {
      const uint32_t stage = static_cast<uint32_t>(fill % S::kStages) * S::kStageBytes;
      if (fill > 0 && fill % kBatch == 0) {
        tokens = next_tokens;
        next_tokens = look(first + fill + kBatch);
      }
#pragma unroll
      for (int i = 0; i < kRowCopies; ++i) {
        const int32_t token = __shfl_sync(0xffffffffu, tokens, fill % kBatch * kRowCopies + i);
        copy8<T, FAST>(row_to + stage + i * 8 * 128, x + static_cast<int64_t>(max(token, 0)) * p.row_stride,
                       token >= 0 ? columns_left : 0);
      }
    };
    auto copy_low = [&](int fill) {
      const uint32_t stage = static_cast<uint32_t>(fill % S::kStages) * S::kStageBytes;
      const int slot = begin + (first + fill) * S::kTokens + row_of_low;
      const bool in = low_in && slot < end;
#pragma unroll
      for (int i = 0; i < kLowCopies; ++i) {
        const int plane = (low_row + i * kLowStep) / S::kTokens;
        if (plane >= 2) continue;
        cp_async16(low_to + stage + plane * S::kPlaneBytes + paneled(row_of_low, low_piece, S::kPanelBytes),
                   low + (in ? (plane * p.slots + slot) * p.rank_pad : 0), in);
      }
    };
    const int fills = last - first;
    if constexpr (!kScaled<T>) {
      for (int fill = 0; fill < fills; ++fill) {
        if (fill >= S::kStages && !ring.wait(ring.used, fill - S::kStages, p)) break;
        copy_rows(fill);
        copy_low(fill);
        ring.filled<FAST>(fill);
      }
    } else {
      // Scaled rows: their planes arrive as they are and each thread brings its
      // own pieces to the block's power, that of its largest row, two fillings
      // later. (Pieces loaded into registers took twice the time: an arrival at a
      // barrier waits for the thread's loads, whichever they are for.)
      constexpr int kAhead = 2;
      for (int fill = 0; fill < kAhead; ++fill) {
        if (fill < fills) copy_rows(fill), copy_low(fill);
        cp_async_commit();
      }
      const T* second = static_cast<const T*>(p.low) + p.slots * p.rank_pad;
      auto power = [&](int slot) {
        return slot < end ? *reinterpret_cast<const uint4*>(second + static_cast<int64_t>(slot) * p.rank_pad) : make_uint4(0, 0, 0, 0);
      };
      // Powers of the rows that the warp's pieces are of, for 8 tiles, one or more
      // a lane, read 8 tiles ahead.
      constexpr int kWarpRows = 32 / kLowPieces, kPowers = 8 / kLowPieces;
      auto powers_of = [&](int fill, uint4 (&to)[kPowers]) {
#pragma unroll
        for (int i = 0; i < kPowers; ++i) {
          const int tile = first + fill + i * kLowPieces + lane / kWarpRows;
          const int row = (warp * kWarpRows + lane % kWarpRows) % S::kTokens;
          to[i] = tile < last ? power(begin + tile * S::kTokens + row) : make_uint4(0, 0, 0, 0);
        }
      };
      uint4 next_powers[kPowers];
      uint32_t powers[kPowers];
      powers_of(0, next_powers);
      __shared__ uint32_t warps[kFillThreads / 32];
      uint32_t most = 1;
#pragma unroll 4
      for (int slot = begin + first * S::kTokens + tid; slot < begin + last * S::kTokens; slot += kFillThreads) {
        most = max(most, back_of(power(slot)));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      if (lane == 0) warps[warp] = most;
      named_barrier(1, kFillThreads);
      back = __reduce_max_sync(0xffffffffu, warps[lane % (kFillThreads / 32)]);

      for (int fill = 0; fill < fills; ++fill) {
        const int ahead = fill + kAhead;
        if (ahead < fills) {
          if (ahead >= S::kStages && !ring.wait(ring.used, ahead - S::kStages, p)) break;
          copy_rows(ahead);
          copy_low(ahead);
        }
        cp_async_commit();
        if (fill % 8 == 0) {
#pragma unroll
          for (int i = 0; i < kPowers; ++i) powers[i] = back_of(next_powers[i]);
          powers_of(fill + 8, next_powers);
        }
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kPowers; ++i) {
          const uint32_t other = __shfl_sync(0xffffffffu, powers[i], fill % kLowPieces * kWarpRows + lane / kLowPieces);
          if (fill % 8 / kLowPieces == i) mine = other;
        }
        const float scale = power_of_two(static_cast<uint32_t>(max(127 + static_cast<int>(mine) - static_cast<int>(back), 0)));
        const uint32_t stage = static_cast<uint32_t>(fill % S::kStages) * S::kStageBytes;
        cp_async_wait<kAhead>();
#pragma unroll
        for (int i = 0; i < kLowCopies; ++i) {
          const int plane = (low_row + i * kLowStep) / S::kTokens;
          if (plane >= 2) continue;
          const uint32_t at = low_to + stage + plane * S::kPlaneBytes + paneled(row_of_low, low_piece, S::kPanelBytes);
          Raw8<T> raw;
          raw.w[0] = load_shared4(at);
          float v[8];
          unpack8(raw, v);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] *= scale;
          const uint4 w = pack8<T>(v).w[0];
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
        }
        mbar_arrive(&ring.full[fill % S::kStages]);
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
  } else {
    constexpr uint32_t kInstruction = idesc_f16<T>(128, 2 * RANK, true, true);
    // Groups of 8 slots are 1024 bytes apart, runs of 64 columns kSubBytes.
    const uint64_t a = smem_desc(stages, S::kSubBytes, 1024, 2);
    const uint64_t b = smem_desc(stages + S::kRowBytes, 128, S::kPanelBytes, 0);
    ring.multiply(last - first, p, [&](int fill) {
      // Addresses advance in the descriptors' units of 16 bytes.
      const uint64_t stage = static_cast<uint64_t>(fill % S::kStages) * (S::kStageBytes / 16);
#pragma unroll
      for (int k = 0; k < S::kTokens / 16; ++k) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          mma_bf16(accumulator + half * 2 * RANK, a + stage + half * (2 * S::kSubBytes / 16) + k * 128, b + stage + k * 16,
                   kInstruction, fill > 0 || k > 0);
        }
      }
    });
  }
  float* part = reinterpret_cast<float*>(shared);
  if (first < last) ring.wait(ring.used, last - 1 - first, p);
  tc_fence_after();
  __syncthreads();
  if (warp < 8) {
    const int half = warp / 4, c = half * 128 + warp % 4 * 32 + lane;
    store_part<RANK, 2>(part + c * S::kPartPitch, accumulator + (static_cast<uint32_t>(warp % 4) << 21) + half * 2 * RANK,
                        first < last && !ring.gave_up(), ring.instead(), power_of_two(back));
  }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(accumulator, S::kTensorColumns);
  // Each block adds up its share of the columns, beside its own sums (which
  // the others may still be reading), then writes it in memory order.
  const int share = (S::kColumns + static_cast<int>(splits) - 1) / static_cast<int>(splits);
  const int c_first = static_cast<int>(split) * share, c_count = max(0, min(share, S::kColumns - c_first));
  float* mine = part;
  if (splits > 1) {
    mine = part + S::kColumns * S::kPartPitch;
    constexpr int kQuads = RANK / 4;
    for (int e = tid; e < c_count * kQuads; e += S::kThreads) {
      const int c = e / kQuads, q = e % kQuads * 4;
      *reinterpret_cast<float4*>(mine + c * S::kPartPitch + q) = sum_cluster(part, (c_first + c) * S::kPartPitch + q, splits);
    }
    cluster_sync();
  }
  T* out = static_cast<T*>(p.out) + static_cast<int64_t>(adapter) * p.rank * p.width;
  const bool columns_fast = p.out_stride == 1;
  for (int e = tid; e < c_count * RANK; e += S::kThreads) {
    const int c = columns_fast ? e % c_count : e / RANK;
    const int r = columns_fast ? e / c_count : e % RANK;
    const int64_t column = column0 + c_first + c;
    if (column >= p.width || rank0 + r >= p.rank) continue;
    out[column * p.out_stride + (rank0 + r) * p.out_rank_stride] = from_float<T>(mine[c * S::kPartPitch + r]);
  }
}

// -------------------------------------------------------------------- host ----

template <typename Kernel>
int launch_clustered(Kernel kernel, const AdapterParams& p, dim3 grid, int threads, int cluster, int shared,
                     bool dependent, cudaStream_t stream) {
  const int rc = allow_shared(reinterpret_cast<const void*>(kernel), shared);
  if (rc != SDC_OK) return rc;
  if (cluster > kPortableSplit) SDC_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
  // Slots are looked up ahead in 32 bits, up to 576 of them.
  SDC_REQUIRE(tokens >= 0 && tokens <= INT_MAX - 1024, "low-rank adapters take fewer than 2^31 - 1024 tokens");
  SDC_REQUIRE(width > 0 && width < INT_MAX - 512, "low-rank adapter widths must be positive and fit padded int32 extents");
  SDC_REQUIRE(rank >= 1 && rank <= kMaxRank, "low-rank adapters take ranks of 1 to 256");
  SDC_REQUIRE(adapters >= 1 && adapters <= 65535, "low-rank adapters take 1 to 65535 adapters");
  return SDC_OK;
}

int set_watchdog(AdapterParams& p) {
  p.watchdog = watchdog_ptr();
  if (p.watchdog == nullptr) return fail(SDC_ERR_CUDA, "low-rank adapters have no watchdog word on this device");
  const WatchdogSettings watch = watchdog_settings();
  p.wait_limit_ns = watch.wait_limit_ns;
  p.expire = watch.pace_extra > 0;
  return SDC_OK;
}

int pad_rank(int rank) { return (rank + 15) / 16 * 16; }
int rank_tile(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : 64; }

bool vector_rows(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

// Stands in for the kernels of clusters where the runtime is asked how many run
// at once: of kernels that allocate tensor memory it assumes one block an SM. It
// is never launched.
__global__ void __launch_bounds__(kTensorThreads, 2) cluster_probe(AdapterParams) {}

int ask_clusters(int size, int shared) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(size));
  config.blockDim = dim3(kTensorThreads);
  config.dynamicSmemBytes = static_cast<size_t>(shared);
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = static_cast<unsigned>(size);
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (allow_shared(reinterpret_cast<const void*>(cluster_probe), shared) != SDC_OK ||
      (size > kPortableSplit &&
       cudaFuncSetAttribute(cluster_probe, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) ||
      cudaOccupancyMaxActiveClusters(&clusters, cluster_probe, &config) != cudaSuccess) {
    cudaGetLastError();  // no cluster of that size here, and no error of the call's
    return 0;
  }
  return clusters;
}

// Clusters of `size` blocks that run at once when an SM holds two blocks (100 KB
// of shared memory), 0 where the device has none. Those beyond the portable size
// must also fit with one block an SM. Asked of the runtime once for each device
// and size. B200 with 148 SMs: 296, 148, 93, 71, 56, 45, 37, 33, 30, 26, 21, 21,
// 17, 14, 14 and 14 of 1 to 16 blocks.
int cluster_room(int size) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxSplit + 1] = {};  // 0: not asked yet, else 1 more
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kDevices) return 0;
  int room = known[device][size].load(std::memory_order_relaxed) - 1;
  if (room < 0) {
    room = size <= kPortableSplit || ask_clusters(size, 150 * 1024) > 0 ? ask_clusters(size, 100 * 1024) : 0;
    known[device][size].store(room + 1, std::memory_order_relaxed);
  }
  return room;
}

// Blocks that share a tile's sum: as many as fill the SMs' `resident` blocks
// each once, as long as each keeps two chunks (four of more than eight blocks),
// and no more than let all clusters run at once: a few that waited for a second
// turn would double the time. Outer products of 16384 rows and one adapter:
// 3584 columns, rank 32, in 14 clusters of 16 blocks 29 us, of 8 35; 1024
// columns, rank 16, 21 and 33. 37 tiles of shrink (3584 columns, rank 32) in
// clusters of 7 take 14 us, of 8 19; 42 clusters of outer products are the other
// way round, 6 blocks 36 us and 7 33.
int split_count(int64_t clusters, int64_t chunks, int resident, int most) {
  const int64_t wanted = std::min<int64_t>(static_cast<int64_t>(resident) * sm_count() / std::max<int64_t>(clusters, 1), chunks / 2);
  int split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(wanted, most)));
  if (split > kPortableSplit && chunks / split < 4) split = kPortableSplit;
  while (split > 1 && clusters > static_cast<int64_t>(cluster_room(split)) * resident / 2) --split;
  return split;
}

template <typename T, int ROWS, int RANK, bool TRANS>
int launch_shrink(AdapterParams p, int64_t tiles, cudaStream_t stream) {
  using S = std::conditional_t<ROWS == kWide, WideShape<RANK, TRANS>, NarrowShape<RANK, TRANS>>;
  const int64_t chunks = ceil_div(p.width, S::kChunk);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int split = split_count(tiles * rank_blocks, chunks, ROWS == kWide ? 2 : 4, kPortableSplit);
  p.chunks_per_split = static_cast<int>(ceil_div(chunks, split));
  const dim3 grid(static_cast<unsigned>(tiles * split), rank_blocks);
  const bool fast = p.vector_rows && p.vector_weight && p.width % 8 == 0 && (!TRANS || p.rank % 8 == 0);
  auto launch = [&](auto kernel) { return launch_clustered(kernel, p, grid, S::kThreads, split, S::kBytes, false, stream); };
  int rc;
  if constexpr (ROWS == kWide) {
    rc = fast ? launch(adapter_shrink_wide<T, RANK, TRANS, true>) : launch(adapter_shrink_wide<T, RANK, TRANS, false>);
  } else {
    rc = fast ? launch(adapter_shrink<T, RANK, TRANS, true>) : launch(adapter_shrink<T, RANK, TRANS, false>);
  }
  if constexpr (kScaled<T>) {
    if (rc != SDC_OK || rank_blocks == 1) return rc;
    adapter_split<T><<<static_cast<unsigned>(tiles), 256, 0, stream>>>(p);
    SDC_CUDA_CHECK(cudaGetLastError());
  }
  return rc;
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

bool expand_fast(const AdapterParams& p, bool trans) {
  return p.vector_rows && p.vector_out && p.vector_weight && p.width % 8 == 0 && (trans || p.rank % 8 == 0);
}

template <typename T, bool TRANS>
int launch_expand_narrow(AdapterParams p, int64_t tiles, bool dependent, cudaStream_t stream) {
  using S = NarrowExpand;
  const int64_t blocks = ceil_div(p.width, S::kColumns) * tiles;
  SDC_REQUIRE(blocks <= INT_MAX, "low-rank adapters have too many tiles for one launch");
  while ((8 << p.piece_bits) < p.rank_pad) ++p.piece_bits;
  auto launch = [&](auto kernel) {
    return launch_clustered(kernel, p, dim3(static_cast<unsigned>(blocks)), S::kThreads, 0, S::bytes(p.rank_pad, TRANS),
                            dependent, stream);
  };
  if (!expand_fast(p, TRANS)) return launch(adapter_expand<T, TRANS, false, 0>);
  switch (p.rank_pad) {
    case 16: return launch(adapter_expand<T, TRANS, true, 16>);
    case 32: return launch(adapter_expand<T, TRANS, true, 32>);
    case 64: return launch(adapter_expand<T, TRANS, true, 64>);
    default: return launch(adapter_expand<T, TRANS, true, 0>);
  }
}

template <typename T, bool TRANS>
int launch_expand_wide(AdapterParams p, int64_t tiles, cudaStream_t stream) {
  const int64_t column_blocks = ceil_div(p.width, ExpandWide::kColumns);
  // Runs of tiles that fill the SMs' two blocks once.
  const int64_t runs = std::max<int64_t>(1, 2 * sm_count() / column_blocks);
  p.tile_count = static_cast<int>(tiles);
  p.tiles_per_block = static_cast<int>(ceil_div(tiles, runs));
  const int64_t blocks = column_blocks * ceil_div(tiles, p.tiles_per_block);
  SDC_REQUIRE(blocks <= INT_MAX, "low-rank adapters have too many tiles for one launch");
  // Two buffers of weights where two blocks of an SM have the room (ranks up to 48).
  p.weights = ExpandWide::bytes(p.rank_pad, 2) <= ExpandWide::kBlockBytes ? 2 : 1;
  auto launch = [&](auto kernel) {
    return launch_clustered(kernel, p, dim3(static_cast<unsigned>(blocks)), ExpandWide::kThreads, 0,
                            ExpandWide::bytes(p.rank_pad, p.weights), false, stream);
  };
  return expand_fast(p, TRANS) ? launch(adapter_expand_wide<T, TRANS, true>) : launch(adapter_expand_wide<T, TRANS, false>);
}

template <typename T>
int expand_typed(const AdapterParams& p, int tile_rows, bool trans, int64_t tiles, bool dependent, cudaStream_t stream) {
  if (tile_rows == kWide) return trans ? launch_expand_wide<T, true>(p, tiles, stream) : launch_expand_wide<T, false>(p, tiles, stream);
  return trans ? launch_expand_narrow<T, true>(p, tiles, dependent, stream)
               : launch_expand_narrow<T, false>(p, tiles, dependent, stream);
}

template <typename T, int RANK>
int launch_outer(const AdapterParams& p, cudaStream_t stream) {
  using S = OuterShape<RANK, kScaled<T>>;
  const int64_t columns = ceil_div(p.width, S::kColumns);
  const unsigned rank_blocks = static_cast<unsigned>(ceil_div(p.rank, RANK));
  const int64_t tiles = ceil_div(ceil_div(p.slots, p.adapters), S::kTokens);
  const int split = split_count(columns * p.adapters * rank_blocks, tiles, 2, kMaxSplit);
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
  SDC_REQUIRE(tile_count >= 0 && tile_count <= INT_MAX / kPortableSplit, "low-rank adapters have too many tiles for one launch");
  if (tile_count == 0) return SDC_OK;
  SDC_REQUIRE(x != nullptr && rows != nullptr && tiles != nullptr && weight != nullptr && low != nullptr && aligned16(low),
              "low-rank adapter pointers must not be null and the low-rank rows must be 16-byte aligned");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  AdapterParams p{};
  rc = set_watchdog(p);
  if (rc != SDC_OK) return rc;
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
  rc = set_watchdog(p);
  if (rc != SDC_OK) return rc;
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
  rc = set_watchdog(p);
  if (rc != SDC_OK) return rc;
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
