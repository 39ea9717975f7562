// Norm of each query and key head with the rotation by position in one pass,
// forward and backward.
//
//   forward   r = rsqrt(mean_d x^2 + eps),  u = x r,  y = Rot(w u)
//   backward  g = Rot^T dy,  dx = r (g w - u mean_d(g w u)),  dw = sum g u
//
// Rot turns pair p < rotary/2 of a head by the position's angle p: elements
// (p, p + rotary/2), or (2p, 2p+1) when interleaved; elements from `rotary`
// on pass, each by itself. Without weights the heads are only turned.
//
// Both directions move bytes and little else (about 10 flops an element), so
// the layout serves the loads: a thread owns 8 pairs of a head, both members
// of each, so the rotation needs no exchange between threads; in the common
// forms its 16 elements are two (16-bit types) or four (fp32) 16-byte words.
// dim/16 neighbouring lanes share a head and exchange only the sum of squares
// (and, backward, of products). A group of lanes keeps a few heads and walks
// the tokens in steps of all groups, so weights are read once and angles once
// for its heads; the heads of the tokens to come are copied to shared memory
// meanwhile, each thread its own words, so that no barrier is needed and loads
// never stop.
#include <algorithm>
#include <climits>
#include <cmath>

#include "mma.cuh"

namespace sdc {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryBlocks = 2;  // on an SM
// Tokens of a group under way, by the 16-byte words that a thread copies of
// one: two blocks share an SM's shared memory.
constexpr int stages_for(int words) { return words >= 8 ? 3 : words >= 4 ? 5 : 8; }
constexpr int kMaxHeadDim = 512;  // 32 lanes of 16 elements

struct RotaryParams {
  const void* x[2];      // q, k
  const void* dy[2];     // backward only
  void* y[2];            // outputs, contiguous [batch, sequence, heads, dim]
  const void* weight[2]; // null: no norm
  int64_t xs[2][3];      // strides of batch, sequence, head in elements
  int64_t dys[2][3];
  int64_t position_strides[2];
  const void* positions;
  const float* table;
  int64_t table_rows;
  uint32_t sequence;     // tokens per batch entry
  uint32_t tokens;
  uint32_t chunks;       // head chunks per token: q's, then k's
  uint32_t q_chunks;
  int heads[2];
  int group_heads;       // heads of a group
  int dim, rotary;
  float eps, inv_dim;
  bool positions_64, weight_f32, vector_table, vector_weight;
  float* partials;       // backward: [blocks][2][dim]
};

__device__ __forceinline__ int64_t load_position(const RotaryParams& p, uint32_t token) {
  const int64_t batch = token / p.sequence, seq = token - static_cast<uint32_t>(batch) * p.sequence;
  const int64_t at = batch * p.position_strides[0] + seq * p.position_strides[1];
  return p.positions_64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
}

template <bool INTERLEAVED>
__device__ __forceinline__ int element_of(int pair, int member, int rotary) {
  if (!INTERLEAVED && pair < rotary / 2) return pair + member * (rotary / 2);
  return 2 * pair + member;  // passing elements pair up in order as well
}

// v[i], v[8 + i]: members of this lane's pair i. VECTOR: the 8 pairs are two
// runs of 8 elements, and neighbouring lanes' runs are neighbours: half-split
// rotary pairs have their first members in one and their second in the other;
// interleaved or passing pairs lie within a run, the lanes' first runs in the
// first half of their part of the head, their second runs in the other.
template <typename T, bool INTERLEAVED, bool VECTOR>
struct HeadIO {
  static constexpr bool kTogether = VECTOR && !INTERLEAVED;  // a lane's pairs turn (split) or pass together
  int first_pair, rotary, pairs, low_run, high_run;
  bool active, split;

  __device__ __forceinline__ HeadIO(const RotaryParams& p, int lane)
      : first_pair(lane * 8), rotary(p.rotary), pairs(p.dim / 2), active(lane * 8 < p.dim / 2),
        split(!INTERLEAVED && lane * 8 < p.rotary / 2) {
    const int part = INTERLEAVED ? 0 : p.rotary;  // where interleaved or passing pairs begin
    low_run = split ? first_pair : part + first_pair - part / 2;
    high_run = split ? first_pair + rotary / 2 : low_run + (p.dim - part) / 2;
  }
  __device__ __forceinline__ int element(int i, int member) const {
    if (!VECTOR) return element_of<INTERLEAVED>(first_pair + i, member, rotary);
    if (split) return (member ? high_run : low_run) + i;
    return (i < 4 ? low_run + 2 * i : high_run + 2 * (i - 4)) + member;
  }
  // Index of pair i's angle (rotary / 2 or more: none, the pair passes).
  __device__ __forceinline__ int angle(int i) const {
    if (!VECTOR || !INTERLEAVED) return first_pair + i;
    return element(i, 0) / 2;
  }

  struct Raw {
    Raw8<T> a, b;
  };
  __device__ __forceinline__ Raw load(const T* head) const {
    Raw r;
    if constexpr (VECTOR) {
      r.a = load8(head + low_run);
      r.b = load8(head + high_run);
    } else {
      T* a = reinterpret_cast<T*>(&r.a);
      T* b = reinterpret_cast<T*>(&r.b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = first_pair + i;
        const bool in = pair < pairs;
        a[i] = in ? head[element_of<INTERLEAVED>(pair, 0, rotary)] : from_float<T>(0.f);
        b[i] = in ? head[element_of<INTERLEAVED>(pair, 1, rotary)] : from_float<T>(0.f);
      }
    }
    return r;
  }
  // The same through this thread's own words of shared memory: words `at`,
  // `at` + kRotaryThreads, ... of 16 bytes.
  static constexpr int kWords = 2 * static_cast<int>(sizeof(Raw8<T>)) / 16;
  __device__ __forceinline__ void issue(const T* head, uint32_t at) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      const T* run = head + (i < kWords / 2 ? low_run : high_run);
      cp_async16(at + i * kRotaryThreads * 16, reinterpret_cast<const uint4*>(run) + i % (kWords / 2));
    }
  }
  __device__ __forceinline__ Raw fetch(uint32_t at) const {
    Raw r;
    uint4* words[2] = {r.a.w, r.b.w};
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      uint4& w = words[i / (kWords / 2)][i % (kWords / 2)];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                   : "r"(at + i * kRotaryThreads * 16));
    }
    return r;
  }
  __device__ __forceinline__ void unpack(const Raw& r, float* v) const { unpack_runs<T>(r.a, r.b, v); }
  template <typename E>
  __device__ __forceinline__ void unpack_runs(const Raw8<E>& ra, const Raw8<E>& rb, float* v) const {
    float a[8], b[8];
    unpack8(ra, a);
    unpack8(rb, b);
    const bool runs = !split;  // even elements are the first members
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (VECTOR) {
        const float e0 = i < 4 ? a[(2 * i) & 7] : b[(2 * i) & 7];
        const float e1 = i < 4 ? a[(2 * i + 1) & 7] : b[(2 * i + 1) & 7];
        v[i] = runs ? e0 : a[i];
        v[8 + i] = runs ? e1 : b[i];
      } else {
        v[i] = a[i];
        v[8 + i] = b[i];
      }
    }
  }
  // Pairs that pass together come from `passed`.
  __device__ __forceinline__ void store(T* head, const float* v, const float* passed) const {
    if constexpr (VECTOR) {
      float a[8], b[8];
      const float* r = kTogether ? passed : v;  // runs
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool runs = !split;
        a[2 * i] = runs ? r[i] : v[2 * i];
        a[2 * i + 1] = runs ? r[8 + i] : v[2 * i + 1];
        b[2 * i] = runs ? r[4 + i] : v[8 + 2 * i];
        b[2 * i + 1] = runs ? r[12 + i] : v[8 + 2 * i + 1];
      }
      store8(head + low_run, pack8<T>(a));
      store8(head + high_run, pack8<T>(b));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int pair = first_pair + i;
        if (pair >= pairs) continue;
        head[element_of<INTERLEAVED>(pair, 0, rotary)] = from_float<T>(v[i]);
        head[element_of<INTERLEAVED>(pair, 1, rotary)] = from_float<T>(v[8 + i]);
      }
    }
  }
  // The weights of this lane's elements, in the order of unpack().
  __device__ __forceinline__ void weights(const void* weight, bool f32, bool vector, float* w) const {
    if (VECTOR && vector) {
      if (f32) {
        const float* from = static_cast<const float*>(weight);
        unpack_runs<float>(load8(from + low_run), load8(from + high_run), w);
      } else {
        unpack(load(static_cast<const T*>(weight)), w);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int member = 0; member < 2; ++member) {
        const int e = element(i, member);
        float value = 0.f;
        if (first_pair + i < pairs) {
          value = f32 ? static_cast<const float*>(weight)[e] : to_float(static_cast<const T*>(weight)[e]);
        }
        w[8 * member + i] = value;
      }
    }
  }
};

// The position's cosine and sine for this lane's 8 pairs; beyond the rotary
// pairs 1 and -0 (an angle of 0 whose sign marks a pair that passes). A
// position outside the table gives NaN, not a stray read.
constexpr uint32_t kPasses = 0x80000000u;
struct Angles {
  float cosine[8], sine[8];
};
template <typename IO>
__device__ __forceinline__ void load_angles(const RotaryParams& p, int64_t position, const IO& io, Angles& a) {
  const int half = p.rotary / 2;
  const bool inside = position >= 0 && position < p.table_rows;
  const float* row = p.table + (inside ? position : 0) * p.rotary;
  const float nan = __int_as_float(0x7fffffff);
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int first = io.angle(4 * part);
    if (inside && p.vector_table && first + 4 <= half) {
      const float4 c = *reinterpret_cast<const float4*>(row + first);
      const float4 s = *reinterpret_cast<const float4*>(row + half + first);
      a.cosine[4 * part] = c.x, a.cosine[4 * part + 1] = c.y, a.cosine[4 * part + 2] = c.z, a.cosine[4 * part + 3] = c.w;
      a.sine[4 * part] = s.x, a.sine[4 * part + 1] = s.y, a.sine[4 * part + 2] = s.z, a.sine[4 * part + 3] = s.w;
      continue;
    }
#pragma unroll
    for (int i = 4 * part; i < 4 * part + 4; ++i) {
      const int pair = io.angle(i);
      const bool turned = pair < half;
      a.cosine[i] = turned ? (inside ? row[pair] : nan) : 1.f;
      a.sine[i] = turned ? (inside ? row[half + pair] : nan) : __uint_as_float(kPasses);
    }
  }
}

// Turns the lane's pairs by their angles, or (BACK) by their opposites. Pairs
// that pass are kept apart: a product with a sine of 0 would carry an infinity
// or a NaN of one element over to the other. Where a lane's pairs pass together
// the caller keeps v instead.
template <bool BACK, typename IO>
__device__ __forceinline__ void turn(const IO& io, const Angles& a, const float* v, float* out) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool passes = !IO::kTogether && __float_as_uint(a.sine[i]) == kPasses;
    const float sine = BACK ? -a.sine[i] : a.sine[i];
    const float x = v[i], y = v[8 + i];
    out[i] = x * a.cosine[i] - (passes ? 0.f : y) * sine;
    out[8 + i] = y * a.cosine[i] + (passes ? 0.f : x) * sine;
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int step = LANES / 2; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
  return x;
}

// What a group of lanes works on: one chunk of heads of every walkers-th token.
// All lanes of a warp run the same number of rounds (their sums are exchanged
// by the whole warp); lanes without work there are not `live`.
template <typename T, int LANES, bool INTERLEAVED, bool VECTOR, int HEADS, int TENSORS>
struct Walk {
  using IO = HeadIO<T, INTERLEAVED, VECTOR>;
  static constexpr int kGroups = kRotaryThreads / LANES;
  static constexpr int kStages = stages_for(TENSORS * HEADS * IO::kWords);
  static constexpr int kStageBytes = TENSORS * HEADS * IO::kWords * kRotaryThreads * 16;
  const RotaryParams& p;
  const IO io;
  uint32_t walkers, walker, shared;
  int role, head0, heads;
  bool working;

  __device__ __forceinline__ Walk(const RotaryParams& params, uint32_t shared_base)
      : p(params), io(params, threadIdx.x % LANES), shared(shared_base + threadIdx.x * 16) {
    const uint32_t group = blockIdx.x * kGroups + threadIdx.x / LANES;
    walkers = gridDim.x * kGroups / p.chunks;
    walker = group / p.chunks;
    const uint32_t chunk = group - walker * p.chunks;
    role = chunk >= p.q_chunks;
    head0 = static_cast<int>(chunk - (role ? p.q_chunks : 0)) * HEADS;
    heads = min(HEADS, p.heads[role] - head0);
    working = walker < walkers && io.active;
  }
  __device__ __forceinline__ uint32_t rounds() const { return (p.tokens + walkers - 1) / walkers; }
  __device__ __forceinline__ uint32_t token(uint32_t round) const { return round * walkers + walker; }
  __device__ __forceinline__ bool live(uint32_t round) const { return working && token(round) < p.tokens; }
  __device__ __forceinline__ const T* head_at(const void* base, const int64_t* strides, uint32_t token, int h) const {
    const uint32_t batch = token / p.sequence, seq = token - batch * p.sequence;
    return static_cast<const T*>(base) + batch * strides[0] + seq * strides[1] + (head0 + h) * strides[2];
  }
  __device__ __forceinline__ uint32_t slot(uint32_t round, int tensor, int h) const {
    return shared + round % kStages * kStageBytes + (tensor * HEADS + h) * IO::kWords * kRotaryThreads * 16;
  }
  // Starts the copies of a round's heads (tensor 0: x, 1: dy).
  __device__ __forceinline__ void issue(uint32_t round, int tensor, const void* base, const int64_t* strides) const {
    if (!VECTOR || !live(round)) return;
    const T* first = head_at(base, strides, token(round), 0);
#pragma unroll
    for (int h = 0; h < HEADS; ++h) {
      if (h < heads) io.issue(first + h * strides[2], slot(round, tensor, h));
    }
  }
  __device__ __forceinline__ typename IO::Raw head(uint32_t round, int tensor, const void* base, const int64_t* strides,
                                                   int h) const {
    if constexpr (VECTOR) return io.fetch(slot(round, tensor, h));
    else return io.load(head_at(base, strides, token(round), h));
  }
};

// Bound by memory: 16384 tokens of 28 + 4 heads of 128 bf16 take 44 us (268 MB,
// 6.1 TB/s), without the norm 40; of 14 + 2 heads of 64 16.2 us (67 MB, half of
// it still in L2 when the launch ends); 8192 of 28 + 4 of 128 fp32 60 us (268 MB,
// 4.5 TB/s: groups of two heads have half the copies under way). One token takes
// 3.7 us, a launch.
template <typename T, int LANES, bool INTERLEAVED, bool VECTOR, int kHeads>
__global__ void __launch_bounds__(kRotaryThreads, kRotaryBlocks) rotary_forward(RotaryParams p) {
  extern __shared__ uint4 copies[];
  using W = Walk<T, LANES, INTERLEAVED, VECTOR, kHeads, 1>;
  constexpr int kStages = W::kStages;
  const W walk(p, smem_u32(copies));
  const int role = walk.role;
  const uint32_t rounds = walk.rounds();
#pragma unroll
  for (uint32_t round = 0; round < kStages - 1; ++round) {
    walk.issue(round, 0, p.x[role], p.xs[role]);
    cp_async_commit();
  }
  // Angles one round ahead, positions two.
  Angles angles, next_angles;
  int64_t position = 0;
  if (walk.live(0)) load_angles(p, load_position(p, walk.token(0)), walk.io, next_angles);
  if (walk.live(1)) position = load_position(p, walk.token(1));
  float w[16];
  const bool norm = p.weight[role] != nullptr;
  if (norm && walk.working) walk.io.weights(p.weight[role], p.weight_f32, p.vector_weight, w);

  for (uint32_t round = 0; round < rounds; ++round) {
    walk.issue(round + kStages - 1, 0, p.x[role], p.xs[role]);
    cp_async_commit();
    angles = next_angles;
    if (walk.live(round + 1)) load_angles(p, position, walk.io, next_angles);
    if (walk.live(round + 2)) position = load_position(p, walk.token(round + 2));
    cp_async_wait<kStages - 1>();
    const bool live = walk.live(round);
    T* y = static_cast<T*>(p.y[role]) + (static_cast<int64_t>(walk.token(round)) * p.heads[role] + walk.head0) * p.dim;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const bool mine = live && h < walk.heads;
      float v[16];
      if (mine) walk.io.unpack(walk.head(round, 0, p.x[role], p.xs[role], h), v);
      if (norm) {
        float squares = 0.f;
        if (mine) {
#pragma unroll
          for (int i = 0; i < 16; ++i) squares = fmaf(v[i], v[i], squares);
        }
        const float r = rsqrtf(group_sum<LANES>(squares) * p.inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = v[i] * r * w[i];
      }
      if (!mine) continue;
      float out[16];
      turn<false>(walk.io, angles, v, out);
      walk.io.store(y + h * p.dim, out, v);
    }
  }
}

// As the forward pass, over x and dy; a thread's 16 weight gradients stay in
// registers for the whole launch, the block adds its groups' sums in a fixed
// order and writes one partial per role. 16384 tokens of 28 + 4 heads of 128
// bf16 take 87 us (403 MB, 4.6 TB/s), of 14 + 2 heads of 64 26.6 us (101 MB,
// 3.8 TB/s), 8192 of 28 + 4 of 128 fp32 108 us (3.7 TB/s): half the issue slots
// at two blocks an SM, whose 128 registers a thread (x, dy, weights and their
// gradients) leave no room for a third. Without the norm 49 us (268 MB, 5.5 TB/s).
template <typename T, int LANES, bool INTERLEAVED, bool VECTOR, int kHeads>
__global__ void __launch_bounds__(kRotaryThreads, kRotaryBlocks) rotary_backward(RotaryParams p) {
  extern __shared__ uint4 copies[];
  using W = Walk<T, LANES, INTERLEAVED, VECTOR, kHeads, 2>;
  constexpr int kStages = W::kStages;
  const W walk(p, smem_u32(copies));
  const int role = walk.role;
  const bool norm = p.weight[role] != nullptr;
  const uint32_t rounds = walk.rounds();
  auto issue = [&](uint32_t round) {
    walk.issue(round, 1, p.dy[role], p.dys[role]);
    if (norm) walk.issue(round, 0, p.x[role], p.xs[role]);
    cp_async_commit();
  };
#pragma unroll
  for (uint32_t round = 0; round < kStages - 1; ++round) issue(round);
  Angles angles, next_angles;
  int64_t position = 0;
  if (walk.live(0)) load_angles(p, load_position(p, walk.token(0)), walk.io, next_angles);
  if (walk.live(1)) position = load_position(p, walk.token(1));
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f, w[i] = 1.f;
  if (norm && walk.working) walk.io.weights(p.weight[role], p.weight_f32, p.vector_weight, w);

  for (uint32_t round = 0; round < rounds; ++round) {
    issue(round + kStages - 1);
    angles = next_angles;
    if (walk.live(round + 1)) load_angles(p, position, walk.io, next_angles);
    if (walk.live(round + 2)) position = load_position(p, walk.token(round + 2));
    cp_async_wait<kStages - 1>();
    const bool live = walk.live(round);
    T* dx = static_cast<T*>(p.y[role]) + (static_cast<int64_t>(walk.token(round)) * p.heads[role] + walk.head0) * p.dim;
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      const bool mine = live && h < walk.heads;
      float v[16], g[16];
      if (mine) {
        walk.io.unpack(walk.head(round, 1, p.dy[role], p.dys[role], h), g);
        if (!W::IO::kTogether || walk.io.split) turn<true>(walk.io, angles, g, g);
      }
      if (norm) {
        float squares = 0.f, products = 0.f;
        if (mine) {
          walk.io.unpack(walk.head(round, 0, p.x[role], p.xs[role], h), v);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            squares = fmaf(v[i], v[i], squares);
            products = fmaf(g[i] * w[i], v[i], products);
          }
        }
        const float r = rsqrtf(group_sum<LANES>(squares) * p.inv_dim + p.eps);
        const float mean = group_sum<LANES>(products) * r * p.inv_dim;
        if (mine) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float u = v[i] * r;
            dw[i] = fmaf(g[i], u, dw[i]);
            g[i] = r * (g[i] * w[i] - u * mean);
          }
        }
      }
      if (mine) walk.io.store(dx + h * p.dim, g, g);
    }
  }
  if (p.partials == nullptr) return;

  // sums[group][element] (the copies are all used: their place is free).
  constexpr int kGroups = W::kGroups;
  float* sums = reinterpret_cast<float*>(copies);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (walk.io.active && walk.io.first_pair + i % 8 < walk.io.pairs) {
      sums[threadIdx.x / LANES * LANES * 16 + walk.io.element(i % 8, i / 8)] = walk.working ? dw[i] : 0.f;
    }
  }
  __syncthreads();
  const uint32_t first_group = blockIdx.x * kGroups;
  for (int e = threadIdx.x; e < 2 * p.dim; e += kRotaryThreads) {
    const int r = e >= p.dim;
    const int at = e - r * p.dim;
    float total = 0.f;
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t c = (first_group + g) % p.chunks;
      if (static_cast<int>(c >= p.q_chunks) == r) total += sums[g * LANES * 16 + at];
    }
    p.partials[static_cast<int64_t>(blockIdx.x) * 2 * p.dim + e] = total;
  }
}

// dweight[role][e] = sum over blocks: 32 strands of every 32nd block, each
// ascending, joined in a fixed order (3 us for 296 blocks, a launch).
template <typename W>
__global__ void __launch_bounds__(1024) rotary_weight_grad(const float* partials, int blocks, int dim, int columns,
                                                           W* dq, W* dk) {
  __shared__ float strand[32][33];
  const int lane = threadIdx.x, y = threadIdx.y;
  const int column = blockIdx.x * 32 + lane;
  float total = 0.f;
  if (column < columns) {
#pragma unroll 4
    for (int b = y; b < blocks; b += 32) total += partials[static_cast<int64_t>(b) * 2 * dim + column];
  }
  strand[y][lane] = total;
  __syncthreads();
  total = strand[lane][y];  // column y's strands, one a lane
#pragma unroll
  for (int step = 16; step > 0; step /= 2) total += __shfl_xor_sync(0xffffffffu, total, step);
  const int mine = blockIdx.x * 32 + y;
  if (lane == 0 && mine < columns) {
    if (mine < dim) dq[mine] = from_float<W>(total);
    else dk[mine - dim] = from_float<W>(total);
  }
}

int lanes_for(int dim) {
  int lanes = 1;
  while (lanes * 16 < dim) lanes *= 2;
  return lanes;
}

// Enough blocks for every (token, chunk), at most the resident ones, at least
// one group per chunk.
int rotary_blocks(int64_t tokens, uint32_t chunks, int dim) {
  const int groups = kRotaryThreads / lanes_for(dim);
  const int64_t wanted = ceil_div(tokens * chunks, groups);
  const int64_t least = ceil_div(chunks, groups);
  return static_cast<int>(std::max(least, std::min<int64_t>(wanted, static_cast<int64_t>(sm_count()) * kRotaryBlocks)));
}

// Heads of a group: as many as keep the copies within the shared memory, half
// of that where groups would be left short by more than a tenth (14 + 2 heads
// are four groups of 4, 4, 4, 2 and one of 2, but eight of 2).
int heads_per_group(int dtype, int heads_q, int heads_k, bool backward) {
  const int most = (dtype == kF32 ? 2 : 4) / (backward ? 2 : 1);
  const int64_t places = (ceil_div(heads_q, most) + ceil_div(heads_k, most)) * most;
  return most > 1 && 10 * (heads_q + heads_k) < 9 * places ? most / 2 : most;
}

template <typename T, bool INTERLEAVED, bool VECTOR, int HEADS>
int launch_heads(const RotaryParams& p, bool backward, int blocks, cudaStream_t stream) {
  auto run = [&](auto lanes) -> int {
    constexpr int L = decltype(lanes)::value;
    // HEADS counts forward; the backward pass copies twice as much a head.
    constexpr int kBackHeads = HEADS > 1 ? HEADS / 2 : 1;
    using Forward = Walk<T, L, INTERLEAVED, VECTOR, HEADS, 1>;
    using Backward = Walk<T, L, INTERLEAVED, VECTOR, kBackHeads, 2>;
    void (*kernel)(RotaryParams) =
        backward ? rotary_backward<T, L, INTERLEAVED, VECTOR, kBackHeads> : rotary_forward<T, L, INTERLEAVED, VECTOR, HEADS>;
    constexpr int kSums = kRotaryThreads * 16 * 4;
    // Without the copies only the weight gradients' sums need shared memory.
    const int shared = VECTOR ? (backward ? std::max(Backward::kStages * Backward::kStageBytes, kSums)
                                          : Forward::kStages * Forward::kStageBytes)
                              : backward ? kSums : 0;
    const int rc = allow_shared(reinterpret_cast<const void*>(kernel), shared);
    if (rc != SDC_OK) return rc;
    kernel<<<blocks, kRotaryThreads, shared, stream>>>(p);
    SDC_CUDA_CHECK(cudaGetLastError());
    return SDC_OK;
  };
  switch (lanes_for(p.dim)) {
    case 1: return run(std::integral_constant<int, 1>{});
    case 2: return run(std::integral_constant<int, 2>{});
    case 4: return run(std::integral_constant<int, 4>{});
    case 8: return run(std::integral_constant<int, 8>{});
    case 16: return run(std::integral_constant<int, 16>{});
    default: return run(std::integral_constant<int, 32>{});
  }
}

template <typename T, bool INTERLEAVED, bool VECTOR>
int launch_rotary(const RotaryParams& p, bool backward, int blocks, cudaStream_t stream) {
  constexpr int kMost = sizeof(T) == 2 ? 4 : 2;
  if (p.group_heads * (backward ? 2 : 1) == kMost) {
    return launch_heads<T, INTERLEAVED, VECTOR, kMost>(p, backward, blocks, stream);
  }
  return launch_heads<T, INTERLEAVED, VECTOR, kMost / 2>(p, backward, blocks, stream);
}

int dispatch_rotary(const RotaryParams& p, int dtype, bool interleaved, bool vector, bool backward, int blocks,
                    cudaStream_t stream) {
  auto typed = [&](auto element) -> int {
    using T = decltype(element);
    if (interleaved) {
      return vector ? launch_rotary<T, true, true>(p, backward, blocks, stream)
                    : launch_rotary<T, true, false>(p, backward, blocks, stream);
    }
    return vector ? launch_rotary<T, false, true>(p, backward, blocks, stream)
                  : launch_rotary<T, false, false>(p, backward, blocks, stream);
  };
  if (dtype == kF32) return typed(float{});
  if (dtype == kBF16) return typed(__nv_bfloat16{});
  return typed(__half{});
}

bool strides_aligned(const int64_t* strides, int dtype) {
  const int64_t unit = 16 / static_cast<int64_t>(element_size(dtype));
  return strides[0] % unit == 0 && strides[1] % unit == 0 && strides[2] % unit == 0;
}

int fill_params(RotaryParams& p, int dtype, const void* q, const int64_t* q_strides, const void* k,
                const int64_t* k_strides, int64_t batch, int64_t sequence, int heads_q, int heads_k, int dim,
                const float* table, int64_t table_rows, int rotary, const void* positions, int positions_64,
                const int64_t* position_strides, const void* q_weight, const void* k_weight, int weight_f32,
                float eps, void* q_out, void* k_out, bool backward) {
  SDC_REQUIRE(dtype == kF32 || dtype == kBF16 || dtype == kF16,
              "head norm rotation takes FP32 (0), BF16 (1) or FP16 (2) heads");
  SDC_REQUIRE(batch >= 0 && sequence >= 0 && heads_q > 0 && heads_k >= 0, "head norm rotation sizes must not be negative and q needs a head");
  SDC_REQUIRE(dim >= 2 && dim % 2 == 0 && dim <= kMaxHeadDim, "head dimension must be even and at most 512");
  SDC_REQUIRE(rotary >= 2 && rotary % 2 == 0 && rotary <= dim, "rotary dimension must be even and within the head");
  SDC_REQUIRE((q_weight == nullptr) == (k_weight == nullptr) || heads_k == 0,
              "head norm weights must be given for both q and k, or for neither");
  SDC_REQUIRE(std::isfinite(eps) && eps >= 0.f, "head norm eps must be finite and not negative");
  if (batch == 0 || sequence == 0) return SDC_OK;
  SDC_REQUIRE(batch <= INT_MAX / sequence, "head norm rotation takes at most 2^31 - 1 tokens");
  SDC_REQUIRE(q != nullptr && q_out != nullptr && table != nullptr && positions != nullptr && table_rows > 0 &&
                  (heads_k == 0 || (k != nullptr && k_out != nullptr)),
              "head norm rotation pointers must not be null");
  p.x[0] = q, p.x[1] = k;
  p.y[0] = q_out, p.y[1] = k_out;
  p.weight[0] = q_weight, p.weight[1] = k_weight;
  for (int i = 0; i < 3; ++i) {
    p.xs[0][i] = q_strides[i];
    p.xs[1][i] = heads_k > 0 ? k_strides[i] : 0;
  }
  p.position_strides[0] = position_strides[0], p.position_strides[1] = position_strides[1];
  p.positions = positions;
  p.table = table;
  p.table_rows = table_rows;
  p.sequence = static_cast<uint32_t>(sequence);
  p.tokens = static_cast<uint32_t>(batch * sequence);
  p.heads[0] = heads_q, p.heads[1] = heads_k;
  const int heads_per_group = p.group_heads = sdc::heads_per_group(dtype, heads_q, heads_k, backward);
  p.q_chunks = static_cast<uint32_t>(ceil_div(heads_q, heads_per_group));
  p.chunks = p.q_chunks + static_cast<uint32_t>(ceil_div(heads_k, heads_per_group));
  SDC_REQUIRE(static_cast<int64_t>(p.tokens) * p.chunks < INT_MAX - 512,
              "head norm rotation has too many heads for one launch");
  p.dim = dim;
  p.rotary = rotary;
  p.eps = eps;
  p.inv_dim = 1.f / static_cast<float>(dim);
  p.positions_64 = positions_64 != 0;
  p.weight_f32 = weight_f32 != 0;
  p.vector_table = rotary % 8 == 0 && aligned16(table);
  p.vector_weight = aligned16(q_weight) && aligned16(k_weight);
  return SDC_OK;
}

// Runs of 8 elements that start on 16 bytes: the half-split form needs whole
// runs on either side of the rotary part's middle and end.
bool vector_layout(const RotaryParams& p, int dtype, bool interleaved) {
  if (p.dim % 16 != 0 || !(interleaved || p.rotary % 16 == 0)) return false;
  for (int role = 0; role < 2; ++role) {
    if (p.heads[role] == 0) continue;
    if (!aligned16(p.x[role]) || !aligned16(p.y[role]) || !strides_aligned(p.xs[role], dtype)) return false;
  }
  return true;
}

}  // namespace
}  // namespace sdc

extern "C" {

int sdc_head_norm_rotary(int dtype, const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                         int64_t batch, int64_t sequence, int heads_q, int heads_k, int dim, const float* table,
                         int64_t table_rows, int rotary, int interleaved, const void* positions, int positions_64,
                         const int64_t* position_strides, const void* q_weight, const void* k_weight, int weight_f32,
                         float eps, void* q_out, void* k_out, sdc_stream_t stream) {
  using namespace sdc;
  RotaryParams p{};
  int rc = fill_params(p, dtype, q, q_strides, k, k_strides, batch, sequence, heads_q, heads_k, dim, table,
                       table_rows, rotary, positions, positions_64, position_strides, q_weight, k_weight, weight_f32,
                       eps, q_out, k_out, false);
  if (rc != SDC_OK || batch == 0 || sequence == 0) return rc;
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  const int blocks = rotary_blocks(p.tokens, p.chunks, dim);
  return dispatch_rotary(p, dtype, interleaved != 0, vector_layout(p, dtype, interleaved != 0), false, blocks, stream);
}

size_t sdc_head_norm_rotary_workspace_bytes(int64_t batch, int64_t sequence, int heads_q, int heads_k, int dim) {
  using namespace sdc;
  if (batch <= 0 || sequence <= 0 || heads_q <= 0 || heads_k < 0 || dim < 2 || dim > kMaxHeadDim) return 0;
  // As many chunks as there are heads, the most that any type has.
  const uint32_t chunks = static_cast<uint32_t>(heads_q + heads_k);
  return static_cast<size_t>(rotary_blocks(batch * sequence, chunks, dim)) * 2 * dim * sizeof(float);
}

int sdc_head_norm_rotary_backward(int dtype, const void* dq_out, const int64_t* dq_strides, const void* dk_out,
                                  const int64_t* dk_strides, const void* q, const int64_t* q_strides, const void* k,
                                  const int64_t* k_strides, int64_t batch, int64_t sequence, int heads_q, int heads_k,
                                  int dim, const float* table, int64_t table_rows, int rotary, int interleaved,
                                  const void* positions, int positions_64, const int64_t* position_strides,
                                  const void* q_weight, const void* k_weight, int weight_f32, float eps, void* dq,
                                  void* dk, void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes,
                                  sdc_stream_t stream) {
  using namespace sdc;
  RotaryParams p{};
  int rc = fill_params(p, dtype, q, q_strides, k, k_strides, batch, sequence, heads_q, heads_k, dim, table,
                       table_rows, rotary, positions, positions_64, position_strides, q_weight, k_weight, weight_f32,
                       eps, dq, dk, true);
  if (rc != SDC_OK) return rc;
  const bool norm = q_weight != nullptr;
  SDC_REQUIRE(!norm || (dq_weight != nullptr && (heads_k == 0 || dk_weight != nullptr)),
              "head norm weight gradients must not be null");
  const bool empty = batch == 0 || sequence == 0;
  SDC_REQUIRE(empty || (dq_out != nullptr && (heads_k == 0 || dk_out != nullptr)),
              "head norm rotation gradients must not be null");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  int blocks = 0;
  if (!empty) {
    p.dy[0] = dq_out, p.dy[1] = dk_out;
    for (int i = 0; i < 3; ++i) {
      p.dys[0][i] = dq_strides[i];
      p.dys[1][i] = heads_k > 0 ? dk_strides[i] : 0;
    }
    blocks = rotary_blocks(p.tokens, p.chunks, dim);
    if (norm) {
      if (workspace == nullptr || workspace_bytes < static_cast<size_t>(blocks) * 2 * dim * sizeof(float)) {
        return fail(SDC_ERR_WORKSPACE, "head norm rotation workspace is missing or too small");
      }
      p.partials = static_cast<float*>(workspace);
    }
    bool vector = vector_layout(p, dtype, interleaved != 0);
    for (int role = 0; role < 2; ++role) {
      if (p.heads[role] > 0) vector = vector && aligned16(p.dy[role]) && strides_aligned(p.dys[role], dtype);
    }
    rc = dispatch_rotary(p, dtype, interleaved != 0, vector, true, blocks, stream);
    if (rc != SDC_OK) return rc;
  }
  if (!norm) return SDC_OK;
  const int columns = (heads_k > 0 ? 2 : 1) * dim;
  const unsigned grid = static_cast<unsigned>(ceil_div(columns, 32));
  auto reduce = [&](auto element) {
    using W = decltype(element);
    rotary_weight_grad<W><<<grid, dim3(32, 32), 0, stream>>>(p.partials, blocks, dim, columns, static_cast<W*>(dq_weight),
                                                            static_cast<W*>(dk_weight));
  };
  if (weight_f32 || dtype == kF32) reduce(float{});
  else if (dtype == kBF16) reduce(__nv_bfloat16{});
  else reduce(__half{});
  SDC_CUDA_CHECK(cudaGetLastError());
  return SDC_OK;
}

}  // extern "C"
