// Norm of each query and key head with the rotation by position in one pass,
// forward and backward.
//
//   forward   r = rsqrt(mean_d x^2 + eps),  u = x r,  y = Rot(w u)
//   backward  g = Rot^T dy,  dx = r (g w - u mean_d(g w u)),  dw = sum g u
//
// Rot turns pair p < rotary/2 of a head by the position's angle p: elements
// (p, p + rotary/2), or (2p, 2p+1) when interleaved; elements from `rotary`
// on pass. Without weights the heads are only turned.
//
// Both directions move bytes and little else (about 10 flops an element), so
// the layout serves the loads: a thread owns 8 pairs of a head, both members
// of each, so the rotation needs no exchange between threads; in the common
// forms its 16 elements are two (16-bit types) or four (fp32) 16-byte words.
// dim/16 neighbouring lanes share a head and exchange only the sum of squares
// (and, backward, of products). A group of lanes takes up to kForwardHeads
// heads of one token: all their loads are issued before the first is used,
// and the angles and weights are read once for them.
#include <algorithm>
#include <climits>
#include <cmath>

#include "layers.cuh"

namespace sdc {
namespace {

constexpr int kRotaryThreads = 256;
constexpr int kForwardHeads = 4;
constexpr int kBackwardHeads = 2;
constexpr int kForwardBlocks = 2, kBackwardBlocks = 2;  // on an SM at least
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
  int dim, rotary;
  float eps, inv_dim;
  bool positions_64, weight_f32, vector_table, vector_weight;
  float* partials;       // backward: [blocks][2][dim]
};

// The position's cosine and sine for this lane's 8 pairs; identity beyond the
// rotary pairs. A position outside the table gives NaN, not a stray read.
__device__ __forceinline__ void load_angles(const RotaryParams& p, int64_t batch, int64_t seq, int first_pair,
                                            float* cosine, float* sine) {
  const int64_t at = batch * p.position_strides[0] + seq * p.position_strides[1];
  const int64_t position = p.positions_64 ? static_cast<const int64_t*>(p.positions)[at]
                                          : static_cast<const int32_t*>(p.positions)[at];
  const int half = p.rotary / 2;
  const bool inside = position >= 0 && position < p.table_rows;
  const float* row = p.table + (inside ? position : 0) * p.rotary;
  if (inside && p.vector_table && first_pair + 8 <= half) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 c = reinterpret_cast<const float4*>(row + first_pair)[i];
      const float4 s = reinterpret_cast<const float4*>(row + half + first_pair)[i];
      cosine[4 * i] = c.x, cosine[4 * i + 1] = c.y, cosine[4 * i + 2] = c.z, cosine[4 * i + 3] = c.w;
      sine[4 * i] = s.x, sine[4 * i + 1] = s.y, sine[4 * i + 2] = s.z, sine[4 * i + 3] = s.w;
    }
    return;
  }
  const float nan = __int_as_float(0x7fffffff);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int pair = first_pair + i;
    const bool turned = pair < half;
    cosine[i] = turned ? (inside ? row[pair] : nan) : 1.f;
    sine[i] = turned ? (inside ? row[half + pair] : nan) : 0.f;
  }
}

// Where this lane's pairs lie in a head: member 0 and member 1 of pair i are
// at first + i * step and second + i * step.
struct PairLayout {
  int first, second, step;
};

template <bool INTERLEAVED>
__device__ __forceinline__ int element_of(int pair, int member, int rotary) {
  if (!INTERLEAVED && pair < rotary / 2) return pair + member * (rotary / 2);
  return 2 * pair + member;  // passing elements pair up in order as well
}

// v[i], v[8 + i]: members of pair i. VECTOR: the 8 pairs are two runs of 8
// elements (half-split rotary pairs) or one run of 16.
template <typename T, bool INTERLEAVED, bool VECTOR>
struct HeadIO {
  int first_pair, rotary, pairs;
  bool active, split;

  __device__ __forceinline__ HeadIO(const RotaryParams& p, int lane)
      : first_pair(lane * 8), rotary(p.rotary), pairs(p.dim / 2), active(lane * 8 < p.dim / 2),
        split(!INTERLEAVED && lane * 8 < p.rotary / 2) {}

  __device__ __forceinline__ int low_run() const { return split ? first_pair : 2 * first_pair; }
  __device__ __forceinline__ int high_run() const { return split ? first_pair + rotary / 2 : 2 * first_pair + 8; }

  struct Raw {
    Raw8<T> a, b;
  };
  __device__ __forceinline__ Raw load(const T* head) const {
    Raw r;
    if constexpr (VECTOR) {
      r.a = load8(head + low_run());
      r.b = load8(head + high_run());
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
  __device__ __forceinline__ void unpack(const Raw& r, float* v) const { unpack_runs<T>(r.a, r.b, v); }
  template <typename E>
  __device__ __forceinline__ void unpack_runs(const Raw8<E>& ra, const Raw8<E>& rb, float* v) const {
    float a[8], b[8];
    unpack8(ra, a);
    unpack8(rb, b);
    const bool runs = VECTOR && !split;  // 16 elements in order: even ones are the first members
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (VECTOR) {
        const float e0 = i < 4 ? a[(2 * i) & 7] : b[(2 * i) & 7];
        const float e1 = i < 4 ? a[(2 * i + 1) & 7] : b[(2 * i + 1) & 7];
        v[i] = INTERLEAVED || runs ? e0 : a[i];
        v[8 + i] = INTERLEAVED || runs ? e1 : b[i];
      } else {
        v[i] = a[i];
        v[8 + i] = b[i];
      }
    }
  }
  __device__ __forceinline__ void store(T* head, const float* v) const {
    if constexpr (VECTOR) {
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool runs = INTERLEAVED || !split;
        a[2 * i] = runs ? v[i] : v[2 * i];
        a[2 * i + 1] = runs ? v[8 + i] : v[2 * i + 1];
        b[2 * i] = runs ? v[4 + i] : v[8 + 2 * i];
        b[2 * i + 1] = runs ? v[12 + i] : v[8 + 2 * i + 1];
      }
      store8(head + low_run(), pack8<T>(a));
      store8(head + high_run(), pack8<T>(b));
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
        unpack_runs<float>(load8(from + low_run()), load8(from + high_run()), w);
      } else {
        unpack(load(static_cast<const T*>(weight)), w);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int member = 0; member < 2; ++member) {
        const int pair = first_pair + i;
        const int e = element_of<INTERLEAVED>(pair, member, rotary);
        float value = 0.f;
        if (pair < pairs) {
          value = f32 ? static_cast<const float*>(weight)[e] : to_float(static_cast<const T*>(weight)[e]);
        }
        w[8 * member + i] = value;
      }
    }
  }
};

template <int LANES>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int step = LANES / 2; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
  return x;
}

template <typename T, int LANES, bool INTERLEAVED, bool VECTOR>
__global__ void __launch_bounds__(kRotaryThreads, kForwardBlocks) rotary_forward(RotaryParams p) {
  constexpr int kGroups = kRotaryThreads / LANES;
  const uint32_t item = blockIdx.x * kGroups + threadIdx.x / LANES;
  const uint32_t token = item / p.chunks;
  const uint32_t chunk = item - token * p.chunks;
  const HeadIO<T, INTERLEAVED, VECTOR> io(p, threadIdx.x % LANES);
  // Whole groups are idle or active; idle lanes still take part in the sums.
  const bool live = token < p.tokens && io.active;
  const int role = chunk >= p.q_chunks;
  const int head0 = static_cast<int>(chunk - (role ? p.q_chunks : 0)) * kForwardHeads;
  const int64_t batch = live ? token / p.sequence : 0, seq = live ? token % p.sequence : 0;
  const T* x = static_cast<const T*>(p.x[role]) + batch * p.xs[role][0] + seq * p.xs[role][1];
  T* y = static_cast<T*>(p.y[role]) + static_cast<int64_t>(token) * p.heads[role] * p.dim;

  typename HeadIO<T, INTERLEAVED, VECTOR>::Raw raw[kForwardHeads];
#pragma unroll
  for (int h = 0; h < kForwardHeads; ++h) {
    if (live && head0 + h < p.heads[role]) raw[h] = io.load(x + (head0 + h) * p.xs[role][2]);
  }
  float cosine[8], sine[8], w[16];
  const bool norm = p.weight[role] != nullptr;
  if (live) {
    load_angles(p, batch, seq, io.first_pair, cosine, sine);
    if (norm) io.weights(p.weight[role], p.weight_f32, p.vector_weight, w);
  }
#pragma unroll
  for (int h = 0; h < kForwardHeads; ++h) {
    const bool mine = live && head0 + h < p.heads[role];
    float v[16];
    if (mine) io.unpack(raw[h], v);
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
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      out[i] = v[i] * cosine[i] - v[8 + i] * sine[i];
      out[8 + i] = v[8 + i] * cosine[i] + v[i] * sine[i];
    }
    io.store(y + (head0 + h) * p.dim, out);
  }
}

// A group keeps one chunk of heads and walks the tokens, so that a thread's
// 16 weight gradients stay in registers for the whole launch; the block adds
// its groups' sums in a fixed order and writes one partial per role.
template <typename T, int LANES, bool INTERLEAVED, bool VECTOR>
__global__ void __launch_bounds__(kRotaryThreads, kBackwardBlocks) rotary_backward(RotaryParams p) {
  constexpr int kGroups = kRotaryThreads / LANES;
  __shared__ float sums[kRotaryThreads * 16];
  const uint32_t group = blockIdx.x * kGroups + threadIdx.x / LANES;
  const uint32_t walkers = gridDim.x * kGroups / p.chunks;
  const uint32_t walker = group / p.chunks;
  const uint32_t chunk = group - walker * p.chunks;
  const HeadIO<T, INTERLEAVED, VECTOR> io(p, threadIdx.x % LANES);
  const int role = chunk >= p.q_chunks;
  const int head0 = static_cast<int>(chunk - (role ? p.q_chunks : 0)) * kBackwardHeads;
  const bool norm = p.weight[role] != nullptr;
  const bool working = walker < walkers;
  float w[16], dw[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) dw[i] = 0.f, w[i] = 1.f;
  if (norm && io.active) io.weights(p.weight[role], p.weight_f32, p.vector_weight, w);

  // All lanes of a warp run the same number of rounds: the sums are exchanged
  // by the whole warp.
  const uint32_t rounds = (p.tokens + walkers - 1) / walkers;
  for (uint32_t round = 0; round < rounds; ++round) {
    const uint32_t token = round * walkers + walker;
    const bool live = working && token < p.tokens && io.active;
    const int64_t batch = live ? token / p.sequence : 0, seq = live ? token % p.sequence : 0;
    const T* x = static_cast<const T*>(p.x[role]) + batch * p.xs[role][0] + seq * p.xs[role][1];
    const T* dy = static_cast<const T*>(p.dy[role]) + batch * p.dys[role][0] + seq * p.dys[role][1];
    T* dx = static_cast<T*>(p.y[role]) + static_cast<int64_t>(token) * p.heads[role] * p.dim;
    typename HeadIO<T, INTERLEAVED, VECTOR>::Raw rx[kBackwardHeads], rdy[kBackwardHeads];
#pragma unroll
    for (int h = 0; h < kBackwardHeads; ++h) {
      if (!live || head0 + h >= p.heads[role]) continue;
      rdy[h] = io.load(dy + (head0 + h) * p.dys[role][2]);
      if (norm) rx[h] = io.load(x + (head0 + h) * p.xs[role][2]);
    }
    float cosine[8], sine[8];
    if (live) load_angles(p, batch, seq, io.first_pair, cosine, sine);
#pragma unroll
    for (int h = 0; h < kBackwardHeads; ++h) {
      const bool mine = live && head0 + h < p.heads[role];
      float v[16], g[16];
      if (mine) {
        float dv[16];
        io.unpack(rdy[h], dv);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          g[i] = dv[i] * cosine[i] + dv[8 + i] * sine[i];
          g[8 + i] = dv[8 + i] * cosine[i] - dv[i] * sine[i];
        }
      }
      if (norm) {
        float squares = 0.f, products = 0.f;
        if (mine) {
          io.unpack(rx[h], v);
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
      if (mine) io.store(dx + (head0 + h) * p.dim, g);
    }
  }
  if (p.partials == nullptr) return;

  // sums[group][16 * lane + i]: element order within a lane as in unpack().
#pragma unroll
  for (int i = 0; i < 16; ++i) sums[threadIdx.x * 16 + i] = working ? dw[i] : 0.f;
  __syncthreads();
  const uint32_t first_group = blockIdx.x * kGroups;
  for (int e = threadIdx.x; e < 2 * p.dim; e += kRotaryThreads) {
    const int r = e >= p.dim;
    const int at = e - r * p.dim;
    // Lane and slot that hold element `at`.
    int pair, member;
    if (!INTERLEAVED && at < p.rotary) {
      member = at >= p.rotary / 2;
      pair = at - member * (p.rotary / 2);
    } else {
      pair = at / 2;
      member = at & 1;
    }
    const int slot = (pair / 8) * 16 + member * 8 + pair % 8;
    float total = 0.f;
    for (int g = 0; g < kGroups; ++g) {
      const uint32_t c = (first_group + g) % p.chunks;
      if (static_cast<int>(c >= p.q_chunks) == r) total += sums[g * LANES * 16 + slot];
    }
    p.partials[static_cast<int64_t>(blockIdx.x) * 2 * p.dim + e] = total;
  }
}

// dweight[role][e] = sum over blocks: 32 strands of every 32nd block, each
// ascending, joined in a fixed order.
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

int backward_blocks(int64_t tokens, uint32_t chunks, int dim) {
  const int groups = kRotaryThreads / lanes_for(dim);
  // Enough blocks for every (token, chunk), at most 4 resident blocks per SM,
  // at least one group per chunk.
  const int64_t wanted = ceil_div(tokens * chunks, groups);
  const int64_t least = ceil_div(chunks, groups);
  return static_cast<int>(std::max(least, std::min<int64_t>(wanted, static_cast<int64_t>(sm_count()) * 4)));
}

template <typename T, bool INTERLEAVED, bool VECTOR>
int launch_rotary(const RotaryParams& p, bool backward, int blocks, cudaStream_t stream) {
  auto run = [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    if (backward) rotary_backward<T, L, INTERLEAVED, VECTOR><<<blocks, kRotaryThreads, 0, stream>>>(p);
    else rotary_forward<T, L, INTERLEAVED, VECTOR><<<blocks, kRotaryThreads, 0, stream>>>(p);
  };
  switch (lanes_for(p.dim)) {
    case 1: run(std::integral_constant<int, 1>{}); break;
    case 2: run(std::integral_constant<int, 2>{}); break;
    case 4: run(std::integral_constant<int, 4>{}); break;
    case 8: run(std::integral_constant<int, 8>{}); break;
    case 16: run(std::integral_constant<int, 16>{}); break;
    default: run(std::integral_constant<int, 32>{}); break;
  }
  SDC_CUDA_CHECK(cudaGetLastError());
  return SDC_OK;
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
                float eps, void* q_out, void* k_out, int heads_per_group) {
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
                       eps, q_out, k_out, kForwardHeads);
  if (rc != SDC_OK || batch == 0 || sequence == 0) return rc;
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  const int groups = kRotaryThreads / lanes_for(dim);
  const int blocks = static_cast<int>(ceil_div(static_cast<int64_t>(p.tokens) * p.chunks, groups));
  return dispatch_rotary(p, dtype, interleaved != 0, vector_layout(p, dtype, interleaved != 0), false, blocks, stream);
}

size_t sdc_head_norm_rotary_workspace_bytes(int64_t batch, int64_t sequence, int heads_q, int heads_k, int dim) {
  using namespace sdc;
  if (batch <= 0 || sequence <= 0 || heads_q <= 0 || heads_k < 0 || dim < 2 || dim > kMaxHeadDim) return 0;
  const uint32_t chunks = static_cast<uint32_t>(ceil_div(heads_q, kBackwardHeads) + ceil_div(heads_k, kBackwardHeads));
  return static_cast<size_t>(backward_blocks(batch * sequence, chunks, dim)) * 2 * dim * sizeof(float);
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
                       eps, dq, dk, kBackwardHeads);
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
    blocks = backward_blocks(p.tokens, p.chunks, dim);
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
