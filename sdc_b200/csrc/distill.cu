// Distillation loss against a teacher's top logits, and its gradient.
//
// For a row of student logits s[0..V) and the teacher's list (i_k, t_k), with
// temperature tau, c = log2(e) / tau:
//
//   p_k = softmax_k(t_k / tau) over the list,  q = softmax(s / tau) over V
//   loss = tau^2 sum_k p_k (ln p_k - ln q[i_k])
//   d loss / d s_j = tau (q_j - sum_{k: i_k = j} p_k)
//
// Entries with a negative index are no entries; a row without any (or whose
// teacher logits are all -inf) has loss 0 and gradient 0 whatever its student
// logits are. An index beyond the vocabulary makes the row's loss and
// gradient NaN (never a stray access).
//
// All of it is bound by the bytes of the student's logits: V * 2 bytes a row
// against about 8 instructions an element. The loss reads them once (running
// maximum and sum per thread, joined across the row). Loss with gradient is
// also one read and one write: a cluster of blocks shares a row, each block
// keeps its slice in shared memory, the (max, sum) pairs cross the cluster
// through distributed shared memory, and the second pass over the slice
// writes the gradient. Softmax statistics are fp32; the exponents are formed
// as fma(s, c, -max c) with the same rounded max c in the sum and in the
// gradient, so its rounding cancels; where max c could overflow (rows masked
// with the type's lowest value throughout) as (s - max) c instead.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "layers.cuh"

namespace sdc {
namespace {

constexpr int kRowThreads = 512;               // threads that stream the slice
constexpr int kRowBlock = kRowThreads + 32;    // and one warp for the teacher's list
constexpr int kUnroll = 4;
constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr size_t kSharedLimit = 227 * 1024;
// Two blocks per SM: one loads while the other computes or writes.
constexpr size_t kSliceTarget = 100 * 1024;
constexpr int kBackThreads = 256;
constexpr int kBackGranules = 8;               // 16-byte words per thread

struct DistillParams {
  const void* logits;
  int64_t row_stride;
  int64_t vocab;
  const void* indices;
  int64_t index_stride;
  const void* teacher;
  int64_t teacher_stride;
  int top;
  bool indices_64;
  int teacher_type;
  float c;                  // log2(e) / temperature
  float tau, inv_tau;
  float* loss;              // [rows], nullable
  float4* stats;            // [rows]: max, 1 / sum, teacher max, 1 / teacher sum; nullable
  void* grad;
  int64_t grad_stride;
  const float* upstream;    // nullable: 1
  int64_t upstream_stride;  // 0 or 1
  const float* upstream_scale;  // nullable: 1
  int slice;                // 16-byte words of a row per block
  int chunks;               // backward: blocks per row
};

// 1 / sum of a row without teacher entries.
constexpr float kEmptyRow = -1.f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int64_t index_at(const DistillParams& p, int64_t row, int k) {
  const int64_t at = row * p.index_stride + k;
  return p.indices_64 ? static_cast<const int64_t*>(p.indices)[at] : static_cast<const int32_t*>(p.indices)[at];
}

__device__ __forceinline__ float teacher_at(const DistillParams& p, int64_t row, int k) {
  const int64_t at = row * p.teacher_stride + k;
  if (p.teacher_type == kF32) return static_cast<const float*>(p.teacher)[at];
  if (p.teacher_type == kBF16) return to_float(static_cast<const __nv_bfloat16*>(p.teacher)[at]);
  return to_float(static_cast<const __half*>(p.teacher)[at]);
}

__device__ __forceinline__ bool is_entry(int64_t index, float t) { return index >= 0 && t != -INFINITY; }

// A row as 16-byte words: the row starts `phase` elements into word 0.
template <typename T>
struct RowWords {
  static constexpr int kPer = 16 / sizeof(T);
  T* row;
  int phase;
  int64_t vocab;
  __device__ __forceinline__ RowWords(T* r, int64_t v)
      : row(r), phase(static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))), vocab(v) {}
  __device__ __forceinline__ int64_t words() const { return (phase + vocab + kPer - 1) / kPer; }
  __device__ __forceinline__ bool whole(int64_t word) const {
    const int64_t e = word * kPer - phase;
    return e >= 0 && e + kPer <= vocab;
  }
  __device__ __forceinline__ T* at(int64_t word) const { return row + (word * kPer - phase); }
  // Elements outside the row read as -inf.
  __device__ __forceinline__ uint4 load(int64_t word) const {
    if (whole(word)) return *reinterpret_cast<const uint4*>(at(word));
    using Value = std::remove_const_t<T>;
    uint4 r;
    Value* v = reinterpret_cast<Value*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = word * kPer - phase + i;
      v[i] = e >= 0 && e < vocab ? row[e] : from_float<Value>(-INFINITY);
    }
    return r;
  }
  __device__ __forceinline__ void store(int64_t word, const uint4& r) const {
    if (whole(word)) {
      *reinterpret_cast<uint4*>(at(word)) = r;
      return;
    }
    store_elements(word, r);
  }
  __device__ __forceinline__ void store_elements(int64_t word, const uint4& r) const {
    const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t e = word * kPer - phase + i;
      if (e >= 0 && e < vocab) row[e] = v[i];
    }
  }
};

template <typename T>
__device__ __forceinline__ void unpack_word(const uint4& r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack_word(const float* v) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

// Whether (s - m) c cannot be formed as s c - m c: a finite m with m c near
// the end of fp32's range.
__device__ __forceinline__ bool is_wild(float m, float c) { return fabsf(m) * c > 1e38f && fabsf(m) < INFINITY; }

// 2^((s - m) c) for a row or thread maximum m.
struct Exponent {
  float m, mc;
  bool wild;
  __device__ __forceinline__ Exponent(float top, float c)
      : m(top), mc(top == -INFINITY ? 0.f : top * c), wild(is_wild(top, c)) {}
  __device__ __forceinline__ float operator()(float s, float c) const {
    return exp2_fast(wild ? (s - m) * c : fmaf(s, c, -mc));
  }
  // v[i] = 2^((v[i] - m) c) * scale, the choice made once.
  template <int N>
  __device__ __forceinline__ void apply(float* v, float c, float scale) const {
    if (!wild) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = exp2_fast(fmaf(v[i], c, -mc)) * scale;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = exp2_fast((v[i] - m) * c) * scale;
    }
  }
};

// Running maximum m and sum of 2^((s - m) c). While nothing above -inf was
// seen m c counts as 0, so that -inf terms add 0.
struct Softmax {
  float m = -INFINITY, mc = 0.f, sum = 0.f;
  bool wild = false;

  __device__ __forceinline__ void raise(float to, float c) {
    const Exponent next(to, c);
    sum = m == -INFINITY ? sum : sum * next(m, c);
    m = to;
    mc = next.mc;
    wild = next.wild;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* v, float c) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, v[i]);
    if (top > m) raise(top, c);
    float part = 0.f;
    if (!wild) {
#pragma unroll
      for (int i = 0; i < N; ++i) part += exp2_fast(fmaf(v[i], c, -mc));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) part += exp2_fast((v[i] - m) * c);
    }
    sum += part;
  }
  __device__ __forceinline__ void join(float m2, float sum2, float c) {
    if (m2 > m) raise(m2, c);
    sum += m2 == -INFINITY ? sum2 : sum2 * Exponent(m, c)(m2, c);
  }
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int step = 16; step > 0; step /= 2) x += __shfl_xor_sync(0xffffffffu, x, step);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int step = 16; step > 0; step /= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, step));
  return x;
}

// What the list warp keeps of an entry.
struct Entry {
  float p;     // teacher probability
  float log_p; // its natural logarithm
  float s;     // student logit
  int at;      // index, -1: no entry
};

// A cluster of blocks per row; GRAD stages the slice and writes the gradient.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kRowBlock) distill_rows(DistillParams p) {
  extern __shared__ uint4 shared[];
  __shared__ float warp_m[kRowThreads / 32], warp_s[kRowThreads / 32];
  __shared__ float2 parts[kMaxCluster];
  constexpr int kPer = 16 / sizeof(T);
  Entry* list = reinterpret_cast<Entry*>(shared);
  uint4* stage = shared + p.top;  // an Entry is 16 bytes

  const uint32_t rank = cluster_ctarank();
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  // The other blocks' shared memory may be written once they have started;
  // the wait comes just before.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t row = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool lists = threadIdx.x >= kRowThreads;

  const RowWords<const T> in(static_cast<const T*>(p.logits) + row * p.row_stride, p.vocab);
  const int64_t first = static_cast<int64_t>(rank) * p.slice;
  const int count = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(p.slice), in.words() - first)));

  // The first words are on their way while the list is looked at.
  uint4 ahead[kUnroll];
  if (!lists) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int w = threadIdx.x + u * kRowThreads;
      if (w < count) ahead[u] = in.load(first + w);
    }
  }
  bool some = false;
  for (int k = 0; k < p.top && !some; k += 32) {
    bool entry = false;
    if (k + lane < p.top) entry = is_entry(index_at(p, row, k + lane), teacher_at(p, row, k + lane));
    some = __any_sync(0xffffffffu, entry);
  }
  if (!some) {  // the same for every thread of the cluster
    if (GRAD && !lists) {
      const RowWords<T> out(static_cast<T*>(p.grad) + row * p.grad_stride, p.vocab);
      const int64_t words = out.words();
      for (int64_t w = static_cast<int64_t>(rank) * kRowThreads + threadIdx.x; w < words;
           w += static_cast<int64_t>(ranks) * kRowThreads) {
        out.store(w, make_uint4(0, 0, 0, 0));
      }
    }
    if (rank == 0 && threadIdx.x == 0) {
      if (p.loss != nullptr) p.loss[row] = 0.f;
      if (p.stats != nullptr) p.stats[row] = make_float4(0.f, kEmptyRow, 0.f, 0.f);
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }

  Softmax mine;
  float teacher_max = 0.f, teacher_inv = 0.f;
  bool stray = false;
  if (lists) {
    float m = -INFINITY;
    for (int k = lane; k < p.top; k += 32) {
      const int64_t index = index_at(p, row, k);
      const float t = teacher_at(p, row, k);
      Entry e{t, 0.f, 0.f, -1};
      if (index >= p.vocab) stray = true;
      else if (is_entry(index, t)) {
        e.at = static_cast<int>(index);
        e.s = to_float(in.row[index]);
        m = fmaxf(m, t);
      }
      list[k] = e;
    }
    m = warp_max(m);
    stray = __any_sync(0xffffffffu, stray);
    teacher_max = m;
    float sum = 0.f;
    for (int k = lane; k < p.top; k += 32) {
      if (list[k].at >= 0) sum += exp2_fast((list[k].p - m) * p.c);
    }
    sum = warp_sum(sum);
    teacher_inv = 1.f / sum;
    const float log_sum = logf(sum);
    for (int k = lane; k < p.top; k += 32) {
      const float x = list[k].p - m;
      list[k].log_p = x * p.inv_tau - log_sum;
      list[k].p = exp2_fast(x * p.c) * teacher_inv;
    }
    __syncwarp();
  } else {
    for (int base = 0; base < count; base += kUnroll * kRowThreads) {
      uint4 next[kUnroll];
      const int after = base + kUnroll * kRowThreads + threadIdx.x;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (after + u * kRowThreads < count) next[u] = in.load(first + after + u * kRowThreads);
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int w = base + threadIdx.x + u * kRowThreads;
        if (w < count) {
          if constexpr (GRAD) stage[w] = ahead[u];
          float v[kPer];
          unpack_word<T>(ahead[u], v);
          mine.add<kPer>(v, p.c);
        }
        ahead[u] = next[u];
      }
    }
#pragma unroll
    for (int step = 16; step > 0; step /= 2) {
      const float m2 = __shfl_xor_sync(0xffffffffu, mine.m, step);
      const float s2 = __shfl_xor_sync(0xffffffffu, mine.sum, step);
      mine.join(m2, s2, p.c);
    }
    if (lane == 0) warp_m[warp] = mine.m, warp_s[warp] = mine.sum;
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < ranks) {  // one thread per block of the cluster
    Softmax block;
    for (int i = 0; i < kRowThreads / 32; ++i) block.join(warp_m[i], warp_s[i], p.c);
    const uint32_t to = mapa_shared(&parts[rank], threadIdx.x);
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(block.m), "f"(block.sum) : "memory");
  }
  cluster_sync();
  Softmax all;
  for (uint32_t i = 0; i < ranks; ++i) all.join(parts[i].x, parts[i].y, p.c);
  float inv = 1.f / all.sum;

  if (lists) {
    if (stray) inv = __int_as_float(0x7fffffff);
    if (rank == 0) {
      const float log_sum = logf(all.sum);
      float total = 0.f;
      for (int k = lane; k < p.top; k += 32) {
        const Entry e = list[k];
        if (e.at >= 0 && e.p != 0.f) total += e.p * (e.log_p - ((e.s - all.m) * p.inv_tau - log_sum));
      }
      total = warp_sum(total);
      if (lane == 0) {
        const float nan = __int_as_float(0x7fffffff);
        if (p.loss != nullptr) p.loss[row] = stray ? nan : total * p.tau * p.tau;
        if (p.stats != nullptr) p.stats[row] = make_float4(all.m, inv, teacher_max, teacher_inv);
      }
    }
  }
  if constexpr (GRAD) {
    __shared__ float row_inv;
    if (threadIdx.x == kRowThreads) row_inv = inv;
    __syncthreads();
    inv = row_inv;
    float a = p.tau;
    if (p.upstream != nullptr) a *= p.upstream[row * p.upstream_stride];
    const float scaled = a * inv;
    const RowWords<T> out(static_cast<T*>(p.grad) + row * p.grad_stride, p.vocab);
    const bool same_phase = out.phase == in.phase;
    const Exponent power(all.m, p.c);
    if (!lists) {
      for (int w = threadIdx.x; w < count; w += kRowThreads) {
        float v[kPer];
        unpack_word<T>(stage[w], v);
        power.template apply<kPer>(v, p.c, scaled);
        const uint4 r = pack_word<T>(v);
        if (same_phase) {
          out.store(first + w, r);
        } else {
          const RowWords<T> shifted = [&] { RowWords<T> s = out; s.phase = in.phase; return s; }();
          shifted.store_elements(first + w, r);
        }
      }
    }
    __syncthreads();
    if (!lists) return;
    // The list's columns again, with the teacher's part. Each entry leaves
    // its number in its (no longer needed) staged logit: one that finds
    // another number there shares its column.
    T* slot = reinterpret_cast<T*>(stage);
    auto local = [&](int k) -> int64_t {
      if (list[k].at < 0) return -1;
      const int64_t e = list[k].at + in.phase - first * kPer;
      return e >= 0 && e < static_cast<int64_t>(count) * kPer ? e : -1;
    };
    using Mark = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
    Mark* mark = reinterpret_cast<Mark*>(slot);
    for (int k = lane; k < p.top; k += 32) {
      const int64_t e = local(k);
      if (e >= 0) mark[e] = static_cast<Mark>(k);
    }
    __syncwarp();
    bool shared_column = false;
    for (int k = lane; k < p.top; k += 32) {
      const int64_t e = local(k);
      if (e >= 0 && mark[e] != static_cast<Mark>(k)) shared_column = true;
    }
    shared_column = __any_sync(0xffffffffu, shared_column);
    for (int k = lane; k < p.top; k += 32) {
      if (local(k) < 0) continue;
      const Entry e = list[k];
      float prob = e.p;
      if (shared_column) {  // every entry of the column writes the same sum
        prob = 0.f;
        for (int j = 0; j < p.top; ++j) {
          if (list[j].at == e.at) prob += list[j].p;
        }
      }
      const float q = power(e.s, p.c) * inv;
      out.row[e.at] = from_float<T>(a * (q - prob));
    }
  }
}

// The gradient from the row statistics: one read, one write, blocks of a row
// independent of each other.
template <typename T>
__global__ void __launch_bounds__(kBackThreads) distill_backward(DistillParams p) {
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kWords = kBackThreads * kBackGranules;
  constexpr int kEntries = kMaxTop / kBackThreads;
  __shared__ uint32_t seen[(kWords * kPer + 31) / 32];
  __shared__ int shared_column;
  const int64_t row = blockIdx.x / p.chunks;
  const int64_t first = static_cast<int64_t>(blockIdx.x % p.chunks) * kWords;
  const RowWords<const T> in(static_cast<const T*>(p.logits) + row * p.row_stride, p.vocab);
  const RowWords<T> out(static_cast<T*>(p.grad) + row * p.grad_stride, p.vocab);
  const int64_t words = in.words();

  uint4 raw[kBackGranules];
#pragma unroll
  for (int u = 0; u < kBackGranules; ++u) {
    const int64_t w = first + threadIdx.x + u * kBackThreads;
    if (w < words) raw[u] = in.load(w);
  }
  const float4 stats = p.stats[row];
  float a = p.tau;
  if (p.upstream != nullptr) a *= p.upstream[row * p.upstream_stride];
  if (p.upstream_scale != nullptr) a *= *p.upstream_scale;
  const bool empty = stats.y == kEmptyRow;
  const float scaled = a * stats.y;
  const Exponent power(stats.x, p.c);

  // This block's entries of the list; their logits before they are
  // overwritten (the gradient may replace the logits).
  int64_t at[kEntries];
  float s[kEntries];
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    at[i] = -1;
    const int k = threadIdx.x + i * kBackThreads;
    if (empty || k >= p.top) continue;
    const int64_t index = index_at(p, row, k);
    const int64_t word = (index + in.phase) / kPer;
    if (index < 0 || index >= p.vocab || word < first || word >= first + kWords) continue;
    if (!is_entry(index, teacher_at(p, row, k))) continue;
    at[i] = index;
    s[i] = to_float(in.row[index]);
  }
  for (int i = threadIdx.x; i < static_cast<int>(sizeof(seen) / 4); i += kBackThreads) seen[i] = 0;
  if (threadIdx.x == 0) shared_column = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    if (at[i] < 0) continue;
    const uint32_t e = static_cast<uint32_t>(at[i] + in.phase - first * kPer);
    if (atomicOr(&seen[e / 32], 1u << (e % 32)) >> (e % 32) & 1u) shared_column = 1;
  }
#pragma unroll
  for (int u = 0; u < kBackGranules; ++u) {
    const int64_t w = first + threadIdx.x + u * kBackThreads;
    if (w >= words) continue;
    float v[kPer];
    unpack_word<T>(raw[u], v);
    power.apply<kPer>(v, p.c, scaled);
    const uint4 r = empty ? make_uint4(0, 0, 0, 0) : pack_word<T>(v);
    if (out.phase == in.phase) {
      out.store(w, r);
    } else {
      const RowWords<T> shifted = [&] { RowWords<T> o = out; o.phase = in.phase; return o; }();
      shifted.store_elements(w, r);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    if (at[i] < 0) continue;
    const int k = threadIdx.x + i * kBackThreads;
    float prob = exp2_fast((teacher_at(p, row, k) - stats.z) * p.c) * stats.w;
    if (shared_column) {
      prob = 0.f;
      for (int j = 0; j < p.top; ++j) {
        if (index_at(p, row, j) != at[i]) continue;
        const float t = teacher_at(p, row, j);
        if (t != -INFINITY) prob += exp2_fast((t - stats.z) * p.c) * stats.w;
      }
    }
    const float q = power(s[i], p.c) * stats.y;
    out.row[at[i]] = from_float<T>(a * (q - prob));
  }
}

// out[0] = sum or mean of the losses over the rows that have entries (0 when
// none has), out[1] = what a row's loss was multiplied with. One block, fixed
// order.
__global__ void __launch_bounds__(1024) distill_reduce(const float* loss, const float4* stats, int64_t rows, bool mean,
                                                       float* out) {
  __shared__ float sums[32];
  __shared__ int counts[32];
  float sum = 0.f;
  int count = 0;
  for (int64_t r = threadIdx.x; r < rows; r += 1024) {
    sum += loss[r];
    count += stats[r].y != kEmptyRow;
  }
  sum = warp_sum(sum);
  count = __reduce_add_sync(0xffffffffu, count);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x / 32] = sum, counts[threadIdx.x / 32] = count;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  sum = warp_sum(sums[threadIdx.x]);
  count = __reduce_add_sync(0xffffffffu, counts[threadIdx.x]);
  if (threadIdx.x == 0) {
    const float scale = mean ? 1.f / static_cast<float>(max(count, 1)) : 1.f;
    out[0] = sum * scale;
    out[1] = scale;
  }
}

int check_distill(int dtype, const void* logits, int64_t rows, int64_t vocab, const void* indices, const void* teacher,
                  int teacher_dtype, int top, float temperature) {
  SDC_REQUIRE(dtype == kF32 || dtype == kBF16 || dtype == kF16, "distillation takes FP32 (0), BF16 (1) or FP16 (2) logits");
  SDC_REQUIRE(teacher_dtype == kF32 || teacher_dtype == kBF16 || teacher_dtype == kF16,
              "distillation takes FP32 (0), BF16 (1) or FP16 (2) teacher logits");
  SDC_REQUIRE(rows >= 0 && vocab > 0 && vocab < INT_MAX - 64, "distillation needs a vocabulary of 1 to 2^31 - 66 tokens");
  SDC_REQUIRE(top >= 1 && top <= kMaxTop, "distillation takes 1 to 1024 teacher logits a row");
  SDC_REQUIRE(std::isfinite(temperature) && temperature > 1e-30f, "distillation temperature must be positive and finite");
  SDC_REQUIRE(rows == 0 || (logits != nullptr && indices != nullptr && teacher != nullptr),
              "distillation pointers must not be null");
  SDC_REQUIRE(reinterpret_cast<uintptr_t>(logits) % element_size(dtype) == 0, "distillation logits must be aligned to their type");
  return SDC_OK;
}

DistillParams distill_params(const void* logits, int64_t vocab, int64_t row_stride, const void* indices,
                             int indices_64, int64_t index_stride, const void* teacher, int teacher_dtype,
                             int64_t teacher_stride, int top, float temperature) {
  DistillParams p{};
  p.logits = logits;
  p.row_stride = row_stride;
  p.vocab = vocab;
  p.indices = indices;
  p.indices_64 = indices_64 != 0;
  p.index_stride = index_stride;
  p.teacher = teacher;
  p.teacher_type = teacher_dtype;
  p.teacher_stride = teacher_stride;
  p.top = top;
  p.c = static_cast<float>(1.4426950408889634 / static_cast<double>(temperature));
  p.tau = temperature;
  p.inv_tau = 1.f / temperature;
  return p;
}

int max_words(int64_t vocab, int dtype) {
  const int per = 16 / static_cast<int>(element_size(dtype));
  return static_cast<int>(ceil_div(vocab + per - 1, per));  // whatever the row's phase
}

size_t shared_bytes(int64_t vocab, int dtype, int top, int cluster, bool grad) {
  return static_cast<size_t>(top) * sizeof(Entry) +
         (grad ? static_cast<size_t>(ceil_div(max_words(vocab, dtype), cluster)) * 16 : 0);
}

// Blocks per row: the gradient's slice should let two blocks share an SM
// (and must fit one); beyond that, few rows are split until the blocks fill
// the SMs. 0: a row does not fit a cluster.
int cluster_size(int64_t rows, int64_t vocab, int dtype, int top, bool grad) {
  int cluster = 1;
  while (cluster < kMaxCluster && shared_bytes(vocab, dtype, top, cluster, grad) > kSliceTarget) cluster *= 2;
  if (shared_bytes(vocab, dtype, top, cluster, grad) > kSharedLimit - 2048) return 0;
  while (cluster < kMaxCluster && rows * cluster < 2 * sm_count() && max_words(vocab, dtype) / cluster > 2 * kRowThreads) {
    cluster *= 2;
  }
  return cluster;
}

template <typename T, bool GRAD>
int launch_rows(DistillParams p, int64_t rows, int cluster, size_t shared, cudaStream_t stream) {
  static std::atomic<uint64_t> prepared{0};
  int device = 0;
  SDC_CUDA_CHECK(cudaGetDevice(&device));
  const uint64_t bit = 1ull << (device & 63);
  if ((prepared.load(std::memory_order_relaxed) & bit) == 0) {
    SDC_CUDA_CHECK(cudaFuncSetAttribute(distill_rows<T, GRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>(kSharedLimit - 2048)));
    prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(rows * cluster));
  config.blockDim = dim3(kRowBlock);
  config.dynamicSmemBytes = shared;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attribute[0].val.clusterDim.y = 1;
  attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  SDC_CUDA_CHECK(cudaLaunchKernelEx(&config, distill_rows<T, GRAD>, p));
  return SDC_OK;
}

template <bool GRAD>
int run_rows(DistillParams p, int dtype, int64_t rows, int cluster, cudaStream_t stream) {
  SDC_REQUIRE(rows <= INT_MAX / cluster, "distillation has too many rows for one launch");
  p.slice = static_cast<int>(ceil_div(max_words(p.vocab, dtype), cluster));
  const size_t shared = shared_bytes(p.vocab, dtype, p.top, cluster, GRAD);
  if (dtype == kF32) return launch_rows<float, GRAD>(p, rows, cluster, shared, stream);
  if (dtype == kBF16) return launch_rows<__nv_bfloat16, GRAD>(p, rows, cluster, shared, stream);
  return launch_rows<__half, GRAD>(p, rows, cluster, shared, stream);
}

int run_backward(DistillParams p, int dtype, int64_t rows, cudaStream_t stream) {
  p.chunks = static_cast<int>(ceil_div(max_words(p.vocab, dtype), kBackThreads * kBackGranules));
  SDC_REQUIRE(rows <= INT_MAX / p.chunks, "distillation has too many rows for one launch");
  const unsigned grid = static_cast<unsigned>(rows * p.chunks);
  if (dtype == kF32) distill_backward<float><<<grid, kBackThreads, 0, stream>>>(p);
  else if (dtype == kBF16) distill_backward<__nv_bfloat16><<<grid, kBackThreads, 0, stream>>>(p);
  else distill_backward<__half><<<grid, kBackThreads, 0, stream>>>(p);
  SDC_CUDA_CHECK(cudaGetLastError());
  return SDC_OK;
}

}  // namespace
}  // namespace sdc

extern "C" {

int sdc_distill_loss(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t row_stride,
                     const void* indices, int indices_64, int64_t index_stride, const void* teacher,
                     int teacher_dtype, int64_t teacher_stride, int top, float temperature, float* loss, float* stats,
                     sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_distill(dtype, logits, rows, vocab, indices, teacher, teacher_dtype, top, temperature);
  if (rc != SDC_OK) return rc;
  if (rows == 0) return SDC_OK;
  SDC_REQUIRE(loss != nullptr && stats != nullptr && aligned16(stats),
              "distillation losses must not be null and row statistics must be 16-byte aligned");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  DistillParams p = distill_params(logits, vocab, row_stride, indices, indices_64, index_stride, teacher,
                                   teacher_dtype, teacher_stride, top, temperature);
  p.loss = loss;
  p.stats = reinterpret_cast<float4*>(stats);
  return run_rows<false>(p, dtype, rows, cluster_size(rows, vocab, dtype, top, false), stream);
}

int sdc_distill_reduce(const float* loss, const float* stats, int64_t rows, int mean, float* out,
                       sdc_stream_t stream) {
  using namespace sdc;
  SDC_REQUIRE(rows >= 0 && out != nullptr && (rows == 0 || (loss != nullptr && stats != nullptr && aligned16(stats))),
              "distillation reduction pointers must not be null and row statistics must be 16-byte aligned");
  int rc = check_current_device();
  if (rc != SDC_OK) return rc;
  distill_reduce<<<1, 1024, 0, stream>>>(loss, reinterpret_cast<const float4*>(stats), rows, mean != 0, out);
  SDC_CUDA_CHECK(cudaGetLastError());
  return SDC_OK;
}

int sdc_distill_backward(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t row_stride,
                         const void* indices, int indices_64, int64_t index_stride, const void* teacher,
                         int teacher_dtype, int64_t teacher_stride, int top, float temperature, const float* stats,
                         const float* grad_loss, int64_t grad_loss_stride, const float* grad_scale, void* grad,
                         int64_t grad_stride, sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_distill(dtype, logits, rows, vocab, indices, teacher, teacher_dtype, top, temperature);
  if (rc != SDC_OK) return rc;
  if (rows == 0) return SDC_OK;
  SDC_REQUIRE(stats != nullptr && aligned16(stats) && grad != nullptr && (rows == 1 || grad_stride >= vocab),
              "distillation gradient rows must not overlap and row statistics must be 16-byte aligned");
  SDC_REQUIRE(grad_loss_stride == 0 || grad_loss_stride == 1, "distillation upstream gradients are one value or one a row");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  DistillParams p = distill_params(logits, vocab, row_stride, indices, indices_64, index_stride, teacher,
                                   teacher_dtype, teacher_stride, top, temperature);
  p.stats = const_cast<float4*>(reinterpret_cast<const float4*>(stats));
  p.upstream = grad_loss;
  p.upstream_stride = grad_loss_stride;
  p.upstream_scale = grad_scale;
  p.grad = grad;
  p.grad_stride = grad_stride;
  return run_backward(p, dtype, rows, stream);
}

int sdc_distill_loss_and_grad(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t row_stride,
                              const void* indices, int indices_64, int64_t index_stride, const void* teacher,
                              int teacher_dtype, int64_t teacher_stride, int top, float temperature,
                              const float* grad_loss, int64_t grad_loss_stride, float* loss, float* stats, void* grad,
                              int64_t grad_stride, sdc_stream_t stream) {
  using namespace sdc;
  int rc = check_distill(dtype, logits, rows, vocab, indices, teacher, teacher_dtype, top, temperature);
  if (rc != SDC_OK) return rc;
  if (rows == 0) return SDC_OK;
  SDC_REQUIRE(loss != nullptr && stats != nullptr && aligned16(stats) && grad != nullptr,
              "distillation losses must not be null and row statistics must be 16-byte aligned");
  SDC_REQUIRE(rows == 1 || grad_stride >= vocab, "distillation gradient rows must not overlap");
  SDC_REQUIRE(grad_loss_stride == 0 || grad_loss_stride == 1, "distillation upstream gradients are one value or one a row");
  rc = check_current_device();
  if (rc != SDC_OK) return rc;
  DistillParams p = distill_params(logits, vocab, row_stride, indices, indices_64, index_stride, teacher,
                                   teacher_dtype, teacher_stride, top, temperature);
  p.loss = loss;
  p.stats = reinterpret_cast<float4*>(stats);
  p.upstream = grad_loss;
  p.upstream_stride = grad_loss_stride;
  p.grad = grad;
  p.grad_stride = grad_stride;
  const int cluster = cluster_size(rows, vocab, dtype, top, true);
  if (cluster > 0) return run_rows<true>(p, dtype, rows, cluster, stream);
  // A row beyond what a cluster's shared memory holds is read twice.
  rc = run_rows<false>(p, dtype, rows, cluster_size(rows, vocab, dtype, top, false), stream);
  return rc == SDC_OK ? run_backward(p, dtype, rows, stream) : rc;
}

}  // extern "C"
