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
// writes the gradient. Softmax statistics are fp32.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <type_traits>

#include "layers.cuh"

namespace sdc {
namespace {

constexpr int kRowThreads = 256;               // threads that stream the slice
constexpr int kRowBlock = kRowThreads + 32;    // and one warp for the teacher's list
constexpr int kUnroll = 4;                      // words at once from global memory
constexpr int kAtOnce = 2;                      // and from shared memory
constexpr int kChunks = 2;                     // pieces of a slice copied under one barrier each
constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kGradBlocks = 3;
constexpr size_t kSharedLimit = 227 * 1024;
// Three blocks of loss with gradient on an SM: some compute while others
// exchange. At 4096 x 151936 bf16, compared in one run before the last steps,
// this took 520 us; two blocks of 80 KB 560, four of 50 KB 550 (the exchange
// costs each block about a microsecond a row), one of 152 KB 550.
constexpr size_t kSliceTarget = 74 * 1024;
constexpr int kBackThreads = 256;
constexpr int kBackWords = 4;                  // 16-byte words per thread of the backward pass

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
  int32_t* watchdog;
  uint64_t wait_limit_ns;
  bool expire;              // test hook: a wait that nothing ends
  int64_t rows;             // loss with gradient: rows and log2 of the hash table's size
  int hash_bits;
};

// 1 / sum of a row without teacher entries.
constexpr float kEmptyRow = -1.f;

// A relative error of about 2^-22, as much as the rounding of the exponent adds;
// tests hold a loss to 2^-17 of its terms.
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

// A row as 16-byte words: the row starts `phase` elements into word 0. Words
// of a block are counted from `first`; those of [lo, hi) lie in the row.
template <typename T>
struct RowWords {
  static constexpr int kPer = 16 / sizeof(T);
  const T* row;
  const uint4* words;  // word `first`, if it were whole
  int phase, vocab, first, count, lo, hi;

  __device__ __forceinline__ RowWords(const T* r, int v, int first_word, int at_most)
      : row(r), phase(static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))), vocab(v), first(first_word) {
    words = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(r) & ~uintptr_t{15}) + first;
    const int all = (phase + vocab + kPer - 1) / kPer;
    count = max(0, min(at_most, all - first));
    lo = first == 0 && phase > 0;
    hi = max(lo, count - (first + count == all && (phase + vocab) % kPer != 0));
  }
  __device__ __forceinline__ int element(int word) const { return (first + word) * kPer - phase; }
  __device__ __forceinline__ bool holds(int e) const {
    return e + phase >= first * kPer && e + phase < (first + count) * kPer;
  }
  // Word with elements outside the row; they read as -inf.
  __device__ __forceinline__ uint4 load_partial(int word) const {
    uint4 r;
    T* v = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = element(word) + i;
      v[i] = e >= 0 && e < vocab ? row[e] : from_float<T>(-INFINITY);
    }
    return r;
  }
  // The same word of another row (a gradient's), which may start elsewhere in its words.
  __device__ __forceinline__ void store(T* to, bool same_phase, int word, const uint4& r) const {
    if (same_phase && word >= lo && word < hi) {
      *reinterpret_cast<uint4*>(to + element(word)) = r;
      return;
    }
    const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = element(word) + i;
      if (e >= 0 && e < vocab) to[e] = v[i];
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

// Two fp32 lanes in one register pair.
struct Pair {
  uint64_t v;
  __device__ __forceinline__ Pair() {}
  __device__ __forceinline__ explicit Pair(float x) : Pair(x, x) {}
  __device__ __forceinline__ Pair(float lo, float hi) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  }
  __device__ __forceinline__ void split(float& lo, float& hi) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
  }
};
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Pair exp2_fast(Pair a) {
  float lo, hi;
  a.split(lo, hi);
  return Pair(exp2_fast(lo), exp2_fast(hi));
}

// Largest element of a word (NaN only if all are).
template <typename T>
__device__ __forceinline__ float word_max(const uint4& r) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(&r);
    const T2 top = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float2 f = unpack2<T>(*reinterpret_cast<const uint32_t*>(&top));
    return fmaxf(f.x, f.y);
  }
}

template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& r, Pair* v) {
  float f[16 / sizeof(T)];
  unpack_word<T>(r, f);
#pragma unroll
  for (int i = 0; i < static_cast<int>(8 / sizeof(T)); ++i) v[i] = Pair(f[2 * i], f[2 * i + 1]);
}

// 2^((s - m) c) for a maximum m. The difference is formed first: s c - m c
// would be one instruction less, but overflows where a row is masked with the
// type's lowest value throughout. While nothing above -inf was seen m counts
// as 0, so that -inf terms give 0.
struct Exponent {
  float shift;
  __device__ __forceinline__ explicit Exponent(float m) : shift(m == -INFINITY ? 0.f : -m) {}
  __device__ __forceinline__ float operator()(float s, float c) const { return exp2_fast((s + shift) * c); }
  __device__ __forceinline__ Pair operator()(Pair s, float c) const {
    return exp2_fast(mul2(add2(s, Pair(shift)), Pair(c)));
  }
};

// Running maximum m and sum of 2^((s - m) c) of one thread.
struct Softmax {
  float m = -INFINITY;
  Exponent power{-INFINITY};
  Pair sums{0.f};

  // N words at once: one look at the maximum, and their exponents do not wait for one another.
  template <typename T, int N>
  __device__ __forceinline__ void add(const uint4* words, float c) {
    constexpr int kPairs = 8 / sizeof(T);
    float top = word_max<T>(words[0]);
#pragma unroll
    for (int n = 1; n < N; ++n) top = fmaxf(top, word_max<T>(words[n]));
    if (top > m) {
      const Exponent next(top);
      if (m != -INFINITY) sums = mul2(sums, Pair(next(m, c)));
      m = top;
      power = next;
    }
    Pair part[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      Pair v[kPairs];
      unpack_pairs<T>(words[n], v);
      part[n] = power(v[0], c);
#pragma unroll
      for (int i = 1; i < kPairs; ++i) part[n] = add2(part[n], power(v[i], c));
    }
#pragma unroll
    for (int n = 1; n < N; ++n) part[0] = add2(part[0], part[n]);
    sums = add2(sums, part[0]);
  }
  __device__ __forceinline__ float2 pair() const {
    float lo, hi;
    sums.split(lo, hi);
    return make_float2(m, lo + hi);
  }
};

// Joins the lanes' (max, sum) over groups of WIDTH lanes; every lane gets it.
template <int WIDTH>
__device__ __forceinline__ float2 join_lanes(float2 mine, float c) {
  float m = mine.x;
#pragma unroll
  for (int step = WIDTH / 2; step > 0; step /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, step));
  float sum = mine.x == -INFINITY ? mine.y : mine.y * Exponent(m)(mine.x, c);
#pragma unroll
  for (int step = WIDTH / 2; step > 0; step /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, step);
  return make_float2(m, sum);
}
// Joins pairs[0 .. count), count <= 32, read one a lane.
__device__ __forceinline__ float2 join_parts(const float2* pairs, int count, int lane, float c) {
  return join_lanes<32>(lane < count ? pairs[lane] : make_float2(-INFINITY, 0.f), c);
}

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
  float p;      // teacher probability
  float column; // that of all entries with the same index (loss with gradient)
  float s;      // student logit
  int at;       // index, -1: no entry
};

struct TeacherSoftmax {
  float max, inv;
  float entropy;  // -sum p ln p
  bool stray;     // an index beyond the vocabulary
  bool empty;     // no entry
};

// Fills `list` (one warp): the teacher's softmax, and the student's logits at
// the indices of this block's slice, or `everywhere`. Four entries a lane are
// on their way at a time.
template <typename T>
__device__ __forceinline__ TeacherSoftmax read_list(const DistillParams& p, int64_t row, const RowWords<T>& in,
                                                    bool everywhere, int lane, Entry* list) {
  TeacherSoftmax t{-INFINITY, 0.f, 0.f, false, true};
  for (int base = lane; base < p.top; base += 128) {
    int64_t index[4];
    Entry e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in_list = base + 32 * i < p.top;
      index[i] = in_list ? index_at(p, row, base + 32 * i) : -1;
      e[i] = Entry{in_list ? teacher_at(p, row, base + 32 * i) : 0.f, 0.f, 0.f, -1};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!is_entry(index[i], e[i].p)) continue;
      t.empty = false;
      if (index[i] >= p.vocab) {
        t.stray = true;
        continue;
      }
      e[i].at = static_cast<int>(index[i]);
      if (everywhere || in.holds(e[i].at)) e[i].s = to_float(in.row[e[i].at]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e[i].at >= 0) t.max = fmaxf(t.max, e[i].p);
      if (base + 32 * i < p.top) list[base + 32 * i] = e[i];
    }
  }
  t.max = warp_max(t.max);
  t.stray = __any_sync(0xffffffffu, t.stray);
  t.empty = __all_sync(0xffffffffu, t.empty);
  if (t.empty) return t;
  float sum = 0.f;
  for (int k = lane; k < p.top; k += 32) {
    if (list[k].at >= 0) sum += exp2_fast((list[k].p - t.max) * p.c);
  }
  sum = warp_sum(sum);
  t.inv = 1.f / sum;
  const float log_sum = logf(sum);
  for (int k = lane; k < p.top; k += 32) {
    const float x = list[k].p - t.max;
    const float prob = exp2_fast(x * p.c) * t.inv;
    if (list[k].at >= 0 && prob != 0.f) t.entropy -= prob * (x * p.inv_tau - log_sum);
    list[k].p = list[k].column = prob;
  }
  t.entropy = warp_sum(t.entropy);
  __syncwarp();
  return t;
}

// Row maximum and sum over the threads of a cluster's blocks: every thread of
// every block calls it, `mine` counts for the streaming ones. The cluster
// barrier's first phase was arrived at when the kernel started: the other
// blocks' shared memory may be written once they have started as well.
__device__ __forceinline__ float2 join_row(const Softmax& mine, float c, uint32_t rank, uint32_t ranks) {
  __shared__ float2 warps[kRowThreads / 32];
  __shared__ float2 blocks[kMaxCluster];
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < kRowThreads) {
    const float2 part = join_lanes<32>(mine.pair(), c);
    if (lane == 0) warps[threadIdx.x / 32] = part;
  }
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < 32) {
    const float2 block = join_parts(warps, kRowThreads / 32, lane, c);
    if (lane < static_cast<int>(ranks)) {
      const uint32_t to = mapa_shared(&blocks[rank], static_cast<uint32_t>(lane));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(block.x), "f"(block.y) : "memory");
    }
    __syncwarp();
  }
  cluster_sync();
  return join_parts(blocks, static_cast<int>(ranks), lane, c);
}

// The row's loss and statistics (the list warp of block 0).
__device__ __forceinline__ void write_loss(const DistillParams& p, int64_t row, const Entry* list, int lane,
                                           float2 all, float inv, const TeacherSoftmax& teacher) {
  const float log_sum = logf(all.y);
  float total = 0.f;
  for (int k = lane; k < p.top; k += 32) {
    const Entry e = list[k];
    if (e.at >= 0 && e.p != 0.f) total -= e.p * ((e.s - all.x) * p.inv_tau - log_sum);
  }
  total = warp_sum(total) - teacher.entropy;
  if (lane == 0) {
    p.loss[row] = teacher.stray ? __int_as_float(0x7fffffff) : total * p.tau * p.tau;
    p.stats[row] = make_float4(all.x, inv, teacher.max, teacher.inv);
  }
}

__device__ __forceinline__ void write_empty(const DistillParams& p, int64_t row) {
  p.loss[row] = 0.f;
  p.stats[row] = make_float4(0.f, kEmptyRow, 0.f, 0.f);
}

// The losses alone: a cluster of blocks per row streams it through registers.
// Bound by memory: 4096 rows of 151936 bf16 take 191 us (1245 MB, 6.5 TB/s),
// 509 rows 33.8 us (4.6 TB/s: the start and the last, partly filled wave cost
// more of so few rows); one row 6.0 us.
template <typename T>
__global__ void __launch_bounds__(kRowBlock, 4) distill_loss_rows(DistillParams p) {
  extern __shared__ uint4 shared[];
  __shared__ volatile int empty_row;
  Entry* list = reinterpret_cast<Entry*>(shared);
  const uint32_t rank = cluster_ctarank();
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int64_t row = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31;
  const bool lists = threadIdx.x >= kRowThreads;
  if (threadIdx.x == 0) empty_row = 0;
  __syncthreads();

  const T* logits = static_cast<const T*>(p.logits) + row * p.row_stride;
  const RowWords<T> in(logits, static_cast<int>(p.vocab), static_cast<int>(rank) * p.slice, p.slice);
  Softmax mine;
  TeacherSoftmax teacher{};
  if (lists) {
    teacher = read_list(p, row, in, rank == 0, lane, list);
    if (teacher.empty) empty_row = 1;
  } else {
    // Whole words, kUnroll at once while the next ones are on their way.
    constexpr int kStep = kUnroll * kRowThreads;
    const uint4* from = in.words + in.lo + threadIdx.x;
    const int words = in.hi - in.lo, rounds = words / kStep;
    uint4 ahead[kUnroll];
    if (rounds > 0) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) ahead[u] = from[u * kRowThreads];
    }
    for (int round = 1; round <= rounds; ++round) {
      uint4 now[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) now[u] = ahead[u];
      if (round < rounds) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) ahead[u] = from[round * kStep + u * kRowThreads];
      }
      if (empty_row) break;  // nothing of the row counts
      mine.add<T, kUnroll>(now, p.c);
    }
    for (int w = rounds * kStep + static_cast<int>(threadIdx.x); w < words; w += kRowThreads) {
      mine.add<T, 1>(in.words + in.lo + w, p.c);
    }
    if ((threadIdx.x == 0 && in.lo > 0 && in.count > 0) || (threadIdx.x == 1 && in.hi < in.count)) {
      const uint4 word = in.load_partial(threadIdx.x == 0 ? 0 : in.count - 1);
      mine.add<T, 1>(&word, p.c);
    }
    __syncwarp();
  }
  const float2 all = join_row(mine, p.c, rank, ranks);
  if (!lists || rank != 0) return;
  if (empty_row) {
    if (lane == 0) write_empty(p, row);
    return;
  }
  const float inv = teacher.stray ? __int_as_float(0x7fffffff) : 1.f / all.y;
  write_loss(p, row, list, lane, all, inv, teacher);
}

// ------------------------------------------------ loss with gradient ----

// Loss and gradient in one pass over the logits. A cluster of blocks walks
// the rows; a block keeps its slice of a row in shared memory. The streaming
// warps add the slice chunk by chunk as its bulk copies arrive, exchange
// (max, sum) with the other blocks, then turn the slice into the gradient
// chunk by chunk; a chunk they have read for the last time is refilled with
// the next row's at once. The list warp looks ahead for rows without entries
// (which are not read at all), issues the copies, and after the streaming
// warps writes the list's columns again with the teacher's part. 4096 rows of
// 151936 bf16 take 507 us (2489 MB, 4.9 TB/s): two exponentials an element
// keep their unit 56 % busy, and a row's exchange costs about a microsecond in
// which its block reads but does not write. Loss and backward pass one after
// the other take 568 us.
struct GradBarriers {
  uint64_t full[kChunks];   // the chunk's copy has arrived
  uint64_t empty[kChunks];  // every streaming warp has read the chunk for the last time
  uint64_t joined;          // every streaming warp's pair is there, and the list has been read
  uint64_t exchanged[2];    // the pairs of all blocks, of alternate rows
  uint64_t never;
};

enum RowState : int { kEmptyList = 1, kStrayIndex = 2 };

// Sums the probabilities of entries that name the same column of this block's
// slice: a hash table of indices, at most half full, finds them (one warp).
template <typename T>
__device__ __forceinline__ void join_columns(const DistillParams& p, const RowWords<T>& in, Entry* list, int* table,
                                             int lane) {
  constexpr int kTwice = static_cast<int>(0x80000000u);
  const int size = 1 << p.hash_bits;
  for (int i = lane; i < size; i += 32) table[i] = -1;
  __syncwarp();
  auto first_slot = [&](int at) {
    return static_cast<int>((static_cast<uint32_t>(at) * 2654435761u) >> (32 - p.hash_bits));
  };
  bool found = false;
  for (int k = lane; k < p.top; k += 32) {
    const int at = list[k].at;
    if (at < 0 || !in.holds(at)) continue;
    for (int slot = first_slot(at);; slot = (slot + 1) & (size - 1)) {
      const int old = atomicCAS(&table[slot], -1, at);
      if (old == -1) break;
      if ((old & ~kTwice) == at) {
        atomicOr(&table[slot], kTwice);
        found = true;
        break;
      }
    }
  }
  if (!__any_sync(0xffffffffu, found)) return;
  __syncwarp();
  for (int k = lane; k < p.top; k += 32) {
    const int at = list[k].at;
    if (at < 0 || !in.holds(at)) continue;
    int slot = first_slot(at);
    while ((table[slot] & ~kTwice) != at) slot = (slot + 1) & (size - 1);
    if ((table[slot] & kTwice) == 0) continue;
    float column = 0.f;
    for (int j = 0; j < p.top; ++j) {
      if (list[j].at == at) column += list[j].p;
    }
    list[k].column = column;
  }
  __syncwarp();
}

template <typename T>
__global__ void __launch_bounds__(kRowBlock, kGradBlocks) distill_grad_rows(DistillParams p) {
  extern __shared__ uint4 shared[];
  __shared__ GradBarriers bars;
  __shared__ int states[2];
  __shared__ float upstream[2];
  __shared__ int32_t abort, cluster_abort;
  __shared__ float2 warp_parts[kRowThreads / 32];
  __shared__ float2 parts[2][kMaxCluster];
  constexpr int kPer = 16 / sizeof(T);
  Entry* lists_of[2] = {reinterpret_cast<Entry*>(shared), reinterpret_cast<Entry*>(shared + p.top)};
  int* table = reinterpret_cast<int*>(shared + 2 * p.top);
  uint4* stage = shared + 2 * p.top + (1 << p.hash_bits) / 4;
  const uint32_t rank = cluster_ctarank();
  uint32_t ranks;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int64_t clusters = gridDim.x / ranks;
  const int64_t first_row = blockIdx.x / ranks;
  const int tid = threadIdx.x, lane = tid & 31;
  const bool lists = tid >= kRowThreads;
  const uint32_t exchange_bytes = ranks * sizeof(float2);
  if (tid == kRowThreads) {
    for (int i = 0; i < kChunks; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], kRowThreads / 32);
    }
    mbar_init(&bars.joined, kRowThreads / 32 + 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.exchanged[i], 1);
      mbar_arrive_expect_tx(&bars.exchanged[i], exchange_bytes);
    }
    mbar_init(&bars.never, 1);
    fence_barrier_init();
    abort = cluster_abort = 0;
  }
  cluster_sync();

  // False for the whole warp once a wait of the block has run out. Every wait
  // is of this kind, so the warps then leave their loops one after the other
  // and meet at the cluster's last barrier, behind which all of the cluster's
  // rows become NaN.
  auto wait = [&](uint64_t* bar, uint32_t phase) {
    return __all_sync(0xffffffffu, mbar_wait(bar, phase, kWaitDistill, &abort, p.watchdog, p.wait_limit_ns)) != 0;
  };
  auto words_of = [&](int64_t row) {
    return RowWords<T>(static_cast<const T*>(p.logits) + row * p.row_stride, static_cast<int>(p.vocab),
                       static_cast<int>(rank) * p.slice, p.slice);
  };
  // All rows use chunks of the same size: a slot is refilled by the next row's.
  const int chunk = (p.slice + kChunks * kRowThreads - 1) / (kChunks * kRowThreads) * kRowThreads;
  auto row_softmax = [&](uint32_t exchange) {
    return join_parts(parts[exchange & 1], static_cast<int>(ranks), lane, p.c);
  };

  uint32_t exchange = 0;  // rows with entries so far
  if (lists) {
    // A row's list is read while the row before it is worked on. (The row's
    // logits are still there: no block replaces them with the gradient before
    // this one has sent its pair for the row.)
    auto prepare = [&](int64_t row, uint32_t turn) {
      Entry* list = lists_of[turn & 1];
      const RowWords<T> in = words_of(row);
      const TeacherSoftmax t = read_list(p, row, in, rank == 0, lane, list);
      if (!t.empty) join_columns(p, in, list, table, lane);
      if (lane == 0) {
        states[turn & 1] = (t.empty ? kEmptyList : 0) | (t.stray ? kStrayIndex : 0);
        upstream[turn & 1] = p.upstream != nullptr ? p.upstream[row * p.upstream_stride] : 1.f;
      }
      __syncwarp();
      return t;
    };
    uint32_t issued = 0;  // parity of each chunk's latest copy
    auto issue = [&](const RowWords<T>& in, bool read, int i, uint32_t turn) {
      issued = (issued & ~(1u << i)) | (turn & 1) << i;
      if (lane != 0) return;
      const int from = max(in.lo, i * chunk), to = min(in.hi, (i + 1) * chunk);
      if (read && in.count > 0) {
        if (in.lo > 0 && i == 0) stage[0] = in.load_partial(0);
        if (in.hi < in.count && (in.count - 1) / chunk == i) stage[in.count - 1] = in.load_partial(in.count - 1);
      }
      if (read && from < to) {
        const uint32_t bytes = static_cast<uint32_t>(to - from) * 16;
        // The chunk's last row was read, and words at its ends written, by
        // ordinary accesses; rows start elsewhere in their words.
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(&bars.full[i], bytes);
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(stage + from)),
            "l"(in.words + from), "r"(bytes), "r"(smem_u32(&bars.full[i]))
            : "memory");
      } else {
        mbar_arrive(&bars.full[i]);
      }
    };
    TeacherSoftmax teacher{};
    if (first_row < p.rows) {
      teacher = prepare(first_row, 0);
      const RowWords<T> in = words_of(first_row);
      for (int i = 0; i < kChunks; ++i) issue(in, !teacher.empty, i, 0);
      __syncwarp();
    }
    uint32_t turn = 0;
    for (int64_t row = first_row; row < p.rows; row += clusters, ++turn) {
      if (p.expire && !wait(&bars.never, 0)) break;
      const Entry* list = lists_of[turn & 1];
      const bool some = !teacher.empty;
      const RowWords<T> in = words_of(row);
      T* grad = static_cast<T*>(p.grad) + row * p.grad_stride;
      if (some && lane == 0) mbar_arrive(&bars.joined);
      const float a = p.tau * upstream[turn & 1];
      TeacherSoftmax next_teacher{};
      const bool more = row + clusters < p.rows;
      if (more) next_teacher = prepare(row + clusters, turn + 1);
      float2 all{0.f, 0.f};
      float inv = 0.f;
      if (some) {
        if (!wait(&bars.exchanged[exchange & 1], exchange >> 1 & 1)) break;
        all = row_softmax(exchange);
        ++exchange;
        inv = teacher.stray ? __int_as_float(0x7fffffff) : 1.f / all.y;
        if (rank == 0) write_loss(p, row, list, lane, all, inv, teacher);
      } else if (rank == 0 && lane == 0) {
        write_empty(p, row);
      }
      const RowWords<T> next = words_of(more ? row + clusters : row);
      bool drained = true;
      for (int i = 0; i < kChunks && drained; ++i) {
        drained = wait(&bars.empty[i], turn & 1);
        if (more && drained) issue(next, !next_teacher.empty, i, turn + 1);
      }
      __syncwarp();
      if (!drained) break;
      if (some) {
        for (int k = lane; k < p.top; k += 32) {
          const Entry e = list[k];
          if (e.at < 0 || !in.holds(e.at)) continue;
          grad[e.at] = from_float<T>(a * (Exponent(all.x)(e.s, p.c) * inv - e.column));
        }
        __syncwarp();
      }
      teacher = next_teacher;
    }
    if (abort != 0 && lane == 0) {  // leave no copy behind in flight
      for (int i = 0; i < kChunks; ++i) mbar_drain(&bars.full[i], issued >> i & 1);
    }
  } else {
    uint32_t turn = 0;
    for (int64_t row = first_row; row < p.rows; row += clusters, ++turn) {
      const RowWords<T> in = words_of(row);
      T* grad = static_cast<T*>(p.grad) + row * p.grad_stride;
      const bool same_phase = static_cast<int>((reinterpret_cast<uintptr_t>(grad) & 15) / sizeof(T)) == in.phase;
      if (!wait(&bars.full[0], turn & 1)) break;
      const int state = states[turn & 1];
      const float a = p.tau * upstream[turn & 1];
      bool arrived = true;
      if (state & kEmptyList) {
        for (int i = 1; i < kChunks && arrived; ++i) arrived = wait(&bars.full[i], turn & 1);
        if (!arrived) break;
        for (int w = tid; w < in.count; w += kRowThreads) in.store(grad, same_phase, w, make_uint4(0, 0, 0, 0));
        __syncwarp();
        if (lane == 0) {
          for (int i = 0; i < kChunks; ++i) mbar_arrive(&bars.empty[i]);
        }
        continue;
      }
      Softmax mine;
      for (int i = 0; i < kChunks && arrived; ++i) {
        if (i > 0) arrived = wait(&bars.full[i], turn & 1);
        const int to = min(in.count, (i + 1) * chunk);
        int w = i * chunk + tid;
        for (; w + (kAtOnce - 1) * kRowThreads < to; w += kAtOnce * kRowThreads) {
          uint4 words[kAtOnce];
#pragma unroll
          for (int u = 0; u < kAtOnce; ++u) words[u] = stage[w + u * kRowThreads];
          mine.add<T, kAtOnce>(words, p.c);
        }
        for (; w < to; w += kRowThreads) mine.add<T, 1>(stage + w, p.c);
      }
      __syncwarp();
      if (!arrived) break;
      const float2 part = join_lanes<32>(mine.pair(), p.c);
      if (lane == 0) {
        warp_parts[tid / 32] = part;
        mbar_arrive(&bars.joined);
      }
      if (tid < 32) {
        if (!wait(&bars.joined, exchange & 1)) break;
        const float2 block = join_parts(warp_parts, kRowThreads / 32, lane, p.c);
        if (lane < static_cast<int>(ranks)) {  // one lane per block of the cluster
          asm volatile(
              "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                  mapa_shared(&parts[exchange & 1][rank], static_cast<uint32_t>(lane))),
              "f"(block.x), "f"(block.y),
              "r"(mapa_shared(&bars.exchanged[exchange & 1], static_cast<uint32_t>(lane)))
              : "memory");
        }
        __syncwarp();
      }
      if (!wait(&bars.exchanged[exchange & 1], exchange >> 1 & 1)) break;
      // For the row after the next one: no block sends its pair before this
      // one has sent the next row's.
      if (tid == 0) mbar_arrive_expect_tx(&bars.exchanged[exchange & 1], exchange_bytes);
      const float2 all = row_softmax(exchange);
      ++exchange;
      const float inv = (state & kStrayIndex) ? __int_as_float(0x7fffffff) : 1.f / all.y;
      const Exponent power(all.x);
      const Pair scaled(a * inv);
      auto gradient = [&](const uint4& word) {
        Pair v[kPer / 2];
        unpack_pairs<T>(word, v);
        float f[kPer];
#pragma unroll
        for (int e = 0; e < kPer / 2; ++e) mul2(power(v[e], p.c), scaled).split(f[2 * e], f[2 * e + 1]);
        return pack_word<T>(f);
      };
      for (int i = 0; i < kChunks; ++i) {
        const int from = i * chunk, to = min(in.count, (i + 1) * chunk);
        if (same_phase) {
          uint4* out = reinterpret_cast<uint4*>(grad + in.element(0));  // only whole words of it are written
          const int end = min(in.hi, to);
          int w = max(in.lo, from) + tid;
          for (; w + (kAtOnce - 1) * kRowThreads < end; w += kAtOnce * kRowThreads) {
            uint4 words[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) words[u] = gradient(stage[w + u * kRowThreads]);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) out[w + u * kRowThreads] = words[u];
          }
          for (; w < end; w += kRowThreads) out[w] = gradient(stage[w]);
          if (tid == 0 && from < in.lo && from < to) in.store(grad, false, 0, gradient(stage[0]));
          if (tid == 0 && in.hi >= from && in.hi < to) in.store(grad, false, in.hi, gradient(stage[in.hi]));
        } else {
          for (int w = from + tid; w < to; w += kRowThreads) in.store(grad, false, w, gradient(stage[w]));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.empty[i]);
      }
    }
  }
  __syncwarp();
  if (abort != 0 && lane < static_cast<int>(ranks)) {
    const uint32_t to = mapa_shared(&cluster_abort, static_cast<uint32_t>(lane));
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(1) : "memory");
  }
  cluster_sync();  // the other blocks may still be sending their pairs
  if (cluster_abort == 0) return;
  const float nan = __int_as_float(0x7fffffff);
  float nans[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) nans[i] = nan;
  for (int64_t row = first_row; row < p.rows; row += clusters) {
    const RowWords<T> in = words_of(row);
    T* grad = static_cast<T*>(p.grad) + row * p.grad_stride;
    for (int w = tid; w < in.count; w += kRowBlock) in.store(grad, false, w, pack_word<T>(nans));
    if (rank == 0 && tid == 0) {
      p.loss[row] = nan;
      p.stats[row] = make_float4(nan, nan, nan, nan);
    }
  }
}

// The gradient from the row statistics: one read, one write, blocks of a row
// independent of each other. A warp of its own collects the block's entries of
// the list meanwhile (their logits before they are overwritten: the gradient
// may replace them) and writes their columns last. Bound by memory: 4096 rows
// of 151936 bf16 take 377 us (2489 MB, 6.6 TB/s).
struct BackEntry {
  float s, p;
  int at;
};

template <typename T>
__global__ void __launch_bounds__(kBackThreads + 32, 6) distill_backward(DistillParams p) {
  extern __shared__ uint4 shared[];
  constexpr int kPer = 16 / sizeof(T);
  constexpr int kWords = kBackThreads * kBackWords;
  __shared__ uint32_t seen[(kWords * kPer + 31) / 32];
  BackEntry* list = reinterpret_cast<BackEntry*>(shared);
  const int64_t row = blockIdx.x / p.chunks;
  const T* logits = static_cast<const T*>(p.logits) + row * p.row_stride;
  T* grad = static_cast<T*>(p.grad) + row * p.grad_stride;
  const RowWords<T> in(logits, static_cast<int>(p.vocab), static_cast<int>(blockIdx.x % p.chunks) * kWords, kWords);
  const int tid = threadIdx.x, lane = tid & 31;

  if (tid < kBackThreads) {
    uint4 raw[kBackWords];
#pragma unroll
    for (int u = 0; u < kBackWords; ++u) {
      const int w = tid + u * kBackThreads;
      if (w >= in.lo && w < in.hi) raw[u] = in.words[w];
      else if (w < in.count) raw[u] = in.load_partial(w);
    }
    const float4 stats = p.stats[row];
    float a = p.tau;
    if (p.upstream != nullptr) a *= p.upstream[row * p.upstream_stride];
    if (p.upstream_scale != nullptr) a *= *p.upstream_scale;
    const Exponent power(stats.x);
    const Pair scaled(a * stats.y);
    const bool same_phase = static_cast<int>((reinterpret_cast<uintptr_t>(grad) & 15) / sizeof(T)) == in.phase;
    __syncthreads();  // the list's logits have been read
#pragma unroll
    for (int u = 0; u < kBackWords; ++u) {
      const int w = tid + u * kBackThreads;
      if (w >= in.count) continue;
      Pair v[kPer / 2];
      unpack_pairs<T>(raw[u], v);
      float f[kPer];
#pragma unroll
      for (int i = 0; i < kPer / 2; ++i) mul2(power(v[i], p.c), scaled).split(f[2 * i], f[2 * i + 1]);
      in.store(grad, same_phase, w, stats.y == kEmptyRow ? make_uint4(0, 0, 0, 0) : pack_word<T>(f));
    }
    __syncthreads();
    return;
  }

  for (int i = lane; i < static_cast<int>(sizeof(seen) / 4); i += 32) seen[i] = 0;
  __syncwarp();
  const float4 stats = p.stats[row];
  int count = 0;
  bool shared_column = false;
  for (int base = 0; base < p.top && stats.y != kEmptyRow; base += 32) {
    BackEntry e{0.f, 0.f, -1};
    if (base + lane < p.top) {
      const int64_t index = index_at(p, row, base + lane);
      const float t = teacher_at(p, row, base + lane);
      if (is_entry(index, t) && index < p.vocab) {
        const int local = static_cast<int>(index) + in.phase - in.first * kPer;
        if (in.holds(static_cast<int>(index))) {
          e = BackEntry{to_float(logits[index]), exp2_fast((t - stats.z) * p.c) * stats.w, static_cast<int>(index)};
          if (atomicOr(&seen[local / 32], 1u << (local % 32)) >> (local % 32) & 1u) shared_column = true;
        }
      }
    }
    const uint32_t mask = __ballot_sync(0xffffffffu, e.at >= 0);
    if (e.at >= 0) list[count + __popc(mask & ((1u << lane) - 1))] = e;
    count += __popc(mask);
  }
  shared_column = __any_sync(0xffffffffu, shared_column);
  __syncthreads();
  float a = p.tau;
  if (p.upstream != nullptr) a *= p.upstream[row * p.upstream_stride];
  if (p.upstream_scale != nullptr) a *= *p.upstream_scale;
  __syncthreads();
  for (int k = lane; k < count; k += 32) {
    const BackEntry e = list[k];
    float prob = e.p;
    if (shared_column) {  // every entry of a column writes the same sum
      prob = 0.f;
      for (int j = 0; j < count; ++j) {
        if (list[j].at == e.at) prob += list[j].p;
      }
    }
    grad[e.at] = from_float<T>(a * (Exponent(stats.x)(e.s, p.c) * stats.y - prob));
  }
}

// out[0] = sum or mean of the losses over the rows that have entries (0 when
// none has), out[1] = what a row's loss was multiplied with. One block, fixed
// order: 2.4 us for 333 rows.
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

int hash_bits(int top) {
  int bits = 6;
  while ((1 << bits) < 2 * top) ++bits;
  return bits;
}

size_t shared_bytes(int64_t vocab, int dtype, int top, int cluster, bool grad) {
  return static_cast<size_t>(top) * sizeof(Entry) * (grad ? 2 : 1) +
         (grad ? (sizeof(int) << hash_bits(top)) + static_cast<size_t>(ceil_div(max_words(vocab, dtype), cluster)) * 16 : 0);
}

// Blocks per row: the gradient's slice should let three blocks share an SM
// (and must fit one); beyond that, few rows are split until the blocks fill
// the SMs. 0: a row does not fit a cluster.
int cluster_size(int64_t rows, int64_t vocab, int dtype, int top, bool grad) {
  int cluster = 1;
  while (cluster < kMaxCluster && grad && shared_bytes(vocab, dtype, top, cluster, grad) > kSliceTarget) ++cluster;
  if (shared_bytes(vocab, dtype, top, cluster, grad) > kSharedLimit - 2048) return 0;
  while (cluster < kMaxCluster && rows * cluster < 4 * sm_count() && max_words(vocab, dtype) / cluster > 2 * kRowThreads) {
    cluster = std::min(2 * cluster, kMaxCluster);
  }
  return cluster;
}

template <typename T, bool GRAD>
int launch_rows(DistillParams p, int64_t rows, int cluster, size_t shared, cudaStream_t stream) {
  void (*kernel)(DistillParams) = GRAD ? distill_grad_rows<T> : distill_loss_rows<T>;
  int64_t clusters = rows;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
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
  if (GRAD) {
    // As many clusters as are resident at a time walk the rows. Asked once
    // for each device, cluster size and amount of shared memory in use.
    struct Resident {
      int device = -1, cluster = 0, clusters = 0;
      size_t shared = 0;
    };
    static thread_local Resident last;
    int device = 0;
    SDC_CUDA_CHECK(cudaGetDevice(&device));
    if (last.device != device || last.cluster != cluster || last.shared != shared) {
      const int rc = allow_shared(reinterpret_cast<const void*>(kernel), static_cast<int>(shared));
      if (rc != SDC_OK) return rc;
      config.gridDim = dim3(static_cast<unsigned>(cluster));
      SDC_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&last.clusters, kernel, &config));
      last.device = device, last.cluster = cluster, last.shared = shared;
    }
    clusters = std::min<int64_t>(rows, std::max(last.clusters, 1));
    config.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
  }
  SDC_CUDA_CHECK(cudaLaunchKernelEx(&config, kernel, p));
  return SDC_OK;
}

template <bool GRAD>
int run_rows(DistillParams p, int dtype, int64_t rows, int cluster, cudaStream_t stream) {
  SDC_REQUIRE(rows <= INT_MAX / cluster, "distillation has too many rows for one launch");
  p.slice = static_cast<int>(ceil_div(max_words(p.vocab, dtype), cluster));
  p.rows = rows;
  p.hash_bits = hash_bits(p.top);
  p.watchdog = watchdog_ptr();
  if (p.watchdog == nullptr) return fail(SDC_ERR_CUDA, "distillation has no watchdog word on this device");
  const WatchdogSettings watch = watchdog_settings();
  p.wait_limit_ns = watch.wait_limit_ns;
  p.expire = watch.pace_extra > 0;
  const size_t shared = shared_bytes(p.vocab, dtype, p.top, cluster, GRAD);
  if (dtype == kF32) return launch_rows<float, GRAD>(p, rows, cluster, shared, stream);
  if (dtype == kBF16) return launch_rows<__nv_bfloat16, GRAD>(p, rows, cluster, shared, stream);
  return launch_rows<__half, GRAD>(p, rows, cluster, shared, stream);
}

int run_backward(DistillParams p, int dtype, int64_t rows, cudaStream_t stream) {
  p.chunks = static_cast<int>(ceil_div(max_words(p.vocab, dtype), kBackThreads * kBackWords));
  SDC_REQUIRE(rows <= INT_MAX / p.chunks, "distillation has too many rows for one launch");
  const unsigned grid = static_cast<unsigned>(rows * p.chunks);
  const size_t shared = static_cast<size_t>(p.top) * sizeof(BackEntry);
  if (dtype == kF32) distill_backward<float><<<grid, kBackThreads + 32, shared, stream>>>(p);
  else if (dtype == kBF16) distill_backward<__nv_bfloat16><<<grid, kBackThreads + 32, shared, stream>>>(p);
  else distill_backward<__half><<<grid, kBackThreads + 32, shared, stream>>>(p);
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
