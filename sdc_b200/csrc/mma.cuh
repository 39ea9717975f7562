// Copies into shared memory that every thread can make on its own, and
// warp-level matrix instructions for products of 16 rows (16-bit operands from
// shared memory, fp32 accumulators in registers): the tensor memory's
// instructions take 64 rows at least, and so few rows wait for their weights
// whatever multiplies them.
#pragma once

#include "layers.cuh"

namespace sdc {

// Four 8x8 matrices of 16-bit elements; lane l gives the shared address of
// row l % 8 of matrix l / 8.
__device__ __forceinline__ void ldmatrix_x4(uint32_t* r, uint32_t row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(row));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t* r, uint32_t row) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(row));
}

// d[16 x 8] += a[16 x 16] b[16 x 8].
template <typename T>
__device__ __forceinline__ void mma_16816(float* d, const uint32_t* a, const uint32_t* b);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float* d, const uint32_t* a, const uint32_t* b) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float* d, const uint32_t* a, const uint32_t* b) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// 16 bytes from global to shared memory, or zeros (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t shared, const void* global, bool copied = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared), "l"(global), "r"(copied ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Eight elements from global to shared memory, zeros beyond `valid`. FAST:
// the source is 16-byte aligned and whole or absent, and the copy runs on its
// own; else one by one. Either way visible after cp_async_wait and a barrier.
template <typename T, bool FAST>
__device__ __forceinline__ void copy8(uint32_t shared, const T* global, int valid) {
  if constexpr (FAST) {
    cp_async16(shared, global, valid > 0);
  } else {
    uint4 w = make_uint4(0, 0, 0, 0);
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < valid) e[i] = global[i];
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(shared), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                 : "memory");
  }
}

// A float of another block's shared memory (cluster address from mapa_shared).
__device__ __forceinline__ float load_cluster_f32(uint32_t address) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
  return v;
}

}  // namespace sdc
