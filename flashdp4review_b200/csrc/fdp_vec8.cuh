// Eight adjacent elements as one (16-bit types) or two (fp32) 16-byte vectors: the unit of the channels-last and elementwise
// kernels, whatever the type, because the keep-mask of the dropout is drawn for eight elements at a time.
#pragma once
#include "fdp_async.cuh"
#include "fdp_common.cuh"

namespace fdp {

template <typename T> struct Vec8 { uint4 v[sizeof(T) / 2]; };
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T>& r, float f[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) unpack16<T>(r.v[i], f + i * (16 / sizeof(T)));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float f[8]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = pack16<T>(f + i * (16 / sizeof(T)));
}

// copies of 16 bytes into shared memory that the thread waits for by itself, all but its N newest groups of them
__device__ __forceinline__ void copy_async16(void* shared, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(shared)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace fdp
