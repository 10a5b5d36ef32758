// Dropout without a stored mask: y = keep * x / (1 - p) (+ residual), the mask drawn from the element's number.
// HBM-bound: one read and one write an element (and the residual's read); the backward is the same kernel on the
// gradient.  A kept infinity or NaN stays what it is, a dropped one becomes 0 (the mask selects, it does not multiply).
#include "fdp_dropout.cuh"
#include "fdp_kernels.h"
#include "fdp_vec8.cuh"

namespace fdp {

// Three blocks of 256 threads an SM: with four, held to 64 registers, the keys of the rounds are fetched again in every
// turn (134 M elements bf16: 97 us against 94), with five and six registers spill (114, 137).
constexpr int DROP_THREADS = 256, DROP_PER_SM = 3;

// the m elements (1 to 8) from number 8 g on, one by one
template <typename T, bool RES>
__device__ __forceinline__ void dropout_some(const T* x, const T* residual, T* y, uint64_t g, int m, const DropKey& key, uint32_t step) {
  const Draw d = draw8(key, step, g);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e < m) {
      float v = draw_keeps(d.w[e / 2], d.bound, e & 1) ? to_f32<T>(x[g * 8 + e]) * key.scale : 0.f;
      if (RES) v += to_f32<T>(residual[g * 8 + e]);
      y[g * 8 + e] = from_f32<T>(v);
    }
  }
}
// A thread's next D groups are copied (cp.async) into slots of shared memory of its own, which takes no registers: 148 x 768
// threads have 64 to 128 bytes each in flight.  x, residual and y may be one buffer: an element is read before it is
// written, by the same thread.
//
// 134 M elements bf16: 94 to 98 us, 82 at the speed of a copy; 124 instructions a group of eight, 64 of them on the integer
// pipe, which is 65% busy.  (Two groups a thread loaded into registers, 76 of them: 119.)
template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(DROP_THREADS, DROP_PER_SM) dropout_kernel(const T* x, const T* residual, T* y, uint64_t n, const __grid_constant__ DropKey key) {
  constexpr int PARTS = sizeof(T) / 2, COPIES = PARTS * (RES ? 2 : 1), D = COPIES == 1 ? 4 : COPIES == 2 ? 3 : 2;
  const uint32_t step = drop_step(key);
  const uint64_t full = VEC ? n / 8 : 0, groups = (n + 7) / 8, stride = static_cast<uint64_t>(gridDim.x) * DROP_THREADS;
  uint64_t g = static_cast<uint64_t>(blockIdx.x) * DROP_THREADS + threadIdx.x;
  if constexpr (VEC) {
    __shared__ uint4 ring[D][COPIES][DROP_THREADS];
    // a thread's groups, counted in 32 bits (64-bit comparisons for each copy and each turn: 4 us of 134 M elements)
    int todo = g < full ? static_cast<int>((full - g + stride - 1) / stride) : 0, ahead = todo;
    const T* from[2] = {x + g * 8, RES ? residual + g * 8 : x};
    T* to = y + g * 8;
    auto copy = [&](int slot) {
      if (ahead > 0) {
#pragma unroll
        for (int c = 0; c < COPIES; ++c) copy_async16(&ring[slot][c][threadIdx.x], from[c / PARTS] + (c % PARTS) * (16 / sizeof(T)));
        from[0] += stride * 8;
        if (RES) from[1] += stride * 8;
        --ahead;
      }
      copy_commit();
    };
#pragma unroll
    for (int a = 0; a < D; ++a) copy(a);
    for (int slot = 0; todo > 0; --todo, g += stride) {
      copy_wait<D - 1>();
      Vec8<T> a, b;
#pragma unroll
      for (int c = 0; c < COPIES; ++c) (c < PARTS ? a : b).v[c % PARTS] = ring[slot][c][threadIdx.x];
      float f[8], r[8];
      unpack8(a, f);
      drop_v<8>(key, step, g * 8, f);
      if (RES) {
        unpack8(b, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += r[e];
      }
      copy(slot);
      store8(to, f);
      to += stride * 8;
      slot = slot + 1 == D ? 0 : slot + 1;
    }
  }
  for (; g < groups; g += stride) dropout_some<T, RES>(x, residual, y, g, n - g * 8 < 8 ? static_cast<int>(n - g * 8) : 8, key, step);
}

template <typename T>
static void dropout_typed(const void* x, const void* residual, void* y, size_t n, const DropKey& key, cudaStream_t s) {
  const bool vec = aligned16(x) && aligned16(y) && (residual == nullptr || aligned16(residual));
  const size_t blocks = ((n + 7) / 8 + DROP_THREADS - 1) / DROP_THREADS;
  const unsigned grid = static_cast<unsigned>(blocks < 148 * DROP_PER_SM ? blocks : 148 * DROP_PER_SM);
  const T *xt = static_cast<const T*>(x), *rt = static_cast<const T*>(residual);
  T* yt = static_cast<T*>(y);
  if (residual != nullptr) {
    if (vec) dropout_kernel<T, true, true><<<grid, 256, 0, s>>>(xt, rt, yt, n, key);
    else dropout_kernel<T, false, true><<<grid, 256, 0, s>>>(xt, rt, yt, n, key);
  } else {
    if (vec) dropout_kernel<T, true, false><<<grid, 256, 0, s>>>(xt, rt, yt, n, key);
    else dropout_kernel<T, false, false><<<grid, 256, 0, s>>>(xt, rt, yt, n, key);
  }
  note_launch();
}

void dropout(const void* x, const void* residual, void* y, size_t n, int dt, const fdp_dropout_params* p, cudaStream_t s) {
  const DropKey key = make_drop_key(p);
  if (dt == FDP_F32) dropout_typed<float>(x, residual, y, n, key, s);
  else if (dt == FDP_BF16) dropout_typed<__nv_bfloat16>(x, residual, y, n, key, s);
  else dropout_typed<__half>(x, residual, y, n, key, s);
}

}  // namespace fdp
