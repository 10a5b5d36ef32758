// Dropout without a stored mask: y = keep * x / (1 - p) (+ residual), the mask drawn from the element's number.
// HBM-bound: one read and one write an element (and the residual's read); the backward is the same kernel on the
// gradient.  A kept infinity or NaN stays what it is, a dropped one becomes 0 (the mask selects, it does not multiply).
#include "fdp_dropout.cuh"
#include "fdp_kernels.h"
#include "fdp_vec8.cuh"

namespace fdp {

// one group of eight elements from number 8 g on
template <typename T, bool VEC, bool RES>
__device__ __forceinline__ void dropout_group(const Vec8<T>& a, const Vec8<T>& b, const T* x, const T* residual, T* y, uint64_t g, uint64_t n, const DropKey& key,
                                              uint32_t step) {
  const uint64_t i = g * 8;
  if (VEC && i + 8 <= n) {
    float f[8], r[8];
    unpack8(a, f);
    drop_v<8>(key, step, i, f);
    if (RES) {
      unpack8(b, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += r[e];
    }
    store8(y + i, f);
  } else {
    const Draw d = draw8(key, step, g);
    const int m = n - i < 8 ? static_cast<int>(n - i) : 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e < m) {
        float v = (e & 1 ? d.w[e / 2] : d.w[e / 2] << 16) > d.bound ? to_f32<T>(x[i + e]) * key.scale : 0.f;
        if (RES) v += to_f32<T>(residual[i + e]);
        y[i + e] = from_f32<T>(v);
      }
    }
  }
}
// Two groups a thread at a time, both loaded before either's numbers are drawn: 2048 threads an SM then have 64 KB in flight.
template <typename T, bool VEC, bool RES>
__global__ void __launch_bounds__(256) dropout_kernel(const T* x, const T* residual, T* y, uint64_t n, DropKey key) {
  // (x, residual and y may be one buffer: an element is read before it is written, by the same thread)
  const uint32_t step = drop_step(key);
  const uint64_t groups = (n + 7) / 8, stride = static_cast<uint64_t>(gridDim.x) * 512;
  for (uint64_t g = static_cast<uint64_t>(blockIdx.x) * 512 + threadIdx.x; g < groups; g += stride) {
    const uint64_t h = g + 256;
    Vec8<T> a0{}, a1{}, b0{}, b1{};
    if (VEC && g * 8 + 8 <= n) {
      a0 = load8(x + g * 8);
      if (RES) b0 = load8(residual + g * 8);
    }
    if (VEC && h * 8 + 8 <= n) {
      a1 = load8(x + h * 8);
      if (RES) b1 = load8(residual + h * 8);
    }
    dropout_group<T, VEC, RES>(a0, b0, x, residual, y, g, n, key, step);
    if (h < groups) dropout_group<T, VEC, RES>(a1, b1, x, residual, y, h, n, key, step);
  }
}

template <typename T>
static void dropout_typed(const void* x, const void* residual, void* y, size_t n, const DropKey& key, cudaStream_t s) {
  const bool vec = aligned16(x) && aligned16(y) && (residual == nullptr || aligned16(residual));
  const size_t blocks = ((n + 7) / 8 + 511) / 512;
  const unsigned grid = static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8);
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
