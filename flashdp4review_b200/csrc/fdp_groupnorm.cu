// Group norm over channels-last input [B, T, C] with the activation, and optionally the dropout, behind it.
//
//   xhat = (x - mean) * rstd, mean and rstd of one sample's T x C/G numbers;  z = xhat * gamma + beta;  y = drop(act(z))
//   gz = drop(dy) * act'(z);  per sample dbeta_b = sum_t gz, dgamma_b = sum_t gz * xhat;
//   dx = rstd * (gamma * gz - s1 - xhat * s2), s1 = sum_{c in g} gamma dbeta_b / n, s2 = sum_{c in g} gamma dgamma_b / n, n = T * C/G
//
// The per-channel sums that the group sums are made of are the per-sample parameter gradients that get clipped, so one
// pass over (dy, x) serves both.  HBM-bound: a first kernel reduces, a second one reads the same data again (out of
// L2 where the tensors fit it) and writes.  A row is C contiguous numbers; a thread keeps one column of eight channels and
// walks rows, so that channel sums and parameters stay in registers.  All reductions run in a fixed order.
#include "fdp_dropout.cuh"
#include "fdp_kernels.h"
#include "fdp_vec8.cuh"

namespace fdp {
namespace {

constexpr int GN_THREADS = 256;

// V adjacent elements (V = 8 as 16-byte vectors, else one)
template <typename T, int V>
__device__ __forceinline__ void load_v(const T* p, float f[V]) {
  if constexpr (V == 8) unpack8(load8(p), f);
  else f[0] = to_f32<T>(*p);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float f[V]) {
  if constexpr (V == 8) store8(p, f);
  else *p = from_f32<T>(f[0]);
}
template <int V>
__device__ __forceinline__ uint32_t keep_v(const DropKey& k, uint32_t step, size_t element) {
  if constexpr (V == 8) return keep8(k, step, element >> 3);
  else return keep1(k, step, element) ? 1u : 0u;
}

// ---- activations -----------------------------------------------------------------------------------
// exp for 16-bit tensors: two instructions, relative error 2^-22 for the arguments that matter, far below their rounding
template <bool FAST> __device__ __forceinline__ float act_exp(float v) { return FAST ? __expf(v) : expf(v); }
template <bool FAST> __device__ __forceinline__ float act_sigmoid(float v) {
  const float d = 1.f + act_exp<FAST>(-v);
  return FAST ? __fdividef(1.f, d) : 1.f / d;
}
constexpr float SQRT_2_PI = 0.7978845608028654f, INV_SQRT_2PI = 0.3989422804014327f, SQRT_HALF = 0.7071067811865476f;
// gelu_tanh: (1 + tanh u) / 2 = sigmoid(2 u), which loses nothing where tanh u is near -1
template <bool FAST> __device__ __forceinline__ float gelu_half(float z) {
  return act_sigmoid<FAST>(2.f * SQRT_2_PI * z * fmaf(0.044715f * z, z, 1.f));
}
// act(z) of V values
template <bool FAST, int V>
__device__ __forceinline__ void activate(int act, const float z[V], float a[V]) {
  switch (act) {
    case FDP_ACT_RELU:
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = z[e] > 0.f || isnan(z[e]) ? z[e] : 0.f;
      break;
    case FDP_ACT_SILU:
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = z[e] * act_sigmoid<FAST>(z[e]);
      break;
    case FDP_ACT_GELU:
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = z[e] * fmaf(0.5f, erff(z[e] * SQRT_HALF), 0.5f);
      break;
    case FDP_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = z[e] * gelu_half<FAST>(z[e]);
      break;
    default:
#pragma unroll
      for (int e = 0; e < V; ++e) a[e] = z[e];
  }
}
// g[e] *= act'(z[e])
template <bool FAST, int V>
__device__ __forceinline__ void times_slope(int act, const float z[V], float g[V]) {
  switch (act) {
    case FDP_ACT_RELU:
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = z[e] > 0.f ? g[e] : 0.f;
      break;
    case FDP_ACT_SILU:
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float s = act_sigmoid<FAST>(z[e]);
        g[e] *= s * fmaf(z[e], 1.f - s, 1.f);
      }
      break;
    case FDP_ACT_GELU:
#pragma unroll
      for (int e = 0; e < V; ++e)
        g[e] *= fmaf(z[e] * INV_SQRT_2PI, act_exp<FAST>(-0.5f * z[e] * z[e]), fmaf(0.5f, erff(z[e] * SQRT_HALF), 0.5f));
      break;
    case FDP_ACT_GELU_TANH:
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = gelu_half<FAST>(z[e]);
        g[e] *= fmaf(z[e] * (h * (1.f - h)), 2.f * SQRT_2_PI * fmaf(3.f * 0.044715f * z[e], z[e], 1.f), h);
      }
      break;
    default:
      break;
  }
}

// ---- a block's share: rows [r0, r1) of sample b ------------------------------------------------------
struct Span { int b, chunk, r0, r1; };
__device__ __forceinline__ Span span_of(int chunks, int rows_per_chunk, int T) {
  Span s;
  s.b = blockIdx.x / chunks;
  s.chunk = blockIdx.x - s.b * chunks;
  s.r0 = s.chunk * rows_per_chunk;
  s.r1 = min(T, s.r0 + rows_per_chunk);
  return s;
}
// a thread's place: column group `col` of `cols`, row `row` of `rg` rows that the block takes at a time.  Rows of more
// columns than threads are walked `col`, `col` + GN_THREADS, ...
struct Place { int cols, rg, col, row; bool on; };
__device__ __forceinline__ Place place_of(int cols) {
  Place p;
  p.cols = cols;
  p.rg = cols < GN_THREADS ? GN_THREADS / cols : 1;
  p.row = cols < GN_THREADS ? static_cast<int>(threadIdx.x) / cols : 0;
  p.col = cols < GN_THREADS ? static_cast<int>(threadIdx.x) - p.row * cols : static_cast<int>(threadIdx.x);
  p.on = p.row < p.rg;
  return p;
}
int rows_at_a_time(int cols) { return cols < GN_THREADS ? GN_THREADS / cols : 1; }

// sums over groups of consecutive entries of a shared array: f(group, lane-strided loop body) is run by one warp a group, or by
// the whole block where there are fewer groups than warps
template <typename Body>
__device__ __forceinline__ void for_groups(int G, Body body) {
  const int warp = threadIdx.x >> 5;
  for (int g = warp; g < G; g += GN_THREADS / 32) body(g);
}

// ---- forward, first pass: mean and sum of squared deviations of every (sample, chunk, group) ------------
// A thread takes sums about the first number it sees of each channel: the squares then lose nothing to a mean that is
// large against the spread, and a first number far off the others is itself part of the spread.  What the threads have is
// put together as (count, mean, squared deviations).
template <typename T, int V>
__global__ void __launch_bounds__(GN_THREADS) gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ part, int Tn, int C, int G,
                                                              int rows_per_chunk, int chunks) {
  extern __shared__ float2 gn_ent[];       // [rg][C]: mean and squared deviations of a channel over a row class's rows
  const Span sp = span_of(chunks, rows_per_chunk, Tn);
  const Place pl = place_of(C / V);
  pdl_trigger();
  const T* xb = x + static_cast<size_t>(sp.b) * Tn * C;
  if (pl.on) {
    for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
      float p0[V], s1[V], s2[V];
#pragma unroll
      for (int e = 0; e < V; ++e) p0[e] = s1[e] = s2[e] = 0.f;
      const int first = sp.r0 + pl.row;
      if (first < sp.r1) load_v<T, V>(xb + static_cast<size_t>(first) * C + col * V, p0);
      int n = first < sp.r1 ? 1 : 0;
#pragma unroll 4
      for (int r = first + pl.rg; r < sp.r1; r += pl.rg) {
        float f[V];
        load_v<T, V>(xb + static_cast<size_t>(r) * C + col * V, f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = f[e] - p0[e];
          s1[e] += d;
          s2[e] = fmaf(d, d, s2[e]);
        }
        ++n;
      }
      const float inv = n > 0 ? 1.f / n : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float m = s1[e] * inv;
        gn_ent[static_cast<size_t>(pl.row) * C + col * V + e] = make_float2(p0[e] + m, fmaxf(s2[e] - s1[e] * m, 0.f));
      }
    }
  }
  __syncthreads();
  const int cg = C / G, lane = threadIdx.x & 31, span_rows = sp.r1 - sp.r0;
  for_groups(G, [&](int g) {
    const float ref = gn_ent[g * cg].x;
    float sum = 0.f, cnt = 0.f;
    for (int k = 0; k < pl.rg; ++k) {
      const float n = static_cast<float>((span_rows - k + pl.rg - 1) / pl.rg);     // rows of class k (0 from the last row on)
      if (n <= 0.f) break;
      for (int c = lane; c < cg; c += 32) { sum = fmaf(n, gn_ent[static_cast<size_t>(k) * C + g * cg + c].x - ref, sum); cnt += n; }
    }
    sum = warp_sum(sum);
    cnt = warp_sum(cnt);
    const float mean = ref + sum / cnt;
    float m2 = 0.f;
    for (int k = 0; k < pl.rg; ++k) {
      const float n = static_cast<float>((span_rows - k + pl.rg - 1) / pl.rg);
      if (n <= 0.f) break;
      for (int c = lane; c < cg; c += 32) {
        const float2 v = gn_ent[static_cast<size_t>(k) * C + g * cg + c];
        const float d = v.x - mean;
        m2 += fmaf(n * d, d, v.y);
      }
    }
    m2 = warp_sum(m2);
    if (lane == 0) part[(static_cast<size_t>(sp.b) * chunks + sp.chunk) * G + g] = make_float2(mean, m2);
  });
}

// ---- forward, second pass -------------------------------------------------------------------------------
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS) gn_apply_kernel(const T* __restrict__ x, const void* __restrict__ gamma, const void* __restrict__ beta,
                                                              const float2* __restrict__ part, T* __restrict__ y, float* __restrict__ mean,
                                                              float* __restrict__ rstd, int Tn, int C, int G, int pdt, float eps, int act,
                                                              int rows_per_chunk, int chunks, int part_rows, int part_chunks, DropKey key) {
  extern __shared__ float2 gn_stat[];      // [G]: mean, rstd
  const Span sp = span_of(chunks, rows_per_chunk, Tn);
  const Place pl = place_of(C / V);
  const int cg = C / G;
  pdl_trigger();
  pdl_wait();
  for (int g = threadIdx.x; g < G; g += GN_THREADS) {
    const float2* p = part + static_cast<size_t>(sp.b) * part_chunks * G + g;
    const float ref = p[0].x;
    float sum = 0.f;
    for (int k = 0; k < part_chunks; ++k) sum = fmaf(static_cast<float>(min(part_rows, Tn - k * part_rows)), p[static_cast<size_t>(k) * G].x - ref, sum);
    const float m = ref + sum / Tn;
    float m2 = 0.f;
    for (int k = 0; k < part_chunks; ++k) {
      const float2 v = p[static_cast<size_t>(k) * G];
      const float d = v.x - m;
      m2 += fmaf(static_cast<float>(min(part_rows, Tn - k * part_rows)) * cg * d, d, v.y);
    }
    const float rs = 1.0f / sqrtf(m2 / (static_cast<float>(Tn) * cg) + eps);
    gn_stat[g] = make_float2(m, rs);
    if (sp.chunk == 0) { mean[sp.b * G + g] = m; rstd[sp.b * G + g] = rs; }
  }
  __syncthreads();
  if (!pl.on) return;
  const uint32_t step = DROP ? drop_step(key) : 0;
  const size_t base = static_cast<size_t>(sp.b) * Tn * C;
  for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
    float mu[V], A[V], Bt[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = col * V + e;
      const float2 st = gn_stat[c / cg];
      mu[e] = st.x;
      A[e] = gamma != nullptr ? st.y * load_as(gamma, pdt, c) : st.y;
      Bt[e] = beta != nullptr ? load_as(beta, pdt, c) : 0.f;
    }
#pragma unroll 2
    for (int r = sp.r0 + pl.row; r < sp.r1; r += pl.rg) {
      const size_t i = base + static_cast<size_t>(r) * C + col * V;
      float z[V], a[V];
      load_v<T, V>(x + i, z);
#pragma unroll
      for (int e = 0; e < V; ++e) z[e] = fmaf(z[e] - mu[e], A[e], Bt[e]);
      activate<sizeof(T) == 2, V>(act, z, a);
      if (DROP) {
        const uint32_t keep = keep_v<V>(key, step, i);
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = (keep >> e) & 1u ? a[e] * key.scale : 0.f;
      }
      store_v<T, V>(y + i, a);
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------------------
// per-channel constants of a thread's column: z = xhat * gamma + beta, xhat = (x - mu) * rs
template <int V>
struct Column { float mu[V], rs[V], ga[V], be[V]; };
template <int V>
__device__ __forceinline__ void load_column(Column<V>& k, const void* gamma, const void* beta, const float* mean, const float* rstd, int pdt,
                                            int b, int G, int cg, int col) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int c = col * V + e, g = b * G + c / cg;
    k.mu[e] = __ldg(mean + g);
    k.rs[e] = __ldg(rstd + g);
    k.ga[e] = gamma != nullptr ? load_as(gamma, pdt, c) : 1.f;
    k.be[e] = beta != nullptr ? load_as(beta, pdt, c) : 0.f;
  }
}
// gz and xhat of V elements at flat index i
template <typename T, int V, bool DROP>
__device__ __forceinline__ void gz_xhat(const T* dy, const T* x, size_t i, const Column<V>& k, int act, const DropKey& key, uint32_t step,
                                        float gz[V], float xh[V]) {
  float z[V];
  load_v<T, V>(dy + i, gz);
  load_v<T, V>(x + i, xh);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    xh[e] = (xh[e] - k.mu[e]) * k.rs[e];
    z[e] = fmaf(xh[e], k.ga[e], k.be[e]);
  }
  if (DROP) {
    const uint32_t keep = keep_v<V>(key, step, i);
#pragma unroll
    for (int e = 0; e < V; ++e) gz[e] = (keep >> e) & 1u ? gz[e] * key.scale : 0.f;
  }
  times_slope<sizeof(T) == 2, V>(act, z, gz);
}

// first pass: part[0][b][chunk][c] = sum gz * xhat, part[1] = sum gz; gpart[b][chunk][g] = (sum_c gamma * sum gz, the same with xhat)
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS) gn_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ gamma,
                                                                 const void* __restrict__ beta, const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, float* __restrict__ part,
                                                                 float2* __restrict__ gpart, int B, int Tn, int C, int G, int pdt, int act,
                                                                 int rows_per_chunk, int chunks, DropKey key) {
  extern __shared__ float2 gn_sum[];       // [rg][C]: (sum gz, sum gz * xhat) of a row class, then [0][C] of the chunk
  const Span sp = span_of(chunks, rows_per_chunk, Tn);
  const Place pl = place_of(C / V);
  const int cg = C / G;
  pdl_trigger();
  const uint32_t step = DROP ? drop_step(key) : 0;
  const size_t base = static_cast<size_t>(sp.b) * Tn * C;
  if (pl.on) {
    for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
      Column<V> k;
      load_column<V>(k, gamma, beta, mean, rstd, pdt, sp.b, G, cg, col);
      float s1[V], s2[V];
#pragma unroll
      for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
#pragma unroll 2
      for (int r = sp.r0 + pl.row; r < sp.r1; r += pl.rg) {
        float gz[V], xh[V];
        gz_xhat<T, V, DROP>(dy, x, base + static_cast<size_t>(r) * C + col * V, k, act, key, step, gz, xh);
#pragma unroll
        for (int e = 0; e < V; ++e) { s1[e] += gz[e]; s2[e] = fmaf(gz[e], xh[e], s2[e]); }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) gn_sum[static_cast<size_t>(pl.row) * C + col * V + e] = make_float2(s1[e], s2[e]);
    }
  }
  __syncthreads();
  const size_t at = (static_cast<size_t>(sp.b) * chunks + sp.chunk) * C, second = static_cast<size_t>(B) * chunks * C;
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    float2 t = gn_sum[c];
    for (int k = 1; k < pl.rg; ++k) { const float2 v = gn_sum[static_cast<size_t>(k) * C + c]; t.x += v.x; t.y += v.y; }
    part[at + c] = t.y;
    part[second + at + c] = t.x;
    const float ga = gamma != nullptr ? load_as(gamma, pdt, c) : 1.f;
    gn_sum[c] = make_float2(ga * t.x, ga * t.y);
  }
  if (gpart == nullptr) return;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for_groups(G, [&](int g) {
    float a = 0.f, b = 0.f;
    for (int c = lane; c < cg; c += 32) { const float2 v = gn_sum[g * cg + c]; a += v.x; b += v.y; }
    a = warp_sum(a);
    b = warp_sum(b);
    if (lane == 0) gpart[(static_cast<size_t>(sp.b) * chunks + sp.chunk) * G + g] = make_float2(a, b);
  });
}

// second pass: dx
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS) gn_bwd_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x, const void* __restrict__ gamma,
                                                               const void* __restrict__ beta, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, const float2* __restrict__ gpart, T* __restrict__ dx,
                                                               int Tn, int C, int G, int pdt, int act, int rows_per_chunk, int chunks, DropKey key) {
  extern __shared__ float2 gn_s[];         // [G]: s1, s2
  const Span sp = span_of(chunks, rows_per_chunk, Tn);
  const Place pl = place_of(C / V);
  const int cg = C / G;
  pdl_trigger();
  pdl_wait();
  const float inv_n = 1.f / (static_cast<float>(Tn) * cg);
  for (int g = threadIdx.x; g < G; g += GN_THREADS) {
    const float2* p = gpart + static_cast<size_t>(sp.b) * chunks * G + g;
    float a = 0.f, b = 0.f;
    for (int k = 0; k < chunks; ++k) { const float2 v = p[static_cast<size_t>(k) * G]; a += v.x; b += v.y; }
    gn_s[g] = make_float2(a * inv_n, b * inv_n);
  }
  __syncthreads();
  if (!pl.on) return;
  const uint32_t step = DROP ? drop_step(key) : 0;
  const size_t base = static_cast<size_t>(sp.b) * Tn * C;
  for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
    Column<V> k;
    load_column<V>(k, gamma, beta, mean, rstd, pdt, sp.b, G, cg, col);
    float s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { const float2 s = gn_s[(col * V + e) / cg]; s1[e] = s.x; s2[e] = s.y; }
#pragma unroll 2
    for (int r = sp.r0 + pl.row; r < sp.r1; r += pl.rg) {
      const size_t i = base + static_cast<size_t>(r) * C + col * V;
      float gz[V], xh[V];
      gz_xhat<T, V, DROP>(dy, x, i, k, act, key, step, gz, xh);
#pragma unroll
      for (int e = 0; e < V; ++e) gz[e] = k.rs[e] * (fmaf(k.ga[e], gz[e], -s1[e]) - xh[e] * s2[e]);
      store_v<T, V>(dx + i, gz);
    }
  }
}

template <typename T, int V>
size_t entry_bytes(int C) { return sizeof(float2) * static_cast<size_t>(rows_at_a_time(C / V)) * C; }

// (the entries of wide rows take up to 64 KB)
template <auto KERNEL>
bool opt_in(size_t bytes) {
  static bool done[64];
  static std::mutex mu;
  return bytes <= 48 * 1024 || smem_opt_in(done, mu, KERNEL, GN_MAX_CHANNELS * sizeof(float2));
}

template <typename T, int V>
int fwd_typed(const GnArgs& a, const GnPlan& pl, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(static_cast<size_t>(a.B) * pl.chunks);
  const size_t ent = entry_bytes<T, V>(a.C), stat = sizeof(float2) * a.G;
  float2* part = static_cast<float2*>(a.workspace);
  const DropKey key = a.drop != nullptr ? make_drop_key(a.drop) : DropKey{};
  if (!opt_in<gn_stats_kernel<T, V>>(ent)) return FDP_ERR_LAUNCH;
  gn_stats_kernel<T, V><<<grid, GN_THREADS, ent, s>>>(static_cast<const T*>(a.x), part, a.T, a.C, a.G, pl.rows_per_chunk, pl.chunks);
  note_launch();
#define FDP_GN_APPLY(DROP)                                                                                                                  \
  do {                                                                                                                                       \
    if (!opt_in<gn_apply_kernel<T, V, DROP>>(stat)) return FDP_ERR_LAUNCH;                                                                   \
    launch_dependent(gn_apply_kernel<T, V, DROP>, dim3(grid), dim3(GN_THREADS), stat, s, static_cast<const T*>(a.x), a.gamma, a.beta, part,  \
                     static_cast<T*>(a.y), a.mean, a.rstd, a.T, a.C, a.G, a.pdt, a.eps, a.act, pl.rows_per_chunk, pl.chunks,                 \
                     pl.rows_per_chunk, pl.chunks, key);                                                                                     \
  } while (0)
  if (a.drop != nullptr) FDP_GN_APPLY(true); else FDP_GN_APPLY(false);
#undef FDP_GN_APPLY
  note_launch();
  return FDP_OK;
}

template <typename T, int V, bool DROP>
int bwd_typed(const GnArgs& a, const GnPlan& pl, float* part, float2* gpart, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(static_cast<size_t>(a.B) * pl.chunks);
  const size_t ent = entry_bytes<T, V>(a.C), stat = sizeof(float2) * a.G;
  const DropKey key = a.drop != nullptr ? make_drop_key(a.drop) : DropKey{};
  if (!opt_in<gn_bwd_sums_kernel<T, V, DROP>>(ent) || !opt_in<gn_bwd_dx_kernel<T, V, DROP>>(stat)) return FDP_ERR_LAUNCH;
  gn_bwd_sums_kernel<T, V, DROP><<<grid, GN_THREADS, ent, s>>>(
      static_cast<const T*>(a.dy), static_cast<const T*>(a.x), a.gamma, a.beta, a.mean, a.rstd, part, a.dx != nullptr ? gpart : nullptr, a.B, a.T,
      a.C, a.G, a.pdt, a.act, pl.rows_per_chunk, pl.chunks, key);
  note_launch();
  if (a.dx != nullptr) {
    launch_dependent(gn_bwd_dx_kernel<T, V, DROP>, dim3(grid), dim3(GN_THREADS), stat, s, static_cast<const T*>(a.dy), static_cast<const T*>(a.x),
                     a.gamma, a.beta, a.mean, a.rstd, gpart, static_cast<T*>(a.dx), a.T, a.C, a.G, a.pdt, a.act, pl.rows_per_chunk, pl.chunks, key);
    note_launch();
  }
  return FDP_OK;
}

template <typename T>
int fwd_any(const GnArgs& a, const GnPlan& pl, cudaStream_t s) {
  return pl.vec && aligned16(a.x) && aligned16(a.y) ? fwd_typed<T, 8>(a, pl, s) : fwd_typed<T, 1>(a, pl, s);
}
template <typename T>
int bwd_any(const GnArgs& a, const GnPlan& pl, float* part, float2* gpart, cudaStream_t s) {
  const bool vec = pl.vec && aligned16(a.x) && aligned16(a.dy) && (a.dx == nullptr || aligned16(a.dx));
  if (a.drop != nullptr) return vec ? bwd_typed<T, 8, true>(a, pl, part, gpart, s) : bwd_typed<T, 1, true>(a, pl, part, gpart, s);
  return vec ? bwd_typed<T, 8, false>(a, pl, part, gpart, s) : bwd_typed<T, 1, false>(a, pl, part, gpart, s);
}

}  // namespace

GnPlan gn_plan(int B, int T, int C) {
  GnPlan pl;
  pl.vec = C % 8 == 0;
  // six blocks an SM, each with at least four rows a thread
  const int rg = rows_at_a_time(pl.vec ? C / 8 : C);
  const long long most = (static_cast<long long>(T) + 4 * rg - 1) / (4 * rg);
  long long chunks = (148 * 6 + B - 1) / B;
  if (chunks > most) chunks = most;
  pl.rows_per_chunk = static_cast<int>((T + chunks - 1) / chunks);
  pl.chunks = ceil_div(T, pl.rows_per_chunk);
  return pl;
}

int gn_fwd(const GnArgs& a, int dt, cudaStream_t s) {
  const GnPlan pl = gn_plan(a.B, a.T, a.C);
  if (dt == FDP_F32) return fwd_any<float>(a, pl, s);
  if (dt == FDP_BF16) return fwd_any<__nv_bfloat16>(a, pl, s);
  return fwd_any<__half>(a, pl, s);
}
int gn_bwd(const GnArgs& a, int dt, float* part, float* gpart, cudaStream_t s) {
  const GnPlan pl = gn_plan(a.B, a.T, a.C);
  float2* gp = reinterpret_cast<float2*>(gpart);
  if (dt == FDP_F32) return bwd_any<float>(a, pl, part, gp, s);
  if (dt == FDP_BF16) return bwd_any<__nv_bfloat16>(a, pl, part, gp, s);
  return bwd_any<__half>(a, pl, part, gp, s);
}

}  // namespace fdp
