// Group norm over channels-last input [B, T, C] with the activation, and optionally the dropout, behind it.
//
//   xhat = (x - mean) * rstd, mean and rstd of one sample's T x C/G numbers;  z = xhat * gamma + beta;  y = drop(act(z))
//   gz = drop(dy) * act'(z);  per sample dbeta_b = sum_t gz, dgamma_b = sum_t gz * xhat;
//   dx = rstd * (gamma * gz - s1 - xhat * s2), s1 = sum_{c in g} gamma dbeta_b / n, s2 = sum_{c in g} gamma dgamma_b / n, n = T * C/G
//
// The per-channel sums that the group sums are made of are the per-sample parameter gradients that get clipped, so one
// pass over (dy, x) serves both.
//
// Each direction reads its inputs twice, reductions first, then the result; the second pass runs from the back, so that what
// the first one read last is still in L2.  A row is C contiguous numbers; a thread keeps one column (16 bytes) of channels
// and walks rows, so that channel sums and parameters stay in registers.  All sums run in a fixed order.  What bounds it is
// latency and the ends of passes: 46 to 62 % of the issue slots are used, by 22 to 35 % of the warps that an SM could hold (80
// registers, with dropout 127), and a pass's start and end move nothing.  (At the memory's speed a 16-bit element leaves 22 issue slots
// for a read and a write or two reads; the statistics take 10, the other passes 14 to 18 with silu and 25 to 33 with gelu and
// dropout, a third of that what a block does beside its rows.)  16 x 4096 x 320 bf16 with silu: 77 us both ways (the reads and writes of both
// ways once: 32); with 16 x 324 x 320 a pass takes 7 to 13 us from cold, so its start and end are much of it.  8 x 16384 x 256
// fp32, whose tensors do not stay in L2: 190 us of 164.
// (Tried: one kernel a direction whose blocks draw reductions and results from a counter, so that nothing drains between the
// passes.  A block that drew a result waited for reductions still running beside it: 16 x 4096 x 320 bf16 144 us for both
// directions against 117 then with a kernel a pass.  Tried: sets of samples whose second pass finds all of them in L2:
// 8 x 16384 x 256 fp32 217 us in sets of 100 MB, 292 of 48 MB, 199 without sets; each pass more costs more than its DRAM reads save.)
#include "fdp_async.cuh"
#include "fdp_dropout.cuh"
#include "fdp_kernels.h"
#include "fdp_vec8.cuh"

namespace fdp {
namespace {

constexpr int GN_THREADS = 256, GN_WARPS = GN_THREADS / 32;
// blocks an SM holds, by their registers: with the generator's words and keys beside the numbers only two
constexpr int gn_per_sm(bool drop) { return drop ? 2 : 3; }
// rows a turn of the loops: with the mask's draw two at once only lengthen the code (16 x 1024 x 1024 bf16: 107 us against 104 then)
__host__ __device__ constexpr int gn_unroll(bool drop) { return drop ? 1 : 2; }

// ---- V numbers of a thread --------------------------------------------------------------------------
// As pairs of fp32 in 64-bit registers, on which one instruction does two operations (rounded as single ones are); V = 1 is a
// plain float.  The pairs stay pairs: taken apart and put together again around every operation they cost more
// instructions than they save.
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair_of(float lo, float hi) {
  pair_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void pair_get(pair_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ pair_t pair_add(pair_t a, pair_t b) { pair_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ pair_t pair_mul(pair_t a, pair_t b) { pair_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ pair_t pair_fma(pair_t a, pair_t b, pair_t c) {
  pair_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
template <int V> struct Nums { pair_t p[V / 2]; };
template <> struct Nums<1> { float x; };
template <int V> __device__ __forceinline__ Nums<V> n_all(float v) {
  Nums<V> r;
  if constexpr (V == 1) { r.x = v; } else {
    const pair_t q = pair_of(v, v);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = q;
  }
  return r;
}
template <int V> __device__ __forceinline__ Nums<V> operator+(const Nums<V>& a, const Nums<V>& b) {
  Nums<V> r;
  if constexpr (V == 1) { r.x = a.x + b.x; } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pair_add(a.p[i], b.p[i]);
  }
  return r;
}
template <int V> __device__ __forceinline__ Nums<V> operator*(const Nums<V>& a, const Nums<V>& b) {
  Nums<V> r;
  if constexpr (V == 1) { r.x = a.x * b.x; } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pair_mul(a.p[i], b.p[i]);
  }
  return r;
}
template <int V> __device__ __forceinline__ Nums<V> n_fma(const Nums<V>& a, const Nums<V>& b, const Nums<V>& c) {
  Nums<V> r;
  if constexpr (V == 1) { r.x = fmaf(a.x, b.x, c.x); } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pair_fma(a.p[i], b.p[i], c.p[i]);
  }
  return r;
}
template <int V> __device__ __forceinline__ Nums<V> operator*(const Nums<V>& a, float s) { return a * n_all<V>(s); }
template <int V> __device__ __forceinline__ void n_get(const Nums<V>& a, float f[V]) {
  if constexpr (V == 1) { f[0] = a.x; } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) pair_get(a.p[i], f[2 * i], f[2 * i + 1]);
  }
}
template <int V> __device__ __forceinline__ Nums<V> n_of(const float f[V]) {
  Nums<V> r;
  if constexpr (V == 1) { r.x = f[0]; } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.p[i] = pair_of(f[2 * i], f[2 * i + 1]);
  }
  return r;
}

// V adjacent elements of a tensor: one vector of 16 bytes (8 of 16 bits, 4 of 32), or of 4 bytes (2 of 16 bits: rows whose length
// is only even), or one
template <typename T, int V> struct Raw { uint4 w; };
template <typename T> struct Raw<T, 2> { uint32_t w; };
template <typename T, int V>
__device__ __forceinline__ Nums<V> unpack_v(const Raw<T, V>& r) {
  float g[8];
  if constexpr (V == 2) unpack16<T>(make_uint4(r.w, 0, 0, 0), g);
  else unpack16<T>(r.w, g);
  return n_of<V>(g);
}
template <typename T, int V>
__device__ __forceinline__ Nums<V> load_v(const T* p) {
  if constexpr (V == 1) return Nums<1>{to_f32<T>(*p)};
  else return unpack_v<T, V>(*reinterpret_cast<const Raw<T, V>*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const Nums<V>& a) {
  float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  n_get<V>(a, f);
  if constexpr (V == 1) *p = from_f32<T>(f[0]);
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(p) = pack16<T>(f).x;
  else *reinterpret_cast<uint4*>(p) = pack16<T>(f);
}
template <int V>
__device__ __forceinline__ Nums<V> n_drop(const DropKey& k, uint32_t step, uint64_t element, const Nums<V>& a) {
  float f[V];
  n_get<V>(a, f);
  drop_v<V>(k, step, element, f);
  return n_of<V>(f);
}

// ---- activations -----------------------------------------------------------------------------------
// ex2.approx is off by 2^-22 of its result and rcp.approx by 2^-23, and rounding v log2(e) adds |v| 2^-23; where |v| is large
// enough for that to matter the result it is relative to has become small against z, so the error of an activation stays
// at a few 2^-23 of z.
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f, SQRT_2_PI = 0.7978845608028654f, INV_SQRT_2PI = 0.3989422804014327f, SQRT_HALF = 0.7071067811865476f;
// 1 / (1 + 2^u); 2^u may be infinite.  (Tried: two reciprocals out of one, 1 / a = b / (a b), to spare the special-function
// units.  They are not what bounds the passes, 16 instructions of eight cycles for every eight numbers; holding u down so
// that a product of two stays finite cost more issue slots than it saved.)
template <int V> __device__ __forceinline__ Nums<V> n_sigmoid2(const Nums<V>& u) {
  float a[V];
  n_get<V>(u, a);
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = ex2(a[e]);
  n_get<V>(n_of<V>(a) + n_all<V>(1.f), a);
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = rcp(a[e]);
  return n_of<V>(a);
}
// gelu_tanh: (1 + tanh w) / 2 = 1 / (1 + e^(-2 w)), which loses nothing where tanh w is near -1; w = sqrt(2/pi) (z + 0.044715 z^3)
template <int V> __device__ __forceinline__ Nums<V> n_gelu_half(const Nums<V>& z) {
  constexpr float K = -2.f * SQRT_2_PI * LOG2E;
  return n_sigmoid2<V>(n_fma<V>(z * z, n_all<V>(K * 0.044715f), n_all<V>(K)) * z);
}
// act(z).  The activation is a constant of the loop over rows: a choice inside it would keep the instructions of two rows apart.
template <int ACT, int V>
__device__ __forceinline__ Nums<V> activate(const Nums<V>& z) {
  switch (ACT) {
    case FDP_ACT_RELU: {
      float f[V];
      n_get<V>(z, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = f[e] > 0.f || isnan(f[e]) ? f[e] : 0.f;
      return n_of<V>(f);
    }
    case FDP_ACT_SILU:
      return n_sigmoid2<V>(z * -LOG2E) * z;
    case FDP_ACT_GELU: {
      float f[V];
      n_get<V>(z, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] *= fmaf(0.5f, erff(f[e] * SQRT_HALF), 0.5f);
      return n_of<V>(f);
    }
    case FDP_ACT_GELU_TANH:
      return n_gelu_half<V>(z) * z;
    default:
      return z;
  }
}
// body(Constant) of an activation known at run time
template <int N> struct Constant { static constexpr int value = N; };
template <typename Body>
__device__ __forceinline__ void with_activation(int act, Body body) {
  switch (act) {
    case FDP_ACT_RELU: body(Constant<FDP_ACT_RELU>{}); break;
    case FDP_ACT_SILU: body(Constant<FDP_ACT_SILU>{}); break;
    case FDP_ACT_GELU: body(Constant<FDP_ACT_GELU>{}); break;
    case FDP_ACT_GELU_TANH: body(Constant<FDP_ACT_GELU_TANH>{}); break;
    default: body(Constant<FDP_ACT_NONE>{});
  }
}
// g * act'(z)
template <int ACT, int V>
__device__ __forceinline__ Nums<V> times_slope(const Nums<V>& z, const Nums<V>& g) {
  switch (ACT) {
    case FDP_ACT_RELU: {
      float f[V], h[V];
      n_get<V>(z, f);
      n_get<V>(g, h);
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = f[e] > 0.f ? h[e] : 0.f;
      return n_of<V>(h);
    }
    case FDP_ACT_SILU: {                  // s (1 + z (1 - s)) = s + z s (1 - s)
      const Nums<V> s = n_sigmoid2<V>(z * -LOG2E);
      return g * n_fma<V>(n_fma<V>(s, n_all<V>(-1.f), n_all<V>(1.f)) * z, s, s);
    }
    case FDP_ACT_GELU: {
      float f[V];
      n_get<V>(z, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = fmaf(f[e] * INV_SQRT_2PI, ex2(-0.5f * LOG2E * f[e] * f[e]), fmaf(0.5f, erff(f[e] * SQRT_HALF), 0.5f));
      return g * n_of<V>(f);
    }
    case FDP_ACT_GELU_TANH: {             // h + z h (1 - h) 2 sqrt(2/pi) (1 + 3 * 0.044715 z^2)
      constexpr float K = 2.f * SQRT_2_PI;
      const Nums<V> h = n_gelu_half<V>(z);
      const Nums<V> t = n_fma<V>(z * z, n_all<V>(K * 3.f * 0.044715f), n_all<V>(K)) * z;
      return g * n_fma<V>(t, n_fma<V>(h, n_all<V>(-1.f), n_all<V>(1.f)) * h, h);
    }
    default:
      return g;
  }
}

// ---- a block's share: rows [r0, r1) and channels [c0, c0 + C) of sample b ---------------------------------
// Channels are those of whole groups: G of them from g0 on, of the sample's allC / allG.
struct Shape {
  int B, T, allC, allG, C, G, chunks, rows_per_chunk;
  // What follows is worked out by the host: a division takes a thread 25 instructions, and what a thread does beside its
  // rows was as much as 40 rows (16 x 4096 x 320 bf16, 18 rows a thread: 1200 instructions of 2000 in the first pass).
  int cols, rg, cg, lanes_channels, lanes_chunks;    // columns, rows at a time, channels of a group, threads a group (group_lanes)
  float inv_cols, inv_cg, inv_T, inv_n;              // inv_n: of a group's T x cg numbers
  unsigned by_chunks, by_rg;                         // ceil(2^32 / d), see quotient()
};
// n / d for n below 2^31 (by = ceil(2^32 / d), 0 for d = 1): the product may be one too large
__device__ __forceinline__ int quotient(int n, int d, unsigned by) {
  if (by == 0) return n;
  const int q = static_cast<int>(__umulhi(static_cast<unsigned>(n), by));
  return static_cast<unsigned>(q) * static_cast<unsigned>(d) > static_cast<unsigned>(n) ? q - 1 : q;
}
// n / d for n below 2^16 by multiplication: (n + 1/2) / d is at least 1 / (2 d) off the next whole number
__device__ __forceinline__ int small_quotient(int n, float inv) { return static_cast<int>((static_cast<float>(n) + 0.5f) * inv); }
struct Share { int b, chunk, r0, r1, c0, g0; };
__device__ __forceinline__ Share share_of(const Shape& h, int b, int slab, int chunk) {
  Share s;
  s.b = b;
  s.chunk = chunk;
  s.r0 = min(h.T, chunk * h.rows_per_chunk);
  s.r1 = min(h.T, s.r0 + h.rows_per_chunk);
  s.c0 = slab * h.C;
  s.g0 = slab * h.G;
  return s;
}
// whole rows, sample by sample
__device__ __forceinline__ Share share_of(const Shape& h, int block) {
  const int b = quotient(block, h.chunks, h.by_chunks);
  return share_of(h, b, 0, block - b * h.chunks);
}
// a thread's place: column group `col` of `cols`, row `row` of `rg` rows that the block takes at a time.  Rows of more
// columns than threads are walked `col`, `col` + GN_THREADS, ...
struct Place { int cols, rg, col, row; bool on; };
__device__ __forceinline__ Place place_of(const Shape& h) {
  Place p;
  p.cols = h.cols;
  p.rg = h.rg;
  p.row = h.cols < GN_THREADS ? small_quotient(threadIdx.x, h.inv_cols) : 0;
  p.col = static_cast<int>(threadIdx.x) - p.row * h.cols;
  p.on = p.row < p.rg;
  return p;
}
int rows_at_a_time(int cols) { return cols < GN_THREADS ? GN_THREADS / cols : 1; }

// ---- rows on their way ------------------------------------------------------------------------------------
// A thread reads NT tensors at the same flat indices, a row class's rows one after the other.  Where they are vectors its next D
// rows are copied (cp.async) into slots of shared memory that nobody else touches, so nothing is waited for but the thread's own
// oldest copy, and what is in flight takes no registers: with loads into registers, two rows ahead, the passes ran at a quarter of
// the memory's speed (16 x 4096 x 320 bf16: 15, 32, 42 and 46 us from cold).
template <typename T, int V, int NT>
struct Rows {
  static constexpr bool RING = V > 1;
  static constexpr int WIDE = V * static_cast<int>(sizeof(T));                    // bytes a copy
  static constexpr int SLOT = GN_THREADS * WIDE * NT;
  static constexpr int D = !RING ? 0 : 32768 / SLOT < 3 ? 3 : 32768 / SLOT > 16 ? 16 : 32768 / SLOT;
  static constexpr int BYTES = D * SLOT;
  const T* src[NT];     // where the block's share begins
  uint32_t slots;       // this thread's first slot
  uint32_t next;        // the next row to be copied, in elements from there (a share has less than 2^30)
  uint32_t stride;
  int left;             // rows not copied yet
  int slot;

  __device__ __forceinline__ void issue(int d) {
    if (left > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t to = slots + (d * NT + t) * (GN_THREADS * WIDE);
        if constexpr (WIDE == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src[t] + next) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(src[t] + next) : "memory");
      }
      next += stride;
      --left;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // `rows` rows from `first` on, `step` apart
  __device__ __forceinline__ void start(uint32_t ring, uint32_t first, uint32_t step, int rows) {
    next = first;
    stride = step;
    left = rows;
    slot = 0;
    if constexpr (RING) {
      slots = ring + threadIdx.x * WIDE;
#pragma unroll
      for (int d = 0; d < D; ++d) issue(d);
    }
  }
  // the next row of all tensors
  __device__ __forceinline__ void take(Nums<V> f[NT]) {
    if constexpr (RING) {
      asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint32_t from = slots + (slot * NT + t) * (GN_THREADS * WIDE);
        Raw<T, V> r;
        if constexpr (WIDE == 16)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.w.x), "=r"(r.w.y), "=r"(r.w.z), "=r"(r.w.w) : "r"(from) : "memory");
        else
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r.w) : "r"(from) : "memory");
        f[t] = unpack_v<T, V>(r);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) f[t] = load_v<T, V>(src[t] + next);
      next += stride;
    }
  }
  // after the numbers of take() have been used: their slot is filled again
  __device__ __forceinline__ void advance() {
    if constexpr (RING) {
      issue(slot);
      slot = slot + 1 == D ? 0 : slot + 1;
    }
  }
};

// the rows of a block's share that its thread takes, in the column `col`; none for a thread without a place
template <typename Stream>
__device__ __forceinline__ int gn_begin(Stream& in, uint8_t* ring, const Shape& h, const Share& sh, const Place& pl, int V, int col) {
  const int n = pl.on && col < pl.cols ? quotient(max(0, sh.r1 - sh.r0 - pl.row + pl.rg - 1), pl.rg, h.by_rg) : 0;
  in.start(smem_u32(ring), static_cast<uint32_t>(pl.row) * h.allC + col * V, static_cast<uint32_t>(pl.rg) * h.allC, n);
  return n;
}
// flat index of a share's first element
__device__ __forceinline__ size_t share_start(const Shape& h, const Share& sh) { return (static_cast<size_t>(sh.b) * h.T + sh.r0) * h.allC + sh.c0; }

// Sums over each group's entries 0 .. n-1: `lanes` adjacent threads (a power of two) take a group, so that the block works
// on GN_THREADS / lanes groups at once; every thread of a group gets the sum.  lanes is chosen for the block to be full.
inline int group_lanes(int G, int n) {
  int l = 32;
  while (l > 1 && (l * G > GN_THREADS || l / 2 >= n)) l >>= 1;
  return l;
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// body(g, k, valid): thread k of the `lanes` of group g (valid: there is such a group); all threads come along for the shuffles
template <typename Body>
__device__ __forceinline__ void for_groups(int G, int lanes, Body body) {
  const int k = threadIdx.x & (lanes - 1), shift = __popc(lanes - 1), step = GN_THREADS >> shift;
  for (int g0 = 0; g0 < G; g0 += step) {
    const int g = g0 + static_cast<int>(threadIdx.x >> shift);
    body(g < G ? g : G - 1, k, g < G);
  }
}

// Where the sums of channel c lie in shared memory, two floats each: a thread writes those of V adjacent channels, and with these in
// order the lanes of a warp would be 8 V bytes apart, V (of up to eight) on the same banks.
template <int V> __device__ __forceinline__ int spread(int c) { return c ^ ((c >> 4) & (V - 1)); }

// ---- forward, first pass: mean and sum of squared deviations of every (sample, chunk, group) ------------
// A thread takes its sums about the first number that it sees of a channel: the squares then lose nothing to a mean that is
// large against the spread, and a first number far off the others is itself part of the spread (n deviations about it lose
// n 2^-24 of what they add up to, n the few rows of a thread; about one number for the whole chunk the same loss has all its
// rows for n).  What the threads have is put together as (count, mean, squared deviations).  Squares that overflow stay infinite, so
// that the group's rstd is 0.
template <typename T, int V>
__device__ __forceinline__ void gn_stats(const Shape& h, const Share& sh, const Place& pl, uint8_t* gn_raw, const T* x, float2* part) {
  using Stream = Rows<T, V, 1>;
  const int C = h.C, G = h.G;
  float2* gn_ent = reinterpret_cast<float2*>(gn_raw + Stream::BYTES);       // [rg][C]: mean and squared deviations of a row class, then [0][C] of the chunk
  const int span_rows = sh.r1 - sh.r0;
  Stream in;
  in.src[0] = x + share_start(h, sh);
  for (int col = pl.col; col < pl.cols && pl.on; col += GN_THREADS) {
    const int n = gn_begin(in, gn_raw, h, sh, pl, V, col);
    Nums<V> p0 = n_all<V>(0.f), s1 = p0, s2 = p0, f[1];
    if (n > 0) {
      in.take(f);
      in.advance();
      p0 = f[0] * -1.f;
    }
#pragma unroll 2
    for (int r = 1; r < n; ++r) {
      in.take(f);
      const Nums<V> d = f[0] + p0;
      in.advance();
      s1 = s1 + d;
      s2 = n_fma<V>(d, d, s2);
    }
    float fp[V], f1[V], f2[V];
    n_get<V>(p0, fp);
    n_get<V>(s1, f1);
    n_get<V>(s2, f2);
    const float inv = __fdividef(1.f, static_cast<float>(max(1, n)));
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float m = f1[e] * inv;
      gn_ent[pl.row * C + spread<V>(col * V + e)] = make_float2(m - fp[e], isinf(f2[e]) ? f2[e] : fmaxf(f2[e] - f1[e] * m, 0.f));
    }
  }
  __syncthreads();
  // row classes: those before `longer` have one row more than the others
  const int classes = min(pl.rg, span_rows), base_rows = quotient(span_rows, pl.rg, h.by_rg), longer = span_rows - base_rows * pl.rg;
  const float inv = 1.f / max(1, span_rows);
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    float2* e = gn_ent + spread<V>(c);
    const float2 first = e[0];
    float sum = 0.f, m2 = first.y;
    for (int k = 1; k < classes; ++k) sum = fmaf(static_cast<float>(base_rows + (k < longer)), e[k * C].x - first.x, sum);
    const float m = sum * inv;               // the channel's mean, less the first class's
    m2 = fmaf(static_cast<float>(base_rows + (0 < longer)) * m, m, m2);
    for (int k = 1; k < classes; ++k) {
      const float2 v = e[k * C];
      const float d = v.x - first.x - m;
      m2 += fmaf(static_cast<float>(base_rows + (k < longer)) * d, d, v.y);
    }
    e[0] = make_float2(first.x + m, m2);
  }
  __syncthreads();
  const int cg = h.cg, lanes = h.lanes_channels;
  for_groups(G, lanes, [&](int g, int k, bool valid) {
    const int c0 = g * cg;
    const float ref = gn_ent[spread<V>(c0)].x;
    float sum = 0.f;
    for (int c = k; c < cg; c += lanes) sum += gn_ent[spread<V>(c0 + c)].x - ref;
    const float mean = fmaf(lanes_sum(sum, lanes), h.inv_cg, ref);
    float m2 = 0.f;
    for (int c = k; c < cg; c += lanes) {
      const float2 v = gn_ent[spread<V>(c0 + c)];
      const float d = v.x - mean;
      m2 += fmaf(span_rows * d, d, v.y);
    }
    m2 = lanes_sum(m2, lanes);
    if (valid && k == 0) part[(static_cast<size_t>(sh.b) * h.chunks + sh.chunk) * h.allG + sh.g0 + g] = make_float2(mean, m2);
  });
}

template <typename T, int V>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(false)) gn_stats_kernel(const Shape h, const T* x, float2* part) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  pdl_trigger();
  gn_stats<T, V>(h, share_of(h, blockIdx.x), place_of(h), gn_raw, x, part);
}

// floats of a per-channel array in shared memory: what follows it is 16-byte aligned again, whatever C is
__host__ __device__ __forceinline__ int gn_pad(int C) { return (C + 3) & ~3; }

// ---- per-channel constants in shared memory ----------------------------------------------------------------
// A thread's column of channels may lie in one group or in several: the constants are laid out by channel, and a thread
// takes its own into registers.
template <int V>
__device__ __forceinline__ Nums<V> take_v(const float* s, int col) {
  float f[V];
  if constexpr (V >= 4) {
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
      const float4 v = *reinterpret_cast<const float4*>(s + col * V + 4 * h);
      f[4 * h] = v.x; f[4 * h + 1] = v.y; f[4 * h + 2] = v.z; f[4 * h + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = s[col * V + e];
  }
  return n_of<V>(f);
}

// (mean, squared deviations) of a sample's group from its chunks', by `lanes` threads.  (From L2: in a cluster the others' are new.)
__device__ __forceinline__ float2 gn_moments(const Shape& h, const float2* p, int chunks, int rows_per_chunk, int lanes, int k) {
  constexpr int KEEP = 8;
  const float ref = __ldcg(p).x;
  if (chunks <= KEEP * lanes) {                // (one way to L2 instead of two)
    float2 v[KEEP];
    float rows[KEEP], sum = 0.f, m2 = 0.f;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const int i = k + j * lanes;
      rows[j] = 0.f;
      v[j] = make_float2(ref, 0.f);
      if (i < chunks) {
        rows[j] = static_cast<float>(max(0, min(rows_per_chunk, h.T - i * rows_per_chunk)));
        if (rows[j] > 0.f) v[j] = __ldcg(p + static_cast<size_t>(i) * h.allG);
      }
    }
#pragma unroll
    for (int j = 0; j < KEEP; ++j) sum = fmaf(rows[j], v[j].x - ref, sum);
    const float off = lanes_sum(sum, lanes) * h.inv_T;
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
      const float d = v[j].x - ref - off;
      m2 += fmaf(rows[j] * h.cg * d, d, v[j].y);
    }
    return make_float2(ref + off, lanes_sum(m2, lanes));
  }
  float sum = 0.f;
#pragma unroll 4
  for (int i = k; i < chunks; i += lanes) {
    const int rows = min(rows_per_chunk, h.T - i * rows_per_chunk);
    if (rows > 0) sum = fmaf(static_cast<float>(rows), __ldcg(p + static_cast<size_t>(i) * h.allG).x - ref, sum);
  }
  const float off = lanes_sum(sum, lanes) * h.inv_T;
  float m2 = 0.f;
#pragma unroll 4
  for (int i = k; i < chunks; i += lanes) {
    const int rows = min(rows_per_chunk, h.T - i * rows_per_chunk);
    if (rows > 0) {
      const float2 v = __ldcg(p + static_cast<size_t>(i) * h.allG);
      const float d = v.x - ref - off;
      m2 += fmaf(static_cast<float>(rows) * h.cg * d, d, v.y);
    }
  }
  return make_float2(ref + off, lanes_sum(m2, lanes));
}
// 1 / sqrt(v), one Newton step behind the approximate instruction; infinite for 0 and 0 for infinity
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  return isinf(r) || isinf(v) ? r : r * fmaf(-0.5f * v * r, r, 1.5f);
}
__device__ __forceinline__ float2 gn_total(const float2* p, int stride, int chunks, int lanes, int k) {
  float a = 0.f, b = 0.f;
#pragma unroll 4
  for (int i = k; i < chunks; i += lanes) { const float2 v = __ldcg(p + static_cast<size_t>(i) * stride); a += v.x; b += v.y; }
  return make_float2(lanes_sum(a, lanes), lanes_sum(b, lanes));
}
// Many chunks a sample (a few large ones): put together once, a block a sample, rather than by every block of the second pass.
constexpr int GN_MERGE_CHUNKS = 64;
template <bool MOMENTS>
__global__ void __launch_bounds__(GN_THREADS) gn_merge_kernel(const Shape h, const float2* part, float2* whole) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, lanes = h.lanes_chunks;
  for_groups(h.G, lanes, [&](int g, int k, bool valid) {
    const float2* p = part + static_cast<size_t>(b) * h.chunks * h.allG + g;
    const float2 v = MOMENTS ? gn_moments(h, p, h.chunks, h.rows_per_chunk, lanes, k) : gn_total(p, h.allG, h.chunks, lanes, k);
    if (valid && k == 0) whole[static_cast<size_t>(b) * h.allG + g] = v;
  });
}

// ---- forward, second pass -------------------------------------------------------------------------------
// shared: mean, rstd by group, then by channel -mean, A = rstd * gamma, beta; z = (x - mean) * A + beta
struct GnApply { const void *gamma, *beta; float *mean, *rstd; int pdt, act; float eps; };
// merge_chunks: how many of `part` there are a sample (one, of all rows, behind gn_merge_kernel)
template <typename T, int V, bool DROP, typename Wait>
__device__ __forceinline__ void gn_apply(const Shape& h, const Share& sh, const Place& pl, uint8_t* gn_raw, const T* x, const float2* part, int merge_chunks,
                                         T* y, const GnApply& q, const DropKey& key, Wait wait) {
  using Stream = Rows<T, V, 1>;
  const int C = h.C, G = h.G, cp = gn_pad(C);
  float* gn_c = reinterpret_cast<float*>(gn_raw + Stream::BYTES);
  float *c_mu = gn_c, *c_a = c_mu + cp, *c_b = c_a + cp;
  float2* stat = reinterpret_cast<float2*>(c_b + cp);
  Stream in;
  in.src[0] = x + share_start(h, sh);
  int n = gn_begin(in, gn_raw, h, sh, pl, V, pl.col);                // (rows and parameters need not wait for the statistics)
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    c_a[c] = q.gamma != nullptr ? load_as(q.gamma, q.pdt, sh.c0 + c) : 1.f;
    c_b[c] = q.beta != nullptr ? load_as(q.beta, q.pdt, sh.c0 + c) : 0.f;
  }
  wait();
  const int lanes = merge_chunks == h.chunks ? h.lanes_chunks : 1, rows = merge_chunks == h.chunks ? h.rows_per_chunk : h.T;
  for_groups(G, lanes, [&](int g, int k, bool valid) {
    const float2 v = gn_moments(h, part + static_cast<size_t>(sh.b) * merge_chunks * h.allG + sh.g0 + g, merge_chunks, rows, lanes, k);
    if (valid && k == 0) {
      const float rs = inv_sqrt(fmaf(v.y, h.inv_n, q.eps));
      stat[g] = make_float2(v.x, rs);
      if (sh.chunk == 0) {
        q.mean[static_cast<size_t>(sh.b) * h.allG + sh.g0 + g] = v.x;
        q.rstd[static_cast<size_t>(sh.b) * h.allG + sh.g0 + g] = rs;
      }
    }
  });
  __syncthreads();
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    const float2 st = stat[small_quotient(c, h.inv_cg)];
    c_mu[c] = -st.x;
    c_a[c] *= st.y;
  }
  __syncthreads();
  if (!pl.on) return;
  const uint32_t step = DROP ? drop_step(key) : 0;
  const size_t start = share_start(h, sh);
  T* out = y + start;
  for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
    const Nums<V> mu = take_v<V>(c_mu, col), A = take_v<V>(c_a, col), Bt = take_v<V>(c_b, col);
    if (col != pl.col) n = gn_begin(in, gn_raw, h, sh, pl, V, col);
    with_activation(q.act, [&](auto activation) {
      uint32_t i = static_cast<uint32_t>(pl.row) * h.allC + col * V;
#pragma unroll gn_unroll(DROP)
      for (int r = 0; r < n; ++r, i += in.stride) {
        Nums<V> f[1];
        in.take(f);
        const Nums<V> d = f[0] + mu;
        in.advance();
        Nums<V> a = activate<decltype(activation)::value, V>(n_fma<V>(d, A, Bt));
        if (DROP) a = n_drop<V>(key, step, start + i, a);
        store_v<T, V>(out + i, a);
      }
    });
  }
}

template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(DROP)) gn_apply_kernel(const Shape h, const T* x, const float2* part, int merge_chunks, T* y, const GnApply q,
                                                                 const DropKey key) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  pdl_trigger();
  // from the back: what the first pass read last is in L2
  gn_apply<T, V, DROP>(h, share_of(h, gridDim.x - 1 - blockIdx.x), place_of(h), gn_raw, x, part, merge_chunks, y, q, key, [] { pdl_wait(); });
}

// ---- both passes in one kernel --------------------------------------------------------------------------
// A cluster of h.chunks blocks takes some groups of one sample, reduces, meets at the cluster's barrier and writes: no
// block waits for another cluster, and while one cluster's blocks wait others of their SM work.
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ Share cluster_share(const Shape& h) {
  const int slabs = h.allG / h.G, id = quotient(blockIdx.x, h.chunks, h.by_chunks);
  return share_of(h, id / slabs, id % slabs, blockIdx.x - id * h.chunks);
}
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(DROP)) gn_fwd_cluster_kernel(const Shape h, const T* x, float2* part, T* y, const GnApply q, const DropKey key) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  const Share sh = cluster_share(h);
  const Place pl = place_of(h);
  gn_stats<T, V>(h, sh, pl, gn_raw, x, part);
  __syncthreads();
  gn_apply<T, V, DROP>(h, sh, pl, gn_raw, x, part, h.chunks, y, q, key, [] { cluster_meet(); });
}

// ---- backward ---------------------------------------------------------------------------------------------
// shared constants by channel: -mean, A = rstd * gamma, beta
__device__ __forceinline__ void bwd_constants(float* c_mu, float* c_a, float* c_b, const void* gamma, const void* beta, const float* mean,
                                              const float* rstd, int pdt, const Shape& h, const Share& sh) {
  const int C = h.C;
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    const size_t g = static_cast<size_t>(sh.b) * h.allG + sh.g0 + small_quotient(c, h.inv_cg);
    c_mu[c] = -__ldg(mean + g);
    const float rs = __ldg(rstd + g);
    c_a[c] = gamma != nullptr ? rs * load_as(gamma, pdt, sh.c0 + c) : rs;
    c_b[c] = beta != nullptr ? load_as(beta, pdt, sh.c0 + c) : 0.f;
  }
}
// f[0] = dy becomes gz, f[1] = x becomes x - mean, for V elements at flat index i
template <int ACT, int V, bool DROP>
__device__ __forceinline__ void gz_dev(Nums<V> f[2], size_t i, const Nums<V>& mu, const Nums<V>& A, const Nums<V>& Bt, const DropKey& key,
                                       uint32_t step) {
  f[1] = f[1] + mu;
  if (DROP) f[0] = n_drop<V>(key, step, i, f[0]);
  if (ACT != FDP_ACT_NONE) f[0] = times_slope<ACT, V>(n_fma<V>(f[1], A, Bt), f[0]);
}

// first pass: part[0][b][chunk][c] = sum gz * xhat, part[1] = sum gz; gpart[b][chunk][g] = (sum_c gamma * sum gz, the same with xhat)
struct GnBwd { const void *gamma, *beta; const float *mean, *rstd; int pdt, act; };
template <typename T, int V, bool DROP>
__device__ __forceinline__ void gn_bwd_sums(const Shape& h, const Share& sh, const Place& pl, uint8_t* gn_raw, const T* dy, const T* x, const GnBwd& q,
                                            float* part, float2* gpart, const DropKey& key) {
  using Stream = Rows<T, V, 2>;
  const int C = h.C, G = h.G, cp = gn_pad(C), cg = h.cg;
  float* gn_c = reinterpret_cast<float*>(gn_raw + Stream::BYTES);
  float *c_mu = gn_c, *c_a = c_mu + cp, *c_b = c_a + cp;
  float2* ent = reinterpret_cast<float2*>(gn_c);       // the sums [rg][C] take the constants' place afterwards
  Stream in;
  in.src[0] = dy + share_start(h, sh);
  in.src[1] = x + share_start(h, sh);
  int n = gn_begin(in, gn_raw, h, sh, pl, V, pl.col);
  bwd_constants(c_mu, c_a, c_b, q.gamma, q.beta, q.mean, q.rstd, q.pdt, h, sh);
  __syncthreads();
  const uint32_t step = DROP ? drop_step(key) : 0;
  float* wide = gn_c + 3 * cp;                          // rows of more columns than threads: sums apart from the constants
  const bool apart = pl.cols > GN_THREADS;
  const size_t start = share_start(h, sh);
  float s1[V], s2[V];
  for (int col = pl.col; col < pl.cols && pl.on; col += GN_THREADS) {
    const Nums<V> mu = take_v<V>(c_mu, col), A = take_v<V>(c_a, col), Bt = take_v<V>(c_b, col);
    Nums<V> t1 = n_all<V>(0.f), t2 = t1;
    if (col != pl.col) n = gn_begin(in, gn_raw, h, sh, pl, V, col);
    with_activation(q.act, [&](auto activation) {
      uint32_t i = static_cast<uint32_t>(pl.row) * h.allC + col * V;
#pragma unroll gn_unroll(DROP)
      for (int r = 0; r < n; ++r, i += in.stride) {
        Nums<V> f[2];
        in.take(f);
        gz_dev<decltype(activation)::value, V, DROP>(f, start + i, mu, A, Bt, key, step);
        in.advance();
        t1 = t1 + f[0];
        t2 = n_fma<V>(f[0], f[1], t2);
      }
    });
    n_get<V>(t1, s1);
    n_get<V>(t2, s2);
    if (apart) {
#pragma unroll
      for (int e = 0; e < V; ++e) reinterpret_cast<float2*>(wide)[spread<V>(col * V + e)] = make_float2(s1[e], s2[e]);
    }
  }
  __syncthreads();
  if (apart) {
    ent = reinterpret_cast<float2*>(wide);
  } else {
    if (pl.on) {
#pragma unroll
      for (int e = 0; e < V; ++e) ent[pl.row * C + spread<V>(pl.col * V + e)] = make_float2(s1[e], s2[e]);
    }
    __syncthreads();
  }
  const size_t at = (static_cast<size_t>(sh.b) * h.chunks + sh.chunk) * h.allC + sh.c0, second = static_cast<size_t>(h.B) * h.chunks * h.allC;
  for (int c = threadIdx.x; c < C; c += GN_THREADS) {
    float2* e = ent + spread<V>(c);
    float2 t = e[0];
    for (int k = 1; k < pl.rg; ++k) { const float2 v = e[k * C]; t.x += v.x; t.y += v.y; }
    t.y *= __ldg(q.rstd + static_cast<size_t>(sh.b) * h.allG + sh.g0 + small_quotient(c, h.inv_cg));
    part[at + c] = t.y;
    part[second + at + c] = t.x;
    const float ga = q.gamma != nullptr ? load_as(q.gamma, q.pdt, sh.c0 + c) : 1.f;
    e[0] = make_float2(ga * t.x, ga * t.y);
  }
  if (gpart == nullptr) return;
  __syncthreads();
  const int lanes = h.lanes_channels;
  for_groups(G, lanes, [&](int g, int k, bool valid) {
    float u = 0.f, v = 0.f;
    for (int c = k; c < cg; c += lanes) { const float2 e = ent[spread<V>(g * cg + c)]; u += e.x; v += e.y; }
    u = lanes_sum(u, lanes);
    v = lanes_sum(v, lanes);
    if (valid && k == 0) gpart[(static_cast<size_t>(sh.b) * h.chunks + sh.chunk) * h.allG + sh.g0 + g] = make_float2(u, v);
  });
}
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(DROP)) gn_bwd_sums_kernel(const Shape h, const T* dy, const T* x, const GnBwd q, float* part, float2* gpart,
                                                                               const DropKey key) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  pdl_trigger();
  gn_bwd_sums<T, V, DROP>(h, share_of(h, blockIdx.x), place_of(h), gn_raw, dy, x, q, part, gpart, key);
}

// per-sample gradients from their chunks: out[tensor][b][c], and the sums of squares of every 32 columns, one block's
// share: 32 columns of one sample and tensor, one of each warp a column
__device__ __forceinline__ void gn_psgrad(int piece, float* red, const float* part, float* out, float* sumsq, int chunks, int C) {
  const int nblk = (C + 31) / 32, sample = piece / nblk, l = threadIdx.x & 31, k0 = threadIdx.x >> 5;
  const int c = (piece - sample * nblk) * 32 + l;
  const float* p = part + static_cast<size_t>(sample) * chunks * C + c;
  float t = 0.f;
  if (c < C)
#pragma unroll 8
    for (int k = k0; k < chunks; k += GN_WARPS) t += p[static_cast<size_t>(k) * C];
  red[threadIdx.x] = t;
  __syncthreads();
  if (k0 == 0) {
#pragma unroll
    for (int k = 1; k < GN_WARPS; ++k) t += red[k * 32 + l];
    if (c < C) out[static_cast<size_t>(sample) * C + c] = t;
    t = warp_sum(t * t);
    if (l == 0) sumsq[piece] = t;
  }
}
__global__ void __launch_bounds__(GN_THREADS) gn_psgrad_kernel(const float* part, float* out, float* sumsq, int chunks, int C) {
  __shared__ float red[GN_THREADS];
  pdl_trigger();
  pdl_wait();
  gn_psgrad(blockIdx.x, red, part, out, sumsq, chunks, C);
}
// second pass: dx = A * gz - c1 - (x - mean) * c2, c1 = rstd * s1, c2 = rstd^2 * s2
template <typename T, int V, bool DROP, typename Wait>
__device__ __forceinline__ void gn_bwd_dx(const Shape& h, const Share& sh, const Place& pl, uint8_t* gn_raw, const T* dy, const T* x, const GnBwd& q,
                                          const float2* gpart, int merge_chunks, T* dx, const DropKey& key, Wait wait) {
  using Stream = Rows<T, V, 2>;
  const int C = h.C, G = h.G, cp = gn_pad(C), cg = h.cg;
  float* gn_c = reinterpret_cast<float*>(gn_raw + Stream::BYTES);
  float *c_mu = gn_c, *c_a = c_mu + cp, *c_b = c_a + cp, *c_1 = c_b + cp, *c_2 = c_1 + cp;
  Stream in;
  in.src[0] = dy + share_start(h, sh);
  in.src[1] = x + share_start(h, sh);
  int n = gn_begin(in, gn_raw, h, sh, pl, V, pl.col);
  bwd_constants(c_mu, c_a, c_b, q.gamma, q.beta, q.mean, q.rstd, q.pdt, h, sh);
  wait();
  const float inv_n = h.inv_n;
  const int lanes = merge_chunks == h.chunks ? h.lanes_chunks : h.lanes_channels;
  for_groups(G, lanes, [&](int g, int k, bool valid) {
    const float2 v = gn_total(gpart + static_cast<size_t>(sh.b) * merge_chunks * h.allG + sh.g0 + g, h.allG, merge_chunks, lanes, k);
    if (valid) {
      const float rs = __ldg(q.rstd + static_cast<size_t>(sh.b) * h.allG + sh.g0 + g);
      for (int c = g * cg + k; c < (g + 1) * cg; c += lanes) { c_1[c] = -rs * (v.x * inv_n); c_2[c] = -rs * rs * (v.y * inv_n); }
    }
  });
  __syncthreads();
  if (!pl.on) return;
  const uint32_t step = DROP ? drop_step(key) : 0;
  const size_t start = share_start(h, sh);
  T* out = dx + start;
  for (int col = pl.col; col < pl.cols; col += GN_THREADS) {
    const Nums<V> mu = take_v<V>(c_mu, col), A = take_v<V>(c_a, col), Bt = take_v<V>(c_b, col), k1 = take_v<V>(c_1, col), k2 = take_v<V>(c_2, col);
    if (col != pl.col) n = gn_begin(in, gn_raw, h, sh, pl, V, col);
    with_activation(q.act, [&](auto activation) {
      uint32_t i = static_cast<uint32_t>(pl.row) * h.allC + col * V;
#pragma unroll gn_unroll(DROP)
      for (int r = 0; r < n; ++r, i += in.stride) {
        Nums<V> f[2];
        in.take(f);
        gz_dev<decltype(activation)::value, V, DROP>(f, start + i, mu, A, Bt, key, step);
        in.advance();
        store_v<T, V>(out + i, n_fma<V>(f[0], A, n_fma<V>(f[1], k2, k1)));
      }
    });
  }
}

// The launch has blocks behind those of dx that form the per-sample gradients, which need the first pass only: no launch of their
// own.  (In front they kept the others from starting: 16 x 4096 x 320 bf16 80 us both ways, now 77.)
struct GnPsgrad { int pieces; const float* part; float *out, *sumsq; };
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(DROP)) gn_bwd_dx_kernel(const Shape h, const T* dy, const T* x, const GnBwd q, const float2* gpart,
                                                                             int merge_chunks, T* dx, const GnPsgrad ps, const DropKey key) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  pdl_trigger();
  const int blocks = static_cast<int>(gridDim.x) - ps.pieces;
  if (static_cast<int>(blockIdx.x) >= blocks) {
    pdl_wait();
    gn_psgrad(blockIdx.x - blocks, reinterpret_cast<float*>(gn_raw), ps.part, ps.out, ps.sumsq, h.chunks, h.C);
    return;
  }
  gn_bwd_dx<T, V, DROP>(h, share_of(h, blocks - 1 - blockIdx.x), place_of(h), gn_raw, dy, x, q, gpart, merge_chunks, dx, key,
                              [] { pdl_wait(); });
}
// In a cluster every block also forms its part of the sample's gradients: one of h.chunks stretches of the channels.
template <typename T, int V, bool DROP>
__global__ void __launch_bounds__(GN_THREADS, gn_per_sm(DROP)) gn_bwd_cluster_kernel(const Shape h, const T* dy, const T* x, const GnBwd q, float* part,
                                                                                  float2* gpart, T* dx, const GnPsgrad ps, const DropKey key) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  const Share sh = cluster_share(h);
  const Place pl = place_of(h);
  pdl_trigger();
  gn_bwd_sums<T, V, DROP>(h, sh, pl, gn_raw, dy, x, q, part, gpart, key);
  __syncthreads();
  auto gradients = [&] {
    cluster_meet();
    if (ps.out == nullptr) return;
    const int width = (h.C + h.chunks - 1) / h.chunks, first = sh.chunk * width, last = min(h.C, first + width);
    float sq[2] = {0.f, 0.f};
    for (int v = threadIdx.x; v < 2 * width; v += GN_THREADS) {
      const int tensor = v >= width ? 1 : 0, c = first + v - tensor * width;
      if (c >= last) continue;
      const size_t row = static_cast<size_t>(tensor) * h.B + sh.b;
      const float* p = ps.part + row * h.chunks * h.allC + sh.c0 + c;
      float t = 0.f;
#pragma unroll 8
      for (int k = 0; k < h.chunks; ++k) t += __ldcg(p + static_cast<size_t>(k) * h.allC);
      ps.out[row * h.allC + sh.c0 + c] = t;
      if (tensor == 0) sq[0] = fmaf(t, t, sq[0]); else sq[1] = fmaf(t, t, sq[1]);
    }
    __shared__ float red[32];
    const int parts = h.allG / h.G * h.chunks, at = sh.g0 / h.G * h.chunks + sh.chunk;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float v = block_sum(sq[t], red);
      if (threadIdx.x == 0) ps.sumsq[(static_cast<size_t>(t) * h.B + sh.b) * parts + at] = v;
    }
  };
  if (dx != nullptr) gn_bwd_dx<T, V, DROP>(h, sh, pl, gn_raw, dy, x, q, gpart, h.chunks, dx, key, gradients);
  else gradients();
}

// clip factors from the sums of squares (`lanes` threads a sample), clipped sum over the samples, mean, noise: 32 columns of one
// tensor a block, eight threads a column, whose first numbers are on their way while the factors are formed
__global__ void __launch_bounds__(GN_THREADS) gn_clip_kernel(const float* psgrad, const float* sumsq, int nparts, int lanes, float Cc, float clamp, float* norms0,
                                                             float* norms1, void* out0, void* out1, int B, int C, int out_dt, float inv_div, NoiseKey nk0,
                                                             NoiseKey nk1) {
  extern __shared__ __align__(16) uint8_t gn_raw[];
  float* fac = reinterpret_cast<float*>(gn_raw);      // [B]
  __shared__ float red[GN_THREADS];
  const int tensor = blockIdx.y, l = threadIdx.x & 31, k0 = threadIdx.x >> 5, c = blockIdx.x * 32 + l;
  pdl_wait();
  constexpr int AHEAD = 8;
  const float* p = psgrad + static_cast<size_t>(tensor) * B * C + c;
  float v[AHEAD];
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) {
    const int b = k0 + j * GN_WARPS;
    v[j] = c < C && b < B ? p[static_cast<size_t>(b) * C] : 0.f;
  }
  for_groups(B, lanes, [&](int b, int k, bool valid) {
    const float* part = sumsq + (static_cast<size_t>(tensor) * B + b) * nparts;
    float sq = 0.f;
#pragma unroll 4
    for (int i = k; i < nparts; i += lanes) sq += part[i];
    sq = lanes_sum(sq, lanes);
    if (valid && k == 0) {
      const float n = norm_of_sumsq(sq);
      fac[b] = clip_factor(n, Cc, clamp);
      float* no = tensor == 0 ? norms0 : norms1;
      if (blockIdx.x == 0 && no != nullptr) no[b] = n;
    }
  });
  __syncthreads();
  float acc = 0.f;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j)
    if (k0 + j * GN_WARPS < B) acc = fmaf(fac[k0 + j * GN_WARPS], v[j], acc);
  if (c < C)
#pragma unroll 8
    for (int b = k0 + AHEAD * GN_WARPS; b < B; b += GN_WARPS) acc = fmaf(fac[b], p[static_cast<size_t>(b) * C], acc);
  red[threadIdx.x] = acc;
  __syncthreads();
  if (k0 == 0 && c < C) {
#pragma unroll
    for (int k = 1; k < GN_WARPS; ++k) acc += red[k * 32 + l];
    float mean = acc * inv_div;
    const NoiseKey& nk = tensor == 0 ? nk0 : nk1;
    if (nk.std != 0.f) mean += noise_at(nk, c);
    store_as(tensor == 0 ? out0 : out1, out_dt, c, mean);
  }
}

// constants of GN_MAX_CHANNELS channels (five floats, or three and two sums) beside a ring of 32 KB
constexpr size_t GN_SMEM_MOST = GN_MAX_CHANNELS * 20 + 32768;
static_assert(GN_SMEM_MOST <= 227 * 1024 && Rows<float, 4, 2>::BYTES <= 32768 && Rows<__half, 8, 2>::BYTES <= 32768, "shared memory of a block");
template <auto KERNEL>
bool opt_in(size_t bytes) {
  static bool done[64];
  static std::mutex mu;
  return bytes <= 47 * 1024 || smem_opt_in(done, mu, KERNEL, GN_SMEM_MOST);      // (a kernel may have some of its own)
}
template <auto KERNEL, typename... Args>
int gn_launch(unsigned grid, size_t smem, bool dependent, cudaStream_t s, Args... args) {
  if (!opt_in<KERNEL>(smem)) return FDP_ERR_LAUNCH;
  if (dependent) launch_dependent(KERNEL, dim3(grid), dim3(GN_THREADS), smem, s, args...);
  else KERNEL<<<grid, GN_THREADS, smem, s>>>(args...);
  note_launch();
  return FDP_OK;
}
// blocks in clusters of `cluster`
template <auto KERNEL, typename... Args>
int gn_launch_clusters(unsigned grid, int cluster, size_t smem, cudaStream_t s, Args... args) {
  static bool done[64];
  static std::mutex mu;
  if (!opt_in<KERNEL>(smem)) return FDP_ERR_LAUNCH;
  if (cluster > 8) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return FDP_ERR_LAUNCH; }
    std::lock_guard<std::mutex> lk(mu);
    if (!done[dev] && cudaFuncSetAttribute(KERNEL, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) { cudaGetLastError(); return FDP_ERR_LAUNCH; }
    done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(GN_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, KERNEL, args...) != cudaSuccess) { cudaGetLastError(); return FDP_ERR_LAUNCH; }
  note_launch();
  return FDP_OK;
}

Shape shape_of(const GnArgs& a, const GnPlan& pl, int V) {
  Shape h{};
  h.B = a.B; h.T = a.T; h.allC = a.C; h.allG = a.G;
  h.C = a.C / pl.slabs; h.G = a.G / pl.slabs;
  h.chunks = pl.chunks; h.rows_per_chunk = pl.rows_per_chunk;
  h.cols = h.C / V; h.rg = rows_at_a_time(h.cols); h.cg = a.C / a.G;
  h.lanes_channels = group_lanes(h.G, h.cg); h.lanes_chunks = group_lanes(h.G, pl.chunks);
  h.inv_cols = 1.0f / h.cols; h.inv_cg = 1.0f / h.cg; h.inv_T = static_cast<float>(1.0 / a.T);
  h.inv_n = static_cast<float>(1.0 / (static_cast<double>(a.T) * h.cg));
  const auto by = [](int d) { return d == 1 ? 0u : static_cast<unsigned>(((1ull << 32) + d - 1) / d); };
  h.by_chunks = by(pl.chunks); h.by_rg = by(h.rg);
  return h;
}

template <typename T, int V, bool DROP>
int fwd_typed(const GnArgs& a, const GnPlan& pl, cudaStream_t s) {
  constexpr size_t ring = Rows<T, V, 1>::BYTES;
  const Shape h = shape_of(a, pl, V);
  const size_t ent = ring + sizeof(float2) * static_cast<size_t>(rows_at_a_time(h.C / V)) * h.C;
  const size_t con = ring + sizeof(float) * (3 * gn_pad(h.C) + 2 * h.G);
  float2 *part = reinterpret_cast<float2*>(a.gpart), *whole = reinterpret_cast<float2*>(a.gsum);
  const DropKey key = a.drop != nullptr ? make_drop_key(a.drop) : DropKey{};
  const GnApply q{a.gamma, a.beta, a.mean, a.rstd, a.pdt, a.act, a.eps};
  const unsigned grid = static_cast<unsigned>(static_cast<size_t>(a.B) * pl.slabs * pl.chunks);
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  if (pl.cluster) return gn_launch_clusters<gn_fwd_cluster_kernel<T, V, DROP>>(grid, pl.chunks, ent > con ? ent : con, s, h, x, part, y, q, key);
  const bool merge = pl.chunks > GN_MERGE_CHUNKS;
  int st = gn_launch<gn_stats_kernel<T, V>>(grid, ent, false, s, h, x, part);
  if (st == FDP_OK && merge) st = gn_launch<gn_merge_kernel<true>>(a.B, 0, true, s, h, static_cast<const float2*>(part), whole);
  if (st == FDP_OK)
    st = gn_launch<gn_apply_kernel<T, V, DROP>>(grid, con, true, s, h, x, static_cast<const float2*>(merge ? whole : part), merge ? 1 : pl.chunks, y, q, key);
  return st;
}

// nparts: sums of squares a sample
template <typename T, int V, bool DROP>
int bwd_typed(const GnArgs& a, const GnPlan& pl, bool need_dw, int* nparts, cudaStream_t s) {
  constexpr size_t ring = Rows<T, V, 2>::BYTES;
  const Shape h = shape_of(a, pl, V);
  const size_t con = sizeof(float) * 3 * gn_pad(h.C), ent = sizeof(float2) * static_cast<size_t>(rows_at_a_time(h.C / V)) * h.C;
  const size_t sums = ring + (h.C / V > GN_THREADS ? con + sizeof(float2) * h.C : ent > con ? ent : con);
  size_t out = ring + sizeof(float) * 5 * gn_pad(h.C);
  if (out < sizeof(float) * GN_THREADS) out = sizeof(float) * GN_THREADS;
  float2 *gpart = reinterpret_cast<float2*>(a.gpart), *whole = reinterpret_cast<float2*>(a.gsum);
  const DropKey key = a.drop != nullptr ? make_drop_key(a.drop) : DropKey{};
  const GnBwd q{a.gamma, a.beta, a.mean, a.rstd, a.pdt, a.act};
  const unsigned grid = static_cast<unsigned>(static_cast<size_t>(a.B) * pl.slabs * pl.chunks);
  const T *x = static_cast<const T*>(a.x), *dy = static_cast<const T*>(a.dy);
  T* dx = static_cast<T*>(a.dx);
  GnPsgrad ps{0, a.part, need_dw ? a.psgrad : nullptr, a.sumsq};
  if (pl.cluster) {
    *nparts = pl.slabs * pl.chunks;
    return gn_launch_clusters<gn_bwd_cluster_kernel<T, V, DROP>>(grid, pl.chunks, sums > out ? sums : out, s, h, dy, x, q, a.part,
                                                                       dx != nullptr ? gpart : nullptr, dx, ps, key);
  }
  *nparts = ceil_div(a.C, 32);
  const bool merge = pl.chunks > GN_MERGE_CHUNKS;
  const int pieces = need_dw ? 2 * a.B * *nparts : 0;
  int st = gn_launch<gn_bwd_sums_kernel<T, V, DROP>>(grid, sums, false, s, h, dy, x, q, a.part, dx != nullptr ? gpart : nullptr, key);
  if (st == FDP_OK && dx != nullptr) {
    if (merge) st = gn_launch<gn_merge_kernel<false>>(a.B, 0, true, s, h, static_cast<const float2*>(gpart), whole);
    ps.pieces = pieces;
    if (st == FDP_OK)
      st = gn_launch<gn_bwd_dx_kernel<T, V, DROP>>(grid + pieces, out, true, s, h, dy, x, q, static_cast<const float2*>(merge ? whole : gpart),
                                                         merge ? 1 : pl.chunks, dx, ps, key);
  } else if (st == FDP_OK && need_dw) {
    st = gn_launch<gn_psgrad_kernel>(pieces, 0, true, s, static_cast<const float*>(a.part), a.psgrad, a.sumsq, pl.chunks, a.C);
  }
  return st;
}

template <typename T, bool DROP>
int fwd_any(const GnArgs& a, const GnPlan& pl, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = aligned16(a.x) && aligned16(a.y);
  if (pl.vec == V && aligned) return fwd_typed<T, V, DROP>(a, pl, s);
  if constexpr (V == 8)
    if (pl.vec == 2 && aligned) return fwd_typed<T, 2, DROP>(a, pl, s);
  return fwd_typed<T, 1, DROP>(a, pl, s);
}
template <typename T, bool DROP>
int bwd_any(const GnArgs& a, const GnPlan& pl, bool need_dw, int* nparts, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = aligned16(a.x) && aligned16(a.dy) && (a.dx == nullptr || aligned16(a.dx));
  if (pl.vec == V && aligned) return bwd_typed<T, V, DROP>(a, pl, need_dw, nparts, s);
  if constexpr (V == 8)
    if (pl.vec == 2 && aligned) return bwd_typed<T, 2, DROP>(a, pl, need_dw, nparts, s);
  return bwd_typed<T, 1, DROP>(a, pl, need_dw, nparts, s);
}
template <typename T>
int fwd_drop(const GnArgs& a, const GnPlan& pl, cudaStream_t s) { return a.drop != nullptr ? fwd_any<T, true>(a, pl, s) : fwd_any<T, false>(a, pl, s); }
template <typename T>
int bwd_drop(const GnArgs& a, const GnPlan& pl, bool need_dw, int* nparts, cudaStream_t s) {
  return a.drop != nullptr ? bwd_any<T, true>(a, pl, need_dw, nparts, s) : bwd_any<T, false>(a, pl, need_dw, nparts, s);
}

}  // namespace

// How the work is cut up.  Must not depend on the device in use, nor on pointers: the workspace query has to agree.
//
// Small tensors, where launches are what counts: clusters.  A sample's groups go to `slabs` clusters, its rows to the `chunks`
// blocks of each, and both passes are one kernel.  On the device a kernel a pass is as fast or faster (16 x 64 x 256 bf16, forward
// and backward 5.8 + 8.5 us against 6.9 + 9.8; 2 x 1600 x 256 13.0 + 14.3 against 8.8 + 14.3), but up to 2 MB a call takes the host
// longer than either, and a launch more is 2 to 3 us of it.  (In a captured step the host's time does not count and the difference on
// the device is lost.  Rows of a slab are at least 64 bytes, where they are no vectors 32:
// 3 x 1369 x 90 fp16 backward 13.1 us with one slab, 11.8 with three.)
// Others: a kernel a pass over whole rows, which keeps the SMs fuller (16 x 4096 x 320 bf16: 91 us then, in clusters of 16 blocks
// 113 to 142), in the number of chunks that takes the fewest (rows a thread + fixed cost of a block) a wave of blocks.
GnPlan gn_plan(int B, int T, int C, int G, int element, int tensors, bool drop) {
  constexpr int FIXED_ROWS = 6, SEGMENT = 64;          // rows a thread that a block's fixed cost is worth; bytes of a slab's row
  constexpr long long PIECE = 96 << 10, SMALL = 2 << 20;
  const int GN_WAVE = 148 * gn_per_sm(drop);
  GnPlan pl{};
  const int wide = 16 / element;
  pl.vec = C % wide == 0 ? wide : wide == 8 && C % 2 == 0 ? 2 : 1;
  pl.slabs = 1;
  const long long sample = static_cast<long long>(T) * C * element * tensors;
  if (sample * B <= SMALL) {
    // the fewest slabs (whole groups, whole vectors) whose clusters of up to 16 blocks make a block an SM, or the most there are
    int best = 1, best_chunks = 1;
    for (int d = 1; d <= G; ++d) {
      if (G % d != 0) continue;
      const int cs = C / d;
      if (d > 1 && cs * element < (pl.vec == wide ? SEGMENT : SEGMENT / 2)) break;
      if (cs % pl.vec != 0) continue;
      const int most = ceil_div(T, 2 * rows_at_a_time(cs / pl.vec));            // chunks of at least two rows a thread
      int k = 1;
      while (k < 16 && 2 * k <= most && (sample / d / k > PIECE || static_cast<long long>(B) * d * k < GN_WAVE)) k *= 2;
      best = d;
      best_chunks = k;
      if (static_cast<long long>(B) * d * k >= GN_WAVE && sample / d / k <= PIECE) break;
    }
    pl.cluster = true;
    pl.slabs = best;
    pl.chunks = best_chunks;
    pl.rows_per_chunk = ceil_div(T, best_chunks);
    return pl;
  }
  const int rg = rows_at_a_time(C / pl.vec), most = ceil_div(T, 2 * rg);
  int best = 1;
  long long best_cost = -1;
  for (int waves = 1; waves <= 4; ++waves) {
    long long ch = static_cast<long long>(waves) * GN_WAVE / B;
    if (ch < 1) ch = 1;
    if (ch > most) ch = most;
    const int rows = ceil_div(T, static_cast<int>(ch)), n = ceil_div(T, rows);
    const long long w = (static_cast<long long>(B) * n + GN_WAVE - 1) / GN_WAVE;
    const long long cost = w * (ceil_div(rows, rg) + FIXED_ROWS);
    if (best_cost < 0 || cost < best_cost) { best_cost = cost; best = n; }
  }
  pl.rows_per_chunk = ceil_div(T, best);
  pl.chunks = ceil_div(T, pl.rows_per_chunk);
  return pl;
}

int gn_fwd(const GnArgs& a, int dt, cudaStream_t s) {
  const GnPlan pl = gn_plan(a.B, a.T, a.C, a.G, static_cast<int>(dtype_size(dt)), 1, a.drop != nullptr);
  if (dt == FDP_F32) return fwd_drop<float>(a, pl, s);
  if (dt == FDP_BF16) return fwd_drop<__nv_bfloat16>(a, pl, s);
  return fwd_drop<__half>(a, pl, s);
}
int gn_sumsq_parts(int C, const GnPlan& pl) { return pl.cluster ? pl.slabs * pl.chunks : ceil_div(C, 32); }
int gn_bwd(const GnArgs& a, int dt, const fdp_dp_params* p, void* dgamma, void* dbeta, float* norms_gamma, float* norms_beta, cudaStream_t s) {
  const GnPlan pl = gn_plan(a.B, a.T, a.C, a.G, static_cast<int>(dtype_size(dt)), 2, a.drop != nullptr);
  const bool need_dw = dgamma != nullptr;
  int nparts = 0;
  const int st = dt == FDP_F32 ? bwd_drop<float>(a, pl, need_dw, &nparts, s)
                 : dt == FDP_BF16 ? bwd_drop<__nv_bfloat16>(a, pl, need_dw, &nparts, s) : bwd_drop<__half>(a, pl, need_dw, &nparts, s);
  if (st != FDP_OK || !need_dw) return st;
  const int div = p->batch_divisor > 0 ? p->batch_divisor : a.B;
  const float inv_div = 1.0f / static_cast<float>(div);
  const NoiseKey nk0 = make_noise_key(p, p->param_id), nk1 = make_noise_key(p, p->param_id2);
  if (a.B <= 8192) {
    launch_dependent(gn_clip_kernel, dim3(ceil_div(a.C, 32), 2), dim3(GN_THREADS), sizeof(float) * a.B, s, a.psgrad, a.sumsq, nparts, group_lanes(a.B, nparts), p->C,
                     p->clamp_value, norms_gamma, norms_beta, dgamma, dbeta, a.B, a.C, a.pdt, inv_div, nk0, nk1);
    note_launch();
  } else {
    ln_clip_finalize(a.psgrad, a.sumsq, nparts, p->C, p->clamp_value, a.factors, norms_gamma, norms_beta, dgamma, dbeta, a.B, 1, a.C, a.pdt,
                     inv_div, nk0, nk1, s);
  }
  return FDP_OK;
}

}  // namespace fdp
