// The keep-mask of the counter-based dropout, shared by the dropout kernel and the group norm that drops its output.
//
// Elements are taken in groups of eight (element i of the tensor, in row-major order, is number i % 8 of group i / 8), one
// Philox4x32-10 draw a group: key (seed lo, seed hi ^ "DROP"), counter (group lo, group hi, stream, step).  The key keeps
// these draws apart from the noise's.  Number e of a group has 16 bits of the draw (word e / 2, low half first) and, below
// them, the same 16 bits of a second draw whose counter has bit 63 of the group set; it is dropped where these 32 bits are
// less than T = round(p * 2^32), so P(drop) is p to 2^-33.  The second draw decides only where the first 16 bits equal T's:
// one element in 65536, so it is made in a branch that a warp of 256 elements enters once in 256 times.  (With 32 bits of
// one draw an element the generator would take twice the instructions, and a 16-bit tensor leaves an element
// about 22 issue slots at the speed of the memory: 148 SMs x 128 lanes x 1.9 GHz against 1.6e12 elements a second.)
#pragma once
#include "fdp_common.cuh"

namespace fdp {

struct DropKey {
  uint32_t k0[10], k1[10];  // the key of each round: constants of the launch, which cost an instruction nothing
  uint32_t stream, step;
  uint32_t hi;              // T >> 16 (65536 for p = 1: everything is dropped)
  uint32_t lo;              // T & 65535
  float scale;              // 1 / (1 - p)
  uint64_t offset;          // added to the group number
  const uint32_t* step_dev; // null, or a device counter added to `step` when the kernel runs
};

inline DropKey make_drop_key(const fdp_dropout_params* p) {
  DropKey k;
  k.k0[0] = static_cast<uint32_t>(p->seed);
  k.k1[0] = static_cast<uint32_t>(p->seed >> 32) ^ 0x44524F50u;
  for (int i = 1; i < 10; ++i) { k.k0[i] = k.k0[i - 1] + 0x9E3779B9u; k.k1[i] = k.k1[i - 1] + 0xBB67AE85u; }
  k.stream = p->stream_id;
  k.step = p->step;
  const unsigned long long t = static_cast<unsigned long long>(__builtin_nearbyint(p->p * 4294967296.0));
  k.hi = static_cast<uint32_t>(t >> 16);
  k.lo = static_cast<uint32_t>(t & 65535u);
  k.scale = p->p < 1.0 ? static_cast<float>(1.0 / (1.0 - p->p)) : 0.f;
  k.offset = p->offset;
  k.step_dev = p->step_device;
  return k;
}

__device__ __forceinline__ uint32_t drop_step(const DropKey& k) { return k.step_dev != nullptr ? k.step + __ldg(k.step_dev) : k.step; }

__device__ __forceinline__ void drop_philox(const DropKey& k, uint32_t step, uint64_t group, uint32_t r[4]) {
  uint32_t c0 = static_cast<uint32_t>(group), c1 = static_cast<uint32_t>(group >> 32), c2 = k.stream, c3 = step;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = static_cast<uint64_t>(0xD2511F53u) * c0, b = static_cast<uint64_t>(0xCD9E8D57u) * c2;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k.k0[i];
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k.k1[i];
    c1 = static_cast<uint32_t>(b);
    c3 = static_cast<uint32_t>(a);
  }
  r[0] = c0; r[1] = c1; r[2] = c2; r[3] = c3;
}

// A group's 16-bit numbers, two a word, after the border has been settled: number e is kept if it is at least the half of
// `bound` that it faces.
struct Draw { uint32_t w[4], bound; };
__device__ __forceinline__ Draw draw8(const DropKey& k, uint32_t step, uint64_t group) {
  group += k.offset;
  Draw d;
  drop_philox(k, step, group, d.w);
  const uint32_t both = k.hi | (k.hi << 16);
  d.bound = both + 0x00010001u;
  // a half of w ^ both that is zero has 16 bits like T's
  const uint32_t m = __vminu2(__vminu2(d.w[0] ^ both, d.w[1] ^ both), __vminu2(d.w[2] ^ both, d.w[3] ^ both));
  if (((m - 0x00010001u) & ~m & 0x80008000u) != 0 || k.hi >= 65535u) {  // (from 65535 on no number is above T's 16 bits: settled one by one)
    uint32_t q[4];
    drop_philox(k, step, group | (1ull << 63), q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t l = d.w[j] & 0xFFFFu, h = d.w[j] >> 16;
      const bool kl = l > k.hi || (l == k.hi && (q[j] & 0xFFFFu) >= k.lo), kh = h > k.hi || (h == k.hi && (q[j] >> 16) >= k.lo);
      d.w[j] = (kl ? 0xFFFFu : 0u) | (kh ? 0xFFFF0000u : 0u);
    }
    d.bound = 0x80008000u;
  }
  return d;
}
__device__ __forceinline__ bool draw_keeps(uint32_t word, uint32_t bound, int half) { return (half ? word >> 16 : word & 0xFFFFu) >= (bound & 0xFFFFu); }
// a * b of pairs, as one instruction
__device__ __forceinline__ void drop_scale2(float& a, float& b, float s) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}" : "+f"(a), "+f"(b) : "f"(s));
}
// V adjacent elements from number `element` on, a multiple of V (1, 2, 4 or 8): times 1 / (1 - p), or 0
template <int V>
__device__ __forceinline__ void drop_v(const DropKey& k, uint32_t step, uint64_t element, float f[V]) {
  const Draw d = draw8(k, step, element >> 3);
  if constexpr (V == 1) {
    const uint32_t j = (element >> 1) & 3, w = j == 0 ? d.w[0] : j == 1 ? d.w[1] : j == 2 ? d.w[2] : d.w[3];
    f[0] = draw_keeps(w, d.bound, element & 1) ? f[0] * k.scale : 0.f;
  } else {
    uint32_t w[V / 2];
    if constexpr (V == 8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = d.w[j];
    } else if constexpr (V == 4) {
      const bool upper = (element & 4) != 0;
      w[0] = upper ? d.w[2] : d.w[0];
      w[1] = upper ? d.w[3] : d.w[1];
    } else {
      const uint32_t j = (element >> 1) & 3;
      w[0] = j == 0 ? d.w[0] : j == 1 ? d.w[1] : j == 2 ? d.w[2] : d.w[3];
    }
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      drop_scale2(f[2 * j], f[2 * j + 1], k.scale);
      f[2 * j] = (w[j] << 16) >= (d.bound << 16) ? f[2 * j] : 0.f;
      f[2 * j + 1] = w[j] >= (d.bound & 0xFFFF0000u) ? f[2 * j + 1] : 0.f;
    }
  }
}

}  // namespace fdp
