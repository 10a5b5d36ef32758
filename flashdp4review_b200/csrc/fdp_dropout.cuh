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
  uint32_t k0, k1, stream, step;
  uint32_t hi;              // T >> 16 (65536 for p = 1: everything is dropped)
  uint32_t lo;              // T & 65535
  float scale;              // 1 / (1 - p)
  uint64_t offset;          // added to the group number
  const uint32_t* step_dev; // null, or a device counter added to `step` when the kernel runs
};

inline DropKey make_drop_key(const fdp_dropout_params* p) {
  DropKey k;
  k.k0 = static_cast<uint32_t>(p->seed);
  k.k1 = static_cast<uint32_t>(p->seed >> 32) ^ 0x44524F50u;
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

// bit e: number e of the group is kept.  `step` is drop_step(k), read once a thread.
__device__ __forceinline__ uint32_t keep8(const DropKey& k, uint32_t step, uint64_t group) {
  group += k.offset;
  uint32_t r[4];
  philox4x32_10(static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32), k.stream, step, k.k0, k.k1, r);
  const uint32_t both = k.hi | (k.hi << 16);
  uint32_t bits = 0, tie = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bits |= ((r[j] & 0xFFFFu) > k.hi ? 1u : 0u) << (2 * j);
    bits |= ((r[j] >> 16) > k.hi ? 1u : 0u) << (2 * j + 1);
    const uint32_t x = r[j] ^ both;                  // a half that is zero has 16 bits like T's
    tie |= (x - 0x00010001u) & ~x & 0x80008000u;     // (a half above a zero half may report itself too: looked at again below)
  }
  if (tie != 0 && k.hi < 65536u) {
    uint32_t q[4];
    philox4x32_10(static_cast<uint32_t>(group), static_cast<uint32_t>(group >> 32) | 0x80000000u, k.stream, step, k.k0, k.k1, q);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((r[j] & 0xFFFFu) == k.hi && (q[j] & 0xFFFFu) >= k.lo) bits |= 1u << (2 * j);
      if ((r[j] >> 16) == k.hi && (q[j] >> 16) >= k.lo) bits |= 1u << (2 * j + 1);
    }
  }
  return bits;
}
// one element on its own, for layouts in which a thread's elements are no whole group
__device__ __forceinline__ bool keep1(const DropKey& k, uint32_t step, uint64_t element) {
  return (keep8(k, step, element >> 3) >> (element & 7)) & 1u;
}

}  // namespace fdp
