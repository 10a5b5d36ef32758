// tcgen05 / TMA / CTA-pair wrappers and the epilogue warps' output boxes, shared by the tensor-core kernels.
// (mbarrier helpers live in fdp_async.cuh)
#pragma once
#include <cuda.h>
#include <stdint.h>

#include "fdp_async.cuh"

namespace fdp {

constexpr int BOX_ROWS = 32, BOX_BYTES = BOX_ROWS * 128;   // an epilogue warp's output box: 32 rows of 128 bytes
constexpr int MAX_SMS = 148;           // workers the split-K parking area is sized for
constexpr int TMEM_COLS = 512;

// ---- PTX wrappers (mbarrier helpers live in fdp_async.cuh) --------------------------------------------
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
// ---- CTA-pair (cta_group::2) helpers: the even CTA of a 2-CTA cluster issues one 256-row MMA for both;
// loads are per CTA (no multicast), completion is signalled on the leader's mbarrier ------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// shared::cluster address of the same shared-memory offset in CTA `rank` of the cluster
__device__ __forceinline__ uint32_t mapa_u32(uint32_t local_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Hands an accumulator back to the leader's MMA warp.  Relaxed: no memory is handed over with it, the accumulator's loads
// have completed (tcgen05.wait::ld), and tcgen05.fence::before_thread_sync here and ::after_thread_sync behind the MMA warp's
// wait order them before its MMAs, for which the PTX manual's patterns between threads use a relaxed arrive and wait too.  A release at cluster scope waits for the warp's
// own earlier stores and took 1300 to 2500 cycles, in which the pair's tensor cores ran dry (weight gradients in six products,
// 16 x 197 rows 768 -> 3072: 151 us, now 134; 5 x 704, 64 -> 7928: 153 / 121; one pair alone in three products, 8192 deep: 89 / 64).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(leader_bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(leader_bar) : "memory");
}
// arrives on the barrier at this offset in both CTAs of the pair.  (One commit to both, not one each: a commit holds
// the tensor pipe up by about 30 cycles; 32768 rows 4096 -> 4096 bf16: 732 -> 699 us.)
__device__ __forceinline__ void tc_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t r[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// shared-memory matrix descriptor (sm_100 format): start address, leading / stride byte offsets in
// 16-byte units, version 1, 128-byte swizzle.  The low word holds the address (and the leading offset), so that what
// moves with the stage and the K slice is one 32-bit addition.
struct Desc { uint32_t lo, hi; };
__device__ __forceinline__ Desc make_desc(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  Desc d;
  d.lo = ((saddr >> 4) & 0x3FFF) | (((lbo_bytes >> 4) & 0x3FFF) << 16);
  d.hi = ((sbo_bytes >> 4) & 0x3FFF) | (1u << 14) /* descriptor version of sm_100 */ | (2u << 29) /* SWIZZLE_128B */;
  return d;
}
// one lane of the warp, the same one every time
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// ---- output boxes ------------------------------------------------------------------------------------
// After tcgen05.ld a lane holds one row of the tile, so direct stores put the 32 lanes of an instruction
// on 32 different rows: half-used sectors, 32 lines per request (16384 rows, 1024 -> 3072, bf16 forward with
// bias: 171 us, tensor pipe 27 % busy; 86 us with the boxes and add_bias32).  Instead every epilogue warp
// writes boxes of 32 rows x 128 bytes into its own 4 KB of shared memory, in the 128-byte swizzle of the
// tensor map (16-byte chunk j of row r at slot j ^ (r & 7): no bank conflicts), and one lane hands each box
// to the copy engine, which also clips what lies past the matrix.
__device__ __forceinline__ void box_wait(int lane) {      // the previous box has been read out
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
__device__ __forceinline__ void box_put(uint32_t box, int lane, int j, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
               ::"r"(box + lane * 128 + ((j ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void box_send(uint32_t box, const CUtensorMap* map, int col, int row, int lane) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(col), "r"(row), "r"(box) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
__device__ __forceinline__ void box_drain(int lane) {     // before the CTA leaves
  if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
// 32 fp32 values per lane = one box
__device__ __forceinline__ void store_f32x32(uint32_t box, const CUtensorMap* map, const float v[32], int col, int row, int lane) {
  box_wait(lane);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    box_put(box, lane, j, __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
            __float_as_uint(v[4 * j + 3]));
  box_send(box, map, col, row, lane);
}
// ---- host side (fdp_tc.cu) ------------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn();
int launch_sms();                      // SMs the next persistent GEMM grid may occupy, an even number
// map of an output matrix [rows, cols] for the epilogue warps' boxes
bool make_out_map(CUtensorMap* m, void* base, uint64_t rows, uint64_t cols, int dt);

}  // namespace fdp
