// Tensor-core building blocks: TMA tensor maps, tcgen05 matrix instructions
// and tensor memory.  No load is multicast; a pair's commit arrives on both its
// CTAs' barriers.
#pragma once

#include <cuda.h>

#include "afb_device.cuh"
#include "afb_launch.h"

namespace afb {

// ---------------------------------------------------------------- host side --
// A 2-D tensor map over a row-major matrix of `rows` rows of `cols` elements,
// row stride `ld` bytes, box `bcols` x `brows`.  Out of bounds reads as zero.
inline cudaError_t make_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base,
                            uint64_t cols, uint64_t rows, uint64_t ld, uint32_t bcols, uint32_t brows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult res{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (encode == nullptr) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld};
  const cuuint32_t box[2] = {bcols, brows}, es[2] = {1, 1};
  const CUresult r = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// -------------------------------------------------------------- device side --
// The warp's index, the same register in all its lanes for the compiler too.
__device__ __forceinline__ int warp_index() { return __shfl_sync(kFull, static_cast<int>(threadIdx.x >> 5), 0); }
// True in one lane of a converged warp.  Copies and matrix instructions take
// their operands from uniform registers: issued under this predicate by a warp
// whose lanes all run the loop, a stage's four instructions take about half
// the time of the same loop run by lane 0 alone.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
// Box at (x, y) of the map into shared memory; x times the element size is a
// multiple of 16 bytes.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(m), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// Tensor memory: `cols` columns (a power of two, 32..512) of 128 lanes; the
// whole warp calls.  The address is written to shared memory.
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor; lbo and sbo in bytes.  The rows of 128, 64 or
// 32 bytes (`row`) are swizzled over as many bytes, in groups of 8.
// K-major (rows along k): sbo = 8 rows, between groups of 8 of m or n; lbo
// unused.  MN-major (rows along m or n): lbo between rows' lengths of m or n,
// sbo = 8 rows, between groups of 8 of k.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo, int row = 128) {
  const uint64_t mode = row == 128 ? 2 : row == 64 ? 4 : 6;
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) |
         (static_cast<uint64_t>(sbo >> 4) << 32) | (uint64_t{1} << 46) | (mode << 61);
}

// D[tmem] (+)= A * B, 8-bit integers, 32 k.
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
// The same for 16-bit floats, 16 k.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
// ---- a pair of CTAs (a cluster of two) working on one tile of 256 rows ------
// Box into this CTA's shared memory, signalled on `bar`, which may lie in the
// pair's other CTA.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* m, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(m), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Both CTAs call these with one warp each, between cluster barriers: the pair's
// other CTA has to be running.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// The pair's first CTA issues: 128 rows of A and half of B in each CTA, at the
// same places of their shared memory.
__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
      : "memory");
}
// Arrives on `bar` of both CTAs when the matrix instructions issued so far are
// done.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}
// mbar_wait for a barrier on which the cluster's other CTAs arrive.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kMaxWaitSpins; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  atomicOr(&g_afb_device_status, kStatusWaitTimeout);
  return false;
}
// Arrives on a barrier of any CTA of the cluster.  What the arrival announces
// (tensor memory read, or shared memory written and fenced for the matrix
// unit) concerns this CTA's own units, so the default release is enough; one of
// cluster scope waits for the thread's global stores and cost 1900 cycles here.
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Arrives on `bar` when the matrix instructions issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// 16 or 32 columns of the warp's 32 lanes: v[c] is column c of the lane.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
// 16 lanes by 8 * NB columns as matrix fragments: v[4 * i + j] of thread t is
// column 8 i + 2 (t % 4) + j % 2 of lane t / 4 + 8 (j / 2).
__device__ __forceinline__ void tmem_ld_frag2(uint32_t addr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(addr));
}
// Four 8x8 matrices of 16-bit elements, transposed: thread t gives elements
// (2 (t % 4), t / 4) and (2 (t % 4) + 1, t / 4) of matrix g in v[g]; lane
// 8 g + r gives the address of row r of matrix g.
__device__ __forceinline__ void stmatrix_trans(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ uint4 lds16a(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Writes `cols` columns of a warp's 32 accumulator lanes at `acc` as rows of a
// row-major 16-bit matrix: column c, lane l goes to y[c * ld + run + l], where
// run + l < ld.  value(c, g, lo, hi) gives the pair of columns c, c + 1 of lane
// 8 g + t / 4 (t the thread's lane), rounded, from their 32 bits.
//
// 16 columns at a time: fragments of 8 lanes x 8 columns are transposed into
// rows of 32 in the warp's own shared memory (st0: twice 1024 bytes, 128-byte
// aligned), which leave as whole 64-byte runs.  The rows' 16-byte pieces are
// swizzled, so that neither side meets a bank twice.  Lane by lane, in 2-byte
// stores, the same took 1.8 times as long as the matrix instructions of a tile
// with k = 2048.
template <typename F>
__device__ __forceinline__ void emit_columns(uint32_t acc, uint32_t st0, int cols, uint16_t* y, int ld, int run, F value) {
  const int lane = threadIdx.x & 31;
  const bool wide = ld % 8 == 0;
#pragma unroll 2
  for (int c = 0; c < cols; c += 16) {
    const uint32_t stage = st0 + ((c >> 4) & 1) * 1024;
    uint32_t v[2][8];
    tmem_ld_frag2(acc + c, v[0]);
    tmem_ld_frag2(acc + (16u << 16) + c, v[1]);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t o[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint32_t* p = &v[g >> 1][4 * i + 2 * (g & 1)];
        o[g] = value(c + 8 * i + 2 * (lane & 3), g, p[0], p[1]);
      }
      const int row = 8 * i + (lane & 7);
      stmatrix_trans(stage + row * 64 + (((lane >> 3) ^ (row >> 1)) & 3) * 16, o);
    }
    __syncwarp();
    if (wide) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = 8 * i + (lane >> 2), at = run + (lane & 3) * 8;
        const uint4 w = lds16a(stage + row * 64 + (((lane & 3) ^ (row >> 1)) & 3) * 16);
        if (c + row < cols && at < ld) st16(y + static_cast<int64_t>(c + row) * ld + at, w);
      }
    } else {
      // a channel a lane; eight rows are read before the first is written
#pragma unroll
      for (int r0 = 0; r0 < 16; r0 += 8) {
        uint16_t w[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int row = r0 + r;
          asm volatile("ld.shared.u16 %0, [%1];"
                       : "=h"(w[r])
                       : "r"(stage + row * 64 + (((lane >> 3) ^ (row >> 1)) & 3) * 16 + (lane & 7) * 2)
                       : "memory");
        }
        if (run + lane < ld) {
          uint16_t* at = y + static_cast<int64_t>(c + r0) * ld + run + lane;
#pragma unroll
          for (int r = 0; r < 8; ++r, at += ld)
            if (c + r0 + r < cols) *at = w[r];
        }
      }
    }
  }
}

// Clusters.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address of `addr` (this CTA's shared memory) in the CTA `rank`.
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint4 peer_ld16(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr));
  return r;
}
// The 16 bytes at `addr` of every CTA of a cluster of up to 8; zero above it.
// All are asked for before the first is used.
__device__ __forceinline__ void peer_ld_all(uint32_t addr, int split, uint4 (&p)[8]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) p[r] = r < split ? peer_ld16(peer_addr(addr, r)) : make_uint4(0, 0, 0, 0);
}

// Launch with a cluster of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace afb
