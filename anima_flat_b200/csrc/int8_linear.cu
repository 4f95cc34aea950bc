// Matrix product in 8-bit integers with a scale per token and per channel:
//   y[m, n] = (sum_k q[m, k] w[n, k]) * s[m] * v[n] + bias[n]
// The sum is exact in 32-bit integers (K <= 131072: 127^2 K < 2^31), so the
// order of its parts does not matter.
//
// A tile is 128 channels by BN tokens: the weight rows are the first operand
// of the matrix instruction (tensor-memory lanes), the tokens the second
// (columns), so that a warp of the epilogue keeps its 32 channels' scales and
// biases in registers.  TMA brings both in blocks of 128 bytes along k; one
// thread issues the copies, one the matrix instructions, four warps the
// epilogue, which for large products overlaps the next tile's main loop (two
// accumulators in tensor memory).  Few tiles are split along k over a cluster,
// whose parts are added through distributed shared memory.
#include "int8_common.cuh"
#include "tc_device.cuh"

#include <algorithm>

namespace afb {

struct LinearArgs {
  const float* s;        // [M]
  const float* v;        // [N] or null (1)
  const uint16_t* bias;  // [N] or null
  uint16_t* y;           // [M, N]
  int M, N, K;
  int ntiles, tiles;     // tiles along N, and in all
};

constexpr int kTileN = 128;    // channels of a tile
constexpr int kKBlock = 128;   // k of a stage: one swizzled row of 128 bytes
constexpr int kThreads = 192;  // copy, matrix, four epilogue warps

__host__ __device__ constexpr int lin_stage_bytes(int bn) { return (kTileN + bn) * kKBlock; }
__host__ __device__ constexpr int lin_stages(int bn) { return bn >= 128 ? 3 : bn >= 64 ? 4 : 5; }
__host__ __device__ constexpr int lin_smem(int bn) { return lin_stages(bn) * lin_stage_bytes(bn) + 1024; }
__host__ __device__ constexpr int lin_tmem(int bn) { return 2 * bn < 32 ? 32 : 2 * bn; }

__device__ __forceinline__ float scale_of(const LinearArgs& a, int n) { return a.v != nullptr ? __ldg(a.v + n) : 1.0f; }
__device__ __forceinline__ float scaled(uint32_t acc, float s, float v, float b) {
  return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(acc)), s), v), b);
}

// The warp's 32 channels from `run` and `cols` tokens from m0 of an accumulator
// at `acc`, scaled.  sm: the tokens' scales; vn, b: scale and bias of the
// lane's channel.
template <int DT>
__device__ __forceinline__ void emit(const LinearArgs& a, uint32_t acc, const float* sm, uint32_t st0, int run, int m0,
                                     int cols, float vn, float b) {
  const int lane = threadIdx.x & 31;
  float vf[4], bf[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    vf[g] = __shfl_sync(kFull, vn, (lane >> 2) + 8 * g);
    bf[g] = __shfl_sync(kFull, b, (lane >> 2) + 8 * g);
  }
  emit_columns(acc, st0, cols, a.y + static_cast<int64_t>(m0) * a.N, a.N, run,
               [&](int c, int g, uint32_t lo, uint32_t hi) {
                 const float2 s2 = *reinterpret_cast<const float2*>(&sm[c]);
                 return pack2<DT>(scaled(lo, s2.x, vf[g], bf[g]), scaled(hi, s2.y, vf[g], bf[g]));
               });
}

template <int BN, int DT>
__global__ void __launch_bounds__(kThreads, 2)
int8_linear_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap qmap,
                   const LinearArgs a, int split) {
  constexpr int ST = lin_stages(BN), SB = lin_stage_bytes(BN);
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * ST + 4];
  __shared__ __align__(8) float sm[2][BN];
  __shared__ __align__(128) uint8_t out[4][2][1024];  // a warp's 16 tokens x 32 channels, twice
  __shared__ uint32_t tslot;
  const uint32_t ring = (smem_addr(dyn) + 1023) & ~1023u;
  const uint32_t full = smem_addr(bars), empty = full + 8 * ST, accf = empty + 8 * ST, acce = accf + 16;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_map(&wmap);
    prefetch_map(&qmap);
    for (int i = 0; i < ST; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accf + 8 * i, 1);
      mbar_init(acce + 8 * i, 4);
    }
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(smem_addr(&tslot), lin_tmem(BN));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  pdl_wait();
  pdl_trigger();

  const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int blocks = (a.K + kKBlock - 1) / kKBlock;
  const int kb0 = static_cast<int>(static_cast<int64_t>(blocks) * rank / split);
  const int kb1 = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / split);
  const int first = static_cast<int>(blockIdx.x) / split, step = static_cast<int>(gridDim.x) / split;

  if (warp == 0) {
    // Copies: a stage is refilled once the matrix instructions that read it
    // are done.
    int it = 0, sent = 0;
    bool ok = true;
    for (int tile = first; ok && tile < a.tiles; tile += step) {
      const int n0 = (tile % a.ntiles) * kTileN, m0 = (tile / a.ntiles) * BN;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % ST;
        if (it >= ST && !mbar_wait(empty + 8 * st, ((it / ST) - 1) & 1)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(full + 8 * st, SB);
          tma_load(ring + st * SB, &wmap, kb * kKBlock, n0, full + 8 * st);
          tma_load(ring + st * SB + kTileN * kKBlock, &qmap, kb * kKBlock, m0, full + 8 * st);
        }
        __syncwarp();
        sent = it + 1;
      }
    }
    // After a wait that gave up: the copies still in flight land before the
    // block ends.
    if (!ok)
      for (int i = sent > ST ? sent - ST : 0; i < sent; ++i) mbar_wait(full + 8 * (i % ST), (i / ST) & 1);
  } else if (warp == 1) {
    // 32-bit sums of signed bytes, BN columns, 128 lanes.
    constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(BN >> 3) << 17) | (uint32_t(kTileN >> 4) << 24);
    const uint64_t desc0 = smem_desc(ring, 16, 1024);
    const int total = first < a.tiles ? ((a.tiles - first - 1) / step + 1) * (kb1 - kb0) : 0;
    int it = 0, n = 0;
    bool ok = true;
    for (int tile = first; ok && tile < a.tiles; tile += step, ++n) {
      const int buf = n & 1;
      if (n >= 2 && !mbar_wait(acce + 8 * buf, ((n >> 1) - 1) & 1)) break;
      tc_fence_after();
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % ST;
        if (!mbar_wait(full + 8 * st, (it / ST) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t da = desc0 + static_cast<uint64_t>(st * (SB >> 4));
          const uint64_t db = da + (kTileN * kKBlock >> 4);
#pragma unroll
          for (int k = 0; k < kKBlock / 32; ++k)
            mma_i8(tmem + buf * BN, da + 2 * k, db + 2 * k, idesc, kb > kb0 || k > 0);
          if (it + ST < total) mma_commit(empty + 8 * st);  // the last ones are not waited for
        }
        __syncwarp();
      }
      if (elect_one()) mma_commit(accf + 8 * buf);
      __syncwarp();
    }
  } else if (warp >= 2) {
    const int quad = warp & 3;  // the tensor-memory lanes that this warp may read
    const int et = static_cast<int>(threadIdx.x) - 64;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    int n = 0;
    bool ok = true;  // after a wait that gave up, only the barriers go on
    for (int tile = first; tile < a.tiles; tile += step, ++n) {
      const int buf = n & 1;
      const int n0 = (tile % a.ntiles) * kTileN, m0 = (tile / a.ntiles) * BN;
      const int ch = n0 + quad * 32 + lane;
      const bool nok = ch < a.N;
      const float vn = nok ? scale_of(a, ch) : 0.0f;
      const float b = nok && a.bias != nullptr ? load1<DT>(a.bias + ch) : 0.0f;
      for (int i = et; i < BN; i += 128) sm[buf][i] = m0 + i < a.M ? __ldcg(a.s + m0 + i) : 0.0f;
      named_bar_sync(1, 128);
      ok = ok && mbar_wait(accf + 8 * buf, (n >> 1) & 1);
      if (!ok) continue;
      tc_fence_after();
      const int cols = min(BN, a.M - m0);
      if (split == 1) {
        emit<DT>(a, trow + buf * BN, sm[buf], smem_addr(out[warp - 2][0]), n0 + quad * 32, m0, cols, vn, b);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce + 8 * buf);
      } else {
        // The ring is free: all its copies were read by the instructions that
        // the accumulator waited for.  Column c, lane l at (c * 128 + l) * 4.
        const uint32_t at = ring + (quad * 32 + lane) * 4;
#pragma unroll 1
        for (int c = 0; c < cols; c += 16) {
          uint32_t v[16];
          tmem_ld16(trow + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + (c + i) * 512), "r"(kb1 > kb0 ? v[i] : 0u) : "memory");
        }
      }
    }
  }
  if (split > 1) {
    __syncwarp();
    cluster_sync();
    // Four channels a lane, a column a warp and step.
    const int n0 = (first % a.ntiles) * kTileN, m0 = (first / a.ntiles) * BN;
    const int cols = min(BN, a.M - m0), ch = n0 + 4 * lane;
    if (ch < a.N) {
      float vn[4], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        vn[j] = ch + j < a.N ? scale_of(a, ch + j) : 0.0f;
        b[j] = a.bias != nullptr && ch + j < a.N ? load1<DT>(a.bias + ch + j) : 0.0f;
      }
      for (int c = rank + split * warp; c < cols; c += split * (kThreads / 32)) {
        uint4 p[8];
        peer_ld_all(ring + c * 512 + lane * 16, split, p);
        const float s = sm[0][c];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t acc = 0;
#pragma unroll
          for (int r = 0; r < 8; ++r) acc += word(p[r], j);
          f[j] = scaled(acc, s, vn[j], b[j]);
        }
        uint16_t* y = a.y + static_cast<int64_t>(m0 + c) * a.N + ch;
        const uint2 o = make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]));
        if (a.N % 4 == 0) {
          st8(y, o);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (ch + j < a.N) y[j] = static_cast<uint16_t>((j < 2 ? o.x : o.y) >> (16 * (j & 1)));
        }
      }
    }
    __syncwarp();
    cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free(tmem, lin_tmem(BN));
  }
}

// The same for large products, by pairs of CTAs: a tile is 256 channels by BN
// tokens, a CTA brings and emits its 128 channels and brings half of the
// tokens, the first CTA issues the matrix instructions for both.  A stage then
// costs a CTA (128 + BN / 2) rows from L2 for the work of 128 x BN: alone, with
// 256 tokens, it asks for 96 bytes a clock, more than L2 gives.
//
// No arrival is under way to the other CTA's shared memory when a CTA leaves:
// only those that someone waits for are made.  (With an arrival that nobody
// waited for just before the last cluster barrier, a chain of several hundred
// calls stopped.)
constexpr int kPairTok = 256;  // tokens of a pair's widest tile
constexpr int kPairStages = 6, kPairStageBytes = (kTileN + kPairTok / 2) * kKBlock;
constexpr int kPairSmem = kPairStages * kPairStageBytes + 1024;
constexpr int kPairThreads = 64 + 256;  // eight warps of the epilogue: 8192 x 256 -> 8192 39 us, 53 with four

template <int DT>
__global__ void __launch_bounds__(kPairThreads, 1)
int8_linear_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap qmap,
                        const LinearArgs a, int bn) {
  constexpr int BN = kPairTok, ST = kPairStages, SB = kPairStageBytes;  // the widest tile's
  const uint32_t stage_bytes = (kTileN + bn / 2) * kKBlock;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * ST + 4];
  __shared__ __align__(8) float sm[2][BN];
  __shared__ __align__(128) uint8_t out[8][2][1024];
  __shared__ uint32_t tslot;
  const uint32_t ring = (smem_addr(dyn) + 1023) & ~1023u;
  const uint32_t full = smem_addr(bars), empty = full + 8 * ST, accf = empty + 8 * ST, acce = accf + 16;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  if (threadIdx.x == 0) {
    prefetch_map(&wmap);
    prefetch_map(&qmap);
    for (int i = 0; i < ST; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accf + 8 * i, 1);
      mbar_init(acce + 8 * i, 16);
    }
    fence_mbar_init();
  }
  // Both CTAs run, and their barriers are ready, before the pair allocates.
  cluster_sync();
  __syncwarp();
  if (warp == 1) tmem_alloc_pair(smem_addr(&tslot), lin_tmem(BN));
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tslot;
  pdl_wait();
  pdl_trigger();

  const int blocks = (a.K + kKBlock - 1) / kKBlock;
  const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
  auto channel0 = [&](int tile) { return (tile % a.ntiles) * 2 * kTileN + rank * kTileN; };

  if (warp == 0) {
    const uint32_t full0 = peer_addr(full, 0);
    int it = 0, sent = 0;
    bool ok = true;
    for (int tile = first; ok && tile < a.tiles; tile += step) {
      const int n0 = channel0(tile), m0 = (tile / a.ntiles) * bn + rank * (bn / 2);
      for (int kb = 0; kb < blocks; ++kb, ++it) {
        const int st = it % ST;
        if (it >= ST && !mbar_wait(empty + 8 * st, ((it / ST) - 1) & 1)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full + 8 * st, 2 * stage_bytes);
          tma_load_pair(ring + st * SB, &wmap, kb * kKBlock, n0, full0 + 8 * st);
          tma_load_pair(ring + st * SB + kTileN * kKBlock, &qmap, kb * kKBlock, m0, full0 + 8 * st);
        }
        __syncwarp();
        sent = it + 1;
      }
    }
    // After a wait that gave up: the first CTA's barriers count both CTAs'
    // copies, and neither leaves before the cluster's last barrier.
    if (!ok && rank == 0)
      for (int i = sent > ST ? sent - ST : 0; i < sent; ++i) mbar_wait(full + 8 * (i % ST), (i / ST) & 1);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc =
          (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(bn >> 3) << 17) | (uint32_t(2 * kTileN >> 4) << 24);
      const uint64_t desc0 = smem_desc(ring, 16, 1024);
      const int total = first < a.tiles ? ((a.tiles - first - 1) / step + 1) * blocks : 0;
      int it = 0, n = 0;
      bool ok = true;
      for (int tile = first; ok && tile < a.tiles; tile += step, ++n) {
        const int buf = n & 1;
        if (n >= 2 && !mbar_wait_cluster(acce + 8 * buf, ((n >> 1) - 1) & 1)) break;
        tc_fence_after();
        for (int kb = 0; kb < blocks; ++kb, ++it) {
          const int st = it % ST;
          if (!mbar_wait_cluster(full + 8 * st, (it / ST) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = desc0 + static_cast<uint64_t>(st * (SB >> 4));
            const uint64_t db = da + (kTileN * kKBlock >> 4);
#pragma unroll
            for (int k = 0; k < kKBlock / 32; ++k)
              mma_i8_pair(tmem + buf * BN, da + 2 * k, db + 2 * k, idesc, kb > 0 || k > 0);
            if (it + ST < total) mma_commit_pair(empty + 8 * st);
          }
          __syncwarp();
        }
        if (elect_one()) mma_commit_pair(accf + 8 * buf);
        __syncwarp();
      }
    }
  } else {
    // Two warps for each quarter of the lanes, half of the tokens each.
    const int quad = warp & 3, from = ((warp - 2) >> 2) * (bn / 2);
    const int et = static_cast<int>(threadIdx.x) - 64;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t acce0 = peer_addr(acce, 0);
    int n = 0;
    bool ok = true;
    for (int tile = first; tile < a.tiles; tile += step, ++n) {
      const int buf = n & 1;
      const int n0 = channel0(tile), m0 = (tile / a.ntiles) * bn;
      const int ch = n0 + quad * 32 + lane;
      const float vn = ch < a.N ? scale_of(a, ch) : 0.0f;
      const float b = ch < a.N && a.bias != nullptr ? load1<DT>(a.bias + ch) : 0.0f;
      for (int i = et; i < bn; i += 256) sm[buf][i] = m0 + i < a.M ? __ldcg(a.s + m0 + i) : 0.0f;
      named_bar_sync(1, 256);
      ok = ok && mbar_wait(accf + 8 * buf, (n >> 1) & 1);
      if (!ok) continue;
      tc_fence_after();
      emit<DT>(a, trow + buf * BN + from, sm[buf] + from, smem_addr(out[warp - 2][0]), n0 + quad * 32, m0 + from,
               min(bn / 2, a.M - m0 - from), vn, b);
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && tile + 2 * step < a.tiles) mbar_arrive_at(acce0 + 8 * buf);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free_pair(tmem, lin_tmem(BN));
  }
  cluster_sync();  // neither CTA leaves while the pair frees
}

template <int DT>
static cudaError_t launch_pair(const void* q, const void* w, LinearArgs a, int bn, cudaStream_t st) {
  CUtensorMap wmap, qmap;
  const uint64_t K = static_cast<uint64_t>(a.K);
  cudaError_t e = make_map(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, w, K, a.N, K, kKBlock, kTileN);
  if (e == cudaSuccess)
    e = make_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, q, K, a.M, K, kKBlock, bn / 2);
  if (e == cudaSuccess) e = ensure_smem(int8_linear_pair_kernel<DT>, kPairSmem);
  if (e != cudaSuccess) return e;
  a.ntiles = (a.N + 2 * kTileN - 1) / (2 * kTileN);
  a.tiles = a.ntiles * ((a.M + bn - 1) / bn);
  const int grid = 2 * std::min(a.tiles, device_info().sms / 2);
  return launch_cluster(int8_linear_pair_kernel<DT>, dim3(grid), dim3(kPairThreads), kPairSmem, 2, st, wmap, qmap, a, bn);
}

template <int BN, int DT>
static cudaError_t launch_linear(const void* q, const void* w, LinearArgs a, int split, cudaStream_t st) {
  CUtensorMap wmap, qmap;
  const uint64_t K = static_cast<uint64_t>(a.K);
  cudaError_t e = make_map(&wmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, w, K, a.N, K, kKBlock, kTileN);
  if (e == cudaSuccess)
    e = make_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, q, K, a.M, K, kKBlock, BN);
  if (e == cudaSuccess) e = ensure_smem(int8_linear_kernel<BN, DT>, lin_smem(BN));
  if (e != cudaSuccess) return e;
  a.ntiles = (a.N + kTileN - 1) / kTileN;
  a.tiles = a.ntiles * ((a.M + BN - 1) / BN);
  const int grid = split > 1 ? a.tiles * split : std::min(a.tiles, device_info().sms * 2);
  return launch_cluster(int8_linear_kernel<BN, DT>, dim3(grid), dim3(kThreads), lin_smem(BN), split, st, wmap, qmap, a,
                        split);
}

// Tokens of a tile and parts along k, for single CTAs.  Up to 128 tokens one
// tile holds them all; above, 128.  Few tiles are split along k, two blocks a
// multiprocessor (264 fit in clusters of eight), into parts of four k blocks at
// least, or two while half of the multiprocessors would have none: 512 x 8192 ->
// 2048 14.8 us in 4 parts, 17.5 in 2; 128 x 2048 -> 2048 6.7 in 4, 8.2 in 8;
// 77 x 1024 -> 2047 5.1 in 4, 6.2 in 2.
static void linear_shape(int M, int N, int K, int sms, int* bn, int* split) {
  const int64_t nt = (N + kTileN - 1) / kTileN;
  auto tiles = [&](int b) { return nt * ((M + b - 1) / b); };
  int b = 16;
  while (b < 128 && b < M) b *= 2;
  const int blocks = (K + kKBlock - 1) / kKBlock;
  int s = 1;
  while (s < 8 && tiles(b) * s * 2 <= 2 * sms - 32 && blocks / (2 * s) >= (tiles(b) * s * 2 <= sms / 2 ? 2 : 4)) s *= 2;
  *bn = b;
  *split = s;
}

// Whether pairs of CTAs take a product of more than 128 tokens.  Always where
// 128 x 256 tiles would give every multiprocessor one.  For fewer, from eight
// k blocks on, where they take less by what was measured: a pair 4 us and 0.21 a
// k block and round of tiles; single CTAs 4 us, 7 in a cluster, and 0.30 a k
// block of a part, 0.48 where two share a multiprocessor.  1024 x 2048 -> 2048
// 8.2 us (11.2 single), 512 x 8192 -> 2048 17.1 (14.8).
static bool linear_by_pairs(int M, int N, int K, int bn, int split, int sms) {
  if (M <= 128) return false;
  const int64_t nt = (N + kTileN - 1) / kTileN, blocks = (K + kKBlock - 1) / kKBlock;
  if (nt * ((M + 255) / 256) >= sms) return true;
  if (blocks < 8) return false;
  const int64_t rounds = ((nt + 1) / 2 * ((M + 255) / 256) + sms / 2 - 1) / (sms / 2);
  const int64_t ctas = nt * ((M + bn - 1) / bn) * split;
  const int64_t single = (split > 1 ? 700 : 400) + (ctas + 2 * sms - 1) / (2 * sms) * (blocks / split) * (ctas > sms ? 48 : 30);
  return 400 + rounds * blocks * 21 < single;
}

// Tokens of a pair's tile: of 256, 224, 192 and 160 the one whose whole rounds
// of tiles take least, by the cycles of a block of k: 2 for a token's matrix
// instructions, or what L2 takes for its (128 + bn / 2) rows of 128 bytes at 66
// bytes a cycle.  1024 x 2048 -> 6144, 1.3 rounds of 256 or 1.9 of 192: 15.9 us
// and 13.8.
static int pair_tokens(int M, int N, int pairs) {
  const int64_t nt = (N + 2 * kTileN - 1) / (2 * kTileN);
  int best = kPairTok;
  int64_t least = INT64_MAX;
  for (int bn = kPairTok; bn >= 160; bn -= 32) {
    const int64_t rounds = (nt * ((M + bn - 1) / bn) + pairs - 1) / pairs;
    const int64_t cost = rounds * std::max(2 * bn, (kTileN + bn / 2) * kKBlock / 66);
    if (cost < least) {
      least = cost;
      best = bn;
    }
  }
  return best;
}

template <int DT>
static cudaError_t linear(const void* q, const void* w, const LinearArgs& a, cudaStream_t st) {
  const DeviceInfo& d = device_info();
  if (d.error != cudaSuccess) return d.error;
  int bn, split;
  linear_shape(a.M, a.N, a.K, d.sms, &bn, &split);
  if (linear_by_pairs(a.M, a.N, a.K, bn, split, d.sms))
    return launch_pair<DT>(q, w, a, pair_tokens(a.M, a.N, d.sms / 2), st);
  switch (bn) {
    case 16: return launch_linear<16, DT>(q, w, a, split, st);
    case 32: return launch_linear<32, DT>(q, w, a, split, st);
    case 64: return launch_linear<64, DT>(q, w, a, split, st);
    default: return launch_linear<128, DT>(q, w, a, split, st);
  }
}

// ------------------------------------------------------------------ few rows --
// A few short tokens, from their unquantised rows, in one launch.  The weight is
// read once and nothing else matters, so a block owns a contiguous range of
// channels, whose codes it asks into L2 before it waits for its predecessor;
// meanwhile it quantises the tokens itself into shared memory (296 blocks
// repeat that).  A warp then takes R channels at a
// time, 16 codes a lane and load, with dp4a.
struct FewArgs {
  const uint16_t* x;     // [M, K]
  const float* cols;     // [K] or null
  const int8_t* w;       // [N, K]
  const float* v;        // [N] or null
  const uint16_t* bias;  // [N] or null
  uint16_t* y;           // [M, N]
  int M, N, K;
  int per;  // channels of a block
};
constexpr int kFewRows = 4;
constexpr int64_t kFewK = 2048, kFewWeight = 1 << 24;
constexpr int kFewWarps = 8;

template <int MP, int DT>
__global__ void __launch_bounds__(kFewWarps * 32) int8_linear_few_kernel(const FewArgs a) {
  constexpr int W = kFewWarps / MP;        // warps that quantise a row
  constexpr int R = MP <= 2 ? 4 : 2;       // channels of a warp at a time
  extern __shared__ __align__(16) uint8_t dyn[];  // codes [MP][K]
  __shared__ uint32_t red[kFewWarps];
  __shared__ float scales[MP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n0 = blockIdx.x * a.per, n1 = min(n0 + a.per, a.N);
  const int64_t bytes = static_cast<int64_t>(n1 - n0) * a.K;
  for (int64_t at = static_cast<int64_t>(threadIdx.x) * 8192; at < bytes; at += kFewWarps * 32 * 8192)
    prefetch_l2(a.w + static_cast<int64_t>(n0) * a.K + at, static_cast<uint32_t>(min(bytes - at, static_cast<int64_t>(8192))));
  pdl_wait();
  pdl_trigger();
  {
    const int m = warp / W, t = (warp % W) * 32 + lane;
    const uint16_t* x = a.x + static_cast<int64_t>(m) * a.K;
    auto load = [&](int e, f2_t(&f)[4]) {
      const uint4 v = ld_keep(x + e);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = unpack2<DT>(word(v, j));
      if (a.cols != nullptr) {
        const float4 lo = ld_keep_f4(a.cols + e), hi = ld_keep_f4(a.cols + e + 4);
        f[0] = mul2(f[0], f2(lo.x, lo.y));
        f[1] = mul2(f[1], f2(lo.z, lo.w));
        f[2] = mul2(f[2], f2(hi.x, hi.y));
        f[3] = mul2(f[3], f2(hi.z, hi.w));
      }
    };
    float amax = 0.0f;
    if (m < a.M) {
#pragma unroll 4
      for (int e = t * 8; e < a.K; e += W * 256) {
        f2_t f[4];
        load(e, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max_abs_nan(amax, f[j]);
      }
    }
    const uint32_t top = warp_max_u32(__float_as_uint(amax));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    const uint32_t all = group_max_u32<W>(&red[m * W]);
    const RowScale r = row_scale(all);
    if (t == 0) scales[m] = scale_value(all);
#pragma unroll 4
    for (int e = t * 8; e < a.K; e += W * 256) {
      uint2 c = make_uint2(0, 0);
      if (m < a.M) {
        f2_t f[4];
        load(e, f);
        c = codes8(f, r);
      }
      st8(dyn + m * a.K + e, c);
    }
  }
  __syncthreads();
  for (int n = n0 + warp * R; n < n1; n += kFewWarps * R) {
    int acc[MP][R] = {};
#pragma unroll 4
    for (int k = lane * 16; k < a.K; k += 512) {
      uint4 w[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        w[r] = n + r < n1 ? ld_stream(a.w + static_cast<int64_t>(n + r) * a.K + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MP; ++m) {
        const uint4 q = lds16(dyn + m * a.K + k);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          acc[m][r] = __dp4a(static_cast<int>(w[r].x), static_cast<int>(q.x), acc[m][r]);
          acc[m][r] = __dp4a(static_cast<int>(w[r].y), static_cast<int>(q.y), acc[m][r]);
          acc[m][r] = __dp4a(static_cast<int>(w[r].z), static_cast<int>(q.z), acc[m][r]);
          acc[m][r] = __dp4a(static_cast<int>(w[r].w), static_cast<int>(q.w), acc[m][r]);
        }
      }
    }
    // Lane m R + r writes token m, channel n + r.
    int mine = 0;
#pragma unroll
    for (int m = 0; m < MP; ++m)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int sum = __reduce_add_sync(kFull, acc[m][r]);
        if (lane == m * R + r) mine = sum;
      }
    const int m = lane / R, c = n + lane % R;
    if (m < a.M && c < n1) {
      const float v = a.v != nullptr ? __ldg(a.v + c) : 1.0f, b = a.bias != nullptr ? load1<DT>(a.bias + c) : 0.0f;
      a.y[static_cast<int64_t>(m) * a.N + c] =
          static_cast<uint16_t>(pack2<DT>(scaled(static_cast<uint32_t>(mine), scales[m], v, b), 0.0f));
    }
  }
}

// Measured against quantise and product on their own: 1 x 2048 -> 6144 5.0 us
// (7.3), 4 x 2048 -> 6144 7.0 (7.7), 1 x 512 -> 2048 2.3 (4.8); but 1 x 2048 ->
// 24576 15.2 (12.7), 8 x 2048 -> 6144 9.3 (7.8) and 1 x 8192 -> 8192 28 (15.5),
// where tiles and TMA keep more of the weight coming.
static bool few_rows(int64_t M, int64_t N, int64_t K) { return M <= kFewRows && K <= kFewK && N * K <= kFewWeight; }

template <int DT>
static cudaError_t linear_few(FewArgs a, cudaStream_t st) {
  const DeviceInfo& d = device_info();
  if (d.error != cudaSuccess) return d.error;
  const int step = kFewWarps * (a.M <= 2 ? 4 : 2);
  // two blocks a multiprocessor, in whole rounds of their warps
  const int per = (a.N + 2 * d.sms - 1) / (2 * d.sms);
  a.per = per < step ? (per + 7) / 8 * 8 : (per + step - 1) / step * step;
  const dim3 grid((a.N + a.per - 1) / a.per), block(kFewWarps * 32);
  const int mp = a.M <= 2 ? 2 : 4;  // one token: 6.9 us with eight warps on its row, for 5.0
  const size_t smem = static_cast<size_t>(mp) * a.K;
  return mp == 2 ? launch_pdl(int8_linear_few_kernel<2, DT>, grid, block, smem, st, a)
                 : launch_pdl(int8_linear_few_kernel<4, DT>, grid, block, smem, st, a);
}

cudaError_t read_status_int8_linear(int* status, bool clear) { return tu_status(status, clear); }

}  // namespace afb

using namespace afb;

static bool check_linear(const void* w, const void* v, const void* bias, void* y, int64_t M, int64_t N, int64_t K,
                         int64_t most_k, int dtype) {
  return check(M >= 0 && M <= (1 << 30), "M must be in [0, 2^30]") &&
         check(N >= 1 && N <= (1 << 30), "N must be in [1, 2^30]") &&
         check(((M + 15) / 16) * ((N + kTileN - 1) / kTileN) <= (1 << 27), "M * N is too large") &&
         check_k(K, most_k) &&
         check_dtype(dtype) &&
         (M == 0 || (check_ptrs({w, y}, {"w", "y"}) && check(aligned(v, 4), "v is not 4-byte aligned") &&
                     check(aligned(bias, 2), "bias is not 2-byte aligned")));
}

static cudaError_t run_linear(const void* q, const void* s, const void* w, const void* v, const void* bias, void* y,
                              int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  LinearArgs a{};
  a.s = static_cast<const float*>(s);
  a.v = static_cast<const float*>(v);
  a.bias = static_cast<const uint16_t*>(bias);
  a.y = static_cast<uint16_t*>(y);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == kBf16 ? linear<kBf16>(q, w, a, st) : linear<kFp16>(q, w, a, st);
}

extern "C" int afb_int8_linear(const void* q, const void* s, const void* w, const void* v, const void* bias, void* y,
                               int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  ApiGuard g("afb_int8_linear");
  if (!check_linear(w, v, bias, y, M, N, K, 131072, dtype)) return g.fail();
  if (M == 0) return 0;
  if (!check_ptrs({q}, {"q"}) || !check_ptr4(s, "s") || !check_ptr4(v, "v")) return g.fail();
  return g.done(run_linear(q, s, w, v, bias, y, M, N, K, dtype, stream));
}

extern "C" size_t afb_int8_linear_x_workspace(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (M > (1 << 30) || N > (1 << 30) || K > 16384) return SIZE_MAX;
  if (few_rows(M, N, K)) return 0;
  return static_cast<size_t>(M) * (K + 4);
}

extern "C" int afb_int8_linear_x(const void* x, const void* cols, const void* w, const void* v, const void* bias,
                                 void* y, int64_t M, int64_t N, int64_t K, int dtype, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  ApiGuard g("afb_int8_linear_x");
  if (!check_linear(w, v, bias, y, M, N, K, 16384, dtype)) return g.fail();
  if (M == 0) return 0;
  if (!check_ptrs({x}, {"x"}) || !check(aligned(cols, 16), "cols is not 16-byte aligned") ||
      !check(workspace_bytes >= afb_int8_linear_x_workspace(M, N, K), "workspace too small"))
    return g.fail();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_rows(M, N, K)) {
    FewArgs f{};
    f.x = static_cast<const uint16_t*>(x);
    f.cols = static_cast<const float*>(cols);
    f.w = static_cast<const int8_t*>(w);
    f.v = static_cast<const float*>(v);
    f.bias = static_cast<const uint16_t*>(bias);
    f.y = static_cast<uint16_t*>(y);
    f.M = static_cast<int>(M);
    f.N = static_cast<int>(N);
    f.K = static_cast<int>(K);
    return g.done(dtype == kBf16 ? linear_few<kBf16>(f, st) : linear_few<kFp16>(f, st));
  }
  if (!check_ptrs({workspace}, {"workspace"})) return g.fail();
  int8_t* q = static_cast<int8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + M * K);
  const cudaError_t e = quantize_rows(x, cols, q, s, M, K, dtype, st);
  if (e != cudaSuccess) return g.done(e);
  return g.done(run_linear(q, s, w, v, bias, y, M, N, K, dtype, stream));
}
