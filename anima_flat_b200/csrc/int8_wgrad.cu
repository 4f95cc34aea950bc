// Weight gradient from 8-bit checkpoints:
//   dw[n, k] = sum_t dy[t, n] (q[t, k] s[t])
// over the tokens t, with the codes and scales that the forward product read.
//
// The sum runs along the rows of both operands, so both enter the matrix
// instruction with their k index (the token) outermost, after groups of four
// warps have turned a stage of 64 tokens into its operands.  A token's scale
// goes with dy: the codes are exact in bf16, and g = dy s, formed in fp32, enters
// as the two bf16 values hi = RN(g) and lo = RN(g - hi), whose sum is g to 2^-16
// of it (2^-8 of bf16's half-step, 2^-5 of fp16's).  Both products add into one
// fp32 sum.  With q s rounded to 16 bits instead, one product is enough, but the
// error is 1.4 times that of rounding dw once, and fp16 ends at 65504 where codes
// with fp32 scales do not; bf16 has fp32's range.
//
// A tile is 128 channels (tensor-memory lanes) by BN columns of dy.  For an
// adapter's few columns the kernel reads the codes once at memory speed; for a
// full weight it is bound by the matrix instructions.  Few tiles are split
// along the tokens over a cluster, whose parts are added in order of rank
// through distributed shared memory: the order is fixed by the sizes alone.
#include "int8_common.cuh"
#include "tc_device.cuh"

#include <algorithm>

namespace afb {

struct WgradArgs {
  const float* s;  // [T]
  uint16_t* dw;    // [N, K]
  int T, N, K;
  int ld;  // row length of dy, a multiple of 8
  int ktiles;
};

constexpr int kTok = 64;  // tokens of a stage
constexpr int kCh = 128;  // channels of a tile

// A stage's copies (codes, and BN columns of dy in chunks of 64 at most) and
// its converted codes have rings of their own, since copies take longest.  hi
// takes the place of dy, and lo that of the codes; what of it does not fit there
// (a second chunk) follows the converted codes.  Two blocks share a
// multiprocessor up to 64 columns: with one, 120 blocks at most run at once in
// clusters of eight.
__host__ __device__ constexpr int wg_width(int bn) { return bn < 64 ? bn : 64; }  // columns of a chunk
__host__ __device__ constexpr int wg_chunks(int bn) { return bn / wg_width(bn); }
__host__ __device__ constexpr int wg_raw_bytes(int bn) { return kTok * kCh + bn * kTok * 2; }
__host__ __device__ constexpr int wg_conv_bytes(int bn) { return kCh * kTok * 2 + (wg_chunks(bn) - 1) * kTok * 128; }
__host__ __device__ constexpr int wg_raw(int bn) { return bn == 16 || bn >= 128 ? 6 : 3; }
// Groups of four warps that convert, one for each converted stage, and then
// write the results.  Sixteen warps on one stage after another took 0.58 us a
// stage, the latency of one pass from wait to arrival.  A group meets its
// stages of either ring in every phase: a wait by parity may be one phase
// behind its barrier, not two.
constexpr int kGroups = 3;
constexpr int kWgThreads = 64 + 128 * kGroups;
__host__ __device__ constexpr int wg_smem(int bn) { return kGroups * wg_conv_bytes(bn) + wg_raw(bn) * wg_raw_bytes(bn) + 1024; }
__host__ __device__ constexpr int wg_tmem(int bn) { return bn < 32 ? 32 : bn; }

// Sixteen codes to two 16-byte pieces of bf16.
__device__ __forceinline__ void convert16(const uint4 q, uint4& lo, uint4& hi) {
  uint32_t o[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = word(q, j) ^ 0x80808080u;  // code + 128 in each byte
    // 2^23 + 128 + code, then minus 2^23 + 128
    const f2_t a = f2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)),
                      __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)));
    const f2_t b = f2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)),
                      __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)));
    const f2_t base = splat2(8388736.0f);
    o[2 * j] = pack2<kBf16>(sub2(a, base));
    o[2 * j + 1] = pack2<kBf16>(sub2(b, base));
  }
  lo = make_uint4(o[0], o[1], o[2], o[3]);
  hi = make_uint4(o[4], o[5], o[6], o[7]);
}

__device__ __forceinline__ void sts16a(uint32_t addr, const uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// A token's 16 channels 16 part .. of a stage, converted, to the operand at
// `dst`: chunk of 64 channels, row of the token, 16-byte pieces swizzled by it.
__device__ __forceinline__ void put_converted(uint32_t dst, int t, int part, const uint4 code) {
  uint4 lo, hi;
  convert16(code, lo, hi);
  const uint32_t row = dst + (part >> 2) * (kTok * 128) + t * 128;
  const uint32_t p0 = ((2 * (part & 3)) ^ (t & 7)) * 16;
  sts16a(row + p0, lo);
  sts16a(row + (p0 ^ 16), hi);
}

// The warp's 16 rows of a chunk of dy at `src`, ROW bytes a token, times their
// scales: hi in their place, lo at `dst`.  A piece's place within the swizzled
// rows stays what it is.  The scale of row r comes from lane half + r.  An
// infinity or a NaN is in hi alone: as lo it would make a NaN of either.
template <int DT, int ROW>
__device__ __forceinline__ void split_rows(uint32_t src, uint32_t dst, float scales, int half) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < ROW / 32; ++j) {
    const int p = lane + 32 * j;
    const f2_t s = splat2(__shfl_sync(kFull, scales, half + p / (ROW / 16)));
    const uint4 v = lds16a(src + 16 * p);
    uint4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f2_t g = mul2(unpack2<DT>(word(v, k)), s);
      const uint32_t h = pack2<kBf16>(g);
      const f2_t r = sub2(g, unpack2<kBf16>(h));
      const float a = f2lo(r), b = f2hi(r);
      word_ref(hi, k) = h;
      word_ref(lo, k) = pack2<kBf16>(fabsf(a) < 0x1p127f ? a : 0.0f, fabsf(b) < 0x1p127f ? b : 0.0f);
    }
    sts16a(src + 16 * p, hi);
    sts16a(dst + 16 * p, lo);
  }
}

// Both operands bf16, outermost along k (bits 15, 16), `rows` by `cols`, fp32 sums.
__host__ __device__ constexpr uint32_t wg_idesc(int rows, int cols) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | (uint32_t(cols >> 3) << 17) | (uint32_t(rows >> 4) << 24);
}

template <int BN, int DT>
__global__ void __launch_bounds__(kWgThreads, BN <= 64 ? 2 : 1)
int8_wgrad_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                  const WgradArgs a, int split) {
  constexpr int R = wg_raw(BN), RB = wg_raw_bytes(BN), CB = wg_conv_bytes(BN), G = kGroups;
  constexpr int kGOff = kTok * kCh, kRow = wg_width(BN) * 2;  // bytes of a chunk's row
  static_assert(R % G == 0, "");
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[2 * R + 2 * G + 1];
  __shared__ uint32_t tslot;
  const uint32_t ring = (smem_addr(dyn) + 1023) & ~1023u, raw = ring + G * CB;
  const uint32_t full = smem_addr(bars), empty = full + 8 * R, conv = empty + 8 * R, cempty = conv + 8 * G;
  const uint32_t accf = cempty + 8 * G;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_map(&qmap);
    prefetch_map(&gmap);
    for (int i = 0; i < R; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < G; ++i) {
      mbar_init(conv + 8 * i, 4);
      mbar_init(cempty + 8 * i, 1);
    }
    mbar_init(accf, 1);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(smem_addr(&tslot), wg_tmem(BN));
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tslot;
  pdl_wait();
  pdl_trigger();

  const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / split;
  const int k0 = (tile % a.ktiles) * kCh, n0 = (tile / a.ktiles) * BN;
  const int blocks = (a.T + kTok - 1) / kTok;
  const int b0 = static_cast<int>(static_cast<int64_t>(blocks) * rank / split);
  const int nb = static_cast<int>(static_cast<int64_t>(blocks) * (rank + 1) / split) - b0;

  bool done = false;  // the accumulator holds this part's sum
  if (warp == 0) {
    int sent = 0;
    bool ok = true;
    for (int it = 0; it < nb; ++it) {
      const int st = it % R;
      const uint32_t base = raw + st * RB;
      if (it >= R && !mbar_wait(empty + 8 * st, ((it / R) - 1) & 1)) {
        ok = false;
        break;
      }
      if (elect_one()) {
        mbar_arrive_expect_tx(full + 8 * st, RB);
        tma_load(base, &qmap, k0, (b0 + it) * kTok, full + 8 * st);
#pragma unroll
        for (int c = 0; c < wg_chunks(BN); ++c)
          tma_load(base + kGOff + c * kTok * kRow, &gmap, n0 + 64 * c, (b0 + it) * kTok, full + 8 * st);
      }
      __syncwarp();
      sent = it + 1;
    }
    if (!ok)  // copies still in flight land before the block ends
      for (int i = sent > R ? sent - R : 0; i < sent; ++i) mbar_wait(full + 8 * (i % R), (i / R) & 1);
  } else if (warp == 1) {
    constexpr uint32_t idesc = wg_idesc(kCh, BN), idesc_lo = wg_idesc(kCh, wg_width(BN));
    const uint64_t ca = smem_desc(ring, kTok * 128, 1024);
    const uint64_t cb = smem_desc(raw + kGOff, kTok * kRow, 8 * kRow, kRow);
    const uint64_t cl = smem_desc(raw, kTok * kRow, 8 * kRow, kRow);
    for (int it = 0; it < nb; ++it) {
      const int st = it % R, cs = it % G;
      if (!mbar_wait(conv + 8 * cs, (it / G) & 1)) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t da = ca + static_cast<uint64_t>(cs * (CB >> 4)), db = cb + static_cast<uint64_t>(st * (RB >> 4));
        const uint64_t dl = cl + static_cast<uint64_t>(st * (RB >> 4));
#pragma unroll
        for (int k = 0; k < kTok / 16; ++k) {  // 16 tokens: two groups of 8 rows
          mma_f16(tmem, da + k * (2048 >> 4), db + k * (16 * kRow >> 4), idesc, it > 0 || k > 0);
          mma_f16(tmem, da + k * (2048 >> 4), dl + k * (2048 >> 4), idesc_lo, true);
          if (wg_chunks(BN) > 1)  // after the converted codes
            mma_f16(tmem + 64, da + k * (2048 >> 4), da + ((kCh * kTok * 2 + k * 2048) >> 4), idesc_lo, true);
        }
        // the last ones are not waited for
        if (it + R < nb) mma_commit(empty + 8 * st);
        if (it + G < nb) mma_commit(cempty + 8 * cs);
      }
      __syncwarp();
    }
    if (elect_one()) mma_commit(accf);
    __syncwarp();
  } else if (warp >= 2) {
    // A warp converts 16 tokens of a stage, four at a time: 8 lanes read a
    // token's 128 codes.  Its lo rows then take the place of its own codes, 2048
    // bytes.  Lane l keeps the scale of the warp's token l % 16, in this stage of
    // the group or its next one (l / 16), and asks for the two after them when
    // these begin, so that no stage waits for the load.
    const int w = (warp - 2) & 3, part = lane & 7;
    auto scale_at = [&](int it) {
      const int at = it + (lane >> 4) * G;
      const int t = (b0 + at) * kTok + w * 16 + (lane & 15);
      return at < nb && t < a.T ? __ldcg(a.s + t) : 0.0f;
    };
    const int g = (warp - 2) >> 2;
    const uint32_t dst = ring + g * CB;
    float now = 0.0f, next = scale_at(g);
    int half = 0;
    for (int it = g; it < nb; it += G, half ^= 16) {
      const int st = it % R;
      const uint32_t src = raw + st * RB + w * 2048, dy = raw + st * RB + kGOff + w * 16 * kRow;
      if (half == 0) {
        now = next;
        next = scale_at(it + 2 * G);
      }
      if (!mbar_wait(full + 8 * st, (it / R) & 1)) break;
      if (it >= G && !mbar_wait(cempty + 8 * g, ((it / G) - 1) & 1)) break;
      uint4 code[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) code[i] = lds16a(src + (4 * i + (lane >> 3)) * kCh + part * 16);
      __syncwarp();  // all of the warp's codes are read
      split_rows<DT, kRow>(dy, src, now, half);
      if (wg_chunks(BN) > 1) split_rows<DT, kRow>(dy + kTok * kRow, dst + kCh * kTok * 2 + w * 2048, now, half);
#pragma unroll
      for (int i = 0; i < 4; ++i) put_converted(dst, w * 16 + 4 * i + (lane >> 3), part, code[i]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(conv + 8 * g);
    }
    done = mbar_wait(accf, 0);
    tc_fence_after();
  }

  const int quad = warp & 3, group = (warp - 2) >> 2;  // lanes, and every G-th block of columns
  const int ch = k0 + quad * 32 + lane;
  const int cols = min(BN, a.N - n0);
  const uint32_t trow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
  const uint32_t at = ring + (quad * 32 + lane) * 4;
  if (warp >= 2 && done) {
#pragma unroll 1
    for (int c = 16 * group; c < cols; c += 16 * G) {
      uint32_t v[16];
      tmem_ld16(trow + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (nb == 0) v[i] = 0;
        if (split > 1) {
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + (c + i) * 512), "r"(v[i]) : "memory");
        } else if (ch < a.K && c + i < cols) {
          a.dw[static_cast<int64_t>(n0 + c + i) * a.K + ch] = static_cast<uint16_t>(pack2<DT>(__uint_as_float(v[i]), 0.0f));
        }
      }
    }
  }
  if (split > 1) {
    __syncwarp();
    cluster_sync();
    // Four channels a lane, a column a warp and step.
    if (warp >= 2 && k0 + 4 * lane < a.K) {
      for (int c = rank + split * (warp - 2); c < cols; c += split * 4 * G) {
        uint4 p[8];
        peer_ld_all(ring + c * 512 + lane * 16, split, p);
        float f[4] = {};
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) f[j] += __uint_as_float(word(p[r], j));
        st8(a.dw + static_cast<int64_t>(n0 + c) * a.K + k0 + 4 * lane, make_uint2(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3])));
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
    tmem_free(tmem, wg_tmem(BN));
  }
}

template <int BN, int DT>
static cudaError_t launch_wgrad(const void* dy, const void* q, WgradArgs a, int split, cudaStream_t st) {
  CUtensorMap qmap, gmap;
  cudaError_t e = make_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_NONE, q, a.K, a.T, a.K, kCh, kTok);
  constexpr CUtensorMapSwizzle swizzle = BN >= 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                         : BN == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                    : CU_TENSOR_MAP_SWIZZLE_32B;
  if (e == cudaSuccess)
    e = make_map(&gmap, CU_TENSOR_MAP_DATA_TYPE_UINT16, swizzle, dy, a.ld, a.T, static_cast<uint64_t>(a.ld) * 2, wg_width(BN),
                 kTok);
  if (e == cudaSuccess) e = ensure_smem(int8_wgrad_kernel<BN, DT>, wg_smem(BN), true);
  if (e != cudaSuccess) return e;
  a.ktiles = (a.K + kCh - 1) / kCh;
  const int tiles = a.ktiles * ((a.N + BN - 1) / BN);
  return launch_cluster(int8_wgrad_kernel<BN, DT>, dim3(tiles * split), dim3(kWgThreads), wg_smem(BN), split, st, qmap,
                        gmap, a, split);
}

// The same for many columns, by pairs of CTAs: a tile is 256 channels by 256
// columns, a CTA converts and emits its 128 channels and brings and converts half
// of the columns; the first CTA issues the matrix instructions for both.  Codes,
// dy (then hi) and converted stages (codes, then lo) have rings of their own.  A
// stage's matrix instructions take 1024 cycles, and its bytes about 1280 of shared
// memory's: 4096 tokens, 8192 x 2048 235 us, the matrix units at the measured
// sustained rate 197.
constexpr int kPairCols = 256;
constexpr int kQRing = 3, kDRing = 6, kCRing = 3;
constexpr int kQBytes = kTok * kCh, kDBytes = kPairCols / 2 * kTok * 2, kABytes = kCh * kTok * 2, kCBytes = kABytes + kDBytes;
constexpr int kPairSmem = kQRing * kQBytes + kDRing * kDBytes + kCRing * kCBytes + 1024;
// Copies of dy, matrix instructions, copies of codes, one idle; four warps of
// the epilogue; kCRing groups of four that convert.
constexpr int kPairThreads = 128 + 128 + 128 * kCRing;

template <int DT>
__global__ void __launch_bounds__(kPairThreads, 1)
int8_wgrad_pair_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap gmap,
                       const WgradArgs a, int tiles) {
  // a group meets its stages of every ring in every phase
  static_assert(kQRing % kCRing == 0 && kDRing % kCRing == 0, "");
  constexpr int kBars = 2 * (kQRing + kDRing + kCRing) + 4;
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[kBars];
  __shared__ __align__(128) uint8_t out[4][2][1024];
  __shared__ uint32_t tslot;
  const uint32_t cring = (smem_addr(dyn) + 1023) & ~1023u;
  const uint32_t dring = cring + kCRing * kCBytes, qring = dring + kDRing * kDBytes;
  const uint32_t qfull = smem_addr(bars), qempty = qfull + 8 * kQRing, dfull = qempty + 8 * kQRing;
  const uint32_t dempty = dfull + 8 * kDRing, cfull = dempty + 8 * kDRing, cempty = cfull + 8 * kCRing;
  const uint32_t accf = cempty + 8 * kCRing, acce = accf + 16;
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  if (threadIdx.x == 0) {
    prefetch_map(&qmap);
    prefetch_map(&gmap);
    for (int i = 0; i < kQRing; ++i) {
      mbar_init(qfull + 8 * i, 1);
      mbar_init(qempty + 8 * i, 4);
    }
    for (int i = 0; i < kDRing; ++i) {
      mbar_init(dfull + 8 * i, 1);
      mbar_init(dempty + 8 * i, 1);
    }
    for (int i = 0; i < kCRing; ++i) {
      mbar_init(cfull + 8 * i, 8);
      mbar_init(cempty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(accf + 8 * i, 1);
      mbar_init(acce + 8 * i, 8);
    }
    fence_mbar_init();
  }
  // Both CTAs run, and their barriers are ready, before the pair allocates.
  cluster_sync();
  __syncwarp();
  if (warp == 1) tmem_alloc_pair(smem_addr(&tslot), 2 * kPairCols);
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tslot;
  pdl_wait();
  pdl_trigger();

  const int blocks = (a.T + kTok - 1) / kTok;
  const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;
  const int mine = first < tiles ? (tiles - first + step - 1) / step : 0;
  auto channel0 = [&](int tile) { return (tile % a.ktiles) * 2 * kCh + rank * kCh; };
  auto column0 = [&](int tile) { return (tile / a.ktiles) * kPairCols; };

  if (warp == 0) {
    int it = 0, sent = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step) {
      const int n0 = column0(tile) + rank * (kPairCols / 2);
      for (int t = 0; t < blocks; ++t, ++it) {
        const int st = it % kDRing;
        if (it >= kDRing && !mbar_wait(dempty + 8 * st, ((it / kDRing) - 1) & 1)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(dfull + 8 * st, kDBytes);
#pragma unroll
          for (int c = 0; c < kPairCols / 128; ++c)
            tma_load(dring + st * kDBytes + c * kTok * 128, &gmap, n0 + 64 * c, t * kTok, dfull + 8 * st);
        }
        __syncwarp();
        sent = it + 1;
      }
    }
    if (!ok)  // copies still in flight land before the block ends
      for (int i = sent > kDRing ? sent - kDRing : 0; i < sent; ++i) mbar_wait(dfull + 8 * (i % kDRing), (i / kDRing) & 1);
  } else if (warp == 2) {
    int it = 0, sent = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step) {
      const int k0 = channel0(tile);
      for (int t = 0; t < blocks; ++t, ++it) {
        const int st = it % kQRing;
        if (it >= kQRing && !mbar_wait(qempty + 8 * st, ((it / kQRing) - 1) & 1)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          mbar_arrive_expect_tx(qfull + 8 * st, kQBytes);
          tma_load(qring + st * kQBytes, &qmap, k0, t * kTok, qfull + 8 * st);
        }
        __syncwarp();
        sent = it + 1;
      }
    }
    if (!ok)
      for (int i = sent > kQRing ? sent - kQRing : 0; i < sent; ++i) mbar_wait(qfull + 8 * (i % kQRing), (i / kQRing) & 1);
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = wg_idesc(2 * kCh, kPairCols);
      const uint64_t ca = smem_desc(cring, kTok * 128, 1024), cb = smem_desc(dring, kTok * 128, 1024);
      int it = 0;
      bool ok = true;
      for (int n = 0; ok && n < mine; ++n) {
        const int buf = n & 1;
        if (n >= 2 && !mbar_wait_cluster(acce + 8 * buf, ((n >> 1) - 1) & 1)) break;
        tc_fence_after();
        for (int t = 0; t < blocks; ++t, ++it) {
          const int ds = it % kDRing, cs = it % kCRing;
          if (!mbar_wait_cluster(cfull + 8 * cs, (it / kCRing) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t da = ca + static_cast<uint64_t>(cs * (kCBytes >> 4));
            const uint64_t db = cb + static_cast<uint64_t>(ds * (kDBytes >> 4));
#pragma unroll
            for (int k = 0; k < kTok / 16; ++k) {
              mma_f16_pair(tmem + buf * kPairCols, da + k * (2048 >> 4), db + k * (2048 >> 4), idesc, t > 0 || k > 0);
              mma_f16_pair(tmem + buf * kPairCols, da + k * (2048 >> 4), da + ((kABytes + k * 2048) >> 4), idesc, true);
            }
            // No arrival is under way to the other CTA when a CTA leaves:
            // only those that someone waits for are made.
            if (it + kDRing < mine * blocks) mma_commit_pair(dempty + 8 * ds);
            if (it + kCRing < mine * blocks) mma_commit_pair(cempty + 8 * cs);
          }
          __syncwarp();
        }
        if (elect_one()) mma_commit_pair(accf + 8 * buf);
        __syncwarp();
      }
    }
  } else if (warp >= 8) {
    // As in the kernel above: a warp converts 16 tokens of its group's stages.
    const int w = warp & 3, g = (warp - 8) >> 2, part = lane & 7;
    const int total = mine * blocks;
    const uint32_t cfull0 = peer_addr(cfull, 0);
    auto scale_at = [&](int it) {
      const int at = it + (lane >> 4) * kCRing;
      const int t = (at % blocks) * kTok + w * 16 + (lane & 15);
      return at < total && t < a.T ? __ldcg(a.s + t) : 0.0f;
    };
    float now = 0.0f, next = scale_at(g);
    int half = 0;
    for (int it = g; it < total; it += kCRing, half ^= 16) {
      const int qs = it % kQRing, ds = it % kDRing;
      const uint32_t dst = cring + g * kCBytes, src = qring + qs * kQBytes + w * 2048, dy = dring + ds * kDBytes + w * 2048;
      if (half == 0) {
        now = next;
        next = scale_at(it + 2 * kCRing);
      }
      if (!mbar_wait(qfull + 8 * qs, (it / kQRing) & 1) || !mbar_wait(dfull + 8 * ds, (it / kDRing) & 1)) break;
      if (it >= kCRing && !mbar_wait(cempty + 8 * g, ((it / kCRing) - 1) & 1)) break;
      uint4 code[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) code[i] = lds16a(src + (4 * i + (lane >> 3)) * kCh + part * 16);
#pragma unroll
      for (int c = 0; c < kPairCols / 128; ++c)
        split_rows<DT, 128>(dy + c * kTok * 128, dst + kABytes + c * kTok * 128 + w * 2048, now, half);
#pragma unroll
      for (int i = 0; i < 4; ++i) put_converted(dst, w * 16 + 4 * i + (lane >> 3), part, code[i]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(qempty + 8 * qs);
        mbar_arrive_at(cfull0 + 8 * g);
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3;
    const uint32_t trow = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t acce0 = peer_addr(acce, 0);
    int n = 0;
    for (int tile = first; tile < tiles; tile += step, ++n) {
      const int buf = n & 1, n0 = column0(tile);
      if (!mbar_wait(accf + 8 * buf, (n >> 1) & 1)) break;
      tc_fence_after();
      emit_columns(trow + buf * kPairCols, smem_addr(out[quad][0]), min(kPairCols, a.N - n0),
                   a.dw + static_cast<int64_t>(n0) * a.K, a.K, channel0(tile) + quad * 32,
                   [](int, int, uint32_t lo, uint32_t hi) { return pack2<DT>(__uint_as_float(lo), __uint_as_float(hi)); });
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && tile + 2 * step < tiles) mbar_arrive_at(acce0 + 8 * buf);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_free_pair(tmem, 2 * kPairCols);
  }
  cluster_sync();  // neither CTA leaves while the pair frees
}

template <int DT>
static cudaError_t launch_wgrad_pair(const void* dy, const void* q, WgradArgs a, cudaStream_t st) {
  CUtensorMap qmap, gmap;
  cudaError_t e = make_map(&qmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_NONE, q, a.K, a.T, a.K, kCh, kTok);
  if (e == cudaSuccess)
    e = make_map(&gmap, CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_128B, dy, a.ld, a.T,
                 static_cast<uint64_t>(a.ld) * 2, 64, kTok);
  if (e == cudaSuccess) e = ensure_smem(int8_wgrad_pair_kernel<DT>, kPairSmem);
  if (e != cudaSuccess) return e;
  a.ktiles = (a.K + 2 * kCh - 1) / (2 * kCh);
  const int tiles = a.ktiles * ((a.N + kPairCols - 1) / kPairCols);
  const int grid = 2 * std::min(tiles, device_info().sms / 2);
  return launch_cluster(int8_wgrad_pair_kernel<DT>, dim3(grid), dim3(kPairThreads), kPairSmem, 2, st, qmap, gmap, a, tiles);
}

// Columns of a tile and parts along the tokens, for single CTAs: the narrowest
// tile that holds all columns, up to 128.  Few tiles are split into parts of at
// least two stages: up to 64 columns two blocks share a multiprocessor and 264
// run at once in clusters of eight; above, 132 in clusters of four but only 120
// in clusters of eight (128 columns of 2048 channels: 18.1 us in 4 parts).
static void wgrad_shape(int T, int N, int K, int sms, int* bn, int* split) {
  const int64_t kt = (K + kCh - 1) / kCh;
  int b = 16;
  while (b < 128 && b < N) b *= 2;
  const int64_t tiles = kt * ((N + b - 1) / b);
  const int blocks = (T + kTok - 1) / kTok;
  const int most = b <= 64 ? 8 : 4, fit = b <= 64 ? 2 * sms - 32 : sms - 16;
  int s = 1;
  while (s < most && tiles * s * 2 <= fit && blocks / (2 * s) >= 2) s *= 2;
  *bn = b;
  *split = s;
}

// Whether pairs of CTAs take a gradient of more than 128 columns, by what was
// measured: a pair 4 us and 0.75 a stage and round of tiles, single CTAs 5 us
// and 0.72 a stage of a part and round.  4096 tokens: 2048 x 2048 57 us (101
// single), 1024 x 1024 51 (30).
static bool wgrad_by_pairs(int T, int N, int K, int split, int sms) {
  if (N <= 128) return false;
  const int64_t blocks = (T + kTok - 1) / kTok, kt = (K + kCh - 1) / kCh;
  const int64_t pair_rounds = ((kt + 1) / 2 * ((N + 255) / 256) + sms / 2 - 1) / (sms / 2);
  const int64_t rounds = (kt * ((N + 127) / 128) * split + sms - 1) / sms;
  return 400 + pair_rounds * blocks * 75 < 500 + rounds * (blocks / split) * 72;
}

template <int DT>
static cudaError_t wgrad(const void* dy, const void* q, const WgradArgs& a, cudaStream_t st) {
  const DeviceInfo& d = device_info();
  if (d.error != cudaSuccess) return d.error;
  int bn, split;
  wgrad_shape(a.T, a.N, a.K, d.sms, &bn, &split);
  if (wgrad_by_pairs(a.T, a.N, a.K, split, d.sms)) return launch_wgrad_pair<DT>(dy, q, a, st);
  switch (bn) {
    case 16: return launch_wgrad<16, DT>(dy, q, a, split, st);
    case 32: return launch_wgrad<32, DT>(dy, q, a, split, st);
    case 64: return launch_wgrad<64, DT>(dy, q, a, split, st);
    default: return launch_wgrad<128, DT>(dy, q, a, split, st);
  }
}

// Rows of N elements into rows of ld: the copies of dy need rows of a multiple
// of 16 bytes.  Eight elements a thread; a row may start at an odd place, so the
// aligned words that hold them are shifted into order.  (An element a thread
// took 126 us for 4096 x 8191.)
__global__ void __launch_bounds__(256) pad_rows_kernel(const uint16_t* x, uint16_t* y, int64_t chunks, DivU32 per_row, int N) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= chunks) return;
  const int64_t r = div_u32(per_row, i);
  const int c = static_cast<int>(i - r * per_row.d) * 8;
  const int64_t off = r * N + c;
  uint32_t o[4] = {};
  if (c + 8 < N) {  // the word after the last element is this row's too
    const uint32_t* p = reinterpret_cast<const uint32_t*>(x) + (off >> 1);
    uint32_t w[5];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __ldcg(p + k);
    w[4] = (off & 1) ? __ldcg(p + 4) : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (off & 1) ? __funnelshift_r(w[k], w[k + 1], 16) : w[k];
  } else {
    for (int k = 0; k < 8 && c + k < N; ++k) o[k >> 1] |= static_cast<uint32_t>(x[off + k]) << (16 * (k & 1));
  }
  st16(y + i * 8, make_uint4(o[0], o[1], o[2], o[3]));
}

cudaError_t read_status_int8_wgrad(int* status, bool clear) { return tu_status(status, clear); }

}  // namespace afb

using namespace afb;

extern "C" size_t afb_int8_wgrad_workspace(int64_t rows, int64_t N, int64_t K) {
  (void)K;
  if (rows <= 0 || N <= 0 || N % 8 == 0) return 0;
  if (rows > (1 << 30) || N > (1 << 20)) return SIZE_MAX;
  return static_cast<size_t>(rows) * ((N + 7) / 8 * 8) * 2;
}

extern "C" int afb_int8_wgrad(const void* dy, const void* q, const void* s, void* dw, int64_t rows, int64_t N,
                              int64_t K, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  ApiGuard g("afb_int8_wgrad");
  if (!check(rows >= 0 && rows <= (1 << 30), "rows must be in [0, 2^30]") ||
      !check(N >= 1 && N <= (1 << 20), "N must be in [1, 2^20]") ||
      !check_k(K, 1 << 20) ||
      !check_dtype(dtype) || !check_ptrs({dw}, {"dw"}))
    return g.fail();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) return g.done(cudaMemsetAsync(dw, 0, static_cast<size_t>(N) * K * 2, st));
  if (!check_ptrs({dy, q}, {"dy", "q"}) || !check_ptr4(s, "s") ||
      !check(workspace_bytes >= afb_int8_wgrad_workspace(rows, N, K), "workspace too small"))
    return g.fail();
  WgradArgs a{};
  a.s = static_cast<const float*>(s);
  a.dw = static_cast<uint16_t*>(dw);
  a.T = static_cast<int>(rows);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.ld = static_cast<int>((N + 7) / 8 * 8);
  if (N % 8 != 0) {
    if (!check_ptrs({workspace}, {"workspace"})) return g.fail();
    const int64_t chunks = rows * (a.ld / 8);
    if (!check((chunks + 255) / 256 <= INT64_C(0x7fffffff), "rows * N is too large")) return g.fail();
    const cudaError_t e = launch_pdl(pad_rows_kernel, dim3(static_cast<unsigned>((chunks + 255) / 256)), dim3(256), 0, st,
                                     static_cast<const uint16_t*>(dy), static_cast<uint16_t*>(workspace), chunks,
                                     make_divu32(a.ld / 8), a.N);
    if (e != cudaSuccess) return g.done(e);
    dy = workspace;
  }
  return g.done(dtype == kBf16 ? wgrad<kBf16>(dy, q, a, st) : wgrad<kFp16>(dy, q, a, st));
}
