// Weight gradient from 8-bit checkpoints:
//   dw[n, k] = sum_t dy[t, n] (q[t, k] s[t])
// over the tokens t, with the codes and scales that the forward product read.
#include "int8_common.cuh"

namespace afb {

struct WgradArgs {
  const uint16_t* dy;  // [T, N]
  const int8_t* q;     // [T, K]
  const float* s;      // [T]
  uint16_t* dw;        // [N, K]
  int T, N, K;
};

// 64 x 64 outputs a block of 256 threads, 16 tokens a step, fp32.
template <int DT>
__global__ void __launch_bounds__(256) int8_wgrad_kernel(const WgradArgs a) {
  __shared__ float dy[16][65], x[16][65];
  pdl_wait();
  pdl_trigger();
  const int n0 = blockIdx.y * 64, k0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int t0 = 0; t0 < a.T; t0 += 16) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int t = t0 + i / 64, c = i % 64;
      dy[i / 64][c] = t < a.T && n0 + c < a.N ? load1<DT>(a.dy + static_cast<int64_t>(t) * a.N + n0 + c) : 0.0f;
      x[i / 64][c] = t < a.T && k0 + c < a.K
                         ? static_cast<float>(a.q[static_cast<int64_t>(t) * a.K + k0 + c]) * __ldg(a.s + t) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(dy[t][ty + 16 * i], x[t][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + ty + 16 * i, k = k0 + tx + 16 * j;
      if (n < a.N && k < a.K)
        a.dw[static_cast<int64_t>(n) * a.K + k] = static_cast<uint16_t>(pack2<DT>(acc[i][j], 0.0f));
    }
}

}  // namespace afb

using namespace afb;

extern "C" int afb_int8_wgrad(const void* dy, const void* q, const void* s, void* dw, int64_t rows, int64_t N,
                              int64_t K, int dtype, void* stream) {
  ApiGuard g("afb_int8_wgrad");
  if (!check(rows >= 0 && rows <= (1 << 30), "rows must be in [0, 2^30]") ||
      !check(N >= 8 && N % 8 == 0 && N <= (1 << 20), "N must be a multiple of 8 in [8, 2^20], got " + std::to_string(N)) ||
      !check(K >= 16 && K % 16 == 0 && K <= (1 << 20), "K must be a multiple of 16 in [16, 2^20], got " + std::to_string(K)) ||
      !check_dtype(dtype) || !check_ptrs({dw}, {"dw"}))
    return g.fail();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows != 0 && (!check_ptrs({dy, q}, {"dy", "q"}) || !check_ptr4(s, "s"))) return g.fail();
  WgradArgs a{static_cast<const uint16_t*>(dy), static_cast<const int8_t*>(q), static_cast<const float*>(s),
              static_cast<uint16_t*>(dw), static_cast<int>(rows), static_cast<int>(N), static_cast<int>(K)};
  const dim3 grid(static_cast<unsigned>((K + 63) / 64), static_cast<unsigned>((N + 63) / 64));
  return g.done(dtype == kBf16 ? launch_pdl(int8_wgrad_kernel<kBf16>, grid, dim3(256), 0, st, a)
                               : launch_pdl(int8_wgrad_kernel<kFp16>, grid, dim3(256), 0, st, a));
}
