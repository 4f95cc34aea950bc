// Matrix product in 8-bit integers with a scale per token and per channel:
//   y[m, n] = (sum_k q[m, k] w[n, k]) * s[m] * v[n] + bias[n]
// The sum is exact in 32-bit integers (K <= 131072: 127^2 K < 2^31).
#include "int8_common.cuh"

namespace afb {

struct LinearArgs {
  const int8_t* q;       // [M, K]
  const float* s;        // [M]
  const int8_t* w;       // [N, K]
  const float* v;        // [N]
  const uint16_t* bias;  // [N] or null
  uint16_t* y;           // [M, N]
  int M, N, K;
};

// 64 x 64 outputs a block of 256 threads, 64 k a step, dp4a.
template <int DT>
__global__ void __launch_bounds__(256) int8_linear_kernel(const LinearArgs a) {
  __shared__ int aq[64][17], bw[64][17];
  pdl_wait();
  pdl_trigger();
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 4;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 64) {
    const bool kok = k0 + lc * 4 < a.K;
    const int4 z = make_int4(0, 0, 0, 0);
    const int4 qa = kok && m0 + lr < a.M
                        ? *reinterpret_cast<const int4*>(a.q + static_cast<int64_t>(m0 + lr) * a.K + k0 + lc * 4) : z;
    const int4 wa = kok && n0 + lr < a.N
                        ? *reinterpret_cast<const int4*>(a.w + static_cast<int64_t>(n0 + lr) * a.K + k0 + lc * 4) : z;
    aq[lr][lc] = qa.x; aq[lr][lc + 1] = qa.y; aq[lr][lc + 2] = qa.z; aq[lr][lc + 3] = qa.w;
    bw[lr][lc] = wa.x; bw[lr][lc + 1] = wa.y; bw[lr][lc + 2] = wa.z; bw[lr][lc + 3] = wa.w;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(aq[ty + 16 * i][k], bw[tx + 16 * j][k], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= a.M || n >= a.N) continue;
      float f = static_cast<float>(acc[i][j]) * __ldg(a.s + m) * __ldg(a.v + n);
      if (a.bias != nullptr) f += load1<DT>(a.bias + n);
      a.y[static_cast<int64_t>(m) * a.N + n] = static_cast<uint16_t>(pack2<DT>(f, 0.0f));
    }
}

}  // namespace afb

using namespace afb;

extern "C" int afb_int8_linear(const void* q, const void* s, const void* w, const void* v, const void* bias, void* y,
                               int64_t M, int64_t N, int64_t K, int dtype, void* stream) {
  ApiGuard g("afb_int8_linear");
  if (!check(M >= 0 && M <= (1 << 30), "M must be in [0, 2^30]") || !check(N >= 1 && N <= (1 << 30), "N must be in [1, 2^30]") ||
      !check(K >= 16 && K % 16 == 0 && K <= 131072, "K must be a multiple of 16 in [16, 131072], got " + std::to_string(K)) ||
      !check_dtype(dtype))
    return g.fail();
  if (M == 0) return 0;
  if (!check_ptrs({q, w}, {"q", "w"}) || !check_ptr4(s, "s") || !check_ptr4(v, "v") ||
      !check(y != nullptr && aligned(y, 2), "y is null or not 2-byte aligned") ||
      !check(aligned(bias, 2), "bias is not 2-byte aligned"))
    return g.fail();
  LinearArgs a{static_cast<const int8_t*>(q), static_cast<const float*>(s), static_cast<const int8_t*>(w),
               static_cast<const float*>(v), static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(y),
               static_cast<int>(M), static_cast<int>(N), static_cast<int>(K)};
  const dim3 grid(static_cast<unsigned>((N + 63) / 64), static_cast<unsigned>((M + 63) / 64));
  if (!check(grid.y <= 65535, "M is too large")) return g.fail();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g.done(dtype == kBf16 ? launch_pdl(int8_linear_kernel<kBf16>, grid, dim3(256), 0, st, a)
                               : launch_pdl(int8_linear_kernel<kFp16>, grid, dim3(256), 0, st, a));
}
