// Shared by the 8-bit integer and sandwich-norm kernels: the two 16-bit
// activation types, and the row quantisation to 8-bit codes.
#pragma once

#include <cuda_fp16.h>

#include "afb_device.cuh"
#include "afb_launch.h"

namespace afb {

// The 16-bit types of an activation; the values are the C ABI's dtype codes.
constexpr int kBf16 = 0;
constexpr int kFp16 = 1;

template <int DT>
__device__ __forceinline__ f2_t unpack2(uint32_t w) {
  if (DT == kBf16) return bf2f2(w);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return f2(f.x, f.y);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (DT == kBf16) return pack2_rn(lo, hi);
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(f2_t v) {
  return pack2<DT>(f2lo(v), f2hi(v));
}
template <int DT>
__device__ __forceinline__ float load1(const uint16_t* p) {
  const uint32_t w = __ldg(p);
  return f2lo(unpack2<DT>(w));
}

// Integer maximum of the bit patterns of non-negative floats: it orders
// finite < infinity < NaN, so a row with a non-finite value keeps it.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t max_bits2(uint32_t m, f2_t v) {
  return max(m, max(abs_bits(f2lo(v)), abs_bits(f2hi(v))));
}
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) { return __reduce_max_sync(kFull, v); }

// Row quantisation.  With a = max(max|y|, 1e-30):
//   s = a / 127,  q = rint(127 y / a), half to even.
// A row with a non-finite value gets the non-finite scale and zero codes, so
// whatever is computed from it is NaN.
//
// The codes are those of the IEEE quotient RN(RN(127 y) / a) without a
// division per element: t = y * RN(127 / a) is within 127 * 3 * 2^-24 < 2.3e-5
// of it, so rint(t) is the code unless t lies within 5e-5 of a half; a vector
// with such an element takes the division.  For a 16-bit y both 127 y and the
// ties are exact in fp32, so the code is the exactly rounded one.
struct RowScale {
  float a;    // max(max|y|, 1e-30)
  float inv;  // 127 / a, or 0 for a row with a non-finite value
  float s;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  RowScale r;
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) {
    r.a = 1.0f;
    r.inv = 0.0f;
    r.s = __fdiv_rn(amax, 127.0f);
  } else {
    r.a = fmaxf(amax, 1e-30f);
    r.inv = __fdiv_rn(127.0f, r.a);
    r.s = __fdiv_rn(r.a, 127.0f);
  }
  return r;
}

// The quotient for one element.  Rows of values near the top of the fp32
// range are scaled down by a power of two, which changes no quotient of
// interest and keeps 127 y finite.
static __device__ __noinline__ int code_exact(float y, RowScale r) {
  if (r.inv == 0.0f) return 0;
  const float k = r.a > 0x1p100f ? 0x1p-20f : 1.0f;
  return static_cast<int>(rintf(__fdiv_rn(__fmul_rn(127.0f, __fmul_rn(y, k)), __fmul_rn(r.a, k))));
}

// Eight codes of four pairs, element k in byte k.
__device__ __forceinline__ uint2 codes8(const f2_t (&y)[4], const RowScale& r) {
  const f2_t inv = splat2(r.inv);
  const f2_t magic = splat2(12582912.0f);  // 1.5 * 2^23: the sum's low byte is the code
  uint32_t w[8];
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f2_t t = mul2(y[j], inv);
    const f2_t m = add2(t, magic);
    const f2_t e = sub2(t, sub2(m, magic));
    far = max_abs2(far, f2lo(e), f2hi(e));
    w[2 * j] = __float_as_uint(f2lo(m));
    w[2 * j + 1] = __float_as_uint(f2hi(m));
  }
  if (far > 0.49995f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[2 * j] = static_cast<uint32_t>(code_exact(f2lo(y[j]), r));
      w[2 * j + 1] = static_cast<uint32_t>(code_exact(f2hi(y[j]), r));
    }
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410);
  // t is NaN where a non-finite element met the zero factor
  if (r.inv == 0.0f) o = make_uint2(0, 0);
  return o;
}

// Two codes (bytes 2j and 2j+1 of w) as floats.
__device__ __forceinline__ f2_t code_pair(uint32_t w, int j) {
  const int v = static_cast<int>(w);
  return j == 0 ? f2(static_cast<float>(static_cast<int8_t>(v)), static_cast<float>(static_cast<int8_t>(v >> 8)))
                : f2(static_cast<float>(static_cast<int8_t>(v >> 16)), static_cast<float>(v >> 24));
}

// Codes and scales of x, or of x * cols where cols is not null (int8_quant.cu).
cudaError_t quantize_rows(const void* x, const void* cols, int8_t* q, float* s, int64_t rows, int64_t K, int dtype,
                          cudaStream_t st);

inline bool check_dtype(int dtype) { return check(dtype == kBf16 || dtype == kFp16, "dtype must be 0 (bf16) or 1 (fp16)"); }

}  // namespace afb
