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

// max(m, |lo|, |hi|) in one three-input maximum; NaN stays NaN.
__device__ __forceinline__ float max_abs_nan(float m, f2_t v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(f2lo(v))), "f"(fabsf(f2hi(v))));
  return r;
}
// Maximum over the warp of bit patterns of non-negative floats: it orders
// finite < infinity < NaN, so a row with a non-finite value keeps it.
__device__ __forceinline__ uint32_t warp_max_u32(uint32_t v) { return __reduce_max_sync(kFull, v); }
// The group's maximum from its warps' in red[0 .. GROUP).
template <int GROUP>
__device__ __forceinline__ uint32_t group_max_u32(const uint32_t* red) {
  return warp_max_u32(red[(threadIdx.x & 31) % GROUP]);
}

// Row quantisation.  With a = max(max|y|, 1e-30):
//   s = a / 127,  q = rint(127 y / a), half to even.
// A row with a non-finite value gets the non-finite scale and zero codes, so
// whatever is computed from it is NaN.
//
// The quotient is formed without a division, by Markstein's correction ("IA-64
// and Elementary Functions", 2000): with c = RN(127 y), t1 = RN(y (127 rcp(a)))
// and the exact remainder r = c - t1 a, t = RN(t1 + r rcp(a)) is c / a to half a
// unit in its last place and 2^-40.  A 16-bit y makes c exact, a tie c / a =
// n + 1/2 comes out as itself, and any other quotient is further from a tie
// than t from the quotient, so the code is the exactly rounded one.  A test of
// each vector for elements near a tie, with a division for those, took 1.6
// times as long in all: among 16-bit values exact ties are common.
struct RowScale {
  float a;    // max(max|y|, 1e-30)
  float rcp;  // 1 / a nearly, or 0 for a row with a non-finite value
  bool big;   // near the top of the fp32 range: y and a are to be scaled down
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  RowScale r;
  const float amax = __uint_as_float(amax_bits);
  const bool finite = amax_bits < 0x7f800000u;
  r.big = finite && amax > 0x1p100f;
  r.a = finite ? fmaxf(r.big ? amax * 0x1p-20f : amax, 1e-30f) : 1.0f;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r.rcp) : "f"(r.a));
  if (!finite) r.rcp = 0.0f;
  return r;
}
// The row's scale, from the same maximum.
__device__ __forceinline__ float scale_value(uint32_t amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  return __fdiv_rn(amax_bits < 0x7f800000u ? fmaxf(amax, 1e-30f) : amax, 127.0f);
}

// Eight codes of four pairs, element k in byte k.  EXACT: by the corrected
// quotient; else rint(y (127 rcp(a))), within 3.1e-5 of the quotient, for values
// that are approximations themselves.
template <bool EXACT = true>
__device__ __forceinline__ uint2 codes8(const f2_t (&y)[4], const RowScale& r) {
  if (r.rcp == 0.0f) return make_uint2(0, 0);
  f2_t v[4] = {y[0], y[1], y[2], y[3]};
  if (r.big) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], splat2(0x1p-20f));
  }
  const f2_t inv = splat2(127.0f * r.rcp), rcp = splat2(r.rcp), na = splat2(-r.a);
  const f2_t magic = splat2(12582912.0f);  // 1.5 * 2^23: the sum's low byte is the code
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f2_t t1 = mul2(v[j], inv);
    f2_t t = t1;
    if (EXACT) t = fma2(fma2(t1, na, mul2(v[j], splat2(127.0f))), rcp, t1);
    const f2_t m = add2(t, magic);
    w[2 * j] = __float_as_uint(f2lo(m));
    w[2 * j + 1] = __float_as_uint(f2hi(m));
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410);
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

// The length of a row of codes.  (The message is made only where it is needed.)
inline bool check_k(int64_t K, int64_t most) {
  return (K >= 16 && K % 16 == 0 && K <= most) ||
         check(false, "K must be a multiple of 16 in [16, " + std::to_string(most) + "], got " + std::to_string(K));
}
inline bool check_dtype(int dtype) { return check(dtype == kBf16 || dtype == kFp16, "dtype must be 0 (bf16) or 1 (fp16)"); }

}  // namespace afb
