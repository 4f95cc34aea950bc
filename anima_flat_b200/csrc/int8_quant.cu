// Row quantisation to 8-bit integers, the GELU whose input is kept in 8 bits
// for the backward pass, and the restoring of codes.
//
// Per row of K elements, with a = max(max|y|, 1e-30) (afb::RowScale):
//   s = a / 127,  q = rint(127 y / a)
// where y is the input, the input times a vector over its columns (the
// gradient entering a product with scaled weight rows), or GELU(input).
//
// Quantising is memory bound, 3 bytes an element (8192 x 8192: 31.8 us, floor
// 30.7).  GELU, which writes its own codes and those of its input, 4 bytes, is
// bound by its instructions, 23 an element on 72% of the issue slots (62.7 us,
// floor 41).  A row lives in the registers of a group of
// GROUP warps from its only read to the write of its codes; 16 elements a
// thread and step make each access 16 bytes wide.
#include "int8_common.cuh"

namespace afb {

struct QuantArgs {
  const uint16_t* x;  // [rows, K]
  const float* cols;  // [K] or null: factors of the columns
  int8_t* q;          // [rows, K]: codes of x, x * cols or GELU(x)
  float* s;           // [rows]
  int8_t* c;          // GELU only: codes of x, and their scales
  float* cs;
  int64_t rows;
  int K;
};

enum QuantMode { kPlain = 0, kCols = 1, kGelu = 2 };  // kGelu has its own kernel

__host__ __device__ constexpr int quant_block_warps(int group) { return group > 4 ? group : 4; }

template <int CPL, int GROUP, int DT, int MODE>
__global__ void __launch_bounds__(quant_block_warps(GROUP) * 32)
rowquant_int8_kernel(const QuantArgs a) {
  constexpr int BW = quant_block_warps(GROUP);
  __shared__ uint32_t red[BW];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int t = (warp % GROUP) * 32 + lane;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (BW / GROUP) + warp / GROUP;
  const bool row_ok = row < a.rows;
  const int K = a.K;
  const int64_t base = (row_ok ? row : 0) * K;

  uint4 xv[CPL][2];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 16;
    const bool ok = row_ok && e < K;
    xv[c][0] = ok ? ld_stream(a.x + base + e) : make_uint4(0, 0, 0, 0);
    xv[c][1] = ok ? ld_stream(a.x + base + e + 8) : make_uint4(0, 0, 0, 0);
  }
  f2_t y[CPL][2][4];
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 16;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
      if (MODE == kCols) {
        const bool ok = row_ok && e < K;
        const float4 lo = ok ? ld_keep_f4(a.cols + e + 8 * h) : make_float4(0, 0, 0, 0);
        const float4 hi = ok ? ld_keep_f4(a.cols + e + 8 * h + 4) : make_float4(0, 0, 0, 0);
        f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
        f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2_t v = unpack2<DT>(word(xv[c][h], j));
        y[c][h][j] = MODE == kCols ? mul2(v, f2(f[2 * j], f[2 * j + 1])) : v;
        amax = max_abs_nan(amax, y[c][h][j]);
      }
    }
  }
  uint32_t top = warp_max_u32(__float_as_uint(amax));
  if (GROUP > 1) {
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = group_max_u32<GROUP>(&red[(warp / GROUP) * GROUP]);
  }
  if (!row_ok) return;
  const RowScale r = row_scale(top);
  if (t == 0) a.s[row] = scale_value(top);
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 16;
    if (e >= K) continue;
    const uint2 lo = codes8(y[c][0], r), hi = codes8(y[c][1], r);
    st16(a.q + base + e, make_uint4(lo.x, lo.y, hi.x, hi.y));
  }
}

// GELU of a pair (erf form), by Abramowitz & Stegun 7.1.26: with r = poly(t)
// exp(-x^2 / 2), 1 - erf(|x| / sqrt 2) up to 1.5e-7,
//   gelu(x) = max(x, 0) - |x| r / 2,
// which nothing cancels below zero: there it is -|x| r / 2, within 2^-8 of GELU
// down to -6 (r's relative error), where x / 2 (1 + erf) would keep a step of
// 2^-24 |x|, more than GELU itself.  A row with nothing larger takes its scale and
// codes from such values.
__device__ __forceinline__ f2_t gelu2(f2_t x) {
  constexpr f2_t kAbs = 0x7fffffff7fffffffull;
  const f2_t hx = mul2(x, splat2(0.5f)), hax = hx & kAbs;
  const f2_t den = fma2(hax, splat2(2.0f * (0.3275911f * 0.707106769084930419921875f)), splat2(1.0f));
  float t0, t1, e0, e1;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(f2lo(den)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(f2hi(den)));
  const f2_t t = f2(t0, t1);
  f2_t n = fma2(splat2(-1.061405429f), t, splat2(1.453152027f));  // n = -poly(t)
  n = fma2(n, t, splat2(-1.421413741f));
  n = fma2(n, t, splat2(0.284496736f));
  n = fma2(n, t, splat2(-0.254829592f));
  n = mul2(n, t);
  const f2_t arg = mul2(mul2(x, x), splat2(-0.721347520444481703680f));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(f2lo(arg)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(f2hi(arg)));
  return fma2(hax, mul2(n, f2(e0, e1)), add2(hx, hax));  // x / 2 + |x| / 2 is exact
}

// GELU and its input's codes.  |GELU| is at most 0.17 below zero and increases
// above it, so from x = 0.34 on the row's largest |GELU| is that of its largest
// x: the row's scale is known before any GELU is formed, and each is formed and
// coded on the spot, where holding them until a maximum is known took 57
// registers a thread.  A row without such an x forms them twice.
template <int CPL, int GROUP, int DT>
__global__ void __launch_bounds__(quant_block_warps(GROUP) * 32)
gelu_int8_kernel(const QuantArgs a) {
  constexpr int BW = quant_block_warps(GROUP);
  __shared__ uint32_t red[3][BW];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int t = (warp % GROUP) * 32 + lane, w0 = (warp / GROUP) * GROUP;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (BW / GROUP) + warp / GROUP;
  const bool row_ok = row < a.rows;
  const int K = a.K;
  const int64_t base = (row_ok ? row : 0) * K;
  // The group's maximum; its warps alone meet.
  auto group_max = [&](float v, int buf) {
    uint32_t m = warp_max_u32(__float_as_uint(v));
    if (GROUP > 1) {
      if (lane == 0) red[buf][warp] = m;
      named_bar_sync(1 + warp / GROUP, GROUP * 32);
      m = group_max_u32<GROUP>(&red[buf][w0]);
    }
    return m;
  };

  uint4 xv[CPL][2];
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 16;
    const bool ok = row_ok && e < K;
    xv[c][0] = ok ? ld_stream(a.x + base + e) : make_uint4(0, 0, 0, 0);
    xv[c][1] = ok ? ld_stream(a.x + base + e + 8) : make_uint4(0, 0, 0, 0);
  }
  float amax = 0.0f, pmax = 0.0f;  // of |x|, and of x above zero
#pragma unroll
  for (int c = 0; c < CPL; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const f2_t v = unpack2<DT>(word(xv[c][j >> 2], j & 3));
      amax = max_abs_nan(amax, v);
      pmax = fmaxf(pmax, fmaxf(f2lo(v), f2hi(v)));
    }
  const uint32_t top = group_max(amax, 0);
  const float most = __uint_as_float(group_max(pmax, 1));
  uint32_t gtop = __float_as_uint(f2lo(gelu2(splat2(most))));
  if (top >= 0x7f800000u) {
    gtop = top;
  } else if (most < 0.34f) {
    float g = 0.0f;
#pragma unroll
    for (int c = 0; c < CPL; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) g = max_abs_nan(g, gelu2(unpack2<DT>(word(xv[c][j >> 2], j & 3))));
    gtop = group_max(g, 2);
  }
  if (!row_ok) return;
  const RowScale rg = row_scale(gtop), rx = row_scale(top);
  if (t == 0) {
    a.s[row] = scale_value(gtop);
    a.cs[row] = scale_value(top);
  }
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 16;
    if (e >= K) continue;
    uint2 q[2], x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f2_t v[4], g[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = unpack2<DT>(word(xv[c][h], j));
        g[j] = gelu2(v[j]);
      }
      q[h] = codes8<false>(g, rg);
      x[h] = codes8(v, rx);
    }
    st16(a.q + base + e, make_uint4(q[0].x, q[0].y, q[1].x, q[1].y));
    st16(a.c + base + e, make_uint4(x[0].x, x[0].y, x[1].x, x[1].y));
  }
}

// Warps of a row's group and chunks of 16 a thread.  The plain forms take two
// chunks a thread (one where 32 threads hold the row): 8192 rows of 8192 take
// 31.8 us so, 40.5 with one, which waits on twice the warps.  GELU takes one up
// to 8 warps (4096 x 2048: 10.2 us, 2.3 more with two) and two from there on
// (8192 x 8192: 62.7 us with 8 warps, 14 more with 16).
template <int MODE>
static bool quant_shape(int64_t K, int* group, int* cpl) {
  const int64_t chunks = K / 16;
  int g = 1;
  if (MODE == kGelu)
    while (g < 8 && chunks > 32 * g) g <<= 1;
  while (g < 16 && chunks > 64 * g) g <<= 1;
  *group = g;
  *cpl = chunks > 32 * g ? 2 : 1;
  return K >= 16 && K % 16 == 0 && chunks <= 64 * g;
}
// Which of them quant_shape gives: one chunk with one warp, or for GELU with up
// to 8; two with any number, for GELU with 8 and 16.
template <int MODE, int GROUP, int CPL>
constexpr bool quant_used() {
  if (MODE == kGelu) return CPL == 1 ? GROUP <= 8 : GROUP >= 8;
  return CPL == 2 || GROUP == 1;
}

template <int CPL, int GROUP, int DT, int MODE>
static auto quant_kernel() {
  if constexpr (MODE == kGelu) return gelu_int8_kernel<CPL, GROUP, DT>;
  else return rowquant_int8_kernel<CPL, GROUP, DT, MODE>;
}
template <int GROUP, int DT, int MODE>
static cudaError_t launch_quant_g(const QuantArgs& a, int cpl, cudaStream_t st) {
  constexpr int BW = quant_block_warps(GROUP);
  const int64_t per = BW / GROUP;
  const dim3 grid(static_cast<unsigned>((a.rows + per - 1) / per)), block(BW * 32);
  if constexpr (quant_used<MODE, GROUP, 2>())
    if (cpl == 2) return launch_pdl(quant_kernel<2, GROUP, DT, MODE>(), grid, block, 0, st, a);
  if constexpr (quant_used<MODE, GROUP, 1>())
    if (cpl == 1) return launch_pdl(quant_kernel<1, GROUP, DT, MODE>(), grid, block, 0, st, a);
  return cudaErrorInvalidValue;
}

template <int DT, int MODE>
static cudaError_t launch_quant(const QuantArgs& a, cudaStream_t st) {
  int group = 0, cpl = 0;
  if (!quant_shape<MODE>(a.K, &group, &cpl)) return cudaErrorInvalidValue;
  switch (group) {
    case 1: return launch_quant_g<1, DT, MODE>(a, cpl, st);
    case 2: return launch_quant_g<2, DT, MODE>(a, cpl, st);
    case 4: return launch_quant_g<4, DT, MODE>(a, cpl, st);
    case 8: return launch_quant_g<8, DT, MODE>(a, cpl, st);
    default: return launch_quant_g<16, DT, MODE>(a, cpl, st);
  }
}

cudaError_t quantize_rows(const void* x, const void* cols, int8_t* q, float* s, int64_t rows, int64_t K, int dtype,
                          cudaStream_t st) {
  QuantArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.cols = static_cast<const float*>(cols);
  a.q = q;
  a.s = s;
  a.rows = rows;
  a.K = static_cast<int>(K);
  if (cols != nullptr) return dtype == kBf16 ? launch_quant<kBf16, kCols>(a, st) : launch_quant<kFp16, kCols>(a, st);
  return dtype == kBf16 ? launch_quant<kBf16, kPlain>(a, st) : launch_quant<kFp16, kPlain>(a, st);
}

// ------------------------------------------------------------ restore, GELU' --
struct RestoreArgs {
  const int8_t* q;     // [rows, K]
  const float* s;      // [rows]
  const uint16_t* dy;  // GELU' only: [rows, K]
  uint16_t* y;         // [rows, K]
  int64_t chunks;      // rows * K / 16
  DivU32 per_row;      // K / 16
};

// d/dv of v * Phi(v) = Phi(v) + v phi(v), with erf by Abramowitz & Stegun
// 7.1.26 (|error| <= 1.5e-7): for a = |v| / sqrt 2, t = 1 / (1 + p a),
// 1 - erf(a) = poly(t) exp(-a^2), and phi(v) holds the same exponential.
__device__ __forceinline__ float gelu_slope(float v) {
  const float a = fabsf(v);
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(__fmaf_rn(a, 0.3275911f * 0.707106769084930419921875f, 1.0f)));
  float p = __fmaf_rn(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
  p = __fmaf_rn(p, t, 0.5f * 1.421413741f);
  p = __fmaf_rn(p, t, 0.5f * -0.284496736f);
  p = __fmaf_rn(p, t, 0.5f * 0.254829592f);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((v * v) * -0.721347520444481703680f));
  const float tail = p * t * e;  // 1 - Phi(|v|)
  const float cdf = v < 0.0f ? tail : 1.0f - tail;
  return __fmaf_rn(v * 0.3989422804014327f, e, cdf);
}

template <int DT, bool SLOPE>
__global__ void __launch_bounds__(256) restore_kernel(const RestoreArgs a) {
  pdl_wait();
  pdl_trigger();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.chunks) return;
  const uint4 qv = ld_stream(a.q + i * 16);
  uint4 g[2] = {};
  if (SLOPE) {
    g[0] = ld_stream(a.dy + i * 16);
    g[1] = ld_stream(a.dy + i * 16 + 8);
  }
  const float s = __ldcg(a.s + div_u32(a.per_row, i));
  uint4 o[2];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const f2_t v = mul2(code_pair(word(qv, k >> 1), k & 1), splat2(s));
    uint32_t& w = word_ref(o[k >> 2], k & 3);
    if (SLOPE) {
      const f2_t d = unpack2<DT>(word(g[k >> 2], k & 3));
      w = pack2<DT>(f2lo(d) * gelu_slope(f2lo(v)), f2hi(d) * gelu_slope(f2hi(v)));
    } else {
      w = pack2<DT>(v);
    }
  }
  st16(a.y + i * 16, o[0]);
  st16(a.y + i * 16 + 8, o[1]);
}

template <bool SLOPE>
static cudaError_t launch_restore(const RestoreArgs& a, int dtype, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((a.chunks + 255) / 256));
  return dtype == kBf16 ? launch_pdl(restore_kernel<kBf16, SLOPE>, grid, dim3(256), 0, st, a)
                        : launch_pdl(restore_kernel<kFp16, SLOPE>, grid, dim3(256), 0, st, a);
}

// rows * K / 16 chunks of 256-thread blocks must fit the grid's x extent.
static bool check_quant(int64_t rows, int64_t K, int dtype) {
  return check(rows >= 0 && rows <= INT64_C(0x7fffffff), "rows must be in [0, 2^31)") && check_k(K, 16384) &&
         check_dtype(dtype);
}

}  // namespace afb

using namespace afb;

extern "C" int afb_rowquant_int8(const void* x, const void* cols, void* q, void* s, int64_t rows, int64_t K,
                                 int dtype, void* stream) {
  ApiGuard g("afb_rowquant_int8");
  if (!check_quant(rows, K, dtype)) return g.fail();
  if (rows == 0) return 0;
  if (!check_ptrs({x, q}, {"x", "q"}) || !check_ptr4(s, "s") ||
      !check(cols == nullptr || aligned(cols, 16), "cols is not 16-byte aligned"))
    return g.fail();
  return g.done(quantize_rows(x, cols, static_cast<int8_t*>(q), static_cast<float*>(s), rows, K, dtype,
                              static_cast<cudaStream_t>(stream)));
}

extern "C" int afb_gelu_int8(const void* x, void* q, void* s, void* c, void* cs, int64_t rows, int64_t K,
                             int dtype, void* stream) {
  ApiGuard g("afb_gelu_int8");
  if (!check_quant(rows, K, dtype)) return g.fail();
  if (rows == 0) return 0;
  if (!check_ptrs({x, q, c}, {"x", "q", "c"}) || !check_ptr4(s, "s") || !check_ptr4(cs, "cs")) return g.fail();
  QuantArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.q = static_cast<int8_t*>(q);
  a.s = static_cast<float*>(s);
  a.c = static_cast<int8_t*>(c);
  a.cs = static_cast<float*>(cs);
  a.rows = rows;
  a.K = static_cast<int>(K);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g.done(dtype == kBf16 ? launch_quant<kBf16, kGelu>(a, st) : launch_quant<kFp16, kGelu>(a, st));
}

static int restore(const char* name, const void* dy, const void* q, const void* s, void* y, int64_t rows, int64_t K,
                   int dtype, void* stream) {
  ApiGuard g(name);
  if (!check_quant(rows, K, dtype)) return g.fail();
  if (rows == 0) return 0;
  if (!check_ptrs({q, y}, {"q", "y"}) || !check_ptr4(s, "s") ||
      !check(dy == nullptr || aligned(dy, 16), "dy is not 16-byte aligned"))
    return g.fail();
  RestoreArgs a{};
  a.q = static_cast<const int8_t*>(q);
  a.s = static_cast<const float*>(s);
  a.dy = static_cast<const uint16_t*>(dy);
  a.y = static_cast<uint16_t*>(y);
  a.chunks = rows * (K / 16);
  a.per_row = make_divu32(K / 16);
  if (!check((a.chunks + 255) / 256 <= INT64_C(0x7fffffff), "rows * K is too large")) return g.fail();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g.done(dy != nullptr ? launch_restore<true>(a, dtype, st) : launch_restore<false>(a, dtype, st));
}

extern "C" int afb_int8_restore(const void* q, const void* s, void* y, int64_t rows, int64_t K, int dtype,
                                void* stream) {
  return restore("afb_int8_restore", nullptr, q, s, y, rows, K, dtype, stream);
}

extern "C" int afb_gelu_int8_bwd(const void* dy, const void* c, const void* cs, void* dx, int64_t rows, int64_t K,
                                 int dtype, void* stream) {
  ApiGuard g("afb_gelu_int8_bwd");
  if (rows != 0 && !check(dy != nullptr, "dy is null")) return g.fail();
  return restore("afb_gelu_int8_bwd", dy, c, cs, dx, rows, K, dtype, stream);
}
