// Norms before and after a block, fused with its gate and residual scale.
//
// Per row of D elements, b = row / S, rms(v) = v / sqrt(mean(v^2) + eps):
//   z = round(alpha * res + gate_b * (rms(x) * post))
//   h = rms(z) * pre * scale_b + shift_b
// x is the block's output, post the norm after it, pre the norm before the
// next block.  h is formed from z as stored, so the backward pass, which has
// z alone, differentiates exactly what was computed.
//
// Backward, with xh = rms(x), zh = rms(z), r1, r2 the reciprocal roots:
//   p = gh scale pre;   dz = gz + r2 (p - zh mean(p zh));  dres = alpha dz
//   m = dz gate post;   dx = r1 (m - xh mean(m xh))
//   P = sum_t gh zh, Q = sum_t dz xh, sum_t gh     over the rows of b
//   dscale = pre P, dpre = sum_b scale P, dgate = post Q, dpost = sum_b gate Q
//
// Sums and statistics are fp32, in an order that the shape alone fixes.
#include "int8_common.cuh"

namespace afb {

// Factors of the columns: a per-sample vector of the activations' type, or
// null for a constant.
struct SandwichArgs {
  const uint16_t* x;      // [B*S, D]
  const uint16_t* res;    // [B*S, D]
  const uint16_t* gate;   // [B, D] or null (1)
  const float* post;      // [D]
  const float* pre;       // [D]
  const uint16_t* shift;  // [B, D] or null (0)
  const uint16_t* scale;  // [B, D] or null (1)
  uint16_t* h;            // [B*S, D]
  uint16_t* z;            // [B*S, D]
  int8_t* q;              // codes of h instead of h
  float* s;
  int64_t rows;
  DivU32 seq;
  int D;
  float alpha, eps;
};

template <int DT>
__device__ __forceinline__ void load8(const uint16_t* p, float fallback, float (&f)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = fallback;
    return;
  }
  const uint4 v = ld_keep(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f2_t t = unpack2<DT>(word(v, j));
    f[2 * j] = f2lo(t);
    f[2 * j + 1] = f2hi(t);
  }
}
__device__ __forceinline__ void load8f(const float* p, float (&f)[8]) {
  const float4 lo = ld_keep_f4(p), hi = ld_keep_f4(p + 4);
  f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
  f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
}
template <int DT>
__device__ __forceinline__ void unpack8t(const uint4 v, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f2_t t = unpack2<DT>(word(v, j));
    f[2 * j] = f2lo(t);
    f[2 * j + 1] = f2hi(t);
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8t(const float (&f)[8]) {
  return make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float rms_scale(float sum, float inv_d, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fmaf_rn(sum, inv_d, eps)));
}

// ------------------------------------------------------------------ forward --
// A group of GROUP warps owns a row and holds it in registers, VPL vectors of
// 8 elements a lane.
template <int VPL, int GROUP, int DT, bool INT8>
__global__ void __launch_bounds__((GROUP > 4 ? GROUP : 4) * 32) sandwich_fwd_kernel(const SandwichArgs a) {
  constexpr int BW = GROUP > 4 ? GROUP : 4;
  __shared__ float red[2][BW];
  __shared__ uint32_t redu[BW];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = (warp % GROUP) * 32 + lane, w0 = (warp / GROUP) * GROUP;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (BW / GROUP) + warp / GROUP;
  const bool row_ok = row < a.rows;
  const int64_t base = (row_ok ? row : 0) * a.D;
  const int64_t bd = row_ok ? div_u32(a.seq, row) * a.D : 0;
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(a.D));

  auto group_sum = [&](float v, int buf) {
    v = warp_sum(v);
    if (GROUP > 1) {
      if (lane == 0) red[buf][warp] = v;
      __syncthreads();
      v = 0.0f;
#pragma unroll
      for (int w = 0; w < GROUP; ++w) v += red[buf][w0 + w];
    }
    return v;
  };

  uint4 xv[VPL], zv[VPL];
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 8;
    const bool ok = row_ok && e < a.D;
    xv[c] = ok ? ld_stream(a.x + base + e) : make_uint4(0, 0, 0, 0);
    zv[c] = ok ? ld_stream(a.res + base + e) : make_uint4(0, 0, 0, 0);
  }
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    float f[8];
    unpack8t<DT>(xv[c], f);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum = __fmaf_rn(f[k], f[k], sum);
  }
  const float r1 = rms_scale(group_sum(sum, 0), inv_d, a.eps);
  sum = 0.0f;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 8;
    if (row_ok && e < a.D) {
      float x[8], r[8], g[8], p[8];
      unpack8t<DT>(xv[c], x);
      unpack8t<DT>(zv[c], r);
      load8<DT>(a.gate ? a.gate + bd + e : nullptr, 1.0f, g);
      load8f(a.post + e, p);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] = __fmaf_rn(g[k], x[k] * r1 * p[k], a.alpha * r[k]);
      zv[c] = pack8t<DT>(r);
      st16(a.z + base + e, zv[c]);
      unpack8t<DT>(zv[c], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum = __fmaf_rn(r[k], r[k], sum);
    }
  }
  const float r2 = rms_scale(group_sum(sum, 1), inv_d, a.eps);
  f2_t h[VPL][4];
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 8;
    if (row_ok && e < a.D) {
      float z[8], p[8], sc[8], sh[8];
      unpack8t<DT>(zv[c], z);
      load8f(a.pre + e, p);
      load8<DT>(a.scale ? a.scale + bd + e : nullptr, 1.0f, sc);
      load8<DT>(a.shift ? a.shift + bd + e : nullptr, 0.0f, sh);
#pragma unroll
      for (int k = 0; k < 8; ++k) z[k] = __fmaf_rn(z[k] * r2 * p[k], sc[k], sh[k]);
      if (!INT8) {
        st16(a.h + base + e, pack8t<DT>(z));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          h[c][j] = f2(z[2 * j], z[2 * j + 1]);
          amax = max_abs_nan(amax, h[c][j]);
        }
      }
    }
  }
  if (INT8) {
    uint32_t top = warp_max_u32(__float_as_uint(amax));
    if (GROUP > 1) {
      if (lane == 0) redu[warp] = top;
      __syncthreads();
      top = group_max_u32<GROUP>(&redu[w0]);
    }
    if (!row_ok) return;
    const RowScale r = row_scale(top);
    if (t == 0) a.s[row] = scale_value(top);
#pragma unroll
    for (int c = 0; c < VPL; ++c) {
      const int e = (t + 32 * GROUP * c) * 8;
      if (e < a.D) st8(a.q + base + e, codes8(h[c], r));
    }
  }
}

template <int VPL, int GROUP, bool INT8>
static cudaError_t launch_fwd_g(const SandwichArgs& a, int dtype, cudaStream_t st) {
  constexpr int BW = GROUP > 4 ? GROUP : 4;
  const dim3 grid(static_cast<unsigned>((a.rows + BW / GROUP - 1) / (BW / GROUP))), block(BW * 32);
  return dtype == kBf16 ? launch_pdl(sandwich_fwd_kernel<VPL, GROUP, kBf16, INT8>, grid, block, 0, st, a)
                        : launch_pdl(sandwich_fwd_kernel<VPL, GROUP, kFp16, INT8>, grid, block, 0, st, a);
}

template <bool INT8>
static cudaError_t launch_fwd(const SandwichArgs& a, int dtype, cudaStream_t st) {
  const int nv = a.D / 8;
  if (nv <= 32) return launch_fwd_g<1, 1, INT8>(a, dtype, st);
  if (nv <= 64) return launch_fwd_g<2, 1, INT8>(a, dtype, st);
  if (nv <= 128) return launch_fwd_g<4, 1, INT8>(a, dtype, st);
  if (nv <= 256) return launch_fwd_g<4, 2, INT8>(a, dtype, st);
  return launch_fwd_g<4, 4, INT8>(a, dtype, st);
}

// ----------------------------------------------------------------- backward --
struct SandwichBwdArgs {
  const uint16_t *gh, *gz, *z, *x;  // [B*S, D]; gz may be null
  const uint16_t* gate;             // [B, D] or null
  const float* post;                // [D]
  const float* pre;                 // [D]
  const uint16_t* scale;            // [B, D] or null
  uint16_t *dx, *dres;              // [B*S, D]
  float* part;                      // [B][chunks][3][D]: P, Q, sum gh
  int64_t S;
  int chunk;   // rows of a block
  int D;
  float alpha, eps;
};

constexpr int kBwdRows = 2;  // rows a block holds at once

// A block owns `chunk` rows of one sample; a thread owns 8 columns, whose
// three sums stay in its registers.
template <int DT>
__global__ void __launch_bounds__(512) sandwich_bwd_kernel(const SandwichBwdArgs a) {
  constexpr int R = kBwdRows;
  __shared__ float red[2][R][4][16];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int e = threadIdx.x * 8;
  const bool col = e < a.D;
  const int64_t b = blockIdx.y, r0 = static_cast<int64_t>(blockIdx.x) * a.chunk;
  const int64_t r1 = min(r0 + a.chunk, a.S);
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(a.D));
  float gw[8] = {}, pw[8] = {};  // gate * post, scale * pre
  if (col) {
    float u[8];
    load8<DT>(a.gate ? a.gate + b * a.D + e : nullptr, 1.0f, gw);
    load8f(a.post + e, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) gw[k] *= u[k];
    load8<DT>(a.scale ? a.scale + b * a.D + e : nullptr, 1.0f, pw);
    load8f(a.pre + e, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) pw[k] *= u[k];
  }
  float P[8] = {}, Q[8] = {}, G[8] = {};
  for (int64_t r = r0; r < r1; r += R) {
    uint4 ghv[R], gzv[R], zv[R], xv[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool ok = col && r + i < r1;
      const int64_t at = (b * a.S + r + i) * a.D + e;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      ghv[i] = ok ? ld_stream(a.gh + at) : zero;
      gzv[i] = ok && a.gz ? ld_stream(a.gz + at) : zero;
      zv[i] = ok ? ld_stream(a.z + at) : zero;
      xv[i] = ok ? ld_stream(a.x + at) : zero;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float g[8], z[8], x[8], s0 = 0.0f, s1 = 0.0f, s2 = 0.0f;
      unpack8t<DT>(ghv[i], g);
      unpack8t<DT>(zv[i], z);
      unpack8t<DT>(xv[i], x);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s0 = __fmaf_rn(z[k], z[k], s0);
        s1 = __fmaf_rn(g[k] * pw[k], z[k], s1);
        s2 = __fmaf_rn(x[k], x[k], s2);
      }
      s0 = warp_sum(s0);
      s1 = warp_sum(s1);
      s2 = warp_sum(s2);
      if (lane == 0) {
        red[0][i][0][warp] = s0;
        red[0][i][1][warp] = s1;
        red[0][i][2][warp] = s2;
      }
    }
    __syncthreads();
    float dz[R][8], rx[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
      for (int w = 0; w < nw; ++w) {
        s0 += red[0][i][0][w];
        s1 += red[0][i][1][w];
        s2 += red[0][i][2][w];
      }
      const float rz = rms_scale(s0, inv_d, a.eps);
      rx[i] = rms_scale(s2, inv_d, a.eps);
      const float c = s1 * rz * inv_d;  // mean(p zh)
      float g[8], z[8], x[8], gz[8];
      unpack8t<DT>(ghv[i], g);
      unpack8t<DT>(zv[i], z);
      unpack8t<DT>(xv[i], x);
      unpack8t<DT>(gzv[i], gz);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float zh = z[k] * rz, xh = x[k] * rx[i];
        dz[i][k] = __fmaf_rn(rz, __fmaf_rn(-zh, c, g[k] * pw[k]), gz[k]);
        s3 = __fmaf_rn(dz[i][k] * gw[k], xh, s3);
        P[k] = __fmaf_rn(g[k], zh, P[k]);
        Q[k] = __fmaf_rn(dz[i][k], xh, Q[k]);
        G[k] += g[k];
      }
      s3 = warp_sum(s3);
      if (lane == 0) red[1][i][3][warp] = s3;
      if (col && r + i < r1) {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = a.alpha * dz[i][k];
        st16(a.dres + (b * a.S + r + i) * a.D + e, pack8t<DT>(o));
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float s3 = 0.0f;
      for (int w = 0; w < nw; ++w) s3 += red[1][i][3][w];
      const float c = s3 * inv_d;
      if (col && r + i < r1) {
        float x[8];
        unpack8t<DT>(xv[i], x);
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = rx[i] * __fmaf_rn(-(x[k] * rx[i]), c, dz[i][k] * gw[k]);
        st16(a.dx + (b * a.S + r + i) * a.D + e, pack8t<DT>(x));
      }
    }
  }
  if (col) {
    float* p = a.part + (b * gridDim.x + blockIdx.x) * 3 * a.D + e;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      p[k] = P[k];
      p[a.D + k] = Q[k];
      p[2 * a.D + k] = G[k];
    }
  }
}

struct SandwichFinalArgs {
  const float* part;
  const uint16_t *gate, *scale;  // [B, D] or null
  const float *post, *pre;       // [D]
  uint16_t *dgate, *dshift, *dscale;  // [B, D] or null
  float *dpost, *dpre;                // [D]
  int64_t B;
  int chunks, D;
};

// 32 columns a block; its 32 warps each sum every 32nd chunk.
template <int DT>
__global__ void __launch_bounds__(1024) sandwich_final_kernel(const SandwichFinalArgs a) {
  __shared__ float red[32][3][33];
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const bool ok = c < a.D;
  float dpost = 0.0f, dpre = 0.0f;
  for (int64_t b = 0; b < a.B; ++b) {
    float s[3] = {};
    if (ok) {
      for (int n = warp; n < a.chunks; n += 32) {
        const float* p = a.part + (b * a.chunks + n) * 3 * a.D + c;
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] += __ldg(p + static_cast<int64_t>(i) * a.D);
      }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) red[warp][i][lane] = s[i];
    __syncthreads();
    if (warp == 0 && ok) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        s[i] = 0.0f;
        for (int w = 0; w < 32; ++w) s[i] += red[w][i][lane];
      }
      const int64_t at = b * a.D + c;
      dpre = __fmaf_rn(a.scale ? load1<DT>(a.scale + at) : 1.0f, s[0], dpre);
      dpost = __fmaf_rn(a.gate ? load1<DT>(a.gate + at) : 1.0f, s[1], dpost);
      if (a.dscale) a.dscale[at] = static_cast<uint16_t>(pack2<DT>(a.pre[c] * s[0], 0.0f));
      if (a.dgate) a.dgate[at] = static_cast<uint16_t>(pack2<DT>(a.post[c] * s[1], 0.0f));
      if (a.dshift) a.dshift[at] = static_cast<uint16_t>(pack2<DT>(s[2], 0.0f));
    }
    __syncthreads();
  }
  if (warp == 0 && ok) {
    a.dpost[c] = dpost;
    a.dpre[c] = dpre;
  }
}

// Rows of a backward block: enough blocks for two a multiprocessor, and no
// fewer than 8 rows each, so that the column sums that a block leaves stay
// below its rows' own traffic.  148 multiprocessors, whatever the device.
static int64_t bwd_chunk(int64_t B, int64_t S) {
  const int64_t per = (B * S + 295) / 296;
  const int64_t c = ((per < 8 ? 8 : per) + kBwdRows - 1) / kBwdRows * kBwdRows;
  return c < S ? c : S;
}
static bool check_sandwich(int64_t B, int64_t S, int64_t D, int dtype) {
  return check(B >= 0 && B <= 65535, "batch must be in [0, 65535]") &&
         check(S >= 0 && S <= (1 << 30), "seq must be in [0, 2^30]") &&
         check(B * S <= INT64_C(0x7fffffff), "batch * seq must be below 2^31") &&
         check(D >= 8 && D % 8 == 0 && D <= kMaxRowDim,
               "dim must be a multiple of 8 in [8, " + std::to_string(kMaxRowDim) + "], got " + std::to_string(D)) &&
         check_dtype(dtype);
}
static bool check_opt16(const void* p, const char* n) {
  return check(aligned(p, 16), std::string(n) + " is not 16-byte aligned");
}

}  // namespace afb

using namespace afb;

static int sandwich_fwd(const char* name, const void* x, const void* res, const void* gate, const void* post,
                        const void* pre, const void* shift, const void* scale, void* h, void* q, void* s, void* z,
                        int64_t B, int64_t S, int64_t D, float alpha, float eps, int dtype, void* stream) {
  ApiGuard g(name);
  if (!check_sandwich(B, S, D, dtype)) return g.fail();
  if (B == 0 || S == 0) return 0;
  if (!check_ptrs({x, res, post, pre, z}, {"x", "residual", "post_weight", "pre_weight", "z"}) ||
      !check_opt16(gate, "gate") || !check_opt16(shift, "shift") || !check_opt16(scale, "scale"))
    return g.fail();
  SandwichArgs a{};
  a.x = static_cast<const uint16_t*>(x);
  a.res = static_cast<const uint16_t*>(res);
  a.gate = static_cast<const uint16_t*>(gate);
  a.post = static_cast<const float*>(post);
  a.pre = static_cast<const float*>(pre);
  a.shift = static_cast<const uint16_t*>(shift);
  a.scale = static_cast<const uint16_t*>(scale);
  a.h = static_cast<uint16_t*>(h);
  a.z = static_cast<uint16_t*>(z);
  a.q = static_cast<int8_t*>(q);
  a.s = static_cast<float*>(s);
  a.rows = B * S;
  a.seq = make_divu32(S);
  a.D = static_cast<int>(D);
  a.alpha = alpha;
  a.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g.done(q != nullptr ? launch_fwd<true>(a, dtype, st) : launch_fwd<false>(a, dtype, st));
}

extern "C" int afb_sandwich_norm(const void* x, const void* residual, const void* gate, const void* post_weight,
                                 const void* pre_weight, const void* shift, const void* scale, void* h, void* z,
                                 int64_t batch, int64_t seq, int64_t dim, float residual_scale, float eps, int dtype,
                                 void* stream) {
  ApiGuard g("afb_sandwich_norm");
  if (batch > 0 && seq > 0 && !check_ptrs({h}, {"h"})) return g.fail();
  return sandwich_fwd("afb_sandwich_norm", x, residual, gate, post_weight, pre_weight, shift, scale, h, nullptr,
                      nullptr, z, batch, seq, dim, residual_scale, eps, dtype, stream);
}

extern "C" int afb_sandwich_norm_int8(const void* x, const void* residual, const void* gate, const void* post_weight,
                                      const void* pre_weight, const void* shift, const void* scale, void* q, void* s,
                                      void* z, int64_t batch, int64_t seq, int64_t dim, float residual_scale,
                                      float eps, int dtype, void* stream) {
  ApiGuard g("afb_sandwich_norm_int8");
  if (batch > 0 && seq > 0 && (!check_ptr8(q, "q") || !check_ptr4(s, "s"))) return g.fail();
  return sandwich_fwd("afb_sandwich_norm_int8", x, residual, gate, post_weight, pre_weight, shift, scale, nullptr, q,
                      s, z, batch, seq, dim, residual_scale, eps, dtype, stream);
}

extern "C" size_t afb_sandwich_norm_bwd_workspace(int64_t batch, int64_t seq, int64_t dim) {
  if (batch <= 0 || seq <= 0 || dim <= 0) return 0;
  if (batch > 65535 || seq > (1 << 30) || dim > kMaxRowDim) return SIZE_MAX;
  const int64_t c = bwd_chunk(batch, seq);
  return static_cast<size_t>(batch * ((seq + c - 1) / c) * 3 * dim) * sizeof(float);
}

extern "C" int afb_sandwich_norm_bwd(const void* gh, const void* gz, const void* z, const void* x, const void* gate,
                                     const void* post_weight, const void* pre_weight, const void* scale, void* dx,
                                     void* dres, void* dgate, void* dpost, void* dpre, void* dshift, void* dscale,
                                     int64_t batch, int64_t seq, int64_t dim, float residual_scale, float eps,
                                     int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  ApiGuard g("afb_sandwich_norm_bwd");
  if (!check_sandwich(batch, seq, dim, dtype) || !check(batch >= 1 && seq >= 1, "batch and seq must be >= 1") ||
      !check_ptrs({gh, z, x, post_weight, pre_weight, dx, dres, dpost, dpre, workspace},
                  {"gh", "z", "x", "post_weight", "pre_weight", "dx", "dres", "dpost", "dpre", "workspace"}) ||
      !check_opt16(gz, "gz") || !check_opt16(gate, "gate") || !check_opt16(scale, "scale") ||
      !check(workspace_bytes >= afb_sandwich_norm_bwd_workspace(batch, seq, dim), "workspace too small"))
    return g.fail();
  SandwichBwdArgs a{};
  a.gh = static_cast<const uint16_t*>(gh);
  a.gz = static_cast<const uint16_t*>(gz);
  a.z = static_cast<const uint16_t*>(z);
  a.x = static_cast<const uint16_t*>(x);
  a.gate = static_cast<const uint16_t*>(gate);
  a.post = static_cast<const float*>(post_weight);
  a.pre = static_cast<const float*>(pre_weight);
  a.scale = static_cast<const uint16_t*>(scale);
  a.dx = static_cast<uint16_t*>(dx);
  a.dres = static_cast<uint16_t*>(dres);
  a.part = static_cast<float*>(workspace);
  a.S = seq;
  a.chunk = static_cast<int>(bwd_chunk(batch, seq));
  a.D = static_cast<int>(dim);
  a.alpha = residual_scale;
  a.eps = eps;
  SandwichFinalArgs f{};
  f.part = a.part;
  f.gate = a.gate;
  f.scale = a.scale;
  f.post = a.post;
  f.pre = a.pre;
  f.dgate = static_cast<uint16_t*>(dgate);
  f.dshift = static_cast<uint16_t*>(dshift);
  f.dscale = static_cast<uint16_t*>(dscale);
  f.dpost = static_cast<float*>(dpost);
  f.dpre = static_cast<float*>(dpre);
  f.B = batch;
  f.chunks = static_cast<int>((seq + a.chunk - 1) / a.chunk);
  f.D = a.D;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(f.chunks), static_cast<unsigned>(batch));
  const dim3 block(static_cast<unsigned>((dim / 8 + 31) / 32 * 32));
  cudaError_t e = dtype == kBf16 ? launch_pdl(sandwich_bwd_kernel<kBf16>, grid, block, 0, st, a)
                                 : launch_pdl(sandwich_bwd_kernel<kFp16>, grid, block, 0, st, a);
  if (e != cudaSuccess) return g.done(e);
  const dim3 fg(static_cast<unsigned>((dim + 31) / 32));
  return g.done(dtype == kBf16 ? launch_pdl(sandwich_final_kernel<kBf16>, fg, dim3(1024), 0, st, f)
                               : launch_pdl(sandwich_final_kernel<kFp16>, fg, dim3(1024), 0, st, f));
}
