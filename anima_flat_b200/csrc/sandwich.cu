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

// Eight factors of the columns as pairs: a per-sample vector of the activations'
// type, or a constant where it is null.
template <int DT>
__device__ __forceinline__ void load4p(const uint16_t* p, float fallback, f2_t (&f)[4]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = splat2(fallback);
    return;
  }
  const uint4 v = ld_keep(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = unpack2<DT>(word(v, j));
}
__device__ __forceinline__ void load4pf(const float* p, f2_t (&f)[4]) {
  const ulonglong2 lo = __ldg(reinterpret_cast<const ulonglong2*>(p)), hi = __ldg(reinterpret_cast<const ulonglong2*>(p + 4));
  f[0] = lo.x;
  f[1] = lo.y;
  f[2] = hi.x;
  f[3] = hi.y;
}
template <int DT>
__device__ __forceinline__ void unpack4p(const uint4 v, f2_t (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = unpack2<DT>(word(v, j));
}
template <int DT>
__device__ __forceinline__ uint4 pack4p(const f2_t (&f)[4]) {
  return make_uint4(pack2<DT>(f[0]), pack2<DT>(f[1]), pack2<DT>(f[2]), pack2<DT>(f[3]));
}
__device__ __forceinline__ float sum2(f2_t v) { return f2lo(v) + f2hi(v); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
__device__ __forceinline__ float rms_scale(float sum, float inv_d, float eps) {
  return rsqrtf(__fmaf_rn(sum, inv_d, eps));
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
  f2_t sum = 0;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    f2_t f[4];
    unpack4p<DT>(xv[c], f);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma2(f[j], f[j], sum);
  }
  const f2_t r1 = splat2(rms_scale(group_sum(sum2(sum), 0), inv_d, a.eps)), alpha = splat2(a.alpha);
  sum = 0;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 8;
    if (row_ok && e < a.D) {
      f2_t x[4], r[4], g[4], p[4];
      unpack4p<DT>(xv[c], x);
      unpack4p<DT>(zv[c], r);
      load4p<DT>(a.gate ? a.gate + bd + e : nullptr, 1.0f, g);
      load4pf(a.post + e, p);
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = fma2(mul2(g[j], p[j]), mul2(x[j], r1), mul2(alpha, r[j]));
      zv[c] = pack4p<DT>(r);
      st16(a.z + base + e, zv[c]);
      unpack4p<DT>(zv[c], r);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fma2(r[j], r[j], sum);
    }
  }
  const f2_t r2 = splat2(rms_scale(group_sum(sum2(sum), 1), inv_d, a.eps));
  f2_t h[VPL][4];
  float amax = 0.0f;
#pragma unroll
  for (int c = 0; c < VPL; ++c) {
    const int e = (t + 32 * GROUP * c) * 8;
    if (row_ok && e < a.D) {
      f2_t z[4], p[4], sc[4], sh[4];
      unpack4p<DT>(zv[c], z);
      load4pf(a.pre + e, p);
      load4p<DT>(a.scale ? a.scale + bd + e : nullptr, 1.0f, sc);
      load4p<DT>(a.shift ? a.shift + bd + e : nullptr, 0.0f, sh);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[c][j] = fma2(mul2(z[j], r2), mul2(p[j], sc[j]), sh[j]);
        if (INT8) amax = max_abs_nan(amax, h[c][j]);
      }
      if (!INT8) st16(a.h + base + e, pack4p<DT>(h[c]));
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

// Many rows: a block owns a chunk of one sample's rows, its teams of D / 8
// threads take four rows at a time.  A thread owns 8 columns and keeps their
// factors in registers; in the kernel above every row reads them again, 14 bytes
// an element from L1 for 8 from memory.  Bulk copies keep the next rows coming.
// Which sizes: fwd_by_teams.
constexpr int64_t kManyWide = 1 << 19, kManyNarrow = 1 << 22;
constexpr int kFwdRows = 4;
constexpr int kFwdStages = 3;
constexpr int kTeamThreads = 512;
static int team_threads_of(int D) { return (D / 8 + 31) / 32 * 32; }
static int teams_of(int D) {
  const int t = kTeamThreads / team_threads_of(D);
  return t < 8 ? t : 8;
}
static size_t fwd_smem(int D) { return static_cast<size_t>(teams_of(D)) * kFwdStages * kFwdRows * 2 * D * 2; }

// Sums, or maxima of bit patterns, of four values over the warp: lane l returns
// that of value l / 8.
__device__ __forceinline__ float warp_sum4(const float (&v)[4]) {
  const int lane = threadIdx.x & 31;
  float b[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool up = lane & 16;
    b[i] = (up ? v[i + 2] : v[i]) + __shfl_xor_sync(kFull, up ? v[i] : v[i + 2], 16);
  }
  const bool up = lane & 8;
  float c = (up ? b[1] : b[0]) + __shfl_xor_sync(kFull, up ? b[0] : b[1], 8);
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) c += __shfl_xor_sync(kFull, c, o);
  return c;
}
// The team's sum of value l / 8 from its warps' in red[value][warp].
__device__ __forceinline__ float team_sum4(const float (*red)[16]) {
  const int lane = threadIdx.x & 31;
  const float2 p = *reinterpret_cast<const float2*>(&red[lane >> 3][2 * (lane & 7)]);
  float c = p.x + p.y;
#pragma unroll
  for (int o = 4; o >= 1; o >>= 1) c += __shfl_xor_sync(kFull, c, o);
  return c;
}

template <int DT, bool INT8>
__global__ void __launch_bounds__(kTeamThreads, 1)
sandwich_rows_kernel(const SandwichArgs a, int64_t S, int chunk, int team_threads, int teams) {
  constexpr int R = kFwdRows, NS = kFwdStages;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[8 * NS];
  __shared__ __align__(16) float red[2][8][R][16];
  __shared__ uint32_t redu[8][R][16];
  const int lane = threadIdx.x & 31;
  const int team = static_cast<int>(threadIdx.x) / team_threads, tid = static_cast<int>(threadIdx.x) % team_threads;
  const int warp = tid >> 5, e = tid * 8;
  const bool col = e < a.D;
  const int64_t b = blockIdx.y, r0 = static_cast<int64_t>(blockIdx.x) * chunk;
  const int rows = static_cast<int>(min(static_cast<int64_t>(chunk), S - r0));
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(a.D));
  const uint32_t row_bytes = static_cast<uint32_t>(a.D) * 2, stage_bytes = R * 2 * row_bytes;
  const uint32_t ring = smem_addr(dyn) + team * NS * stage_bytes, bar0 = smem_addr(bars) + team * NS * 8;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(bar0 + 8 * i, 1);
    fence_mbar_init();
  }
  for (int i = static_cast<int>(threadIdx.x); i < 8 * R * 16; i += static_cast<int>(blockDim.x)) {
    (&red[0][0][0][0])[i] = (&red[1][0][0][0])[i] = 0.0f;
    (&redu[0][0][0])[i] = 0;
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // Group i of the team: rows (i * teams + team) * R of the chunk.
  const int groups = (rows + R - 1) / R;
  const int mine = groups > team ? (groups - team + teams - 1) / teams : 0;
  auto request = [&](int i) {
    const int r = (i * teams + team) * R, n = min(R, rows - r);
    const uint32_t bar = bar0 + 8 * (i % NS), dst = ring + (i % NS) * stage_bytes;
    const int64_t at = (b * S + r0 + r) * a.D;
    mbar_arrive_expect_tx(bar, n * 2 * row_bytes);
    bulk_g2s(dst, a.x + at, n * row_bytes, bar);  // neighbouring rows are one piece
    bulk_g2s(dst + R * row_bytes, a.res + at, n * row_bytes, bar);
  };
  int asked = 0;
  if (tid == 0)
    for (; asked < NS - 1 && asked < mine; ++asked) request(asked);

  f2_t gp[4] = {}, ps[4] = {}, sh[4] = {};  // gate * post, pre * scale, shift
  if (col) {
    f2_t u[4];
    load4pf(a.post + e, u);
    load4p<DT>(a.gate ? a.gate + b * a.D + e : nullptr, 1.0f, gp);
#pragma unroll
    for (int j = 0; j < 4; ++j) gp[j] = mul2(gp[j], u[j]);
    load4pf(a.pre + e, u);
    load4p<DT>(a.scale ? a.scale + b * a.D + e : nullptr, 1.0f, ps);
#pragma unroll
    for (int j = 0; j < 4; ++j) ps[j] = mul2(ps[j], u[j]);
    load4p<DT>(a.shift ? a.shift + b * a.D + e : nullptr, 0.0f, sh);
  }
  const f2_t alpha = splat2(a.alpha);
  bool ok = true;
  for (int i = 0; i < mine; ++i) {
    const int r = (i * teams + team) * R;
    // A thread reads its own 16 bytes of each row alone; one past the last
    // column reads column 0 and counts nothing.
    const uint8_t* at = dyn + (team * NS + i % NS) * stage_bytes + (col ? tid * 16 : 0);
    ok = ok && mbar_wait(bar0 + 8 * (i % NS), (i / NS) & 1);
    const int64_t out = (b * S + r0 + r) * a.D + e;
    float part[R];
    uint4 xv[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      // rows past the chunk's last hold what was there: they are not written
      f2_t x[4], s = 0;
      xv[k] = lds16(at + k * row_bytes);
      unpack4p<DT>(xv[k], x);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fma2(x[j], x[j], s);
      part[k] = col ? sum2(s) : 0.0f;
    }
    const float own = warp_sum4(part);
    if ((lane & 7) == 0) red[0][team][lane >> 3][warp] = own;
    named_bar_sync(1 + team, team_threads);
    // The team is done with group i - 1: its stage takes group i + 2.
    if (tid == 0 && ok && asked < mine) {
      fence_proxy_async_smem();
      request(asked++);
    }
    const float root = rms_scale(team_sum4(red[0][team]), inv_d, a.eps);
    uint4 zv[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const f2_t r1 = splat2(__shfl_sync(kFull, root, 8 * k));
      f2_t x[4], z[4], s = 0;
      unpack4p<DT>(xv[k], x);
      unpack4p<DT>(lds16(at + (R + k) * row_bytes), z);
#pragma unroll
      for (int j = 0; j < 4; ++j) z[j] = fma2(gp[j], mul2(x[j], r1), mul2(alpha, z[j]));
      zv[k] = pack4p<DT>(z);
      if (col && r + k < rows) st16(a.z + out + static_cast<int64_t>(k) * a.D, zv[k]);
      unpack4p<DT>(zv[k], z);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = fma2(z[j], z[j], s);
      part[k] = col ? sum2(s) : 0.0f;
    }
    const float own2 = warp_sum4(part);
    if ((lane & 7) == 0) red[1][team][lane >> 3][warp] = own2;
    named_bar_sync(1 + team, team_threads);
    const float root2 = rms_scale(team_sum4(red[1][team]), inv_d, a.eps);
    f2_t h[INT8 ? R : 1][4];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const f2_t r2 = splat2(__shfl_sync(kFull, root2, 8 * k));
      f2_t(&o)[4] = h[INT8 ? k : 0];
      f2_t z[4];
      float amax = 0.0f;
      unpack4p<DT>(zv[k], z);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        o[j] = fma2(ps[j], mul2(z[j], r2), sh[j]);
        if (INT8) amax = max_abs_nan(amax, o[j]);
      }
      if (!INT8) {
        if (col && r + k < rows) st16(a.h + out + static_cast<int64_t>(k) * a.D, pack4p<DT>(o));
      } else {
        const uint32_t m = warp_max_u32(col ? __float_as_uint(amax) : 0u);
        if (lane == k) top = m;
      }
    }
    if (INT8) {
      if (lane < R) redu[team][lane][warp] = top;
      named_bar_sync(1 + team, team_threads);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const uint32_t m = group_max_u32<16>(redu[team][k]);
        const RowScale rs = row_scale(m);
        if (col && r + k < rows) {
          st8(a.q + out + static_cast<int64_t>(k) * a.D, codes8(h[INT8 ? k : 0], rs));
          if (tid == 0) a.s[b * S + r0 + r + k] = scale_value(m);
        }
      }
    }
  }
  // After a wait that gave up: copies in flight land before the block ends.
  if (tid == 0 && !ok)
    for (int i = asked > NS ? asked - NS : 0; i < asked; ++i) mbar_wait(bar0 + 8 * (i % NS), (i / NS) & 1);
}

// Rows of a block: one block a multiprocessor (148, whatever the device), of at
// least `least` rows.
static int64_t rows_of_block(int64_t B, int64_t S, int64_t least) {
  const int64_t per_sample = B < 148 ? 148 / B : 1;
  const int64_t c = (S + per_sample - 1) / per_sample;
  return c > least ? c : least;
}

// Whether teams take a forward pass.  Where a block a multiprocessor holds all
// samples: from 2^19 elements on for rows of 1024 and more (256 x 2048: 4.0 us
// against 4.2 by groups of warps, 1024 x 2048: 5.5 against 6.5; 128 x 2048: 4.0 and
// 4.0), from 2^22 for shorter ones (8192 x 512: 8.6 against 9.1; 2048 x 512: 4.4
// against 3.6).  A block takes one sample's rows, so more samples are more blocks,
// one after another, each with its start and its factors to load: by what was
// measured, in ns, 2500 a round of 148 and 0.195 an element of a block (0.12 in a
// round of few, and all 15% more for codes), where groups of warps take 2400 and
// 0.002 an element in all (0.0016 in short rows).  4096 samples of one row of 2048: 93
// us by teams, 21 by groups; 256 of 64: 45 and 67.
static bool fwd_by_teams(int64_t B, int64_t S, int64_t D, bool int8) {
  const int64_t all = B * S * D;
  if (all < (D >= 1024 ? kManyWide : kManyNarrow)) return false;
  const int64_t chunk = rows_of_block(B, S, teams_of(static_cast<int>(D)) * kFwdRows);
  const int64_t blocks = B * ((S + chunk - 1) / chunk), rounds = blocks / 148, rest = blocks % 148;
  if (blocks <= 148) return true;
  const int64_t mine = (S < chunk ? S : chunk) * D;
  const int64_t teams = rounds * (2500 + mine * 195 / 1000) + (rest ? 2500 + mine * (120 + 75 * rest / 148) / 1000 : 0);
  const int64_t groups = 2400 + all * (D >= 1024 ? 20 : 16) / 10000;
  return teams * (int8 ? 115 : 100) / 100 < groups;
}

template <bool INT8>
static cudaError_t launch_rows(const SandwichArgs& a, int64_t B, int64_t S, int dtype, cudaStream_t st) {
  const int team = team_threads_of(a.D), teams = teams_of(a.D);
  const int64_t chunk = rows_of_block(B, S, teams * kFwdRows);
  const size_t smem = fwd_smem(a.D);
  const dim3 grid(static_cast<unsigned>((S + chunk - 1) / chunk), static_cast<unsigned>(B)), block(team * teams);
  auto kernel = dtype == kBf16 ? sandwich_rows_kernel<kBf16, INT8> : sandwich_rows_kernel<kFp16, INT8>;
  const cudaError_t e = ensure_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(kernel, grid, block, smem, st, a, S, static_cast<int>(chunk), team, teams);
}

template <int VPL, int GROUP, bool INT8>
static cudaError_t launch_fwd_g(const SandwichArgs& a, int dtype, cudaStream_t st) {
  constexpr int BW = GROUP > 4 ? GROUP : 4;
  const dim3 grid(static_cast<unsigned>((a.rows + BW / GROUP - 1) / (BW / GROUP))), block(BW * 32);
  return dtype == kBf16 ? launch_pdl(sandwich_fwd_kernel<VPL, GROUP, kBf16, INT8>, grid, block, 0, st, a)
                        : launch_pdl(sandwich_fwd_kernel<VPL, GROUP, kFp16, INT8>, grid, block, 0, st, a);
}

template <bool INT8>
static cudaError_t launch_fwd(const SandwichArgs& a, int64_t B, int64_t S, int dtype, cudaStream_t st) {
  const int nv = a.D / 8;
  if (fwd_by_teams(B, S, a.D, INT8)) return launch_rows<INT8>(a, B, S, dtype, st);
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

// A block owns `chunk` rows of one sample.  Its teams of D / 8 threads (rounded
// up to warps) take pairs of rows in turn; a thread owns 8 columns, whose three
// sums stay in its registers, so a row is read once.  Bulk copies keep the next
// two pairs of every team on their way in shared memory: with the loads in the
// row loop itself the kernel ran at 39% of memory speed, on their latency.
//
// All six sums of a row are taken at once, with t = x gate post, since
//   sum m xh = r1 (sum gz t + r2 (sum p t - r2 mean(p zh) sum z t)):
// one barrier a pair of rows, and dx in the pass that forms dz: 1.1 us less at
// 8192 x 2048 than with a barrier of its own for sum m xh.  Both launches, with the
// sums' kernel below: 8192 x 2048 43.5 us, 4096 x 2048 27.8, some 12 of which do not depend on the rows (launches,
// first and last copies, the columns' sums).  In the row loop 16 warps fill 52%
// of the issue slots, with 43 instructions an element; they wait for barriers and
// shared memory in equal parts.
constexpr int kBwdRows = 2;    // rows a team holds at once
constexpr int kBwdStages = 3;  // of kBwdRows rows each
static size_t bwd_smem(int D) { return static_cast<size_t>(teams_of(D)) * kBwdStages * kBwdRows * 4 * D * 2; }

// Sums of eight values over the warp: lane l returns that of value l / 4.
// Each step halves the values a lane carries, 9 exchanges for the 40 of eight
// butterflies.
__device__ __forceinline__ float warp_sum8(const float (&v)[8]) {
  const int lane = threadIdx.x & 31;
  float a[4], b[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool up = lane & 16;
    a[i] = (up ? v[i + 4] : v[i]) + __shfl_xor_sync(kFull, up ? v[i] : v[i + 4], 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool up = lane & 8;
    b[i] = (up ? a[i + 2] : a[i]) + __shfl_xor_sync(kFull, up ? a[i] : a[i + 2], 8);
  }
  const bool up = lane & 4;
  float c = (up ? b[1] : b[0]) + __shfl_xor_sync(kFull, up ? b[0] : b[1], 4);
  c += __shfl_xor_sync(kFull, c, 2);
  return c + __shfl_xor_sync(kFull, c, 1);
}
// The team's sum of value l / 4, for every lane l, from its warps' in
// red[value][warp] (zero above the team's warps).
__device__ __forceinline__ float team_sum8(const float (*red)[16]) {
  const int lane = threadIdx.x & 31;
  const float4 p = *reinterpret_cast<const float4*>(&red[lane >> 2][4 * (lane & 3)]);
  float c = (p.x + p.y) + (p.z + p.w);
  c += __shfl_xor_sync(kFull, c, 2);
  return c + __shfl_xor_sync(kFull, c, 1);
}
template <int DT>
__global__ void __launch_bounds__(kTeamThreads, 1) sandwich_bwd_kernel(const SandwichBwdArgs a, int team_threads, int teams) {
  constexpr int R = kBwdRows, NS = kBwdStages;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ __align__(8) uint64_t bars[8 * NS];
  // per team, for steps in turn: the rows' sums by warp, of z^2, x^2, p z and
  // gz t, and of p t and z t, with t = x gate post
  __shared__ __align__(16) float red8[2][8][8][16], red4[2][8][4][16];
  const int lane = threadIdx.x & 31;
  const int team = static_cast<int>(threadIdx.x) / team_threads, tid = static_cast<int>(threadIdx.x) % team_threads;
  const int warp = tid >> 5;
  const int e = tid * 8;
  const bool col = e < a.D;
  const int64_t b = blockIdx.y, r0 = static_cast<int64_t>(blockIdx.x) * a.chunk;
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.S - r0));
  const float inv_d = __fdiv_rn(1.0f, static_cast<float>(a.D));
  const uint32_t row_bytes = static_cast<uint32_t>(a.D) * 2, stage_bytes = R * 4 * row_bytes;
  const uint32_t ring = smem_addr(dyn) + team * NS * stage_bytes, bar0 = smem_addr(bars) + team * NS * 8;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(bar0 + 8 * i, 1);
    fence_mbar_init();
  }
  for (int i = static_cast<int>(threadIdx.x); i < 2 * 8 * 8 * 16; i += static_cast<int>(blockDim.x)) {
    (&red8[0][0][0][0])[i] = 0.0f;
    if (i < 2 * 8 * 4 * 16) (&red4[0][0][0][0])[i] = 0.0f;
  }
  __syncthreads();
  pdl_wait();
  pdl_trigger();

  // Pair i of the team: rows (i * teams + team) * R of the chunk.
  const int pairs = (rows + R - 1) / R;
  const int mine = pairs > team ? (pairs - team + teams - 1) / teams : 0;
  const uint16_t* src[4] = {a.gh, a.gz, a.z, a.x};
  auto request = [&](int i) {
    const int r = (i * teams + team) * R, n = min(R, rows - r);
    const uint32_t bar = bar0 + 8 * (i % NS), dst = ring + (i % NS) * stage_bytes;
    mbar_arrive_expect_tx(bar, n * (a.gz ? 4 : 3) * row_bytes);
    for (int k = 0; k < n; ++k)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (src[t] != nullptr)
          bulk_g2s(dst + (k * 4 + t) * row_bytes, src[t] + (b * a.S + r0 + r + k) * a.D, row_bytes, bar);
  };
  int asked = 0;
  if (tid == 0)
    for (; asked < NS - 1 && asked < mine; ++asked) request(asked);

  f2_t gw[4] = {}, pw[4] = {};  // gate * post, scale * pre
  if (col) {
    f2_t u[4];
    load4pf(a.post + e, u);
    load4p<DT>(a.gate ? a.gate + b * a.D + e : nullptr, 1.0f, gw);
#pragma unroll
    for (int j = 0; j < 4; ++j) gw[j] = mul2(gw[j], u[j]);
    load4pf(a.pre + e, u);
    load4p<DT>(a.scale ? a.scale + b * a.D + e : nullptr, 1.0f, pw);
#pragma unroll
    for (int j = 0; j < 4; ++j) pw[j] = mul2(pw[j], u[j]);
  }
  f2_t P[4] = {}, Q[4] = {}, G[4] = {};
  bool ok = true;
  const f2_t alpha = splat2(a.alpha);
  for (int i = 0; i < mine; ++i) {
    const int r = (i * teams + team) * R;
    // A thread reads its own 16 bytes of each row alone; one past the last
    // column reads nothing, and its sums are zero.
    uint8_t* at = dyn + (team * NS + i % NS) * stage_bytes + (col ? tid * 16 : 0);
    auto piece = [&](int k, int t) -> uint8_t* { return at + (k * 4 + t) * row_bytes; };
    ok = ok && mbar_wait(bar0 + 8 * (i % NS), (i / NS) & 1);
    if (col) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        if (r + k < rows) continue;
#pragma unroll
        for (int t = 0; t < 4; ++t) st16(piece(k, t), make_uint4(0, 0, 0, 0));  // no such row
      }
    }
    float sums[8] = {}, more[4] = {};
    if (col) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        f2_t g[4], z[4], x[4], gz[4] = {}, s0 = 0, s1 = 0, s2 = 0, s3 = 0, s4 = 0, s5 = 0;
        unpack4p<DT>(lds16(piece(k, 0)), g);
        if (a.gz != nullptr) unpack4p<DT>(lds16(piece(k, 1)), gz);
        unpack4p<DT>(lds16(piece(k, 2)), z);
        unpack4p<DT>(lds16(piece(k, 3)), x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f2_t p = mul2(g[j], pw[j]), t = mul2(x[j], gw[j]);
          s0 = fma2(z[j], z[j], s0);
          s1 = fma2(x[j], x[j], s1);
          s2 = fma2(p, z[j], s2);
          s3 = fma2(gz[j], t, s3);
          s4 = fma2(p, t, s4);
          s5 = fma2(z[j], t, s5);
        }
        sums[k] = sum2(s0);
        sums[2 + k] = sum2(s1);
        sums[4 + k] = sum2(s2);
        sums[6 + k] = sum2(s3);
        more[k] = sum2(s4);
        more[2 + k] = sum2(s5);
      }
    }
    const float own = warp_sum8(sums), own4 = warp_sum4(more);
    if ((lane & 3) == 0) red8[i & 1][team][lane >> 2][warp] = own;
    if ((lane & 7) == 0) red4[i & 1][team][lane >> 3][warp] = own4;
    named_bar_sync(1 + team, team_threads);
    // The team is done with pair i - 1: its stage takes pair i + 2.
    if (tid == 0 && ok && asked < mine) {
      fence_proxy_async_smem();
      request(asked++);
    }
    // Lanes of the first four values turn them into reciprocal roots.
    const float all = team_sum8(red8[i & 1][team]), all4 = team_sum4(red4[i & 1][team]);
    const float root = rms_scale(all, inv_d, a.eps);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const float rz = __shfl_sync(kFull, root, 4 * k), rx = __shfl_sync(kFull, root, 8 + 4 * k);
      const float c = __shfl_sync(kFull, all, 16 + 4 * k) * rz * inv_d;  // mean(p zh)
      const float gzt = __shfl_sync(kFull, all, 24 + 4 * k);
      const float pt = __shfl_sync(kFull, all4, 8 * k), zt = __shfl_sync(kFull, all4, 16 + 8 * k);
      // mean(m xh)
      const float d = __fmaf_rn(rz, __fmaf_rn(-c * rz, zt, pt), gzt) * rx * inv_d;
      if (!col) continue;
      f2_t g[4], z[4], x[4], gz[4] = {}, o[4];
      unpack4p<DT>(lds16(piece(k, 0)), g);
      if (a.gz != nullptr) unpack4p<DT>(lds16(piece(k, 1)), gz);
      unpack4p<DT>(lds16(piece(k, 2)), z);
      unpack4p<DT>(lds16(piece(k, 3)), x);
      const f2_t rz2 = splat2(rz), rx2 = splat2(rx), nc = splat2(-c), nd = splat2(-d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f2_t zh = mul2(z[j], rz2), xh = mul2(x[j], rx2);
        const f2_t dz = fma2(rz2, fma2(zh, nc, mul2(g[j], pw[j])), gz[j]);
        P[j] = fma2(g[j], zh, P[j]);
        Q[j] = fma2(dz, xh, Q[j]);
        G[j] = add2(G[j], g[j]);
        o[j] = mul2(alpha, dz);
        x[j] = mul2(rx2, fma2(xh, nd, mul2(dz, gw[j])));
      }
      if (r + k < rows) {
        const int64_t to = (b * a.S + r0 + r + k) * a.D + e;
        st16(a.dres + to, pack4p<DT>(o));
        st16(a.dx + to, pack4p<DT>(x));
      }
    }
  }
  // After a wait that gave up: copies in flight land before the block ends.
  if (tid == 0 && !ok)
    for (int i = asked > NS ? asked - NS : 0; i < asked; ++i) mbar_wait(bar0 + 8 * (i % NS), (i / NS) & 1);

  // The teams' column sums, in order, through the ring.
  f2_t* sums[3] = {P, Q, G};
  if (teams > 1) {
    f2_t* f = reinterpret_cast<f2_t*>(dyn);
    const int half = a.D / 2;
    __syncthreads();
    if (team > 0 && col)
#pragma unroll
      for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[((team - 1) * 3 + n) * half + tid * 4 + j] = sums[n][j];
    __syncthreads();
    if (team == 0 && col)
      for (int t = 0; t + 1 < teams; ++t)
#pragma unroll
        for (int n = 0; n < 3; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) sums[n][j] = add2(sums[n][j], f[(t * 3 + n) * half + tid * 4 + j]);
  }
  if (team == 0 && col) {
    f2_t* p = reinterpret_cast<f2_t*>(a.part + (b * gridDim.x + blockIdx.x) * 3 * a.D + e);
#pragma unroll
    for (int n = 0; n < 3; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) p[n * (a.D / 2) + j] = sums[n][j];
  }
}

constexpr int kFinCols = 16, kFinSlots = 16, kFinThreads = kFinCols * kFinSlots;
constexpr int kFinBatch = 5;  // chunks that a thread has under way

struct SandwichFinalArgs {
  const float* part;
  const uint16_t *gate, *scale;  // [B, D] or null
  const float *post, *pre;       // [D]
  uint16_t *dgate, *dshift, *dscale;  // [B, D] or null
  float *dpost, *dpre;                // [D]
  int64_t B;
  int chunks, D;
};

// 16 columns a block, so that 2048 columns take most multiprocessors; a thread
// sums every 16th chunk (of a group's samples) of one column, then one thread a
// sum and column adds the slots.  Five chunks are asked for at once: 148 blocks'
// are two round trips to L2.  With 32 columns and 1024 threads, added by warps,
// both kernels took 9.4 us for 64 x 2048, 8.1 so.
template <int DT>
__global__ void __launch_bounds__(kFinThreads) sandwich_final_kernel(const SandwichFinalArgs a) {
  __shared__ float red[3][kFinSlots][kFinCols + 1];
  __shared__ float both[4][2][kFinCols];  // dpre and dpost of the groups
  const int t = static_cast<int>(threadIdx.x), c = t % kFinCols, at = static_cast<int>(blockIdx.x) * kFinCols + c;
  const bool col = at < a.D;
  // Groups of slots take samples in turn; a slot adds every `per`-th chunk.
  const int groups = a.B >= 4 ? 4 : a.B >= 2 ? 2 : 1, per = kFinSlots / groups;
  const int slot = t / kFinCols, g = slot / per, w = slot % per;
  // The thread that adds the slots of sum i: 0 P, 1 Q, 2 gh.
  const int sg = slot / 3, i = slot % 3;
  uint16_t* out = i == 0 ? a.dscale : i == 1 ? a.dgate : a.dshift;
  const uint16_t* factor = i == 0 ? a.scale : a.gate;
  pdl_wait();
  pdl_trigger();
  const float norm = !col || i == 2 ? 1.0f : __ldg((i == 0 ? a.pre : a.post) + at);
  float dnorm = 0.0f;
  for (int64_t b0 = 0; b0 < a.B; b0 += groups) {
    float s[3] = {};
    if (col && b0 + g < a.B) {
      const float* base = a.part + (b0 + g) * a.chunks * 3 * a.D + at;
      for (int n0 = w; n0 < a.chunks; n0 += kFinBatch * per) {
        float v[kFinBatch][3];
#pragma unroll
        for (int u = 0; u < kFinBatch; ++u)
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const int n = n0 + u * per;
            v[u][k] = n < a.chunks ? __ldcg(base + (static_cast<int64_t>(n) * 3 + k) * a.D) : 0.0f;
          }
#pragma unroll
        for (int u = 0; u < kFinBatch; ++u)
#pragma unroll
          for (int k = 0; k < 3; ++k) s[k] += v[u][k];
      }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) red[k][slot][c] = s[k];
    __syncthreads();
    if (col && sg < groups && b0 + sg < a.B) {
      const int64_t o = (b0 + sg) * a.D + at;
      float sum = 0.0f;
      for (int k = 0; k < per; ++k) sum += red[i][sg * per + k][c];
      if (i < 2) dnorm = __fmaf_rn(factor ? load1<DT>(factor + o) : 1.0f, sum, dnorm);
      if (out) out[o] = static_cast<uint16_t>(pack2<DT>(norm * sum, 0.0f));
    }
    __syncthreads();
  }
  if (sg < groups && i < 2) both[sg][i][c] = dnorm;
  __syncthreads();
  if (slot < 2 && col) {
    float sum = 0.0f;
    for (int k = 0; k < groups; ++k) sum += both[k][slot][c];
    (slot == 0 ? a.dpre : a.dpost)[at] = sum;
  }
}

// The order of the column sums follows from the sizes alone.
static int64_t bwd_chunk(int64_t B, int64_t S, int64_t D) {
  return rows_of_block(B, S, teams_of(static_cast<int>(D)) * kBwdRows);
}
static bool check_sandwich(int64_t B, int64_t S, int64_t D, int dtype) {
  return check(B >= 0 && B <= 65535, "batch must be in [0, 65535]") &&
         check(S >= 0 && S <= (1 << 30), "seq must be in [0, 2^30]") &&
         check(B * S <= INT64_C(0x7fffffff), "batch * seq must be below 2^31") &&
         ((D >= 8 && D % 8 == 0 && D <= kMaxRowDim) ||
          check(false, "dim must be a multiple of 8 in [8, " + std::to_string(kMaxRowDim) + "], got " + std::to_string(D))) &&
         check_dtype(dtype);
}
static bool check_opt16(const void* p, const char* n) {
  return aligned(p, 16) || check(false, std::string(n) + " is not 16-byte aligned");
}

cudaError_t read_status_sandwich(int* status, bool clear) { return tu_status(status, clear); }

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
  return g.done(q != nullptr ? launch_fwd<true>(a, B, S, dtype, st) : launch_fwd<false>(a, B, S, dtype, st));
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
  if (batch > 65535 || seq > (1 << 30) || dim > kMaxRowDim || dim % 8 != 0) return SIZE_MAX;
  const int64_t c = bwd_chunk(batch, seq, dim);
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
  a.chunk = static_cast<int>(bwd_chunk(batch, seq, dim));
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
  const int team = team_threads_of(a.D), teams = teams_of(a.D);
  const dim3 block(static_cast<unsigned>(team * teams));
  const size_t smem = bwd_smem(a.D);
  cudaError_t e = dtype == kBf16 ? ensure_smem(sandwich_bwd_kernel<kBf16>, smem) : ensure_smem(sandwich_bwd_kernel<kFp16>, smem);
  if (e != cudaSuccess) return g.done(e);
  e = dtype == kBf16 ? launch_pdl(sandwich_bwd_kernel<kBf16>, grid, block, smem, st, a, team, teams)
                     : launch_pdl(sandwich_bwd_kernel<kFp16>, grid, block, smem, st, a, team, teams);
  if (e != cudaSuccess) return g.done(e);
  const dim3 fg(static_cast<unsigned>((dim + kFinCols - 1) / kFinCols));
  return g.done(dtype == kBf16 ? launch_pdl(sandwich_final_kernel<kBf16>, fg, dim3(kFinThreads), 0, st, f)
                               : launch_pdl(sandwich_final_kernel<kFp16>, fg, dim3(kFinThreads), 0, st, f));
}
