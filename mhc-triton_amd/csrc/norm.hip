// RMS norm of a branch's input rows, with the residual's addition in front, backward, and with an
// output in 8 bits; and the 8-bit quantiser alone.
//
//   h = x + residual   (rounded to the rows' type: the residual stream as it is stored)
//   r = 1 / sqrt(mean_d h_d^2 + eps),   y_d = h_d r w_d
//   dh_d = r (g_d - n_d mean_k(g_k n_k)) + (gradient of h),   g = w dy,  n = r h
//   dw_d = sum_rows dy_d n_d
//
// All of it in fp32 from the stored values.  y is the norm of the *stored* h: the next layer reads
// that h, and the backward has nothing else, so forward and backward see the same function.
//
// A team (a wave, or a workgroup) holds one row in registers, NV vectors per lane, so
// each tensor passes the bus once; a workgroup walks over rows with the weight kept in registers.
#include "stream_kernels.hpp"

namespace mhc {

int check_workspace(const char* who, const void* ws, size_t have, size_t need);

// Sum over the wave, the same bits in every lane: DPP inside rows of 16, then two lane swaps.
__device__ __forceinline__ float wave_total(float v) {
  v = sum_all16(v);
  const uint32_t b = __float_as_uint(v);
  const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  const uint32_t c = __float_as_uint(v);
  const auto q = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// The same in fp64: both halves of a value take the same lanes.
template <class F>
__device__ __forceinline__ double both_halves(double v, F&& f) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)f((uint32_t)(b >> 32)) << 32 | f((uint32_t)b));
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  return both_halves(v, [](uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false); });
}
__device__ __forceinline__ double wave_total(double v) {
  v += dpp64<kDppQuadXor1>(v);
  v += dpp64<kDppQuadXor2>(v);
  v += dpp64<kDppRowRor8>(v);
  v += dpp64<kDppRowRor4>(v);
  v = both_halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false)[0]; }) +
      both_halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane16_swap(x, x, false, false)[1]; });
  return both_halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false)[0]; }) +
         both_halves(v, [](uint32_t x) { return __builtin_amdgcn_permlane32_swap(x, x, false, false)[1]; });
}

// 1 / sqrt(m) to about 2^-45 of itself: fp32's and one Newton step where fp32 holds m.  What it is for is rounded to
// fp32.
__device__ __forceinline__ double rsqrt64(double m) {
  const float f = (float)m;
  if (!(f > 1e-37f && f < 1e37f)) return 1. / sqrt(m);
  const double r = (double)__builtin_amdgcn_rsqf(f);
  return r * (1.5 - 0.5 * m * r * r);
}

// A team is a wave (WAVE: four rows a workgroup of 256) or the whole workgroup, of as many waves as the row
// needs, 16 at most.
constexpr int kTeamWaves = 16;

template <bool WAVE>
__device__ __forceinline__ uint32_t team_lane() { return WAVE ? threadIdx.x & 63 : threadIdx.x; }
template <bool WAVE>
__device__ __forceinline__ uint32_t team_size() { return WAVE ? 64 : blockDim.x; }
template <bool WAVE>
constexpr int kTeamRows = WAVE ? 4 : 1;

// Sum over a team, in wave order.  `turn` alternates between the halves of `lds`, so one barrier per row
// is enough.
template <bool WAVE, typename F>
__device__ __forceinline__ F team_sum(F v, F (&lds)[2][kTeamWaves], int turn) {
  v = wave_total(v);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) lds[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[turn][0];
    for (uint32_t i = 1; i < blockDim.x / 64; ++i) v += lds[turn][i];
  }
  return v;
}

// The vectors of a row that a lane holds: c = lane + v * team, `ok` where c is inside the row.
template <int W, bool RAG, bool WAVE, int NV>
struct RowPart {
  uint32_t col[NV], skip[NV];
  bool ok[NV];
  __device__ __forceinline__ RowPart(uint32_t D) {
    const uint32_t lane = team_lane<WAVE>(), nch = (D + W - 1) / W;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const uint32_t c = lane + v * team_size<WAVE>();
      ok[v] = c < nch;
      const RowCol<W, RAG> rc(ok[v] ? c : 0, D);
      col[v] = rc.col;
      skip[v] = rc.skip;
    }
  }
};

template <typename T, int W, bool RAG, int NV, bool NT, typename P>
__device__ __forceinline__ void load_row(const T* row, int64_t D, const P& p, Frag<T, W> (&f)[NV]) {
  const typename SpanOf<T, W, RAG>::type sp(row, D);
#pragma unroll
  for (int v = 0; v < NV; ++v)
    if (p.ok[v]) f[v].template load<NT>(sp, p.col[v]);
}

template <int W, int NV, typename P>
__device__ __forceinline__ void load_weight(const float* w, const P& p, float (&f)[NV][W]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
#pragma unroll
    for (int e = 0; e < W; ++e) f[v][e] = p.ok[v] ? 1.f : 0.f;
    if (!w || !p.ok[v]) continue;
    if constexpr (W >= 4) {
#pragma unroll
      for (int q = 0; q < W / 4; ++q) RawVec<float>::unpack(__builtin_bit_cast(f32x4, load16_any(w + p.col[v] + 4 * q, false)), f[v] + 4 * q);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) f[v][e] = w[p.col[v] + e];
    }
  }
}

// 8-bit microscaled output: the smallest power of two that brings a block's largest magnitude to 448
// (the largest e4m3 value) or below, so nothing saturates; bytes are 127 + exponent, 255 (NaN) for a
// block that holds an infinity or a NaN.  From the bits: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t mx_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  if (b >= 0x7f800000u) return 255;
  const int k = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b == 0 || k < -127 ? 0 : (uint32_t)(k + 127);
}

// 2^-k of the scale byte 127 + k (exact; k = -127 gives 2^127).
__device__ __forceinline__ float mx_inverse(uint32_t scale) { return __uint_as_float((254u - scale) << 23); }

// W values over their block's scale in 8 bits, W / 4 dwords.  A block of scale NaN gets NaN throughout.
template <int W>
__device__ __forceinline__ void mx_pack(const float (&y)[W], uint32_t scale, uint32_t (&q)[W / 4]) {
  const float inv = mx_inverse(scale);
#pragma unroll
  for (int i = 0; i < W / 4; ++i) {
    int d = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i] * inv, y[4 * i + 1] * inv, 0, false);
    d = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2] * inv, y[4 * i + 3] * inv, d, true);
    q[i] = scale == 255 ? 0x7f7f7f7fu : (uint32_t)d;
  }
}

// Largest magnitude of a block of 32: 4 lanes of 8 values or 8 lanes of 4.  A NaN counts as the
// largest (its bits, sign cleared, are above infinity's), so bits are compared.
template <int W>
__device__ __forceinline__ float block_amax(const float (&y)[W]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < W; ++e) m = max(m, __float_as_uint(y[e]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, kDppQuadXor1, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, kDppQuadXor2, 0xF, 0xF, false));
  if constexpr (W == 4) m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));  // row_half_mirror
  return __uint_as_float(m);
}

constexpr int kMxBlock = 32;

template <int W>
__device__ __forceinline__ void mx_store(uint8_t* q, const uint32_t (&d)[W / 4]) {
  if constexpr (W == 8) __builtin_nontemporal_store((uint64_t)d[1] << 32 | d[0], reinterpret_cast<uint64_t*>(q));
  else __builtin_nontemporal_store(d[0], reinterpret_cast<uint32_t*>(q));
}

struct NormArgs {
  const void *x, *res;
  const float* w;
  void *y, *h;        // y: rows in T, or 8-bit values
  uint8_t* scales;    // 8-bit output only
  float* rstd;        // may be null
  int64_t R, D, ns;   // ns: scale bytes per row
  float eps;
};

// Forward.  Bound by the bus: x and the residual in, y and h out, each once.  16384 x 4096 bf16 with a residual
// 86.6 us (6.2 TB/s), the same in fp32 174 (6.2), 8192 x 7168 into 8 bits 72 us (5.7 TB/s), one row of 4096 2.6 us.  Ragged
// rows of three or four vectors a lane leave one wave a SIMD: 3069 x 1500 fp16 8-9 us, 1504 5.4; beyond a wave bf16
// 8192 x 4098 with a residual 52 us (5.2 TB/s).
template <typename T, int W, bool RAG, bool WAVE, int NV, bool RES, bool MX>
__global__ __launch_bounds__(WAVE ? 256 : 64 * kTeamWaves) void norm_fwd_kernel(NormArgs a) {
  constexpr int ROWS = kTeamRows<WAVE>;
  // 8 bits: the sum and r in fp64, and y = h w r from fp32 products with their errors, rounded to fp32 once.  A
  // block's scale doubles where its largest value passes a boundary, so an error of y there is one of the
  // whole block.
  using Sum = std::conditional_t<MX, double, float>;
  __shared__ Sum lds[2][kTeamWaves];
  const int64_t D = a.D;
  const RowPart<W, RAG, WAVE, NV> p((uint32_t)D);
  float w[NV][W];
  load_weight(a.w, p, w);
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + (WAVE ? threadIdx.x / 64 : 0); row < a.R; row += (int64_t)gridDim.x * ROWS) {
    Frag<T, W> xf[NV], rf[NV];
    load_row<T, W, RAG, NV, true>((const T*)a.x + row * D, D, p, xf);
    if constexpr (RES) load_row<T, W, RAG, NV, true>((const T*)a.res + row * D, D, p, rf);
    float h[NV][W];
    Sum ss = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!p.ok[v]) {
#pragma unroll
        for (int e = 0; e < W; ++e) h[v][e] = 0.f;
        continue;
      }
      xf[v].unpack(h[v]);
      if constexpr (RES) {
        float r[W];
        rf[v].unpack(r);
#pragma unroll
        for (int e = 0; e < W; ++e) h[v][e] = to_f32(from_f32<T>(h[v][e] + r[e]));
        const typename SpanOf<T, W, RAG>::type hs((T*)a.h + row * D, D);
        st_from<T, W, true>(hs, p.col[v], h[v], p.skip[v]);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) ss += RAG && (uint32_t)e < p.skip[v] ? (Sum)0 : (Sum)h[v][e] * (Sum)h[v][e];
    }
    ss = team_sum<WAVE>(ss, lds, turn);
    turn ^= 1;
    Sum r;
    if constexpr (MX) r = rsqrt64(ss / (double)D + (double)a.eps);
    else r = 1.f / sqrtf(ss * inv_d + a.eps);
    if (a.rstd && team_lane<WAVE>() == 0) a.rstd[row] = (float)r;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float y[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        if constexpr (MX) {
          const float hi = (float)r, lo = (float)(r - (double)hi);
          const float p = h[v][e] * w[v][e], err = fmaf(h[v][e], w[v][e], -p);
          const float q = p * hi, rest = fmaf(p, lo, fmaf(err, hi, fmaf(p, hi, -q)));
          y[e] = q + (rest == rest ? rest : 0.f);  // no error term for what is not finite
        } else {
          y[e] = h[v][e] * r * w[v][e];
        }
      }
      if constexpr (MX) {
        const uint32_t s = mx_scale(block_amax(y));
        uint32_t q[W / 4];
        mx_pack(y, s, q);
        if (p.ok[v]) {
          mx_store<W>((uint8_t*)a.y + row * D + p.col[v], q);
          if (p.col[v] % kMxBlock == 0) a.scales[row * a.ns + p.col[v] / kMxBlock] = (uint8_t)s;
        }
      } else if (p.ok[v]) {
        const typename SpanOf<T, W, RAG>::type ys((T*)a.y + row * D, D);
        st_from<T, W, true>(ys, p.col[v], y, p.skip[v]);
      }
    }
    if constexpr (MX) {  // the scale row's filling
      const int64_t pad = D / kMxBlock + team_lane<WAVE>();
      if (pad < a.ns) a.scales[row * a.ns + pad] = 0;
    }
  }
}

struct NormBwdArgs {
  const void *dy, *h, *dh;  // dh may be null
  const float *w, *rstd;
  void* dx;                 // may be null
  float* part;              // [row_blocks][D] partial weight gradients; null without one
  float* dw;                // few rows: the weight gradient itself, by the workgroups past row_blocks
  int64_t R, D;
  uint32_t row_blocks;
};

// The weight gradient of few rows: 64 columns a workgroup, its waves a share of the rows each.
constexpr int64_t kFewRows = 64;

template <typename T>
__device__ __forceinline__ void few_rows_dw(const NormBwdArgs& a) {
  __shared__ double sum[kTeamWaves][64];
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t d = (int64_t)(blockIdx.x - a.row_blocks) * 64 + (threadIdx.x & 63);
  double s = 0.;
  if (d < a.D) {
#pragma unroll 4
    for (int64_t r = wave; r < a.R; r += waves)
      s += (double)(to_f32(((const T*)a.dy)[r * a.D + d]) * (to_f32(((const T*)a.h)[r * a.D + d]) * a.rstd[r]));
  }
  sum[wave][threadIdx.x & 63] = s;
  __syncthreads();
  if (wave || d >= a.D) return;
  for (int i = 1; i < waves; ++i) s += sum[i][threadIdx.x];
  a.dw[d] = (float)s;
}

// Backward.  Bound by the bus (dy, h and dh in, dx out); the weight gradient stays in registers over all of a team's
// rows.  16384 x 4096 bf16 with dh 87 us and 4.7 us for the reduction (5.8 TB/s together), the same in fp32 177 (6.1);
// 3069 x 1500 fp16 13 us (one wave a SIMD), 8192 x 4098 bf16 56 (4.8 TB/s).  The launch bound of 16 waves leaves 128
// registers: some of ragged 16-bit rows beyond a wave and of fp32 rows beyond 8192 are spilled (8 to 66 of them; 4096 x
// 16384 fp32 228 us, 4.7 TB/s, 16383 370).
template <typename T, int W, bool RAG, bool WAVE, int NV, bool DH>
__global__ __launch_bounds__(WAVE ? 256 : 64 * kTeamWaves) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int ROWS = kTeamRows<WAVE>;
  __shared__ float lds[2][kTeamWaves];
  if (blockIdx.x >= a.row_blocks) return few_rows_dw<T>(a);
  const int64_t D = a.D;
  const RowPart<W, RAG, WAVE, NV> p((uint32_t)D);
  float w[NV][W], dw[NV][W];
  load_weight(a.w, p, w);
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < W; ++e) dw[v][e] = 0.f;
  const float inv_d = 1.f / (float)D;
  int turn = 0;
  const int64_t step = (int64_t)a.row_blocks * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + (WAVE ? threadIdx.x / 64 : 0);
  Frag<T, W> yf[NV], hf[NV], gf[NV];
  float r = 0.f;
  auto load = [&](int64_t row) {
    load_row<T, W, RAG, NV, true>((const T*)a.dy + row * D, D, p, yf);
    load_row<T, W, RAG, NV, true>((const T*)a.h + row * D, D, p, hf);
    if constexpr (DH) load_row<T, W, RAG, NV, true>((const T*)a.dh + row * D, D, p, gf);
    r = a.rstd[row];
  };
  if (row < a.R) load(row);
  for (; row < a.R; row += step) {
    float g[NV][W], n[NV][W], u[NV][W];
    const float rs = r;
    float c = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!p.ok[v]) continue;
      yf[v].unpack(g[v]);
      hf[v].unpack(n[v]);
      if constexpr (DH) gf[v].unpack(u[v]);
    }
    if (row + step < a.R) load(row + step);  // on their way while this row is summed
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!p.ok[v]) continue;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        n[v][e] *= rs;
        dw[v][e] += g[v][e] * n[v][e];
        g[v][e] *= w[v][e];
        c += RAG && (uint32_t)e < p.skip[v] ? 0.f : g[v][e] * n[v][e];
      }
    }
    c = team_sum<WAVE>(c, lds, turn) * inv_d;
    turn ^= 1;
    if (!a.dx) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!p.ok[v]) continue;
      float d[W];
#pragma unroll
      for (int e = 0; e < W; ++e) {
        d[e] = rs * (g[v][e] - n[v][e] * c);
        if constexpr (DH) d[e] += u[v][e];
      }
      const typename SpanOf<T, W, RAG>::type ds((T*)a.dx + row * D, D);
      st_from<T, W, true>(ds, p.col[v], d, p.skip[v]);
    }
  }
  if (!a.part) return;
  float* out = a.part + (int64_t)blockIdx.x * D;
  if constexpr (WAVE) {  // the workgroup's four rows' sums, in wave order
    constexpr int TEAM = 64;
    __shared__ float sum[ROWS][TEAM * NV * W];
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < W; ++e) sum[team][(v * W + e) * TEAM + lane] = dw[v][e];
    __syncthreads();
    if (team) return;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int i = (v * W + e) * TEAM + lane;
        dw[v][e] = (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
      }
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (!p.ok[v]) continue;
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (!RAG || (uint32_t)e >= p.skip[v]) out[p.col[v] + e] = dw[v][e];
  }
}

// dw[d] = sum over the partial records in fp64 (they are the sum's largest terms): 16 columns a workgroup, 16
// groups of records side by side, eight loads of a lane in flight.
constexpr int kDwCols = 16, kDwGroups = 16;

__global__ __launch_bounds__(kDwCols * kDwGroups) void norm_dw_reduce_kernel(const float* __restrict__ part,
                                                                            float* __restrict__ dw, int n, int64_t D) {
  __shared__ double sum[kDwGroups][kDwCols];
  const int col = threadIdx.x % kDwCols, grp = threadIdx.x / kDwCols;
  const int64_t d = (int64_t)blockIdx.x * kDwCols + col;
  double s = 0.;
  if (d < D) {
    int i = grp;
    for (; i + 7 * kDwGroups < n; i += 8 * kDwGroups) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = part[(int64_t)(i + k * kDwGroups) * D + d];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    for (; i < n; i += kDwGroups) s += part[(int64_t)i * D + d];
  }
  sum[grp][col] = s;
  __syncthreads();
  if (grp || d >= D) return;
#pragma unroll
  for (int i = 1; i < kDwGroups; ++i) s += sum[i][col];
  dw[d] = (float)s;
}

// The quantiser alone: a lane per vector, rows of whole blocks.  Bound by the bus: 8192 x 7168 bf16 35 us (5.1 TB/s),
// fp32 57 (5.2), experts' weights of 32768 x 7168 bf16 125 us (5.7), 64 x 4096 3.2 us.
template <typename T, int W>
__global__ __launch_bounds__(kThreads) void quantize_mx_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                               uint8_t* __restrict__ scales, int64_t R, int64_t D,
                                                               int64_t ns) {
  // A row has ns blocks; those past D are filled.  Lanes of one block are neighbours.
  constexpr int LANES = kMxBlock / W;
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t block = i / LANES, row = block / ns, b = block - row * ns;
  const int64_t col = b * kMxBlock + (i % LANES) * W;
  const bool in = row < R && col < D;
  float v[W];
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = 0.f;
  if (in) ld<T, W, true>(x + row * D + col, v);
  const uint32_t s = mx_scale(block_amax(v));
  uint32_t d[W / 4];
  mx_pack(v, s, d);
  if (in) mx_store<W>(q + row * D + col, d);
  if (row < R && i % LANES == 0) scales[row * ns + b] = (uint8_t)s;
}

// Rows of up to this many elements fit the registers of the widest team.
constexpr int64_t kNormMaxDim = 16384;

// A workgroup a row (or four) forward, four of them a CU: they start and end apart, which is worth the
// weight's vectors read again for each.  16384 x 4096 bf16 with a residual: two to eight workgroups a CU that
// loop over rows 92-99 us, a row each 86.6 (6.2 TB/s) and 89.0 without the limit.
constexpr int64_t kNormFwdBlocks = ((int64_t)1 << 22) - 1;
static_assert(kNormFwdBlocks * 64 * kTeamWaves < (int64_t)1 << 32, "the runtime takes fewer than 2^32 work items");

// Workgroups of the backward at most, each with a partial weight gradient: half as many of four waves that
// each hold a sum.  More write and add up more partials, fewer leave CUs waiting (us at 256 / 512 / 1024):
// 16384 x 4096 bf16 with a residual 117 / 92 / 104, 3069 x 1500 fp16 (waves) 12.5 / 17 / 21.  A team has two
// rows at least, for the same reason: 1000 x 256 bf16 7.6 -> 5.7 us.
constexpr int64_t kNormBwdBlocks = 512;
constexpr int kBwdRows = 2;

template <bool W, int N>
struct Team {
  static constexpr bool WAVE = W;
  static constexpr int NV = N;
};

// The team for rows of `nch` vectors of W, fn(Team, threads): a wave up to 256 vectors; beyond, a workgroup
// of as many waves as two vectors a lane need (four, past 16 waves).  D = 7168 bf16, seven waves of two
// against four of four: to 8 bits 75.7 -> 72.1 us.  A wave against a workgroup of two vectors a lane, 16384 rows of
// 1024 / 1536 / 2048 bf16 with a residual (us): forward 25 / 37 / 47 and 39 / 47 / 54, backward 29 / 41 / 50 and
// 57 / 61 / 65; ragged, of 1030 / 2044: backward 35 / 47 and 71 / 67, but forward 60 / 71 and 54 / 59.  Single
// elements are rows below one vector, and 16-bit rows end at 16 waves of two.
template <int W, class F>
static int with_team(int64_t nch, F&& fn) {
  if (W == 1 || nch <= 64) return fn(Team<true, 1>{}, 256);
  if constexpr (W > 1) {
    if (nch <= 128) return fn(Team<true, 2>{}, 256);
    if (nch <= 256) return fn(Team<true, 4>{}, 256);
    if (W >= 8 || nch <= 2 * 64 * kTeamWaves) return fn(Team<false, 2>{}, (int)((nch + 127) / 128 * 64));
    if constexpr (W < 8) return fn(Team<false, 4>{}, (int)((nch + 255) / 256 * 64));
  }
}
static_assert(kNormMaxDim <= 8 * 2 * 64 * kTeamWaves && kNormMaxDim <= 4 * 4 * 64 * kTeamWaves, "the widest rows fit");

// Whole vectors, ragged vectors, or (rows below one vector) single elements.
template <int WV, class F>
static int with_row_width(int64_t D, std::initializer_list<const void*> ptrs, F&& fn) {
  bool vec = D % WV == 0;
  for (const void* p : ptrs) vec = vec && (!p || aligned16(p));
  if (vec) return fn(std::integral_constant<int, WV>{}, std::false_type{});
  if (D >= WV) return fn(std::integral_constant<int, WV>{}, std::true_type{});
  return fn(std::integral_constant<int, 1>{}, std::false_type{});
}

static int64_t norm_blocks(int64_t R, int rows, int64_t cap) {
  const int64_t n = (R + rows - 1) / rows;
  return n < cap ? n : cap;
}

static int check_rows(const char* who, int64_t R, int64_t D) {
  if (R < 0 || D < 0) {
    set_error("%s: negative size (R=%lld D=%lld)", who, (long long)R, (long long)D);
    return MHC_ERR_ARG;
  }
  if (D > kNormMaxDim) {
    set_error("%s: rows of %lld elements; at most %lld", who, (long long)D, (long long)kNormMaxDim);
    return MHC_ERR_ARG;
  }
  return MHC_OK;
}

static int64_t mx_scale_row(int64_t D) { return (D + 127) / 128 * 4; }

template <bool MX>
static int norm_forward(const char* who, NormArgs a, int dtype, hipStream_t st) {
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    auto go = [&](auto wc, auto rag) {
      constexpr int W = decltype(wc)::value;
      constexpr bool RAG = decltype(rag)::value;
      return with_team<W>((a.D + W - 1) / W, [&](auto team, int threads) -> int {
        constexpr bool WAVE = decltype(team)::WAVE;
        constexpr int NV = decltype(team)::NV;
        const dim3 grid((unsigned)norm_blocks(a.R, kTeamRows<WAVE>, kNormFwdBlocks));
        const size_t cap = WAVE || threads > 512 ? 0 : occupancy_lds(4);
        if (a.res) norm_fwd_kernel<T, W, RAG, WAVE, NV, true, MX><<<grid, threads, cap, st>>>(a);
        else norm_fwd_kernel<T, W, RAG, WAVE, NV, false, MX><<<grid, threads, cap, st>>>(a);
        return hip_status(hipGetLastError(), who);
      });
    };
    if constexpr (MX) return go(std::integral_constant<int, Vec<T>::N>{}, std::false_type{});
    else return with_row_width<Vec<T>::N>(a.D, {a.x, a.res, a.y, a.h}, go);
  });
}

static bool all_aligned16(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return true;
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_rms_norm_forward(const void* x, const void* residual, int dtype, const float* weight, void* y,
                                    void* h, float* rstd, int64_t R, int64_t D, float eps, mhc_stream_t stream) {
  if (int rc = check_rows("rms_norm_forward", R, D)) return rc;
  if (R * D == 0) return MHC_OK;
  if (!x || !y || (residual && !h)) {
    set_error("rms_norm_forward: null pointer");
    return MHC_ERR_ARG;
  }
  return norm_forward<false>("rms_norm_forward launch",
                             NormArgs{x, residual, weight, y, h, nullptr, rstd, R, D, 0, eps}, dtype,
                             (hipStream_t)stream);
}

extern "C" int mhc_rms_norm_mx_forward(const void* x, const void* residual, int dtype, const float* weight, void* q,
                                       void* scales, void* h, int64_t R, int64_t D, float eps, mhc_stream_t stream) {
  if (int rc = check_rows("rms_norm_mx_forward", R, D)) return rc;
  if (R * D == 0) return MHC_OK;
  if (!x || !q || !scales || (residual && !h)) {
    set_error("rms_norm_mx_forward: null pointer");
    return MHC_ERR_ARG;
  }
  if (D % kMxBlock || !all_aligned16({x, residual, q, h})) {
    set_error("rms_norm_mx_forward: rows of whole blocks of %d and 16-byte aligned tensors required", kMxBlock);
    return MHC_ERR_ARG;
  }
  return norm_forward<true>("rms_norm_mx_forward launch",
                            NormArgs{x, residual, weight, q, h, (uint8_t*)scales, nullptr, R, D, mx_scale_row(D), eps},
                            dtype, (hipStream_t)stream);
}

extern "C" size_t mhc_rms_norm_backward_workspace_bytes(int64_t R, int64_t D) {
  if (R <= kFewRows || D <= 0) return 0;
  return (size_t)(norm_blocks(R, kBwdRows, kNormBwdBlocks) * D) * sizeof(float);
}

extern "C" int mhc_rms_norm_backward(const void* dy, const void* h, const void* dh, int dtype, const float* weight,
                                     const float* rstd, void* dx, float* dweight, int64_t R, int64_t D,
                                     void* workspace, size_t workspace_bytes, mhc_stream_t stream) {
  if (int rc = check_rows("rms_norm_backward", R, D)) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (R * D == 0) return dweight ? fill_zero(dweight, D, st) : (int)MHC_OK;  // an empty sum
  if (!dy || !h || !rstd || (!dx && !dweight)) {
    set_error("rms_norm_backward: null pointer");
    return MHC_ERR_ARG;
  }
  if (dweight)
    if (int rc = check_workspace("rms_norm_backward", workspace, workspace_bytes,
                                 mhc_rms_norm_backward_workspace_bytes(R, D)))
      return rc;
  // Few rows: the weight gradient in the same launch, without partials (64 x 4096 bf16 6.7 -> 3.5 us, and a
  // launch less on the host).
  const bool few = dweight && R <= kFewRows;
  NormBwdArgs a{dy, h, dh, weight, rstd, dx, dweight && !few ? (float*)workspace : nullptr, few ? dweight : nullptr, R, D, 0};
  unsigned blocks = 0;
  const int rc = MHC_DISPATCH_DTYPE(dtype, [&] {
    return with_row_width<Vec<T>::N>(D, {dy, h, dh, dx}, [&](auto wc, auto rag) {
      constexpr int W = decltype(wc)::value;
      constexpr bool RAG = decltype(rag)::value;
      return with_team<W>((D + W - 1) / W, [&](auto team, int threads) -> int {
        constexpr bool WAVE = decltype(team)::WAVE;
        constexpr int NV = decltype(team)::NV;
        blocks = (unsigned)norm_blocks(R, kBwdRows * kTeamRows<WAVE>, WAVE ? kNormBwdBlocks / 2 : kNormBwdBlocks);
        a.row_blocks = !few ? blocks : dx ? (unsigned)norm_blocks(R, kTeamRows<WAVE>, kNormBwdBlocks) : 0;
        const dim3 grid(a.row_blocks + (few ? (unsigned)((D + 63) / 64) : 0));
        if (dh) norm_bwd_kernel<T, W, RAG, WAVE, NV, true><<<grid, threads, 0, st>>>(a);
        else norm_bwd_kernel<T, W, RAG, WAVE, NV, false><<<grid, threads, 0, st>>>(a);
        return hip_status(hipGetLastError(), "rms_norm_backward launch");
      });
    });
  });
  if (rc || !dweight || few) return rc;
  norm_dw_reduce_kernel<<<dim3((unsigned)((D + kDwCols - 1) / kDwCols)), kDwCols * kDwGroups, 0, st>>>(a.part, dweight, (int)blocks, D);
  return hip_status(hipGetLastError(), "rms_norm_backward reduce launch");
}

extern "C" int mhc_quantize_mx(const void* x, int dtype, void* q, void* scales, int64_t R, int64_t D,
                               mhc_stream_t stream) {
  if (R < 0 || D < 0 || D % kMxBlock) {
    set_error("quantize_mx: bad size (R=%lld D=%lld; D in whole blocks of %d)", (long long)R, (long long)D, kMxBlock);
    return MHC_ERR_ARG;
  }
  if (R * D == 0) return MHC_OK;
  if (!x || !q || !scales || !all_aligned16({x, q})) {
    set_error("quantize_mx: null pointer, or a tensor that is not 16-byte aligned");
    return MHC_ERR_ARG;
  }
  const int64_t ns = mx_scale_row(D);
  hipStream_t st = (hipStream_t)stream;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    constexpr int W = Vec<T>::N;
    // the runtime takes fewer than 2^32 work items: whole rows of as many, a launch each
    const int64_t lanes = ns * (kMxBlock / W), most = (((int64_t)1 << 32) - kThreads) / lanes;
    if (most < 1) {
      set_error("quantize_mx: rows of %lld elements are too wide", (long long)D);
      return (int)MHC_ERR_ARG;
    }
    for (int64_t r = 0; r < R; r += most) {
      const int64_t rows = R - r < most ? R - r : most, n = (rows * lanes + kThreads - 1) / kThreads;
      quantize_mx_kernel<T, W><<<dim3((unsigned)n), kThreads, 0, st>>>(
          (const T*)x + r * D, (uint8_t*)q + r * D, (uint8_t*)scales + r * ns, rows, D, ns);
      if (int rc = hip_status(hipGetLastError(), "quantize_mx launch")) return rc;
    }
    return (int)MHC_OK;
  });
}
