// Kernels of linear attention with a decay for each head (decay.hip).
//
// One scan serves the forward and every gradient.  Over a sequence's tokens t = 0, 1, ... (from its first row on, or
// from its last one backwards), with l = exp(log decay) of the head and weights q, k, v:
//
//   o_t = a b sum_{s <= t} l^(t-s) (q_t . k_s) v_s  +  a l^(t+L) q_t X_0
//   X_n = l^n X_0 + b sum_{j < n} l^(n-L-j) k_j^T v_j
//
// X is the state that n tokens leave.  Forward L = 1, and the scale is a; backwards L = 0, because X_0 is the gradient of
// a state that the last token has already entered, and the scale is b, because that gradient has none.  A chunk of 64 tokens is matrix products: P = (Q K^T) o (weights, lower triangle),
// O = P V + weights Q X, X' = l^n X + (K^T) (weighted V).
//
// A workgroup takes a segment of a sequence, a head and 64 of the state's columns; each of its four waves holds
// 16 columns of the state, all rows, in registers from the first chunk to the last, and never passes it on.  Q, K
// and V of a chunk go through LDS, the next chunk's are in flight.  P is made once for the four waves and passes
// through LDS.  Segments but the last are first run for their state alone (STATE_ONLY), so that long sequences with
// few heads fill the card; each then starts from the sum of the states before it.
//
// Precision.  The matrix instructions multiply bf16.  Every operand is a sum of bf16 parts: inputs exactly (bf16 one part,
// fp16 two, fp32 three), what is computed (P, the state, weighted V) in as many as keep the error far below one rounding to the
// output's type (two for 16-bit types, three for fp32); the states go out in fp32, so weighted V has three in every type.
// Products of parts whose size is below the last part's are left out.  Sums are fp32.
#pragma once

#include "grouped_kernels.hpp"

namespace mhc {

constexpr int kChunk = 64;     // tokens of a chunk
constexpr int kStateCols = 64; // columns of the state that a workgroup holds

template <typename T> constexpr int kRaw = sizeof(T) == 4 ? 3 : (__is_same(T, __bf16) ? 1 : 2);  // parts of an input
template <typename T> constexpr int kMade = sizeof(T) == 4 ? 3 : 2;                             // of P and the state
constexpr int kWeighted = 3;                                                                     // of weighted V

struct DecayArgs {
  const void *q, *k, *v;
  void* o;
  const float* log_decay;    // [H]
  const int32_t* offsets;    // ends of the packed sequences; null: N sequences of T rows each
  const float* first;        // X_0 of each sequence, or null
  float* last;               // where X goes, or null
  float* parts;              // states that segments leave by themselves, [tile][H][Dk][Dv]
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements; o is contiguous
  int64_t state_row, state_col;                         // of first and last: X's rows and columns
  int64_t R, T;
  int H, N, Dk, Dv, seg, tiles, col_tiles;
  float out_scale, in_scale;  // a, b
  int lag;                    // L
  bool reverse;
};

// Segment `s` of sequence e, whose rows are lo to hi; e = N: rows past the last sequence; -1: none.
struct Segment {
  int e, s;
  int64_t lo, hi;
};

// Tile t: every sequence has a segment at least, so that one without tokens hands its state on.
__device__ __forceinline__ Segment find_segment(const DecayArgs& a, int t) {
  if (!a.offsets) {
    const int per = (int)max((int64_t)1, (a.T + a.seg - 1) / a.seg);
    const int e = t / per;
    return {e < a.N ? e : -1, t - e * per, e * a.T, (e + 1) * a.T};
  }
  const int lane = threadIdx.x & 63;
  int before = 0, end = 0;
  for (int base = 0; base <= a.N; base += 64) {
    const Group g = groups_of(a.offsets, base, a.N, a.R, &end);
    int n = (int)((g.hi - g.lo + a.seg - 1) / a.seg);
    if (base + lane < a.N) n = max(n, 1);
    int upto = n;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    upto += before;
    const uint64_t found = __ballot(t < upto);
    if (found) {
      const int src = __builtin_ctzll(found);
      return {base + src, t - __shfl(upto - n, src, 64), __shfl((int)g.lo, src, 64), __shfl((int)g.hi, src, 64)};
    }
    before = __shfl(upto, 63, 64);
  }
  return {-1, 0, 0, 0};
}

// D[m][n] += sum_k A[m][k] B[n][k] of 16 x 16 x 32: a lane gives row (column) lane % 16 and the eight k of its group
// lane / 16, and holds rows 4 (lane / 16) + r of column lane % 16.
__device__ __forceinline__ f32x4 mm(u32x4 m, u32x4 n, f32x4 acc) { return mma<__bf16>(m, n, acc); }

// sum over parts i of A and j of B with i + j <= TOP
template <int NA, int NB, int TOP>
__device__ __forceinline__ f32x4 mm_parts(const u32x4 (&m)[NA], const u32x4 (&n)[NB], f32x4 acc) {
#pragma unroll
  for (int i = NA - 1; i >= 0; --i)
#pragma unroll
    for (int j = NB - 1; j >= 0; --j)
      if (i + j <= TOP) acc = mm(m[i], n[j], acc);
  return acc;
}

// Two floats as bf16 in a dword, rounded to nearest even, and their values back.
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 p = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(p, bf16x2));
}
__device__ __forceinline__ float low2(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high2(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// N dwords of bf16 pairs in P parts: part p of f is what parts 0 .. p - 1 leave of it, rounded.
template <int P, int N>
__device__ __forceinline__ void split(float (&f)[2 * N], uint32_t (&out)[P][N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t v = pack2(f[2 * i], f[2 * i + 1]);
      out[p][i] = v;
      if (p + 1 < P) {
        f[2 * i] -= low2(v);
        f[2 * i + 1] -= high2(v);
      }
    }
  }
}
template <int P>
__device__ __forceinline__ void split8(float (&f)[8], u32x4 (&out)[P]) {
  uint32_t t[P][4];
  split<P, 4>(f, t);
#pragma unroll
  for (int p = 0; p < P; ++p) out[p] = u32x4{t[p][0], t[p][1], t[p][2], t[p][3]};
}

// A plane of 64 rows of bf16, D = 128 or 64 columns, in 16-byte chunks.  Of the rows that half a wave (transposed
// reads: eight rows of two chunks each) or a quarter (plain reads: 16 rows of one) reads at a time no two meet in a bank.
template <int D>
__device__ __forceinline__ int plane_slot(int r, int c) {
  static_assert(D == 64 || D == 128, "rows of 8 or 16 chunks");
  const int s = D == 128 ? ((r & 7) << 1 | ((r >> 3) & 1)) : (((r >> 1) & 3) << 1 | ((r >> 3) & 1));
  return r * (D / 8) + (c ^ s);
}
// P: read plainly only; columns in the order in which the lanes' k run (below).
__device__ __forceinline__ int p_slot(int r, int c) { return r * 8 + (c ^ ((r >> 1) & 7)); }

// Which token (or state row) of 32 the e-th k of lane group g is: two runs of four, because that is what a transposed
// read or two tiles of a product's result give a lane.
__device__ __forceinline__ int order(int g, int e) { return 16 * (e >> 2) + 4 * g + (e & 3); }

// Transposed: columns c0 .. c0 + 15 of tokens 32 ks .. 32 ks + 31; lane % 16 gets its column's eight tokens in order().
template <int D>
__device__ __forceinline__ u32x4 read_columns(const u32x4* plane, int c0, int ks) {
#ifdef __HIP_DEVICE_COMPILE__
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const int r = 32 * ks + 4 * g + (i >> 2), c = (c0 >> 3) + ((i & 3) >> 1);
  const char* p = reinterpret_cast<const char*>(plane) + (i & 1) * 8;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + plane_slot<D>(r, c) * 16));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + plane_slot<D>(r + 16, c) * 16));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return u32x4{};
#endif
}
// Row r0 + lane % 16, columns 32 ks .. 32 ks + 31 as they lie, or (ORDERED) in order().
template <int D, bool ORDERED>
__device__ __forceinline__ u32x4 read_rows(const u32x4* plane, int r0, int ks) {
  const int lane = threadIdx.x & 63, g = lane >> 4, r = r0 + (lane & 15);
  if constexpr (!ORDERED) return plane[plane_slot<D>(r, 4 * ks + g)];
  const uint64_t* p = reinterpret_cast<const uint64_t*>(plane);
  const uint64_t lo = p[2 * plane_slot<D>(r, 4 * ks + (g >> 1)) + (g & 1)];
  const uint64_t hi = p[2 * plane_slot<D>(r, 4 * ks + 2 + (g >> 1)) + (g & 1)];
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// A chunk's rows of one operand: global memory -> registers -> planes of parts.  CHUNKS: whole aligned vectors.
template <typename T, int D, bool CHUNKS>
struct Feed {
  static constexpr int PER = D / 8, CH = kChunk * PER / kThreads;  // eights of a row; eights of a thread
  static constexpr int W = sizeof(T) / 2;                          // 16-byte loads of an eight
  u32x4 r[CH][W];

  // Token i < n is row i of `base`, or (reverse) row n - 1 - i; rows of `ld` elements, of which `cols` exist.
  __device__ __forceinline__ void load(const T* base, int64_t ld, int cols, int n, bool reverse) {
    [[maybe_unused]] const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(base), 0, (int)(((n - 1) * ld + cols) * (int64_t)sizeof(T)), kBufRsrcDword3);
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int at = q * kThreads + threadIdx.x, i = at / PER, c = at % PER * 8;
      const int row = reverse ? n - 1 - i : i;
      if constexpr (CHUNKS) {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int off = (int)(row * ld + c + 4 * w) * (int)sizeof(T);
          const bool in = i < n && c + 4 * w < cols;
          r[q][w] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? off : kNowhere, 0, 0);
        }
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int left = i < n ? cols - c - 4 * w : 0;
          r[q][w] = load_chunk<T>(base + (i < n ? row * ld + c + 4 * w : 0), left, cols >= kElems<T>);
        }
      }
    }
  }

  // Into kRaw<T> planes.
  __device__ __forceinline__ void store(u32x4* planes) const {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int at = q * kThreads + threadIdx.x, slot = plane_slot<D>(at / PER, at % PER);
      if constexpr (__is_same(T, __bf16)) {
        planes[slot] = r[q][0];
      } else {
        float f[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r[q][e / 4][e % 4]);
        } else {
          RawVec<T>::unpack(__builtin_bit_cast(typename RawVec<T>::type, r[q][0]), f);
        }
        u32x4 p[kRaw<T>];
        split8<kRaw<T>>(f, p);
#pragma unroll
        for (int i = 0; i < kRaw<T>; ++i) planes[i * kChunk * PER + slot] = p[i];
      }
    }
  }
};

// exp(x) of x <= 0 in fp64, as two floats.
struct Power {
  float hi, lo;
};
__device__ __forceinline__ Power power(float log_decay, int64_t n) {
  if (n == 0) return {1.f, 0.f};
  const double p = exp((double)log_decay * (double)n);
  const float hi = (float)p;
  return {hi, (float)(p - (double)hi)};
}

// LDS in 16-byte chunks: K and V, and for outputs Q and P.
template <typename T, int DK, bool STATE_ONLY>
constexpr int kDecayLds = kRaw<T> * kChunk * (DK / 8 * (STATE_ONLY ? 1 : 2) + 8) + (STATE_ONLY ? 0 : kMade<T> * kChunk * 8);

template <typename T, int DK, bool CHUNKS, bool STATE_ONLY>
__global__ __launch_bounds__(kThreads, (kDecayLds<T, DK, STATE_ONLY> * 16 <= 80 * 1024 ? 2 : 1)) void decay_kernel(DecayArgs a) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int RAW = kRaw<T>, MADE = kMade<T>, TD = DK / 16, KS = DK / 32;
  constexpr int QK = kChunk * DK / 8;  // chunks of a plane of Q or K
  __shared__ u32x4 lds[kDecayLds<T, DK, STATE_ONLY>];
  __shared__ float pow_of[kChunk + 1];  // l^0 .. l^64
  u32x4 *lk = lds, *lv = lk + RAW * QK, *lq = lv + RAW * kChunk * 8, *lp = lq + RAW * QK;

  // column tiles of one (segment, head) side by side on one XCD: they read the same Q and K
  const int run = blockIdx.x / 8, unit = run / a.col_tiles * 8 + blockIdx.x % 8, col_tile = run % a.col_tiles;
  if (unit >= a.tiles * a.H) return;
  const int tile = unit / a.H, h = unit - tile * a.H;
  const Segment sg = find_segment(a, tile);
  const int e = __builtin_amdgcn_readfirstlane(sg.e), seg = __builtin_amdgcn_readfirstlane(sg.s);
  if (e < 0) return;
  const int64_t lo = __builtin_amdgcn_readfirstlane((int)sg.lo), hi = __builtin_amdgcn_readfirstlane((int)sg.hi);
  const int len = (int)(hi - lo), begin = seg * a.seg, stop = min(begin + a.seg, len);  // tokens
  const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = col_tile * kStateCols + 16 * wave + li;  // of X and V
  if constexpr (STATE_ONLY) {
    if (e == a.N || stop == len) return;
  } else if (e == a.N) {  // rows of no sequence: zeros
    const int cols = min(a.Dv - col_tile * kStateCols, kStateCols);
    if (!a.o) return;
    T* o = (T*)a.o + ((lo + begin) * a.H + h) * a.Dv + col_tile * kStateCols;
    for (int i = threadIdx.x; i < (stop - begin) * cols; i += kThreads) o[(int64_t)(i / cols) * a.H * a.Dv + i % cols] = from_f32<T>(0.f);
    return;
  }
  const float given = a.log_decay[h], ld = given > 0.f ? 0.f : given;
  if (threadIdx.x <= kChunk) pow_of[threadIdx.x] = power(ld, threadIdx.x).hi;

  // X: rows 16 td + 4 g + r of the wave's columns
  f32x4 x[TD];
#pragma unroll
  for (int td = 0; td < TD; ++td) x[td] = f32x4{0.f, 0.f, 0.f, 0.f};
  if constexpr (!STATE_ONLY) {
    auto add = [&](const float* s, int64_t row, int64_t column, float w) {
#pragma unroll
      for (int td = 0; td < TD; ++td)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 16 * td + 4 * g + r;
          if (d < a.Dk && col < a.Dv) x[td][r] += w * s[d * row + col * column];
        }
    };
    const int64_t size = (int64_t)a.Dk * a.Dv;
    if (a.first) add(a.first + ((int64_t)e * a.H + h) * size, a.state_row, a.state_col, power(ld, begin).hi);
    for (int s = 0; s < seg; ++s)
      add(a.parts + ((int64_t)(tile - seg + s) * a.H + h) * size, a.Dv, 1, power(ld, (int64_t)(seg - 1 - s) * a.seg).hi);
    // the halves of P's 32-token rows that lie above the diagonal
    for (int p = 0; p < MADE; ++p)
      for (int i = threadIdx.x; i < 32 * 8; i += kThreads) {
        const int r = i / 8 < 16 ? i / 8 : 16 + i / 8;
        lp[p * kChunk * 8 + p_slot(r, i % 8)] = u32x4{0, 0, 0, 0};
      }
  }
  __syncthreads();

  // P's ten tiles in or below the diagonal: wave w makes tiles w, w + 4 and w + 8
  constexpr int kTiles = 3;
  int ti[kTiles], tj[kTiles];
  float pw[kTiles][4], qw[4], vw[2][8];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int t = wave + 4 * n;
    ti[n] = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
    tj[n] = t - ti[n] * (ti[n] + 1) / 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int far = 16 * (ti[n] - tj[n]) + li - 4 * g - r;
      pw[n][r] = far >= 0 && t < 10 ? a.out_scale * a.in_scale * pow_of[far] : 0.f;
    }
  }
#pragma unroll
  for (int it = 0; it < 4; ++it) qw[it] = a.out_scale * pow_of[16 * it + li + a.lag];
  auto weigh_v = [&](int n) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) vw[ks][i] = a.in_scale * pow_of[max(n - a.lag - 32 * ks - order(g, i), 0)];
  };
  weigh_v(kChunk);
  Power whole = power(ld, kChunk);

  const T* q = (const T*)a.q + h * a.q_head;
  const T* k = (const T*)a.k + h * a.k_head;
  const T* v = (const T*)a.v + h * a.v_head + col_tile * kStateCols;
  Feed<T, DK, CHUNKS> fq, fk;
  Feed<T, kStateCols, CHUNKS> fv;
  auto first_row = [&](int t, int n) { return a.reverse ? hi - t - n : lo + t; };
  auto load = [&](int t) {
    const int n = min(kChunk, stop - t);
    const int64_t row = first_row(t, n);
    fk.load(k + row * a.k_row, a.k_row, a.Dk, n, a.reverse);
    fv.load(v + row * a.v_row, a.v_row, a.Dv - col_tile * kStateCols, n, a.reverse);
    if constexpr (!STATE_ONLY) fq.load(q + row * a.q_row, a.q_row, a.Dk, n, a.reverse);
  };
  if (begin < stop) load(begin);
  for (int t = begin; t < stop; t += kChunk) {
    const int n = min(kChunk, stop - t);
    fk.store(lk);
    fv.store(lv);
    if constexpr (!STATE_ONLY) fq.store(lq);
    __syncthreads();
    if (t + kChunk < stop) load(t + kChunk);

    u32x4 vr[2][RAW];  // the wave's columns of V
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int p = 0; p < RAW; ++p) vr[ks][p] = read_columns<kStateCols>(lv + p * kChunk * 8, 16 * wave, ks);

    if constexpr (!STATE_ONLY) {
      // P: keys are the product's rows, so that a lane gets four neighbouring keys of one query
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        if (m == 2 && wave > 1) break;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 kf[RAW], qf[RAW];
#pragma unroll
          for (int p = 0; p < RAW; ++p) {
            kf[p] = read_rows<DK, false>(lk + p * QK, 16 * tj[m], ks);
            qf[p] = read_rows<DK, false>(lq + p * QK, 16 * ti[m], ks);
          }
          s = mm_parts<RAW, RAW, RAW - 1>(kf, qf, s);
        }
        float f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) f[r] = pw[m][r] != 0.f ? s[r] * pw[m][r] : 0.f;  // a masked NaN goes, too
        uint32_t parts[MADE][2];
        split<MADE, 2>(f, parts);
        const int slot = p_slot(16 * ti[m] + li, 4 * (tj[m] >> 1) + g);
#pragma unroll
        for (int p = 0; p < MADE; ++p)
          reinterpret_cast<uint64_t*>(lp + p * kChunk * 8 + slot)[tj[m] & 1] = (uint64_t)parts[p][1] << 32 | parts[p][0];
      }
      // Q X: results are (column, query), a lane's query is li of each tile
      f32x4 o[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = x[2 * ks + i / 4][i % 4];
        u32x4 xs[MADE];
        split8<MADE>(f, xs);
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          u32x4 qf[RAW];
#pragma unroll
          for (int p = 0; p < RAW; ++p) qf[p] = read_rows<DK, true>(lq + p * QK, 16 * it, ks);
          o[it] = mm_parts<MADE, RAW, MADE - 1>(xs, qf, o[it]);
        }
      }
      __syncthreads();
      // P V
      f32x4 pv[4];
      float finite = 0.f;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        pv[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks <= it / 2; ++ks) {
          u32x4 pf[MADE];
#pragma unroll
          for (int p = 0; p < MADE; ++p) pf[p] = lp[p * kChunk * 8 + p_slot(16 * it + li, 4 * ks + g)];
          pv[it] = mm_parts<RAW, MADE, MADE - 1>(vr[ks], pf, pv[it]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) finite = __builtin_fmaf(pv[it][r], 0.f, finite);
      }
      if (__any(finite != 0.f)) {
        // An infinity or a NaN among V: zeros above the diagonal have spread it to earlier tokens.  One by one.
        for (int it = 0; it < 4; ++it) {
          pv[it] = f32x4{0.f, 0.f, 0.f, 0.f};
          const int i = 16 * it + li;
          for (int j = 0; j <= 16 * it + 15; ++j) {
            const int at = j & 31, gj = (at >> 2) & 3, ej = (at >> 4) * 4 + (at & 3);  // order(gj, ej) = at
            float pij = 0.f;
            for (int p = 0; p < MADE; ++p)
              pij += to_f32(reinterpret_cast<const __bf16*>(lp + p * kChunk * 8 + p_slot(i, 4 * (j >> 5) + gj))[ej]);
            for (int r = 0; r < 4; ++r) {
              const int c = 16 * wave + 4 * g + r;
              float vj = 0.f;
              for (int p = 0; p < RAW; ++p)
                vj += to_f32(reinterpret_cast<const __bf16*>(lv + p * kChunk * 8 + plane_slot<kStateCols>(j, c >> 3))[c & 7]);
              if (j <= i) pv[it][r] += pij * vj;
            }
          }
        }
      }
      T* out = (T*)a.o;
      const int64_t row = first_row(t, n);
      const int c = col_tile * kStateCols + 16 * wave + 4 * g;
      const bool vec = a.Dv % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const int i = 16 * it + li;
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = pv[it][r] + o[it][r] * qw[it];
        if (i < n && out) store4(out + ((row + (a.reverse ? n - 1 - i : i)) * a.H + h) * a.Dv + c, y, a.Dv - c, vec);
      }
    }

    // X' = l^n X + K^T (weighted V)
    if (n < kChunk) {
      weigh_v(n);
      whole = power(ld, n);
    }
#pragma unroll
    for (int td = 0; td < TD; ++td)
#pragma unroll
      for (int r = 0; r < 4; ++r) x[td][r] = __builtin_fmaf(x[td][r], whole.hi, x[td][r] * whole.lo);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = 0.f;
#pragma unroll
        for (int p = RAW - 1; p >= 0; --p) f[i] += i % 2 ? high2(vr[ks][p][i / 2]) : low2(vr[ks][p][i / 2]);
        f[i] *= vw[ks][i];
      }
      u32x4 vs[kWeighted];
      split8<kWeighted>(f, vs);
#pragma unroll
      for (int td = 0; td < TD; ++td) {
        u32x4 kf[RAW];
#pragma unroll
        for (int p = 0; p < RAW; ++p) kf[p] = read_columns<DK>(lk + p * QK, 16 * td, ks);
        x[td] = mm_parts<RAW, kWeighted, 2>(kf, vs, x[td]);
      }
    }
    __syncthreads();
  }

  float* to = nullptr;
  int64_t row = a.Dv, column = 1;
  if constexpr (STATE_ONLY) {
    to = a.parts + ((int64_t)tile * a.H + h) * a.Dk * a.Dv;
  } else if (a.last && stop == len) {
    to = a.last + ((int64_t)e * a.H + h) * a.Dk * a.Dv;
    row = a.state_row;
    column = a.state_col;
  }
  if (to) {
#pragma unroll
    for (int td = 0; td < TD; ++td)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * td + 4 * g + r;
        if (d < a.Dk && col < a.Dv) to[d * row + col * column] = x[td][r];
      }
  }
#endif
}

// ---------------------------------------------------------------------------
// One token a sequence: X' = l X + k^T v, o = c q X'.  Bound by the states, read and written once.
// ---------------------------------------------------------------------------
struct DecayStepArgs {
  const void *q, *k, *v;
  void* o;
  const float* log_decay;
  const float* state;
  float* state_out;
  const int32_t* slots;  // null: row r has state r
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  int64_t pool;
  int R, H, Dk, Dv, col_tiles;
  float scale;
};

constexpr int kStepCols = 64;   // columns of a workgroup
constexpr int kStepRows = 128;  // most rows of a state

// A lane holds four neighbouring columns of every 16th row.  VEC: they are one aligned load.  Rows that share a slot are
// tokens in their order: the first row's workgroup takes them all, the others leave.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void decay_step_kernel(DecayStepArgs a) {
  constexpr int LANES = kStepCols / 4, TEAMS = kThreads / LANES, Q = kStepRows / TEAMS;
  static_assert(2 * kStepRows == kThreads, "a thread brings one value of k or q");
  __shared__ float sum[TEAMS][kStepCols];
  __shared__ float kq[2][kStepRows];
  __shared__ int next_of;
  const int unit = blockIdx.x / a.col_tiles, c0 = (int)(blockIdx.x % a.col_tiles) * kStepCols;
  const int first = unit / a.H, h = unit - first * a.H;
  const int team = threadIdx.x / LANES, at = (int)threadIdx.x % LANES * 4, col = c0 + at;
  const int64_t slot = a.slots ? a.slots[first] : first;
  T* out = (T*)a.o;
  const bool writes = threadIdx.x < kStepCols && c0 + (int)threadIdx.x < a.Dv;
  if (slot < 0 || slot >= a.pool) {  // a row of no sequence
    if (writes) out[((int64_t)first * a.H + h) * a.Dv + c0 + threadIdx.x] = from_f32<T>(0.f);
    return;
  }
  // the next row behind `from` with this slot (R: none), or -1 if one before the first has it
  auto find_next = [&](int from) {
    if (!a.slots) return a.R;
    if (threadIdx.x == 0) next_of = a.R;
    __syncthreads();
    for (int i = threadIdx.x; i < a.R; i += kThreads)
      if (a.slots[i] == slot) {
        if (i < first) atomicMin(&next_of, -1);
        else if (i > from) atomicMin(&next_of, i);
      }
    __syncthreads();
    return next_of;
  };
  int next = find_next(first);
  if (next < 0) return;
  const float ld = a.log_decay[h], l = expf(ld > 0.f ? 0.f : ld);
  const int64_t base = (slot * a.H + h) * (int64_t)a.Dk * a.Dv;
  float x[Q][4];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int d = team + i * TEAMS;
    const float* p = a.state + base + (int64_t)d * a.Dv + col;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if constexpr (VEC) {
      if (d < a.Dk && col < a.Dv) s = *reinterpret_cast<const f32x4*>(p);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (d < a.Dk && col + w < a.Dv) s[w] = p[w];
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) x[i][w] = s[w];
  }
  for (int r = first;;) {
    const int d0 = threadIdx.x % kStepRows;
    const T* src = threadIdx.x < kStepRows ? (const T*)a.k + r * a.k_row + h * a.k_head : (const T*)a.q + r * a.q_row + h * a.q_head;
    kq[threadIdx.x / kStepRows][d0] = d0 < a.Dk ? to_f32(src[d0]) : 0.f;
    const T* v = (const T*)a.v + r * a.v_row + h * a.v_head;
    float vf[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) vf[w] = col + w < a.Dv ? to_f32(v[col + w]) : 0.f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const float kd = kq[0][team + i * TEAMS], qd = kq[1][team + i * TEAMS];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        x[i][w] = __builtin_fmaf(l, x[i][w], kd * vf[w]);
        o[w] = __builtin_fmaf(qd, x[i][w], o[w]);
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) sum[team][at + w] = o[w];
    __syncthreads();
    if (writes) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < TEAMS; ++i) s += sum[i][threadIdx.x];
      out[((int64_t)r * a.H + h) * a.Dv + c0 + threadIdx.x] = from_f32<T>(a.scale * s);
    }
    if (next >= a.R) break;
    r = next;
    next = find_next(r);  // its barriers also free kq and sum
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int d = team + i * TEAMS;
    float* p = a.state_out + base + (int64_t)d * a.Dv + col;
    if constexpr (VEC) {
      if (d < a.Dk && col < a.Dv) *reinterpret_cast<f32x4*>(p) = f32x4{x[i][0], x[i][1], x[i][2], x[i][3]};
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (d < a.Dk && col + w < a.Dv) p[w] = x[i][w];
    }
  }
}

}  // namespace mhc
