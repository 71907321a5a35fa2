// Kernels of linear attention with a decay for each head (decay.hip).
//
// One scan serves the forward and every gradient.  Over a sequence's tokens t = 0, 1, ... (from its first row on, or
// from its last one backwards), with l = exp(log decay) of the head and weights q, k, v:
//
//   o_t = a b sum_{s <= t} l^(t-s) (q_t . k_s) v_s  +  a l^(t+L) q_t X_0
//   X_n = l^n X_0 + b sum_{j < n} l^(n-L-j) k_j^T v_j
//
// X is the state that n tokens leave.  Forward L = 1, and the scale is a; backwards L = 0, because X_0 is the gradient of
// a state that the last token has already entered, and the scale is b, because that gradient has none.  A chunk of 64
// tokens is matrix products: P = (Q K^T) o (weights, lower triangle), O = P V + weights Q X, X' = l^n X + (K^T) (weighted V).
//
// A workgroup of WAVES waves takes a segment of a sequence and a head, whose state has at most 16 WAVES columns; each wave holds
// 16 columns of the state, all rows, in registers from the first chunk to the last, and never passes it on.  Q, K
// and V of a chunk go through LDS; P is made once for all waves and passes through LDS.  Registers are held below 128
// for bf16, for four waves a SIMD: phases that wait for LDS, for the matrix cores and for the VALU then overlap (four
// waves of 64 columns each and two a SIMD: 198 us where this takes 139; 32 columns a wave: spills, 399 where 16 take 158).
// Segments but the last are first run for their state alone (STATE_ONLY), so that long sequences with
// few heads fill the card; each then starts from the sum of the states before it, which decay_join_kernel has made in
// sequences of more than kSummed.
//
// Bound by the phases of a chunk, which follow one another, and not far behind by memory.  bf16, 4 x 4096 tokens of 32 heads
// of 128: forward 142 us (3.8 TB/s) and 46 for the segments' states, the gradients' three scans together 375 us (2.5 TB/s) and
// 45.  That is 4.4 us a chunk with one workgroup a CU; a second one gains 14% (the scans of k and v side by side 247 us, one
// alone 143).  Left out for a trial (of 195 us, then): stores 18%, Q X 7, loads 4, P 3, P V 3, loads and stores together
// 28%.  fp32, which has six products for one, 3069 packed tokens of 12 heads of 100 and 72: forward 44 us, gradients 102, states 20
// each; waves whose columns lie past Dv, and zeros past Dk, cost as much as others.
//
// Precision.  The matrix instructions multiply bf16.  Every operand is a sum of bf16 parts: inputs exactly (bf16 one part,
// fp16 two, fp32 three), what is computed (P, the state, weighted V) in as many as keep the error far below one rounding to
// the output's type (two for 16-bit types, three for fp32).  Where the last state is wanted, which is fp32, weighted V has
// three (WEIGHTED; two in its place are 16 matrix and 40 VALU instructions fewer a wave and chunk).
// Products of parts whose size is below the last part's are left out.  Sums are fp32.
#pragma once

#include "grouped_kernels.hpp"

namespace mhc {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kChunk = 64;     // tokens of a chunk

template <typename T> constexpr int kRaw = sizeof(T) == 4 ? 3 : (__is_same(T, __bf16) ? 1 : 2);  // parts of an input
template <typename T> constexpr int kMade = sizeof(T) == 4 ? 3 : 2;                              // of P and the state

struct DecayArgs {
  const void *q, *k, *v;
  void* o;
  const float* log_decay;    // [H]
  const int32_t* offsets;    // ends of the packed sequences; null: N sequences of T rows each, or with N = 0 none
  const float* first;        // X_0 of each sequence, or null
  float* last;               // where X goes, or null
  const int32_t* table;      // [tiles + joins][4]: what find_segment finds, or null
  float* parts;              // [place][H][Dk][Dv]: states that segments leave by themselves; joined: that the next start from
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements; o is contiguous
  int state_row, state_col;                             // of first and last: X's rows and columns
  int part_row, part_col;                               // of parts
  bool joined;  // decay_join_kernel runs
  int64_t R, T;
  int H, N, Dk, Dv, seg, tiles;
  float out_scale, in_scale;  // a, b
  int lag;                    // L
  bool reverse;
};

// Scans that run side by side: the three gradients read the same four tensors, and their workgroups of a segment and
// head are neighbours, so that the second and the third find them in the caches.
constexpr int kMaxJobs = 3;

// A segment adds up the states before it, in sequences of up to this many segments; in others decay_join_kernel does it once
// for all of them.  Summed / joined, us: backward of 32 heads of 8192 tokens as 16 segments 301 / 246, forward of 8 heads of
// 32768 as 64 192 / 139; forward of 32 heads of 2048 as 8 47 / 51.
constexpr int kSummed = 8;
struct DecayJobs {
  DecayArgs job[kMaxJobs];
  int n;
};

// Place among the parts of segment s of a sequence from row lo on.  Only segments with a successor have one; each is `seg` rows,
// so that places differ and stay below (R - 1) / seg, however the rows are split into sequences.
__device__ __forceinline__ int64_t part_place(const DecayArgs& a, int64_t lo, int s) { return (int)lo / a.seg + s; }

// Segment `s` of sequence e, whose rows are lo to hi; e = N: rows past the last sequence; -1: none.
struct Segment {
  int e, s;
  int64_t lo, hi;
};

__device__ __forceinline__ int segments_of(const DecayArgs& a, int64_t lo, int64_t hi) {
  return (int)(((uint32_t)(hi - lo) + (uint32_t)a.seg - 1) / (uint32_t)a.seg);
}

// Tile t: every sequence has a segment at least, so that one without tokens hands its state on.  JOINED: the first segment
// of the t-th sequence of more than kSummed.
template <bool JOINED = false>
__device__ __forceinline__ Segment find_segment(const DecayArgs& a, int t) {
  if (a.table) {
    const int32_t* p = a.table + 4 * ((int64_t)t + (JOINED ? a.tiles : 0));
    return {p[0], p[1], p[2], p[3]};
  }
  if (!a.offsets && a.N) {
    const int per = JOINED ? 1 : max(1, segments_of(a, 0, a.T));
    const int e = t / per;
    return {e < a.N ? e : -1, t - e * per, e * a.T, (e + 1) * a.T};
  }
  const int lane = threadIdx.x & 63;
  int before = 0, end = 0;
  for (int base = 0; base <= a.N; base += 64) {
    const Group g = groups_of(a.offsets, base, a.N, a.R, &end);
    int n = segments_of(a, g.lo, g.hi);
    if (JOINED) n = base + lane < a.N && n > kSummed;
    else if (base + lane < a.N) n = max(n, 1);
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

// The table: every tile's Segment, then the first segments of the sequences of more than kSummed; entries without one have
// e = -1.  One workgroup, a thread a sequence.  For many packed sequences: a tile's own search reads the offsets of all before
// it.
constexpr int kTableThreads = 1024;

__global__ __launch_bounds__(kTableThreads) void decay_table_kernel(DecayArgs a, int32_t* table, int joins) {
  constexpr int W = kTableThreads / 64;
  __shared__ int most[W];
  __shared__ uint64_t sums[W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int end = 0;        // of the sequences so far
  uint64_t done = 0;  // their segments; above 2^32 those of more than kSummed
  auto put = [&](int64_t at, int e, int s, int lo, int hi) {
    int32_t* p = table + 4 * at;
    p[0] = e, p[1] = s, p[2] = lo, p[3] = hi;
  };
  for (int64_t base = 0; base <= a.N; base += kTableThreads) {
    const int64_t e = base + threadIdx.x;
    int hi = e < a.N ? end_of(a.offsets, (int)e, a.R) : (int)a.R;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int v = __shfl_up(hi, off, 64);
      if (lane >= off) hi = max(hi, v);
    }
    if (lane == 63) most[wave] = hi;
    __syncthreads();
    int before = end;
    for (int w = 0; w < W; ++w) {
      if (w < wave) before = max(before, most[w]);
      end = max(end, most[w]);
    }
    hi = max(hi, before);
    const int up = __shfl_up(hi, 1, 64), lo = lane ? up : before;
    int n = segments_of(a, lo, hi);
    const bool joined = e < a.N && n > kSummed;
    n = e < a.N ? max(n, 1) : e == a.N ? n : 0;
    const uint64_t mine = (uint64_t)joined << 32 | (uint32_t)n;
    uint64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t v = __shfl_up(upto, off, 64);
      if (lane >= off) upto += v;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint64_t at = done + upto - mine;
    for (int w = 0; w < W; ++w) {
      if (w < wave) at += sums[w];
      done += sums[w];
    }
    for (int s = 0; s < n; ++s) put((int64_t)(uint32_t)at + s, (int)e, s, lo, hi);
    if (joined && (int)(at >> 32) < joins) put(a.tiles + (int64_t)(at >> 32), (int)e, 0, lo, hi);
    __syncthreads();  // sums and most have been read
  }
  for (int64_t t = (uint32_t)done + threadIdx.x; t < a.tiles; t += kTableThreads) put(t, -1, 0, 0, 0);
  for (int64_t t = (done >> 32) + threadIdx.x; t < joins; t += kTableThreads) put(a.tiles + t, -1, 0, 0, 0);
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

// A plane of 64 rows of bf16, D = 128 or 64 columns, as 16-byte chunks, each row followed by an empty one: every lane's
// accesses lie at constant distances from one address, and of the rows that half a wave (transposed reads: every second
// of 16 rows, two chunks each) or 16 lanes (plain reads: a chunk of 16 rows) read at a time no two meet in a bank.
template <int D> constexpr int kPitch = D / 8 + 1;
template <int D> constexpr int kPlane = kChunk * kPitch<D>;

// Which of 32 tokens the e-th k of lane group g is, and which of 16 keys row m of a product's tile is, so that a lane's
// four results are four neighbouring k of P.
__device__ __forceinline__ int token_of(int g, int e) { return 16 * (e >> 2) + 8 * (g & 1) + 2 * (e & 3) + (g >> 1); }
__device__ __forceinline__ int key_of(int m) { return 8 * ((m >> 2) & 1) + 2 * (m & 3) + (m >> 3); }
// Which of 16 rows of X its tile td holds as row 4 g.  Odd tiles swap neighbouring lane groups, so that the two runs of
// four that a lane reads of a row of Q for two tiles never share a bank with another lane's.
__device__ __forceinline__ int run_of(int td, int g) { return 4 * (td & 1 ? g ^ 1 : g); }

// Transposed: columns c0 .. c0 + 15 of tokens 32 ks .. 32 ks + 31; lane % 16 gets its column's eight, token_of(g, e).
// SWAP: with neighbouring runs of four columns swapped.
template <int D, bool SWAP = false>
__device__ __forceinline__ u32x4 read_columns(const u32x4* plane, int c0, int ks) {
#ifdef __HIP_DEVICE_COMPILE__
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  const char* p = reinterpret_cast<const char*>(plane) + token_of(g, i >> 2) * kPitch<D> * 16 + ((i & 3) ^ (SWAP ? 1 : 0)) * 8;
  p += (32 * ks * kPitch<D> + (c0 >> 3)) * 16;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16 * kPitch<D> * 16));
  return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
  return u32x4{};
#endif
}
// Row r0 + lane % 16 (KEYS: r0 + key_of(lane % 16)), columns 32 ks .. 32 ks + 31 as they lie.
template <int D, bool KEYS = false>
__device__ __forceinline__ u32x4 read_rows(const u32x4* plane, int r0, int ks) {
  const int lane = threadIdx.x & 63, r = KEYS ? key_of(lane & 15) : lane & 15;
  return plane[r * kPitch<D> + (lane >> 4) + r0 * kPitch<D> + 4 * ks];
}
// The same columns in the order in which two tiles of X hold their rows: run_of(0, g) of the first 16, run_of(1, g) of the
// second.
template <int D>
__device__ __forceinline__ u32x4 read_rows_tiled(const u32x4* plane, int r0, int ks) {
  const int lane = threadIdx.x & 63, g = lane >> 4;
  const uint64_t* p = reinterpret_cast<const uint64_t*>(plane) + 2 * (lane & 15) * kPitch<D> + 2 * (r0 * kPitch<D> + 4 * ks);
  const uint64_t lo = p[g], hi = p[4 + (g ^ 1)];
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// A chunk's rows of one operand: global memory -> registers -> planes of parts.  CHUNKS: whole aligned vectors.
template <typename T, int D, int NTH, bool CHUNKS>
struct Feed {
  static constexpr int PER = D / 8, CH = kChunk * PER / NTH;  // eights of a row; eights of a thread
  static constexpr int W = sizeof(T) / 2;                     // 16-byte loads of an eight
  static constexpr int ROWS = NTH / PER;                      // rows that the workgroup brings at a time
  u32x4 r[CH][W];
  int first, step;  // CHUNKS: byte offset of the thread's first eight, and from one to the next

  // Rows of `ld` elements, of which `cols` exist.
  __device__ __forceinline__ Feed(int64_t ld, int cols, bool reverse) {
    const int i = (int)threadIdx.x / PER, c = (int)threadIdx.x % PER * 8;
    first = c < cols ? (int)((reverse ? kChunk - 1 - i : i) * ld + c) * (int)sizeof(T) : kNowhere;
    step = (int)(reverse ? -ROWS * ld : ROWS * ld) * (int)sizeof(T);
  }

  // The n rows from `base` on become the chunk's last n, in their order or (reverse) the other way round, behind zeros.
  // Ranges are checked by the buffer, below its start as offsets past its end: a branch around the loads would have the
  // compiler wait for all of them, and the stores behind them, at once.
  __device__ __forceinline__ void load(const T* base, int64_t ld, int cols, int n, bool reverse) {
    if constexpr (CHUNKS) {
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<T*>(base), 0, n > 0 ? (int)(((n - 1) * ld + cols) * (int64_t)sizeof(T)) : 0, kBufRsrcDword3);
      const int back = reverse ? 0 : (int)((kChunk - n) * ld) * (int)sizeof(T);
#pragma unroll
      for (int q = 0; q < CH; ++q)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          // an eight of fp32 may end behind its first half
          const bool in = w == 0 || (int)threadIdx.x % PER * 8 + 4 * w < cols;
          r[q][w] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? first + q * step - back + 16 * w : kNowhere, 0, 0);
        }
    } else {
#pragma unroll
      for (int q = 0; q < CH; ++q) {
        const int at = q * NTH + threadIdx.x, i = at / PER, c = at % PER * 8;
        const int row = reverse ? kChunk - 1 - i : i - (kChunk - n);
        const bool in = row >= 0 && row < n;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const int left = in ? cols - c - 4 * w : 0;
          r[q][w] = load_chunk<T>(base + (in ? row * ld + c + 4 * w : 0), left, cols >= kElems<T>);
        }
      }
    }
  }

  // Into kRaw<T> planes.
  __device__ __forceinline__ void store(u32x4* planes) const {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int at = q * NTH + threadIdx.x, slot = at / PER * kPitch<D> + at % PER;
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
        for (int i = 0; i < kRaw<T>; ++i) planes[i * kPlane<D> + slot] = p[i];
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

// Keeps the compiler from starting the next step's LDS reads here: their registers would cost others' places.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// LDS in 16-byte chunks: K and V, and for outputs Q and P.  P takes V's place (two barriers more a chunk) where they do not
// fit side by side: fp32, 128 columns and keys.
template <typename T, int DK, int WAVES>
constexpr bool kInPlace = (kRaw<T> * (2 * kPlane<DK> + kPlane<16 * WAVES>) + kMade<T> * kPlane<kChunk>) * 16 > 160 * 1024;
template <typename T, int DK, int WAVES, bool STATE_ONLY>
constexpr int kDecayLds = kRaw<T> * (kPlane<DK> * (STATE_ONLY ? 1 : 2) + kPlane<16 * WAVES>) +
                          (STATE_ONLY || kInPlace<T, DK, WAVES> ? 0 : kMade<T> * kPlane<kChunk>);
// Waves a SIMD: what two workgroups a CU come to, where their LDS fits.
template <typename T, int DK, int WAVES, bool STATE_ONLY>
constexpr int kDecayWaves = WAVES / 4 * (kDecayLds<T, DK, WAVES, STATE_ONLY> * 16 <= 80 * 1024 ? 2 : 1);

template <typename T, int DK, int WAVES, int WEIGHTED, bool CHUNKS, bool STATE_ONLY>
__global__ __launch_bounds__(64 * WAVES, (kDecayWaves<T, DK, WAVES, STATE_ONLY>)) void decay_kernel(DecayJobs jobs) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int RAW = kRaw<T>, MADE = kMade<T>, TD = DK / 16, KS = DK / 32, COLS = 16 * WAVES, NTH = 64 * WAVES;
  constexpr int QK = kPlane<DK>, VP = kPlane<COLS>;
  __shared__ u32x4 lds[kDecayLds<T, DK, WAVES, STATE_ONLY>];
  __shared__ float pow_of[kChunk + 1];  // l^0 .. l^64
  constexpr bool IN_PLACE = !STATE_ONLY && kInPlace<T, DK, WAVES>;
  u32x4 *lk = lds, *lv = lk + RAW * QK, *lq = lv + RAW * VP, *lp = IN_PLACE ? lv : lq + RAW * QK;

  // scans of one (segment, head) side by side on one XCD
  const int run = blockIdx.x / 8, unit = run / jobs.n * 8 + blockIdx.x % 8;
  const DecayArgs a = jobs.job[run % jobs.n];
  if (unit >= a.tiles * a.H) return;
  const int tile = unit / a.H, h = unit - tile * a.H;
  const Segment sg = find_segment(a, tile);
  const int e = __builtin_amdgcn_readfirstlane(sg.e), seg = __builtin_amdgcn_readfirstlane(sg.s);
  if (e < 0) return;
  const int64_t lo = __builtin_amdgcn_readfirstlane((int)sg.lo), hi = __builtin_amdgcn_readfirstlane((int)sg.hi);
  const int len = (int)(hi - lo), begin = seg * a.seg;
  const int stop = begin + min(a.seg, len - begin);  // tokens; begin + a.seg may lie past 2^31
  const int lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = 16 * wave + li;  // of X and V
  if constexpr (STATE_ONLY) {
    if (e == a.N || stop == len) return;
  } else if (e == a.N) {  // rows of no sequence: zeros
    if (!a.o) return;
    T* o = (T*)a.o + ((lo + begin) * a.H + h) * a.Dv;
    for (int i = threadIdx.x; i < (stop - begin) * a.Dv; i += NTH) o[(int64_t)(i / a.Dv) * a.H * a.Dv + i % a.Dv] = from_f32<T>(0.f);
    return;
  }
  const float given = a.log_decay[h], ld = given > 0.f ? 0.f : given;
  if (threadIdx.x <= kChunk) pow_of[threadIdx.x] = power(ld, threadIdx.x).hi;

  // X: rows 16 td + run_of(td, g) + r of the wave's columns
  f32x4 x[TD];
#pragma unroll
  for (int td = 0; td < TD; ++td) x[td] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t size = (int64_t)a.Dk * a.Dv;
  // where x[td][r] is in a state, for a buffer
  auto place_of = [&](int td, int r, int row, int column) {
    const int d = 16 * td + run_of(td, g) + r;
    return d < a.Dk && col < a.Dv ? (d * row + col * column) * 4 : kNowhere;
  };
  if constexpr (!STATE_ONLY) {
    auto add = [&](const float* s, int row, int column, float w) {
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(s), 0, (int)size * 4, kBufRsrcDword3);
      // transposed: a lane's four rows are neighbours, and its columns lines apart from the other lanes'
      if (row == 1 && ((column | a.Dk) & 3) == 0 && ((uintptr_t)s & 15) == 0) {
#pragma unroll
        for (int td = 0; td < TD; ++td)
          x[td] += w * __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, place_of(td, 0, 1, column), 0, 0));
        return;
      }
#pragma unroll
      for (int td = 0; td < TD; ++td) {
        f32x4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          y[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc, place_of(td, r, row, column), 0, 0));
        x[td] += w * y;
      }
    };
    const bool joined = a.joined && seg && segments_of(a, lo, hi) > kSummed;
    if (a.first && !joined) add(a.first + ((int64_t)e * a.H + h) * size, a.state_row, a.state_col, power(ld, begin).hi);
    for (int s = joined ? seg - 1 : 0; s < seg; ++s)
      add(a.parts + (part_place(a, lo, s) * a.H + h) * size, a.part_row, a.part_col, power(ld, (int64_t)(seg - 1 - s) * a.seg).hi);
    // P above the diagonal, where a row's 32 tokens reach past it
    for (int i = threadIdx.x; i < MADE * kPlane<kChunk> && !IN_PLACE; i += NTH) lp[i] = u32x4{0, 0, 0, 0};
  }
  __syncthreads();

  // P's ten tiles in or below the diagonal: wave w makes tiles w, w + WAVES, ...
  constexpr int kTiles = (10 + WAVES - 1) / WAVES;
  int ti[kTiles], tj[kTiles];
#pragma unroll
  for (int n = 0; n < kTiles; ++n) {
    const int t = min(wave + WAVES * n, 9);
    ti[n] = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
    tj[n] = t - ti[n] * (ti[n] + 1) / 2;
  }
  const int key = li - key_of(4 * g);  // query - key of a tile on the diagonal, at r = 0
  float pw[kTiles][4];
#pragma unroll
  for (int n = 0; n < kTiles; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) pw[n][r] = a.out_scale * a.in_scale * pow_of[max(16 * (ti[n] - tj[n]) + key - 2 * r, 0)];
  // A chunk's tokens are its last n.  A result's state weight is l^(li + L) times the tile's; a token's weight on the
  // chunk's end one of its lane group's times one of its place in it, which all lanes share.
  const float out_w = a.out_scale * pow_of[li + a.lag];
  float in_w = a.in_scale * pow_of[10 - a.lag - token_of(g, 0)];
  float place[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) place[i] = uniform(pow_of[22 - token_of(0, i)]);
  const float l16 = uniform(pow_of[16]), l32 = uniform(pow_of[32]);
  // l^64 in fp32 is off by up to 2^-25 of itself, always the same way.  Every 16th chunk puts that right: chunks in
  // between are off by 2^-21 at most where l^64 is so close to 1 that it matters.
  constexpr int kMend = 16;
  const Power p64 = power(ld, kChunk);
  const float whole = uniform(p64.hi), mend = uniform(p64.hi > 0.f ? 1.f + kMend * (p64.lo / p64.hi) : 1.f);
  int since = 0;

  const T* q = (const T*)a.q + h * a.q_head;
  const T* k = (const T*)a.k + h * a.k_head;
  const T* v = (const T*)a.v + h * a.v_head;
  Feed<T, DK, NTH, CHUNKS> fq(a.q_row, a.Dk, a.reverse), fk(a.k_row, a.Dk, a.reverse);
  Feed<T, COLS, NTH, CHUNKS> fv(a.v_row, a.Dv, a.reverse);
  // where the lane's results go: row li of a tile of 16 in a whole chunk, four columns
  const int o_col = 16 * wave + 4 * g, o_row = a.H * a.Dv * (int)sizeof(T);
  const int o_first = o_col < a.Dv ? (a.reverse ? kChunk - 1 - li : li) * o_row + o_col * (int)sizeof(T) : kNowhere;
  const int o_step = a.reverse ? -16 * o_row : 16 * o_row;
  auto first_row = [&](int t, int n) { return a.reverse ? hi - t - n : lo + t; };
  auto load = [&](int t) {
    const int n = max(min(kChunk, stop - t), 0);
    const int64_t row = n ? first_row(t, n) : lo;
    fk.load(k + row * a.k_row, a.k_row, a.Dk, n, a.reverse);
    fv.load(v + row * a.v_row, a.v_row, a.Dv, n, a.reverse);
    if constexpr (!STATE_ONLY) fq.load(q + row * a.q_row, a.q_row, a.Dk, n, a.reverse);
  };
  load(begin);
  for (int t = begin; t < stop; t += kChunk) {
    const int n = min(kChunk, stop - t);
    asm volatile("" : "+v"(in_w));  // its products with `place` are made anew: kept, they would be spilled
    fk.store(lk);
    if constexpr (!IN_PLACE) fv.store(lv);
    if constexpr (!STATE_ONLY) fq.store(lq);
    if constexpr (IN_PLACE) {
      __syncthreads();  // the last chunk's P has been read
      fv.store(lv);
    }
    __syncthreads();
    if constexpr (STATE_ONLY) load(t + kChunk);

    u32x4 vr[2][RAW];  // the wave's columns of V
    auto read_v = [&] {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int p = 0; p < RAW; ++p) vr[ks][p] = read_columns<COLS>(lv + p * VP, 16 * wave, ks);
    };
    [[maybe_unused]] f32x4 o[4];
    if constexpr (!STATE_ONLY) {
      if constexpr (IN_PLACE) read_v();
      auto put = [&](int i, int j, const uint32_t (&parts)[MADE][2]) {
        uint64_t* to = reinterpret_cast<uint64_t*>(lp) + 2 * ((16 * i + li) * kPitch<kChunk> + 4 * (j >> 1) + g) + (j & 1);
#pragma unroll
        for (int p = 0; p < MADE; ++p) to[2 * p * kPlane<kChunk>] = (uint64_t)parts[p][1] << 32 | parts[p][0];
      };
      uint32_t made[kTiles][MADE][2];
      // P: keys are the product's rows, so that a lane gets four neighbouring k of one query
#pragma unroll
      for (int m = 0; m < kTiles; ++m) {
        if ((m + 1) * WAVES > 10 && wave + m * WAVES >= 10) break;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          u32x4 kf[RAW], qf[RAW];
#pragma unroll
          for (int p = 0; p < RAW; ++p) {
            kf[p] = read_rows<DK, true>(lk + p * QK, 16 * tj[m], ks);
            qf[p] = read_rows<DK>(lq + p * QK, 16 * ti[m], ks);
          }
          s = mm_parts<RAW, RAW, RAW - 1>(kf, qf, s);
        }
        float f[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int far = 16 * (ti[m] - tj[m]) + key - 2 * r;
          const float w = pw[m][r] * s[r];
          f[r] = far >= 0 ? w : 0.f;
        }
        split<MADE, 2>(f, made[m]);
        if constexpr (!IN_PLACE) put(ti[m], tj[m], made[m]);
      }
      if constexpr (IN_PLACE) {
        __syncthreads();  // V has been read
#pragma unroll
        for (int m = 0; m < kTiles; ++m)
          if ((m + 1) * WAVES <= 10 || wave + m * WAVES < 10) put(ti[m], tj[m], made[m]);
        // above the diagonal, where a row's 32 tokens reach past it
        if (wave >= WAVES - 2) put(wave == WAVES - 1 ? 0 : 2, wave == WAVES - 1 ? 1 : 3, {});
      }
      // Q X: results are (column, query), a lane's query is li of each tile
#pragma unroll
      for (int it = 0; it < 4; ++it) o[it] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        u32x4 qf[4][RAW], xs[MADE];
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
          for (int p = 0; p < RAW; ++p) qf[it][p] = read_rows_tiled<DK>(lq + p * QK, 16 * it, ks);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = x[2 * ks + i / 4][i % 4];
        split8<MADE>(f, xs);
#pragma unroll
        for (int i = MADE - 1; i >= 0; --i)
#pragma unroll
          for (int j = RAW - 1; j >= 0; --j)
#pragma unroll
            for (int it = 0; it < 4; ++it)
              if (i + j < MADE) o[it] = mm(xs[i], qf[it][j], o[it]);
        fence();
      }
      float w = out_w;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        if (__builtin_expect(n < kChunk, false)) w = a.out_scale * pow_of[max(16 * it + li + a.lag - (kChunk - n), 0)];
        o[it] *= w;
        w *= l16;
      }
    }

    // X' = l^n X + K^T (weighted V)
    if constexpr (!IN_PLACE) read_v();
    float by = whole;
    if (__builtin_expect(n < kChunk, false)) by = power(ld, n).hi;
    if (++since == kMend) {  // what rounding l^64 has cost since the last time
      since = 0;
      by *= mend;
    }
#pragma unroll
    for (int td = 0; td < TD; ++td) x[td] *= by;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] = 0.f;
#pragma unroll
        for (int p = RAW - 1; p >= 0; --p) f[i] += i % 2 ? high2(vr[ks][p][i / 2]) : low2(vr[ks][p][i / 2]);
      }
      const float w = ks ? in_w : in_w * l32;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= w * place[i];
      u32x4 vs[WEIGHTED];
      split8<WEIGHTED>(f, vs);
#pragma unroll
      for (int t4 = 0; t4 < TD; t4 += 4) {
        u32x4 kf[4][RAW];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int p = 0; p < RAW; ++p)
            kf[m][p] = m & 1 ? read_columns<DK, true>(lk + p * QK, 16 * (t4 + m), ks) : read_columns<DK>(lk + p * QK, 16 * (t4 + m), ks);
#pragma unroll
        for (int i = RAW - 1; i >= 0; --i)
#pragma unroll
          for (int j = WEIGHTED - 1; j >= 0; --j)
#pragma unroll
            for (int m = 0; m < 4; ++m)
              if (i + j < WEIGHTED) x[t4 + m] = mm(kf[m][i], vs[j], x[t4 + m]);
        fence();
      }
    }
    if constexpr (!STATE_ONLY) {
      fence();  // the next chunk's registers are not there before
      load(t + kChunk);
    }
    __syncthreads();

    if constexpr (!STATE_ONLY) {
      // P V.  An infinity or a NaN among V has reached every row of its column of X (then and ever after), and would
      // through the zeros above the diagonal reach earlier tokens: such a wave takes its tokens one by one.
      if (__builtin_expect(!__any(x[0][0] * 0.f != 0.f), true)) {
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          u32x4 pf[4][MADE];
#pragma unroll
          for (int it = 2 * ks; it < 4; ++it)
#pragma unroll
            for (int p = 0; p < MADE; ++p) pf[it][p] = read_rows<kChunk>(lp + p * kPlane<kChunk>, 16 * it, ks);
#pragma unroll
          for (int i = RAW - 1; i >= 0; --i)
#pragma unroll
            for (int j = MADE - 1; j >= 0; --j)
#pragma unroll
              for (int it = 2 * ks; it < 4; ++it)
                if (i + j < MADE) o[it] = mm(vr[ks][i], pf[it][j], o[it]);
        }
      } else {
#pragma unroll 1
        for (int j = 0; j < kChunk; ++j) {
          // token_of(gj, ej) = j & 31
          const int gj = ((j >> 3) & 1) | (j & 1) << 1, ej = ((j >> 4) & 1) * 4 + ((j >> 1) & 3);
          float pj[4], vj[4];
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            pj[it] = 0.f;
            for (int p = 0; p < MADE; ++p)
              pj[it] += to_f32(reinterpret_cast<const __bf16*>(lp + p * kPlane<kChunk> + (16 * it + li) * kPitch<kChunk> + 4 * (j >> 5) + gj)[ej]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {  // column 4 g + r is lane 16 gj + 4 g + r's
            vj[r] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
              for (int p = 0; p < RAW; ++p)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const uint32_t w = __shfl(vr[ks][p][i], 16 * gj + 4 * g + r, 64);
                  if (ks == j >> 5 && i == ej >> 1) vj[r] += ej & 1 ? high2(w) : low2(w);
                }
          }
#pragma unroll
          for (int it = 0; it < 4; ++it)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (j <= 16 * it + li) o[it][r] += pj[it] * vj[r];
        }
      }
      T* out = (T*)a.o + (first_row(t, n) * a.H + h) * a.Dv;
      [[maybe_unused]] const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          out, 0, a.o ? (n - 1) * o_row + a.Dv * (int)sizeof(T) : 0, kBufRsrcDword3);
      const int back = a.reverse ? 0 : (kChunk - n) * o_row;
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const f32x4 y = o[it];
        if constexpr (CHUNKS) {
          const int off = o_first + it * o_step - back;
          if constexpr (sizeof(T) == 4) {
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, y), rsrc, off, 0, 0);
          } else {
            const T h4[4] = {from_f32<T>(y[0]), from_f32<T>(y[1]), from_f32<T>(y[2]), from_f32<T>(y[3])};
            uint32_t w[2];
            __builtin_memcpy(w, h4, 8);
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{w[0], w[1]}, rsrc, off, 0, 0);
          }
        } else {
          const int at = a.reverse ? kChunk - 1 - 16 * it - li : 16 * it + li - (kChunk - n);
          if (at >= 0 && at < n && a.o) store4(out + (int64_t)at * a.H * a.Dv + o_col, y, a.Dv - o_col, false);
        }
      }
    }
  }

  float* to = nullptr;
  int row = a.Dv, column = 1;
  if constexpr (STATE_ONLY) {
    to = a.parts + (part_place(a, lo, seg) * a.H + h) * size;
  } else if (a.last && stop == len) {
    to = a.last + ((int64_t)e * a.H + h) * size;
    row = a.state_row;
    column = a.state_col;
  }
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(to, 0, to ? (int)size * 4 : 0, kBufRsrcDword3);
#pragma unroll
  for (int td = 0; td < TD; ++td)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[td][r]), rsrc, place_of(td, r, row, column), 0, 0);
#endif
}

// From the states that a sequence's segments leave by themselves to those that the next ones start from, in place:
//   X_0 = first,  X_(s+1) = l^seg X_s + part_s
// A workgroup has a sequence of more than kSummed segments, a head and every `blocks`-th kJoin values of the state; the next
// segments' loads are in flight.
constexpr int kJoin = 4 * kThreads;

__global__ __launch_bounds__(kThreads) void decay_join_kernel(DecayArgs a, int blocks) {
  const int unit = blockIdx.x / blocks, nth = unit / a.H, h = unit - nth * a.H;
  const Segment sg = find_segment<true>(a, nth);
  if (sg.e < 0) return;
  const int segments = segments_of(a, sg.lo, sg.hi), size = a.Dk * a.Dv;
  const float given = a.log_decay[h];
  const Power l = power(given > 0.f ? 0.f : given, a.seg);
  const int64_t step = (int64_t)a.H * size;  // from a segment's state to the next one's
  float* part = a.parts + (part_place(a, sg.lo, 0) * a.H + h) * size;
  const float* first = a.first ? a.first + ((int64_t)sg.e * a.H + h) * size : nullptr;
  constexpr int V = kJoin / kThreads, AHEAD = 4;
  for (int block = blockIdx.x % blocks; block * kJoin < size; block += blocks) {
    int at[V];
    float x[V], p[AHEAD][V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      at[i] = block * kJoin + i * kThreads + (int)threadIdx.x;
      // parts are [Dk][Dv]; first has strides
      x[i] = first && at[i] < size ? first[at[i] / a.Dv * a.state_row + at[i] % a.Dv * a.state_col] : 0.f;
    }
    auto load = [&](int s, float (&to)[V]) {
#pragma unroll
      for (int i = 0; i < V; ++i) to[i] = s + 1 < segments && at[i] < size ? part[s * step + at[i]] : 0.f;
    };
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) load(n, p[n]);
    for (int s = 0; s + 1 < segments; s += AHEAD) {
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[i] = __builtin_fmaf(x[i], l.hi, __builtin_fmaf(x[i], l.lo, p[n][i]));
          if (s + n + 1 < segments && at[i] < size) part[(s + n) * step + at[i]] = x[i];
        }
        load(s + n + AHEAD, p[n]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// One token a sequence: X' = l X + k^T v, o = c q X'.  Bound by the states, read and written once: 128 rows of 32 heads of
// 128 x 128 102 us from one pool to another (5.3 TB/s), one row 4.7.  Streaming accesses: that case takes 110 without them, and
// in place, the same states again and again, 16 / 48 / 128 / 256 rows 10.2 / 33.0 / 94.5 / 189 us with and 10.8 / 34.3 / 84.2 / 210
// without; a model's other layers come between.
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
      if (d < a.Dk && col < a.Dv) s = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
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
      if (d < a.Dk && col < a.Dv) __builtin_nontemporal_store(f32x4{x[i][0], x[i][1], x[i][2], x[i][3]}, reinterpret_cast<f32x4*>(p));
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if (d < a.Dk && col + w < a.Dv) p[w] = x[i][w];
    }
  }
}

}  // namespace mhc
