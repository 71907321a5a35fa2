// Kernels of the products grouped by expert (grouped.hip).
//
// A workgroup makes a BM x BN tile of out[i, j] = sum_k A(i, k) B(j, k) of one expert.  An operand is
// stored either with k contiguous ("KC": a row per i) or with k as the row index ("KR": a row per k),
// and a slab of 128 bytes of k per row (64 values of 16 bits, 32 of 32, 128 of 8) passes through LDS:
//   KC: [BM rows][8 chunks of 16 bytes], chunk c of row r at slot c ^ (r & 7);
//   KR: [slab rows][BM columns], 16-byte chunks swapped by row so that a transposed read of 16 columns
//       from four rows touches every bank once.
// The matrix instructions take B as their first operand, so a lane's four results are neighbours in j
// and one store.
#pragma once

#include "common.hpp"

namespace mhc {

struct Mx { uint8_t v; };  // e4m3 values with a power-of-two scale for every 32 of k

template <typename T> constexpr int kElems = 16 / (int)sizeof(T);  // values per 16-byte chunk
template <typename T> constexpr int kSlab = 128 / (int)sizeof(T);  // values of k per slab

constexpr int64_t kMaxRows = ((int64_t)1 << 31) - 4096;
constexpr int64_t kMaxWidth = (int64_t)1 << 20;
constexpr int64_t kMaxExperts = 4096;

enum class Role { kRows, kWeight };

struct GroupedArgs {
  const void *A, *B;
  void* out;
  const int32_t* offsets;
  const uint8_t *sa, *sb;  // Mx: scale rows of ns bytes
  int64_t ns;
  int64_t R, I, J, K;      // rows in all; the product's sizes (kRows: I = R, kWeight: K = R)
  int64_t lda, ldb, ldo, b_expert, o_expert;
  int E, tiles_i, tiles_j, cus;
};

// Rows of one expert.  Whatever the offsets hold, they count clamped to [0, R] and as their running maximum, so that
// the experts' rows never overlap, leave none out and fit the launch's tiles.
struct Group {
  int64_t lo, hi;
};

// Of expert e < E; the whole wave calls.
__device__ __forceinline__ Group group_of(const int32_t* offsets, int e, int64_t R) {
  int lo = 0;
  for (int i = threadIdx.x & 63; i < e; i += 64) lo = max(lo, offsets[i]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) lo = max(lo, __shfl_xor(lo, off, 64));
  lo = min(lo, (int)R);
  return {lo, max(lo, min(offsets[e], (int)R))};
}

// Of experts base to base + 63, a lane each; expert E has the rows past the last offset.  `end` is the last lane's
// end, and before the call that of expert base - 1.
__device__ __forceinline__ Group groups_of(const int32_t* offsets, int base, int E, int64_t R, int* end) {
  const int lane = threadIdx.x & 63, e = base + lane;
  int hi = max(e < E ? min(offsets[e], (int)R) : (int)R, *end);
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(hi, off, 64);
    if (lane >= off) hi = max(hi, v);
  }
  const int before = __shfl_up(hi, 1, 64);
  const Group g{lane ? before : *end, hi};
  *end = __shfl(hi, 63, 64);
  return g;
}

struct RowTile {
  int e;           // the expert; E for the rows past the last offset, -1 past the last tile
  int64_t lo, hi;  // the tile's rows
};

// Row tile t when each expert's rows are cut into tiles of BM: a wave looks at 64 experts at a time.
template <int BM>
__device__ __forceinline__ RowTile find_tile(const int32_t* offsets, int E, int64_t R, int t) {
  const int lane = threadIdx.x & 63;
  int before = 0, end = 0;
  for (int base = 0; base <= E; base += 64) {
    const Group g = groups_of(offsets, base, E, R, &end);
    const int n = (int)((g.hi - g.lo + BM - 1) / BM);
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
      const int first = __shfl(upto - n, src, 64);
      const int64_t lo = __shfl((int)g.lo, src, 64) + (int64_t)(t - first) * BM;
      const int64_t hi = __shfl((int)g.hi, src, 64);
      return {base + src, lo, hi < lo + BM ? hi : lo + BM};
    }
    before = __shfl(upto, 63, 64);
  }
  return {-1, 0, 0};
}

// A 16-byte chunk at p, of any alignment, of which `n` values (the rest zero) may be read.  Of a row of 16-bit
// values of at least a chunk (`wide`) the last, partial chunk is read so that it ends with the row and shifted
// into place: a load a value cost the tiles at a row's end more than all the rest.
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* p, int n, bool wide) {
  u32x4 v = {0, 0, 0, 0};
  if (n <= 0) return v;
  const int back = n < kElems<T> ? kElems<T> - n : 0;
  if (sizeof(T) == 4 && back == 0) {
    v = load16_any(p, false);
  } else if (sizeof(T) == 2 && wide) {
    v = load16_any(p - back, false);
    if (back) {
      uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
      const int bits = back * 8 * (int)sizeof(T);
      lo = bits < 64 ? lo >> bits | hi << (64 - bits) : hi >> (bits - 64);
      hi = bits < 64 ? hi >> bits : 0;
      v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
  } else if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i % 2));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < n) v[i] = reinterpret_cast<const uint32_t*>(p)[i];
  }
  return v;
}

// The same in two steps, for rows of at least a chunk.  The load is the same for every lane, so that the compiler
// can keep count of the loads in flight: a row's last, partial chunk is read so that it ends with the row, one with nothing to read from
// `safe`.  chunk_fix, once it has arrived, shifts the former into place and clears the latter.
template <typename T>
__device__ __forceinline__ u32x4 chunk_load(const T* p, int n, const T* safe) {
  const int back = n < kElems<T> ? kElems<T> - n : 0;
  return load16_any(n > 0 ? p - back : safe, false);
}
template <typename T>
__device__ __forceinline__ u32x4 chunk_fix(u32x4 v, int n) {
  const int bits = n >= kElems<T> ? 0 : (kElems<T> - max(n, 1)) * 8 * (int)sizeof(T);
  uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
  const uint64_t carry = bits == 0 ? 0 : hi << (64 - (bits & 63)) % 64;  // bits = 64: lo is replaced below
  lo = bits < 64 ? lo >> (bits & 63) | carry : hi >> (bits & 63);
  hi = bits < 64 ? hi >> (bits & 63) : 0;
  if (n <= 0) lo = hi = 0;
  return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// Slot of 16-byte chunk c of k-row r (KR, PER chunks a row; its own inverse).  16 bits: the eight rows
// that half a wave reads 32 bytes each from (four by the lanes, two by the groups) fall on different banks;
// 32 bits: the four rows of 64 bytes.
template <typename T, int PER>
__device__ __forceinline__ int kr_slot(int r, int c) {
  if constexpr (sizeof(T) == 4) return c ^ (4 * ((r >> 2) & (PER >= 16 ? 3 : 1)));
  else if constexpr (PER >= 16) return c ^ (2 * ((r & 3) | ((r >> 1) & 4)));
  else if constexpr (PER == 8) return c ^ (2 * (((r >> 1) & 1) | ((r >> 2) & 2)));  // two rows share the banks' width
  else return c ^ (2 * ((r >> 3) & 1));  // four do
}

// Global -> registers -> LDS for one slab of one operand (NTH threads).  16-bit k-rows are loaded in two steps
// (8000 x 2001 x 3001 bf16: dx 260 -> 200 us, dw 297 -> 204), the others with what is past an end left out: there
// loads of rows that are none cost more than the branches (the same product's fwd 161 against 183).
template <typename T, bool KR, int BM, int NTH>
struct Stage {
  static constexpr int CH = BM * 8 / NTH;          // chunks per thread
  static constexpr int PER = BM / kElems<T>;       // KR: chunks per k-row
  static constexpr bool TWO = KR && sizeof(T) == 2;
  u32x4 r[CH];

  __device__ __forceinline__ static int row(int q) { return (q * NTH + (int)threadIdx.x) / (KR ? PER : 8); }
  __device__ __forceinline__ static int chunk(int q) { return (q * NTH + (int)threadIdx.x) % (KR ? PER : 8); }
  // Values of chunk q that exist.  rows: KC valid rows of the tile; KR valid columns.
  __device__ __forceinline__ static int left(int q, int rows, int k0, int klim) {
    const int c = chunk(q) * kElems<T>;
    if constexpr (KR) return k0 + row(q) < klim ? rows - c : 0;
    else return row(q) < rows ? klim - k0 - c : 0;
  }

  // wide: a row in memory has a chunk at least.
  __device__ __forceinline__ void load(const T* base, int64_t ld, int rows, int k0, int klim, bool wide) {
    const bool whole = !KR && k0 + kSlab<T> <= klim;  // no row ends inside the slab
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int c = chunk(q) * kElems<T>, n = left(q, rows, k0, klim);
      const T* p = base + (KR ? (int64_t)(k0 + row(q)) * ld + c : row(q) * ld + k0 + c);
      if (TWO && wide) r[q] = chunk_load<T>(p, n, base + (int64_t)k0 * ld + min(0, rows - kElems<T>));
      else if (whole) r[q] = row(q) < rows ? load16_any(p, false) : u32x4{0, 0, 0, 0};
      else r[q] = load_chunk<T>(p, n, wide);
    }
  }
  __device__ __forceinline__ void store(u32x4* lds, int rows, int k0, int klim, bool wide) const {
    const bool ends = TWO && wide && (rows < BM || k0 + kSlab<T> > klim);  // the operand, or k, ends inside the slab
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const u32x4 v = ends ? chunk_fix<T>(r[q], left(q, rows, k0, klim)) : r[q];
      if constexpr (KR) lds[row(q) * PER + kr_slot<T, PER>(row(q), chunk(q))] = v;
      else lds[row(q) * 8 + (chunk(q) ^ (row(q) & 7))] = v;
    }
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// Half a slab (64 bytes of k) of 16 rows or columns from `row` on: half h, 16 bytes per lane; lane group
// g = lane / 16 holds chunk 4 h + g of row `row + lane % 16`.
template <typename T, bool KR, int BM>
__device__ __forceinline__ u32x4 load_frag(const u32x4* lds, int row, int h) {
  const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
  if constexpr (!KR) {
    const int r = row + i;
    return lds[r * 8 + ((4 * h + g) ^ (r & 7))];
  } else if constexpr (sizeof(T) == 2) {
    constexpr int PER = BM / 8;
    const int c = (row >> 3) + ((i & 3) >> 1);  // chunk of the lane's four columns
    const char* p = reinterpret_cast<const char*>(lds);
    const int r0 = 32 * h + 8 * g + (i >> 2), r1 = r0 + 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (r0 * PER + kr_slot<T, PER>(r0, c)) * 16 + (i & 1) * 8));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (r1 * PER + kr_slot<T, PER>(r1, c)) * 16 + (i & 1) * 8));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    constexpr int PER = BM / 4;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(lds);
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 16 * h + 4 * g + j, c = row + i;
      v[j] = p[(r * PER + kr_slot<T, PER>(r, c >> 2)) * 4 + (c & 3)];
    }
    return v;
  }
}

// acc[j] (lane group g: columns 4 g + j; lane % 16: the row) += the half slab's products.
template <typename T>
__device__ __forceinline__ f32x4 mma(u32x4 b, u32x4 a, f32x4 acc) {
  if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b), __builtin_bit_cast(f16x8, a), acc, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b[j]), __uint_as_float(a[j]), acc, 0, 0, 0);
    return acc;
  }
}

// Both halves of an 8-bit slab at once.  The instruction multiplies k-block s (of four) by the scales
// that the lanes of group s hold for their row.  It accumulates in fp32, but first lines the products of a
// lane group's 16 values up with the largest and drops what lies below 2^-13 of it (as the unscaled 8-bit
// instruction does; measured with powers of two): far below the inputs' 4 significant bits, yet no
// fp32 sum, which is why results are offered in 16 bits only.
__device__ __forceinline__ f32x4 mma_mx(u32x4 b0, u32x4 b1, u32x4 a0, u32x4 a1, uint32_t sb, uint32_t sa, f32x4 acc) {
  const i32x8 b = __builtin_bit_cast(i32x8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
  const i32x8 a = __builtin_bit_cast(i32x8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 0, 0, 0, (int)sb, 0, (int)sa);
}

// Stores four neighbouring results of a row; `n` of them exist.
template <typename TO>
__device__ __forceinline__ void store4(TO* p, f32x4 v, int64_t n, bool vec) {
  if (n >= 4 && vec) {
    if constexpr (sizeof(TO) == 4) {
      *reinterpret_cast<f32x4*>(p) = v;
    } else {
      TO t[4] = {from_f32<TO>(v[0]), from_f32<TO>(v[1]), from_f32<TO>(v[2]), from_f32<TO>(v[3])};
      *reinterpret_cast<uint64_t*>(p) = __builtin_bit_cast(uint64_t, *reinterpret_cast<s16x4*>(t));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) p[i] = from_f32<TO>(v[i]);
  }
}

// Tile t of tiles_i x tiles_j: four row tiles side by side through all column tiles, so that neighbours share
// rows and columns.  Each XCD (every eighth workgroup) takes a run of neighbours, for its L2.
__device__ __forceinline__ void band_tile(int t, int tiles_i, int tiles_j, int* ti, int* tj) {
  const int band = t / (4 * tiles_j), high = min(4, tiles_i - 4 * band), in = t - band * 4 * tiles_j;
  *ti = 4 * band + in % high;
  *tj = in / high;
}

// Place `at` of this workgroup's XCD in n places split into eight runs; false past the run's end.
__device__ __forceinline__ bool xcd_place(int n, int at, int* t) {
  const int run = (n + 7) / 8;
  *t = (blockIdx.x % 8) * run + at;
  return at < run && *t < n;
}

// Row tiles in all.
template <int BM>
__device__ __forceinline__ int count_tiles(const int32_t* offsets, int E, int64_t R) {
  int n = 0, end = 0;
  for (int base = 0; base <= E; base += 64) {
    const Group g = groups_of(offsets, base, E, R, &end);
    n += (int)((g.hi - g.lo + BM - 1) / BM);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  return n;
}

// The tile's results, acc[i][j] of wave (wi, wj), to out rows of ldo: through LDS, so that whole rows of 16-byte
// chunks leave the workgroup.  (Four neighbours a lane straight from the registers cost 20 us a tile of 256 x 256
// bf16; 16384 x 4096 outputs at K = 64: 105 -> 41 us.)  Chunk c of row r waits at slot c ^ (r & 15).
template <typename TO, int BM, int BN, int NTH, int CHUNKS, int FI, int FJ>
__device__ __forceinline__ void store_tile(u32x4* lds, const f32x4 (&acc)[FI][FJ], int wi, int wj, TO* out, int64_t ldo,
                                           int rows, int cols) {
  constexpr int CPR = BN / kElems<TO>, MASK = (CPR < 16 ? CPR : 16) - 1;
  constexpr int RP = BM * CPR <= CHUNKS ? BM : BM / 2;  // rows at a time
  constexpr int Q = (RP * CPR + NTH - 1) / NTH;
  static_assert(RP * CPR <= CHUNKS && RP % 16 == 0, "the tile fits in two passes");
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int p = 0; p < BM / RP; ++p) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      if (RP < BM && (wi + 16 * i) / RP != p) continue;
      const int r = wi + 16 * i + (lane & 15) - p * RP;
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        const int c = wj + 16 * j + 4 * (lane >> 4);
        const f32x4 v = acc[i][j];
        if constexpr (sizeof(TO) == 4) {
          lds[r * CPR + ((c / 4) ^ (r & MASK))] = __builtin_bit_cast(u32x4, v);
        } else {
          TO t[4] = {from_f32<TO>(v[0]), from_f32<TO>(v[1]), from_f32<TO>(v[2]), from_f32<TO>(v[3])};
          reinterpret_cast<s16x4*>(lds)[2 * (r * CPR + ((c / 8) ^ (r & MASK))) + (c / 4) % 2] = *reinterpret_cast<s16x4*>(t);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int at = q * NTH + threadIdx.x, r = at / CPR, c = at % CPR;
      const int n = cols - c * kElems<TO>;  // values of the chunk that exist
      if (r >= RP || p * RP + r >= rows || n <= 0) continue;
      const u32x4 v = lds[r * CPR + (c ^ (r & MASK))];
      TO* to = out + (int64_t)(p * RP + r) * ldo + c * kElems<TO>;
      if (n >= kElems<TO>) {
        store16_any(to, v, false);
      } else {
        for (int k = 0; k < n; ++k) {
          if constexpr (sizeof(TO) == 4) reinterpret_cast<uint32_t*>(to)[k] = v[k];
          else reinterpret_cast<uint16_t*>(to)[k] = (uint16_t)(v[k / 2] >> (16 * (k & 1)));
        }
      }
    }
  }
}

// The general kernel: any size and alignment, operands staged through registers (unaligned 16-byte loads,
// single values at a short row's end).  256 threads, four waves of a quarter of the tile each; the next slab's
// loads are in flight while one is multiplied, and two slabs of LDS make one barrier a slab enough.  Bound by
// the slab's loads (any alignment down to the element's): 3069 x 1500 x 1001 fp16 over 9 experts fwd 32, dx 40, dw 39-45 us,
// where 1504 and 1008 take 28, 23 and 22 in the direct kernel.
template <typename T, bool A_KR, bool B_KR, int BM, int BN, Role ROLE>
__global__ __launch_bounds__(256) void grouped_kernel(GroupedArgs a) {
  constexpr int NTH = 256, FI = BM / 32, FJ = BN / 32;
  __shared__ u32x4 lds[2 * (BM + BN) * 8];
  const T *A = (const T*)a.A, *B = (const T*)a.B;
  T* out = (T*)a.out;
  int64_t i0, j0;
  int rows, k0 = 0, klim;  // the tile's rows, the range of k
  int e;
  int t, ti, tj;
  if constexpr (ROLE == Role::kRows) {
    const int tiles = __builtin_amdgcn_readfirstlane(count_tiles<BM>(a.offsets, a.E, a.R));
    if (!xcd_place(tiles * a.tiles_j, blockIdx.x / 8, &t)) return;
    band_tile(t, tiles, a.tiles_j, &ti, &tj);
    const RowTile k = find_tile<BM>(a.offsets, a.E, a.R, ti);
    if (k.e < 0) return;
    e = k.e;
    rows = (int)(k.hi - k.lo);
    klim = k.e < a.E ? (int)a.K : 0;
    i0 = k.lo;
    A += i0 * a.lda;
    B += (int64_t)(e < a.E ? e : 0) * a.b_expert;
  } else {
    const int run = (a.tiles_i * a.tiles_j + 7) / 8, at = blockIdx.x / 8;
    e = at / run;
    if (!xcd_place(a.tiles_i * a.tiles_j, at - e * run, &t)) return;
    band_tile(t, a.tiles_i, a.tiles_j, &ti, &tj);
    i0 = (int64_t)ti * BM;
    const Group g = group_of(a.offsets, e, a.R);
    rows = (int)(a.I - i0 < BM ? a.I - i0 : BM);
    k0 = (int)g.lo;
    klim = (int)g.hi;
    A += i0;
    out += (int64_t)e * a.o_expert;
  }
  j0 = (int64_t)tj * BN;
  const int cols = (int)(a.J - j0 < BN ? a.J - j0 : BN);
  const bool wa = a.lda >= kElems<T>, wb = a.ldb >= kElems<T>;
  B += B_KR ? j0 : j0 * a.ldb;
  const int wave = threadIdx.x >> 6;
  const int wi = (wave >> 1) * (BM / 2), wj = (wave & 1) * (BN / 2);
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Stage<T, A_KR, BM, NTH> sa;
  Stage<T, B_KR, BN, NTH> sb;
  if (k0 < klim) {
    sa.load(A, a.lda, rows, k0, klim, wa);
    sb.load(B, a.ldb, cols, k0, klim, wb);
  }
  for (int s = 0; k0 < klim; k0 += kSlab<T>, s ^= 1) {
    u32x4 *la = lds + s * (BM + BN) * 8, *lb = la + BM * 8;
    sa.store(la, rows, k0, klim, wa);
    sb.store(lb, cols, k0, klim, wb);
    __syncthreads();
    if (k0 + kSlab<T> < klim) {
      sa.load(A, a.lda, rows, k0 + kSlab<T>, klim, wa);
      sb.load(B, a.ldb, cols, k0 + kSlab<T>, klim, wb);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 fb[FJ];
#pragma unroll
      for (int j = 0; j < FJ; ++j) fb[j] = load_frag<T, B_KR, BN>(lb, wj + 16 * j, h);
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const u32x4 fa = load_frag<T, A_KR, BM>(la, wi + 16 * i, h);
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = mma<T>(fb[j], fa, acc[i][j]);
      }
    }
  }
  store_tile<T, BM, BN, NTH, 2 * (BM + BN) * 8>(lds, acc, wi, wj, out + i0 * a.ldo + j0, a.ldo, rows, cols);
}

// ---------------------------------------------------------------------------
// The direct kernel: operands of whole 16-byte chunks go from global memory into LDS without passing
// registers (buffer loads to LDS; a lane's 16 bytes land at the wave's base + 16 * lane, so the swizzle
// is in the addresses that the lanes read from).  ST slabs are in flight; one barrier a slab: behind it,
// the slab waited for is complete and the one multiplied before is free.
//
// Bound, at 256 x 256, by LDS (256 KB a slab move in the time of its products) and by the clock that the matrix
// cores leave: 8192^3 bf16 fwd 1382, dx 1328, dw 1125 TFLOP/s, 8 bits 2372; 4096^3 fp32 144, 142, 141.  A k-row operand is read transposed,
// with twice the read instructions.
//
// Ranges are checked by the buffer: rows past the tile's and, for a k-row operand, k past the group's end
// read as zeros; chunks past a row's end get an offset past any buffer.
// ---------------------------------------------------------------------------
constexpr int kNowhere = 0x7ffffff0;

template <typename T, bool KR, int BM, int NTH>
struct Direct {
  static constexpr int CH = BM * 8 / NTH;    // loads a lane makes per slab
  static constexpr int PER = BM / kElems<T>; // KR: chunks per k-row
  const char* base;
  int64_t ld;  // bytes
  int off[CH];
  int col;     // KC: the lane's first value in a slab
  int span;    // KC: the buffer's bytes; KR: bytes of a row that may be read

  // rows: KC rows of the tile, KR columns.
  __device__ __forceinline__ Direct(const T* p, int64_t ld_, int rows, int klim) {
    base = reinterpret_cast<const char*>(p);
    ld = ld_ * (int64_t)sizeof(T);
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int i = q * NTH + threadIdx.x;
      if constexpr (KR) {
        const int row = i / PER, c = kr_slot<T, PER>(row, i % PER);
        off[q] = c * kElems<T> < rows ? (int)(row * ld) + c * 16 : kNowhere;
      } else {
        const int row = i / 8;
        off[q] = (int)(row * ld) + (((i % 8) ^ (row & 7)) * 16);
      }
    }
    col = (((int)threadIdx.x % 8) ^ (((int)threadIdx.x / 8) & 7)) * kElems<T>;
    span = KR ? (int)(rows * (int64_t)sizeof(T)) : (int)((rows - 1) * ld + klim * (int64_t)sizeof(T));
  }

  // The slab at k0 into lds; past klim it reads zeros.
  __device__ __forceinline__ void load(u32x4* lds, int k0, int klim) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if constexpr (KR) {
      const int left = klim - k0;
      const int n = left <= 0 ? 0 : min(left, kSlab<T>) - 1;
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(base + k0 * ld), 0, left <= 0 ? 0 : (int)(n * ld) + span, kBufRsrcDword3);
#pragma unroll
      for (int q = 0; q < CH; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + q * NTH + wave * 64),
                                                 16, off[q], 0, 0, 0);
    } else {
      // k goes into the scalar offset, which the range check leaves out: rows past the tile's are caught by
      // their own offsets, k past the row's end (the last slab, or those after it) by the lane.
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, span, kBufRsrcDword3);
      const int k = k0 * (int)sizeof(T);
      const bool in = k0 + col < klim;
#pragma unroll
      for (int q = 0; q < CH; ++q)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + q * NTH + wave * 64),
                                                 16, in ? off[q] : kNowhere, k, 0, 0);
    }
  }
};

// Scales of 8-bit operands on their way to LDS: a thread has a row, and takes four slabs' scales (16 bytes) at a
// time, a slab before they are used.  A dword a slab straight to LDS asked L2 for as many lines as the values
// themselves do (8192 x 7168 x 2048 over 16 experts: 236 -> 219 us).  What fills a row past K / 32 is not used.
struct ScaleFeed {
  __amdgpu_buffer_rsrc_t r;
  int off, ns, blocks;  // the row's offset (past any buffer: none); bytes of a row, and how many of them count
  u32x4 quad;

  __device__ __forceinline__ void load(int slab) {
    if (4 * slab + 16 <= ns) {
      quad = __builtin_amdgcn_raw_buffer_load_b128(r, off, 4 * slab, 0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        quad[j] = __builtin_amdgcn_raw_buffer_load_b32(r, 4 * (slab + j) < ns ? off : kNowhere, 4 * (slab + j), 0);
    }
  }
  // The scales of slab n, which follow one another.
  __device__ __forceinline__ uint32_t take(int n) {
    uint32_t v = n & 2 ? (n & 1 ? quad[3] : quad[2]) : (n & 1 ? quad[1] : quad[0]);
    const int left = blocks - 4 * n;
    if (left < 4) v = left <= 0 ? 0 : v & ((1u << (8 * left)) - 1);
    if ((n & 3) == 3) load(n + 1);
    return v;
  }
};

// Waits until at most N of the wave's loads are in flight and its LDS accesses are done, then for the whole workgroup:
// behind it, slabs may be read that were waited for, and those overwritten that were read before.
template <int N>
__device__ __forceinline__ void slab_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// What a workgroup is to do: `rows` x `cols` results of expert e from (i0, j0) on, k from k0 to klim.
struct Task {
  int e;
  int64_t i0, j0;
  int rows, cols, k0, klim;
};

// LDS of a tile in 16-byte chunks: per slab A, B and (8 bits) a dword of scales for each thread.
template <typename T, int BM, int BN, int NTH>
constexpr int kSlabChunks = (BM + BN) * 8 + (__is_same(T, Mx) ? NTH / 4 : 0);

#ifdef __HIP_DEVICE_COMPILE__  // the host's compiler drops instantiations with 16-byte loads to LDS
template <typename T, typename TO, bool A_KR, bool B_KR, int BM, int BN, int WI, int WJ, int ST, Role ROLE>
__device__ __forceinline__ void direct_tile(const GroupedArgs& a, const Task& task, u32x4* lds) {
  constexpr bool MX = __is_same(T, Mx), AHEAD = sizeof(T) == 2 && BM == 256 && BN == 256;
  constexpr int NTH = 64 * WI * WJ, FI = BM / WI / 16, FJ = BN / WJ / 16;
  constexpr int kSlabChunks = mhc::kSlabChunks<T, BM, BN, NTH>;
  static_assert(!MX || BM + BN <= NTH, "a thread has one row's scales");
  const int e = task.e, rows = task.rows, cols = task.cols, klim = task.klim;
  int k0 = task.k0;
  const int64_t i0 = task.i0, j0 = task.j0;
  const bool row_role = ROLE == Role::kRows;
  const T* A = (const T*)a.A + (row_role ? i0 * a.lda : i0);
  const T* B = (const T*)a.B + (row_role ? (int64_t)(e < a.E ? e : 0) * a.b_expert : 0) + (B_KR ? j0 : j0 * a.ldb);
  TO* out = (TO*)a.out + (row_role ? 0 : (int64_t)e * a.o_expert);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = (wave / WJ) * (BM / WI), wj = (wave % WJ) * (BN / WJ);
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  const Direct<T, A_KR, BM, NTH> da(A, a.lda, rows, klim);
  const Direct<T, B_KR, BN, NTH> db(B, a.ldb, cols, klim);
  constexpr int kLoads = da.CH + db.CH;  // per wave and slab
  ScaleFeed feed{};
  if constexpr (MX) {
    static_assert(BM % 64 == 0, "a wave's rows are all A's or all B's");
    const bool of_a = wave * 64 < BM;
    const int row = (int)threadIdx.x - (of_a ? 0 : BM);
    feed.ns = (int)a.ns;
    feed.blocks = klim / 32;
    feed.r = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t*>(of_a ? a.sa + i0 * a.ns : a.sb + ((int64_t)(e < a.E ? e : 0) * a.J + j0) * a.ns), 0,
        (of_a ? rows : cols) * feed.ns, kBufRsrcDword3);
    feed.off = row < (of_a ? rows : cols) ? row * feed.ns : kNowhere;
    feed.load(0);
  }
  auto issue = [&](int s, int k) {
    u32x4* p = lds + s * kSlabChunks;
    if constexpr (MX) reinterpret_cast<uint32_t*>(p + (BM + BN) * 8)[threadIdx.x] = feed.take(k / kSlab<T>);
    da.load(p, k, klim);
    db.load(p + BM * 8, k, klim);
  };
  auto multiply = [&](int s, int k) {
    const u32x4 *la = lds + s * kSlabChunks, *lb = la + BM * 8;
    if constexpr (MX) {
      // The instruction takes its scale from the low byte.
      const uint32_t* sc = reinterpret_cast<const uint32_t*>(la + (BM + BN) * 8) + (lane & 15);
      const int shift = 8 * (lane >> 4);
      u32x4 fb[FJ][2];
      uint32_t s_b[FJ], s_a[FI];
#pragma unroll
      for (int j = 0; j < FJ; ++j) s_b[j] = sc[BM + wj + 16 * j] >> shift;
#pragma unroll
      for (int i = 0; i < FI; ++i) s_a[i] = sc[wi + 16 * i] >> shift;
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        fb[j][0] = load_frag<T, false, BN>(lb, wj + 16 * j, 0);
        fb[j][1] = load_frag<T, false, BN>(lb, wj + 16 * j, 1);
      }
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const u32x4 a0 = load_frag<T, false, BM>(la, wi + 16 * i, 0), a1 = load_frag<T, false, BM>(la, wi + 16 * i, 1);
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = mma_mx(fb[j][0], fb[j][1], a0, a1, s_b[j], s_a[i], acc[i][j]);
      }
      // one row fragment ahead of the matrix instructions that use it, and no more: registers
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * FJ + 4, 0);
#pragma unroll
      for (int n = 0; n < FI; ++n) {
        __builtin_amdgcn_sched_group_barrier(0x008, FJ, 0);
        if (n < FI - 2) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 fb[FJ];
#pragma unroll
        for (int j = 0; j < FJ; ++j) fb[j] = load_frag<T, B_KR, BN>(lb, wj + 16 * j, h);
#pragma unroll
        for (int i = 0; i < FI; ++i) {
          const u32x4 fa = load_frag<T, A_KR, BM>(la, wi + 16 * i, h);
#pragma unroll
          for (int j = 0; j < FJ; ++j) acc[i][j] = mma<T>(fb[j], fa, acc[i][j]);
        }
      }
      if constexpr (FI >= FJ) {
        // One row fragment ahead of the matrix instructions that use it, and the second half's columns
        // spread over the first half's end.
        constexpr int RA = !A_KR ? 1 : (sizeof(T) == 2 ? 2 : 4), RB = !B_KR ? 1 : (sizeof(T) == 2 ? 2 : 4);
        constexpr int MM = FJ * (sizeof(T) == 4 ? 4 : 1);
        __builtin_amdgcn_sched_group_barrier(0x100, FJ * RB + 2 * RA, 0);
#pragma unroll
        for (int n = 0; n < 2 * FI; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, MM, 0);
          if (n >= FI - FJ && n < FI) __builtin_amdgcn_sched_group_barrier(0x100, RB, 0);
          if (n < 2 * FI - 2) __builtin_amdgcn_sched_group_barrier(0x100, RA, 0);
        }
      }
    }
  };

  if constexpr (AHEAD) {
    // Fragments are read half a slab ahead of the matrix instructions that use them.  Between a slab's halves
    // every wave has read all of it and the next one has arrived: one barrier a slab, and the loads of slab
    // n + 2 go out there, a whole slab's time before they are needed.
    if (k0 < klim) {
      u32x4 fa[2][FI], fb[2][FJ];
      constexpr int RA = !A_KR ? 1 : (sizeof(T) == 2 ? 2 : 4), RB = !B_KR ? 1 : (sizeof(T) == 2 ? 2 : 4);
      constexpr int MM = FI * FJ * (sizeof(T) == 4 ? 4 : 1), DS = FI * RA + FJ * RB;
      auto read = [&](int s, int h) {
        const u32x4 *la = lds + s * kSlabChunks, *lb = la + BM * 8;
#pragma unroll
        for (int j = 0; j < FJ; ++j) fb[h][j] = load_frag<T, B_KR, BN>(lb, wj + 16 * j, h);
#pragma unroll
        for (int i = 0; i < FI; ++i) fa[h][i] = load_frag<T, A_KR, BM>(la, wi + 16 * i, h);
      };
      auto mult = [&](int h) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int j = 0; j < FJ; ++j) acc[i][j] = mma<T>(fb[h][j], fa[h][i], acc[i][j]);
      };
      issue(0, k0);
      issue(1, k0 + kSlab<T>);
      slab_ready<kLoads>();
      read(0, 0);
      int s = 0;
      for (; k0 < klim; k0 += kSlab<T>, s ^= 1) {
        read(s, 1);
        mult(0);
#pragma unroll
        for (int n = 0; n < DS; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, MM / DS, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        issue(s, k0 + 2 * kSlab<T>);
        read(s ^ 1, 0);
        mult(1);
#pragma unroll
        for (int n = 0; n < DS; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          if (n < kLoads) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, MM / DS, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands in LDS after the workgroup's end
    }
  } else if (k0 < klim) {
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) issue(s, k0 + s * kSlab<T>);
    int s = 0;
    for (; k0 < klim; k0 += kSlab<T>) {
      slab_ready<(ST - 2) * kLoads>();
      int next = s + ST - 1;
      next = next >= ST ? next - ST : next;
      issue(next, k0 + (ST - 1) * kSlab<T>);
      multiply(s, k0);
      s = s + 1 == ST ? 0 : s + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing lands in LDS after the workgroup's end
  }
  store_tile<TO, BM, BN, NTH, ST * kSlabChunks>(lds, acc, wi, wj, out + i0 * a.ldo + j0, a.ldo, rows, cols);
}
#endif

// Row tile ti of expert rows, column tile tj.
template <int BM, int BN>
__device__ __forceinline__ Task row_task(const GroupedArgs& a, int ti, int tj) {
  const RowTile t = find_tile<BM>(a.offsets, a.E, a.R, ti);
  Task k;
  k.e = __builtin_amdgcn_readfirstlane(t.e);
  k.i0 = __builtin_amdgcn_readfirstlane((int)t.lo);
  k.rows = __builtin_amdgcn_readfirstlane((int)(t.hi - t.lo));
  k.j0 = (int64_t)tj * BN;
  k.cols = (int)(a.J - k.j0 < BN ? a.J - k.j0 : BN);
  k.k0 = 0;
  k.klim = k.e < a.E ? (int)a.K : 0;  // the rows of no expert: zeros
  return k;
}

template <typename T, typename TO, bool A_KR, bool B_KR, int BM, int BN, int WI, int WJ, int ST, Role ROLE>
__global__ __launch_bounds__(64 * WI * WJ, 2) void grouped_direct_kernel(GroupedArgs a) {
#ifdef __HIP_DEVICE_COMPILE__
  __shared__ u32x4 lds[ST * kSlabChunks<T, BM, BN, 64 * WI * WJ>];
  // Tiles of 256 x 256 of rows: what is left after whole rounds of the CUs, if it is half a round at most, goes in
  // quarters, so that the last round does not leave most CUs idle.
  constexpr bool QUARTERS = BM == 256 && ROLE == Role::kRows;
  int t, ti, tj;
  Task k;
  if constexpr (ROLE == Role::kRows) {
    const int tiles = __builtin_amdgcn_readfirstlane(count_tiles<BM>(a.offsets, a.E, a.R));
    const int total = tiles * a.tiles_j, left = total % a.cus;
    const int split = QUARTERS && left <= a.cus / 2 ? left : 0, whole = total - split;
    const int at = blockIdx.x / 8, runs = (whole + 7) / 8;
    int part = -1;
    if (!xcd_place(whole, at, &t)) {
      if (!QUARTERS || at < runs || !xcd_place(4 * split, at - runs, &t)) return;
      part = t % 4;
      t = whole + t / 4;
    }
    band_tile(t, tiles, a.tiles_j, &ti, &tj);
    k = row_task<BM, BN>(a, ti, tj);
    if (k.e < 0) return;
    if constexpr (QUARTERS) {
      if (part >= 0) {
        const int di = part / 2 * 128, dj = part % 2 * 128;
        if (di >= k.rows || dj >= k.cols) return;
        k.i0 += di;
        k.j0 += dj;
        k.rows = min(k.rows - di, 128);
        k.cols = min(k.cols - dj, 128);
        direct_tile<T, TO, A_KR, B_KR, 128, 128, 2, 4, ST, ROLE>(a, k, lds);
        return;
      }
      if (k.rows <= 128) {  // an expert's last rows
        direct_tile<T, TO, A_KR, B_KR, 128, 256, 2, 4, ST, ROLE>(a, k, lds);
        return;
      }
    }
  } else {
    // Every XCD takes an eighth of each expert's tiles: the experts' rows, and so their tiles' times, differ.
    const int run = (a.tiles_i * a.tiles_j + 7) / 8, at = blockIdx.x / 8;
    k.e = at / run;
    if (!xcd_place(a.tiles_i * a.tiles_j, at - k.e * run, &t)) return;
    band_tile(t, a.tiles_i, a.tiles_j, &ti, &tj);
    const Group g = group_of(a.offsets, k.e, a.R);
    k.i0 = (int64_t)ti * BM;
    k.rows = (int)(a.I - k.i0 < BM ? a.I - k.i0 : BM);
    k.j0 = (int64_t)tj * BN;
    k.cols = (int)(a.J - k.j0 < BN ? a.J - k.j0 : BN);
    k.k0 = __builtin_amdgcn_readfirstlane((int)g.lo);
    k.klim = __builtin_amdgcn_readfirstlane((int)g.hi);
  }
  direct_tile<T, TO, A_KR, B_KR, BM, BN, WI, WJ, ST, ROLE>(a, k, lds);
#endif
}

// ---------------------------------------------------------------------------
// Few rows an expert (decoding): out[i, j] for up to 16 FI rows and 16 NJ columns, both operands with k
// contiguous.  What counts is how fast the weights arrive, and nothing is used twice, so fragments come
// from global memory straight into registers: a lane holds 16-byte chunks g and 4 + g of 128 bytes of a
// row (a unit).  The waves of a workgroup take every WAVES-th unit, each with U of them in flight, and
// add up through LDS in wave order.  64 rows over 28 experts of 2048 to 4096 bf16 75 us (6.2 TB/s of weights), 128
// rows over 30 of 4096 to 4096 in 8 bits 100 us (5.1); with streaming loads, whose lines leave between their
// halves, 84 and 111.
// ---------------------------------------------------------------------------
template <typename T, typename TO, int FI, int NJ, int WAVES, int U, bool CHUNKS>
__global__ __launch_bounds__(64 * WAVES) void grouped_few_kernel(GroupedArgs a) {
  constexpr bool MX = __is_same(T, Mx);
  __shared__ f32x4 sum[WAVES][FI * NJ][64];
  const int ti = blockIdx.x / a.tiles_j;
  const int j0 = (int)(blockIdx.x % a.tiles_j) * 16 * NJ;
  const RowTile t = find_tile<16 * FI>(a.offsets, a.E, a.R, ti);
  if (t.e < 0) return;
  const int e = __builtin_amdgcn_readfirstlane(t.e);
  const int64_t i0 = __builtin_amdgcn_readfirstlane((int)t.lo);
  const int rows = __builtin_amdgcn_readfirstlane((int)(t.hi - t.lo));
  const int klim = e < a.E ? (int)a.K : 0;
  const int cols = min((int)a.J - j0, 16 * NJ);
  const int lane = threadIdx.x & 63, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wrow = (int64_t)(e < a.E ? e : 0) * a.J + j0;  // the tile's first weight row
  const int lda = (int)(a.lda * (int64_t)sizeof(T)), ldb = (int)(a.ldb * (int64_t)sizeof(T));
  const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>((const char*)a.A + i0 * lda), 0, (rows - 1) * lda + klim * (int)sizeof(T), kBufRsrcDword3);
  const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>((const char*)a.B + wrow * ldb), 0, (cols - 1) * ldb + klim * (int)sizeof(T), kBufRsrcDword3);
  const int ns = (int)a.ns;
  const __amdgpu_buffer_rsrc_t rsa = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(MX ? a.sa + i0 * a.ns : nullptr), 0, MX ? rows * ns : 0, kBufRsrcDword3);
  const __amdgpu_buffer_rsrc_t rsb = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint8_t*>(MX ? a.sb + wrow * a.ns : nullptr), 0, MX ? cols * ns : 0, kBufRsrcDword3);
  f32x4 acc[FI][NJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Unit {
    u32x4 a[FI][2], b[NJ][2];
  };
  // Whole chunks: ranges as in the direct kernel, rows past the tile's by the buffer, k past the end by the lane.
  // Otherwise the general kernel's loads.
  auto load = [&](Unit& u, int unit) {
    const int k = unit * kSlab<T>;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = k + (4 * h + g) * kElems<T>;
      const bool in = c < klim;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = 16 * j + (lane & 15);
        if constexpr (CHUNKS) u.b[j][h] = __builtin_amdgcn_raw_buffer_load_b128(rb, in ? row * ldb + (4 * h + g) * 16 : kNowhere, unit * 128, 0);
        else u.b[j][h] = load_chunk<T>((const T*)a.B + (wrow + row) * a.ldb + c, row < cols ? klim - c : 0, klim >= kElems<T>);
      }
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int row = 16 * i + (lane & 15);
        if constexpr (CHUNKS) u.a[i][h] = __builtin_amdgcn_raw_buffer_load_b128(ra, in ? row * lda + (4 * h + g) * 16 : kNowhere, unit * 128, 0);
        else u.a[i][h] = load_chunk<T>((const T*)a.A + (i0 + row) * a.lda + c, row < rows ? klim - c : 0, klim >= kElems<T>);
      }
    }
  };
  const int units = (klim + kSlab<T> - 1) / kSlab<T>;
  Unit u[U];
  if constexpr (MX) {
    // A wave takes four units in a row, whose scales are 16 bytes of a row: one load for all of them (a byte
    // a unit and lane: 120 -> 108 us for 128 rows over 32 experts, 4096 to 4096).
    static_assert(U == 2, "units two ahead");
    const int blocks = klim / 32;
    auto scales = [&](__amdgpu_buffer_rsrc_t r, int row, int unit) -> u32x4 {
      u32x4 v;
      if (4 * unit + 16 <= ns) {
        v = __builtin_amdgcn_raw_buffer_load_b128(r, row * ns, 4 * unit, 0);
      } else {
#pragma unroll
        for (int n = 0; n < 4; ++n)
          v[n] = __builtin_amdgcn_raw_buffer_load_b32(r, 4 * (unit + n) < ns ? row * ns : kNowhere, 4 * (unit + n), 0);
      }
      return v;
    };
    auto first_unit = [&](int group) { return 4 * (wave + group * WAVES); };
    const int groups = (units + 4 * WAVES - 1) / (4 * WAVES);  // of this wave; some past the end
    u32x4 sb[NJ], sa[FI], next_b[NJ], next_a[FI];
    auto load_scales = [&](int unit) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) next_b[j] = scales(rsb, 16 * j + (lane & 15), unit);
#pragma unroll
      for (int i = 0; i < FI; ++i) next_a[i] = scales(rsa, 16 * i + (lane & 15), unit);
    };
    load_scales(first_unit(0));
    load(u[0], first_unit(0));
    load(u[1], first_unit(0) + 1);
    for (int n = 0; n < groups; ++n) {
      const int at = first_unit(n);
#pragma unroll
      for (int j = 0; j < NJ; ++j) sb[j] = next_b[j];
#pragma unroll
      for (int i = 0; i < FI; ++i) sa[i] = next_a[i];
      load_scales(first_unit(n + 1));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool block = 4 * (at + q) + g < blocks;  // a scale row's filling is not used
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            acc[i][j] = mma_mx(u[q % 2].b[j][0], u[q % 2].b[j][1], u[q % 2].a[i][0], u[q % 2].a[i][1],
                               block ? sb[j][q] >> (8 * g) : 0, block ? sa[i][q] >> (8 * g) : 0, acc[i][j]);
        load(u[q % 2], q < 2 ? at + q + 2 : first_unit(n + 1) + q - 2);
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < U; ++n) load(u[n], wave + n * WAVES);  // past the end: zeros
    for (int at = wave; at < units; at += U * WAVES) {
#pragma unroll
      for (int n = 0; n < U; ++n) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[i][j] = mma<T>(u[n].b[j][h], u[n].a[i][h], acc[i][j]);
        load(u[n], at + (U + n) * WAVES);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) sum[wave][i * NJ + j][lane] = acc[i][j];
  __syncthreads();
  TO* out = (TO*)a.out;
  const bool vec = a.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(TO) - 1)) == 0;
  for (int f = wave; f < FI * NJ; f += WAVES) {
    f32x4 v = sum[0][f][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += sum[w][f][lane];
    const int r = f / NJ * 16 + (lane & 15), c = f % NJ * 16 + 4 * g;
    if (r < rows) store4(out + (i0 + r) * a.ldo + j0 + c, v, cols - c, vec);
  }
}

}  // namespace mhc
