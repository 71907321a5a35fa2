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
  int E, tiles_i, tiles_j;
  bool vec;
};

// Rows of one expert, clamped to [0, R) whatever the offsets hold.
struct Group {
  int64_t lo, hi;
};

__device__ __forceinline__ Group group_of(const int32_t* offsets, int e, int E, int64_t R) {
  int64_t lo = e > 0 ? offsets[e - 1] : 0, hi = e < E ? offsets[e] : R;
  lo = lo < 0 ? 0 : (lo > R ? R : lo);
  hi = hi < lo ? lo : (hi > R ? R : hi);
  return {lo, hi};
}

struct RowTile {
  int e;           // the expert; E for the rows past the last offset, -1 past the last tile
  int64_t lo, hi;  // the tile's rows
};

// Row tile t when each expert's rows are cut into tiles of BM: a wave looks at 64 experts at a time.
template <int BM>
__device__ __forceinline__ RowTile find_tile(const int32_t* offsets, int E, int64_t R, int t) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int base = 0; base <= E; base += 64) {
    const int e = base + lane;
    Group g{0, 0};
    if (e <= E) g = group_of(offsets, e, E, R);
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

// A 16-byte chunk at p of which `n` values (the rest zero) may be read.
template <typename T, bool VEC>
__device__ __forceinline__ u32x4 load_chunk(const T* p, int64_t n) {
  u32x4 v = {0, 0, 0, 0};
  if (n >= kElems<T>) {
    if constexpr (VEC) v = *reinterpret_cast<const u32x4*>(p);
    else v = load16_any(p, false);
  } else if (n > 0) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) v[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i % 2));
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) v[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
    // 8-bit rows are whole chunks
  }
  return v;
}

// Slot of 16-byte chunk c of k-row r (KR).
template <typename T>
__device__ __forceinline__ int kr_slot(int r, int c) {
  if constexpr (sizeof(T) == 2) return c ^ (2 * ((r & 3) | ((r >> 1) & 4)));
  else return c ^ (4 * ((r >> 2) & 3));
}

// Global -> registers -> LDS for one slab of one operand (NTH threads).
template <typename T, bool KR, int BM, int NTH, bool VEC>
struct Stage {
  static constexpr int CH = BM * 8 / NTH;          // chunks per thread
  static constexpr int PER = BM / kElems<T>;       // KR: chunks per k-row
  u32x4 r[CH];

  // rows: KC valid rows of the tile; KR valid columns.  k0: the slab's first k, klim: the end of k.
  __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t rows, int64_t k0, int64_t klim) {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int i = q * NTH + threadIdx.x;
      if constexpr (KR) {
        const int row = i / PER, c = (i % PER) * kElems<T>;
        r[q] = load_chunk<T, VEC>(base + (k0 + row) * ld + c, k0 + row < klim ? rows - c : 0);
      } else {
        const int row = i / 8, c = (i % 8) * kElems<T>;
        r[q] = load_chunk<T, VEC>(base + row * ld + k0 + c, row < rows ? klim - k0 - c : 0);
      }
    }
  }
  __device__ __forceinline__ void store(u32x4* lds) const {
#pragma unroll
    for (int q = 0; q < CH; ++q) {
      const int i = q * NTH + threadIdx.x;
      if constexpr (KR) {
        const int row = i / PER;
        lds[row * PER + kr_slot<T>(row, i % PER)] = r[q];
      } else {
        const int row = i / 8;
        lds[row * 8 + ((i % 8) ^ (row & 7))] = r[q];
      }
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
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (r0 * PER + kr_slot<T>(r0, c)) * 16 + (i & 1) * 8));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + (r1 * PER + kr_slot<T>(r1, c)) * 16 + (i & 1) * 8));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    constexpr int PER = BM / 4;
    const uint32_t* p = reinterpret_cast<const uint32_t*>(lds);
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 16 * h + 4 * g + j, c = row + i;
      v[j] = p[(r * PER + kr_slot<T>(r, c >> 2)) * 4 + (c & 3)];
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

// The general kernel: any size and alignment, operands staged through registers.  256 threads, four
// waves of a quarter of the tile each.
template <typename T, typename TO, bool A_KR, bool B_KR, int BM, int BN, Role ROLE, bool VEC>
__global__ __launch_bounds__(256) void grouped_kernel(GroupedArgs a) {
  constexpr int NTH = 256, FI = BM / 32, FJ = BN / 32;
  __shared__ u32x4 lds[(BM + BN) * 8];
  u32x4 *la = lds, *lb = lds + BM * 8;
  const T *A = (const T*)a.A, *B = (const T*)a.B;
  TO* out = (TO*)a.out;
  int64_t rows, k0 = 0, klim, i0 = 0;  // the tile's rows, the range of k, the first row
  int64_t j0;
  int e;
  if constexpr (ROLE == Role::kRows) {
    const int ti = blockIdx.x / a.tiles_j;
    j0 = (int64_t)(blockIdx.x % a.tiles_j) * BN;
    const RowTile t = find_tile<BM>(a.offsets, a.E, a.R, ti);
    if (t.e < 0) return;
    e = t.e;
    rows = t.hi - t.lo;
    klim = t.e < a.E ? a.K : 0;
    i0 = t.lo;
    A += t.lo * a.lda;
    B += (int64_t)(e < a.E ? e : 0) * a.b_expert;
  } else {
    const int per = a.tiles_i * a.tiles_j;
    e = blockIdx.x / per;
    const int t = blockIdx.x % per;
    i0 = (int64_t)(t / a.tiles_j) * BM;
    j0 = (int64_t)(t % a.tiles_j) * BN;
    const Group g = group_of(a.offsets, e, a.E, a.R);
    rows = a.I - i0 < BM ? a.I - i0 : BM;
    k0 = g.lo;
    klim = g.hi;
    A += i0;
    out += (int64_t)e * a.o_expert;
  }
  const int64_t cols = a.J - j0 < BN ? a.J - j0 : BN;
  B += B_KR ? j0 : j0 * a.ldb;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = (wave >> 1) * (BM / 2), wj = (wave & 1) * (BN / 2);
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int i = 0; i < FI; ++i)
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  Stage<T, A_KR, BM, NTH, VEC> sa;
  Stage<T, B_KR, BN, NTH, VEC> sb;
  for (; k0 < klim; k0 += kSlab<T>) {
    sa.load(A, a.lda, rows, k0, klim);
    sb.load(B, a.ldb, cols, k0, klim);
    __syncthreads();
    sa.store(la);
    sb.store(lb);
    __syncthreads();
    if constexpr (__is_same(T, Mx)) {
      uint32_t s_a[FI], s_b[FJ];
      const bool block = k0 + 32 * (lane >> 4) < klim;  // a scale row's filling is not read
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const int r = wi + 16 * i + (lane & 15);
        s_a[i] = block && r < rows ? a.sa[(i0 + r) * a.ns + k0 / 32 + (lane >> 4)] : 0;
      }
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        const int r = wj + 16 * j + (lane & 15);
        s_b[j] = block && r < cols ? a.sb[((int64_t)e * a.J + j0 + r) * a.ns + k0 / 32 + (lane >> 4)] : 0;
      }
      u32x4 fb[FJ][2];
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) fb[j][h] = load_frag<T, false, BN>(lb, wj + 16 * j, h);
#pragma unroll
      for (int i = 0; i < FI; ++i) {
        const u32x4 a0 = load_frag<T, false, BM>(la, wi + 16 * i, 0), a1 = load_frag<T, false, BM>(la, wi + 16 * i, 1);
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = mma_mx(fb[j][0], fb[j][1], a0, a1, s_b[j], s_a[i], acc[i][j]);
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
    }
  }
  const bool vec = a.ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(TO) - 1)) == 0;
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int r = wi + 16 * i + (lane & 15);
    if (r >= rows) continue;
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int c = wj + 16 * j + 4 * (lane >> 4);
      store4(out + (i0 + r) * a.ldo + j0 + c, acc[i][j], cols - c, vec);
    }
  }
}

}  // namespace mhc
