// Host side of the products grouped by expert, shared by grouped.hip and gated.hip: tiles of a launch, its checks and
// the launches.
#pragma once

#include "grouped_kernels.hpp"

namespace mhc {

// Row tiles (kRows) or output tiles (kWeight) of a launch, at most.
template <Role ROLE, int BM, int BN>
static int64_t set_tiles(GroupedArgs& a) {
  a.tiles_j = (int)((a.J + BN - 1) / BN);
  if (ROLE == Role::kWeight) {
    a.tiles_i = (int)((a.I + BM - 1) / BM);
    return (int64_t)a.E * (((int64_t)a.tiles_i * a.tiles_j + 7) / 8 * 8);  // an eighth of each expert's for each XCD
  }
  const int64_t most = a.R / BM + a.E + 1;
  a.tiles_i = (int)(a.R < most ? a.R : most);
  return (int64_t)a.tiles_i * a.tiles_j;
}

static int check_tiles(const char* who, int64_t tiles, int threads) {
  if (tiles < ((int64_t)1 << 32) / threads - 8) return MHC_OK;
  set_error("%s: %lld tiles are too many for a call", who, (long long)tiles);
  return MHC_ERR_ARG;
}

template <typename T, typename TO, bool A_KR, bool B_KR, int BM, int BN, int WI, int WJ, int ST, Role ROLE, bool GATED = false>
static int launch_direct(GroupedArgs a, const char* who, hipStream_t st) {
  constexpr int NTH = 64 * WI * WJ;
  a.cus = num_cus();
  // the 256-tiles of the last round may go in quarters
  const int64_t tiles = set_tiles<ROLE, BM, GATED ? BN / 2 : BN>(a) + (BM == 256 && ROLE == Role::kRows ? 2 * a.cus + 16 : 0);
  if (int rc = check_tiles(who, tiles, NTH)) return rc;
  // whole runs of eight: one for each XCD
  grouped_direct_kernel<T, TO, A_KR, B_KR, BM, BN, WI, WJ, ST, ROLE, GATED>
      <<<dim3((unsigned)((tiles + 7) / 8 * 8)), NTH, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

template <typename T, typename TO, int FI, int NJ, int WAVES, int U, bool CHUNKS, bool GATED = false>
static int launch_few(GroupedArgs a, const char* who, hipStream_t st) {
  const int64_t tiles = set_tiles<Role::kRows, 16 * FI, GATED ? 8 * NJ : 16 * NJ>(a);
  if (int rc = check_tiles(who, tiles, 64 * WAVES)) return rc;
  grouped_few_kernel<T, TO, FI, NJ, WAVES, U, CHUNKS, GATED><<<dim3((unsigned)tiles), 64 * WAVES, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

template <typename T, bool A_KR, bool B_KR, int BM, int BN, Role ROLE, bool GATED = false>
static int launch_general(GroupedArgs a, const char* who, hipStream_t st) {
  const int64_t tiles = set_tiles<ROLE, BM, GATED ? BN / 2 : BN>(a);
  if (int rc = check_tiles(who, tiles, 256)) return rc;
  grouped_kernel<T, A_KR, B_KR, BM, BN, ROLE, GATED><<<dim3((unsigned)((tiles + 7) / 8 * 8)), 256, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

// Tiles that hold rows, as far as the host can tell: an expert's last row tile is half full.
template <Role ROLE, int BM, int BN>
static int64_t likely_tiles(const GroupedArgs& a) {
  const int64_t j = (a.J + BN - 1) / BN;
  if (ROLE == Role::kWeight) return a.E * ((a.I + BM - 1) / BM) * j;
  return ((a.R + BM - 1) / BM + (a.E < a.R ? a.E : a.R) / 2) * j;
}

static int check_grouped(const char* who, int64_t R, int64_t K, int64_t N, int64_t E) {
  if (R < 0 || K < 0 || N < 0 || E < 0) {
    set_error("%s: negative size (R=%lld K=%lld N=%lld E=%lld)", who, (long long)R, (long long)K, (long long)N,
              (long long)E);
    return MHC_ERR_ARG;
  }
  // A row's byte offsets inside a tile are 32-bit, as are tile counts; offsets are int32, and the weight
  // gradient counts up to two slabs past the last row.
  if (R > kMaxRows || K > kMaxWidth || N > kMaxWidth || E > kMaxExperts) {
    set_error("%s: R=%lld K=%lld N=%lld E=%lld exceeds %lld rows, widths of %lld or %lld experts", who, (long long)R,
              (long long)K, (long long)N, (long long)E, (long long)kMaxRows, (long long)kMaxWidth, (long long)kMaxExperts);
    return MHC_ERR_ARG;
  }
  return MHC_OK;
}

static int null_pointer(const char* who) {
  set_error("%s: null pointer", who);
  return MHC_ERR_ARG;
}

// The gradients of grouped.hip without its entries' checks; no offsets: one expert with all rows.
int grouped_input_gradient(const char* who, const void* dy, const void* weight, int dtype, const int32_t* offsets, void* dx,
                           int64_t R, int64_t K, int64_t N, int64_t E, hipStream_t st);
int grouped_weight_gradient(const char* who, const void* dy, const void* x, int dtype, const int32_t* offsets, void* dw,
                            int64_t R, int64_t K, int64_t N, int64_t E, hipStream_t st);

}  // namespace mhc
