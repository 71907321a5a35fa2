// Matrix products grouped by expert: rows [offsets[e-1], offsets[e]) of x belong to expert e.
//
//   forward          y[m, n]     = sum_k x[m, k] w[e][n, k]
//   input gradient   dx[m, k]    = sum_n dy[m, n] w[e][n, k]
//   weight gradient  dw[e][n, k] = sum_{m of e} dy[m, n] x[m, k]
//
// The offsets stay on the device.  A launch has as many row tiles as any split of the rows among the
// experts can need, and each workgroup finds its own in the offsets, so nothing waits for the host and a
// captured graph serves every split.  Rows past the last offset get zeros.
#include "grouped_launch.hpp"

namespace mhc {

// Which kernel; times in us, a captured launch each.  One rule for all types, made for 16 and 8 bits: where a figure
// here speaks against it, the rule has not been refined.
//
// Few rows an expert: at 8 each the kernel that takes weights into registers still wins, past 16 it reads the rows
// too often (1 / 8 / 16 / 32 rows an expert, registers against tiles: 32 experts of 2048 to 4096 bf16
// 100 / 111 / 131 / 211 against 133; 8 bits 56 / 64 / 75 / 123 against 74 to 78).  In 8 bits its four waves need four
// units of four slabs: K = 1024 over 64 experts 38 against 32 us.  fp32 (1 / 4 / 8 / 16 rows): 173 / 216 / 236 / 305 against
// 64-tiles' 251 / 288 / 291 / 292 and 32-tiles' 159 / 228 / 227 / 231.  Rows of any alignment, against the general
// kernel: 1500 to 1001 fp16 18.5 / 21.0 / 23.0 / 27.3 and 21.7 / 22.5 / 22.6 / 23.0, 2047 to 4095 fp32
// 204 / 273 / 300 / 397 and 266 / 306 / 311 / 320, but bf16 of that odd width 173 / 231 / 268 / 401 and 99 / 113 / 120 / 139.
//
// Tiles: the largest of 256, 128, 64 and 32 that gives every CU one, 256 only where experts have as many rows (bf16
// fwd / dx / dw, 256 against 128: 4096 rows of 4096 to 4096 over 8 experts 118 / 126 / 169 and 154 / 167 / 197 us, 8192 of
// 1024 to 1024 over 8, half a tile a CU, 29 / 37 / 38 and 25 / 22 / 23, 4096 of 2048 to 1024 over 32 47 / 32 / 50 and
// 27 / 28 / 45; fp32 dw of 4096 by 1024 over 4, 256 tiles, 452 and 270).
//   128 against 64, 1024 to 1024 over 8 (fwd / dx), with 352, 264 and 208 likely 128-tiles: bf16 20 / 22 and 28 / 37,
//   18 / 21 and 20 / 27, 16 / 21 and 18 / 26 (where the rule takes 64); fp32 130 / 130 and 113 / 116, 129 / 129 and
//   79 / 79, 73 / 74 and 62 / 63.
//   64 against 32, 1024 to 1024 over 4 with 288 and 160 likely 64-tiles: bf16 10 / 12 and 15 / 20, 8.6 / 10.5 each;
//   fp32 40 / 40 and 34 / 34, 25 / 25 and 21 / 22.  512 from 2048 with 48: bf16 16.0 and 13.2, fp32 45 and 21.
//   8 bits, 128 against 64: 288 tiles 22.5 and 32.2, 224 18.3 and 25.4 (where the rule takes 64), 72 10.9 and 7.9.
//
// The general kernel takes what is not whole aligned 16-byte chunks, in 128-tiles from two a CU on (against 64, 1001 to
// 1003 over 4 with 520, 392 and 272 likely 128-tiles: bf16 33 / 39 and 50 / 52, 30 / 37 and 41 / 46,
// 28 / 36 and 29 / 31; fp32 147 / 155 and 165 / 173, 145 / 153 and 140 / 150, 142 / 152 and 88 / 94).
template <typename T, typename TO, bool A_KR, bool B_KR, Role ROLE>
static int launch_grouped(GroupedArgs a, const char* who, hipStream_t st) {
  constexpr bool MX = __is_same(T, Mx);
  const bool chunks = a.lda % kElems<T> == 0 && a.ldb % kElems<T> == 0 && aligned16(a.A) && aligned16(a.B);
  const int cus = num_cus();
  if (chunks) {
    if constexpr (!A_KR && !B_KR)
      if (a.R <= 8 * (int64_t)a.E && (!MX || a.K >= 2048)) return launch_few<T, TO, 1, 2, 4, 2, true>(a, who, st);
    if (likely_tiles<ROLE, 256, 256>(a) >= cus && (ROLE == Role::kWeight || a.R >= 256 * (int64_t)a.E))
      return launch_direct<T, TO, A_KR, B_KR, 256, 256, 2, 4, 2, ROLE>(a, who, st);
    if (likely_tiles<ROLE, 128, 128>(a) >= cus) return launch_direct<T, TO, A_KR, B_KR, 128, 128, 2, 2, 2, ROLE>(a, who, st);
    if (MX || likely_tiles<ROLE, 64, 64>(a) >= cus) return launch_direct<T, TO, A_KR, B_KR, 64, 64, 2, 2, 4, ROLE>(a, who, st);
    if constexpr (!MX) return launch_direct<T, TO, A_KR, B_KR, 32, 32, 2, 2, 4, ROLE>(a, who, st);
  }
  if constexpr (!MX) {
    if constexpr (!A_KR && !B_KR)
      if (a.R <= 8 * (int64_t)a.E) return launch_few<T, TO, 1, 2, 4, 2, false>(a, who, st);
    if (likely_tiles<ROLE, 128, 128>(a) >= 2 * cus) return launch_general<T, A_KR, B_KR, 128, 128, ROLE>(a, who, st);
    return launch_general<T, A_KR, B_KR, 64, 64, ROLE>(a, who, st);
  }
  return MHC_OK;  // 8-bit operands are whole chunks (checked at the entry)
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_grouped_matmul_forward(const void* x, const void* weight, int dtype, const int32_t* offsets, void* y,
                                          int64_t R, int64_t K, int64_t N, int64_t E, mhc_stream_t stream) {
  const char* who = "grouped_matmul_forward";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (R * N == 0) return MHC_OK;
  if (!y || (E && !offsets) || (K && (!x || (E && !weight)))) return null_pointer(who);
  GroupedArgs a{};
  a.A = x; a.B = weight; a.out = y; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = R; a.J = N; a.K = K;
  a.lda = K; a.ldb = K; a.ldo = N; a.b_expert = N * K;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    return launch_grouped<T, T, false, false, Role::kRows>(a, who, (hipStream_t)stream);
  });
}

namespace mhc {

int grouped_input_gradient(const char* who, const void* dy, const void* weight, int dtype, const int32_t* offsets, void* dx,
                           int64_t R, int64_t K, int64_t N, int64_t E, hipStream_t st) {
  GroupedArgs a{};
  a.A = dy; a.B = weight; a.out = dx; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = R; a.J = K; a.K = N;
  a.lda = N; a.ldb = K; a.ldo = K; a.b_expert = N * K;
  return MHC_DISPATCH_DTYPE(dtype, [&] { return launch_grouped<T, T, false, true, Role::kRows>(a, who, st); });
}

int grouped_weight_gradient(const char* who, const void* dy, const void* x, int dtype, const int32_t* offsets, void* dw,
                            int64_t R, int64_t K, int64_t N, int64_t E, hipStream_t st) {
  GroupedArgs a{};
  a.A = dy; a.B = x; a.out = dw; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = N; a.J = K; a.K = R;
  a.lda = N; a.ldb = K; a.ldo = K; a.o_expert = N * K;
  return MHC_DISPATCH_DTYPE(dtype, [&] { return launch_grouped<T, T, true, true, Role::kWeight>(a, who, st); });
}

}  // namespace mhc

extern "C" int mhc_grouped_matmul_backward_input(const void* dy, const void* weight, int dtype, const int32_t* offsets,
                                                 void* dx, int64_t R, int64_t K, int64_t N, int64_t E,
                                                 mhc_stream_t stream) {
  const char* who = "grouped_matmul_backward_input";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (R * K == 0) return MHC_OK;
  if (!dx || (E && !offsets) || (N && (!dy || (E && !weight)))) return null_pointer(who);
  return grouped_input_gradient(who, dy, weight, dtype, offsets, dx, R, K, N, E, (hipStream_t)stream);
}

extern "C" int mhc_grouped_matmul_backward_weight(const void* dy, const void* x, int dtype, const int32_t* offsets,
                                                  void* dw, int64_t R, int64_t K, int64_t N, int64_t E,
                                                  mhc_stream_t stream) {
  const char* who = "grouped_matmul_backward_weight";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (E * N * K == 0) return MHC_OK;
  if (!dw || !offsets || (R && (!dy || !x))) return null_pointer(who);
  return grouped_weight_gradient(who, dy, x, dtype, offsets, dw, R, K, N, E, (hipStream_t)stream);
}

extern "C" int mhc_grouped_matmul_mx(const void* x, const void* x_scales, const void* weight, const void* weight_scales,
                                     const int32_t* offsets, void* y, int dtype_y, int64_t R, int64_t K, int64_t N,
                                     int64_t E, mhc_stream_t stream) {
  const char* who = "grouped_matmul_mx";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (R * N == 0) return MHC_OK;
  if (!y || (E && !offsets) || (K && (!x || !x_scales || (E && (!weight || !weight_scales))))) return null_pointer(who);
  if (K % 32 || !aligned16(x) || !aligned16(weight) || ((uintptr_t)x_scales & 3) || ((uintptr_t)weight_scales & 3)) {
    set_error("%s: K in whole blocks of 32, values aligned to 16 bytes and scales to 4 required", who);
    return MHC_ERR_ARG;
  }
  GroupedArgs a{};
  a.A = x; a.B = weight; a.out = y; a.offsets = offsets;
  a.sa = (const uint8_t*)x_scales; a.sb = (const uint8_t*)weight_scales; a.ns = (K + 127) / 128 * 4;
  a.R = R; a.E = (int)E; a.I = R; a.J = N; a.K = K;
  a.lda = K; a.ldb = K; a.ldo = N; a.b_expert = N * K;
  switch (dtype_y) {
    case MHC_DTYPE_BF16: return launch_grouped<Mx, __bf16, false, false, Role::kRows>(a, who, (hipStream_t)stream);
    case MHC_DTYPE_F16: return launch_grouped<Mx, _Float16, false, false, Role::kRows>(a, who, (hipStream_t)stream);
    default: set_error("%s: results in bf16 or fp16, not dtype code %d", who, dtype_y); return MHC_ERR_DTYPE;
  }
}
