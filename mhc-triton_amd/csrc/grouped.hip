// Matrix products grouped by expert: rows [offsets[e-1], offsets[e]) of x belong to expert e.
//
//   forward          y[m, n]     = sum_k x[m, k] w[e][n, k]
//   input gradient   dx[m, k]    = sum_n dy[m, n] w[e][n, k]
//   weight gradient  dw[e][n, k] = sum_{m of e} dy[m, n] x[m, k]
//
// The offsets stay on the device.  A launch has as many row tiles as any split of the rows among the
// experts can need, and each workgroup finds its own in the offsets, so nothing waits for the host and a
// captured graph serves every split.  Rows past the last offset get zeros.
#include "grouped_kernels.hpp"

namespace mhc {

template <typename T, typename TO, bool A_KR, bool B_KR, Role ROLE>
static int launch_grouped(GroupedArgs a, const char* who, hipStream_t st) {
  constexpr int BM = 128, BN = 128;
  a.vec = a.lda % kElems<T> == 0 && a.ldb % kElems<T> == 0 && aligned16(a.A) && aligned16(a.B);
  a.tiles_j = (int)((a.J + BN - 1) / BN);
  int64_t tiles;
  if (ROLE == Role::kWeight) {
    a.tiles_i = (int)((a.I + BM - 1) / BM);
    tiles = (int64_t)a.E * a.tiles_i * a.tiles_j;
  } else {
    const int64_t most = a.R / BM + a.E + 1;
    a.tiles_i = (int)(a.R < most ? a.R : most);
    tiles = (int64_t)a.tiles_i * a.tiles_j;
  }
  if (tiles >= ((int64_t)1 << 32) / 256) {
    set_error("%s: %lld tiles are too many for a call", who, (long long)tiles);
    return MHC_ERR_ARG;
  }
  if (a.vec) grouped_kernel<T, TO, A_KR, B_KR, BM, BN, ROLE, true><<<dim3((unsigned)tiles), 256, 0, st>>>(a);
  else grouped_kernel<T, TO, A_KR, B_KR, BM, BN, ROLE, false><<<dim3((unsigned)tiles), 256, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

static int check_grouped(const char* who, int64_t R, int64_t K, int64_t N, int64_t E) {
  if (R < 0 || K < 0 || N < 0 || E < 0) {
    set_error("%s: negative size (R=%lld K=%lld N=%lld E=%lld)", who, (long long)R, (long long)K, (long long)N,
              (long long)E);
    return MHC_ERR_ARG;
  }
  // A row's byte offsets inside a tile are 32-bit, as are tile counts; offsets are int32.
  if (R >= ((int64_t)1 << 31) || K > kMaxWidth || N > kMaxWidth || E > kMaxExperts) {
    set_error("%s: R=%lld K=%lld N=%lld E=%lld exceeds 2^31-1 rows, widths of %lld or %lld experts", who, (long long)R,
              (long long)K, (long long)N, (long long)E, (long long)kMaxWidth, (long long)kMaxExperts);
    return MHC_ERR_ARG;
  }
  return MHC_OK;
}

static int null_pointer(const char* who) {
  set_error("%s: null pointer", who);
  return MHC_ERR_ARG;
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

extern "C" int mhc_grouped_matmul_backward_input(const void* dy, const void* weight, int dtype, const int32_t* offsets,
                                                 void* dx, int64_t R, int64_t K, int64_t N, int64_t E,
                                                 mhc_stream_t stream) {
  const char* who = "grouped_matmul_backward_input";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (R * K == 0) return MHC_OK;
  if (!dx || (E && !offsets) || (N && (!dy || (E && !weight)))) return null_pointer(who);
  GroupedArgs a{};
  a.A = dy; a.B = weight; a.out = dx; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = R; a.J = K; a.K = N;
  a.lda = N; a.ldb = K; a.ldo = K; a.b_expert = N * K;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    return launch_grouped<T, T, false, true, Role::kRows>(a, who, (hipStream_t)stream);
  });
}

extern "C" int mhc_grouped_matmul_backward_weight(const void* dy, const void* x, int dtype, const int32_t* offsets,
                                                  void* dw, int64_t R, int64_t K, int64_t N, int64_t E,
                                                  mhc_stream_t stream) {
  const char* who = "grouped_matmul_backward_weight";
  if (int rc = check_grouped(who, R, K, N, E)) return rc;
  if (E * N * K == 0) return MHC_OK;
  if (!dw || !offsets || (R && (!dy || !x))) return null_pointer(who);
  GroupedArgs a{};
  a.A = dy; a.B = x; a.out = dw; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = N; a.J = K; a.K = R;
  a.lda = N; a.ldb = K; a.ldo = K; a.o_expert = N * K;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    return launch_grouped<T, T, true, true, Role::kWeight>(a, who, (hipStream_t)stream);
  });
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
