// The gated product that a feed-forward begins with, its rows grouped by expert as in grouped.hip or all of one:
//
//   g = x Wg^T,  u = x Wu^T,  y = act(g) * u,   Wg the first N rows of a weight [2N, K], Wu the others
//   dg = dy u act'(g),  du = dy act(g),  dx = [dg du] W,  dW = [dg du]^T x
//
// Forward the tiles of grouped_kernels.hpp with gates and values side by side: both products, the activation and their
// product in one launch, x read once.  For a backward it leaves g and u in fp32: rounded to 16 bits they would put
// two more roundings into every gradient (1.7 times the error that one rounding of [dg du] and one of the result give).
// At 16384 rows of 4096 to 8192 in bf16 writing them is 190 of the forward's 1950 us, and [dg du] from them 340 us of the
// backward's 4340.
//
// Bound by the matrix products, for few rows by reading the weight.  fp32, 8192 rows of 2048 to 4096: forward 1950 us
// (141 TFLOP/s, the library's plain product 148), backward 4000 (137).
#include "grouped_launch.hpp"

namespace mhc {

// [dg du] from dy, g and u: a lane four neighbouring columns.
struct GateArgs {
  const void* dy;
  const float* saved;
  void* out;
  int64_t R, N, first;  // first: the launch's first vector
  int act;
};

constexpr int64_t kMaxGate = (((int64_t)1 << 32) / kThreads - 1) * kThreads;  // vectors of a launch

template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void gate_backward_kernel(GateArgs a) {
  const int64_t per = (a.N + 3) / 4, at = a.first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t r = at / per;
  if (r >= a.R) return;
  const int c = (int)(at - r * per) * 4, n = (int)(a.N - c < 4 ? a.N - c : 4);
  const T* dy = (const T*)a.dy + r * a.N + c;
  const float* s = a.saved + r * 2 * a.N + c;
  T* out = (T*)a.out + r * 2 * a.N + c;
  f32x4 d = {0.f, 0.f, 0.f, 0.f}, g = d, u = d;
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      d = *reinterpret_cast<const f32x4*>(dy);
    } else {
      const s16x4 v = *reinterpret_cast<const s16x4*>(dy);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const short bits = v[i];
        d[i] = to_f32(__builtin_bit_cast(T, bits));
      }
    }
    g = *reinterpret_cast<const f32x4*>(s);
    u = *reinterpret_cast<const f32x4*>(s + a.N);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < n) {
        d[i] = to_f32(dy[i]);
        g[i] = s[i];
        u[i] = s[a.N + i];
      }
  }
  f32x4 dg, du;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    dg[i] = d[i] * u[i] * activate_slope(a.act, g[i]);
    du[i] = d[i] * activate(a.act, g[i]);
  }
  store4(out, dg, n, VEC);
  store4(out + a.N, du, n, VEC);
}

template <typename T>
static int launch_gate_backward(GateArgs a, const char* who, hipStream_t st) {
  const int64_t total = a.R * ((a.N + 3) / 4);
  const bool vec = a.N % 4 == 0 && aligned16(a.dy) && aligned16(a.saved) && aligned16(a.out);
  for (a.first = 0; a.first < total; a.first += kMaxGate) {
    const int64_t n = total - a.first < kMaxGate ? total - a.first : kMaxGate;
    const dim3 grid((unsigned)((n + kThreads - 1) / kThreads));
    if (vec) gate_backward_kernel<T, true><<<grid, kThreads, 0, st>>>(a);
    else gate_backward_kernel<T, false><<<grid, kThreads, 0, st>>>(a);
    if (int rc = hip_status(hipGetLastError(), who)) return rc;
  }
  return MHC_OK;
}

// As launch_grouped chooses, a column counting for its gate and its value, with limits of its own for fp32, whose loop is
// bound by the matrix cores at any tile (times in us, cold weights where they matter):
//   few rows an expert: 4096 to 8192, one expert, 1 / 8 / 16 / 32 / 64 rows: weights into registers 30.0 / 30.3 / 31.7 / 53.4 / 97.6,
//   64-tiles 30.8 / 31.8 / 31.1 / 31.5 / 32.4 (4.3 TB/s: the weights alone, from memory).
//   256 against 128, 2048 to 4096, 2304 / 2560 / 4096 / 4608 rows (288 to 576 likely 256-tiles): bf16 85 / 91 / 126 / 152 and
//   92 / 93 / 143 / 163; 2048 to 2048, 1280 / 2304 rows (80 and 144) 50 / 54 and 34 / 58 (the rule takes 128 for both).
//   fp32, 256 against 64, the same: 620 / 628 / 981 / 1113 and 641 / 711 / 1133 / 1274 (the rule takes 64 for the first two);
//   264 / 488 and 186 / 324.
//   128 against 64, 2048 to 2048, 384 / 640 / 896 / 1152 / 1664 / 2176 rows (96 to 544 likely 128-tiles): bf16
//   26.8 / 27.5 / 27.9 / 31.6 / 34.8 / 58.4 and 16.4 / 26.7 / 31.8 / 41.4 / 55.7 / 70.3; fp32 137 / 139 / 139 / 253 / 257 / 385 and
//   76 / 115 / 144 / 185 / 254 / 325.
//   any alignment, 2047 to 2048, the same rows: bf16 44 / 46 / 46 / 51 / 52 / 94 and 29 / 37 / 49 / 66 / 77 / 106; fp32
//   165 / 166 / 166 / 276 / 278 / 439 and 90 / 126 / 162 / 207 / 275 / 357.
template <typename T>
static int launch_gated(GroupedArgs a, const char* who, hipStream_t st) {
  constexpr bool F32 = sizeof(T) == 4;
  const bool chunks = a.lda % kElems<T> == 0 && a.ldb % kElems<T> == 0 && aligned16(a.A) && aligned16(a.B);
  const int cus = num_cus();
  const bool few = a.R <= 8 * (int64_t)a.E;
  if (chunks) {
    if (few) return launch_few<T, T, 1, 2, 4, 2, true, true>(a, who, st);
    if (likely_tiles<Role::kRows, 256, 128>(a) >= (F32 ? 2 : 1) * cus && a.R >= 256 * (int64_t)a.E)
      return launch_direct<T, T, false, false, 256, 256, 2, 4, 2, Role::kRows, true>(a, who, st);
    if constexpr (!F32)
      if (likely_tiles<Role::kRows, 128, 64>(a) >= cus)
        return launch_direct<T, T, false, false, 128, 128, 2, 2, 2, Role::kRows, true>(a, who, st);
    return launch_direct<T, T, false, false, 64, 64, 2, 2, 4, Role::kRows, true>(a, who, st);
  }
  if (few) return launch_few<T, T, 1, 2, 4, 2, false, true>(a, who, st);
  if constexpr (!F32)
    if (likely_tiles<Role::kRows, 128, 64>(a) >= cus) return launch_general<T, false, false, 128, 128, Role::kRows, true>(a, who, st);
  return launch_general<T, false, false, 64, 64, Role::kRows, true>(a, who, st);
}

static int check_gated(const char* who, int64_t R, int64_t K, int64_t N, int64_t E, int act, const int32_t* offsets) {
  if (N < 0 || N > kMaxWidth / 2) {
    set_error("%s: N=%lld; at most %lld", who, (long long)N, (long long)kMaxWidth / 2);
    return MHC_ERR_ARG;
  }
  if (int rc = check_grouped(who, R, K, 2 * N, E)) return rc;
  if (act != MHC_ACT_SILU && act != MHC_ACT_GELU && act != MHC_ACT_GELU_TANH) {
    set_error("%s: unknown activation %d", who, act);
    return MHC_ERR_ARG;
  }
  if (!offsets && E > 1) {  // without experts there are none to read
    set_error("%s: %lld experts need offsets", who, (long long)E);
    return MHC_ERR_ARG;
  }
  return MHC_OK;
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_gated_matmul_forward(const void* x, const void* weight, int dtype, const int32_t* offsets, int act, void* y,
                                        float* saved, int64_t R, int64_t K, int64_t N, int64_t E, mhc_stream_t stream) {
  const char* who = "gated_matmul_forward";
  if (int rc = check_gated(who, R, K, N, E, act, offsets)) return rc;
  if (R * N == 0) return MHC_OK;
  if (!y || (K && (!x || (E && !weight)))) return null_pointer(who);
  GroupedArgs a{};
  a.A = x; a.B = weight; a.out = y; a.saved = saved; a.offsets = offsets;
  a.R = R; a.E = (int)E; a.I = R; a.J = N; a.K = K;
  a.lda = K; a.ldb = K; a.ldo = N; a.b_expert = 2 * N * K;
  a.half = N; a.act = act;
  return MHC_DISPATCH_DTYPE(dtype, [&] { return launch_gated<T>(a, who, (hipStream_t)stream); });
}

extern "C" size_t mhc_gated_matmul_backward_workspace_bytes(int64_t R, int64_t N, int dtype) {
  return R > 0 && N > 0 ? (size_t)R * 2 * N * (dtype == MHC_DTYPE_F32 ? 4 : 2) : 0;
}

extern "C" int mhc_gated_matmul_backward(const void* dy, const float* saved, const void* x, const void* weight, int dtype,
                                         const int32_t* offsets, int act, void* dx, void* dweight, int64_t R, int64_t K,
                                         int64_t N, int64_t E, void* workspace, size_t workspace_bytes,
                                         mhc_stream_t stream) {
  const char* who = "gated_matmul_backward";
  if (int rc = check_gated(who, R, K, N, E, act, offsets)) return rc;
  if (!(dx && R * K) && !(dweight && E * N * K)) return MHC_OK;
  if (R * N && (!dy || !saved)) return null_pointer(who);
  if ((dx && R * K && N && E && !weight) || (dweight && E * N * K && R && !x)) return null_pointer(who);
  const size_t need = mhc_gated_matmul_backward_workspace_bytes(R, N, dtype);
  if (need && (!workspace || workspace_bytes < need)) {
    set_error("%s: workspace of %zu bytes, %zu needed", who, workspace ? workspace_bytes : (size_t)0, need);
    return MHC_ERR_WORKSPACE;
  }
  const hipStream_t st = (hipStream_t)stream;
  if (R * N) {
    const GateArgs g{dy, saved, workspace, R, N, 0, act};
    if (int rc = MHC_DISPATCH_DTYPE(dtype, [&] { return launch_gate_backward<T>(g, who, st); })) return rc;
  }
  if (dx && R * K)
    if (int rc = grouped_input_gradient(who, workspace, weight, dtype, offsets, dx, R, K, 2 * N, E, st)) return rc;
  if (dweight && E * N * K) return grouped_weight_gradient(who, workspace, x, dtype, offsets, dweight, R, K, 2 * N, E, st);
  return MHC_OK;
}
