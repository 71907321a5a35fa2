// Dropout from a counter-based generator: the mask is recomputed from (seed, offset, element index)
// wherever it is needed, forward and backward, and never stored.
//
//   y_i = [residual_i +] (u_i < kept ? x_i * 65536 / kept : 0),   kept = round((1 - p) * 65536)
//
// u_i is the 16-bit half i % 8 of the four words that Philox4x32 with ten rounds (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) makes of the counter (i / 8, offset)
// under the key `seed`.  The probability is thus a multiple of 2^-16, and the kept values are scaled by
// the inverse of the probability that they really have, so the expectation is exact.
//
// Bound by the bus (two or three tensors), as long as the generator stays below it: its twenty 32x32-bit
// products per call are quarter rate, which is why a call serves eight elements (halves) and not four.
// 16384 x 4096 bf16: with a residual 62 us (6.4 TB/s), a gradient 44.5 us (6.0 TB/s).
#include "stream_kernels.hpp"

namespace mhc {

struct Rng {
  uint64_t seed, offset;
};

__device__ __forceinline__ void philox(uint64_t counter, Rng rng, uint32_t (&out)[4]) {
  uint32_t a = (uint32_t)counter, b = (uint32_t)(counter >> 32);
  uint32_t c = (uint32_t)rng.offset, d = (uint32_t)(rng.offset >> 32);
  uint32_t k0 = (uint32_t)rng.seed, k1 = (uint32_t)(rng.seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
    a = (uint32_t)(q >> 32) ^ b ^ k0;
    b = (uint32_t)q;
    c = (uint32_t)(p >> 32) ^ d ^ k1;
    d = (uint32_t)p;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  out[0] = a; out[1] = b; out[2] = c; out[3] = d;
}

struct DropoutArgs {
  const void *x, *res;
  void* y;
  int64_t n, first;  // first: the launch's first generator call
  uint32_t kept;
  float scale;
  Rng rng;
  const int64_t* state;  // {seed, offset} on the device instead of rng; may be null
  int64_t* used;         // where the kernel writes what it drew from; may be null
};

constexpr int kDropWidth = 8;  // elements per generator call

// Workgroups of a launch: the runtime takes fewer than 2^32 work items.
constexpr int64_t kMaxGridX = ((int64_t)1 << 32) / kThreads - 1;

// A lane takes eight neighbouring elements.  VEC: all tensors 16-byte aligned; otherwise the same
// vectors at the elements' own alignment.  The last n % 8 elements go one by one.
template <typename T, bool RES, bool VEC>
__global__ __launch_bounds__(kThreads) void dropout_kernel(DropoutArgs a) {
  const int64_t call = a.first + (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t i = call * kDropWidth;
  if (a.state) {
    a.rng.seed = (uint64_t)a.state[0];
    a.rng.offset = (uint64_t)a.state[1];
  }
  if (call == 0 && a.used) {
    a.used[0] = (int64_t)a.rng.seed;
    a.used[1] = (int64_t)a.rng.offset;
  }
  if (i >= a.n) return;
  const T* x = (const T*)a.x + i;
  const T* res = (const T*)a.res + i;
  T* y = (T*)a.y + i;
  const bool whole = i + kDropWidth <= a.n;
  Frag<T, kDropWidth> xf, rf;
  if (whole) {
    if constexpr (VEC) {
      xf.template load<true>(x);
      if constexpr (RES) rf.template load<true>(res);
    } else {
      xf.template load<true>(RagSpan<T>(x, 0), 0);
      if constexpr (RES) rf.template load<true>(RagSpan<T>(res, 0), 0);
    }
    loads_issued();
  }
  uint32_t w[4];
  philox((uint64_t)call, a.rng, w);
  float v[kDropWidth], r[kDropWidth];
  const int m = whole ? kDropWidth : (int)(a.n - i);
  if (whole) {
    xf.unpack(v);
    if constexpr (RES) rf.unpack(r);
  } else {
#pragma unroll
    for (int e = 0; e < kDropWidth; ++e) {
      v[e] = e < m ? to_f32(x[e]) : 0.f;
      r[e] = RES && e < m ? to_f32(res[e]) : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < kDropWidth; ++e) {
    const uint32_t u = e % 2 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
    v[e] = u < a.kept ? v[e] * a.scale : 0.f;  // a dropped infinity or NaN leaves a zero
    if constexpr (RES) v[e] += r[e];
  }
  if (whole) {
    if constexpr (VEC) st<T, kDropWidth, true>(y, v);
    else st_from<T, kDropWidth, true>(RagSpan<T>(y, 0), 0, v, 0);
  } else {
#pragma unroll
    for (int e = 0; e < kDropWidth; ++e)
      if (e < m) y[e] = from_f32<T>(v[e]);
  }
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_dropout(const void* x, const void* residual, int dtype, void* y, int64_t n, double p,
                           uint64_t seed, uint64_t offset, const int64_t* state, int64_t* used,
                           mhc_stream_t stream) {
  if (n < 0 || !(p >= 0. && p <= 1.)) {
    set_error("dropout: bad size or probability (n=%lld p=%g)", (long long)n, p);
    return MHC_ERR_ARG;
  }
  if (n == 0 && !used) return MHC_OK;
  if (n && (!x || !y)) {
    set_error("dropout: null pointer");
    return MHC_ERR_ARG;
  }
  const int64_t blocks = n ? (n + kDropWidth * kThreads - 1) / (kDropWidth * kThreads) : 1;
  DropoutArgs a{x, residual, y, n, 0, (uint32_t)rint((1. - p) * 65536.), 0.f, {seed, offset}, state, used};
  a.scale = a.kept ? (float)(65536. / a.kept) : 0.f;
  const bool vec = aligned16(x) && aligned16(y) && aligned16(residual);
  hipStream_t st = (hipStream_t)stream;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    auto go = [&](auto res, auto v) {
      for (int64_t b = 0; b < blocks; b += kMaxGridX) {
        a.first = b * kThreads;
        const unsigned nb = (unsigned)(blocks - b < kMaxGridX ? blocks - b : kMaxGridX);
        dropout_kernel<T, decltype(res)::value, decltype(v)::value><<<dim3(nb), kThreads, 0, st>>>(a);
        if (int rc = hip_status(hipGetLastError(), "dropout launch")) return rc;
      }
      return (int)MHC_OK;
    };
    if (residual) return vec ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
    return vec ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
  });
}
