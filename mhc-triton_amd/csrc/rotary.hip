// Rotary positions of queries and keys.
//
//   (a, b) -> m (a cos t - b sin t, b cos t + a sin t),   t = position * frequency[i]
//
// for the i-th of `pairs` pairs of a head: elements (i, pairs + i), or (2i, 2i + 1) interleaved; the head's other
// elements go through as they are.  The inverse turns by -t and is the backward.
//
// Angles are taken in fp64 and brought into half a turn there: in fp32 a position of 2^17 would be off by
// 2^17 2^-24 radians.  Sine and cosine are then fp32 and serve every head of the row, from LDS.
//
// Bound by memory: each element is read and written once; 16384 rows of 40 heads of 128 bf16 58 us (5.7 TB/s).
#include "common.hpp"

namespace mhc {

struct RotaryTensor {
  const void* x;
  void* y;
  int64_t row, head;  // strides of x in elements; y is contiguous
  int heads;
};

struct RotaryArgs {
  RotaryTensor t[2];
  const void* positions;
  int64_t position_count;  // row r has position r % position_count
  const double* frequencies;
  int64_t R;
  int D, pairs, rows, per_group, groups;  // rows of a tile; heads of a group, groups of heads
  float magnitude;
  bool wide, inverse;  // 64-bit positions
};

constexpr int kRotaryPairs = 2048;  // (row, pair) angles that a workgroup holds

// W elements at any alignment; W = 1: one.
template <typename T, int W, bool NT>
__device__ __forceinline__ void rot_load(const T* p, float* f) {
  if constexpr (W == 1) f[0] = to_f32(*p);
  else RawVec<T>::unpack(__builtin_bit_cast(typename RawVec<T>::type, load16_any(p, NT)), f);
}
template <typename T, int W, bool NT>
__device__ __forceinline__ void rot_store(T* p, const float* f) {
  if constexpr (W == 1) *p = from_f32<T>(f[0]);
  else store16_any(p, RawVec<T>::pack(f), NT);
}

// An item is a vector of W elements: of each half of the pairs (half layout), of whole pairs (interleaved), or of what
// goes through.  Where W does not divide a part, its last vector is moved back to end with the part and its first
// elements are computed twice, to the same values.  W = 1 (parts shorter than a vector): a pair or an element an item.
template <typename T, int W, bool INTER, bool NT>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  __shared__ float cs[2 * kRotaryPairs];
  const int group = blockIdx.x % a.groups;
  const int h0 = group * a.per_group, h1 = min(h0 + a.per_group, a.t[0].heads + a.t[1].heads);
  const int turned = INTER ? (W == 1 ? a.pairs : (2 * a.pairs + W - 1) / W) : (a.pairs + W - 1) / W;
  const int items = turned + (a.D - 2 * a.pairs + W - 1) / W;
  const int64_t tiles = (a.R + a.rows - 1) / a.rows;
  for (int64_t tile = blockIdx.x / a.groups; tile < tiles; tile += gridDim.x / a.groups) {
    const int64_t r0 = tile * a.rows;
    const int rows = (int)min((int64_t)a.rows, a.R - r0);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * a.pairs; i += kThreads) {
      const int64_t at = (r0 + i / a.pairs) % a.position_count;
      const int64_t pos = a.wide ? ((const int64_t*)a.positions)[at] : (int64_t)((const int32_t*)a.positions)[at];
      double turns = (double)pos * a.frequencies[i % a.pairs] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      float s, c;
      sincospif(2.f * (float)turns, &s, &c);
      cs[2 * i] = c * a.magnitude;
      cs[2 * i + 1] = (a.inverse ? -s : s) * a.magnitude;
    }
    __syncthreads();
    const int per_row = (h1 - h0) * items;
    for (int i = threadIdx.x; i < rows * per_row; i += kThreads) {
      const int r = i / per_row, in_row = i - r * per_row;
      int h = in_row / items, v = in_row - h * items;
      h += h0;
      const bool second = h >= a.t[0].heads;
      const RotaryTensor& t = a.t[second];
      if (second) h -= a.t[0].heads;
      const T* x = (const T*)t.x + (r0 + r) * t.row + h * t.head;
      T* y = (T*)t.y + ((r0 + r) * t.heads + h) * a.D;
      const float* w = cs + 2 * r * a.pairs;
      if (v >= turned) {
        const int c = min(2 * a.pairs + (v - turned) * W, a.D - W);
        float f[W];
        rot_load<T, W, NT>(x + c, f);
        rot_store<T, W, NT>(y + c, f);
      } else if constexpr (INTER && W > 1) {
        const int c = min(v * W, 2 * a.pairs - W);
        float f[W], g[W];
        rot_load<T, W, NT>(x + c, f);
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          const float co = w[c + e], si = w[c + e + 1];
          g[e] = f[e] * co - f[e + 1] * si;
          g[e + 1] = f[e + 1] * co + f[e] * si;
        }
        rot_store<T, W, NT>(y + c, g);
      } else {
        const int c = INTER ? v : min(v * W, a.pairs - W);  // first pair
        const int ca = INTER ? 2 * c : c, cb = INTER ? 2 * c + 1 : a.pairs + c;
        float f[W], g[W], p[W], q[W];
        rot_load<T, W, NT>(x + ca, f);
        rot_load<T, W, NT>(x + cb, g);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float co = w[2 * (c + e)], si = w[2 * (c + e) + 1];
          p[e] = f[e] * co - g[e] * si;
          q[e] = g[e] * co + f[e] * si;
        }
        rot_store<T, W, NT>(y + ca, p);
        rot_store<T, W, NT>(y + cb, q);
      }
    }
  }
}

template <typename T>
static int launch_rotary(RotaryArgs a, bool interleaved, hipStream_t st) {
  constexpr int N = Vec<T>::N;
  const int turned = interleaved ? 2 * a.pairs : a.pairs, rest = a.D - 2 * a.pairs;
  const bool vec = turned >= N && (rest == 0 || rest >= N);
  const int w = vec ? N : 1;
  const int items = (interleaved && !vec ? a.pairs : (turned + w - 1) / w) + (rest + w - 1) / w;
  const int heads = a.t[0].heads + a.t[1].heads;
  const int cus = num_cus();
  // Few rows: a workgroup takes as many heads of one row as it has lanes for, so that nothing is done one after the
  // other.  Many: all heads of four rows, which share the row's angles.
  a.rows = 1;
  a.per_group = heads;
  if (a.R < 4 * (int64_t)cus) {
    a.per_group = kThreads / items > 0 ? kThreads / items : 1;
    if (a.per_group > heads) a.per_group = heads;
  } else {
    while (a.rows < 4 && 2 * a.rows * a.pairs <= kRotaryPairs) a.rows *= 2;
  }
  a.groups = (heads + a.per_group - 1) / a.per_group;
  const int64_t tiles = (a.R + a.rows - 1) / a.rows;
  const int64_t most = (((int64_t)1 << 32) / kThreads - 1) / a.groups;  // fewer than 2^32 work items
  const dim3 grid((unsigned)((tiles < most ? tiles : most) * a.groups));
  // Streaming accesses where the rows are more than the caches hold: 40 heads of 128 bf16, plain against streaming, 84 MB read
  // and written 15.6 / 17.9 us, 168 MB 30.1 / 32.6 (30.6 / 30.7 right after the rows were made), 336 MB 65.2 / 60.7 (59.7 / 44.9).
  const bool stream = vec && 2 * a.R * heads * a.D * (int64_t)sizeof(T) > ((int64_t)192 << 20);
  auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, st>>>(a); };
  if (vec && interleaved) go(stream ? rotary_kernel<T, N, true, true> : rotary_kernel<T, N, true, false>);
  else if (vec) go(stream ? rotary_kernel<T, N, false, true> : rotary_kernel<T, N, false, false>);
  else if (interleaved) go(rotary_kernel<T, 1, true, false>);
  else go(rotary_kernel<T, 1, false, false>);
  return hip_status(hipGetLastError(), "rotary launch");
}

}  // namespace mhc

using namespace mhc;

extern "C" int mhc_rotary(const void* q, int64_t q_row, int64_t q_head, void* q_out, int64_t q_heads, const void* k,
                          int64_t k_row, int64_t k_head, void* k_out, int64_t k_heads, int dtype, const void* positions,
                          int wide, int64_t position_count, const double* frequencies, int64_t pairs, int64_t R,
                          int64_t D, float magnitude, int interleaved, int inverse, mhc_stream_t stream) {
  const char* who = "rotary";
  if (R < 0 || D < 0 || q_heads < 0 || k_heads < 0 || pairs < 0 || 2 * pairs > D || D > 2 * kRotaryPairs ||
      q_heads + k_heads > 65536 || R > ((int64_t)1 << 40)) {
    set_error("%s: R=%lld D=%lld heads=%lld+%lld pairs=%lld (pairs of a head of at most %d, 65536 heads)", who,
              (long long)R, (long long)D, (long long)q_heads, (long long)k_heads, (long long)pairs, 2 * kRotaryPairs);
    return MHC_ERR_ARG;
  }
  if (R * D * (q_heads + k_heads) == 0) return MHC_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !positions || (pairs && !frequencies)) {
    set_error("%s: null pointer", who);
    return MHC_ERR_ARG;
  }
  if (position_count <= 0) {
    set_error("%s: no positions", who);
    return MHC_ERR_ARG;
  }
  RotaryArgs a{};
  a.t[0] = {q, q_out, q_row, q_head, (int)q_heads};
  a.t[1] = {k, k_out, k_row, k_head, (int)k_heads};
  a.positions = positions;
  a.position_count = position_count;
  a.frequencies = frequencies;
  a.R = R;
  a.D = (int)D;
  a.pairs = (int)pairs;
  a.magnitude = magnitude;
  a.wide = wide;
  a.inverse = inverse;
  return MHC_DISPATCH_DTYPE(dtype, [&] { return launch_rotary<T>(a, interleaved, (hipStream_t)stream); });
}
