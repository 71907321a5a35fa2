// Linear attention with a decay for each head: chunked over sequences with its gradients, and a token at a time.
//
//   S_t = l S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log decay), log decays above 0 counting as 0
//
// The gradients are the same scan with other operands:
//   dq = scan(do, v, k) with the states transposed, dv = scan(k, q, do) and dk = scan(v, do, q) from the last token to
//   the first, whose state begins as the last state's gradient and ends as the first one's.
#include "decay_kernels.hpp"

namespace mhc {

// Tokens of a segment.  Enough segments for two workgroups a CU (the kernel's occupancy), but none shorter than
// kLeast: each costs a state written and read again by those behind it.
constexpr int64_t kLeast = 512;

static int64_t segment_tokens(int64_t R, int64_t N, int64_t H, int64_t Dv, bool packed) {
  const int64_t longest = packed || N == 0 ? R : R / N;
  const int64_t heads = H * ((Dv + kStateCols - 1) / kStateCols);
  const int64_t sequences = packed ? 1 : N;
  int64_t want = 2 * num_cus() / (heads * sequences > 0 ? heads * sequences : 1);
  if (want < 1) want = 1;
  int64_t seg = (longest + want - 1) / want;
  if (seg < kLeast) seg = kLeast;
  return (seg + kChunk - 1) / kChunk * kChunk;
}

static int64_t count_tiles(int64_t R, int64_t N, int64_t seg, bool packed) {
  if (packed) return R / seg + N + 1;
  const int64_t T = N ? R / N : 0;
  return N * (T > seg ? (T + seg - 1) / seg : 1);
}

static int64_t parts_bytes(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, bool packed) {
  const int64_t seg = segment_tokens(R, N, H, Dv, packed);
  if ((packed || N == 0 ? R : R / N) <= seg) return 0;
  return count_tiles(R, N, seg, packed) * H * Dk * Dv * 4;
}

template <typename T, int DK, bool CHUNKS>
static int launch_scan(const DecayArgs& a, bool parts, const char* who, hipStream_t st) {
  const int64_t units = ((int64_t)a.tiles * a.H + 7) / 8 * 8;
  if (units * a.col_tiles * kThreads >= ((int64_t)1 << 32)) {
    set_error("%s: %lld workgroups are too many for a call", who, (long long)(units * a.col_tiles));
    return MHC_ERR_ARG;
  }
  const dim3 grid((unsigned)(units * a.col_tiles));
  if (parts) {
    decay_kernel<T, DK, CHUNKS, true><<<grid, kThreads, 0, st>>>(a);
    if (int rc = hip_status(hipGetLastError(), who)) return rc;
  }
  decay_kernel<T, DK, CHUNKS, false><<<grid, kThreads, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

template <typename T>
static bool whole_chunks(const void* p, int64_t row, int64_t head, int64_t D) {
  return aligned16(p) && row % kElems<T> == 0 && head % kElems<T> == 0 && D % kElems<T> == 0;
}

template <typename T>
static int scan(DecayArgs a, void* workspace, const char* who, hipStream_t st) {
  const bool packed = a.offsets != nullptr;
  a.T = a.N ? a.R / a.N : 0;
  const int64_t seg = segment_tokens(a.R, a.N, a.H, a.Dv, packed);
  a.seg = (int)seg;
  const int64_t tiles = count_tiles(a.R, a.N, seg, packed);
  if (tiles * a.H >= ((int64_t)1 << 31) - 8) {
    set_error("%s: %lld segments of %d heads are too many for a call", who, (long long)tiles, a.H);
    return MHC_ERR_ARG;
  }
  a.tiles = (int)tiles;
  a.col_tiles = (a.Dv + kStateCols - 1) / kStateCols;
  a.parts = (float*)workspace;
  const bool parts = parts_bytes(a.R, a.N, a.H, a.Dk, a.Dv, packed) != 0;
  const bool chunks = whole_chunks<T>(a.q, a.q_row, a.q_head, a.Dk) && whole_chunks<T>(a.k, a.k_row, a.k_head, a.Dk) &&
                      whole_chunks<T>(a.v, a.v_row, a.v_head, a.Dv);
  if (chunks) return a.Dk <= 64 ? launch_scan<T, 64, true>(a, parts, who, st) : launch_scan<T, 128, true>(a, parts, who, st);
  return a.Dk <= 64 ? launch_scan<T, 64, false>(a, parts, who, st) : launch_scan<T, 128, false>(a, parts, who, st);
}

constexpr int64_t kMaxHeadDim = 128;
constexpr int64_t kMaxRowStride = (int64_t)1 << 22;  // byte offsets inside a chunk are 32-bit

static int check_decay(const char* who, int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, bool packed,
                       std::initializer_list<int64_t> row_strides) {
  if (R < 0 || N < 0 || H < 0 || Dk < 1 || Dv < 1 || Dk > kMaxHeadDim || Dv > kMaxHeadDim || R > kMaxRows ||
      N > ((int64_t)1 << 24) || H * (Dk > Dv ? Dk : Dv) > kMaxRowStride || (!packed && (N ? R % N : R))) {
    set_error("%s: R=%lld N=%lld H=%lld Dk=%lld Dv=%lld (heads of 1 to %lld; sequences of R / N rows)", who, (long long)R,
              (long long)N, (long long)H, (long long)Dk, (long long)Dv, (long long)kMaxHeadDim);
    return MHC_ERR_ARG;
  }
  for (int64_t s : row_strides)
    if (s < 0 || s > kMaxRowStride) {
      set_error("%s: rows %lld elements apart; at most %lld", who, (long long)s, (long long)kMaxRowStride);
      return MHC_ERR_ARG;
    }
  return MHC_OK;
}

static int null_in(const char* who) {
  set_error("%s: null pointer", who);
  return MHC_ERR_ARG;
}

static int check_workspace(const char* who, const void* ws, size_t have, size_t need) {
  if (need == 0 || (ws && have >= need)) return MHC_OK;
  set_error("%s: workspace of %zu bytes, %zu needed", who, ws ? have : (size_t)0, need);
  return MHC_ERR_WORKSPACE;
}

template <typename T, bool VEC>
static int launch_step(DecayStepArgs a, const char* who, hipStream_t st) {
  a.col_tiles = (a.Dv + kStepCols - 1) / kStepCols;
  const int64_t n = (int64_t)a.R * a.H * a.col_tiles;
  if (n * kThreads >= ((int64_t)1 << 32)) {
    set_error("%s: %lld workgroups are too many for a call", who, (long long)n);
    return MHC_ERR_ARG;
  }
  decay_step_kernel<T, VEC><<<dim3((unsigned)n), kThreads, 0, st>>>(a);
  return hip_status(hipGetLastError(), who);
}

}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_decay_attention_workspace_bytes(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, int packed) {
  if (R <= 0 || N < 0 || H <= 0 || Dk <= 0 || Dv <= 0) return 0;
  return (size_t)parts_bytes(R, N, H, Dk, Dv, packed);
}

extern "C" int mhc_decay_attention_forward(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                           int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int dtype,
                                           const float* log_decay, const int32_t* offsets, const float* first, void* o,
                                           float* last, int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv,
                                           float scale, void* workspace, size_t workspace_bytes, mhc_stream_t stream) {
  const char* who = "decay_attention_forward";
  if (int rc = check_decay(who, R, N, H, Dk, Dv, offsets != nullptr, {q_row, k_row, v_row})) return rc;
  if (H == 0 || (R == 0 && (N == 0 || !last))) return MHC_OK;
  if (!log_decay || (R && (!q || !k || !v || !o))) return null_in(who);
  const size_t need = mhc_decay_attention_workspace_bytes(R, N, H, Dk, Dv, offsets != nullptr);
  if (int rc = check_workspace(who, workspace, workspace_bytes, need)) return rc;
  DecayArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.log_decay = log_decay; a.offsets = offsets; a.first = first; a.last = last;
  a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
  a.state_row = Dv; a.state_col = 1;
  a.R = R; a.N = (int)N; a.H = (int)H; a.Dk = (int)Dk; a.Dv = (int)Dv;
  a.out_scale = scale; a.in_scale = 1.f; a.lag = 1;
  return MHC_DISPATCH_DTYPE(dtype, [&] { return scan<T>(a, workspace, who, (hipStream_t)stream); });
}

extern "C" size_t mhc_decay_attention_backward_workspace_bytes(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv,
                                                               int packed) {
  const size_t x = mhc_decay_attention_workspace_bytes(R, N, H, Dk, Dv, packed);
  const size_t y = mhc_decay_attention_workspace_bytes(R, N, H, Dv, Dk, packed);
  return x > y ? x : y;
}

extern "C" int mhc_decay_attention_backward(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                            int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* dout,
                                            int64_t do_row, int64_t do_head, int dtype, const float* log_decay,
                                            const int32_t* offsets, const float* first, const float* d_last, void* dq,
                                            void* dk, void* dv, float* d_first, int64_t R, int64_t N, int64_t H,
                                            int64_t Dk, int64_t Dv, float scale, void* workspace, size_t workspace_bytes,
                                            mhc_stream_t stream) {
  const char* who = "decay_attention_backward";
  if (int rc = check_decay(who, R, N, H, Dk, Dv, offsets != nullptr, {q_row, k_row, v_row, do_row})) return rc;
  if (H == 0 || (R == 0 && (N == 0 || !d_first))) return MHC_OK;
  if (!log_decay || (R && (!q || !k || !v || !dout))) return null_in(who);
  const size_t need = mhc_decay_attention_backward_workspace_bytes(R, N, H, Dk, Dv, offsets != nullptr);
  if (int rc = check_workspace(who, workspace, workspace_bytes, need)) return rc;
  DecayArgs base{};
  base.log_decay = log_decay; base.offsets = offsets;
  base.R = R; base.N = (int)N; base.H = (int)H;
  return MHC_DISPATCH_DTYPE(dtype, [&]() -> int {
    if (dq && R) {
      DecayArgs a = base;
      a.q = dout; a.q_row = do_row; a.q_head = do_head;
      a.k = v; a.k_row = v_row; a.k_head = v_head;
      a.v = k; a.v_row = k_row; a.v_head = k_head;
      a.o = dq; a.first = first; a.state_row = 1; a.state_col = Dv;
      a.Dk = (int)Dv; a.Dv = (int)Dk;
      a.out_scale = scale; a.in_scale = 1.f; a.lag = 1;
      if (int rc = scan<T>(a, workspace, who, (hipStream_t)stream)) return rc;
    }
    base.first = d_last;
    base.out_scale = 1.f; base.in_scale = scale; base.lag = 0; base.reverse = true;
    if (dv || (d_first && !dk)) {
      DecayArgs a = base;
      a.q = k; a.q_row = k_row; a.q_head = k_head;
      a.k = q; a.k_row = q_row; a.k_head = q_head;
      a.v = dout; a.v_row = do_row; a.v_head = do_head;
      a.o = dv; a.last = d_first; a.state_row = Dv; a.state_col = 1;
      a.Dk = (int)Dk; a.Dv = (int)Dv;
      if (int rc = scan<T>(a, workspace, who, (hipStream_t)stream)) return rc;
    }
    if (dk) {
      DecayArgs a = base;
      a.q = v; a.q_row = v_row; a.q_head = v_head;
      a.k = dout; a.k_row = do_row; a.k_head = do_head;
      a.v = q; a.v_row = q_row; a.v_head = q_head;
      a.o = dk; a.last = dv ? nullptr : d_first; a.state_row = 1; a.state_col = Dv;
      a.Dk = (int)Dv; a.Dv = (int)Dk;
      if (int rc = scan<T>(a, workspace, who, (hipStream_t)stream)) return rc;
    }
    return MHC_OK;
  });
}

extern "C" int mhc_decay_attention_step(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                        int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int dtype,
                                        const float* log_decay, const int32_t* slots, const float* state,
                                        float* state_out, void* o, int64_t R, int64_t pool, int64_t H, int64_t Dk,
                                        int64_t Dv, float scale, mhc_stream_t stream) {
  const char* who = "decay_attention_step";
  if (R < 0 || pool < 0 || H < 0 || Dk < 1 || Dv < 1 || Dk > kMaxHeadDim || Dv > kMaxHeadDim || R > (1 << 20) ||
      H > 65536 || (!slots && R > pool)) {
    set_error("%s: R=%lld of %lld states, H=%lld Dk=%lld Dv=%lld (heads of 1 to %lld)", who, (long long)R, (long long)pool,
              (long long)H, (long long)Dk, (long long)Dv, (long long)kMaxHeadDim);
    return MHC_ERR_ARG;
  }
  if (R * H == 0) return MHC_OK;
  if (!q || !k || !v || !o || !log_decay || (pool && (!state || !state_out))) return null_in(who);
  DecayStepArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.log_decay = log_decay; a.state = state; a.state_out = state_out; a.slots = slots;
  a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
  a.pool = pool; a.R = (int)R; a.H = (int)H; a.Dk = (int)Dk; a.Dv = (int)Dv; a.scale = scale;
  return MHC_DISPATCH_DTYPE(dtype, [&] {
    if (Dv % 4 == 0 && aligned16(state) && aligned16(state_out)) return launch_step<T, true>(a, who, (hipStream_t)stream);
    return launch_step<T, false>(a, who, (hipStream_t)stream);
  });
}
