// Linear attention with a decay for each head: chunked over sequences with its gradients, and a token at a time.
//
//   S_t = l S_{t-1} + k_t^T v_t,   o_t = scale q_t S_t,   l = exp(log decay), log decays above 0 counting as 0
//
// The gradients are the same scan with other operands:
//   dq = scan(do, v, k) with the states transposed, dv = scan(k, q, do) and dk = scan(v, do, q) from the last token to
//   the first, whose state begins as the last state's gradient and ends as the first one's.
#include "decay_kernels.hpp"

namespace mhc {

// Tokens of a segment.  Enough segments for a workgroup a CU, but none shorter than kLeast: each costs a state written and
// read again.  Forward / backward of bf16 heads of 128: 32 heads of 8192 tokens 112 / 235 us, with two workgroups a CU 118 /
// 250; 8 heads of 2048 43 / 50 us, with kLeast = 512 53 / 59; the other way round from 256 segments of one head on (65536
// tokens 109 / 140, with 512 91 / 116).
constexpr int64_t kLeast = 256;
static int64_t segment_tokens(int64_t R, int64_t N, int64_t H, bool packed) {
  const int64_t longest = packed || N == 0 ? R : R / N;
  const int64_t sequences = packed ? 1 : N;
  int64_t want = num_cus() / (H * sequences > 0 ? H * sequences : 1);
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

// From so many packed sequences on a table says which segment a tile has; the tiles' own searches grow with the square of their
// number.  Heads of 128, sequences of 64 tokens, forward without / with in us: 4 heads, 32 / 64 / 128 / 256 / 1024 sequences
// 15 / 16 / 28 / 53 / 254 and 17 / 18 / 26 / 41 / 141; 32 heads, 32 / 64 / 128 / 256 / 1024 39 / 69 / 150 / 307 / 1694 and
// 39 / 66 / 137 / 264 / 1004.
constexpr int64_t kTableSequences = 128;

// A scan's segments and what they take of the workspace: the states that they leave, then the table.
struct Plan {
  int64_t seg, tiles;
  int64_t parts;  // bytes; 0: no sequence has a second segment
  int64_t joins;  // sequences of more than kSummed segments, at most; 0: decay_join_kernel does not run
  int64_t table;  // bytes; 0: without
};
static Plan plan_scan(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, bool packed) {
  Plan p;
  p.seg = segment_tokens(R, N, H, packed);
  p.tiles = count_tiles(R, N, p.seg, packed);
  const int64_t longest = packed || N == 0 ? R : R / N;
  p.parts = longest > p.seg ? (R - 1) / p.seg * H * Dk * Dv * 4 : 0;  // places of part_place
  // Packed sequences' lengths are not known here, and that one is so long is not likely: from twice as many rows on.  One head of
  // 65536 tokens in 64 sequences, forward / backward in us without and with the launch: split evenly 44 / 81 and 47 / 83, all but 63 in
  // the first 281 / 994 and 111 / 145; 12 heads of 16384 in 256 sequences 110 / 300 and 115 / 304, 169 / 437 and 176 / 417.
  p.joins = longest <= kSummed * p.seg * (packed && N > 1 ? 2 : 1) ? 0 : packed ? (R - 1) / (kSummed * p.seg) : N;
  p.table = packed && N >= kTableSequences ? (p.tiles + p.joins) * 16 : 0;
  return p;
}

template <typename T, int DK, int WAVES, int WEIGHTED, bool CHUNKS>
static int launch_scan(const DecayJobs& jobs, int64_t joins, bool states, bool outputs, const char* who, hipStream_t st) {
  constexpr int NTH = 64 * WAVES;
  const DecayArgs& a = jobs.job[0];
  const int64_t groups = ((int64_t)a.tiles * a.H + 7) / 8 * 8 * jobs.n;
  if (groups * NTH >= ((int64_t)1 << 32)) {
    set_error("%s: %lld workgroups are too many for a call", who, (long long)groups);
    return MHC_ERR_ARG;
  }
  const dim3 grid((unsigned)groups);
  if (states) decay_kernel<T, DK, WAVES, WEIGHTED, CHUNKS, true><<<grid, NTH, 0, st>>>(jobs);
  if (states && joins) {
    const int64_t units = joins * a.H, most = (((int64_t)1 << 32) / kThreads - 1) / units, want = (a.Dk * a.Dv + kJoin - 1) / kJoin;
    const int blocks = (int)(want < most ? want : most);
    decay_join_kernel<<<dim3((unsigned)(units * blocks)), kThreads, 0, st>>>(a, blocks);
  }
  if (outputs) decay_kernel<T, DK, WAVES, WEIGHTED, CHUNKS, false><<<grid, NTH, 0, st>>>(jobs);
  return hip_status(hipGetLastError(), who);
}

// Rows that overlap (one row expanded to all tokens among them) are not: what a buffer over the n rows of a short chunk
// leaves out then lies inside them.
template <typename T>
static bool whole_chunks(const void* p, int64_t row, int64_t head, int64_t D) {
  return aligned16(p) && row >= D && row % kElems<T> == 0 && head % kElems<T> == 0 && D % kElems<T> == 0;
}

// What the scans of a call share, and its table made at `table` where it is null and there is to be one.
static int set_plan(DecayArgs& a, const Plan& plan, void* table, const char* who, hipStream_t st) {
  if (plan.tiles * a.H >= ((int64_t)1 << 31) - 8) {
    set_error("%s: %lld segments of %d heads are too many for a call", who, (long long)plan.tiles, a.H);
    return MHC_ERR_ARG;
  }
  a.T = a.N ? a.R / a.N : 0;
  a.seg = (int)plan.seg;
  a.tiles = (int)plan.tiles;
  a.joined = plan.joins > 0;
  if (!plan.table || a.table) return MHC_OK;
  a.table = (const int32_t*)table;
  decay_table_kernel<<<dim3(1), kTableThreads, 0, st>>>(a, (int32_t*)table, (int)plan.joins);
  return hip_status(hipGetLastError(), who);
}

// The segments' states (needed where there are several), or the outputs, of scans alike in their plan and in how many
// halves of 128 their dims take.  exact: a last state is to come of them.
enum { kStates = 1, kOutputs = 2 };
template <typename T>
static int scan(DecayJobs jobs, const Plan& plan, int what, bool exact, const char* who, hipStream_t st) {
  bool chunks = true;
  for (int j = 0; j < jobs.n; ++j) {
    DecayArgs& a = jobs.job[j];
    chunks = chunks && whole_chunks<T>(a.q, a.q_row, a.q_head, a.Dk) && whole_chunks<T>(a.k, a.k_row, a.k_head, a.Dk) &&
             whole_chunks<T>(a.v, a.v_row, a.v_head, a.Dv) && aligned16(a.o);
  }
  const bool states = what & kStates && plan.parts, outputs = what & kOutputs;
  const DecayArgs& a = jobs.job[0];
  auto launch = [&](auto w, auto parts) {
    constexpr int WAVES = decltype(w)::value, WEIGHTED = decltype(parts)::value;
    if (chunks)
      return a.Dk <= 64 ? launch_scan<T, 64, WAVES, WEIGHTED, true>(jobs, plan.joins, states, outputs, who, st)
                        : launch_scan<T, 128, WAVES, WEIGHTED, true>(jobs, plan.joins, states, outputs, who, st);
    return a.Dk <= 64 ? launch_scan<T, 64, WAVES, WEIGHTED, false>(jobs, plan.joins, states, outputs, who, st)
                      : launch_scan<T, 128, WAVES, WEIGHTED, false>(jobs, plan.joins, states, outputs, who, st);
  };
  using std::integral_constant;
  if constexpr (sizeof(T) == 4) {
    return a.Dv > 64 ? launch(integral_constant<int, 8>(), integral_constant<int, 3>())
                     : launch(integral_constant<int, 4>(), integral_constant<int, 3>());
  } else {
    if (exact) return a.Dv > 64 ? launch(integral_constant<int, 8>(), integral_constant<int, 3>())
                                : launch(integral_constant<int, 4>(), integral_constant<int, 3>());
    return a.Dv > 64 ? launch(integral_constant<int, 8>(), integral_constant<int, 2>())
                     : launch(integral_constant<int, 4>(), integral_constant<int, 2>());
  }
}

constexpr int64_t kMaxHeadDim = 128;
constexpr int64_t kMaxRowStride = (int64_t)1 << 22;  // byte offsets inside a chunk are 32-bit

static int check_decay(const char* who, int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, bool packed,
                       std::initializer_list<int64_t> row_strides) {
  if (R < 0 || N < 0 || H < 0 || Dk < 1 || Dv < 1 || Dk > kMaxHeadDim || Dv > kMaxHeadDim || R > kMaxRows ||
      N > ((int64_t)1 << 24) || H * (Dk > Dv ? Dk : Dv) > kMaxRowStride || (!packed && R % N)) {
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

extern "C" size_t mhc_decay_attention_workspace_bytes(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv, int packed,
                                                      int /*dtype*/) {
  if (R < 0 || N < 0 || H <= 0 || Dk <= 0 || Dv <= 0) return 0;
  const Plan p = plan_scan(R, N, H, Dk, Dv, packed);
  return (size_t)(p.parts + p.table);
}

extern "C" int mhc_decay_attention_forward(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                           int64_t k_head, const void* v, int64_t v_row, int64_t v_head, int dtype,
                                           const float* log_decay, const int32_t* offsets, const float* first, void* o,
                                           float* last, int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv,
                                           float scale, void* workspace, size_t workspace_bytes, mhc_stream_t stream) {
  const char* who = "decay_attention_forward";
  const bool packed = offsets || N == 0;
  if (int rc = check_decay(who, R, N, H, Dk, Dv, packed, {q_row, k_row, v_row})) return rc;
  if (H == 0 || (R == 0 && (N == 0 || !last))) return MHC_OK;
  if (!log_decay || (R && (!q || !k || !v || !o))) return null_in(who);
  const Plan plan = plan_scan(R, N, H, Dk, Dv, packed);
  if (int rc = check_workspace(who, workspace, workspace_bytes, (size_t)(plan.parts + plan.table))) return rc;
  DecayJobs jobs{};
  jobs.n = 1;
  DecayArgs& a = jobs.job[0];
  a.q = q; a.k = k; a.v = v; a.o = o; a.log_decay = log_decay; a.offsets = offsets; a.first = first; a.last = last;
  a.q_row = q_row; a.q_head = q_head; a.k_row = k_row; a.k_head = k_head; a.v_row = v_row; a.v_head = v_head;
  a.state_row = (int)Dv; a.state_col = 1;
  a.parts = (float*)workspace; a.part_row = (int)Dv; a.part_col = 1;
  a.R = R; a.N = (int)N; a.H = (int)H; a.Dk = (int)Dk; a.Dv = (int)Dv;
  a.out_scale = scale; a.in_scale = 1.f; a.lag = 1;
  return MHC_DISPATCH_DTYPE(dtype, [&]() -> int {
    const hipStream_t st = (hipStream_t)stream;
    if (int rc = set_plan(a, plan, (char*)workspace + plan.parts, who, st)) return rc;
    return scan<T>(jobs, plan, kStates | kOutputs, last != nullptr, who, st);
  });
}

// Whether scans over states of Dk x Dv and of Dv x Dk run side by side: the same kernel.
static bool alike(int64_t Dk, int64_t Dv) { return (Dk <= 64) == (Dv <= 64); }

// The states that the segments of the backward scans (dv's and dk's) leave, those of the forward where the caller did not keep
// them, and the table: it is made again, because it says where to write, and what was kept may have been changed since.
extern "C" size_t mhc_decay_attention_backward_workspace_bytes(int64_t R, int64_t N, int64_t H, int64_t Dk, int64_t Dv,
                                                               int packed, int dtype) {
  if (R < 0 || N < 0 || H <= 0 || Dk <= 0 || Dv <= 0) return 0;
  const Plan p = plan_scan(R, N, H, Dk, Dv, packed);
  return (size_t)(2 * p.parts + p.table);
}

extern "C" int mhc_decay_attention_backward(const void* q, int64_t q_row, int64_t q_head, const void* k, int64_t k_row,
                                            int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const void* dout,
                                            int64_t do_row, int64_t do_head, int dtype, const float* log_decay,
                                            const int32_t* offsets, const float* first, const float* kept,
                                            const float* d_last, void* dq, void* dk, void* dv, float* d_first, int64_t R,
                                            int64_t N, int64_t H, int64_t Dk, int64_t Dv, float scale, void* workspace,
                                            size_t workspace_bytes, mhc_stream_t stream) {
  const char* who = "decay_attention_backward";
  const bool packed = offsets || N == 0;
  if (int rc = check_decay(who, R, N, H, Dk, Dv, packed, {q_row, k_row, v_row, do_row})) return rc;
  if (H == 0 || (R == 0 && (N == 0 || !d_first))) return MHC_OK;
  if (!log_decay || (R && (!q || !k || !v || !dout))) return null_in(who);
  const bool same = alike(Dk, Dv);
  const Plan plan = plan_scan(R, N, H, Dk, Dv, packed);
  const int64_t states = (kept ? 1 : 2) * plan.parts;
  if (int rc = check_workspace(who, workspace, workspace_bytes, (size_t)(states + plan.table))) return rc;
  DecayArgs base{};
  base.log_decay = log_decay; base.offsets = offsets;
  base.R = R; base.N = (int)N; base.H = (int)H;
  const int dims[2] = {(int)Dk, (int)Dv};

  // dq: from the first token on, states transposed.  Its segments' states are the forward's.
  DecayArgs of_q = base;
  of_q.q = dout; of_q.q_row = do_row; of_q.q_head = do_head;
  of_q.k = v; of_q.k_row = v_row; of_q.k_head = v_head;
  of_q.v = k; of_q.v_row = k_row; of_q.v_head = k_head;
  of_q.o = dq; of_q.first = first; of_q.state_row = 1; of_q.state_col = dims[1];
  of_q.Dk = dims[1]; of_q.Dv = dims[0];
  of_q.out_scale = scale; of_q.in_scale = 1.f; of_q.lag = 1;
  of_q.parts = kept ? const_cast<float*>(kept) : (float*)workspace;
  of_q.part_row = kept ? 1 : dims[0]; of_q.part_col = kept ? dims[1] : 1;
  // dv and dk: from the last token back, with the same states, dk's transposed
  base.first = d_last;
  base.out_scale = 1.f; base.in_scale = scale; base.lag = 0; base.reverse = true;
  base.parts = (float*)((char*)workspace + (kept ? 0 : plan.parts));
  DecayArgs of_v = base;
  of_v.q = k; of_v.q_row = k_row; of_v.q_head = k_head;
  of_v.k = q; of_v.k_row = q_row; of_v.k_head = q_head;
  of_v.v = dout; of_v.v_row = do_row; of_v.v_head = do_head;
  of_v.o = dv; of_v.last = d_first; of_v.state_row = dims[1]; of_v.state_col = 1;
  of_v.part_row = dims[1]; of_v.part_col = 1;
  of_v.Dk = dims[0]; of_v.Dv = dims[1];
  DecayArgs of_k = base;
  of_k.q = v; of_k.q_row = v_row; of_k.q_head = v_head;
  of_k.k = dout; of_k.k_row = do_row; of_k.k_head = do_head;
  of_k.v = q; of_k.v_row = q_row; of_k.v_head = q_head;
  of_k.o = dk; of_k.state_row = 1; of_k.state_col = dims[1];
  of_k.Dk = dims[1]; of_k.Dv = dims[0];

  const bool want_q = dq && R, want_v = dv || (d_first && !dk), want_k = dk != nullptr, exact = d_first != nullptr;
  if (want_k && !want_v) of_k.last = d_first;
  return MHC_DISPATCH_DTYPE(dtype, [&]() -> int {
    const hipStream_t st = (hipStream_t)stream;
    if (int rc = set_plan(of_q, plan, (char*)workspace + states, who, st)) return rc;
    for (DecayArgs* a : {&of_v, &of_k}) {
      a->table = of_q.table;
      if (int rc = set_plan(*a, plan, nullptr, who, st)) return rc;
    }
    auto one = [&](const DecayArgs& a, int what, bool fine) {
      DecayJobs jobs{};
      jobs.n = 1;
      jobs.job[0] = a;
      return scan<T>(jobs, plan, what, fine, who, st);
    };
    if (!same) {  // each by itself; dk's states take dv's place in the workspace
      of_k.part_row = dims[0]; of_k.part_col = 1;
      if (want_q)
        if (int rc = one(of_q, kept ? kOutputs : kStates | kOutputs, false)) return rc;
      if (want_v)
        if (int rc = one(of_v, kStates | kOutputs, exact)) return rc;
      if (want_k) return one(of_k, kStates | kOutputs, of_k.last != nullptr);
      return MHC_OK;
    }
    // dv's states serve dk, transposed
    of_k.part_row = want_v ? 1 : dims[0]; of_k.part_col = want_v ? dims[1] : 1;
    if (want_q && !kept)
      if (int rc = one(of_q, kStates, false)) return rc;
    if (want_v || want_k)
      if (int rc = one(want_v ? of_v : of_k, kStates, exact)) return rc;
    DecayJobs jobs{};
    if (want_q) jobs.job[jobs.n++] = of_q;
    if (want_v) jobs.job[jobs.n++] = of_v;
    if (want_k) jobs.job[jobs.n++] = of_k;
    return jobs.n ? scan<T>(jobs, plan, kOutputs, exact, who, st) : MHC_OK;
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
