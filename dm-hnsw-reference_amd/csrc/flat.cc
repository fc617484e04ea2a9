// C entries of flat scoring (include/shine_gpu.h shine_flat_*): checks, workspaces and launches.  Kernels:
// flat_kernels.hip.  Nothing is allocated and nothing waits for the GPU here, so every entry can be captured.
#include "flat.h"

#include <algorithm>
#include <string>

#include "index_internal.h"

using namespace shine;
namespace F = shine::flat;

namespace {

// Rows of one launch (the grid's second extent ends at 65,535).  Loops over them count in 64 bits: the number behind the last
// block's first row may be 2^32.
constexpr uint32_t kRowBlock = 32768;
constexpr uint64_t kQuantizeBlock = 1 << 24;  // rows of one quantising launch (threads of a grid are a 32-bit number)
constexpr uint64_t kAlign = 256;

uint64_t aligned(uint64_t bytes) { return (bytes + kAlign - 1) & ~(kAlign - 1); }

// The call's device, and the caller's again afterwards.
struct OnDevice {
  int was = -1;
  hipError_t e;
  explicit OnDevice(int gpu) {
    e = hipGetDevice(&was);
    if (e == hipSuccess && was != gpu) e = hipSetDevice(gpu);
    else if (e == hipSuccess) was = -1;
  }
  ~OnDevice() {
    if (was >= 0) (void)hipSetDevice(was);
  }
};

int fail(const char* what) { return set_error(SHINE_ERR_ARG, what); }
int hip(const char* what, hipError_t e) {
  if (e == hipSuccess) return SHINE_OK;
  (void)hipGetLastError();  // it is reported here, and not by whoever asks for the last error next
  return set_error(SHINE_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}
bool float_elem(int e) { return e == F::kF32 || e == F::kF16 || e == F::kBF16; }
uint64_t elem_size(int e) { return e == F::kF32 ? 4 : 2; }
bool on(const void* p, uint64_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

const char* check_rows(const void* rows, int elem, uint64_t n, uint64_t width, uint64_t ld) {
  if (!float_elem(elem)) return "element type must be SHINE_ELEM_F32, _F16 or _BF16";
  if (n && width && !rows) return "NULL device pointer";
  if (ld < width && n > 1) return "row stride is shorter than a row";
  if (!on(rows, elem_size(elem))) return "a pointer is not aligned to its element type";
  return nullptr;
}

const char* check_table(const shine_flat_table* t) {
  if (!t) return "table is NULL";
  if (t->dim == 0 || t->dim > F::kMaxDim) return "dim must be in [1, 16384]";
  if (t->n > F::kMaxRecords) return "a table holds at most 2^30 records";
  if (t->n && (!t->codes || !t->scales)) return "NULL device pointer";
  if (!on(t->codes, 64) || !on(t->scales, 4) || !on(t->bias, 4)) return "table codes must be 64-byte, scales and bias 4-byte aligned";
  return nullptr;
}

const char* check_adjustment(const shine_flat_adjustment* a, uint32_t nq, uint64_t n) {
  if (a->bias && a->bias_ld && a->bias_ld < n && nq > 1) return "bias row stride is shorter than a row";
  if (a->allow && a->allow_ld && a->allow_ld < (n + 31) / 32 && nq > 1) return "allow row stride is shorter than a row";
  if (a->seen_n > F::kMaxHistory) return "seen_n must be at most 65535";
  if (a->seen_n && !a->seen) return "seen is NULL with seen_n > 0";
  if (a->seen_n && a->seen_ld && a->seen_ld < a->seen_n && nq > 1) return "seen row stride is shorter than a row";
  if (!on(a->bias, 4) || !on(a->allow, 4) || !on(a->seen, 4) || !on(a->repetition, 4) || !on(a->frequency, 4) ||
      !on(a->presence, 4))
    return "an adjustment array is not 4-byte aligned";
  return nullptr;
}

// Rows of width n that share memory without being the same rows; rows of one stride may lie between one another's.
bool tangled(const void* a, uint64_t a_ld, const void* b, uint64_t b_ld, uint64_t nq, uint64_t n, uint64_t size) {
  if (nq < 2) a_ld = b_ld = n;
  if (a == b && a_ld == b_ld) return false;
  const uint64_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  if (x + ((nq - 1) * a_ld + n) * size <= y || y + ((nq - 1) * b_ld + n) * size <= x) return false;
  if (a_ld != b_ld) return true;
  const uint64_t apart = (y > x ? y - x : x - y) % (a_ld * size);
  return apart < n * size || a_ld * size - apart < n * size;
}

F::AdjustArgs adjust_args(const shine_flat_adjustment& a, uint64_t row) {
  F::AdjustArgs r{};
  r.bias = a.bias ? a.bias + row * a.bias_ld : nullptr;
  r.bias_ld = a.bias_ld;
  r.allow = a.allow ? a.allow + row * a.allow_ld : nullptr;
  r.allow_ld = a.allow_ld;
  r.seen = a.seen_n ? a.seen + row * a.seen_ld : nullptr;
  r.seen_ld = a.seen_ld;
  r.seen_n = a.seen_n;
  r.repetition = a.repetition ? a.repetition + row : nullptr;
  r.frequency = a.frequency ? a.frequency + row : nullptr;
  r.presence = a.presence ? a.presence + row : nullptr;
  return r;
}

bool neutral(const shine_flat_adjustment* a) { return !a || (!a->bias && !a->allow && !a->seen_n); }

hipError_t quantize(const void* rows, int elem, uint64_t n, uint32_t dim, uint64_t ld, int8_t* codes, float* scales,
                    float* half_norms, hipStream_t s) {
  for (uint64_t at = 0; at < n; at += kQuantizeBlock) {
    F::QuantizeArgs a{};
    a.rows = static_cast<const char*>(rows) + at * ld * elem_size(elem);
    a.n = std::min(kQuantizeBlock, n - at);
    a.ld = ld;
    a.dim = dim;
    a.codes = codes + at * F::code_pitch(dim);
    a.scales = scales + at;
    a.half_norms = half_norms ? half_norms + at : nullptr;
    if (hipError_t e = F::launch_quantize(elem, a, s); e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Search, stepwise: blocks of rows x chunks of records whose scores fit kChunkScores, scored, adjusted and ranked.
constexpr uint64_t kChunkScores = 1ull << 26;
// Search, fused: bytes that a block of rows may take for its lists, and for its masks.
constexpr uint64_t kListBytes = 256ull << 20;
constexpr uint32_t kMaxPasses = 8;

struct SearchPlan {
  bool fused;
  uint32_t rows;       // rows of a block
  uint64_t cols;       // stepwise: records of a chunk, whole tiles of 4,096
  uint32_t chunks, slices;
  uint32_t passes;     // fused
  uint64_t stride[kMaxPasses], cap, words;
  uint64_t codes, scales, scores, keys, terms, query_terms, limit, count, mask, extra, extra_count, total;  // offsets into the workspace
};

// Fused passes cost less than the score matrix once it is larger than about 24M scores: with 128 codes and k = 10,
// 1024 x 20,000 take 51 us a call (stepwise 48), 256 x 131,072 take 47 (63), 2048 x 20,000 take 69 (79), 1024 x 65,536 take 62
// (133); with few queries the table is read more often than the matrix would be (16 x 1M: 58 and 58, 8 x 1M: 57 and 48).  A
// bias for each row is as large as the matrix itself, and wide rows' queries do not fit the registers: these are searched
// stepwise.
constexpr uint64_t kFusedScores = 24u << 20;
SearchPlan plan_search(uint32_t nq, uint64_t n, uint32_t dim, uint32_t k, const shine_flat_adjustment* a) {
  SearchPlan p{};
  const uint32_t pitch = F::code_pitch(dim), seen_n = a ? a->seen_n : 0;
  p.fused = nq > 16 && nq * n > kFusedScores && pitch <= F::kMaxFusedPitch && seen_n <= F::kMaxSeen &&
            !(a && a->bias && a->bias_ld);
  p.rows = std::min(std::max(nq, 1u), 2048u);
  uint64_t at = 0;
  auto take = [&at](uint64_t bytes) {
    const uint64_t here = at;
    at += aligned(bytes);
    return here;
  };
  if (p.fused) {
    // Blocks of the coarsest pass: 256 where a short list of 128 would take a pass more (256 x 200k x 200, k = 10: 56 us, with
    // 128 66) and for long answers (1024 x 2M x 64, k = 100: 505 us, 547), else 128 (1024 x 1M x 128, k = 10: 219 us, 226).
    const uint64_t blocks = (n + 31) / 32, coarse = k > 64 || (blocks > 128 * 32 && blocks <= 256 * 32) ? 256 : 128;
    uint64_t ratio = 1;
    if (blocks <= 256) {
      p.passes = 1;
      p.stride[0] = 1;
    } else {
      // each pass at most 32 times the one before: its list then holds about 32 k keys
      const uint64_t s0 = (blocks + coarse - 1) / coarse;
      uint32_t steps = 1;
      for (ratio = s0; ratio > 32; ++steps) {
        ratio = 2;
        auto power = [&](uint64_t r) {
          uint64_t v = 1;
          for (uint32_t i = 0; i < steps + 1; ++i) v *= r;
          return v;
        };
        while (power(ratio) < s0) ++ratio;
      }
      p.passes = steps + 1;
      p.stride[0] = s0;
      uint64_t v = 1;
      for (uint32_t i = 0; i < steps; ++i, v *= ratio) p.stride[steps - i] = v;
    }
    p.cap = std::max<uint64_t>((blocks + p.stride[0] - 1) / p.stride[0] * 32, p.passes > 1 ? 2 * k * ratio + 1024 : 0);
    p.words = blocks;
    p.rows = std::min<uint64_t>(p.rows, std::max<uint64_t>(128, kListBytes / (8 * p.cap) / 128 * 128));
    if (seen_n) p.rows = std::min<uint64_t>(p.rows, std::max<uint64_t>(32, kListBytes / (4 * p.words) / 32 * 32));
  } else {
    p.cols = std::max<uint64_t>(4096, kChunkScores / p.rows / 4096 * 4096);
    p.cols = std::min(p.cols, std::max<uint64_t>(1, n));
    p.chunks = static_cast<uint32_t>((n + p.cols - 1) / p.cols);
    p.slices = F::topk_slices(p.rows, p.cols);
  }
  p.codes = take(static_cast<uint64_t>(p.rows) * pitch);
  p.scales = take(4ull * p.rows);
  if (p.fused) {
    p.keys = take(8 * p.cap * p.rows);
    if (p.passes > 1) p.terms = take(F::kTermBytes * 32ull * p.words);
    p.query_terms = take(static_cast<uint64_t>(F::kTermBytes) * p.rows);
    p.limit = take(4ull * p.rows);
    p.count = take(4ull * F::kCountStride * p.rows);
    if (seen_n) {
      p.mask = take(4 * p.words * p.rows);
      p.extra = take(8ull * seen_n * p.rows);
      p.extra_count = take(4ull * p.rows);
    }
  } else {
    p.scores = take(4ull * p.rows * p.cols);
    p.keys = take(8ull * p.rows * p.chunks * p.slices * k);
  }
  p.total = at;
  return p;
}

hipError_t search_fused(const SearchPlan& p, const shine_flat_table& t, const shine_flat_adjustment* a, uint64_t q,
                        uint32_t m, uint32_t k, char* ws, float* values, int32_t* ids, hipStream_t s) {
  F::PassArgs pass{};
  pass.qcodes = reinterpret_cast<int8_t*>(ws + p.codes);
  pass.qscales = reinterpret_cast<float*>(ws + p.scales);
  pass.codes = t.codes;
  pass.scales = t.scales;
  pass.tbias = t.bias;
  pass.nq = m;
  pass.pitch = F::code_pitch(t.dim);
  pass.n = t.n;
  pass.record_terms = ws + p.terms;
  pass.query_terms = ws + p.query_terms;
  pass.limit = reinterpret_cast<int32_t*>(ws + p.limit);
  pass.count = reinterpret_cast<uint32_t*>(ws + p.count);
  pass.keys = reinterpret_cast<uint64_t*>(ws + p.keys);
  pass.cap = p.cap;
  F::SelectArgs sel{};
  if (a) {
    const F::AdjustArgs r = adjust_args(*a, q);
    pass.abias = r.bias;
    pass.allow = r.allow;
    pass.allow_ld = r.allow_ld;
    if (r.seen) {
      F::SeenArgs seen{};
      seen.pass = pass;
      seen.seen = r.seen;
      seen.seen_ld = r.seen_ld;
      seen.seen_n = r.seen_n;
      seen.repetition = r.repetition;
      seen.frequency = r.frequency;
      seen.presence = r.presence;
      seen.mask = reinterpret_cast<uint32_t*>(ws + p.mask);
      seen.mask_ld = p.words;
      seen.extra = reinterpret_cast<uint64_t*>(ws + p.extra);
      seen.extra_count = reinterpret_cast<uint32_t*>(ws + p.extra_count);
      seen.extra_ld = r.seen_n;
      if (hipError_t e = F::launch_seen(seen, s); e != hipSuccess) return e;
      pass.allow = seen.mask;
      pass.allow_ld = seen.mask_ld;
      sel.extra = seen.extra;
      sel.extra_count = seen.extra_count;
      sel.extra_ld = seen.extra_ld;
    }
  }
  const uint64_t* extra = sel.extra;
  for (uint32_t i = 0; i < p.passes; ++i) {
    const bool last = i + 1 == p.passes;
    pass.stride = p.stride[i];
    pass.blocks = (p.words + pass.stride - 1) / pass.stride;
    if (hipError_t e = i ? F::launch_pass(pass, s) : F::launch_sample(pass, s); e != hipSuccess) return e;
    sel.pass = pass;
    sel.k = k;
    sel.sample = i == 0;
    sel.terms = i == 0 && !last && q == 0;  // the same for all blocks of rows
    sel.extra = last ? extra : nullptr;
    sel.last = last;
    sel.values = values;
    sel.ids = ids;
    if (hipError_t e = F::launch_select(sel, s); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

extern "C" {

uint32_t shine_flat_pitch(uint32_t dim) { return F::code_pitch(dim); }

int shine_flat_quantize(int gpu_id, const void* d_rows, int elem, uint64_t n, uint32_t dim, uint64_t ld, int8_t* d_codes,
                        float* d_scales, float* d_half_norms, void* stream) {
  if (dim == 0 || dim > F::kMaxDim) return fail("dim must be in [1, 16384]");
  if (const char* w = check_rows(d_rows, elem, n, dim, ld)) return fail(w);
  if (n == 0) return SHINE_OK;
  if (!d_codes || !d_scales) return fail("NULL device pointer");
  if (!on(d_codes, 8) || !on(d_scales, 4) || !on(d_half_norms, 4)) return fail("codes must be 8-byte, scales and norms 4-byte aligned");
  OnDevice dev(gpu_id);
  if (dev.e != hipSuccess) return hip("flat quantize: device", dev.e);
  return hip("flat quantize", quantize(d_rows, elem, n, dim, ld, d_codes, d_scales, d_half_norms, static_cast<hipStream_t>(stream)));
}

uint64_t shine_flat_scores_workspace(uint32_t nq, uint64_t n, uint32_t dim) {
  if (F::scores_from_rows(nq, F::code_pitch(dim))) return 0;
  const uint64_t rows = std::min(nq, kRowBlock);
  return aligned(rows * F::code_pitch(dim)) + aligned(4 * rows);
}

int shine_flat_scores(int gpu_id, const shine_flat_table* table, const void* d_queries, int elem, uint32_t nq, uint64_t ld,
                      void* d_out, int out_elem, uint64_t out_ld, void* d_workspace, uint64_t workspace_bytes, void* stream) {
  if (const char* w = check_table(table)) return fail(w);
  if (const char* w = check_rows(d_queries, elem, nq, table->dim, ld)) return fail(w);
  if (nq == 0 || table->n == 0) return SHINE_OK;
  if (const char* w = check_rows(d_out, out_elem, nq, table->n, out_ld)) return fail(w);
  const uint64_t need = shine_flat_scores_workspace(nq, table->n, table->dim);
  if (need && (!d_workspace || !on(d_workspace, kAlign) || workspace_bytes < need))
    return fail("workspace is missing, not 256-byte aligned or smaller than shine_flat_scores_workspace");
  OnDevice dev(gpu_id);
  if (dev.e != hipSuccess) return hip("flat scores: device", dev.e);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t pitch = F::code_pitch(table->dim);
  const uint64_t rows = std::min(nq, kRowBlock);
  F::ScoresArgs a{};
  a.codes = table->codes;
  a.scales = table->scales;
  a.bias = table->bias;
  a.pitch = pitch;
  a.n = table->n;
  a.ld = out_ld;
  if (need == 0) {
    a.nq = nq;
    a.out = d_out;
    a.queries = d_queries;
    a.queries_ld = ld;
    a.dim = table->dim;
    return hip("flat scores", F::launch_scores_of_rows(elem, out_elem, a, s));
  }
  int8_t* codes = static_cast<int8_t*>(d_workspace);
  float* scales = reinterpret_cast<float*>(codes + aligned(rows * pitch));
  a.qcodes = codes;
  a.qscales = scales;
  for (uint64_t q = 0; q < nq; q += kRowBlock) {
    const uint32_t m = static_cast<uint32_t>(std::min<uint64_t>(kRowBlock, nq - q));
    if (hipError_t e = quantize(static_cast<const char*>(d_queries) + q * ld * elem_size(elem), elem, m, table->dim, ld,
                                codes, scales, nullptr, s); e != hipSuccess)
      return hip("flat scores", e);
    a.nq = m;
    a.out = static_cast<char*>(d_out) + q * out_ld * elem_size(out_elem);
    if (hipError_t e = F::launch_scores(out_elem, a, s); e != hipSuccess) return hip("flat scores", e);
  }
  return SHINE_OK;
}

int shine_flat_adjust(int gpu_id, const void* d_scores, int elem, uint32_t nq, uint64_t n, uint64_t ld,
                      const shine_flat_adjustment* adjustment, void* d_out, uint64_t out_ld, void* stream) {
  if (!adjustment) return fail("adjustment is NULL");
  if (n > F::kMaxRecords) return fail("a row holds at most 2^30 scores");
  if (const char* w = check_rows(d_scores, elem, nq, n, ld)) return fail(w);
  if (const char* w = check_adjustment(adjustment, nq, n)) return fail(w);
  if (nq == 0 || n == 0) return SHINE_OK;
  if (const char* w = check_rows(d_out, elem, nq, n, out_ld)) return fail(w);
  if (tangled(d_scores, ld, d_out, out_ld, nq, n, elem_size(elem)))
    return fail("out overlaps the scores without being the same rows");
  OnDevice dev(gpu_id);
  if (dev.e != hipSuccess) return hip("flat adjust: device", dev.e);
  for (uint64_t q = 0; q < nq; q += kRowBlock) {
    F::AdjustArgs a = adjust_args(*adjustment, q);
    a.scores = static_cast<const char*>(d_scores) + q * ld * elem_size(elem);
    a.out = static_cast<char*>(d_out) + q * out_ld * elem_size(elem);
    a.ld = ld;
    a.out_ld = out_ld;
    a.nq = static_cast<uint32_t>(std::min<uint64_t>(kRowBlock, nq - q));
    a.n = n;
    if (hipError_t e = F::launch_adjust(elem, a, static_cast<hipStream_t>(stream)); e != hipSuccess) return hip("flat adjust", e);
  }
  return SHINE_OK;
}

uint64_t shine_flat_topk_workspace(uint32_t nq, uint64_t n, uint32_t k) {
  const uint32_t rows = std::min(std::max(nq, 1u), kRowBlock), slices = F::topk_slices(rows, n);
  return slices > 1 ? aligned(8ull * rows * slices * k) : 0;
}

int shine_flat_topk(int gpu_id, const void* d_scores, int elem, uint32_t nq, uint64_t n, uint64_t ld, uint32_t k,
                    void* d_values, int32_t* d_ids, void* d_workspace, uint64_t workspace_bytes, void* stream) {
  if (k == 0 || k > F::kMaxK) return fail("k must be in [1, 256]");
  if (n > F::kMaxRecords) return fail("a row holds at most 2^30 scores");
  if (const char* w = check_rows(d_scores, elem, nq, n, ld)) return fail(w);
  if (nq == 0) return SHINE_OK;
  if (!d_values || !d_ids) return fail("NULL device pointer");
  if (!on(d_values, elem_size(elem)) || !on(d_ids, 4)) return fail("a pointer is not aligned to its element type");
  const uint64_t need = shine_flat_topk_workspace(nq, n, k);
  if (need && (!d_workspace || !on(d_workspace, kAlign) || workspace_bytes < need))
    return fail("workspace is missing, not 256-byte aligned or smaller than shine_flat_topk_workspace");
  OnDevice dev(gpu_id);
  if (dev.e != hipSuccess) return hip("flat topk: device", dev.e);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t slices = F::topk_slices(std::min(nq, kRowBlock), n);
  for (uint64_t q = 0; q < nq; q += kRowBlock) {
    F::TopkArgs a{};
    a.scores = static_cast<const char*>(d_scores) + q * ld * elem_size(elem);
    a.ld = ld;
    a.nq = static_cast<uint32_t>(std::min<uint64_t>(kRowBlock, nq - q));
    a.k = k;
    a.n = n;
    a.slices = slices;
    a.keys = static_cast<uint64_t*>(d_workspace);
    a.key_ld = slices;
    a.values = static_cast<char*>(d_values) + q * k * elem_size(elem);
    a.ids = d_ids + q * k;
    if (hipError_t e = F::launch_topk(elem, false, a, s); e != hipSuccess) return hip("flat topk", e);
    if (slices > 1) {
      F::MergeArgs m{a.keys, static_cast<uint64_t>(slices) * k, a.nq, k, a.values, a.ids};
      if (hipError_t e = F::launch_merge(elem, m, s); e != hipSuccess) return hip("flat topk", e);
    }
  }
  return SHINE_OK;
}

uint64_t shine_flat_search_workspace(uint32_t nq, uint64_t n, uint32_t dim, uint32_t k,
                                     const shine_flat_adjustment* adjustment) {
  // what shine_flat_search refuses: a plan has room for the passes over kMaxRecords records
  if (n > F::kMaxRecords || dim == 0 || dim > F::kMaxDim || k == 0 || k > F::kMaxK) return 0;
  return plan_search(nq, n, dim, k, adjustment).total;
}

int shine_flat_search(int gpu_id, const shine_flat_table* table, const void* d_queries, int elem, uint32_t nq, uint64_t ld,
                      uint32_t k, const shine_flat_adjustment* adjustment, float* d_values, int32_t* d_ids,
                      void* d_workspace, uint64_t workspace_bytes, void* stream) {
  if (const char* w = check_table(table)) return fail(w);
  if (k == 0 || k > F::kMaxK) return fail("k must be in [1, 256]");
  if (const char* w = check_rows(d_queries, elem, nq, table->dim, ld)) return fail(w);
  if (adjustment)
    if (const char* w = check_adjustment(adjustment, nq, table->n)) return fail(w);
  if (nq == 0) return SHINE_OK;
  if (!d_values || !d_ids) return fail("NULL device pointer");
  if (!on(d_values, 4) || !on(d_ids, 4)) return fail("a pointer is not aligned to its element type");
  const SearchPlan p = plan_search(nq, table->n, table->dim, k, adjustment);
  if (!d_workspace || !on(d_workspace, kAlign) || workspace_bytes < p.total)
    return fail("workspace is missing, not 256-byte aligned or smaller than shine_flat_search_workspace");
  OnDevice dev(gpu_id);
  if (dev.e != hipSuccess) return hip("flat search: device", dev.e);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t pitch = F::code_pitch(table->dim);
  char* ws = static_cast<char*>(d_workspace);
  for (uint64_t q = 0; q < nq; q += p.rows) {
    const uint32_t m = static_cast<uint32_t>(std::min<uint64_t>(p.rows, nq - q));
    const char* rows = static_cast<const char*>(d_queries) + q * ld * elem_size(elem);
    const bool from_rows = !p.fused && F::scores_from_rows(m, pitch);
    if (!from_rows)
      if (hipError_t e = quantize(rows, elem, m, table->dim, ld, reinterpret_cast<int8_t*>(ws + p.codes),
                                  reinterpret_cast<float*>(ws + p.scales), nullptr, s); e != hipSuccess)
        return hip("flat search", e);
    if (p.fused) {
      if (hipError_t e = search_fused(p, *table, adjustment, q, m, k, ws, d_values + q * k, d_ids + q * k, s); e != hipSuccess)
        return hip("flat search", e);
      continue;
    }
    for (uint32_t c = 0; c < p.chunks; ++c) {
      const uint64_t first = c * p.cols, cols = std::min(p.cols, table->n - first);
      F::ScoresArgs a{};
      a.qcodes = reinterpret_cast<int8_t*>(ws + p.codes);
      a.qscales = reinterpret_cast<float*>(ws + p.scales);
      a.codes = table->codes + first * pitch;
      a.scales = table->scales + first;
      a.bias = table->bias ? table->bias + first : nullptr;
      a.nq = m;
      a.pitch = pitch;
      a.n = cols;
      a.out = ws + p.scores;
      a.ld = p.cols;
      a.queries = rows;
      a.queries_ld = ld;
      a.dim = table->dim;
      if (hipError_t e = from_rows ? F::launch_scores_of_rows(elem, F::kF32, a, s) : F::launch_scores(F::kF32, a, s);
          e != hipSuccess)
        return hip("flat search", e);
      if (!neutral(adjustment)) {
        F::AdjustArgs b = adjust_args(*adjustment, q);
        b.scores = b.out = a.out;
        b.ld = b.out_ld = p.cols;
        b.nq = m;
        b.n = cols;
        b.first = first;
        if (hipError_t e = F::launch_adjust(F::kF32, b, s); e != hipSuccess) return hip("flat search", e);
      }
      F::TopkArgs t{};
      t.scores = a.out;
      t.ld = p.cols;
      t.nq = m;
      t.k = k;
      t.n = cols;
      t.first = first;
      t.slices = p.slices;
      t.keys = reinterpret_cast<uint64_t*>(ws + p.keys) + static_cast<uint64_t>(c) * p.slices * k;
      t.key_ld = p.chunks * p.slices;
      if (hipError_t e = F::launch_topk(F::kF32, true, t, s); e != hipSuccess) return hip("flat search", e);
    }
    F::MergeArgs g{reinterpret_cast<uint64_t*>(ws + p.keys), static_cast<uint64_t>(p.chunks) * p.slices * k, m, k,
                   d_values + q * k, d_ids + q * k};
    if (hipError_t e = F::launch_merge(F::kF32, g, s); e != hipSuccess) return hip("flat search", e);
  }
  return SHINE_OK;
}

}  // extern "C"
