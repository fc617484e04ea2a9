// Flat scoring: internal interface between the C entries (flat.cc) and the kernels (flat_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace shine::flat {

constexpr uint32_t kMaxDim = 16384;   // sums of dim products of 8-bit codes stay below 2^31 (16384 * 127^2 = 2.6e8)
constexpr uint32_t kMaxK = 256;       // answers of a top-k
constexpr uint64_t kMaxRecords = 1ull << 30;  // ids are int32, a grid's threads a 32-bit number

// bytes of a row of codes: whole 64-byte steps of the matrix instructions, zero behind dim
inline uint32_t code_pitch(uint32_t dim) { return (dim + 63u) & ~63u; }

enum Elem { kF32 = 0, kF16 = 1, kBF16 = 5 };  // SHINE_ELEM_F32 / _F16 / _BF16

struct QuantizeArgs {
  const void* rows;
  uint64_t n, ld;  // ld in elements
  uint32_t dim;
  int8_t* codes;
  float* scales;
  float* half_norms;  // nullable
};

struct ScoresArgs {
  const int8_t* qcodes;
  const float* qscales;
  const int8_t* codes;
  const float* scales;
  const float* bias;  // nullable
  uint32_t nq, pitch;
  uint64_t n;    // records of this launch
  void* out;
  uint64_t ld;   // in elements
  // scores_of_rows: instead of qcodes and qscales
  const void* queries;
  uint64_t queries_ld;
  uint32_t dim;
};
// Few queries are quantised in the launch that scores them (with 128 codes, 1 x 20,000: 8.6 us a call, 13.4 in two launches;
// 16 x 1M: 33.9 and 37.3).
inline bool scores_from_rows(uint32_t nq, uint32_t pitch) { return nq <= 16 && pitch <= 256; }

constexpr uint32_t kCountStride = 32;  // queries' counts lie in memory lines of their own: all XCDs add to them
constexpr uint32_t kTermBytes = 16;    // of a record or a query in the threshold test

// One pass of a fused search over every `stride`-th block of 32 records.
struct PassArgs {
  const int8_t* qcodes;
  const float* qscales;
  const int8_t* codes;
  const float* scales;
  const float* tbias;     // nullable: the table's
  const float* abias;     // nullable: the adjustment's, shared by all queries
  const uint32_t* allow;  // nullable; word w of query q at q * allow_ld + w
  uint64_t allow_ld;
  uint32_t nq, pitch;
  uint64_t n;
  uint64_t blocks;        // ceil(ceil(n / 32) / stride): blocks of this pass
  uint64_t stride;
  // the coarsest pass: every key at keys[q * cap + 32 * block + i]
  uint64_t* keys;
  uint64_t cap;
  // the others: the keys of what reaches the threshold, or lies a little below it, at keys[q * cap + 0 .. count - 1]
  void* record_terms;        // of all records, whole blocks
  void* query_terms;
  int32_t* limit;            // per query
  uint32_t* count;           // query q's at q * kCountStride (may pass cap; the list then holds cap keys)
};

// Selection from a search's lists: the k-th best key between passes, the answers behind the last one.
struct SelectArgs {
  PassArgs pass;          // what a row's scores are computed with
  uint32_t k;
  bool sample;            // every list holds `blocks` x 32 keys; else count[q]
  const uint64_t* extra;  // nullable: extra_count[q] more keys at extra + q * extra_ld
  const uint32_t* extra_count;
  uint64_t extra_ld;
  bool terms;             // write pass.record_terms beside it, as a shared allow, scales and biases have them
  bool last;              // write the answers; else thr, limit and query_terms, and clear count
  float* values;
  int32_t* ids;
};

// A history's records: taken out of the row's mask, and scored with their penalties.
struct SeenArgs {
  PassArgs pass;          // its allow (nullable) is the caller's
  const int32_t* seen;
  uint64_t seen_ld;
  uint32_t seen_n;
  const float *repetition, *frequency, *presence;
  uint32_t* mask;         // nq rows of mask_ld words
  uint64_t mask_ld;
  uint64_t* extra;
  uint32_t* extra_count;
  uint64_t extra_ld;
};
constexpr uint32_t kMaxHistory = 65535;    // longest history (its counts are 16-bit numbers)
constexpr uint32_t kMaxSeen = 4096;       // longest history of a fused search (its ids are sorted in LDS)
constexpr uint32_t kMaxFusedPitch = 256;  // widest rows of a fused search (the queries' codes stay in registers)

struct AdjustArgs {
  const void* scores;
  void* out;
  uint64_t ld, out_ld;
  uint32_t nq;
  uint64_t n;             // columns of this launch
  uint64_t first;         // record of its first column
  const float* bias;      // nullable; record j of row i at bias[i * bias_ld + j]
  uint64_t bias_ld;
  const uint32_t* allow;  // nullable; record j of row i: bit j % 32 of allow[i * allow_ld + j / 32]
  uint64_t allow_ld;
  const int32_t* seen;    // nullable
  uint64_t seen_ld;
  uint32_t seen_n;
  const float *repetition, *frequency, *presence;  // each nullable
};

struct TopkArgs {
  const void* scores;
  uint64_t ld;
  uint32_t nq, k;
  uint64_t n;       // columns of this launch
  uint64_t first;   // record of its first column
  uint32_t slices;  // workgroups per row
  uint64_t* keys;   // slices > 1 or keys_only: k keys of every (row, slice) at (row * key_ld + slice) * k
  uint32_t key_ld;
  void* values;
  int32_t* ids;
};

struct MergeArgs {
  const uint64_t* keys;  // per row: count keys
  uint64_t count;
  uint32_t nq, k;
  void* values;
  int32_t* ids;
};

uint32_t topk_slices(uint32_t nq, uint64_t n);

hipError_t launch_quantize(int elem, const QuantizeArgs& a, hipStream_t s);
hipError_t launch_scores(int out_elem, const ScoresArgs& a, hipStream_t s);
hipError_t launch_sample(const PassArgs& a, hipStream_t s);
hipError_t launch_pass(const PassArgs& a, hipStream_t s);
hipError_t launch_select(const SelectArgs& a, hipStream_t s);
hipError_t launch_seen(const SeenArgs& a, hipStream_t s);
hipError_t launch_scores_of_rows(int elem, int out_elem, const ScoresArgs& a, hipStream_t s);
hipError_t launch_adjust(int elem, const AdjustArgs& a, hipStream_t s);
hipError_t launch_topk(int elem, bool keys_only, const TopkArgs& a, hipStream_t s);
hipError_t launch_merge(int elem, const MergeArgs& a, hipStream_t s);

}  // namespace shine::flat
