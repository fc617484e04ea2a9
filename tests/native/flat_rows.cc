// The C entries of flat scoring (csrc/flat.cc) over as many rows as a call can name, with launches that only count: every
// row is launched once and the loop over blocks of rows ends.
#include <cstdio>

#include "flat.h"
#include "index_internal.h"

namespace {
constexpr uint32_t kRows = 0xFFFFFFFFu;
uint64_t quantised, scored, adjusted, ranked, merged, sampled, selected, launches;
hipError_t launched() { return ++launches > 30'000'000 ? hipErrorUnknown : hipSuccess; }  // an endless loop ends too
}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "too many launches"; }
}

namespace shine {
int set_error(int code, const std::string& what) {
  std::printf("error %d: %s\n", code, what.c_str());
  return code;
}
namespace flat {
uint32_t topk_slices(uint32_t, uint64_t) { return 1; }
hipError_t launch_quantize(int, const QuantizeArgs& a, hipStream_t) { return quantised += a.n, launched(); }
hipError_t launch_scores(int, const ScoresArgs& a, hipStream_t) { return scored += a.nq, launched(); }
hipError_t launch_scores_of_rows(int, int, const ScoresArgs& a, hipStream_t) { return scored += a.nq, launched(); }
hipError_t launch_sample(const PassArgs& a, hipStream_t) { return sampled += a.nq, launched(); }
hipError_t launch_pass(const PassArgs&, hipStream_t) { return launched(); }
hipError_t launch_select(const SelectArgs& a, hipStream_t) { return selected += a.pass.nq, launched(); }
hipError_t launch_seen(const SeenArgs&, hipStream_t) { return launched(); }
hipError_t launch_adjust(int, const AdjustArgs& a, hipStream_t) { return adjusted += a.nq, launched(); }
hipError_t launch_topk(int, bool, const TopkArgs& a, hipStream_t) { return ranked += a.nq, launched(); }
hipError_t launch_merge(int, const MergeArgs& a, hipStream_t) { return merged += a.nq, launched(); }
}  // namespace flat
}  // namespace shine

namespace {
bool all(const char* what, int rc, std::initializer_list<uint64_t> counts) {
  bool ok = rc == SHINE_OK;
  for (uint64_t c : counts) ok = ok && c == kRows;
  std::printf("%s: rc %d, %llu launches%s\n", what, rc, static_cast<unsigned long long>(launches), ok ? "" : ", WRONG");
  quantised = scored = adjusted = ranked = merged = sampled = selected = launches = 0;
  return ok;
}
}  // namespace

int main() {
  char* const p = reinterpret_cast<char*>(1ull << 40);  // addresses that nobody reads
  auto* codes = reinterpret_cast<int8_t*>(p);
  auto* floats = reinterpret_cast<float*>(p);
  auto* ids = reinterpret_cast<int32_t*>(p);
  const uint64_t room = 1ull << 50;
  const shine_flat_table narrow{codes, floats, nullptr, 1, 32, 0}, wide{codes, floats, nullptr, 1, 300, 0};
  const shine_flat_adjustment none{};
  bool ok = true;
  int rc = shine_flat_scores(0, &narrow, p, SHINE_ELEM_F32, kRows, 32, p, SHINE_ELEM_F32, 1, p, room, nullptr);
  ok = all("scores", rc, {quantised, scored}) && ok;
  rc = shine_flat_adjust(0, p, SHINE_ELEM_F32, kRows, 1, 1, &none, p, 1, nullptr);
  ok = all("adjust", rc, {adjusted}) && ok;
  rc = shine_flat_topk(0, p, SHINE_ELEM_F32, kRows, 1, 1, 1, p, ids, p, room, nullptr);
  ok = all("topk", rc, {ranked}) && ok;
  rc = shine_flat_search(0, &narrow, p, SHINE_ELEM_F32, kRows, 32, 1, nullptr, floats, ids, p, room, nullptr);
  ok = all("search in passes", rc, {quantised, sampled, selected}) && ok;
  rc = shine_flat_search(0, &wide, p, SHINE_ELEM_F32, kRows, 300, 1, nullptr, floats, ids, p, room, nullptr);
  ok = all("search by way of the matrix", rc, {quantised, scored, ranked, merged}) && ok;
  std::printf(ok ? "rows ok\n" : "rows wrong\n");
  return ok ? 0 : 1;
}
