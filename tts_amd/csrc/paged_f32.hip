#include "paged_start.h"

namespace ttsamd {
hipError_t start_f32(const AttArgs &g, const PagedLaunch &p, hipStream_t st) { return start_paged<float>(g, p, st); }
void join_f32(const AttArgs &g, hipStream_t st) { join_paged<float>(g, st); }
}  // namespace ttsamd
