#include "paged_start.h"

namespace ttsamd {
hipError_t start_f16(const AttArgs &g, const PagedLaunch &p, hipStream_t st) { return start_paged<_Float16>(g, p, st); }
void join_f16(const AttArgs &g, hipStream_t st) { join_paged<_Float16>(g, st); }
}  // namespace ttsamd
