#include "paged_start.h"

namespace ttsamd {
hipError_t start_bf16(const AttArgs &g, const PagedLaunch &p, hipStream_t st) { return start_paged<__bf16>(g, p, st); }
void join_bf16(const AttArgs &g, hipStream_t st) { join_paged<__bf16>(g, st); }
}  // namespace ttsamd
