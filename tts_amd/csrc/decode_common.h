// Shared by the autoregressive-decoding operators: element types and the checks of their structs.
#pragma once
#include <cstdint>

#include "common.h"
#include "decode_places.h"

namespace ttsamd {

inline int elem_bytes(int dtype) { return dtype == TTSAMD_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == TTSAMD_F32 || dtype == TTSAMD_F16 || dtype == TTSAMD_BF16; }

// Host-side checks of the two structs every cache operator takes; 0 or a negative error code.
int check_paged_kv(const char *what, const ttsamd_paged_kv *c);
int check_paged_batch(const char *what, const ttsamd_paged_batch *b, int tokens);

#if defined(__HIPCC__)
template <class T> __device__ __forceinline__ float to_f(T x) { return static_cast<float>(x); }
#endif
}  // namespace ttsamd
