// Shared by the autoregressive-decoding operators: element types and the checks of their structs.
#pragma once
#include <cstdint>

#include "common.h"
#include "decode_overlap.h"
#include "decode_places.h"

namespace ttsamd {

inline int elem_bytes(int dtype) { return dtype == TTSAMD_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == TTSAMD_F32 || dtype == TTSAMD_F16 || dtype == TTSAMD_BF16; }

// Host-side checks of the two structs every cache operator takes; 0 or a negative error code.
int check_paged_kv(const char *what, const ttsamd_paged_kv *c);
int check_paged_batch(const char *what, const ttsamd_paged_batch *b, int tokens);

// A tensor of a call [tokens][heads][dim], strides in elements.
inline RowSet rows_of(const void *at, int64_t t, int64_t h, int64_t tokens, int64_t heads, int64_t dim, int dtype)
{
    const int64_t es = elem_bytes(dtype);
    return RowSet{at, t * es, h * es, tokens, heads, dim * es};
}
// 0, or an error where rows that are written share memory with each other or with rows that are read (`in_place`: other than being these).
int check_written(const char *what, const char *name, const RowSet &out, const char *from, const RowSet &in, bool in_place);

#if defined(__HIPCC__)
template <class T> __device__ __forceinline__ float to_f(T x) { return static_cast<float>(x); }
#endif
}  // namespace ttsamd
