// Products of a few rows with 4-bit weights: y[m,n] = sum_g s[n,g] sum_{k in g} x[m,k] (level[n,k] - z[n,g]) + bias[n].
// A wave per output column and row: lanes walk the 32-bit words of eight levels, the group's scale on each word's sum.
#include "decode_common.h"

namespace ttsamd {
namespace {

template <class T> __device__ __forceinline__ float ld(const void *p, int64_t i) { return to_f(((const T *)p)[i]); }
__device__ __forceinline__ float ld_any(const void *p, int64_t i, int dtype)
{
    return dtype == TTSAMD_F32 ? ld<float>(p, i) : dtype == TTSAMD_F16 ? ld<_Float16>(p, i) : ld<__bf16>(p, i);
}

template <class T> __global__ __launch_bounds__(64) void linear_w4(ttsamd_linear_w4_args a)
{
    const int n = blockIdx.x, lane = threadIdx.x, kt = (a.k + 127) / 128, groups = kt * (128 / a.group);
    for (int m = blockIdx.y; m < a.m; m += gridDim.y) {
        const T *x = (const T *)a.x + m * a.x_stride;
        float acc = 0.f;
        for (int w = lane; w < a.k / 8; w += 64) {
            const int c = w >> 4, j = (w >> 2) & 3, g = w & 3;
            const uint32_t word = a.levels[(((int64_t)(n >> 4) * kt + c) * 4 + g) * 64 + (n & 15) * 4 + j];
            const int64_t sg = ((int64_t)(n >> 4) * groups + w * 8 / a.group) * 16 + (n & 15);
            const float z = a.zeros ? (float)a.zeros[sg] : 8.f;
            float part = 0.f;
            for (int e = 0; e < 8; ++e) part = fmaf(to_f(x[w * 8 + e]), (float)((word >> (4 * e)) & 15) - z, part);
            acc = fmaf(part, ld_any(a.scales, sg, a.scale_dtype), acc);
        }
        for (int s = 32; s; s >>= 1) acc += __shfl_xor(acc, s);
        if (lane == 0) ((T *)a.y)[m * a.y_stride + n] = (T)(acc + (a.bias ? ld<T>(a.bias, n) : 0.f));
    }
}

}  // namespace
}  // namespace ttsamd

extern "C" int ttsamd_linear_w4(const ttsamd_linear_w4_args *a, void *stream)
{
    using namespace ttsamd;
    TTSAMD_CHECK_ARG(a, "linear_w4: arguments are NULL");
    TTSAMD_CHECK_ARG(known_dtype(a->dtype) && known_dtype(a->scale_dtype), "linear_w4: unknown element type");
    TTSAMD_CHECK_ARG(a->m >= 0 && a->n >= 0 && a->k >= 0, "linear_w4: negative size");
    if (a->group != 32 && a->group != 64 && a->group != 128) {
        set_error("linear_w4: groups of %d (32, 64 or 128)", a->group);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    TTSAMD_CHECK_ARG(a->k > 0 && a->k % a->group == 0, "linear_w4: k = %d is not a multiple of the group %d", a->k, a->group);
    if (a->m == 0 || a->n == 0) return TTSAMD_OK;
    TTSAMD_CHECK_ARG(a->x && a->y && a->levels && a->scales, "linear_w4: a tensor is NULL");
    TTSAMD_CHECK_ARG((((uintptr_t)a->levels | (uintptr_t)a->scales | (uintptr_t)a->zeros) & 15) == 0,
                     "linear_w4: levels, scales and zeros start at multiples of 16 bytes");
    const dim3 grid(a->n, a->m < 65535 ? a->m : 65535);
    hipStream_t st = as_stream(stream);
    if (a->dtype == TTSAMD_F32) linear_w4<float><<<grid, 64, 0, st>>>(*a);
    else if (a->dtype == TTSAMD_F16) linear_w4<_Float16><<<grid, 64, 0, st>>>(*a);
    else linear_w4<__bf16><<<grid, 64, 0, st>>>(*a);
    TTSAMD_LAUNCH_CHECK();
    return TTSAMD_OK;
}
