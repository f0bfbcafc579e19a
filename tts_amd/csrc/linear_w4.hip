// Products of a few rows with 4-bit weights: y[m,n] = sum_g s[n,g] sum_{k in g} x[m,k] (level[n,k] - z[n,g]) + bias[n].
//
// Mathematics.  A level q becomes a 16-bit float without arithmetic: its four bits put into the top of the mantissa of 16.0 give 16 + q,
// exact in bf16 and fp16 alike, two levels for one rotate and one and-or (the image keeps the levels of a word in the order in which
// the pairs come out).  The matrix unit sums x (16 + q) over a group in fp32, started at -(16 + z) sum x, and the group's scale
// multiplies what it leaves: no product is rounded before the sum, and what cancels is at most some six times the result's own size.
// The sums of x come from the matrix unit too (a right operand of ones leaves them in every column, where the start needs them).
// fp32 rows travel as three bf16 parts cut off one after the other (8 + 8 + 8 bits: exact), three products each.
//
// Layout.  16x16x32 products with x as the left operand and 16 outputs as the right one: a lane holds the word of 8 levels of output
// lane % 16, and 16 bytes of the image are the lane's words of four products (128 k): whole lines, read once, straight into registers.
// x needs no staging either: the lane's eight k are neighbours in memory.  Row r of the left operand is row 4 (r % 4) + r / 4 of x, so
// that up to four rows land in one accumulator register of every lane.
// A workgroup owns 16 NT outputs; its waves take the chunks of 128 k in turn and are joined in LDS.
//
// Bound: HBM by its bytes (0.5 + scale / group a weight) once the layer is large, the latency of one workgroup for small layers.
#include "decode_common.h"

namespace ttsamd {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ unsigned rotr(unsigned x, int n) { return __builtin_amdgcn_alignbit(x, x, n); }

// The eight levels of a word as 16 + q: bits 4p and 16 + 4p of the word hold levels 2p and 2p + 1.
template <bool BF> __device__ __forceinline__ uint4 unpack(unsigned w)
{
    constexpr int at = BF ? 3 : 6;                                     // where the mantissa of 16 + q holds q
    constexpr unsigned mask = 0xfu << at | 0xfu << (at + 16), one = BF ? 0x41804180u : 0x4c004c00u;
    return uint4{(rotr(w, (32 - at) & 31) & mask) | one, (rotr(w, (36 - at) & 31) & mask) | one, (rotr(w, (40 - at) & 31) & mask) | one,
                 (rotr(w, (44 - at) & 31) & mask) | one};
}
template <bool BF> __device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float ld_any(const void *p, int64_t i, int dtype)
{
    return dtype == TTSAMD_F32 ? ((const float *)p)[i] : dtype == TTSAMD_F16 ? to_f(((const _Float16 *)p)[i]) : to_f(((const __bf16 *)p)[i]);
}
// The upper halves of x and y.
__device__ __forceinline__ unsigned uppers(unsigned x, unsigned y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); }

template <class T, int MT, int NT, int GROUP, int MAXW> __global__ __launch_bounds__(MAXW * 64) void linear_w4(ttsamd_linear_w4_args a)
{
    constexpr bool F32 = sizeof(T) == 4, BF = !__is_same(T, _Float16);
    constexpr int PARTS = F32 ? 3 : 1, PER = GROUP / 32, GPC = 128 / GROUP;      // products a group, groups a chunk
    extern __shared__ float join[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int tiles = (a.n + 15) / 16, chunks = (a.k + 127) / 128;
    const int n0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT, rows = min(a.m - m0, 16 * MT);
    const int c16 = lane & 15, g4 = lane >> 4, row = 4 * (c16 & 3) + (c16 >> 2);
    const uint4 ones = BF ? uint4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u} : uint4{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
    const uint4 *levels[NT];
    int64_t sg[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const int64_t tile = min(n0 + u, tiles - 1);                             // a tile behind the last is computed twice, stored once
        levels[u] = (const uint4 *)a.levels + tile * chunks * 64 + lane;
        sg[u] = tile * chunks * GPC * 16 + c16;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[u][t] = f32x4{0.f, 0.f, 0.f, 0.f};

    uint4 next[NT];
    if (wave < chunks)
#pragma unroll
        for (int u = 0; u < NT; ++u) next[u] = levels[u][(int64_t)wave * 64];
    for (int c = wave; c < chunks; c += waves) {
        unsigned word[NT][4];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            word[u][0] = next[u].x, word[u][1] = next[u].y, word[u][2] = next[u].z, word[u][3] = next[u].w;
            if (c + waves < chunks) next[u] = levels[u][(int64_t)(c + waves) * 64];
        }
        float scale[NT][GPC], zero[NT][GPC];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const int64_t at = sg[u] + ((int64_t)c * GPC + q) * 16;
                scale[u][q] = ld_any(a.scales, at, a.scale_dtype);
                zero[u][q] = a.zeros ? -16.f - (float)a.zeros[at] : -24.f;
            }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            uint4 x[4][PARTS];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 128 * c + 32 * j + 8 * g4;
                const bool in = 16 * t + row < rows && k < a.k;
                const T *src = (const T *)a.x + (int64_t)(m0 + 16 * t + row) * a.x_stride + k;
                if constexpr (F32) {
                    unsigned f[8] = {};
                    if (in) __builtin_memcpy(f, src, 32);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        x[j][p] = uint4{uppers(f[0], f[1]), uppers(f[2], f[3]), uppers(f[4], f[5]), uppers(f[6], f[7])};
                        if (p + 1 < PARTS)
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] = __float_as_uint(__uint_as_float(f[e]) - __uint_as_float(f[e] & 0xffff0000u));
                    }
                } else {
                    x[j][0] = uint4{0, 0, 0, 0};
                    if (in) __builtin_memcpy(&x[j][0], src, 16);
                }
            }
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < PER; ++j)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) sum = mfma<BF>(x[q * PER + j][p], ones, sum);
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    f32x4 part;
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[i] = sum[i] * zero[u][q];
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const uint4 w = unpack<BF>(word[u][q * PER + j]);
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) part = mfma<BF>(x[q * PER + j][p], w, part);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[u][t][i] = fmaf(part[i], scale[u][q], acc[u][t][i]);
                }
            }
        }
    }
    // join the waves: [wave][x row][output]
    constexpr int LD = 16 * NT + 1;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (16 * t + 4 * i + g4 < rows) join[(wave * rows + 16 * t + 4 * i + g4) * LD + 16 * u + c16] = acc[u][t][i];
    __syncthreads();
    for (int it = threadIdx.x; it < rows * 16 * NT; it += blockDim.x) {
        const int r = it / (16 * NT), col = it % (16 * NT), n = n0 * 16 + col;
        if (n >= a.n) continue;
        float y = 0.f;
        for (int x = 0; x < waves; ++x) y += join[(x * rows + r) * LD + col];
        if (a.bias) y += to_f(((const T *)a.bias)[n]);
        ((T *)a.y)[(int64_t)(m0 + r) * a.y_stride + n] = (T)y;
    }
}

template <class T, int MT, int NT, int GROUP> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    constexpr int MAXW = MT == 1 ? 16 : 8;
    const int chunks = (a.k + 127) / 128, blocks = (a.n + 16 * NT - 1) / (16 * NT), row_blocks = (a.m + 16 * MT - 1) / (16 * MT);
    // Waves share the chunks of k: eight, or sixteen where there are fewer workgroups than compute units.
    int waves = MAXW > 8 && blocks * row_blocks < 256 ? 16 : 8;
    while (waves > 1 && waves > chunks) waves /= 2;
    const int rows = a.m < 16 * MT ? a.m : 16 * MT, bytes = waves * rows * (16 * NT + 1) * 4;
    static std::atomic<unsigned long long> done{0};
    if (hipError_t e = ensure_dynamic_lds((const void *)linear_w4<T, MT, NT, GROUP, MAXW>, MAXW * 16 * MT * (16 * NT + 1) * 4, done)) return e;
    linear_w4<T, MT, NT, GROUP, MAXW><<<dim3(blocks, row_blocks), waves * 64, bytes, st>>>(a);
    return hipSuccess;
}
template <class T, int MT, int NT> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    return a.group == 32 ? start<T, MT, NT, 32>(a, st) : a.group == 64 ? start<T, MT, NT, 64>(a, st) : start<T, MT, NT, 128>(a, st);
}
template <class T, int MT> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    return a.n >= 16 * 1024 ? start<T, MT, 2>(a, st) : start<T, MT, 1>(a, st);
}
template <class T> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    // Rows beyond 16 share the unpacked weights where the output tiles alone fill the chip; else they are workgroups of their own,
    // which read the weights again from the cache.
    const int tiles = (a.n + 15) / 16;
    if (a.m <= 16 || tiles * ((a.m + 15) / 16) <= 512) return start<T, 1>(a, st);
    return a.m <= 32 || tiles * ((a.m + 31) / 32) <= 512 ? start<T, 2>(a, st) : start<T, 4>(a, st);
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
    if (a->m > 65535 * 16) {
        set_error("linear_w4: %d rows (up to 2^20 - 16)", a->m);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    hipStream_t st = as_stream(stream);
    TTSAMD_HIP(a->dtype == TTSAMD_F32 ? start<float>(*a, st) : a->dtype == TTSAMD_F16 ? start<_Float16>(*a, st) : start<__bf16>(*a, st));
    TTSAMD_LAUNCH_CHECK();
    return TTSAMD_OK;
}
