// Products of a few rows with 4-bit weights: y[m,n] = sum_g s[n,g] sum_{k in g} x[m,k] (level[n,k] - z[n,g]) + bias[n].
//
// Mathematics.  The matrix unit sums x (q - z) over a group in fp32, and the group's scale multiplies the sum: q - z is a small integer,
// exact in bf16 and fp16 alike, so no product is rounded, and the sum is no larger on its way than the products are.  (Sums of x q, or of x
// with an offset level, less z times the sum of x would round at the size of the sum of x: weights at the zero point would weigh.)
// fp16: the four bits of a level at the end of the mantissa of 1024.0 give 1024 + q, four bits further up in 64.0 64 + q, two levels for one
// and-or (and a shift for every second pair), less 1024 + z or 64 + z in one packed subtraction.  bf16 has none: a level as the low bits of a
// byte is q 2^-9 in fp8 (e4m3, the subnormals and the first binade), four bytes of a word a mask, two levels a conversion to fp32, and one
// fma a level takes 2^9 and z: nineteen instructions a word of eight, against nine.
// fp32 rows travel as three bf16 parts cut off one after the other (8 + 8 + 8 bits: exact), three products each; up to five rows put their
// parts beside each other into the sixteen rows of one product (8128 -> 1688, one row: 12.3 -> 10.0 us; 10.6 with exact levels).
//
// Layout.  16x16x32 products with x as the left operand and 16 outputs as the right one: a lane holds the word of 8 levels of output
// lane % 16, and 16 bytes of the image are the lane's words of four products (128 k): whole lines, read once, straight into registers.
// x goes through LDS, each wave its own chunk: the lanes of a product hold 16 rows each, and loads of 16 bytes a row cost a line each
// (8128 -> 1688 with 16 rows, fp16 10.6 -> 7.6 us, fp32 17.6 -> 13.9).  Row r of the left operand is row 4 (r % 4) + r / 4 of x, so that
// up to four rows land in one accumulator register of every lane.
// A workgroup owns 16 outputs; its waves take the chunks of 128 k in turn and are joined in LDS.
//
// Bound: memory by its bytes (0.5 + scale / group a weight) once the layer is large (8192 x 8192, group 128, one fp16 row: 34.6 MB in 10.3
// us where many layers take turns, 3.4 TB/s, 9.0 over and over; bf16 10.8, fp32 14.4: its unpacking, and for fp32 the parts of x, come on
// top), the latency of one workgroup for small layers (1024 x 1024: 3.2 us), unpacking and products from some 16 rows on, for every sixteen
// rows anew (64 rows of 8192 x 8192: fp16 29 us, 295 TFLOP/s, bf16 35, fp32 77).
#include <type_traits>

#include "decode_common.h"

namespace ttsamd {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool BF> __device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c)
{
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// The upper halves of x and y.
__device__ __forceinline__ unsigned uppers(unsigned x, unsigned y) { return __builtin_amdgcn_perm(y, x, 0x07060302u); }
// The eight levels of a word less the zero point, as eight 16-bit floats: bits 4p and 16 + 4p of the word hold levels 2p and 2p + 1.
// fp16 takes two offsets, 1024 and 64, twice each, and the zero point on top of them.
struct Offset {
    unsigned low, high;
};
__device__ __forceinline__ uint4 unpack(unsigned w, Offset at, const f16x2 (&z)[2])
{
    const unsigned w8 = w >> 8;
    auto low = [&](unsigned v) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, (v & 0x000f000fu) | at.low) - z[0]); };
    auto high = [&](unsigned v) { return __builtin_bit_cast(unsigned, __builtin_bit_cast(f16x2, (v & 0x00f000f0u) | at.high) - z[1]); };
    return uint4{low(w), high(w), low(w8), high(w8)};
}
__device__ __forceinline__ uint4 unpack(unsigned w, Offset, const float (&zero)[1])
{
    const float z = zero[0];
    const unsigned even = w & 0x0f0f0f0fu, odd = w >> 4 & 0x0f0f0f0fu;       // bytes: levels 0 4 1 5, and 2 6 3 7
    auto two = [&](unsigned bytes, auto upper) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 q = __builtin_amdgcn_cvt_pk_f32_fp8(bytes, decltype(upper)::value);
        return uint2{__float_as_uint(fmaf(q[0], 512.f, -z)), __float_as_uint(fmaf(q[1], 512.f, -z))};
    };
    const uint2 a = two(even, std::false_type()), b = two(even, std::true_type()), c = two(odd, std::false_type()), d = two(odd, std::true_type());
    return uint4{uppers(a.x, b.x), uppers(c.x, d.x), uppers(a.y, b.y), uppers(c.y, d.y)};
}

// Output n of row m product by product, for a sum that is no number: an infinity leaves NaN in its parts, and fp32 values from 2^123 on can
// pass fp32's range before the scale, where x times the weight need not.
template <class T, int GROUP> __device__ float summed(const ttsamd_linear_w4_args &a, int m, int n)
{
    const T *x = (const T *)a.x + (int64_t)m * a.x_stride;
    const int chunks = (a.k + 127) / 128;
    const int64_t tile = n / 16;
    const unsigned *words = a.levels + (tile * chunks * 64 + n % 16) * 4;
    float y = a.bias ? to_f(((const T *)a.bias)[n]) : 0.f;
    for (int q = 0; q < a.k / GROUP; ++q) {
        const int64_t at = (tile * chunks * (128 / GROUP) + q) * 16 + n % 16;
        const float z = a.zeros ? (float)a.zeros[at] : 8.f;
        const float scale = a.scale_dtype == TTSAMD_F32    ? ((const float *)a.scales)[at]
                            : a.scale_dtype == TTSAMD_BF16 ? (float)((const __bf16 *)a.scales)[at]
                                                           : (float)((const _Float16 *)a.scales)[at];
        for (int k = q * GROUP; k < (q + 1) * GROUP; ++k) {
            const unsigned w = words[((int64_t)(k / 128) * 64 + (k / 8 % 4) * 16) * 4 + k / 32 % 4];
            y = fmaf(to_f(x[k]), ((float)(w >> (4 * (k / 2 % 4) + 16 * (k % 2)) & 15) - z) * scale, y);
        }
    }
    return y;
}

// Rows of x that a wave stages a chunk of at most; of few rows, so many that a load each (16 bits) or three of them hold them.
template <class T> constexpr int staged_rows(bool few) { return !few ? 16 : sizeof(T) == 4 ? 6 : 4; }
template <class T> constexpr int few_rows() { return sizeof(T) == 4 ? 5 : 4; }

template <class T, int NT, int GROUP, int MAXW, bool FEW> __global__ __launch_bounds__(MAXW * 64) void linear_w4(ttsamd_linear_w4_args a)
{
    constexpr bool F32 = sizeof(T) == 4, BF = !__is_same(T, _Float16), BESIDE = F32 && FEW;
    constexpr int PARTS = F32 && !BESIDE ? 3 : 1, PER = GROUP / 32, GPC = 128 / GROUP;      // products a group, groups a chunk
    constexpr int ES = sizeof(T), PPR = 8 * ES, RPI = 64 / PPR, XI = staged_rows<T>(FEW) / RPI;   // 16-byte pieces of a chunk of a row; rows a load; loads
    constexpr bool XAHEAD = NT < 4 && !(F32 && !FEW && NT == 2 && GROUP == 32);          // the others have no registers left for it
    extern __shared__ float join[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int chunks = (a.k + 127) / 128, m0 = blockIdx.y * 16, rows = min(a.m - m0, 16), products = BESIDE ? 3 * rows : rows;
    const int c16 = lane & 15, g4 = lane >> 4, row = 4 * (c16 & 3) + (c16 >> 2);
    struct Zero {
        std::conditional_t<BF, float, f16x2> v[BF ? 1 : 2];
    };
    Offset offset = {0x64006400u, 0x54005400u};
    if constexpr (!BF) asm("" : "+v"(offset.low), "+v"(offset.high));      // in vector registers: and-or takes one scalar operand, the mask
    const uint4 *levels[NT];
    int64_t sg[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
        const int64_t tile = min((int)blockIdx.x * NT + u, (a.n + 15) / 16 - 1);      // behind the last: the last again, never stored
        levels[u] = (const uint4 *)a.levels + tile * chunks * 64 + lane;
        sg[u] = tile * chunks * GPC * 16 + c16;
    }
    // a row behind the last is the last one again: no row of a product meets another
    const T *const x0 = (const T *)a.x + (int64_t)m0 * a.x_stride;
    const int piece = lane % PPR, lrow = lane / PPR, arow = min(BESIDE ? row / 3 : row, rows - 1);
    char *const stage = (char *)join + wave * XI * RPI * 16 * PPR;
    const unsigned first = BESIDE && row % 3 > 0 ? 0xffff0000u : 0u, second = BESIDE && row % 3 > 1 ? 0xffff0000u : 0u;     // parts that go before
    f32x4 acc[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Two chunks are on their way at any time: levels, scales and zeros as they lie in memory, x too where the registers allow.
    struct Chunk {
        uint4 word[NT];
        unsigned scale[NT][GPC], zero[NT][GPC];
        uint4 x[XAHEAD ? XI : 1];
    } ahead[2];
    const bool wide = a.scale_dtype == TTSAMD_F32, brain = a.scale_dtype == TTSAMD_BF16, zeros = a.zeros != nullptr;
    auto fetch_x = [&](uint4 &to, int c, int i) {
        const int k = 128 * c + 16 / ES * piece;                                 // behind the last k the weights are 0: any x will do
        __builtin_memcpy(&to, x0 + (int64_t)min(RPI * i + lrow, rows - 1) * a.x_stride + min(k, a.k - 16 / ES), 16);
    };
    auto fetch = [&](Chunk &f, int c) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            f.word[u] = levels[u][(int64_t)c * 64];
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const int64_t at = sg[u] + ((int64_t)c * GPC + q) * 16;
                f.scale[u][q] = wide ? ((const unsigned *)a.scales)[at] : ((const unsigned short *)a.scales)[at];
                if (zeros) f.zero[u][q] = a.zeros[at];
            }
        }
        if constexpr (XAHEAD)
#pragma unroll
            for (int i = 0; i < XI; ++i) fetch_x(f.x[i], c, i);
    };
    auto multiply = [&](Chunk &f, int c) {
        unsigned word[NT][4];
        Zero zero[NT][GPC];
        float scale[NT][GPC];
        // x by way of LDS: loaded as it lies (whole lines), read as the products take it
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            const int r = RPI * i + lrow;
            uint4 w;
            if constexpr (XAHEAD) w = f.x[i];
            else fetch_x(w, c, i);
            *(uint4 *)(stage + r * 16 * PPR + (piece ^ r) * 16) = w;
        }
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            word[u][0] = f.word[u].x, word[u][1] = f.word[u].y, word[u][2] = f.word[u].z, word[u][3] = f.word[u].w;
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                const unsigned r = f.scale[u][q];
                scale[u][q] = wide ? __uint_as_float(r) : brain ? __uint_as_float(r << 16) : (float)__builtin_bit_cast(_Float16, (unsigned short)r);
                const float z = zeros ? (float)f.zero[u][q] : 8.f;
                if constexpr (BF) zero[u][q].v[0] = z;
                else zero[u][q].v[0] = f16x2{(_Float16)(1024.f + z), (_Float16)(1024.f + z)}, zero[u][q].v[1] = f16x2{(_Float16)(64.f + z), (_Float16)(64.f + z)};
            }
        }
        if (c + 2 * waves < chunks) fetch(f, c + 2 * waves);
        uint4 raw[4][ES / 2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int y = 0; y < ES / 2; ++y) raw[j][y] = *(const uint4 *)(stage + arow * 16 * PPR + (((4 * j + g4) * (ES / 2) + y) ^ arow) * 16);
        uint4 x[4][PARTS];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (F32) {
                if constexpr (BESIDE) {
                    unsigned e8[8] = {raw[j][0].x, raw[j][0].y, raw[j][0].z, raw[j][0].w, raw[j][1].x, raw[j][1].y, raw[j][1].z, raw[j][1].w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        e8[e] = __float_as_uint(__uint_as_float(e8[e]) - __uint_as_float(e8[e] & first));
                        e8[e] = __float_as_uint(__uint_as_float(e8[e]) - __uint_as_float(e8[e] & second));
                    }
                    x[j][0] = uint4{uppers(e8[0], e8[1]), uppers(e8[2], e8[3]), uppers(e8[4], e8[5]), uppers(e8[6], e8[7])};
                    continue;
                }
                unsigned e8[8] = {raw[j][0].x, raw[j][0].y, raw[j][0].z, raw[j][0].w, raw[j][1].x, raw[j][1].y, raw[j][1].z, raw[j][1].w};
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    x[j][p] = uint4{uppers(e8[0], e8[1]), uppers(e8[2], e8[3]), uppers(e8[4], e8[5]), uppers(e8[6], e8[7])};
                    if (p + 1 < PARTS)
#pragma unroll
                        for (int e = 0; e < 8; ++e) e8[e] = __float_as_uint(__uint_as_float(e8[e]) - __uint_as_float(e8[e] & 0xffff0000u));
                }
            } else {
                x[j][0] = raw[j][0];
            }
        }
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int q = 0; q < GPC; ++q) {
                f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const uint4 w = unpack(word[u][q * PER + j], offset, zero[u][q].v);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) part = mfma<BF>(x[q * PER + j][p], w, part);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[u][i] = fmaf(part[i], scale[u][q], acc[u][i]);
            }
    };
    if (wave < chunks) fetch(ahead[0], wave);
    if (wave + waves < chunks) fetch(ahead[1], wave + waves);
    for (int c = wave; c < chunks; c += 2 * waves) {
        multiply(ahead[0], c);
        if (c + waves < chunks) multiply(ahead[1], c + waves);
    }
    // join the waves: [wave][x row][output]
    __syncthreads();
    constexpr int LD = 16 * NT + 1;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * i + g4 < products) join[(wave * products + 4 * i + g4) * LD + 16 * u + c16] = acc[u][i];
    __syncthreads();
    for (int it = threadIdx.x; it < rows * 16 * NT; it += blockDim.x) {
        const int r = it / (16 * NT), col = it % (16 * NT), n = blockIdx.x * 16 * NT + col;
        if (n >= a.n) continue;
        float y = a.bias ? to_f(((const T *)a.bias)[n]) : 0.f;
#pragma unroll 4
        for (int x = 0; x < waves; ++x) {
            if constexpr (BESIDE) y += join[(x * products + 3 * r + 2) * LD + col] + join[(x * products + 3 * r + 1) * LD + col] + join[(x * products + 3 * r) * LD + col];
            else y += join[(x * rows + r) * LD + col];
        }
        if (!(fabsf(y) < __builtin_inff())) y = summed<T, GROUP>(a, m0 + r, n);
        ((T *)a.y)[(int64_t)(m0 + r) * a.y_stride + n] = (T)y;
    }
}

template <class T, int NT, int GROUP, bool FEW> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    constexpr int MAXW = NT == 1 && sizeof(T) == 2 && FEW ? 16 : 8;
    const int chunks = (a.k + 127) / 128, blocks = (a.n + 16 * NT - 1) / (16 * NT), row_blocks = (a.m + 15) / 16;
    const bool few = (int64_t)blocks * row_blocks < 256;
    // Waves share the chunks of k: eight, or sixteen where there are fewer workgroups than compute units (and the registers of few rows).
    int waves = MAXW > 8 && few ? 16 : 8;
    while (waves > 1 && waves > chunks) waves /= 2;
    const int rows = a.m < 16 ? a.m : 16, joined = waves * (FEW && sizeof(T) == 4 ? 3 * rows : rows) * (16 * NT + 1) * 4;
    constexpr int staged = staged_rows<T>(FEW) * 128 * (int)sizeof(T), most_joined = MAXW * 16 * (16 * NT + 1) * 4;
    const int bytes = joined > waves * staged ? joined : waves * staged;
    static std::atomic<unsigned long long> done{0};
    if (hipError_t e = ensure_dynamic_lds((const void *)linear_w4<T, NT, GROUP, MAXW, FEW>, most_joined > MAXW * staged ? most_joined : MAXW * staged, done)) return e;
    linear_w4<T, NT, GROUP, MAXW, FEW><<<dim3(blocks, row_blocks), waves * 64, bytes, st>>>(a);
    return hipSuccess;
}
template <class T, int NT, int GROUP> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    return a.m <= few_rows<T>() ? start<T, NT, GROUP, true>(a, st) : start<T, NT, GROUP, false>(a, st);
}
template <class T, int NT> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    return a.group == 32 ? start<T, NT, 32>(a, st) : a.group == 64 ? start<T, NT, 64>(a, st) : start<T, NT, 128>(a, st);
}
template <class T> hipError_t start(const ttsamd_linear_w4_args &a, hipStream_t st)
{
    // Every workgroup reads its rows of x whole: several output tiles a wave read (and, fp32, split) them once, as long as the chip stays
    // full and the registers hold.  us at 1 / 2 / 4 tiles, k = 4096, groups of 64: bf16, 16 rows to 4096 outputs (256 tiles) 6.0 / 8.0 /
    // 12.3, to 8192 8.8 / 8.4 / 12.7, 64 rows to 8192 24.7 / 27.4 / 23.8; fp16, 32 rows to 8192 (1024 tiles) 13.4 / 13.6 / 11.5, to 16384
    // 24.1 / 25.2 / 22.8; fp32, one row to 4096 6.8 / 8.7, to 8192 10.4 / 9.5, 64 rows to 4096 31.5 / 22.8.  Few rows have nothing to gain
    // from four: one bf16 row to 16384 11.7 / 11.8 / 13.1, k = 2048 to 32768 14.1 / 12.3 / 15.4.
    const int64_t tiles = (int64_t)((a.n + 15) / 16) * ((a.m + 15) / 16);
    if (tiles < 512) return start<T, 1>(a, st);
    if constexpr (sizeof(T) == 2)
        if (tiles >= 1024 && a.m > few_rows<T>() && a.group >= 64) return a.group == 64 ? start<T, 4, 64, false>(a, st) : start<T, 4, 128, false>(a, st);
    return start<T, 2>(a, st);
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
    if (a->m > 65535 * 16 || a->n > (1 << 30) || a->k > (1 << 30)) {
        set_error("linear_w4: %d rows, %d by %d weights (up to 2^20 - 16 rows, 2^30 a side)", a->m, a->n, a->k);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    if (int rc = check_written("linear_w4", "y", rows_of(a->y, a->y_stride, 0, a->m, 1, a->n, a->dtype), "x",
                               rows_of(a->x, a->x_stride, 0, a->m, 1, a->k, a->dtype), false))
        return rc;
    hipStream_t st = as_stream(stream);
    TTSAMD_HIP(a->dtype == TTSAMD_F32 ? start<float>(*a, st) : a->dtype == TTSAMD_F16 ? start<_Float16>(*a, st) : start<__bf16>(*a, st));
    TTSAMD_LAUNCH_CHECK();
    return TTSAMD_OK;
}
