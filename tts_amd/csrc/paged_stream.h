// Attention of few rows over a long paged cache: keys and values stream from memory through registers into the matrix unit.
//
// Rows.  All query heads that read one key head, of all new tokens of a sequence, are rows of one problem: row r = token r / G,
// head r % G (G = q_heads / kv_heads).  A workgroup takes NQ tiles of 16 rows; its waves take the tiles of its keys in turn, each with
// a running maximum and sum of its own, and are joined in LDS at the end.
//
// Layout.  S^T = K Q^T is computed with the keys as the matrix rows, so that in the 16x16 result a lane holds one query row (column
// lane % 16) and the keys 4 (lane / 16) + i: maximum, exponential and sum stay in the lane.  The same registers, in T, are the
// right operand of O^T = V^T P^T as they lie, because the order of the keys inside a contraction is free: slot (lane / 16, e) of the
// 32-deep product is key 4 (lane / 16) + e of the first 16 keys for e < 4, of the second for e >= 4.  The left operand V^T wants, per
// lane, eight keys of one channel; a lane loads eight keys of NV = DP / 16 neighbouring channels (16 bytes and whole lines at DP = 128)
// and regroups the halves with one v_perm per pair, so nothing passes through LDS.  fp32 uses the 4-deep fp32 product: no regrouping,
// 16 keys a tile.
//
// A probability travels in two parts of T, the nearest one and the remainder, a product each (together 16 bits of bf16, 22 of fp16), and is
// summed in fp32: rounded to T once it would be off by as much as the result's own rounding.  These kernels wait for memory: 48 fp16 tokens
// over 1007 keys 32.3 -> 32.8 us, three bf16 ones over 65537 77.6 -> 77.7, eight sequences of 40 rows over 2000 keys 24.7 -> 25.6.
//
// The running maximum moves only when a score exceeds it by a good deal (lazy; p stays within every type's range): the cross-lane
// maximum and the scaling of O are skipped in almost every tile.
//
// Where a tile's rows lie (page lookup, one key a lane, keys in lanes 0-31 and values in lanes 32-63) is fetched a tile ahead; a
// key without a place gets the cache's first row and is masked, its value zeroed, so no lane ever reads outside the pages.
//
// A value that is an infinity or NaN must not reach rows that do not see its key, and 0 * infinity would: where a tile is seen by some
// rows only and holds such a value, the rows are computed again key by key.
//
// Bound: memory for single tokens.  48 fp16 sequences of up to 1007 keys, 16 heads of 64: 150 MB in 33.8 us where many caches take turns
// (4.4 TB/s), 27.6 where one stays in the last-level cache; three bf16 ones of up to 65537, 32 heads over 4 of 128: 363 MB in 66 us (5.5
// TB/s; a large copy reaches 5.0 to 5.3), and 5 for the join of 21 splits.
#pragma once
#include <type_traits>

#include "decode_common.h"

namespace ttsamd {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr float kNoMax = -3.402823466e38f;      // a running maximum before the first key: no score lies below it, no difference of two is NaN
constexpr float kFar = 4194304.f;               // 2^22
// How far (log2) a row's largest p lies above 1 when the running maximum moves, and how much further it may rise before it moves again.
// fp16 holds no step below 2^-24: with a largest p of 2^11 to 2^15 a key loses at most 2^-36 of the heaviest one's weight (from 1 to 2^8,
// thousands of keys of 2^-25 each weighed nothing).  bf16 and fp32 have the range.
template <class T> constexpr float lift() { return __is_same(T, _Float16) ? 11.f : 0.f; }
template <class T> constexpr float lazy() { return __is_same(T, _Float16) ? 4.f : 8.f; }

struct AttArgs {
    ttsamd_paged_attention_args a;
    ttsamd_paged_kv c;
    ttsamd_paged_batch b;
    FastDiv by_page, by_group;       // group = query heads a key head
    float scale2;                    // scale * log2 e
    int group, splits, split_keys;   // split_keys: keys of a split (the last takes the rest)
    float *part;                     // splits > 1: [tokens * q_heads][splits][head_dim], then [tokens * q_heads][splits][2]
    float *stat;
};

// p = exp2(s scale2 - m) as one fma takes m, the rounded product of a largest score, from s scale2 unrounded: every p of the row is off by
// the same power of two, half a last place of m at most, in whichever part of the keys it lies, and that falls out of o / l as long as it
// is small.  From |m| = 2^22 on (a quarter) it need not be: for such rows (is_far) the scores are scaled and rounded as the maximum was
// before it is taken away, and its key has p = 1.  Scores are to stay within 2^127 in size, so that their product with log2 e is finite.
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar && m > kNoMax; }

template <class T> __device__ __forceinline__ f32x4_t mfma_16x16x32(uint4 a, uint4 b, f32x4_t c);
template <> __device__ __forceinline__ f32x4_t mfma_16x16x32<__bf16>(uint4 a, uint4 b, f32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4_t mfma_16x16x32<_Float16>(uint4 a, uint4 b, f32x4_t c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}
template <class T> __device__ __forceinline__ f32x4_t mfma_16x16x16(uint2 a, uint2 b, f32x4_t c)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(h4, a), __builtin_bit_cast(h4, b), c, 0, 0, 0);
}
template <class T> __device__ __forceinline__ unsigned pack2(float x, float y)
{
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef T t2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2{x, y}), t2));
}
// x and y in two parts of T each: the nearest one and what it leaves, rounded.
template <class T> __device__ __forceinline__ void split2(float x, float y, unsigned &upper, unsigned &lower)
{
    typedef T t2 __attribute__((ext_vector_type(2)));
    upper = pack2<T>(x, y);
    if constexpr (__is_same(T, __bf16)) {
        lower = pack2<T>(x - __uint_as_float(upper << 16), y - __uint_as_float(upper & 0xffff0000u));
    } else {
        const t2 h = __builtin_bit_cast(t2, upper);
        lower = pack2<T>(x - (float)h[0], y - (float)h[1]);
    }
}
// Both halves of w, added to c in fp32: the probabilities as the products take them, so that what their rounding does to numerator and
// denominator alike falls out.
template <class T> __device__ __forceinline__ float sum2(unsigned w, float c)
{
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w), b2{(__bf16)1.f, (__bf16)1.f}, c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w), h2{(_Float16)1.f, (_Float16)1.f}, c, false);
}
// Whether a 32-bit word of T holds an infinity or NaN.
template <class T> __device__ __forceinline__ bool any_odd(unsigned w)
{
    constexpr unsigned X = __is_same(T, float) ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
    if constexpr (sizeof(T) == 4) return (w & X) == X;
    else return (w & X) == X || (w >> 16 & X) == X;
}

// Which of the 64 keys from `base` a row sees.
__device__ __forceinline__ uint64_t seen_bits(uint64_t ok, int base, Range see)
{
    const int from = max(see.begin - base, 0), to = see.end - base;
    if (from >= 64 || to <= from) return 0;
    return ok & (~0ull << from) & (to >= 64 ? ~0ull : ~(~0ull << to));
}
// x where bit `b` of `bits` is set, else minus infinity.
__device__ __forceinline__ float masked(float x, uint32_t bits, int b)
{
    const uint32_t all = (uint32_t)((int32_t)(bits << (31 - b)) >> 31);
    return __uint_as_float((__float_as_uint(x) & all) | (0xff800000u & ~all));
}

// One row's keys [lo, hi), a wave, key by key: o[d] += p v only for the keys of `see`.  For the rare tile where a value that some row
// must not see is an infinity or NaN.  Lane x owns o[x], o[x + 64], ..; returns the sum of the p (every lane).
template <class T>
__device__ float attend_row(const AttArgs &g, int b, int hk, const T *q, Range see, float *o, float *ml)
{
    const int lane = threadIdx.x & 63, D = g.c.head_dim;
    float m = kNoMax, l = 0.f, acc[4] = {};
    for (int j = see.begin; j < see.end; ++j) {
        int row;
        const int64_t page = page_of(g.b, g.by_page, g.c.pages, b, j, row);
        if (page < 0) continue;
        const T *k = (const T *)g.c.k + page * g.c.k_page + hk * g.c.k_head + row * g.c.k_row;
        const T *v = (const T *)g.c.v + page * g.c.v_page + hk * g.c.v_head + row * g.c.v_row;
        float x = 0.f;
        for (int d = lane; d < D; d += 64) x = fmaf(to_f(q[d]), to_f(k[d]), x);
        for (int y = 32; y; y >>= 1) x += __shfl_xor(x, y);
        const float t = x * g.scale2, to = fmaxf(m, t), fade = __builtin_amdgcn_exp2f(m - to), p = __builtin_amdgcn_exp2f(is_far(to) ? t - to : fmaf(x, g.scale2, -to));
        m = to, l = l * fade + p;
        for (int y = 0; y < 4; ++y)
            if (lane + 64 * y < D) acc[y] = fmaf(p, to_f(v[lane + 64 * y]), acc[y] * fade);
    }
    for (int y = 0; y < 4; ++y)
        if (lane + 64 * y < D) o[lane + 64 * y] = acc[y];
    if (lane == 0) ml[0] = m, ml[1] = l;
    return l;
}

// x of the lane N places on in the row of 16.
template <int N> __device__ __forceinline__ float turned(float x)
{
    return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x120 + N, 0xf, 0xf, true));
}

// Joins the parts o [part][row][DP + 4] and (m, l) [part][row] that lie in LDS and writes the rows r0 .. r0 + nr: to the output, or as one
// split of it.  R: rows of a part.
template <class T, int DP>
__device__ __forceinline__ void join_waves(const AttArgs &g, const Sequence &s, int hk, int split, const float *lds, const float *ml, int r0, int nr,
                                           int R, int parts)
{
    constexpr int LDO = DP + 4;
    const int D = g.c.head_dim, cols = D / 4;
    for (int w = threadIdx.x; w < nr * cols; w += blockDim.x) {
        const int r = w / cols, d = (w - r * cols) * 4;
        float top = kNoMax, sum = 0.f;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int x = 0; x < parts; ++x) top = fmaxf(top, ml[2 * (x * R + r)]);
#pragma unroll 4
        for (int x = 0; x < parts; ++x) {
            const float f = __builtin_amdgcn_exp2f(ml[2 * (x * R + r)] - top);
            sum += f * ml[2 * (x * R + r) + 1];
            acc += *(const f32x4_t *)(lds + (x * R + r) * LDO + d) * f;
        }
        const int row = r0 + r, i = g.by_group.div(row), h = hk * g.group + row - i * g.group;
        const int64_t token = s.start + i;
        if (g.splits > 1) {
            const int64_t at = (token * g.a.q_heads + h) * g.splits + split;
            *(f32x4_t *)(g.part + at * D + d) = acc;
            if (d == 0) g.stat[2 * at] = top, g.stat[2 * at + 1] = sum;
        } else {
            const float inv = sum > 0.f ? 1.f / sum : sum;          // no key: zeros; NaN stays
            acc *= inv;
            T *dst = (T *)g.a.out + token * g.a.o_tstride + (int64_t)h * g.a.o_hstride + d;
            if constexpr (sizeof(T) == 4) *(f32x4_t *)dst = acc;
            else *(uint2 *)dst = uint2{pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3])};
        }
    }
}

template <class T, int DP, int NQ, bool FULL, int MAXW>
__global__ __launch_bounds__(MAXW * 64) void attend_stream(AttArgs g)
{
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int ES = sizeof(T), RB = DP * ES, NS = RB / 64, NV = DP / 16, KT = F32 || DP > 192 ? 16 : 32, NT = KT / 16;
    constexpr int VK = KT / 4;                          // values (keys) a lane holds of a tile
    constexpr int VB = NV * ES, VP = VB % 16 ? 8 : 16;  // bytes of a lane's channels of one key, and of one load
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int c16 = lane & 15, g4 = lane >> 4;
    const int hk = blockIdx.x / g.splits, split = blockIdx.x - hk * g.splits, b = blockIdx.z;
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, b);
    const int D = g.c.head_dim, rows = s.n * g.group;
    const char *kbase = (const char *)g.c.k + (int64_t)hk * g.c.k_head * ES, *vbase = (const char *)g.c.v + (int64_t)hk * g.c.v_head * ES;
    const bool vrole = lane >= 32;
    const uint32_t page16 = (uint32_t)((vrole ? g.c.v_page : g.c.k_page) * ES / 16), row16 = (uint32_t)((vrole ? g.c.v_row : g.c.k_row) * ES / 16);

    // the largest score is found before the scale: it has to be positive (a negative one turns q's sign, zero takes q away)
    const unsigned flip = g.scale2 < 0.f ? F32 ? 0x80000000u : 0x80008000u : 0u, keep = g.scale2 == 0.f ? 0u : ~0u;
    const float scale2 = g.scale2 == 0.f ? 1.f : fabsf(g.scale2);

    for (int tile = (rows + 16 * NQ - 1) / (16 * NQ) - 1 - blockIdx.y; tile >= 0; tile -= gridDim.y) {      // the longest first
        const int r0 = tile * 16 * NQ, last = min(r0 + 16 * NQ, rows) - 1;
        Range mine[NQ];
        uint4 q[NQ][NS];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            const int r = min(r0 + 16 * u + c16, last), i = g.by_group.div(r), h = hk * g.group + r - i * g.group;
            mine[u] = seen_by(s, s.len - s.n + i, g.a.causal, g.a.window);
            const char *src = (const char *)g.a.q + ((int64_t)(s.start + i) * g.a.q_tstride + (int64_t)h * g.a.q_hstride) * ES;
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                const int at = x * 64 + g4 * 16;
                q[u][x] = FULL || at < D * ES ? *(const uint4 *)(src + (FULL || at < D * ES ? at : 0)) : uint4{0, 0, 0, 0};
                q[u][x].x = (q[u][x].x & keep) ^ flip, q[u][x].y = (q[u][x].y & keep) ^ flip;
                q[u][x].z = (q[u][x].z & keep) ^ flip, q[u][x].w = (q[u][x].w & keep) ^ flip;
            }
        }
        const Range first = seen_by(s, s.len - s.n + (int)g.by_group.div(r0), g.a.causal, g.a.window);
        const Range final = seen_by(s, s.len - s.n + (int)g.by_group.div(last), g.a.causal, g.a.window);
        // ranges move to the right with the row: the union is [first.begin, final.end), the intersection [final.begin, first.end)
        const int64_t from = first.begin + (int64_t)split * g.split_keys, to = split + 1 < g.splits ? from + g.split_keys : final.end;
        const int lo = (int)min(from, (int64_t)final.end), hi = (int)min(to, (int64_t)final.end);

        f32x4_t o[NQ][NV];
        float m[NQ], l[NQ];
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            m[u] = kNoMax, l[u] = 0.f;
#pragma unroll
            for (int x = 0; x < NV; ++x) o[u][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }

        bool odd = false, far[NQ] = {};
        int base = lo + wave * KT;
        const int step = waves * KT, idx = lane & (KT - 1);
        uint4 k[NT][NS];
        unsigned v[VK][VB / 4];
        // the table's entry for this lane's key of the tile at `at`, still on its way; what it is worth once it is there
        auto fetch = [&](int at, int &row) { return entry_of(g.b, g.by_page, b, min(at + idx, hi - 1), row); };
        auto place = [&](int at, int entry) { return at + idx < hi && held(entry, g.c.pages) ? entry : -1; };
        auto load_k = [&](uint32_t off) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const char *p = kbase + (uint64_t)(uint32_t)__shfl((int)off, 16 * t + c16) * 16;
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    const int at = x * 64 + g4 * 16;
                    k[t][x] = *(const uint4 *)(p + (FULL || at < D * ES ? at : 0));
                    if (!FULL && at >= D * ES) k[t][x] = uint4{0, 0, 0, 0};
                }
            }
        };
        int row_next = 0, page_next = -1;
        uint32_t off = 0;
        unsigned ok = 0;
        if (base < hi) {
            int row;
            const int page = place(base, fetch(base, row));
            off = page < 0 ? 0 : (uint32_t)page * page16 + (uint32_t)row * row16;
            ok = (unsigned)__ballot(page >= 0) & (KT == 32 ? ~0u : 0xffffu);
            load_k(off);
            page_next = fetch(base + step, row_next);
        }
        for (; base < hi; base += step) {
            // values of this tile: slot e of lane group g4 is key 4 g4 + e (e < 4), 16 + 4 g4 + e - 4
#pragma unroll
            for (int e = 0; e < VK; ++e) {
                const char *p = vbase + (uint64_t)(uint32_t)__shfl((int)off, 32 + (e & 3) + 4 * g4 + (e >> 2) * 16) * 16;
#pragma unroll
                for (int x = 0; x < VB / VP; ++x) {
                    const int at = c16 * VB + x * VP, in = FULL || at < D * ES ? at : 0;
                    if constexpr (VP == 8) {
                        const uint2 w = *(const uint2 *)(p + in);
                        v[e][2 * x] = w.x, v[e][2 * x + 1] = w.y;
                    } else {
                        const uint4 w = *(const uint4 *)(p + in);
                        v[e][4 * x] = w.x, v[e][4 * x + 1] = w.y, v[e][4 * x + 2] = w.z, v[e][4 * x + 3] = w.w;
                    }
                }
            }
            const unsigned ok_now = ok;
            const int page = place(base + step, page_next);
            off = page < 0 ? 0 : (uint32_t)page * page16 + (uint32_t)row_next * row16;
            ok = (unsigned)__ballot(page >= 0) & (KT == 32 ? ~0u : 0xffffu);
            page_next = fetch(base + 2 * step, row_next);

            f32x4_t sc[NQ][NT];
#pragma unroll
            for (int u = 0; u < NQ; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < NS; ++x) {
                        if constexpr (F32) {
                            const f32x4_t kk = __builtin_bit_cast(f32x4_t, k[t][x]), qq = __builtin_bit_cast(f32x4_t, q[u][x]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[j], qq[j], acc, 0, 0, 0);
                        } else {
                            acc = mfma_16x16x32<T>(k[t][x], q[u][x], acc);
                        }
                    }
                    sc[u][t] = acc;
                }
            if (base + step < hi) load_k(off);

            const bool clear = ok_now == (KT == 32 ? ~0u : 0xffffu) && base >= final.begin && base + KT <= first.end;
            if (!clear) {
#pragma unroll
                for (int e = 0; e < VK; ++e) {
                    const bool held = ok_now >> ((e & 3) + 4 * g4 + (e >> 2) * 16) & 1;
#pragma unroll
                    for (int x = 0; x < VB / 4; ++x) {
                        if (!held) v[e][x] = 0;                              // 0 * p stays 0 whatever lies there
                        else if (s.n > 1) odd |= any_odd<T>(v[e][x]);        // 0 * infinity would not
                    }
                }
            }
            float p[NQ][VK];
#pragma unroll
            for (int u = 0; u < NQ; ++u) {
                if (!clear) {
                    const uint32_t bits = (uint32_t)seen_bits(ok_now, base, mine[u]) >> (4 * g4);
#pragma unroll
                    for (int e = 0; e < VK; ++e) sc[u][e >> 2][e & 3] = masked(sc[u][e >> 2][e & 3], bits, (e & 3) + (e >> 2) * 16);
                }
                float top = sc[u][0][0];
#pragma unroll
                for (int e = 1; e < VK; ++e) top = fmaxf(top, sc[u][e >> 2][e & 3]);
                top *= scale2;
                if (__any(top > m[u] + (lift<T>() + lazy<T>()))) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float to = fmaxf(m[u], top - lift<T>()), fade = __builtin_amdgcn_exp2f(m[u] - to);
                    m[u] = to, l[u] *= fade;
#pragma unroll
                    for (int x = 0; x < NV; ++x) o[u][x] *= fade;
                    far[u] = __any(is_far(to));
                }
                float by = scale2, off = m[u];
                if (far[u]) {
                    const bool it = is_far(m[u]);
#pragma unroll
                    for (int e = 0; e < VK; ++e) sc[u][e >> 2][e & 3] = it ? sc[u][e >> 2][e & 3] * scale2 - m[u] : sc[u][e >> 2][e & 3];
                    if (it) by = 1.f, off = 0.f;
                }
#pragma unroll
                for (int e = 0; e < VK; ++e) {
                    p[u][e] = __builtin_amdgcn_exp2f(fmaf(sc[u][e >> 2][e & 3], by, -off));
                    if constexpr (F32) l[u] += p[u][e];
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < VK; ++e)
#pragma unroll
                    for (int x = 0; x < NV; ++x)
#pragma unroll
                        for (int u = 0; u < NQ; ++u)
                            o[u][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[e][x]), p[u][e], o[u][x], 0, 0, 0);
            } else if constexpr (KT == 16) {
                uint2 pb[NQ][2];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    split2<T>(p[u][0], p[u][1], pb[u][0].x, pb[u][1].x), split2<T>(p[u][2], p[u][3], pb[u][0].y, pb[u][1].y);
#pragma unroll
                    for (int e = 0; e < VK; ++e) l[u] += p[u][e];
                }
#pragma unroll
                for (int x = 0; x < NV; ++x) {
                    const unsigned sel = x & 1 ? 0x07060302u : 0x05040100u;
                    const uint2 vt = {__builtin_amdgcn_perm(v[1][x / 2], v[0][x / 2], sel), __builtin_amdgcn_perm(v[3][x / 2], v[2][x / 2], sel)};
#pragma unroll
                    for (int u = 0; u < NQ; ++u) o[u][x] = mfma_16x16x16<T>(vt, pb[u][0], mfma_16x16x16<T>(vt, pb[u][1], o[u][x]));
                }
            } else {
                uint4 pb[NQ][2];
#pragma unroll
                for (int u = 0; u < NQ; ++u) {
                    split2<T>(p[u][0], p[u][1], pb[u][0].x, pb[u][1].x), split2<T>(p[u][2], p[u][3], pb[u][0].y, pb[u][1].y);
                    split2<T>(p[u][4], p[u][5], pb[u][0].z, pb[u][1].z), split2<T>(p[u][6], p[u][7], pb[u][0].w, pb[u][1].w);
#pragma unroll
                    for (int e = 0; e < VK; ++e) l[u] += p[u][e];
                }
#pragma unroll
                for (int x = 0; x < NV; ++x) {
                    const unsigned sel = x & 1 ? 0x07060302u : 0x05040100u;
                    const uint4 vt = {__builtin_amdgcn_perm(v[1][x / 2], v[0][x / 2], sel), __builtin_amdgcn_perm(v[3][x / 2], v[2][x / 2], sel),
                                      __builtin_amdgcn_perm(v[5][x / 2], v[4][x / 2], sel), __builtin_amdgcn_perm(v[7][x / 2], v[6][x / 2], sel)};
#pragma unroll
                    for (int u = 0; u < NQ; ++u) o[u][x] = mfma_16x16x32<T>(vt, pb[u][0], mfma_16x16x32<T>(vt, pb[u][1], o[u][x]));
                }
            }
        }

        // join the waves: o [wave][row][DP + 4], then m, l [wave][row]
        constexpr int R = 16 * NQ, LDO = DP + 4;
        float *const ml = lds + waves * R * LDO;
        const bool redo = __syncthreads_or(odd);            // and the last row tile's readers are done
        if (redo) {
            for (int r = r0 + wave; r <= last; r += waves) {
                const int i = g.by_group.div(r), h = hk * g.group + r - i * g.group;
                Range see = seen_by(s, s.len - s.n + i, g.a.causal, g.a.window);
                see.begin = max(see.begin, lo), see.end = min(see.end, hi);
                attend_row<T>(g, b, hk, (const T *)g.a.q + (int64_t)(s.start + i) * g.a.q_tstride + (int64_t)h * g.a.q_hstride, see,
                              lds + (r - r0) * LDO, ml + 2 * (r - r0));
            }
        }
#pragma unroll
        for (int u = 0; u < NQ; ++u) {
            l[u] += __shfl_xor(l[u], 16);
            l[u] += __shfl_xor(l[u], 32);
            const int row = wave * R + 16 * u + c16;
            if (!redo && r0 + 16 * u + c16 <= last) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < NV; x += 4)
                        *(f32x4_t *)(lds + row * LDO + NV * (4 * g4 + i) + x) = f32x4_t{o[u][x][i], o[u][x + 1][i], o[u][x + 2][i], o[u][x + 3][i]};
                if (g4 == 0) ml[2 * row] = m[u], ml[2 * row + 1] = l[u];
            }
        }
        __syncthreads();
        join_waves<T, DP>(g, s, hk, split, lds, ml, r0, last - r0 + 1, R, redo ? 1 : waves);
    }
}

// One or two fp32 rows: the same stream without the matrix unit, whose fp32 products of 16 rows would leave 14 of them idle at 1152 cycles
// a tile of 16 keys of 64 channels, against some 330 here (one token over 605 keys of 16 heads of 64: 7.3 us a launch of a graph).  A lane holds
// four channels of every 64 of keys 4 (lane / 16) + i: whole rows of 16 lanes add up a score by rotation, so that the lanes of a key know
// it, and each 16 lanes keep a maximum, sum and output of their own until the end.
template <int DP, bool FULL, int R> __global__ __launch_bounds__(512) void attend_few(AttArgs g)
{
    constexpr int NX = DP / 64, KT = 16;
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int c16 = lane & 15, g4 = lane >> 4;
    const int hk = blockIdx.x / g.splits, split = blockIdx.x - hk * g.splits, b = blockIdx.z;
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, b);
    const int D = g.c.head_dim, rows = s.n * g.group;
    const char *kbase = (const char *)g.c.k + (int64_t)hk * g.c.k_head * 4, *vbase = (const char *)g.c.v + (int64_t)hk * g.c.v_head * 4;
    const bool vrole = lane >= 32;
    const uint32_t page16 = (uint32_t)((vrole ? g.c.v_page : g.c.k_page) / 4), row16 = (uint32_t)((vrole ? g.c.v_row : g.c.k_row) / 4);
    const float flip = g.scale2 < 0.f ? -1.f : g.scale2 == 0.f ? 0.f : 1.f, scale2 = g.scale2 == 0.f ? 1.f : fabsf(g.scale2);
    for (int r0 = blockIdx.y * R; r0 < rows; r0 += gridDim.y * R) {
        const int last = min(r0 + R, rows) - 1;
        Range mine[R], all = {0x7fffffff, 0}, both = {0, 0x7fffffff};            // what some row sees, what every row sees
        f32x4_t q[R][NX];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const int r = min(r0 + u, last), i = g.by_group.div(r), h = hk * g.group + r - i * g.group;
            mine[u] = seen_by(s, s.len - s.n + i, g.a.causal, g.a.window);
            all.begin = min(all.begin, mine[u].begin), all.end = max(all.end, mine[u].end);
            both.begin = max(both.begin, mine[u].begin), both.end = min(both.end, mine[u].end);
            const float *src = (const float *)g.a.q + (int64_t)(s.start + i) * g.a.q_tstride + (int64_t)h * g.a.q_hstride;
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                const int d = c16 * 4 + 64 * x;
                q[u][x] = FULL || d < D ? *(const f32x4_t *)(src + (FULL || d < D ? d : 0)) * flip : f32x4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
        const int64_t from = all.begin + (int64_t)split * g.split_keys, to = split + 1 < g.splits ? from + g.split_keys : all.end;
        const int lo = (int)min(from, (int64_t)all.end), hi = (int)min(to, (int64_t)all.end);
        f32x4_t o[R][NX], k[4][NX], v[4][NX];
        float m[R], l[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            m[u] = kNoMax, l[u] = 0.f;
#pragma unroll
            for (int x = 0; x < NX; ++x) o[u][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        const int step = waves * KT;
        int base = lo + wave * KT;
        bool far[R] = {};
        auto fetch = [&](int at, int &row) { return entry_of(g.b, g.by_page, b, min(at + c16, hi - 1), row); };
        auto place = [&](int at, int entry) { return at + c16 < hi && held(entry, g.c.pages) ? entry : -1; };
        // keys in lanes 0-15, values in 32-47: where the four of this lane's sixteen lie
        auto load = [&](f32x4_t(&to)[4][NX], const char *from, uint32_t off, int role) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const char *p = from + (uint64_t)(uint32_t)__shfl((int)off, role + 4 * g4 + i) * 16;
#pragma unroll
                for (int x = 0; x < NX; ++x) {
                    const int d = c16 * 4 + 64 * x;
                    to[i][x] = *(const f32x4_t *)(p + (FULL || d < D ? d * 4 : 0));
                    if (!FULL && d >= D) to[i][x] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                }
            }
        };
        int row_next = 0, entry_next = -1;
        uint32_t off = 0;
        unsigned ok = 0;
        if (base < hi) {
            int row;
            const int page = place(base, fetch(base, row));
            off = page < 0 ? 0 : (uint32_t)page * page16 + (uint32_t)row * row16;
            ok = (unsigned)__ballot(page >= 0) & 0xffffu;
            load(k, kbase, off, 0);
            entry_next = fetch(base + step, row_next);
        }
        for (; base < hi; base += step) {
            load(v, vbase, off, 32);
            const unsigned ok_now = ok;
            const int page = place(base + step, entry_next);
            off = page < 0 ? 0 : (uint32_t)page * page16 + (uint32_t)row_next * row16;
            ok = (unsigned)__ballot(page >= 0) & 0xffffu;
            entry_next = fetch(base + 2 * step, row_next);
            float sc[R][4];
#pragma unroll
            for (int u = 0; u < R; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = 0.f;
#pragma unroll
                    for (int y = 0; y < NX; ++y)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x = fmaf(q[u][y][e], k[i][y][e], x);
                    x += turned<8>(x), x += turned<4>(x), x += turned<2>(x), x += turned<1>(x);
                    sc[u][i] = x;
                }
            if (base + step < hi) load(k, kbase, off, 0);
            auto add = [&](auto whole) {                       // whole: every row sees every key of the tile
                constexpr bool ALL = decltype(whole)::value;
#pragma unroll
                for (int u = 0; u < R; ++u) {
                    const uint32_t bits = ALL ? ~0u : (uint32_t)seen_bits(ok_now, base, mine[u]) >> (4 * g4);
                    float top = kNoMax;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!ALL) sc[u][i] = masked(sc[u][i], bits, i);
                        top = fmaxf(top, sc[u][i] * scale2);
                    }
                    if (__any(top > m[u] + lazy<float>())) {
                        const float to = fmaxf(m[u], top), fade = __builtin_amdgcn_exp2f(m[u] - to);
                        m[u] = to, l[u] *= fade;
#pragma unroll
                        for (int x = 0; x < NX; ++x) o[u][x] *= fade;
                        far[u] = __any(is_far(to));
                    }
                    float by = scale2, off = m[u];
                    if (far[u]) {
                        const bool it = is_far(m[u]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[u][i] = it ? sc[u][i] * scale2 - m[u] : sc[u][i];
                        if (it) by = 1.f, off = 0.f;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(sc[u][i], by, -off));
                        l[u] += p;
#pragma unroll
                        for (int x = 0; x < NX; ++x)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                // a key that is not seen takes no part, whatever its value holds
                                const float value = ALL || (bits >> i & 1) ? v[i][x][e] : 0.f;
                                o[u][x][e] = fmaf(p, value, o[u][x][e]);
                            }
                    }
                }
            };
            if (ok_now == 0xffffu && base >= both.begin && base + KT <= both.end) add(std::true_type());
            else add(std::false_type());
        }
        // join the 16 lanes' results of a wave, then the waves
        constexpr int LDO = DP + 4;
        float *const ml = lds + waves * R * LDO;
        __syncthreads();                                    // the last rows' readers are done
#pragma unroll
        for (int u = 0; u < R; ++u) {
            float top = fmaxf(m[u], __shfl_xor(m[u], 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float f = __builtin_amdgcn_exp2f(m[u] - top);
            float sum = l[u] * f;
            sum += __shfl_xor(sum, 16), sum += __shfl_xor(sum, 32);
#pragma unroll
            for (int x = 0; x < NX; ++x) {
                f32x4_t y = o[u][x] * f;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], 16), y[e] += __shfl_xor(y[e], 32);
                if (g4 == 0) *(f32x4_t *)(lds + (wave * R + u) * LDO + c16 * 4 + 64 * x) = y;
            }
            if (lane == 0) ml[2 * (wave * R + u)] = top, ml[2 * (wave * R + u) + 1] = sum;
        }
        __syncthreads();
        join_waves<float, DP>(g, s, hk, split, lds, ml, r0, last - r0 + 1, R, waves);
    }
}

// Joins the splits: a thread owns eight channels of a row (token, head) and every lanes-th split of it; the lanes of a row are added
// up in LDS, in their order.  lanes: a power of two, lanes * head_dim / 8 <= 256.
template <class T> __global__ __launch_bounds__(256) void join_splits(AttArgs g, int lanes)
{
    constexpr int ES = sizeof(T);
    __shared__ float lds[256 * 9];
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, blockIdx.y);
    const int D = g.c.head_dim, cols = D / 8, team = cols * lanes, teams = 256 / team;
    const int mine = threadIdx.x / team, in_team = threadIdx.x - mine * team, lane = in_team / cols, col = in_team - lane * cols, d = col * 8;
    const int64_t rows = (int64_t)s.n * g.a.q_heads;
    for (int64_t r0 = (int64_t)blockIdx.x * teams; r0 < rows; r0 += (int64_t)gridDim.x * teams) {
        const int64_t row = r0 + mine;
        const bool in = mine < teams && row < rows;
        const int64_t at = ((int64_t)s.start * g.a.q_heads + row) * g.splits;
        float top = kNoMax, all[9] = {};
        if (in) {
            for (int x = lane; x < g.splits; x += lanes) top = fmaxf(top, g.stat[2 * (at + x)]);
#pragma unroll 2
            for (int x = lane; x < g.splits; x += lanes) {
                const float f = __builtin_amdgcn_exp2f(g.stat[2 * (at + x)] - top);
                const f32x4_t a0 = *(const f32x4_t *)(g.part + (at + x) * D + d), a1 = *(const f32x4_t *)(g.part + (at + x) * D + d + 4);
#pragma unroll
                for (int y = 0; y < 4; ++y) all[y] = fmaf(f, a0[y], all[y]), all[4 + y] = fmaf(f, a1[y], all[4 + y]);
                all[8] = fmaf(f, g.stat[2 * (at + x) + 1], all[8]);
            }
        }
        if (lanes > 1) {
            // each lane has a maximum of its own: brought to the largest first
            const int base = mine * team + col;
            __syncthreads();
            lds[threadIdx.x * 9 + 8] = top;
            __syncthreads();
            float best = top;
            if (in)
                for (int x = 0; x < lanes; ++x) best = fmaxf(best, lds[(base + x * cols) * 9 + 8]);
            const float f = __builtin_amdgcn_exp2f(top - best);
            __syncthreads();
#pragma unroll
            for (int y = 0; y < 9; ++y) lds[threadIdx.x * 9 + y] = all[y] * f, all[y] = 0.f;
            __syncthreads();
            if (in && lane == 0)
                for (int x = 0; x < lanes; ++x)
#pragma unroll
                    for (int y = 0; y < 9; ++y) all[y] += lds[(base + x * cols) * 9 + y];
        }
        if (in && lane == 0) {
            alignas(16) T out[8];
            const float inv = all[8] > 0.f ? 1.f / all[8] : all[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) out[y] = (T)(all[y] * inv);
            const int64_t token = s.start + row / g.a.q_heads;
            T *dst = (T *)g.a.out + token * g.a.o_tstride + (row % g.a.q_heads) * g.a.o_hstride + d;
#pragma unroll
            for (int y = 0; y < 8 * ES / 16; ++y) ((uint4 *)dst)[y] = ((const uint4 *)out)[y];
        }
    }
}

}  // namespace ttsamd
