// Attention of many fp32 rows over a paged cache: paged_tile.h with every operand in three bf16 parts.
//
// The fp32 products of the matrix unit run at a sixteenth of the bf16 rate.  x = x0 + x1 + x2 with xi the nearest bf16 to what is left:
// |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x|, and x0..x2 together hold all 24 bits.  A product keeps the six terms xi yj with i + j <= 2, summed
// in fp32; what is dropped is at most 2^-23 |x y|, two roundings of an fp32 product.  The scores' and the values' products are taken so,
// the probabilities split like the rest; maximum, exponential and sums are fp32.
// Keys and values are split once for a workgroup's rows, on their way into LDS (32 at a time, a plane a part, planes permuted as in
// paged_tile.h).  An infinity would leave NaN behind in its parts: where one is met (it shows in what is left after x0), the rows are
// computed again key by key.
//
// Bound: the instructions issued, matrix ones (36 cycles each, 48 of them a wave for 32 keys of 64 channels) and others (4) one after
// the other: about 3200 cycles, against 6200 with the fp32 products (one chunk of 700 tokens over 2048 keys, 16 heads of 64: 79 -> 53 us; two
// ragged prompts of up to 437: 21 us).
#pragma once
#include "paged_tile.h"

namespace ttsamd {

// Eight floats as three pieces of eight bf16; `left` becomes NaN if one of them is an infinity or NaN.
__device__ __forceinline__ void split3(const float (&x)[8], uint4 (&part)[3], float &left)
{
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = pack2<__bf16>(r[2 * e], r[2 * e + 1]);
            if (p < 2) r[2 * e] -= __uint_as_float(w[e] << 16), r[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
            if (p == 0) left = fmaf(r[2 * e], 0.f, fmaf(r[2 * e + 1], 0.f, left));
        }
        part[p] = uint4{w[0], w[1], w[2], w[3]};
    }
}
__device__ __forceinline__ void split3(uint4 a, uint4 b, uint4 (&part)[3], float &left)
{
    const float x[8] = {__uint_as_float(a.x), __uint_as_float(a.y), __uint_as_float(a.z), __uint_as_float(a.w),
                        __uint_as_float(b.x), __uint_as_float(b.y), __uint_as_float(b.z), __uint_as_float(b.w)};
    split3(x, part, left);
}
// c + the six leading terms, the small ones first.
__device__ __forceinline__ f32x16_t mfma_three(const uint4 (&a)[3], const uint4 (&b)[3], f32x16_t c)
{
    c = mfma_32x32x16<__bf16>(a[2], b[0], c);
    c = mfma_32x32x16<__bf16>(a[0], b[2], c);
    c = mfma_32x32x16<__bf16>(a[1], b[1], c);
    c = mfma_32x32x16<__bf16>(a[1], b[0], c);
    c = mfma_32x32x16<__bf16>(a[0], b[1], c);
    return mfma_32x32x16<__bf16>(a[0], b[0], c);
}

template <int DC, bool FULL, int RW, int KG> __global__ __launch_bounds__(64 * RW * KG, DC > 64 ? 1 : 2) void attend_tile3(AttArgs g)
{
    // DC channels are computed, of rows of DP in LDS
    constexpr int DP = tile3_pitch(DC), CH = DP / 8, RB = DP * 2, PLANE = kTile3Keys * RB, NST = kTile3Keys * CH / (64 * RW), kTileRows = 32 * RW, NS = DC / 16,
                  ND = DC / 32;
    constexpr bool WHOLE = FULL && DC == DP;
    extern __shared__ float lds_f[];
    char *const lds = (char *)lds_f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % RW), c32 = lane & 31, h2 = lane >> 5;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * RW)), member = threadIdx.x % (64 * RW);       // KG teams of RW waves take the tiles in turn
    char *const mem = lds + team * 12 * PLANE;
    const int hk = blockIdx.x / g.splits, split = blockIdx.x - hk * g.splits, b = blockIdx.z;
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, b);
    const int D = g.c.head_dim, rows = s.n * g.group, tiles = (rows + kTileRows - 1) / kTileRows;
    const char *kbase = (const char *)g.c.k + (int64_t)hk * g.c.k_head * 4, *vbase = (const char *)g.c.v + (int64_t)hk * g.c.v_head * 4;
    const uint32_t page16 = (uint32_t)((h2 ? g.c.v_page : g.c.k_page) / 4), row16 = (uint32_t)((h2 ? g.c.v_row : g.c.k_row) / 4);
    // within eight pieces where their number is no power of two (rows of 192 channels start at two places of the banks in turn)
    auto k_swz = [](int row) { return CH == 8 ? (row & 7) ^ (row >> 3 & 1) : CH == 16 ? row & 15 : row >> 1 & 7; };
    auto v_swz = [](int row) { return CH == 8 ? (row & 3) << 1 : CH == 16 ? (row & 1) << 2 | (row & 2) * 5 : (row & 2) << 1; };
    const int i16 = lane & 15, vr = 4 * h2 + (i16 >> 2), vc = 2 * (lane >> 4 & 1) + (i16 >> 1 & 1), vb8 = (i16 & 1) * 8;
    const float flip = g.scale2 < 0.f ? -1.f : g.scale2 == 0.f ? 0.f : 1.f, scale2 = g.scale2 == 0.f ? 1.f : fabsf(g.scale2);

    for (int tile = tiles - 1 - blockIdx.y; tile >= 0; tile -= gridDim.y) {         // the longest first
        const int r0 = tile * kTileRows, last = min(r0 + kTileRows, rows) - 1, w0 = min(r0 + 32 * wave, last), w1 = min(r0 + 32 * wave + 31, last);
        auto range_of = [&](int r) { return seen_by(s, s.len - s.n + (int)g.by_group.div(r), g.a.causal, g.a.window); };
        const int my_row = min(r0 + 32 * wave + c32, last), my_i = g.by_group.div(my_row), my_h = hk * g.group + my_row - my_i * g.group;
        const Range mine = range_of(my_row), wfirst = range_of(w0), wlast = range_of(w1), first = range_of(r0), final = range_of(last);
        float left = 0.f;                                    // NaN once an infinity or NaN was met
        uint4 q[NS][3];
        {
            const float *src = (const float *)g.a.q + (int64_t)(s.start + my_i) * g.a.q_tstride + (int64_t)my_h * g.a.q_hstride;
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = x * 16 + h2 * 8 + e;
                    f[e] = FULL || d < D ? src[d] * flip : 0.f;
                }
                split3(f, q[x], left);
            }
        }
        f32x16_t o[ND];
#pragma unroll
        for (int x = 0; x < ND; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) o[x][y] = 0.f;
        float m = kNoMax, l = 0.f;
        bool far = false;

        const int64_t from = first.begin + (int64_t)split * g.split_keys, to = split + 1 < g.splits ? from + g.split_keys : final.end;
        const int lo = (int)min(from, (int64_t)final.end), hi = (int)min(to, (int64_t)final.end);
        uint4 sk[NST][2], sv[NST][2];
        // the table's entry for this lane's key (c32) of the tile at `at`, still on its way; what it is worth once it is there
        auto fetch = [&](int at, int &row) { return entry_of(g.b, g.by_page, b, min(at + c32, hi - 1), row); };
        auto place = [&](int at, int entry) { return at + c32 < hi && held(entry, g.c.pages) ? entry : -1; };
        auto stage = [&](int page, int row) {
            const uint32_t off = page < 0 ? 0 : (uint32_t)page * page16 + (uint32_t)row * row16;      // keys in lanes 0-31, values in 32-63
#pragma unroll
            for (int x = 0; x < NST; ++x) {
                const int i = x * 64 * RW + member, r = i / CH, piece = i % CH, at = WHOLE || piece * 8 < D ? piece * 32 : 0;
                const uint4 *ks = (const uint4 *)(kbase + (uint64_t)(uint32_t)__shfl((int)off, r) * 16 + at);
                const uint4 *vs = (const uint4 *)(vbase + (uint64_t)(uint32_t)__shfl((int)off, 32 + r) * 16 + at);
                sk[x][0] = ks[0], sk[x][1] = ks[1], sv[x][0] = vs[0], sv[x][1] = vs[1];
            }
        };
        auto put = [&](char *buf, uint32_t ok) {
#pragma unroll
            for (int x = 0; x < NST; ++x) {
                const int i = x * 64 * RW + member, r = i / CH, piece = i % CH;
                if (!(ok >> r & 1) || (!WHOLE && piece * 8 >= D)) sk[x][0] = sk[x][1] = sv[x][0] = sv[x][1] = uint4{0, 0, 0, 0};
                uint4 part[3];
                split3(sk[x][0], sk[x][1], part, left);
#pragma unroll
                for (int p = 0; p < 3; ++p) *(uint4 *)(buf + p * PLANE + r * RB + (piece ^ k_swz(r)) * 16) = part[p];
                split3(sv[x][0], sv[x][1], part, left);
#pragma unroll
                for (int p = 0; p < 3; ++p) *(uint4 *)(buf + (3 + p) * PLANE + r * RB + (piece ^ v_swz(r)) * 16) = part[p];
            }
        };

        int cur = 0, page_next = -1, row_next = 0;
        uint32_t ok = 0;
        constexpr int step = KG * kTile3Keys;
        const int begin = lo + team * kTile3Keys;
        __syncthreads();                                     // the last row tile's readers are done
        if (begin < hi) {
            int row;
            const int page = place(begin, fetch(begin, row));
            ok = (uint32_t)__ballot(page >= 0);
            page_next = fetch(begin + step, row_next);
            stage(page, row);
            put(mem, ok);
        }
        for (int base0 = lo; base0 < hi; base0 += step) {
            __syncthreads();
            const int base = base0 + team * kTile3Keys;
            const char *kb = mem + cur * 6 * PLANE, *vb = kb + 3 * PLANE;
            const uint32_t ok_now = ok;
            const bool more = base + step < hi;
            if (more) {
                const int page = place(base + step, page_next);
                ok = (uint32_t)__ballot(page >= 0);
                stage(page, row_next);
                page_next = fetch(base + 2 * step, row_next);
            }
            if (base < hi && base < wlast.end && base + kTile3Keys > wfirst.begin) {
                f32x16_t sc;
#pragma unroll
                for (int y = 0; y < 16; ++y) sc[y] = 0.f;
                const char *kr = kb + c32 * RB;
                const int kswz = k_swz(c32);
                auto k_piece = [&](int x, uint4 (&f)[3]) {
#pragma unroll
                    for (int p = 0; p < 3; ++p) f[p] = *(const uint4 *)(kr + p * PLANE + ((2 * x + h2) ^ kswz) * 16);
                };
                uint4 kf[2][3];
                k_piece(0, kf[0]);
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                    __builtin_amdgcn_sched_barrier(0);       // in this order: the reads stay a step ahead of the products
                    if (x + 1 < NS) k_piece(x + 1, kf[(x + 1) & 1]);
                    sc = mfma_three(kf[x & 1], q[x], sc);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (ok_now != ~0u || base < wlast.begin || base + kTile3Keys > wfirst.end) {
                    const uint32_t bits = (uint32_t)seen_bits(ok_now, base, mine) >> (4 * h2);
#pragma unroll
                    for (int y = 0; y < 16; ++y) sc[y] = masked(sc[y], bits, 8 * (y >> 2) + (y & 3));
                }
                float top = sc[0];
#pragma unroll
                for (int y = 1; y < 16; ++y) top = fmaxf(top, sc[y]);
                top *= scale2;
                if (__any(top > m + lazy<float>())) {
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float to = fmaxf(m, top), fade = __builtin_amdgcn_exp2f(m - to);
                    m = to, l *= fade;
#pragma unroll
                    for (int x = 0; x < ND; ++x) o[x] *= fade;
                    far = __any(is_far(to));
                }
                float by = scale2, off = m;
                if (far) {
                    const bool it = is_far(m);
#pragma unroll
                    for (int y = 0; y < 16; ++y) sc[y] = it ? sc[y] * scale2 - m : sc[y];
                    if (it) by = 1.f, off = 0.f;
                }
                const char *vrow = vb + vr * RB + vb8;
                const int vswz = v_swz(vr);
                auto v_piece = [&](int i, uint4 (&f)[3]) {
                    typedef short s4 __attribute__((ext_vector_type(4)));
#pragma unroll
                    for (int p = 0; p < 3; ++p) {
                        const char *at = vrow + p * PLANE + 16 * (i / ND) * RB + ((4 * (i % ND) + vc) ^ vswz) * 16;
                        const uint2 lower = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at));
                        const uint2 upper = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(at + 8 * RB)));
                        f[p] = uint4{lower.x, lower.y, upper.x, upper.y};
                    }
                };
                uint4 vf[2][3], pb[2][3];
                v_piece(0, vf[0]);
                float unused = 0.f;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float p[8];
#pragma unroll
                    for (int y = 0; y < 8; ++y) {
                        p[y] = __builtin_amdgcn_exp2f(fmaf(sc[8 * u + y], by, -off));
                        l += p[y];
                    }
                    split3(p, pb[u], unused);
                }
#pragma unroll
                for (int i = 0; i < 2 * ND; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (i + 1 < 2 * ND) v_piece(i + 1, vf[(i + 1) & 1]);
                    o[i % ND] = mfma_three(vf[i & 1], pb[i / ND], o[i % ND]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            cur ^= 1;
            if (more) put(mem + cur * 6 * PLANE, ok);
        }
        const bool redo = __syncthreads_or(left != left);
        l += __shfl_xor(l, 32);
        if constexpr (KG == 2)
            if (!redo) join_teams<ND>(lds_f, team, wave, lane, m, l, o);
        if (!redo && team == 0) {
            if (r0 + 32 * wave + c32 <= last) {
                const int64_t token = s.start + my_i, at = (token * g.a.q_heads + my_h) * g.splits + split;
                const float inv = l > 0.f ? 1.f / l : l;      // no key: zeros; NaN stays
                float *dst = (float *)g.a.out + token * g.a.o_tstride + (int64_t)my_h * g.a.o_hstride;
#pragma unroll
                for (int x = 0; x < ND; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int d = 32 * x + 8 * y + 4 * h2;
                        if (!FULL && d >= D) continue;
                        const f32x4_t v = {o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]};
                        if (g.splits > 1) *(f32x4_t *)(g.part + at * D + d) = v;
                        else *(f32x4_t *)(dst + d) = v * inv;
                    }
                if (g.splits > 1 && h2 == 0) g.stat[2 * at] = m, g.stat[2 * at + 1] = l;
            }
        } else if (redo) {
            float *const mine_o = lds_f + (team * RW + wave) * 264;
            for (int r = r0 + team * RW + wave; r <= last; r += RW * KG) {
                const int i = g.by_group.div(r), h = hk * g.group + r - i * g.group;
                const int64_t token = s.start + i, at = (token * g.a.q_heads + h) * g.splits + split;
                Range see = range_of(r);
                see.begin = max(see.begin, lo), see.end = min(see.end, hi);
                const float sum = attend_row<float>(g, b, hk, (const float *)g.a.q + token * g.a.q_tstride + (int64_t)h * g.a.q_hstride, see,
                                                    mine_o, mine_o + 256);
                const float inv = sum > 0.f ? 1.f / sum : sum;
                float *dst = (float *)g.a.out + token * g.a.o_tstride + (int64_t)h * g.a.o_hstride;
                for (int d = lane; d < D; d += 64) {
                    if (g.splits > 1) g.part[at * D + d] = mine_o[d];
                    else dst[d] = mine_o[d] * inv;
                }
                if (g.splits > 1 && lane == 0) g.stat[2 * at] = mine_o[256], g.stat[2 * at + 1] = sum;
            }
        }
    }
}

}  // namespace ttsamd
