// Attention of many rows over a paged cache (chunks of a prompt), 16-bit types: keys and values staged through LDS for 32 RW rows.
//
// A team of RW waves takes 32 rows a wave (row = token x heads of one key head, as in paged_stream.h) and walks the keys 64 at a time;
// KG teams of a workgroup take the tiles of the same rows in turn and are joined in LDS.
// As there, S^T = K Q^T is computed, here in 32x32x16 products: a lane holds one row (column lane % 32) and half of a tile's keys, the
// probabilities are the right operand of O^T = V^T P^T where they lie (slot e of half h of product u is key 16 u + 4 h + e, + 4 for
// e >= 4), and V^T comes out of LDS by the transposing read, four keys of a channel at a time.
//
// LDS.  Two buffers of 64 key rows and 64 value rows: while a tile is multiplied the next one's keys, then its values, travel through
// registers into the other buffer; one barrier a tile.  A row's 16-byte pieces are permuted by an exclusive or with a function of the row,
// so that the reads of 8 (and 16) neighbouring lanes fall on different banks: keys are read a piece a row down a column, values 32 (64)
// bytes of four rows.
//
// The probabilities are rounded to the type for the second product, numerator and denominator alike: a result is off by up to half a step
// of the type of sum p |v|, as large as its own rounding (bf16, two chunks of 2048 behind 6143 others: 0.0017 -> 0.0023 of its size in the
// mean).  A second part, as paged_stream.h takes one, would cost another product for every two: 571 -> 713 us there, 46 -> 55 us for 1000
// tokens over 2000 keys.
//
// Bound: the issue of instructions, 36 cycles a matrix one and 4 any other (the matrix unit is busy for some 40 % of the time, no bank
// conflicts): two chunks of 2048 bf16 tokens behind 6143 others, 32 heads over 8 of 128: 402 GFLOP in 440 to 470 us a call, 860 to 910
// TFLOP/s (526 in the median of a trace: the clock gives way), where 392 us are the sum of its instructions at the full clock.  Reads AHEAD by 2, 3 or 6 products instead of 4, eight waves a workgroup and raised wave priorities gave
// nothing.
#pragma once
#include "paged_launch.h"

namespace ttsamd {

template <class T> __device__ __forceinline__ f32x16_t mfma_32x32x16(uint4 a, uint4 b, f32x16_t c)
{
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Team 1 hands its running maximum, sum and output to team 0, wave by wave and register by register; all waves of the workgroup call it.
template <int ND> __device__ __forceinline__ void join_teams(float *lds, int team, int wave, int lane, float &m, float &l, f32x16_t (&o)[ND])
{
    float *const mine = lds + wave * (ND * 16 + 2) * 64 + lane;
    if (team == 1) {
#pragma unroll
        for (int x = 0; x < ND; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) mine[(x * 16 + y) * 64] = o[x][y];
        mine[ND * 16 * 64] = m, mine[(ND * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (team == 0) {
        const float m2 = mine[ND * 16 * 64], to = fmaxf(m, m2), f = __builtin_amdgcn_exp2f(m - to), f2 = __builtin_amdgcn_exp2f(m2 - to);
        m = to, l = l * f + mine[(ND * 16 + 1) * 64] * f2;
#pragma unroll
        for (int x = 0; x < ND; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) o[x][y] = o[x][y] * f + mine[(x * 16 + y) * 64] * f2;
    }
}

template <class T, int DC, bool FULL, int RW, int KG>
__global__ __launch_bounds__(64 * RW * KG, DC > 128 || (DC > 64 && RW == 2) ? 1 : 2) void attend_tile(AttArgs g)
{
    // DC channels are computed, of rows of DP in LDS
    constexpr int DP = padded_pow2(DC), CH = DP / 8, RB = DP * 2, NSTG = CH / RW, kTileRows = 32 * RW, RPI = 64 / CH, NS = DC / 16,
                  ND = DC / 32, AHEAD = 4;
    constexpr int HALF = kTileKeys * RB;                    // bytes of a tile's keys (or values)
    extern __shared__ float lds_f[];
    char *const lds = (char *)lds_f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) % RW), c32 = lane & 31, h2 = lane >> 5;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * RW));               // KG teams of RW waves take the tiles in turn
    char *const mem = lds + team * 4 * HALF;
    const int hk = blockIdx.x / g.splits, split = blockIdx.x - hk * g.splits, b = blockIdx.z;
    const Sequence s = sequence_of(g.b, g.a.tokens, g.c.page_size, b);
    const int D = g.c.head_dim, rows = s.n * g.group, tiles = (rows + kTileRows - 1) / kTileRows;
    const char *kbase = (const char *)g.c.k + (int64_t)hk * g.c.k_head * 2, *vbase = (const char *)g.c.v + (int64_t)hk * g.c.v_head * 2;
    const uint32_t kpage16 = (uint32_t)(g.c.k_page / 8), krow16 = (uint32_t)(g.c.k_row / 8);
    const uint32_t vpage16 = (uint32_t)(g.c.v_page / 8), vrow16 = (uint32_t)(g.c.v_row / 8);
    auto k_swz = [](int row) { return CH == 8 ? (row & 7) ^ (row >> 3 & 1) : row & 15; };
    auto v_swz = [](int row) { return CH == 8 ? (row & 3) << 1 : (row & 1) << 2 | (row & 2) * 5; };     // 0 4 10 14

    // staging: this thread's piece of NSTG rows
    const int piece = lane % CH, row_of_lane = lane / CH;
    constexpr bool WHOLE = FULL && DC == DP;
    const bool piece_in = WHOLE || piece * 8 < D;
    const char *kbase_l = kbase + (piece_in ? piece * 16 : 0), *vbase_l = vbase + (piece_in ? piece * 16 : 0);
    // reading: a key row per lane; four value rows and a 32-byte span per 16 lanes
    const int i16 = lane & 15, vr = 4 * h2 + (i16 >> 2), vc = 2 * (lane >> 4 & 1) + (i16 >> 1 & 1), vb8 = (i16 & 1) * 8;

    // the largest score is found before the scale: it has to be positive (a negative one turns q's sign, zero takes q away)
    const unsigned flip = g.scale2 < 0.f ? 0x80008000u : 0u, keep = g.scale2 == 0.f ? 0u : ~0u;
    const float scale2 = g.scale2 == 0.f ? 1.f : fabsf(g.scale2);
    for (int tile = tiles - 1 - blockIdx.y; tile >= 0; tile -= gridDim.y) {         // the longest first
        const int r0 = tile * kTileRows, last = min(r0 + kTileRows, rows) - 1, w0 = min(r0 + 32 * wave, last), w1 = min(r0 + 32 * wave + 31, last);
        auto range_of = [&](int r) { return seen_by(s, s.len - s.n + (int)g.by_group.div(r), g.a.causal, g.a.window); };
        const int my_row = min(r0 + 32 * wave + c32, last), my_i = g.by_group.div(my_row), my_h = hk * g.group + my_row - my_i * g.group;
        const Range mine = range_of(my_row), wfirst = range_of(w0), wlast = range_of(w1), first = range_of(r0), final = range_of(last);
        uint4 q[NS];
        {
            const char *src = (const char *)g.a.q + ((int64_t)(s.start + my_i) * g.a.q_tstride + (int64_t)my_h * g.a.q_hstride) * 2;
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                const bool in = FULL || x * 16 + h2 * 8 < D;
                q[x] = in ? *(const uint4 *)(src + (in ? x * 32 + h2 * 16 : 0)) : uint4{0, 0, 0, 0};
                q[x].x = (q[x].x & keep) ^ flip, q[x].y = (q[x].y & keep) ^ flip, q[x].z = (q[x].z & keep) ^ flip, q[x].w = (q[x].w & keep) ^ flip;
            }
        }
        f32x16_t o[ND];
#pragma unroll
        for (int x = 0; x < ND; ++x)
#pragma unroll
            for (int y = 0; y < 16; ++y) o[x][y] = 0.f;
        float m = kNoMax, l = 0.f;
        bool odd = false, far = false;

        const int64_t from = first.begin + (int64_t)split * g.split_keys, to = split + 1 < g.splits ? from + g.split_keys : final.end;
        const int lo = (int)min(from, (int64_t)final.end), hi = (int)min(to, (int64_t)final.end);
        uint4 st[NSTG];                                      // what travels: keys first, then values
        // the table's entry for this lane's key of the tile at `at`, still on its way; what it is worth once it is there
        auto fetch = [&](int at, int &row) { return entry_of(g.b, g.by_page, b, min(at + lane, hi - 1), row); };
        auto place = [&](int at, int entry) { return at + lane < hi && held(entry, g.c.pages) ? entry : -1; };
        auto stage = [&](const char *src, uint32_t off) {
#pragma unroll
            for (int x = 0; x < NSTG; ++x) st[x] = *(const uint4 *)(src + (uint64_t)(uint32_t)__shfl((int)off, (x * RW + wave) * RPI + row_of_lane) * 16);
        };
        auto k_off = [&](int page, int row) { return page < 0 ? 0 : (uint32_t)page * kpage16 + (uint32_t)row * krow16; };
        auto v_off = [&](int page, int row) { return page < 0 ? 0 : (uint32_t)page * vpage16 + (uint32_t)row * vrow16; };
        auto put_k = [&](char *buf) {
#pragma unroll
            for (int x = 0; x < NSTG; ++x) {
                const int r = (x * RW + wave) * RPI + row_of_lane;
                if (!WHOLE && !piece_in) st[x] = uint4{0, 0, 0, 0};
                *(uint4 *)(buf + r * RB + ((piece ^ k_swz(r)) & (CH - 1)) * 16) = st[x];
            }
        };
        auto put_v = [&](char *buf, uint64_t ok, bool mixed) {
            if (mixed) {
#pragma unroll
                for (int x = 0; x < NSTG; ++x) {
                    if (!(ok >> ((x * RW + wave) * RPI + row_of_lane) & 1)) st[x] = uint4{0, 0, 0, 0};
                    odd |= any_odd<T>(st[x].x) || any_odd<T>(st[x].y) || any_odd<T>(st[x].z) || any_odd<T>(st[x].w);
                }
            }
#pragma unroll
            for (int x = 0; x < NSTG; ++x) {
                const int r = (x * RW + wave) * RPI + row_of_lane;
                if (!WHOLE && !piece_in) st[x] = uint4{0, 0, 0, 0};
                *(uint4 *)(buf + HALF + r * RB + ((piece ^ v_swz(r)) & (CH - 1)) * 16) = st[x];
            }
        };
        auto mixed_at = [&](int at, uint64_t ok) { return ok != ~0ull || at < final.begin || at + kTileKeys > first.end; };

        int cur = 0, page_next = -1, row_next = 0;
        uint64_t ok = 0;
        constexpr int step = KG * kTileKeys;
        const int begin = lo + team * kTileKeys;
        __syncthreads();                                     // the last row tile's readers are done
        if (begin < hi) {
            int row;
            const int page = place(begin, fetch(begin, row));
            ok = __ballot(page >= 0);
            page_next = fetch(begin + step, row_next);
            stage(kbase_l, k_off(page, row));
            put_k(mem);
            stage(vbase_l, v_off(page, row));
            put_v(mem, ok, mixed_at(begin, ok));
        }
        for (int base0 = lo; base0 < hi; base0 += step) {
            __syncthreads();
            const int base = base0 + team * kTileKeys;
            const char *kb = mem + cur * 2 * HALF, *vb = kb + HALF;
            char *const next = mem + (cur ^ 1) * 2 * HALF;
            const uint64_t ok_now = ok;
            const bool more = base + step < hi, busy = base < hi && base < wlast.end && base + kTileKeys > wfirst.begin;
            uint32_t voff = 0;
            if (more) {
                const int page = place(base + step, page_next);
                ok = __ballot(page >= 0);
                stage(kbase_l, k_off(page, row_next));
                voff = v_off(page, row_next);
                page_next = fetch(base + 2 * step, row_next);
            }
            f32x16_t sc[2];
            if (busy) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int y = 0; y < 16; ++y) sc[t][y] = 0.f;
                const char *kr = kb + c32 * RB;
                const int kswz = k_swz(c32);                 // rows 32 apart are permuted alike
                auto k_piece = [&](int i) { return *(const uint4 *)(kr + (i & 1) * 32 * RB + (((i & ~1) + h2) ^ kswz) * 16); };
                uint4 kf[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) kf[i] = k_piece(i);
#pragma unroll
                for (int i = 0; i < 2 * NS; ++i) {
                    __builtin_amdgcn_sched_barrier(0);       // in this order: the reads stay AHEAD products ahead
                    sc[i & 1] = mfma_32x32x16<T>(kf[i % AHEAD], q[i >> 1], sc[i & 1]);
                    if (i + AHEAD < 2 * NS) kf[i % AHEAD] = k_piece(i + AHEAD);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (more) {
                put_k(next);
                stage(vbase_l, voff);
            }
            if (busy) {
                // slot y of half h2 of tile t: key 32 t + 8 (y / 4) + 4 h2 + y % 4
                if (ok_now != ~0ull || base < wlast.begin || base + kTileKeys > wfirst.end) {
                    const uint64_t bits = seen_bits(ok_now, base, mine) >> (4 * h2);
#pragma unroll
                    for (int y = 0; y < 32; ++y) sc[y >> 4][y & 15] = masked(sc[y >> 4][y & 15], (uint32_t)(bits >> (y & 16 ? 32 : 0)), 8 * (y >> 2 & 3) + (y & 3));
                }
                float top = sc[0][0];
#pragma unroll
                for (int y = 1; y < 32; ++y) top = fmaxf(top, sc[y >> 4][y & 15]);
                top *= scale2;
                if (__any(top > m + (lift<T>() + lazy<T>()))) {
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float to = fmaxf(m, top - lift<T>()), fade = __builtin_amdgcn_exp2f(m - to);
                    m = to, l *= fade;
#pragma unroll
                    for (int x = 0; x < ND; ++x) o[x] *= fade;
                    far = __any(is_far(to));
                }
                float by = scale2, off = m;
                if (far) {
                    const bool it = is_far(m);
#pragma unroll
                    for (int y = 0; y < 32; ++y) sc[y >> 4][y & 15] = it ? sc[y >> 4][y & 15] * scale2 - m : sc[y >> 4][y & 15];
                    if (it) by = 1.f, off = 0.f;
                }
                typedef short s4 __attribute__((ext_vector_type(4)));
                const char *vrow = vb + vr * RB + vb8;
                const int vswz = v_swz(vr);                  // rows four apart are permuted alike
                // the left operand of product i = u * ND + x: sixteen keys of 32 channels
                auto v_piece = [&](int i) {
                    const char *at = vrow + 16 * (i / ND) * RB + ((4 * (i % ND) + vc) ^ vswz) * 16;
                    const uint2 lower = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)at));
                    const uint2 upper = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(at + 8 * RB)));
                    return uint4{lower.x, lower.y, upper.x, upper.y};
                };
                // two of a group's eight probabilities, rounded
                auto p_pair = [&](int u, int y) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[u >> 1][(u & 1) * 8 + 2 * y], by, -off));
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[u >> 1][(u & 1) * 8 + 2 * y + 1], by, -off));
                    return pack2<T>(p0, p1);
                };
                unsigned pb[2][4];
                uint4 vf[AHEAD];
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) vf[i] = v_piece(i);
#pragma unroll
                for (int y = 0; y < 4; ++y) pb[0][y] = p_pair(0, y);
#pragma unroll
                for (int i = 0; i < 4 * ND; ++i) {
                    const int u = i / ND, x = i % ND;
                    __builtin_amdgcn_sched_barrier(0);
                    o[x] = mfma_32x32x16<T>(vf[i % AHEAD], uint4{pb[u & 1][0], pb[u & 1][1], pb[u & 1][2], pb[u & 1][3]}, o[x]);
                    if (i + AHEAD < 4 * ND) vf[i % AHEAD] = v_piece(i + AHEAD);
                    // while it runs: a share of the next group's probabilities, and this one's sum
#pragma unroll
                    for (int y = x * 4 / ND; y < (x + 1) * 4 / ND; ++y) {
                        if (u < 3) pb[(u + 1) & 1][y] = p_pair(u + 1, y);
                        l = sum2<T>(pb[u & 1][y], l);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (more) put_v(next, ok, mixed_at(base + step, ok));
            cur ^= 1;
        }
        const bool redo = __syncthreads_or(odd);
        l += __shfl_xor(l, 32);
        if constexpr (KG == 2)
            if (!redo) join_teams<ND>(lds_f, team, wave, lane, m, l, o);
        if (!redo && team == 0) {
            if (r0 + 32 * wave + c32 <= last) {
                const int64_t token = s.start + my_i, at = (token * g.a.q_heads + my_h) * g.splits + split;
                const float inv = l > 0.f ? 1.f / l : l;      // no key: zeros; NaN stays
                T *dst = (T *)g.a.out + token * g.a.o_tstride + (int64_t)my_h * g.a.o_hstride;
#pragma unroll
                for (int x = 0; x < ND; ++x)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int d = 32 * x + 8 * y + 4 * h2;
                        if (!FULL && d >= D) continue;
                        const f32x4_t v = {o[x][4 * y], o[x][4 * y + 1], o[x][4 * y + 2], o[x][4 * y + 3]};
                        if (g.splits > 1) *(f32x4_t *)(g.part + at * D + d) = v;
                        else *(uint2 *)(dst + d) = uint2{pack2<T>(v[0] * inv, v[1] * inv), pack2<T>(v[2] * inv, v[3] * inv)};
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
                const float sum = attend_row<T>(g, b, hk, (const T *)g.a.q + token * g.a.q_tstride + (int64_t)h * g.a.q_hstride, see, mine_o,
                                                mine_o + 256);
                const float inv = sum > 0.f ? 1.f / sum : sum;
                T *dst = (T *)g.a.out + token * g.a.o_tstride + (int64_t)h * g.a.o_hstride;
                for (int d = lane; d < D; d += 64) {
                    if (g.splits > 1) g.part[at * D + d] = mine_o[d];
                    else dst[d] = (T)(mine_o[d] * inv);
                }
                if (g.splits > 1 && lane == 0) g.stat[2 * at] = mine_o[256], g.stat[2 * at + 1] = sum;
            }
        }
    }
}

}  // namespace ttsamd
