// Rotary positions and the append to a paged key/value cache: rows of [tokens, heads, head_dim] tensors that move once, some of them
// turning on the way.
//
// Mathematics.  A pair (x1, x2) of channel pair i at position p becomes A (x1 cos a - x2 sin a, x2 cos a + x1 sin a) with a = p f_i.
// The angle is kept as a fraction of the circle in 2^-64 units: p * turns_i modulo 2^64 is one 64-bit multiply and exact at any
// position (fp32 angles are off by 0.06 rad at p = 10^6, and a table of angles would be as many bytes as a small batch itself).  Its
// top 32 bits give the nearest quarter turn and a remainder in [-1/8, 1/8] turn, where the Taylor sums of degree 9 / 10 are off by
// less than 2e-9.
// Bound: memory (one read, one write of every byte) once a call moves more than a few MB: 8192 tokens of 32 fp32 heads of 128, 268 MB in
// 65 us where several such sets take turns (4.1 TB/s; a copy of that size reaches 5.0 to 5.3), 51 where one partly stays in the last-level
// cache; 6 ragged bf16 prompts of up to 1500 tokens with 32 + 2 x 8 heads of 128, 205 MB in 54 us (3.8 TB/s) and 38.  Launch latency
// below: 4 us.  A thread owns one chunk of pairs (two 16-byte pieces) and walks several heads with it,
// because the angles are the same in every head of a token and cost about thirty instructions a pair.
#include "decode_common.h"

namespace ttsamd {

int check_paged_kv(const char *what, const ttsamd_paged_kv *c)
{
    TTSAMD_CHECK_ARG(c && c->k && c->v, "%s: the cache is NULL", what);
    TTSAMD_CHECK_ARG(known_dtype(c->dtype), "%s: unknown element type %d", what, c->dtype);
    TTSAMD_CHECK_ARG(c->pages > 0 && c->kv_heads > 0 && c->page_size > 0, "%s: cache of %d pages, %d heads, %d rows a page", what, c->pages,
                     c->kv_heads, c->page_size);
    TTSAMD_CHECK_ARG(c->head_dim > 0, "%s: head_dim %d", what, c->head_dim);
    if (c->head_dim % 8 != 0 || c->head_dim > 256) {
        set_error("%s: head_dim %d (a multiple of 8 up to 256 is supported)", what, c->head_dim);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    const int per = 16 / elem_bytes(c->dtype);
    const int64_t strides[] = {c->k_page, c->k_head, c->k_row, c->v_page, c->v_head, c->v_row};
    for (int64_t s : strides) TTSAMD_CHECK_ARG(s >= 0 && s % per == 0, "%s: cache stride %lld (multiples of 16 bytes)", what, (long long)s);
    TTSAMD_CHECK_ARG((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "%s: the cache has to start at a multiple of 16 bytes", what);
    return TTSAMD_OK;
}

int check_paged_batch(const char *what, const ttsamd_paged_batch *b, int tokens)
{
    TTSAMD_CHECK_ARG(b, "%s: the batch is NULL", what);
    TTSAMD_CHECK_ARG(b->batch >= 0 && b->batch <= 65535, "%s: batch %d (up to 65535)", what, b->batch);
    TTSAMD_CHECK_ARG(b->batch == 0 || (b->seq_lens && b->q_starts), "%s: seq_lens or q_starts is NULL", what);
    TTSAMD_CHECK_ARG(b->table_width >= 0 && (b->table_width == 0 || b->batch == 0 || b->block_table), "%s: the block table is NULL", what);
    TTSAMD_CHECK_ARG(b->table_stride >= 0 && tokens >= 0 && b->max_new >= 0 && b->max_len >= 0, "%s: negative size", what);
    return TTSAMD_OK;
}

int check_written(const char *what, const char *name, const RowSet &out, const char *from, const RowSet &in, bool in_place)
{
    TTSAMD_CHECK_ARG(!rows_meet(out), "%s: rows of %s overlap each other", what, name);
    TTSAMD_CHECK_ARG((in_place && same_rows(out, in)) || !sets_meet(out, in), "%s: %s overlaps %s%s", what, name, from,
                     in_place ? " (it may be the same rows, in the same order)" : "");
    return TTSAMD_OK;
}

namespace {

// One tensor that moves: source rows, destination rows, and whether they turn.
struct Stream {
    const void *src;
    void *dst;
    int64_t s_t, s_h, d_t, d_h;   // d_t: token stride, or the page stride of a paged destination
    int64_t d_row;
    int heads, turns, paged;
    int first_unit;               // units of one token: [first_unit, next stream's first_unit)
};
struct MoveArgs {
    Stream s[3];
    ttsamd_rotary_plan plan;
    ttsamd_paged_batch batch;     // block_table etc.; seq_lens NULL: no sequences, all tokens in one run, places from `positions`
    const void *positions;
    int position_bytes, tokens, head_dim, pages, page_size, inverse;
    int units;                    // work items of one token
    int heads_per_unit;
    int token_tile;
    FastDiv by_units, by_page;
};

template <class T, int V> struct alignas(sizeof(T) * V) Piece {
    T v[V];
};

__device__ __forceinline__ void unit_circle(uint64_t phase, float &c, float &s)
{
    const uint32_t hi = (uint32_t)(phase >> 32);
    const uint32_t quarter = (hi + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(hi - (quarter << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
    const float x2 = x * x;
    const float sn = x * fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), 1.f);
    const float cs = fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, fmaf(x2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const float a = (quarter & 1) ? sn : cs, b = (quarter & 1) ? cs : sn;
    c = (quarter == 1 || quarter == 2) ? -a : a;
    s = (quarter >= 2) ? -b : b;
}

// x c - y s in fp32, then one rounding to T.  Kept apart from the conversion: folded into a mixed-precision fma (which the compiler
// does for some piece widths and not for others) the same row would differ in its last bit with its alignment.
template <class T> __device__ __forceinline__ T turn(float x, float c, float y, float s)
{
    float r = fmaf(x, c, y * s);
    asm("" : "+v"(r));
    return (T)r;
}

// V elements a piece; a head's row = rotary_dim / 2V turning chunks of two pieces, then (head_dim - rotary_dim) / V copied pieces.
template <class T, int V> __global__ __launch_bounds__(256) void move_rows(MoveArgs a)
{
    int start = 0, n = a.tokens, base = 0, keys = 0;
    const bool seqs = a.batch.seq_lens != nullptr;
    if (seqs) {
        const Sequence s = sequence_of(a.batch, a.tokens, a.page_size, blockIdx.y);
        start = s.start, n = s.n, base = s.len - s.n, keys = s.keys;
    }
    const int half = a.plan.rotary_dim / 2;
    using P = Piece<T, V>;
    // unsigned: the step past the last token of 2^31 is no negative one
    for (unsigned t0 = blockIdx.x * a.token_tile; t0 < (unsigned)n; t0 += gridDim.x * a.token_tile) {
        const int items = min(a.token_tile, n - (int)t0) * a.units;
        for (int w = threadIdx.x; w < items; w += 256) {
            const int lt = a.by_units.div(w), unit = w - lt * a.units;
            const int i = (int)t0 + lt, token = start + i;
            const int which = unit >= a.s[2].first_unit ? 2 : unit >= a.s[1].first_unit ? 1 : 0;
            const Stream &st = a.s[which];
            const int turning = st.turns ? half / V : 0;
            const int chunks = turning + (a.head_dim - 2 * V * turning) / V;
            const int u = unit - st.first_unit, hg = u / chunks, chunk = u - hg * chunks;
            const T *src = (const T *)st.src + (int64_t)token * st.s_t;
            T *dst = (T *)st.dst;
            int64_t place = base + i;
            if (st.paged) {
                if (place < 0 || place >= keys) continue;
                int row;
                const int page = page_of(a.batch, a.by_page, a.pages, blockIdx.y, (int)place, row);
                if (page < 0) continue;
                dst += (int64_t)page * st.d_t + (int64_t)row * st.d_row;
            } else {
                dst += (int64_t)token * st.d_t;
            }
            const int hstep = (st.heads + a.heads_per_unit - 1) / a.heads_per_unit;     // neighbouring threads take neighbouring heads
            if (chunk >= turning) {
                const int at = (2 * turning + chunk - turning) * V;
                if (src + at == dst + at && st.s_h == st.d_h) continue;
                for (int h = hg; h < st.heads; h += hstep)
                    *(P *)(dst + h * st.d_h + at) = *(const P *)(src + h * st.s_h + at);
                continue;
            }
            if (a.positions)
                place = a.position_bytes == 8 ? ((const int64_t *)a.positions)[token] : ((const int32_t *)a.positions)[token];
            const uint64_t p = (uint64_t)(a.inverse ? -place : place);
            const int p0 = a.plan.interleaved ? 2 * chunk * V : chunk * V;
            const int p1 = a.plan.interleaved ? p0 + V : p0 + half;
            float c[V], s[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                unit_circle(p * a.plan.turns[chunk * V + e], c[e], s[e]);
                c[e] *= a.plan.amplitude, s[e] *= a.plan.amplitude;
            }
            for (int h = hg; h < st.heads; h += hstep) {
                const P x = *(const P *)(src + h * st.s_h + p0), y = *(const P *)(src + h * st.s_h + p1);
                P ox, oy;
                if (a.plan.interleaved) {
                    T in[2 * V], out[2 * V];
#pragma unroll
                    for (int e = 0; e < V; ++e) in[e] = x.v[e], in[V + e] = y.v[e];
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float f = to_f(in[2 * e]), g = to_f(in[2 * e + 1]);
                        out[2 * e] = turn<T>(f, c[e], -g, s[e]), out[2 * e + 1] = turn<T>(g, c[e], f, s[e]);
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) ox.v[e] = out[e], oy.v[e] = out[V + e];
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float f = to_f(x.v[e]), g = to_f(y.v[e]);
                        ox.v[e] = turn<T>(f, c[e], -g, s[e]), oy.v[e] = turn<T>(g, c[e], f, s[e]);
                    }
                }
                *(P *)(dst + h * st.d_h + p0) = ox;
                *(P *)(dst + h * st.d_h + p1) = oy;
            }
        }
    }
}

// The widest piece that every row, stride and part of the head allows.
int piece_of(const MoveArgs &a, int esize)
{
    const int half = a.plan.rotary_dim / 2;
    for (int v = 16 / esize; v > 1; v /= 2) {
        bool ok = a.head_dim % v == 0 && half % v == 0;
        for (const Stream &s : a.s) {
            if (!s.heads) continue;
            ok = ok && ((uintptr_t)s.src | (uintptr_t)s.dst) % (v * esize) == 0 && s.s_t % v == 0 && s.s_h % v == 0 && s.d_t % v == 0 &&
                 s.d_h % v == 0 && s.d_row % v == 0;
        }
        if (ok) return v;
    }
    return 1;
}

template <class T> void launch(const MoveArgs &a, int v, dim3 grid, hipStream_t st)
{
    switch (v) {
    case 8: if constexpr (sizeof(T) == 2) { move_rows<T, 8><<<grid, 256, 0, st>>>(a); } break;
    case 4: move_rows<T, 4><<<grid, 256, 0, st>>>(a); break;
    case 2: move_rows<T, 2><<<grid, 256, 0, st>>>(a); break;
    default: move_rows<T, 1><<<grid, 256, 0, st>>>(a); break;
    }
}

int move(MoveArgs &a, int dtype, int longest, int sequences, void *stream)
{
    const int v = piece_of(a, elem_bytes(dtype));
    auto chunks = [&](const Stream &s) { return s.turns ? a.plan.rotary_dim / 2 / v + (a.head_dim - a.plan.rotary_dim) / v : a.head_dim / v; };
    // Heads a thread walks with one set of angles: one while the call cannot fill the chip (latency counts), four beyond (1 / 2 / 4 / 8:
    // 24 tokens of 16 bf16 heads of 64 3.5 / 3.9 / 4.7 / 6.0 us; 8192 of 32 fp32 heads of 128 91 / 72 / 59 / 57; the prompts above 63 / 59 /
    // 50 / 53).
    int64_t items = 0;
    for (const Stream &s : a.s) items += (int64_t)s.heads * (s.heads ? chunks(s) : 0);
    items *= a.tokens;
    a.heads_per_unit = items >= 4 * 256 * 1024 ? 4 : 1;
    a.units = 0;
    for (Stream &s : a.s) {
        s.first_unit = a.units;
        if (s.heads) a.units += (s.heads + a.heads_per_unit - 1) / a.heads_per_unit * chunks(s);
    }
    a.token_tile = a.units >= 256 ? 1 : 256 / a.units;
    a.by_units = fast_div(a.units);
    const int64_t tiles = ((int64_t)longest + a.token_tile - 1) / a.token_tile;
    const dim3 grid((unsigned)(tiles < 1 ? 1 : tiles > 1048576 ? 1048576 : tiles), sequences);
    hipStream_t st = as_stream(stream);
    if (dtype == TTSAMD_F32) launch<float>(a, v, grid, st);
    else if (dtype == TTSAMD_F16) launch<_Float16>(a, v, grid, st);
    else launch<__bf16>(a, v, grid, st);
    TTSAMD_LAUNCH_CHECK();
    return TTSAMD_OK;
}

int check_plan(const char *what, const ttsamd_rotary_plan *p, int head_dim)
{
    TTSAMD_CHECK_ARG(p->rotary_dim >= 0 && p->rotary_dim % 2 == 0 && p->rotary_dim <= head_dim,
                     "%s: rotary_dim %d of a head of %d (an even number up to it)", what, p->rotary_dim, head_dim);
    TTSAMD_CHECK_ARG(p->rotary_dim == 0 || p->turns, "%s: the plan has no turns", what);
    return TTSAMD_OK;
}

}  // namespace
}  // namespace ttsamd

extern "C" int ttsamd_rotary(const ttsamd_rotary_args *r, const ttsamd_rotary_plan *plan, void *stream)
{
    using namespace ttsamd;
    TTSAMD_CHECK_ARG(r && plan, "rotary: arguments are NULL");
    TTSAMD_CHECK_ARG(known_dtype(r->dtype), "rotary: unknown element type %d", r->dtype);
    TTSAMD_CHECK_ARG(r->tokens >= 0 && r->heads >= 0 && r->head_dim >= 0, "rotary: negative size");
    if (int rc = check_plan("rotary", plan, r->head_dim)) return rc;
    if (r->tokens == 0 || r->heads == 0 || r->head_dim == 0) return TTSAMD_OK;
    TTSAMD_CHECK_ARG(r->x && r->y && r->positions, "rotary: a tensor is NULL");
    TTSAMD_CHECK_ARG(r->position_bytes == 4 || r->position_bytes == 8, "rotary: positions of %d bytes", r->position_bytes);
    if ((int64_t)r->heads * r->head_dim > (1 << 20)) {
        set_error("rotary: %d heads of %d channels (up to 2^20 channels a token)", r->heads, r->head_dim);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    const RowSet x = rows_of(r->x, r->x_tstride, r->x_hstride, r->tokens, r->heads, r->head_dim, r->dtype);
    const RowSet y = rows_of(r->y, r->y_tstride, r->y_hstride, r->tokens, r->heads, r->head_dim, r->dtype);
    if (int rc = check_written("rotary", "y", y, "x", x, true)) return rc;
    MoveArgs a = {};
    a.s[0] = {r->x, r->y, r->x_tstride, r->x_hstride, r->y_tstride, r->y_hstride, 0, r->heads, 1, 0, 0};
    a.plan = *plan;
    a.positions = r->positions, a.position_bytes = r->position_bytes;
    a.tokens = r->tokens, a.head_dim = r->head_dim, a.inverse = r->inverse;
    a.page_size = 1, a.by_page = fast_div(1);
    return move(a, r->dtype, r->tokens, 1, stream);
}

extern "C" int ttsamd_kv_append(const ttsamd_kv_append_args *r, const ttsamd_paged_kv *cache, const ttsamd_paged_batch *batch,
                                const ttsamd_rotary_plan *plan, void *stream)
{
    using namespace ttsamd;
    TTSAMD_CHECK_ARG(r, "kv_append: arguments are NULL");
    if (int rc = check_paged_kv("kv_append", cache)) return rc;
    if (int rc = check_paged_batch("kv_append", batch, r->tokens)) return rc;
    if (plan) if (int rc = check_plan("kv_append", plan, cache->head_dim)) return rc;
    if (r->tokens == 0 || batch->batch == 0) return TTSAMD_OK;
    TTSAMD_CHECK_ARG(r->k && r->v && (!r->q || r->q_out), "kv_append: a tensor is NULL");
    TTSAMD_CHECK_ARG(!r->positions || r->position_bytes == 4 || r->position_bytes == 8, "kv_append: positions of %d bytes", r->position_bytes);
    TTSAMD_CHECK_ARG(!r->q || r->q_heads > 0, "kv_append: %d query heads", r->q_heads);
    if ((int64_t)(2 * cache->kv_heads + (r->q ? r->q_heads : 0)) * cache->head_dim > (1 << 20)) {
        set_error("kv_append: more than 2^20 channels a token");
        return TTSAMD_ERR_UNSUPPORTED;
    }
    if (r->q) {
        auto rows = [&](const void *at, int64_t t, int64_t h, int heads) { return rows_of(at, t, h, r->tokens, heads, cache->head_dim, cache->dtype); };
        const RowSet out = rows(r->q_out, r->qo_tstride, r->qo_hstride, r->q_heads);
        if (int rc = check_written("kv_append", "q_out", out, "q", rows(r->q, r->q_tstride, r->q_hstride, r->q_heads), true)) return rc;
        if (int rc = check_written("kv_append", "q_out", out, "k", rows(r->k, r->k_tstride, r->k_hstride, cache->kv_heads), false)) return rc;
        if (int rc = check_written("kv_append", "q_out", out, "v", rows(r->v, r->v_tstride, r->v_hstride, cache->kv_heads), false)) return rc;
    }
    MoveArgs a = {};
    const int turns = plan && plan->rotary_dim > 0;
    a.s[0] = {r->k, cache->k, r->k_tstride, r->k_hstride, cache->k_page, cache->k_head, cache->k_row, cache->kv_heads, turns, 1, 0};
    a.s[1] = {r->v, cache->v, r->v_tstride, r->v_hstride, cache->v_page, cache->v_head, cache->v_row, cache->kv_heads, 0, 1, 0};
    if (r->q) a.s[2] = {r->q, r->q_out, r->q_tstride, r->q_hstride, r->qo_tstride, r->qo_hstride, 0, r->q_heads, turns, 0, 0};
    if (plan) a.plan = *plan;
    a.batch = *batch;
    a.positions = r->positions, a.position_bytes = r->position_bytes;
    a.tokens = r->tokens, a.head_dim = cache->head_dim, a.pages = cache->pages, a.page_size = cache->page_size;
    a.by_page = fast_div(cache->page_size);
    return move(a, cache->dtype, batch->max_new < 1 ? 1 : batch->max_new, batch->batch, stream);
}
