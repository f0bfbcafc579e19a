// Attention of new tokens over a paged key/value cache: the choice of kernel and launch, and the entry points.
//
// out[t,h] = sum_j p_j v_j, p = softmax_j(scale q.k_j) over the keys token t sees, in one pass over the keys with a running maximum m
// and sum l: a tile's scores s give m' = max(m, s), p = exp(s - m'), l = l exp(m - m') + sum p, o = o exp(m - m') + sum p v.
#include "paged_launch.h"

namespace ttsamd {
namespace {

constexpr int kCus = 256;

// How a call is laid over the chip.  Sizes here are hints (max_new, max_len): the kernels compute whatever the device data holds.
PagedLaunch plan_of(const ttsamd_paged_attention_args &a, const ttsamd_paged_kv &c, const ttsamd_paged_batch &b)
{
    PagedLaunch p = {};
    const bool f32 = c.dtype == TTSAMD_F32;
    const int group = a.q_heads / c.kv_heads;
    // Heads between the widths of a power of two have kernels of their own (computed as 256 and 128: 48 single bf16 tokens over 2000 keys of
    // 8 heads of 192 158 -> 112 us; chunks of 2 x 1024 tokens over 2048 keys, 32 heads over 8: bf16 of 192 299 -> 171, of 96 87 -> 82,
    // fp32 of 192 1489 -> 469, of 96 333 -> 283; streamed, 96 are computed as 128: they wait for memory either way).
    p.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : c.head_dim <= 192 ? 192 : 256;
    const int64_t rows = (int64_t)(b.max_new < 1 ? 1 : b.max_new) * group;
    const int64_t room = (int64_t)b.table_width * c.page_size;
    int64_t keys = b.max_len > 0 && b.max_len < room ? b.max_len : room;
    if (a.window > 0 && (int64_t)a.window + b.max_new < keys) keys = (int64_t)a.window + b.max_new;
    // Staged from some rows on (one sequence over 4096 keys; 8 key heads of 128, bf16: 128 / 256 / 1024 rows streamed 28.5 / 30.6 / 57 us,
    // staged 24.6 / 27.2 / 40; 16 of 64, fp32, 2048 keys: 64 / 128 / 256 rows streamed 20.1 / 25.0 / 35, staged 21.5 / 22.9 / 28.6).
    p.tile = f32 ? p.dp <= 192 && rows >= (p.dp == 64 ? 96 : 64) : rows >= 96;
    // One or two fp32 rows go without the matrix unit (one token over 605 keys of 16 heads of 64: 11.4 -> 7.6 us, 48 of up to 1007 keys: 59 ->
    // 56 us; heads over 128 channels would need more registers than they have).
    p.few = f32 && rows <= 2 && p.dp <= 128;
    p.nq = p.few ? (int)rows : rows > 16 && p.dp <= 128 ? 2 : 1;
    const bool pairs = p.tile && (p.dp == 64 || (p.dp == 128 && !f32));               // registers and LDS for two teams
    const int kt = p.tile ? f32 ? kTile3Keys : kTileKeys : f32 || p.dp > 192 ? 16 : 32;
    const int64_t key_tiles = keys < 1 ? 1 : (keys + kt - 1) / kt;
    p.waves = 4;
    if (pairs) {
        // 64 rows a workgroup instead of 128 while such ones are few, or few enough for the chip where two of them share a compute unit
        // or the keys are short: 2 x 437 fp32 tokens, 16 heads of 64: 22.2 against 24.6 us; 256 bf16 tokens over 4096 keys, 32 heads over
        // 8 of 128 (128 of them, one a compute unit): 54 against 39 us.
        const int64_t small = (rows + 63) / 64 * c.kv_heads * b.batch;
        if (small <= 32 || (small <= kCus && (f32 ? key_tiles <= 16 : p.dp == 64))) p.waves = 2;
    }
    const int block_rows = p.tile ? 32 * p.waves : p.few ? p.nq : 16 * p.nq;
    const int64_t tiles = (rows + block_rows - 1) / block_rows, blocks = tiles * c.kv_heads * b.batch;
    p.row_tiles = (int)(tiles < 65535 ? tiles : 65535);
    // Fewer streaming workgroups than compute units: more waves to each, since they are joined in LDS for nothing but a barrier.  (One bf16
    // token of 16 heads over 605 keys: 2 / 4 / 8 waves 12.0 / 9.1 / 8.2 us; 448 workgroups of fp32 rows: 33.4 / 23.2 / 29.5 us.)
    while (!p.tile && p.waves < most_waves(p.dp) && blocks < kCus && key_tiles > p.waves) p.waves *= 2;
    // Staged ones put a second team of waves on the keys where a workgroup has a compute unit to itself (1000 bf16 tokens over 2000 keys, 32
    // heads over 8 of 128: 61 -> 49 us).
    p.teams = pairs && (p.waves == 2 || (blocks <= kCus && key_tiles >= 4)) ? 2 : 1;
    // Still few, and long: the keys are split over workgroups until one round of them fills the chip, and a second launch joins them.
    // (Three tokens over 65537 keys, 12 workgroups of 8 waves, one a compute unit: 21 / 32 / 42 / 85 splits 70.6 / 84.0 / 75.5 / 87.2 us;
    // one bf16 token over 605 keys, 2.4 tiles a wave: whole 8.2 us, two splits 11.0; 32 heads over 8 of 128, 600 keys 11.0 and 11.6, 1000
    // 15.0 and 12.0; one over 4096, 16 tiles a wave: at least 1 / 2 / 4 tiles left to a wave 14.1 / 16.0 / 21.0 us; one fp32 token over 605,
    // 4.8 tiles a wave: whole 8.0 us, two splits 9.1, over 2048: 17.6 and, eight splits, 12.2.)
    p.splits = 1;
    const int waves_held = p.tile ? p.dp > 128 || (f32 && p.dp > 64) || (p.waves == 2 && (f32 || p.dp > 64)) ? 4 : 8 : p.few ? 16 : p.dp == 64 ? 12 : p.dp <= 192 ? 8 : 4;
    const int resident = waves_held / (p.waves * p.teams);                                  // workgroups a compute unit holds, by registers and LDS
    const int64_t fill = (int64_t)kCus * (resident < 1 ? 1 : resident) / blocks, a_wave = p.tile ? p.teams : p.waves;
    // Tiles left to a wave, or a team, of a split: the join costs by the row and the split.  Staged, at least 1 / 2 / 4: 24 workgroups of fp16
    // rows (2 x 84 tokens, 8 heads over 4 of 128) over 600 keys 16.2 / 19.3 / 19.8 us, over 1815 19.6 / 21.2 / 24.7; 12 over 4096 (21 and 16
    // splits) 21.3 / 18.7 / 22.1; 1600 rows of one head of 64 over 1815 16.4 / 14.8 / 16.3; 128 workgroups of 64 over 600 keys 14.9 / 14.0 /
    // 13.0, over 1815 19.6 / 19.6 / 21.2.
    const int least = p.tile ? blocks <= 32 && rows <= 512 ? 1 : blocks >= 64 && key_tiles <= 8 * a_wave ? 4 : 2 : rows > 64 ? 4 : p.few || rows > 32 ? 2 : 1;
    int64_t most = key_tiles / (a_wave * least);
    if (p.tile && least == 1 && most > 16) most = key_tiles / (2 * a_wave) > 16 ? key_tiles / (2 * a_wave) : 16;
    if (fill > 1 && key_tiles > (p.few ? 8 : p.tile || p.dp == 64 ? 4 : 3) * a_wave && most > 1) p.splits = (int)(fill < most ? fill : most);
    // Parts are laid out by the token, whoever owns it: a call whose tokens are mostly padding gets fewer splits, not gigabytes.
    const size_t rows_bytes = (size_t)a.tokens * a.q_heads * (c.head_dim + 2) * sizeof(float), room_bytes = (size_t)256 << 20;
    if (p.splits * rows_bytes > room_bytes) p.splits = rows_bytes * 2 > room_bytes ? 1 : (int)(room_bytes / rows_bytes);
    if ((int64_t)p.splits * c.kv_heads > 65535) p.splits = 65535 / c.kv_heads > 1 ? 65535 / c.kv_heads : 1;
    const int64_t each = (key_tiles + p.splits - 1) / p.splits;
    p.split_keys = (int)(each * kt < 0x7fffffff ? each * kt : 0x7fffffff);
    if (p.tile && p.dp == 128 && c.head_dim <= 96) p.dp = 96;
    if (p.splits > 1) {
        const size_t n = (size_t)a.tokens * a.q_heads * p.splits;
        p.part_bytes = n * c.head_dim * sizeof(float), p.stat_bytes = n * 2 * sizeof(float);
    }
    return p;
}

int check(const ttsamd_paged_attention_args *a, const ttsamd_paged_kv *cache, const ttsamd_paged_batch *batch)
{
    TTSAMD_CHECK_ARG(a, "paged_attention: arguments are NULL");
    if (int rc = check_paged_kv("paged_attention", cache)) return rc;
    if (int rc = check_paged_batch("paged_attention", batch, a->tokens)) return rc;
    TTSAMD_CHECK_ARG(a->q_heads > 0 && a->q_heads % cache->kv_heads == 0, "paged_attention: %d query heads over %d key heads", a->q_heads,
                     cache->kv_heads);
    TTSAMD_CHECK_ARG(a->window >= 0, "paged_attention: window %d", a->window);
    if (a->q_heads > 65535 || (int64_t)a->tokens * a->q_heads > (1 << 30) || (int64_t)batch->table_width * cache->page_size > 0x7fff0000) {
        set_error("paged_attention: %d query heads of %d tokens, tables of %d pages (up to 65535 heads, 2^30 rows, 2^31 - 2^16 positions)",
                  a->q_heads, a->tokens, batch->table_width);
        return TTSAMD_ERR_UNSUPPORTED;
    }
    // row offsets travel in 16-byte units of 32 bits
    const int es = elem_bytes(cache->dtype);
    if ((((int64_t)cache->pages - 1) * cache->k_page + (cache->page_size - 1) * cache->k_row) * es / 16 > 0xffffffffll ||
        (((int64_t)cache->pages - 1) * cache->v_page + (cache->page_size - 1) * cache->v_row) * es / 16 > 0xffffffffll) {
        set_error("paged_attention: a cache that spans over 64 GiB");
        return TTSAMD_ERR_UNSUPPORTED;
    }
    return TTSAMD_OK;
}

}  // namespace
}  // namespace ttsamd

extern "C" size_t ttsamd_paged_attention_workspace_bytes(const ttsamd_paged_attention_args *a, const ttsamd_paged_kv *cache,
                                                         const ttsamd_paged_batch *batch)
{
    using namespace ttsamd;
    if (check(a, cache, batch) != TTSAMD_OK || a->tokens == 0 || batch->batch == 0) return 0;
    const PagedLaunch p = plan_of(*a, *cache, *batch);
    return p.part_bytes + p.stat_bytes;
}

extern "C" int ttsamd_paged_attention(const ttsamd_paged_attention_args *a, const ttsamd_paged_kv *cache, const ttsamd_paged_batch *batch,
                                      void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace ttsamd;
    if (int rc = check(a, cache, batch)) return rc;
    if (a->tokens == 0 || batch->batch == 0) return TTSAMD_OK;
    TTSAMD_CHECK_ARG(a->q && a->out, "paged_attention: a tensor is NULL");
    const int per = 16 / elem_bytes(cache->dtype);
    TTSAMD_CHECK_ARG((((uintptr_t)a->q | (uintptr_t)a->out) & 15) == 0 && a->q_tstride % per == 0 && a->q_hstride % per == 0 &&
                         a->o_tstride % per == 0 && a->o_hstride % per == 0,
                     "paged_attention: q and out start and stride at multiples of 16 bytes");
    const RowSet q = rows_of(a->q, a->q_tstride, a->q_hstride, a->tokens, a->q_heads, cache->head_dim, cache->dtype);
    const RowSet out = rows_of(a->out, a->o_tstride, a->o_hstride, a->tokens, a->q_heads, cache->head_dim, cache->dtype);
    if (int rc = check_written("paged_attention", "out", out, "q", q, true)) return rc;
    const PagedLaunch p = plan_of(*a, *cache, *batch);
    TTSAMD_CHECK_ARG(p.splits == 1 || (workspace && ((uintptr_t)workspace & 15) == 0 && workspace_bytes >= p.part_bytes + p.stat_bytes),
                     "paged_attention: a workspace of %zu bytes at a multiple of 16 is wanted", p.part_bytes + p.stat_bytes);
    AttArgs g = {};
    g.a = *a, g.c = *cache, g.b = *batch;
    g.group = a->q_heads / cache->kv_heads;
    g.by_page = fast_div(cache->page_size), g.by_group = fast_div(g.group);
    g.scale2 = a->scale * 1.4426950408889634f;
    g.splits = p.splits, g.split_keys = p.split_keys;
    g.part = (float *)workspace, g.stat = (float *)((char *)workspace + p.part_bytes);
    hipStream_t st = as_stream(stream);
    TTSAMD_HIP(cache->dtype == TTSAMD_F32 ? start_f32(g, p, st) : cache->dtype == TTSAMD_F16 ? start_f16(g, p, st) : start_bf16(g, p, st));
    TTSAMD_LAUNCH_CHECK();
    if (p.splits > 1) {
        cache->dtype == TTSAMD_F32 ? join_f32(g, st) : cache->dtype == TTSAMD_F16 ? join_f16(g, st) : join_bf16(g, st);
        TTSAMD_LAUNCH_CHECK();
    }
    return TTSAMD_OK;
}
