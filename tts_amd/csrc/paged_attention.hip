// Attention of new tokens over a paged key/value cache: the choice of kernel and launch, and the entry points.
//
// out[t,h] = sum_j p_j v_j, p = softmax_j(scale q.k_j) over the keys token t sees, in one pass over the keys with a running maximum m
// and sum l: a tile's scores s give m' = max(m, s), p = exp(s - m'), l = l exp(m - m') + sum p, o = o exp(m - m') + sum p v.
#include "paged_tile.h"

namespace ttsamd {
namespace {

constexpr int kCus = 256;

struct Launch {
    bool tile;                       // paged_tile.h; else paged_stream.h
    int dp, nq, waves, splits, split_keys, row_tiles;
    size_t part_bytes, stat_bytes;
};

// Waves of a workgroup, by what a wave's registers allow (256 or 512 of them).
constexpr int most_waves(int dp) { return dp <= 128 ? 8 : 4; }

// How a call is laid over the chip.  Sizes here are hints (max_new, max_len): the kernels compute whatever the device data holds.
Launch plan_of(const ttsamd_paged_attention_args &a, const ttsamd_paged_kv &c, const ttsamd_paged_batch &b)
{
    Launch p = {};
    const bool f32 = c.dtype == TTSAMD_F32;
    const int group = a.q_heads / c.kv_heads;
    p.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
    const int64_t rows = (int64_t)(b.max_new < 1 ? 1 : b.max_new) * group;
    // Rows enough for the staged kernel, by type and row: 4096 keys, one sequence, 128 / 256 / 512 / 1024 rows of 8 key heads of 128: streamed
    // 26 / 30 / 39 / 57 us, staged 30 / 33 / 41 / 50; of 16 of 64: 21 / 35 / 48 us (128 / 256 / 512 rows), staged 21 / 25 / 29.
    p.tile = !f32 && rows >= 256;
    p.nq = rows > 16 && p.dp < 256 ? 2 : 1;
    const int block_rows = p.tile ? kTileRows : 16 * p.nq, kt = p.tile ? kTileKeys : f32 || p.dp > 128 ? 16 : 32;
    const int64_t tiles = (rows + block_rows - 1) / block_rows;
    p.row_tiles = (int)(tiles < 65535 ? tiles : 65535);
    const int64_t room = (int64_t)b.table_width * c.page_size;
    int64_t keys = b.max_len > 0 && b.max_len < room ? b.max_len : room;
    if (a.window > 0 && (int64_t)a.window + b.max_new < keys) keys = (int64_t)a.window + b.max_new;
    const int64_t key_tiles = keys < 1 ? 1 : (keys + kt - 1) / kt, blocks = tiles * c.kv_heads * b.batch;
    // Fewer workgroups than compute units: more waves to each, since they are joined in LDS for nothing but a barrier.  (One bf16 token of
    // 16 heads over 605 keys: 2 / 4 / 8 waves 12.0 / 9.1 / 8.2 us; 2 x 437 fp32 tokens, 448 workgroups: 33.4 / 23.2 / 29.5 us.)
    p.waves = 4;
    while (!p.tile && p.waves < most_waves(p.dp) && blocks < kCus && key_tiles > p.waves) p.waves *= 2;
    // Still few, and long: the keys are split over workgroups until one round of them fills the chip, and a second launch joins them.
    // (Three tokens over 65537 keys, 12 workgroups of 8 waves, one a compute unit: 21 / 32 / 42 / 85 splits 70.6 / 84.0 / 75.5 / 87.2 us;
    // one bf16 token over 605 keys, 2.4 tiles a wave: whole 8.2 us, two splits 11.0; one over 4096, 16 tiles a wave: at least 1 / 2 / 4
    // tiles left to a wave 14.1 / 16.0 / 21.0 us.)
    p.splits = 1;
    const int resident = (p.dp > 128 ? 4 : p.dp == 64 && !p.tile ? 12 : 8) / p.waves;    // workgroups a compute unit's registers hold
    const int64_t fill = (int64_t)kCus * (resident < 1 ? 1 : resident) / blocks, a_wave = p.tile ? 1 : p.waves;
    const int64_t most = key_tiles / (a_wave * (p.tile || rows > 64 ? 4 : rows > 32 ? 2 : 1));       // tiles left to a wave: the join costs by the row
    if (fill > 1 && key_tiles > 4 * a_wave) p.splits = (int)(fill < most ? fill : most);
    if ((int64_t)p.splits * c.kv_heads > 65535) p.splits = 65535 / c.kv_heads > 1 ? 65535 / c.kv_heads : 1;
    const int64_t each = (key_tiles + p.splits - 1) / p.splits;
    p.split_keys = (int)(each * kt < 0x7fffffff ? each * kt : 0x7fffffff);
    if (p.splits > 1) {
        const size_t n = (size_t)a.tokens * a.q_heads * p.splits;
        p.part_bytes = n * c.head_dim * sizeof(float), p.stat_bytes = n * 2 * sizeof(float);
    }
    return p;
}

template <class T, int DP, int NQ, bool FULL> hipError_t start(const AttArgs &g, const Launch &p, dim3 grid, hipStream_t st)
{
    constexpr int MAXW = most_waves(DP);
    static std::atomic<unsigned long long> done{0};
    const int bytes = p.waves * 16 * NQ * (DP + 4 + 2) * 4, most = MAXW * 16 * NQ * (DP + 4 + 2) * 4;
    if (hipError_t e = ensure_dynamic_lds((const void *)attend_stream<T, DP, NQ, FULL, MAXW>, most, done)) return e;
    attend_stream<T, DP, NQ, FULL, MAXW><<<grid, p.waves * 64, bytes, st>>>(g);
    return hipSuccess;
}
template <class T, int DP, int NQ> hipError_t start(const AttArgs &g, const Launch &p, dim3 grid, hipStream_t st)
{
    return g.c.head_dim == DP ? start<T, DP, NQ, true>(g, p, grid, st) : start<T, DP, NQ, false>(g, p, grid, st);
}
template <class T, int DP, bool FULL> hipError_t start_tile(const AttArgs &g, dim3 grid, hipStream_t st)
{
    static std::atomic<unsigned long long> done{0};
    constexpr int bytes = 2 * 2 * kTileKeys * DP * 2;
    if (hipError_t e = ensure_dynamic_lds((const void *)attend_tile<T, DP, FULL>, bytes, done)) return e;
    attend_tile<T, DP, FULL><<<grid, 256, bytes, st>>>(g);
    return hipSuccess;
}
template <class T, int DP> hipError_t start_tile(const AttArgs &g, dim3 grid, hipStream_t st)
{
    return g.c.head_dim == DP ? start_tile<T, DP, true>(g, grid, st) : start_tile<T, DP, false>(g, grid, st);
}
template <class T> hipError_t start(const AttArgs &g, const Launch &p, hipStream_t st)
{
    if constexpr (sizeof(T) == 2) {
        const dim3 grid(g.c.kv_heads * p.splits, p.row_tiles, g.b.batch);
        if (p.tile) return p.dp == 64 ? start_tile<T, 64>(g, grid, st) : p.dp == 128 ? start_tile<T, 128>(g, grid, st) : start_tile<T, 256>(g, grid, st);
    }
    const dim3 grid(g.c.kv_heads * p.splits, p.row_tiles, g.b.batch);
    if (p.dp == 64) return p.nq == 2 ? start<T, 64, 2>(g, p, grid, st) : start<T, 64, 1>(g, p, grid, st);
    if (p.dp == 128) return p.nq == 2 ? start<T, 128, 2>(g, p, grid, st) : start<T, 128, 1>(g, p, grid, st);
    return start<T, 256, 1>(g, p, grid, st);
}
template <class T> void join(const AttArgs &g, hipStream_t st)
{
    // a quarter of the splits to a lane, as long as a row's lanes fit a workgroup
    const int cols = g.c.head_dim / 8, n = g.b.max_new < 1 ? 1 : g.b.max_new;
    int lanes = 1;
    while (lanes * 4 < g.splits && lanes * 2 * cols <= 256) lanes *= 2;
    const int teams = 256 / (cols * lanes);
    const int64_t blocks = ((int64_t)n * g.a.q_heads + teams - 1) / teams;
    join_splits<T><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536), g.b.batch), 256, 0, st>>>(g, lanes);
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
    const Launch p = plan_of(*a, *cache, *batch);
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
    const Launch p = plan_of(*a, *cache, *batch);
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
    TTSAMD_HIP(cache->dtype == TTSAMD_F32 ? start<float>(g, p, st) : cache->dtype == TTSAMD_F16 ? start<_Float16>(g, p, st) : start<__bf16>(g, p, st));
    TTSAMD_LAUNCH_CHECK();
    if (p.splits > 1) {
        if (cache->dtype == TTSAMD_F32) join<float>(g, st);
        else if (cache->dtype == TTSAMD_F16) join<_Float16>(g, st);
        else join<__bf16>(g, st);
        TTSAMD_LAUNCH_CHECK();
    }
    return TTSAMD_OK;
}
