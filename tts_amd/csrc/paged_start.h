// What paged_launch.h declares, for one element type T.
#pragma once
#include "paged_tile3.h"

namespace ttsamd {

template <class T, int DP, int NQ, bool FULL> hipError_t start_stream(const AttArgs &g, const PagedLaunch &p, dim3 grid, hipStream_t st)
{
    constexpr int MAXW = most_waves(DP);
    static std::atomic<unsigned long long> done{0};
    const int bytes = p.waves * 16 * NQ * (DP + 4 + 2) * 4, most = MAXW * 16 * NQ * (DP + 4 + 2) * 4;
    if (hipError_t e = ensure_dynamic_lds((const void *)attend_stream<T, DP, NQ, FULL, MAXW>, most, done)) return e;
    attend_stream<T, DP, NQ, FULL, MAXW><<<grid, p.waves * 64, bytes, st>>>(g);
    return hipSuccess;
}
template <class T, int DP, int NQ> hipError_t start_stream(const AttArgs &g, const PagedLaunch &p, dim3 grid, hipStream_t st)
{
    return g.c.head_dim == DP ? start_stream<T, DP, NQ, true>(g, p, grid, st) : start_stream<T, DP, NQ, false>(g, p, grid, st);
}

template <class T, int DC, bool FULL, int RW, int KG> hipError_t start_tile(const AttArgs &g, dim3 grid, hipStream_t st)
{
    static std::atomic<unsigned long long> done{0};
    constexpr int join = KG == 2 ? RW * (DC / 2 + 2) * 64 * 4 : 0;
    if constexpr (sizeof(T) == 4) {
        constexpr int tiles = KG * 2 * 6 * kTile3Keys * tile3_pitch(DC) * 2, bytes = tiles > join ? tiles : join;
        if (hipError_t e = ensure_dynamic_lds((const void *)attend_tile3<DC, FULL, RW, KG>, bytes, done)) return e;
        attend_tile3<DC, FULL, RW, KG><<<grid, 64 * RW * KG, bytes, st>>>(g);
    } else {
        constexpr int tiles = KG * 2 * 2 * kTileKeys * padded_pow2(DC) * 2, bytes = tiles > join ? tiles : join;
        if (hipError_t e = ensure_dynamic_lds((const void *)attend_tile<T, DC, FULL, RW, KG>, bytes, done)) return e;
        attend_tile<T, DC, FULL, RW, KG><<<grid, 64 * RW * KG, bytes, st>>>(g);
    }
    return hipSuccess;
}
template <class T, int DC, int RW, int KG> hipError_t start_tile(const AttArgs &g, dim3 grid, hipStream_t st)
{
    return g.c.head_dim == DC ? start_tile<T, DC, true, RW, KG>(g, grid, st) : start_tile<T, DC, false, RW, KG>(g, grid, st);
}
template <class T, int DC> hipError_t start_tile(const AttArgs &g, const PagedLaunch &p, dim3 grid, hipStream_t st)
{
    if constexpr (DC == 64 || (DC <= 128 && sizeof(T) == 2)) {
        if (p.waves == 2) return start_tile<T, DC, 2, 2>(g, grid, st);
        if (p.teams == 2) return start_tile<T, DC, 4, 2>(g, grid, st);
    }
    return start_tile<T, DC, 4, 1>(g, grid, st);
}

template <int DP, bool FULL, int R> hipError_t start_few(const AttArgs &g, const PagedLaunch &p, dim3 grid, hipStream_t st)
{
    static std::atomic<unsigned long long> done{0};
    const int bytes = p.waves * R * (DP + 4 + 2) * 4, most = most_waves(DP) * R * (DP + 4 + 2) * 4;
    if (hipError_t e = ensure_dynamic_lds((const void *)attend_few<DP, FULL, R>, most, done)) return e;
    attend_few<DP, FULL, R><<<grid, p.waves * 64, bytes, st>>>(g);
    return hipSuccess;
}
template <int DP> hipError_t start_few(const AttArgs &g, const PagedLaunch &p, dim3 grid, hipStream_t st)
{
    if (g.c.head_dim == DP) return p.nq == 1 ? start_few<DP, true, 1>(g, p, grid, st) : start_few<DP, true, 2>(g, p, grid, st);
    return p.nq == 1 ? start_few<DP, false, 1>(g, p, grid, st) : start_few<DP, false, 2>(g, p, grid, st);
}

template <class T> hipError_t start_paged(const AttArgs &g, const PagedLaunch &p, hipStream_t st)
{
    const dim3 grid(g.c.kv_heads * p.splits, p.row_tiles, g.b.batch);
    if (p.tile) {
        if (p.dp == 64) return start_tile<T, 64>(g, p, grid, st);
        if (p.dp == 96) return start_tile<T, 96>(g, p, grid, st);
        if (p.dp == 128) return start_tile<T, 128>(g, p, grid, st);
        if (p.dp == 192) return start_tile<T, 192>(g, p, grid, st);
        if constexpr (sizeof(T) == 2) return start_tile<T, 256>(g, p, grid, st);
    }
    if constexpr (sizeof(T) == 4)
        if (p.few) return p.dp == 64 ? start_few<64>(g, p, grid, st) : start_few<128>(g, p, grid, st);
    if (p.dp == 64) return p.nq == 2 ? start_stream<T, 64, 2>(g, p, grid, st) : start_stream<T, 64, 1>(g, p, grid, st);
    if (p.dp == 128) return p.nq == 2 ? start_stream<T, 128, 2>(g, p, grid, st) : start_stream<T, 128, 1>(g, p, grid, st);
    if (p.dp == 192) return start_stream<T, 192, 1>(g, p, grid, st);
    return start_stream<T, 256, 1>(g, p, grid, st);
}

template <class T> void join_paged(const AttArgs &g, hipStream_t st)
{
    // a quarter of the splits to a lane, as long as a row's lanes fit a workgroup
    const int cols = g.c.head_dim / 8, n = g.b.max_new < 1 ? 1 : g.b.max_new;
    int lanes = 1;
    while (lanes * 4 < g.splits && lanes * 2 * cols <= 256) lanes *= 2;
    const int teams = 256 / (cols * lanes);
    const int64_t blocks = ((int64_t)n * g.a.q_heads + teams - 1) / teams;
    join_splits<T><<<dim3((unsigned)(blocks < 65536 ? blocks : 65536), g.b.batch), 256, 0, st>>>(g, lanes);
}

}  // namespace ttsamd
