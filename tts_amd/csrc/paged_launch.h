// The launches of paged_attention.hip, one translation unit an element type (paged_f32.hip, paged_f16.hip, paged_bf16.hip).
#pragma once
#include "paged_stream.h"

namespace ttsamd {

constexpr int kTileKeys = 64, kTile3Keys = 32;      // keys of a staged tile: 16-bit types, fp32
// Channels of a staged row in LDS, for 64, 96, 128, 192 or 256 computed ones: a power of two, so that its pieces fall evenly on lanes; fp32
// rows of 192 stay as they are (two buffers of six planes would not fit otherwise).
constexpr int padded_pow2(int dc) { return dc <= 64 ? 64 : dc <= 128 ? 128 : 256; }
constexpr int tile3_pitch(int dc) { return dc == 192 ? 192 : padded_pow2(dc); }

struct PagedLaunch {
    bool tile, few;                  // paged_tile.h / paged_tile3.h; one or two fp32 rows (attend_few); else attend_stream
    int dp, nq, waves, teams;        // head_dim padded to what is computed; row tiles a wave (streamed); waves of a workgroup, or of one of its teams (staged)
    int splits, split_keys, row_tiles;
    size_t part_bytes, stat_bytes;
};

// Waves of a streaming workgroup, by what a wave's registers allow (256 or 512 of them).
constexpr int most_waves(int dp) { return dp <= 192 ? 8 : 4; }

hipError_t start_f32(const AttArgs &g, const PagedLaunch &p, hipStream_t st);
hipError_t start_f16(const AttArgs &g, const PagedLaunch &p, hipStream_t st);
hipError_t start_bf16(const AttArgs &g, const PagedLaunch &p, hipStream_t st);
void join_f32(const AttArgs &g, hipStream_t st);
void join_f16(const AttArgs &g, hipStream_t st);
void join_bf16(const AttArgs &g, hipStream_t st);

}  // namespace ttsamd
