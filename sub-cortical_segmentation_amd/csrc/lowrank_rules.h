// Which form of the shared projection's kernels a call takes (scs_lowrank.hip): rules on sizes, types and alignment alone, host code without the device's.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/scs.h"

namespace scs {
namespace {

constexpr int kFewWaves = 8;              // waves of a workgroup of the few-rows form (lowrank_few.h)

// directions of an adapter in tiles of 16, as the kernels are compiled: 1, 2, 4, 8
inline int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }

// ---- shrink
// Up to so many rows a workgroup takes four directions of one row (and reads P once for every row), above a tile of rows.  The whole forward call in us, the one
// way / the other: 540 x 540, f32, rank 8, 128 rows 11.9 / 12.4, 512 rows 17.3 / 17.2, 1024 rows 24.7 / 23.2; 4096 x 512, bf16, rank 16, 26.8 / 31.3, 32.5 / 32.1,
// 40.9 / 32.1; the same of rank 64 35.8 / 46.5, 58.8 / 45.6, 87.5 / 45.6 (the two meet at 256 rows there, at 384 for rank 32: the rule does not look at the rank)
constexpr int kDotRows = 512;

// Above: waves that share a row tile's contraction, about two units of 256 bytes of a row (128 where many directions fill the registers) each; two row tiles
// a wave (P read half as often) where workgroups abound.
struct ShrinkForm { int mt, waves; };
inline ShrinkForm shrink_form(const scs_lowrank& p, int64_t K) {
    const int jt = rank_tiles(p.rank), unit = (jt <= 2 ? 4 : 2) * 64 / (p.dtype == SCS_F32 ? 4 : 2);
    const int64_t units = (K + unit - 1) / unit;
    if (p.rows >= 16384) return {jt <= 2 ? 2 : 1, units >= 16 ? 8 : 4};
    return {1, units >= 32 ? (jt <= 2 ? 16 : 8) : units >= 16 ? 8 : 4};
}

// ---- gradients of the adapters
// Rows of a block of the by-blocks form, 0: the direct form.  Blocks so that there are about 2048 workgroups, of 64 to 512 rows (more where a
// grid's 65535 would not do); direct up to 512 rows (the second launch would cost more than it saves), and where the slots (requests + blocks, rank
// f32 values a column each) would weigh too much: more than four times X's own bytes, or more than X because requests make up four fifths of them (each
// is written and read once, and a request of a few rows costs a block's waves as much as sixteen).  By blocks / direct, us, dA and dB:
//   8192 x 4096 + 4096, bf16, rank 16, adapters 1 and 8: 10 requests 75 / 113 and 70 / 65, 100 requests 136 / 135 and 95 / 72, 400 requests 389 / 189 and
//   204 / 92; 900 requests 403 / 124 (8 adapters), where the slots took 490 MB of workspace
//   60 000 x 540 + 540, f32, rank 8, adapters 1 and 8: 10 requests 126 / 665 and 102 / 167, 400 requests 345 / 739 and 136 / 136
//   4096 x 2048 + 2048, bf16, rank 64, adapters 1 and 8: 10 requests 108 / 194 and 103 / 74, 400 requests 618 / 317 and 434 / 87
// (with several adapters the direct form is the faster one in some of what is left to the blocks, by up to a half; nothing looks at that)
constexpr int kDirectRows = 512;
int wgrad_block_rows(const scs_lowrank& p) {
    const int64_t tiles = (std::max(p.in_features, p.out_features) + 63) / 64;
    const int64_t rows = std::max<int64_t>(std::min<int64_t>(512, std::max<int64_t>(64, (p.rows * tiles / 2048 + 63) / 64 * 64)), (p.rows / 65535 + 64) / 64 * 64);
    const int64_t blocks = (p.rows + rows - 1) / rows;
    const int64_t slots = (p.n_requests + blocks) * p.rank * 4, x = p.rows * (p.dtype == SCS_F32 ? 4 : 2);             // bytes a column
    if (p.rows <= kDirectRows || blocks <= 1 || slots > 4 * x || (slots > x && p.n_requests > 4 * blocks)) return 0;
    return (int)rows;
}

// ---- project: few rows (lowrank_few.h)
struct Few { int mt = 0, splits = 1, tiles_n = 0, tiles_m = 0; size_t part = 0; int tickets = 0; };      // mt 0: the tile kernels
// f32 tiles (lowrank_tiles32.h): columns / 16 of the tile with the least padding; among equals the one that ran fastest at 60 000 x 540 x 540 (6: 306 us,
// 5: 303, 7: 321, 4: 322; 8 pads there)
int f32_columns(int64_t N) {
    int nt = 0;
    int64_t waste = INT64_MAX;
    for (const int n : {6, 5, 8, 7, 4}) {
        const int64_t w = (N + 16 * n - 1) / (16 * n) * 16 * n;
        if (w < waste) { waste = w; nt = n; }
    }
    return nt;
}
// ... and its rows / 64: the higher tile where that still gives every CU one, the lower where that gives most of them one, 0: neither does
int f32_rows(int64_t rows, int64_t N) {
    const int64_t across = (N + 16 * f32_columns(N) - 1) / (16 * f32_columns(N));
    return (rows + 127) / 128 * across >= 256 ? 2 : (rows + 63) / 64 * across >= 192 ? 1 : 0;
}
// The few-rows form: up to 64 rows in 16 bits (128 rows at 4096 x 4096 take 28 us as tiles), in f32 wherever the tiles would leave CUs idle (512 rows
// at 540 x 540: 18 us, as tiles 46).  Row tiles a workgroup, f32: two halve W's reads and the workgroups.  One / two, us: 128 x 2048 x 2048 20.5 / 22.1,
// 256 x 540 x 540 12.1 / 16.6, 512 x 1448 x 1448 43.7 / 48.5 are left to one; 300 x 1500 x 1500 30.6 / 27.6, 400 x 2048 x 1024 37.0 / 32.8 and 256 x 1024 x 2048
// 23.7 / 20.8 gain from two, 256 x 2048 x 1024 20.0 / 21.9 and 700 x 2052 x 1033 62.6 / 69.8 lose a tenth by it
Few few_of(const scs_lowrank& p, int64_t K, int64_t N) {
    Few f;
    if (p.rows == 0) return f;
    if (p.dtype == SCS_F32 ? f32_rows(p.rows, N) != 0 : p.rows > 64) return f;
    f.mt = p.dtype == SCS_F32 ? (p.rows >= 256 && K * N >= (1 << 21) ? 2 : 1) : (int)(p.rows + 15) / 16;
    f.tiles_n = (int)((N + 63) / 64);
    f.tiles_m = (int)((p.rows + 16 * f.mt - 1) / (16 * f.mt));
    const int64_t steps = (K + 31) / 32;
    f.splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / ((int64_t)f.tiles_n * f.tiles_m), steps / (2 * kFewWaves)));
    if (f.splits > 1) {
        f.part = (size_t)f.splits * f.tiles_m * 16 * f.mt * f.tiles_n * 64 * 4;
        f.tickets = f.tiles_n * f.tiles_m;
    }
    return f;
}
// What of a projection's operands has to be laid out anew for the tile kernels: K up to a multiple of 64 (16-bit) or 4 (f32), rows at multiples
// of 16 bytes.  `K`, `N`: of this direction; `x`, `ldx`: X as the call gets it.
struct Pack { bool x = false, w = false; int64_t K = 0, nw = 0, w_rows = 0, w_cols = 0; size_t x_bytes = 0, w_bytes = 0; };
Pack pack_of(const scs_lowrank& p, int64_t K, int64_t N, bool trans, const void* x, int64_t ldx) {
    Pack k;
    const int e = p.dtype == SCS_F32 ? 4 : 2, per = 16 / e, unit = p.dtype == SCS_F32 ? 4 : 64;
    auto whole = [](int64_t v, int64_t u) { return (v + u - 1) / u * u; };
    k.K = whole(K, unit);
    // (2^21: the tile kernels' offsets inside a tile have 32 bits)
    k.x = k.K != K || ldx % per || (uintptr_t)x % 16 || ldx > (1 << 21);
    k.w = k.K != K || p.ldw % per || (uintptr_t)p.w % 16 || (!trans && N % per) || p.ldw > (1 << 21);
    k.nw = trans ? N : whole(N, per);
    k.w_rows = trans ? N : k.K;
    k.w_cols = trans ? k.K : k.nw;
    if (k.x) k.x_bytes = (size_t)p.rows * k.K * e;
    if (k.w) k.w_bytes = (size_t)k.w_rows * k.w_cols * e;
    return k;
}

// ---- project: 16-bit tiles (lowrank_tiles.h)
// the largest 16-bit tile that still gives most of the 256 CUs one
int tile16(int64_t rows, int64_t N) {
    auto tiles = [&](int64_t b) { return (rows + b - 1) / b * ((N + b - 1) / b); };
    return tiles(256) >= 192 ? 256 : tiles(128) >= 192 ? 128 : 64;
}

// ---- launches of two things at once, where neither fills the card and dx does not read what the other writes
// dx of few rows and the gradients in the direct form (not with thousands of adapters: the one launch's threads along x have to stay below 2^32)
inline bool few_beside_wgrad(const scs_lowrank& p, const Few& f) { return f.mt >= 1 && f.mt <= 2 && p.rank <= 32 && p.n_adapters <= 128 && !wgrad_block_rows(p); }
// dx in the smallest 16-bit tiles and the gradients by blocks of rows
inline bool tiles_beside_wgrad(const scs_lowrank& p, const Few& f) {
    return p.dtype != SCS_F32 && !f.mt && p.rank <= 32 && tile16(p.rows, p.in_features) == 64 && wgrad_block_rows(p);
}

}  // namespace
}  // namespace scs
