// How a call of the paged attention is cut into workgroups, and the workspace that this takes: host
// arithmetic alone.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstddef>

#include "../../include/jasmine_hip.h"

namespace jas {

// How a call is launched
struct PagedPlan {
    int rows;  // of a tile: 16 (its waves share the keys), 64 or 128
    long tiles;
    int nsplit, chunk;
};

// Rounds of workgroups that tiles whose keys are split make, and the fewest keys of a split
constexpr int paged_rounds(int rows) { return rows == 16 ? 8 : rows == 64 ? 4 : 2; }
constexpr int paged_least(int rows) { return rows == 16 ? 128 : 256; }

// Tiles of 16 rows stream the keys once for each tile, without LDS: for sequences whose new rows
// (tokens times the query heads of a key head) fit one.  Otherwise tiles of 64 rows, or of 128, which
// read fragments from LDS for twice the products but come in half the number, less evenly loaded.
// (us, tiles of 128 and of 64; lengths spread up to what is named, 32 query heads of 128 on 8 but as said)
//   fp32 rows, 12 heads of 64: 16 x up to 200 tokens over 1024 keys 98, 55; 8 x 1024 92, 81; 2 x 333 over 2001
//     39.5, 38.5; 500 over 8000 93, 102: always 64
//   bf16 rows, 128 give a workgroup to every unit: 4 x 512 over 4096 121, 138; 24 x 256 beside single tokens over
//     2048, e4m3 88, 94
//   only 64 do, with some over: 2 x 512 over 4096 106, 86, int8 135, 112; 6 x 300 over 2048, 16 heads of 64, int8 68, 48
//   neither does: 512 over 8192, int8 135, 212; 300 over 6000 80, 80
inline PagedPlan paged_plan(int n, int B, int H, int n_kv, int max_q, int max_len, int dtype, long cus)
{
    PagedPlan r;
    max_len = std::min(max_len, 0x7fff0000);  // (no table's row holds more: PagedView)
    const long G = H / n_kv, most = std::min((long)max_q, (long)n) * G;
    auto full = [&](int rows) { return std::max((long)B, (long)n * G / rows) * n_kv; };  // tiles, about
    r.rows = most <= 16 ? 16 : most <= 64 || dtype == JAS_F32 || (full(128) < cus && full(64) >= cus + cus / 8) ? 64 : 128;
    // sequence b owns tiles from floor(cu[b] G / rows) + b on
    r.tiles = (long)n * G / r.rows + B;
    // Splits of `chunk` keys: enough workgroups to fill the chip some times over, so that sequences of
    // different lengths even out; a split that a shorter sequence does not need ends at once.
    // Tiles of 16 rows: eight rounds of one workgroup a unit (32 sequences of 1024 to 4096 keys, 8
    // heads, bf16: 75.2, 71.0, 72.1, 78.9 us at 6, 8, 12, 16).  Larger tiles are bound by the matrix
    // cores and their partial results are large: split only where units would be left without one
    // (2 x 333 rows over 2001 keys, 12 heads of 64, fp32: 81, 38.5 us unsplit and split; 4 chunks of 512
    // over 4096, bf16: 121, 167), those of 64 into four rounds (that fp32: 41.7, 38.7, 38.3 at 2, 3, 4),
    // those of 128 into two (512 over 8192, int8: 169, 135, 161, 143 at 1.5, 2, 3, 4).  An odd number of
    // splits: see paged_block.  One plan for the whole call: beside chunks that fill the chip a single token's
    // keys are not split either (3 chunks of 512 over 4096 and one token over 32768 keys: 839 us, 120 and 36 apart).
    if (r.rows > 16 && full(r.rows) >= cus) r.chunk = std::max(max_len, 1), r.nsplit = 1;
    else {
        // (a fraction of a key counts: a chunk below the share makes more splits than paged_bytes allows for)
        const double share = std::ceil((double)full(r.rows) * max_len / (paged_rounds(r.rows) * cus));
        r.chunk = (int)std::min(((long)std::max((double)paged_least(r.rows), std::min(share, (double)max_len)) + 127) / 128 * 128, 0x7fff0000L);
        r.nsplit = (int)std::max(1L, std::min(((long)max_len + r.chunk - 1) / r.chunk, 63L));
        if (r.nsplit > 1) r.nsplit |= 1;
    }
    return r;
}

// Bytes that hold the partial results of every call within the given numbers: fewer rows can need more
// than many, whose keys are not split.  With x = max(B, n G / rows) n_kv there are at most 2 x tiles of
// all heads.  A chunk is at least max_len x / (rounds cus) keys, so a tile has at most rounds cus / x + 1
// splits, and one more to make them odd: 2 rounds cus + 4 x in all, where x is below rounds cus (one split
// otherwise) and for tiles of 64 and 128 below cus (not split otherwise).
inline size_t paged_bytes(int rows, int n, int B, int H, int n_kv, int D, int max_len, double cus)
{
    if (max_len <= paged_least(rows)) return 0;
    const double rounds = paged_rounds(rows), G = H / n_kv;
    const double x = std::min(std::max((double)B, n * G / rows) * n_kv, (rows == 16 ? rounds : 1.0) * cus);
    const double parts = std::min(2 * rounds * cus + 4 * x, (n * G / rows + B) * n_kv * std::min(63.0, (double)max_len / paged_least(rows) + 2));
    return (size_t)parts * rows * (D + 4) * sizeof(float);
}

// Bytes that a plan's workgroups write
inline size_t paged_need(const PagedPlan &r, int n_kv, int D)
{
    return r.nsplit > 1 ? (size_t)r.tiles * n_kv * r.nsplit * r.rows * (D + 4) * sizeof(float) : 0;
}

inline size_t paged_workspace(int n, int B, int H, int n_kv, int D, int max_q, int max_len, double cus)
{
    const double most = std::min((double)max_q, (double)n) * (H / n_kv);
    size_t bytes = paged_bytes(16, n, B, H, n_kv, D, max_len, cus);
    if (most > 16) bytes = std::max(bytes, paged_bytes(64, n, B, H, n_kv, D, max_len, cus));
    if (most > 64) bytes = std::max(bytes, paged_bytes(128, n, B, H, n_kv, D, max_len, cus));
    return bytes;
}

} // namespace jas
