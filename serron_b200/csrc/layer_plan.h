// How a layer norm is laid over the GPU when its rows fit in registers: vector width, vectors per thread, threads,
// cluster and number of blocks, from the sizes and alignments alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace serron {

struct NormPlan {
    bool ok = false;
    bool rows = false;     // inner == 1
    int V = 1;             // elements of a vector
    int NV = 1, R = 1;     // vectors of a row that a thread takes; rows: rows it takes at a time
    bool shifted = false;  // rows: V does not divide len
    bool full = false;     // columns: no thread has fewer than NV
    int tx = 32, ty = 1, clusters = 1;
    int64_t tiles = 0;   // pieces of work: the rows (rows) or columns (columns) that a block takes at a time
    int64_t blocks = 0;  // of clusters, a grid that walks over the tiles
};

constexpr int kSMs = 148;

inline int64_t plan_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The widths tried for elements of `size` bytes, wider first; 0 ends the list.  Columns take four elements of 16 bits
// and not eight: a thread keeps several numbers for each of its V rows beside the elements.
inline const int* plan_widths(bool rows, int size) {
    static const int half[] = {8, 1, 0}, four[] = {4, 1, 0};
    return rows && size == 2 ? half : four;
}

// Rows: the kernels are NV x R = 1 x 4, 2 x 2, 4 x 1 (and 1 x 1, 2 x 1) with vectors of 16 bytes, 4 x 4, 4 x 1 and 16 x 1
// with single elements, which only pointers off a vector's boundary come to.
inline void plan_rows(NormPlan& p, int64_t rows, int64_t len, int size, bool backward) {
    const bool wide = p.V * size == 16;
    p.shifted = len % p.V != 0;
    const int64_t vectors = plan_ceil(len + (p.shifted ? p.V - 1 : 0), p.V);
    constexpr int kMostThreads = 512;
    // a row to as few warps as may be, so that what is done once a row and thread is shared by more elements ((8192,1024)
    // bfloat16 forward: 11.5 us with one warp a row, 17.6 with four warps for four rows); a backward pass also keeps two sums
    // for each of a thread's elements of a row, and takes no more than 16 (22 us against 36 with 32)
    const int most = wide ? (backward && p.V == 8 ? 2 : 4) : 16;
    p.NV = wide ? (vectors <= 32 ? 1 : vectors <= 64 ? 2 : most) : (vectors <= 128 ? 4 : 16);
    p.R = wide ? 4 / p.NV : p.NV == 4 ? 4 : 1;
    int64_t threads = plan_ceil(vectors, p.NV);
    // few rows: one at a time, with fewer vectors per thread and over more blocks (16 rows of 65536 bfloat16 forward: 7 us
    // over clusters of eight blocks, 10 in chunks joined by further launches)
    if (plan_ceil(rows, p.R) * std::max<int64_t>(threads, 32) < int64_t(kSMs) * 512) {
        p.R = 1;
        p.NV = wide ? 1 : 4;
        while (p.NV < most && plan_ceil(vectors, p.NV) > (rows < kSMs ? 4 : 1) * 512) p.NV = wide ? 2 * p.NV : 16;
        threads = plan_ceil(vectors, p.NV);
        while (p.clusters < 8 && rows * p.clusters < kSMs && threads > 256 * p.clusters) p.clusters *= 2;
    }
    while (p.clusters < 8 && threads > 256 * p.clusters) p.clusters *= 2;  // several to an SM
    threads = plan_ceil(threads, p.clusters);
    if (threads > kMostThreads) return;
    if (threads <= 32) {
        p.tx = 1;
        while (p.tx < threads) p.tx *= 2;
        p.ty = 128 / p.tx;
        while (p.ty > 1 && p.tx * p.ty > 32 && int64_t(p.ty / 2) * p.R >= rows) p.ty /= 2;
    } else {
        p.tx = static_cast<int>(plan_ceil(threads, 32)) * 32;
    }
    const int64_t at_once = int64_t(p.ty) * p.R;
    p.tiles = !p.shifted ? plan_ceil(rows, at_once)
              : rows < p.V ? rows
                           : p.V * plan_ceil(plan_ceil(rows, p.V), at_once);
    p.ok = true;
}

// Columns: NV = 4, 8 (and 16 for 16-bit forward passes) with V = 4, NV = 8, 16 with V = 1.
inline void plan_columns(NormPlan& p, int64_t rows, int64_t len, int64_t inner, int size, bool backward) {
    if (len * inner >= int64_t(1) << 31) return;
    const int64_t columns = rows / p.V;
    // what fits in registers but for a few spilled words (48 bytes at most): 64 bytes of each tensor, of the one of a
    // forward pass 128 ((64,32,256,256) bfloat16 forward: 105 us with 16 strides a thread, 147 with 8; backward 165
    // with 8, 249 with 4)
    int per = p.V == 4 ? std::max(4, (backward ? 8 : 16) / (size / 2)) : 16;
    const int least = p.V == 4 ? 4 : 8;
    while (per > least && (len <= per / 2 || columns * plan_ceil(len, per) < int64_t(kSMs) * 512) &&
           plan_ceil(len, per / 2) <= 16)
        per /= 2;
    while (p.clusters < 8 && plan_ceil(len, per) > 16 * p.clusters) p.clusters *= 2;
    const int64_t groups = plan_ceil(plan_ceil(len, per), p.clusters);
    if (groups > 16) return;
    p.NV = per;
    p.ty = static_cast<int>(groups);
    p.full = p.V == 4 && len == int64_t(per) * groups * p.clusters;
    p.tx = 32 * std::max(1, 4 / p.ty);
    p.tiles = plan_ceil(columns, p.tx);
    p.ok = true;
}

// A plan for width V, or one that is not ok.
inline NormPlan norm_plan(int64_t rows, int64_t len, int64_t inner, int V, int size, bool backward) {
    NormPlan p;
    p.rows = inner == 1;
    p.V = V;
    if (rows == 0 || (!p.rows && inner % V != 0)) return p;
    if (rows > (int64_t(1) << 34) / len) return p;  // the join's generator counts blocks of four elements in 32 bits here
    if (p.rows)
        plan_rows(p, rows, len, size, backward);
    else
        plan_columns(p, rows, len, inner, size, backward);
    if (!p.ok) return p;
    // the grid walks over the tiles: as many blocks as are resident, each with the same number of tiles (or one, where that
    // is two rounds of blocks at most)
    const int threads = p.tx * p.ty;
    const int on_an_sm = p.rows && !backward ? 1024 : 512;
    const int64_t resident = std::max<int64_t>(1, int64_t(kSMs) * std::max(1, on_an_sm / threads) / p.clusters);
    int64_t each = p.tiles <= 2 * resident ? 1 : plan_ceil(p.tiles, resident);
    // No more than 128 rows (rows) or 256 pairs of a lane's rows (columns: two a tile) to a thread's part of a float32 sum of
    // the parameters' gradients.  A block adds up its threads' parts in float32 too: the groups one after the other, at
    // most 128 (rows of up to eight elements); the lanes of a warp as a tree, then its four warps.  So no term takes
    // part in more than about 270 additions before the sums of the blocks, which are joined in double.
    if (backward)
        each = std::min<int64_t>(each, 128 / p.R);
    else if (p.rows)  // little is done once a block: rather four rounds of blocks (10.9 us against 14.1)
        each = std::max<int64_t>(1, each / 4);
    p.blocks = plan_ceil(p.tiles, each);
    // a block of shifted rows takes every V-th tile
    if (p.shifted && p.blocks < p.tiles) p.blocks = std::min(p.tiles, plan_ceil(p.blocks, p.V) * p.V);
    p.ok = p.blocks < (int64_t(1) << 31) - 1;
    return p;
}

// Floats of dynamic shared memory that the plan's kernel takes.  Rows: a backward pass joins the parameters' sums of a
// block's groups there.  Columns: column_totals' scratch for one number a row, for two in a backward pass, and at its
// end two sums per channel and warp.  No plan takes more than 48 KB, which need not be asked for.
inline int64_t plan_shared_floats(const NormPlan& p, bool backward) {
    if (p.rows) return backward && p.ty > 1 ? int64_t(p.NV) * p.V * p.tx * p.ty : 0;
    const int64_t totals = (p.ty > 1 || p.clusters > 1) ? (2 * int64_t(p.ty) + 2) * p.tx * p.V : 0;
    return backward ? std::max(2 * totals, int64_t(p.NV) * p.ty * (p.tx / 32) * 2) : totals;
}

}  // namespace serron
