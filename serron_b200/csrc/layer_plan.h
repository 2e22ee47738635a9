// How a layer norm is laid over the GPU when its rows fit in registers: vector width, vectors per thread, threads,
// cluster and number of blocks, from the sizes and alignments alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace serron {

struct NormPlan {
    bool ok = false;
    bool rows = false;  // inner == 1
    int V = 1, NV = 1;
    int tx = 32, ty = 1, clusters = 1;
    int64_t tiles = 0;   // pieces of work: the rows (rows) or columns (columns) that a block takes at a time
    int64_t blocks = 0;  // of clusters: forward one per tile, backward a grid that walks over them
};

constexpr int kSMs = 148;

// The widths tried for elements of `size` bytes, widest first; 0 ends the list.  Columns take four elements of 16 bits
// and not eight: a thread keeps four numbers for each of its V rows beside the elements.
inline const int* plan_widths(bool rows, int size) {
    static const int half[] = {8, 2, 1, 0}, four[] = {4, 1, 0};
    return rows && size == 2 ? half : four;
}

// The vectors per thread that kernels of width V exist for.
inline int round_vectors(bool rows, bool wide, int V, int64_t n) {
    if (rows && wide) return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 0;
    if (rows) return V == 2 ? (n <= 2 ? 2 : n <= 8 ? 8 : 0) : (n <= 4 ? 4 : n <= 16 ? 16 : 0);
    return wide ? (n <= 4 ? 4 : n <= 8 ? 8 : 0) : (n <= 8 ? 8 : n <= 16 ? 16 : 0);
}

inline int64_t plan_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A plan for width V, or one that is not ok.
inline NormPlan norm_plan(int64_t rows, int64_t len, int64_t inner, int V, int size, bool backward) {
    NormPlan p;
    p.rows = inner == 1;
    p.V = V;
    if (rows == 0 || (p.rows ? len : inner) % V != 0) return p;
    const bool wide = p.rows ? V * size == 16 : V == 4;
    if (p.rows) {
        const int most_warps = backward ? 16 : 32;  // of a block
        const int64_t vectors = len / V;
        // few rows: fewer vectors per thread
        int per = wide ? 4 : V == 2 ? 8 : 16;
        while (per > 1 && rows * plan_ceil(vectors, 32 * per) < kSMs * 32) per /= 2;
        const int64_t warps = plan_ceil(vectors, 32 * per);
        while (p.clusters < 8 &&
               (warps > most_warps * p.clusters || (rows * p.clusters < kSMs && warps > 8 * p.clusters)))
            p.clusters *= 2;
        p.tx = static_cast<int>(std::min<int64_t>(plan_ceil(warps, p.clusters), most_warps)) * 32;
        p.ty = p.tx == 32 ? static_cast<int>(std::min<int64_t>(backward ? 8 : 4, rows)) : 1;
        p.NV = round_vectors(true, wide, V, plan_ceil(vectors, int64_t(p.tx) * p.clusters));
        p.tiles = plan_ceil(rows, p.ty);
    } else {
        const int64_t columns = rows / V;
        int per = wide ? 8 : 16;
        if (columns * plan_ceil(len, per) < kSMs * 16 * 32 || len <= per / 2) per /= 2;
        if (plan_ceil(len, per) > 16) per = wide ? 8 : 16;
        while (p.clusters < 8 && plan_ceil(len, per) > 16 * p.clusters) p.clusters *= 2;
        const int64_t groups = plan_ceil(plan_ceil(len, per), p.clusters);
        if (groups > 16) return p;
        p.NV = round_vectors(false, wide, V, per);
        p.ty = static_cast<int>(groups);
        p.tx = 32 * std::max(1, 4 / p.ty);
        p.tiles = plan_ceil(columns, p.tx);
    }
    p.blocks = p.tiles;
    if (backward) {
        // as many blocks as are resident, each with the same number of tiles, and no more than 128 tiles each, which
        // keeps the sums of the parameters' gradients as exact as a tree's
        const int64_t resident = std::max<int64_t>(1, kSMs * (512 / (p.tx * p.ty)) / p.clusters);
        p.blocks = plan_ceil(p.tiles, std::min<int64_t>(plan_ceil(p.tiles, resident), 128));
    }
    p.ok = p.NV > 0 && p.blocks < (int64_t(1) << 31) - 1;
    return p;
}

}  // namespace serron
