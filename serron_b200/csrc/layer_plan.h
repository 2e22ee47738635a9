// How a layer norm is laid over the GPU when its rows fit in registers: vector width, vectors per thread, threads,
// cluster and number of blocks, from the sizes and alignments alone.
#pragma once

#include <algorithm>
#include <cstdint>

namespace serron {

struct NormPlan {
    bool ok = false;
    bool rows = false;  // inner == 1
    int V = 1;          // elements of a vector
    int NV = 1, R = 1;  // vectors of a row that a thread takes; rows: rows it takes at a time
    bool full = false;  // columns: no thread has fewer
    int tx = 32, ty = 1, clusters = 1;
    int64_t tiles = 0;   // pieces of work: the rows (rows) or columns (columns) that a block takes at a time
    int64_t blocks = 0;  // of clusters; a forward pass over rows has one per tile, the others a grid that walks over them
};

constexpr int kSMs = 148;

inline int64_t plan_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The widths tried for elements of `size` bytes, widest first; 0 ends the list.  Columns take four elements of 16 bits
// and not eight: a thread keeps several numbers for each of its V rows beside the elements.
inline const int* plan_widths(bool rows, int size) {
    static const int half[] = {8, 2, 1, 0}, four[] = {4, 1, 0};
    return rows && size == 2 ? half : four;
}

// The (NV, R) that row kernels exist for, by what a vector is: 16 bytes, two elements, one element.
struct RowShape {
    int NV, R;
};
inline const RowShape* row_shapes(bool wide, int V) {
    static const RowShape w[] = {{1, 4}, {2, 2}, {4, 1}, {0, 0}}, pair[] = {{2, 4}, {8, 1}, {0, 0}},
                          single[] = {{4, 4}, {16, 1}, {0, 0}};
    return wide ? w : V == 2 ? pair : single;
}

// A plan for width V, or one that is not ok.
inline NormPlan norm_plan(int64_t rows, int64_t len, int64_t inner, int V, int size, bool backward) {
    NormPlan p;
    p.rows = inner == 1;
    p.V = V;
    if (rows == 0 || (p.rows ? len : inner) % V != 0) return p;
    if (p.rows) {
        constexpr int kMostThreads = 512;
        const int64_t vectors = len / V;
        const RowShape* shape = row_shapes(V * size == 16, V);
        // as few vectors per thread as leave a row to 8 warps, then to 16, then to a cluster
        const RowShape* best = shape;
        for (const RowShape* s = shape; s->NV; ++s) {
            best = s;
            if (vectors <= int64_t(s->NV) * 256) break;
        }
        if (backward && V * size == 16 && best->NV == 4) --best;  // its sums would not fit in registers beside the rows
        p.NV = best->NV;
        p.R = best->R;
        int64_t threads = plan_ceil(vectors, p.NV);
        // few rows: one at a time, over as many blocks as have something to do
        if (plan_ceil(rows, p.R) * threads < int64_t(kSMs) * 512) {
            p.R = 1;
            p.NV = shape->NV;
            threads = plan_ceil(vectors, p.NV);
            while (p.clusters < 8 && rows * p.clusters < kSMs && threads > 256 * p.clusters) p.clusters *= 2;
            while (p.clusters == 8 && threads > int64_t(kMostThreads) * 8 && p.NV < best->NV) {
                p.NV = (++shape)->NV;
                threads = plan_ceil(vectors, p.NV);
            }
        }
        while (p.clusters < 8 && threads > int64_t(kMostThreads) * p.clusters) p.clusters *= 2;
        threads = plan_ceil(threads, p.clusters);
        if (threads > kMostThreads) return p;
        if (threads <= 32) {
            p.tx = 1;
            while (p.tx < threads) p.tx *= 2;
            p.ty = 256 / p.tx;
            while (p.ty > 1 && p.tx * p.ty > 32 && int64_t(p.ty / 2) * p.R >= rows) p.ty /= 2;
        } else {
            p.tx = static_cast<int>(plan_ceil(threads, 32)) * 32;
        }
        p.tiles = plan_ceil(rows, int64_t(p.ty) * p.R);
    } else {
        const int64_t columns = rows / V;
        // what fits in registers without spilling: 64 bytes of each tensor, in float32 128 of the one of a forward pass
        int per = V == 4 ? (backward && size == 4 ? 4 : 8) : 16;
        const int least = V == 4 ? 4 : 8;
        while (per > least && (len <= per / 2 || columns * plan_ceil(len, per) < int64_t(kSMs) * 512) &&
               plan_ceil(len, per / 2) <= 16)
            per /= 2;
        while (p.clusters < 8 && plan_ceil(len, per) > 16 * p.clusters) p.clusters *= 2;
        const int64_t groups = plan_ceil(plan_ceil(len, per), p.clusters);
        if (groups > 16) return p;
        p.NV = per;
        p.ty = static_cast<int>(groups);
        p.full = V == 4 && len == int64_t(per) * groups * p.clusters;
        p.tx = 32 * std::max(1, 4 / p.ty);
        p.tiles = plan_ceil(columns, p.tx);
    }
    p.blocks = p.tiles;
    if (backward || !p.rows) {
        // as many blocks as are resident, each with the same number of tiles; and in a backward pass no more than 128
        // rows to a sum of the parameters' gradients, which keeps those as exact as a tree's
        const int64_t resident = std::max<int64_t>(1, int64_t(kSMs) * (512 / (p.tx * p.ty)) / p.clusters);
        int64_t each = plan_ceil(p.tiles, resident);
        if (backward) each = std::min<int64_t>(each, 128 / p.R);
        p.blocks = plan_ceil(p.tiles, each);
    }
    p.ok = p.blocks < (int64_t(1) << 31) - 1;
    return p;
}

}  // namespace serron
