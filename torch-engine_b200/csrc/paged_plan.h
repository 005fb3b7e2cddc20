// How the work of paged attention is dealt to a fixed number of workers (thread blocks), shared by the kernels and, as
// plain C++, by the host-side tests.
//
// A segment is one (row, head tile): a row's keys and values read by the query heads of one tile.  It consists of tiles of
// `tile` consecutive positions on the absolute grid (so that a tile of aligned pages starts at a page's multiple of 16).
// All segments' tiles are numbered row by row, head tile by head tile; worker w of W takes the units
// [U w / W, U (w + 1) / W) of the U (W <= U: every worker has one): equal shares whatever the lengths, at most one unfinished segment at either end.
#pragma once
#include "kv_place.h"

namespace te {

// Positions [first, n) that a row attends to.
struct RowRange {
    int64_t first, n;
};
TE_HD RowRange row_range(int64_t len, int64_t most, int64_t window) {
    RowRange r;
    r.n = len < 0 ? 0 : len > most ? most : len;
    r.first = window > 0 && r.n > window ? r.n - window : 0;
    return r;
}
TE_HD int row_tiles(const RowRange& r, int tile) {
    return r.n <= r.first ? 0 : (int)((r.n + tile - 1) / tile - r.first / tile);
}

TE_HD int64_t worker_begin(int64_t units, int workers, int w) { return units * w / workers; }
// The worker whose share holds unit u: the smallest w with worker_begin(w + 1) > u.
TE_HD int worker_of(int64_t units, int workers, int64_t u) { return (int)(((u + 1) * workers + units - 1) / units) - 1; }

// Where a worker keeps the part of a segment that it does not finish alone: place 0 for the segment its share begins
// inside of, place 1 for the one that begins in its share and continues behind it.
TE_HD int part_slot(int worker, bool begins_here) { return 2 * worker + (begins_here ? 1 : 0); }

}  // namespace te
