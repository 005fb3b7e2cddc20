// How the work of paged attention is dealt to a fixed number of workers (thread blocks), shared by the kernels and, as
// plain C++, by the host-side tests.
//
// A segment is one (row, head tile): a row's keys and values read by the query heads of one tile.  It consists of tiles of
// `tile` consecutive positions on the absolute grid (so that 16 tokens from a multiple of 16 are never cut), and counts as
// that many units and SEGMENT_COST more for its beginning and end.  All segments' units are numbered row by row, head tile
// by head tile, and dealt to the workers in equal shares, the first U % W of the W workers one unit more (W <= U: every
// worker has one): at most one unfinished segment at either end of a share, whatever the lengths.
//
// Positions and units are 32-bit: positions are below 2^31 (the page table is checked), and the host passes so few rows at
// a time that units are, too.  64-bit division, the first version's, took 2 us of a call for one token.
#pragma once
#include "kv_place.h"

namespace te {

// Positions [first, n) that a row attends to.
struct RowRange {
    int first, n;
};
TE_HD RowRange row_range(int64_t len, int most, int64_t window) {
    RowRange r;
    r.n = len < 0 ? 0 : len > most ? most : (int)len;
    r.first = window > 0 && r.n > window ? r.n - (int)window : 0;
    return r;
}
TE_HD int row_tiles(const RowRange& r, int tile) {
    return r.n <= r.first ? 0 : (int)(((unsigned)r.n + tile - 1) / (unsigned)tile - (unsigned)r.first / (unsigned)tile);
}

struct Shares {
    int workers, base, more;        // units of a share; this many workers have one more
};
TE_HD Shares shares_of(int units, int workers) {
    Shares s;
    s.workers = workers;
    s.base = (int)((unsigned)units / (unsigned)workers);
    s.more = units - s.base * workers;
    return s;
}
TE_HD int share_begin(const Shares& s, int w) { return w * s.base + (w < s.more ? w : s.more); }
// The worker whose share holds unit u.
TE_HD int worker_of(const Shares& s, int u) {
    const int big = s.more * (s.base + 1);
    return u < big ? (int)((unsigned)u / (unsigned)(s.base + 1)) : s.more + (int)((unsigned)(u - big) / (unsigned)s.base);
}

// 1: 16 rows of 20 key heads under a window take 40 us (44 with 0, 41 with 3), 256 rows of up to 300 tokens 27 (27, 29).
constexpr int SEGMENT_COST = 1;
// Units of a row's segment; a row without tiles has none.
TE_HD int segment_units(int tiles) { return tiles > 0 ? tiles + SEGMENT_COST : 0; }

// Where a worker keeps the part of a segment that it does not finish alone: place 0 for the segment its share begins
// inside of, place 1 for the one that begins in its share and continues behind it.
TE_HD int part_slot(int worker, bool begins_here) { return 2 * worker + (begins_here ? 1 : 0); }

// What a worker computes of one segment.
struct Piece {
    int row, head_tile;
    RowRange range;
    int first_tile;            // on the absolute grid
    int tiles;
    bool begins, ends;         // holds the segment's first tile, its last
    int segment_end;           // unit behind the segment
};

// Goes through a worker's pieces in order.  RangeOf: row -> RowRange.
struct Walker {
    int unit, end;             // of the share: what is left
    int segment;               // first unit of the present segment
    int row, head_tile, tiles; // tiles of the present row, -1 before it has been looked at
    RowRange range;

    // The share [unit, end) begins in row `row`, whose units begin at row_begin.
    TE_HD void start(int unit_, int end_, int row_, int row_begin) {
        unit = unit_;
        end = end_;
        segment = row_begin;
        row = row_;
        head_tile = 0;
        tiles = -1;
        range.first = range.n = 0;
    }
    template <class RangeOf>
    TE_HD bool next(const RangeOf& range_of, int head_tiles, int tile, Piece& piece) {
        while (unit < end) {
            if (tiles < 0) {
                range = range_of(row);
                tiles = row_tiles(range, tile);
                if (tiles > 0 && unit - segment >= segment_units(tiles)) {      // only in the share's first row
                    const int skip = (int)((unsigned)(unit - segment) / (unsigned)segment_units(tiles));
                    head_tile = skip;
                    segment += skip * segment_units(tiles);
                }
            }
            if (tiles == 0 || head_tile >= head_tiles) {
                ++row;
                head_tile = 0;
                tiles = -1;
                continue;
            }
            const int segment_end = segment + segment_units(tiles), stop = end < segment_end ? end : segment_end;
            const int a = unit - segment - SEGMENT_COST, b = stop - segment - SEGMENT_COST;
            const int from = a > 0 ? a : 0, to = b > 0 ? b : 0;
            piece.row = row;
            piece.head_tile = head_tile;
            piece.range = range;
            piece.first_tile = range.first / tile + from;
            piece.tiles = to - from;
            piece.begins = from == 0;
            piece.ends = to == tiles;
            piece.segment_end = segment_end;
            unit = stop;
            if (stop == segment_end) {
                segment = segment_end;
                ++head_tile;
            }
            if (to > from) return true;
        }
        return false;
    }
};

}  // namespace te
