// The page numbers that a walk over a paged cache has at hand (dsa_paged_walk.h): which lie where, and when more of them are asked for.  Plain C++, without memory: a test runs it
// on the CPU for every place among the pages that a piece may begin at.
#pragma once

// Numbers go in batches of 64 (a load of one each by the lanes), batch b in half b & 1 of a ring of 128.  Tiles of 32 keys are counted from the piece's first one, which lies anywhere among
// the pages.
struct PageRing {
    int base, pshift;                                    // the piece's first tile; log2 of a page's rows
    constexpr int page(int tile) const { return (base + tile) * 32 >> pshift; }              // of the tile's first row
    constexpr int batch(int tile) const { return page(tile) >> 6; }
    static constexpr int place(int page) { return page & 127; }
    // In front of the walk come the first tile's batch and the one behind it.  In the walk the batch after next is asked for at a batch's first page, by the step that requests V of
    // `tile`, 3 or later: what lies in front of that page has been looked up, so its batch's half is free, and K, three tiles ahead, is far from needing it.
    constexpr bool due(int tile) const { return (page(tile) & 63) == 0; }
    // Tiles 1 and 2 have no such step: where a batch begins with one of them, the one behind it is asked for once they have been looked up.
    constexpr bool due_early() const { return batch(2) != batch(0); }
};
