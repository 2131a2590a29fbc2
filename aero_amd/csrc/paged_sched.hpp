// Which keys an attention call over few query rows walks, and who walks them:
// plain arithmetic for the kernels (attn_rows.hip), the host side and a CPU test.
//
// The keys that some query of positions [q_lo, q_hi] sees are a list of 16-key
// tiles: with a window, those that hold the sinks and those from the window's
// first key on (one run where the two meet), else all up to q_hi. A tile lies
// in one page (pages are 16 tokens or more, a power of two).
//
// The tiles of an item (sequence, kv head, query tile) are grouped into units,
// the units into chunks, one a workgroup: as many of about the same size as fill
// the chip, whatever the items' lengths.
#pragma once

#include <cstdint>

#ifdef __HIP__
#define AERO_HD __host__ __device__ __forceinline__
#else
#define AERO_HD inline
#endif

namespace aero {

struct KeyTiles {
    int32_t n_sink;   // tiles of the sinks: tiles 0 .. n_sink - 1
    int32_t first;    // the tile after them (the window's first)
    int32_t n;        // tiles in all

    // the 16-key tile at place x of the list
    AERO_HD int32_t at(int32_t x) const { return x < n_sink ? x : x - n_sink + first; }
    // the place of tile x (one of the list's)
    AERO_HD int32_t place(int32_t x) const { return x < n_sink ? x : x - first + n_sink; }
    // a page list with no gaps: the sinks' pages, then the window's; the place
    // there of the page of list place x (shift: log2 of tiles a page)
    AERO_HD int32_t page_place(int32_t x, int shift) const {
        const int32_t page = at(x) >> shift;
        return x < n_sink ? page : page - (first >> shift) + sink_pages(shift);
    }
    AERO_HD int32_t sink_pages(int shift) const {
        return (n_sink + (1 << shift) - 1) >> shift;
    }
    // the table column at a place of that list
    AERO_HD int32_t column(int32_t place, int shift) const {
        const int32_t s = sink_pages(shift);
        return place < s ? place : place - s + (first >> shift);
    }
};

// Keys below n_kv seen from positions q_lo .. q_hi (q_hi < q_lo or q_hi < 0:
// none), in tiles of `tile` keys. Positions are those of the keys' places.
AERO_HD KeyTiles key_tiles(int64_t q_lo, int64_t q_hi, int64_t n_kv, int32_t window,
                           int32_t sinks, int32_t tile = 16) {
    KeyTiles t{0, 0, 0};
    const int64_t hi = q_hi + 1 < n_kv ? q_hi + 1 : n_kv;   // keys 0 .. hi - 1
    if (hi <= 0 || q_lo > q_hi) return t;
    const int32_t last = (int32_t)((hi + tile - 1) / tile);
    if (window > 0) {
        int64_t lo = q_lo - window + 1;
        lo = lo < 0 ? 0 : (lo < hi ? lo : hi);
        const int64_t s = sinks < lo ? sinks : lo;
        const int32_t ns = (int32_t)((s + tile - 1) / tile), first = (int32_t)(lo / tile);
        if (ns < first) {
            t.n_sink = ns;
            t.first = first;
            t.n = ns + last - first;
            return t;
        }
    }
    t.n = last;
    return t;
}

// units of an item: at least one, so that some workgroup writes its rows
AERO_HD int32_t item_units(int32_t n_tiles, int32_t tiles_a_unit) {
    const int32_t u = (n_tiles + tiles_a_unit - 1) / tiles_a_unit;
    return u > 0 ? u : 1;
}

// The chunks of an item of u units where all items' units, `total`, are to make
// about `target` chunks: at most total / target units each (rounded up), so no
// more than target + items in all, and no more than 2 target in the items that
// have several.
AERO_HD int32_t item_chunks(int32_t u, int32_t total, int32_t target) {
    const int32_t most = (total - 1) / target + 1;
    return (u - 1) / most + 1;
}
// chunk c of n takes units [chunk_begin(c), chunk_begin(c + 1)) of u
AERO_HD int32_t chunk_begin(int32_t c, int32_t n, int32_t u) {
    const int32_t each = u / n, more = u - each * n;     // (the first `more` take one more)
    return c * each + (c < more ? c : more);
}

}  // namespace aero
