// How the slices of all items are numbered and cut into thread blocks' shares: the arithmetic alone, for the attention kernel
// (attend.cuh) and for a replay on the host.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define UCMX_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define UCMX_HOST_DEVICE inline
#endif

namespace ucmx {
namespace attend {

// One item's part inside a thread block's range, in units (leads included).
struct Seg {
    int32_t begin, end;                // of the whole item
    int32_t lo, hi;                    // the part of it
    int32_t from, to;                  // that part's slices, counted from the item's first
    int32_t r, h, ct;
    int32_t first;                     // offsets[r]
    int32_t n;                         // entries of the request's list; -1: not an item
};

// An item's fixed cost in slices: queries in, four warps' results joined, result out.  Tiles of 16 and 32 columns have more to join
// (24 requests of 8..40 columns: 41.8 us with 16, 37.4 with 24, 38.4 with 32; a tile of 4, 4 bits, 3 requests: 11.4 us with 16, 12.5 with 24).
constexpr int lead_of(bool tiled) { return tiled ? 24 : 16; }
constexpr int kLeadMost = lead_of(true);
constexpr int kMaxScan = 1023;         // requests whose column tiles are counted exactly
// Items up to this many units, for shares of `size` units, are not split.  Where the shares are small a thread block has an item or two
// whatever is done, and whole ones need no joining, up to 32 slices (119 requests of 6 to 18 slices: 10.2 us, 11.7 where the longer of
// them are split; beyond 32 slices the warps' own share of an item grows: 3 requests over 4 bits 17.7 us with 64, 11.4 so).  Where the
// shares are larger a whole item makes one that much longer than the others (the 24 requests above: 42.8 us with 56 units, 37.4 so).
UCMX_HOST_DEVICE constexpr int whole_of(int size, int lead) { return size < 64 ? 32 + lead : size / 8 > 32 ? size / 8 : 32; }

// All units of a launch stay below this, and so does what is added to them (the host refuses a batch whose lists, ascending and
// inside their arrays, could need more).
constexpr int32_t kUnitLimit = INT32_MAX - (1 << 20);
// What the sum over the requests (mult = heads) stops at: more than any batch has that is not refused.
UCMX_HOST_DEVICE int32_t most_units(int32_t heads) { return kUnitLimit / heads; }
inline bool too_many_units(int64_t units, int64_t heads, int64_t tiles)      // on the host: for lists as long as their arrays
{
    return units > INT32_MAX / 2 || units * heads > INT32_MAX / 2 || units * heads * tiles > kUnitLimit - heads;
}

// How the units are shared out.  Request r begins at (base(r) - base(0)) * mult: base(r) = offsets[r] * spe + r * lead with mult = KV heads x
// column tiles; or, where requests may need several tiles, base(r) = the sum of (slices + lead) x tiles of the requests before it,
// built in shared memory, with mult = KV heads (the tiles of a request depend on its number of query tokens).
struct Share {
    const int32_t* scan;               // nullptr: from the offsets
    int32_t mult, tiles;
    int32_t zero;                      // base(0): the lists may begin anywhere in the entry arrays
    int32_t lo, hi;                    // this thread block's units
    int32_t size;                      // units of a thread block
    int32_t whole;
    int32_t step;                      // the first level of the search: every step-th base,
    const int32_t* probes;             // 32 of them in shared memory
};

UCMX_HOST_DEVICE int32_t at_least(int32_t x, int32_t y) { return x > y ? x : y; }
UCMX_HOST_DEVICE int32_t at_most(int32_t x, int32_t y) { return x < y ? x : y; }

// An offset as it is used: inside the entry arrays.
UCMX_HOST_DEVICE int32_t inside(int32_t offset, int32_t total) { return at_least(0, at_most(offset, total)); }

// Offsets of one request that the lists cannot have: reported, and nothing outside the arrays or the workspace is touched for them.
UCMX_HOST_DEVICE bool bad_offsets(int32_t x, int32_t y, int32_t total) { return x < 0 || y < x || y > total; }

// Does place `at` (not negative) lie in the row [t0, t1) of a table of `size` entries?  t0 and t1 may be anything.
UCMX_HOST_DEVICE bool in_row(int32_t t0, int32_t t1, int32_t size, int32_t at)
{
    return t0 >= 0 && (int64_t)t0 + at < at_most(t1, size);
}

// Sum of units that stops at `most` (offsets that go up and down add up to more than there are).
UCMX_HOST_DEVICE int32_t add_units(int32_t x, int32_t y, int32_t most)
{
    const uint32_t sum = (uint32_t)x + (uint32_t)y;
    return sum < (uint32_t)most ? (int32_t)sum : most;
}
// base0, base_end: base(0) and base(n_req).  A sum that reached its end is no batch: none of it is done.
UCMX_HOST_DEVICE void share_out(Share& w, int32_t base0, int32_t base_end, uint32_t block, uint32_t blocks, int lead)
{
    const bool none = base_end < base0 || (w.scan && base_end >= most_units(w.mult));
    const int32_t all = none ? 0 : (base_end - base0) * w.mult;           // (a captured batch may use less than its capacity)
    w.zero = base0;
    w.size = (int32_t)(((uint32_t)all + blocks - 1u) / blocks);           // (the host keeps all + blocks below 2^31)
    w.lo = at_most(all, (int32_t)block * w.size);
    w.hi = w.lo + at_most(w.size, all - w.lo);
    w.whole = whole_of(w.size, lead);
}

// The item that holds unit `at`, and the part of it from there on that ends in this thread block.  a, b: base(r), base(r+1) of the
// request found for it; s.r and s.first are set.  Offsets that do not ascend make items that cannot be: false, with a segment of nothing
// (n < 0) up to the end of the share.  They may also make items that begin before the first unit or end behind the last one; their slices lie
// inside the lists all the same, and parts_of counts the thread blocks that there are.
UCMX_HOST_DEVICE bool place(Seg& s, const Share& w, int32_t a, int32_t b, int32_t tiles, int32_t heads, int32_t spe, int32_t total, int lead, int32_t at)
{
    const int32_t item = w.scan ? (b - a) / tiles : b - a;                // units of one (KV head, column tile)
    const int32_t start = (a - w.zero) * w.mult;
    s.n = (item - lead) / spe;
    if (item < lead || s.n > total - s.first || at < start || at - start >= item * (heads * tiles)) {
        s.begin = s.lo = at;
        s.end = s.hi = at_least(at + 1, w.hi);
        s.from = s.to = 0;
        s.h = s.ct = 0;
        s.n = -1;
        return false;
    }
    const int32_t i = (at - start) / item;
    s.h = i / tiles;
    s.ct = i - s.h * tiles;
    s.begin = start + i * item;
    s.end = s.begin + item;
    s.lo = at;
    s.hi = item <= w.whole || s.end < w.hi ? s.end : w.hi;
    s.from = at_least(0, at - s.begin - lead);
    s.to = s.hi - s.begin - lead;
    return true;
}

// Where the thread block's first segment `s` (at w.lo) begins for it: at the end of an item that the thread block before takes whole, or
// at the beginning of one whose first slice is here.  True: at the end, look there again.
UCMX_HOST_DEVICE bool passes_over(const Share& w, Seg& s, int32_t& begin, int lead)
{
    if (s.begin >= begin) return false;
    if (s.end - s.begin <= w.whole) {
        begin = s.end;
        return true;
    }
    if (begin <= s.begin + lead) begin = s.lo = s.begin;
    return false;
}

// Does the part that begins with the item belong to this thread block?  A split item's first part goes to the one that holds its
// first slice.
UCMX_HOST_DEVICE bool begins_here(const Share& w, const Seg& s, int lead) { return s.end - s.begin <= w.whole || s.begin + lead < w.hi; }

// Thread blocks that hold a part of an item which begins in thread block `block` and ends behind it; no more than follow.
UCMX_HOST_DEVICE int32_t parts_of(const Share& w, const Seg& s, int32_t block, int32_t blocks)
{
    return at_most((s.end - 1) / w.size - block + 1, blocks - block);
}

}  // namespace attend
}  // namespace ucmx
