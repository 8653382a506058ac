// The attention kernel's cut of its work (csrc/split.cuh), thread block by thread block, without a GPU.
#include <cstdint>
#include <vector>

#include "split.cuh"

using namespace ucmx::attend;

namespace {

struct Lists {
    const int32_t* offsets;
    int32_t n_req, total, spe, heads, lead;
    const int32_t* tiles;              // of each request, or NULL: col_tiles for all
    int32_t col_tiles;
    std::vector<int32_t> scan;
    int32_t base(int32_t r) const { return tiles ? scan[r] : inside(offsets[r], total) * spe + r * lead; }
};

// the search as a warp does it: 32 values at a time, the first of them read ahead
int request_of(const Lists& l, const Share& w, int32_t e, int32_t& first, int32_t& next)
{
    int lo = 0, n = l.n_req, step = w.step;
    int32_t v[32];
    for (int i = 0; i < 32; ++i) v[i] = w.probes[i];
    for (;;) {
        int c = 0;
        for (int i = 0; i < 32; ++i) c += i * step < n && v[i] <= e;
        const int adv = (c > 0 ? c - 1 : 0) * step;
        if (step == 1) {
            first = v[c > 0 ? c - 1 : 0];
            next = v[c > 0 ? c : 1];
            return lo + adv;
        }
        lo += adv;
        n = n - adv < step ? n - adv : step;
        step = (n + 30) / 31;
        for (int i = 0; i < 32; ++i) v[i] = l.base(lo + (i * step < n ? i * step : n));
    }
}

}  // namespace

// Rows of `out`: block, request, head, tile, from, to, first entry, entries, 1 if the part begins the item, parts (0: not split).
// Returns their number, or -1 where a loop does not end or `room` is short; *rejected: pieces that were passed over.
extern "C" int64_t replay(const int32_t* offsets, int32_t n_req, int32_t total, int32_t spe, int32_t heads, const int32_t* tiles, int32_t col_tiles,
                          int32_t lead, int32_t blocks, int64_t* out, int64_t room, int64_t* rejected, int32_t* reported)
{
    if (too_many_units((int64_t)total * spe + (int64_t)n_req * kLeadMost, heads, col_tiles)) return -2;      // (the host refuses it)
    Lists l{offsets, n_req, total, spe, heads, lead, tiles, col_tiles, {}};
    *reported = 0;
    for (int r = 0; r < n_req; ++r) *reported |= bad_offsets(offsets[r], offsets[r + 1], total);
    if (tiles) {
        int32_t sum = 0;
        for (int r = 0; r < n_req; ++r) {
            l.scan.push_back(sum);
            const int32_t units = (inside(offsets[r + 1], total) - inside(offsets[r], total)) * spe + lead;
            sum = add_units(sum, at_least(lead, units) * tiles[r], most_units(heads));
        }
        l.scan.push_back(sum);
    }
    *rejected = 0;
    int64_t n = 0;
    for (int block = 0; block < blocks; ++block) {
        Share w{};
        int32_t probes[32];
        w.scan = tiles ? l.scan.data() : nullptr;
        w.tiles = col_tiles;
        w.mult = tiles ? heads : heads * col_tiles;
        w.step = (n_req + 30) / 31;
        for (int i = 0; i < 32; ++i) probes[i] = l.base(i * w.step < n_req ? i * w.step : n_req);
        w.probes = probes;
        share_out(w, probes[0], probes[31], block, blocks, lead);
        auto segment_at = [&](int32_t at) {
            Seg s{};
            int32_t a = 0, b = 0;
            s.r = request_of(l, w, at / w.mult + w.zero, a, b);
            s.first = tiles ? inside(offsets[s.r], total) : (a - s.r * lead) / spe;
            if (!place(s, w, a, b, tiles ? at_least(1, tiles[s.r]) : col_tiles, heads, spe, total, lead, at)) ++*rejected;
            return s;
        };
        int32_t begin = w.lo;
        Seg head{};
        if (begin < w.hi) {
            head = segment_at(begin);
            if (passes_over(w, head, begin, lead) && begin < w.hi) head = segment_at(begin);
        }
        int64_t turns = 0;
        for (int32_t at = begin; at < w.hi;) {
            const Seg s = at == begin ? head : segment_at(at);
            if (!begins_here(w, s, lead)) break;
            at = s.hi;
            if (n == room || ++turns > (int64_t)room) return -1;
            if (s.n < 0) continue;
            const bool split = s.lo == s.begin && s.hi < s.end;
            const int64_t row[10] = {block, s.r, s.h, s.ct, s.from, s.to, s.first, s.n, s.lo == s.begin, split ? parts_of(w, s, block, blocks) : 0};
            for (int i = 0; i < 10; ++i) out[n * 10 + i] = row[i];
            ++n;
        }
    }
    return n;
}

extern "C" int32_t row_holds(int32_t t0, int32_t t1, int32_t size, int32_t at) { return in_row(t0, t1, size, at); }
