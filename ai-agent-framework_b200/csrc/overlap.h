// Which arguments of the paged serving operators share memory: arithmetic on
// addresses and sizes, nothing is read.
#pragma once
#include <algorithm>
#include <string>

#include "paged.h"

namespace b2 {

// `rows` rows of `bytes` bytes, `stride` bytes apart.
struct Region {
    const char* name;
    const void* p;
    __int128 bytes;
    __int128 rows = 1, stride = 0;
};

// Whether one run of bytes (a.rows == 1) meets a row of b: the last row that
// starts before a's end reaches furthest of those that do.
inline bool regions_meet(const Region& a, const Region& b) {
    const __int128 from = (__int128)(uintptr_t)a.p - (uintptr_t)b.p, to = from + a.bytes;  // seen from b's start
    if (to <= 0 || a.bytes <= 0 || b.bytes <= 0) return false;
    const __int128 last = b.rows == 1 ? 0 : std::min(b.rows - 1, (to - 1) / b.stride);
    return last * b.stride + b.bytes > from;
}

// "<output> overlaps <input>" where an output of a page plan shares memory
// with what it reads: its CTAs read the lengths again after others have
// written.  Of the free list only the first entry's place is known here.
inline std::string page_plan_overlap(const PagePlanArgs& a) {
    const __int128 req = a.n_req, tok = a.max_tokens;
    const Region table{"table", a.table, (__int128)4 * a.max_pages, req, (__int128)4 * a.table_stride};
    const Region in[] = {{"cached", a.cached, 4 * req}, {"fresh", a.fresh, 4 * req}, {"free_pages", a.free_pages, 4},
                         {"n_free", a.n_free, 4}};
    const Region out[] = {{"lens", a.lens, 4 * req}, {"starts", a.starts, 4 * (req + 1)}, {"slots", a.slots, 8 * tok},
                          {"positions", a.positions, 4 * tok}, {"token_req", a.token_req, 4 * tok},
                          {"info", a.info, 16}};
    for (const Region& i : in) {
        if (regions_meet(i, table)) return std::string("table overlaps ") + i.name;
        for (const Region& o : out)
            if (regions_meet(i, o)) return std::string(o.name) + " overlaps " + i.name;
    }
    for (const Region& o : out)
        if (regions_meet(o, table)) return std::string(o.name) + " overlaps table";
    return "";
}

// Whether the places of a cache are apart: pages, positions and heads, and k
// and v, each taken with its distance, from the smallest distance up; every
// distance has to pass the extent of the ones before it.  (Distances that
// interleave without meeting in any other way are refused too.)
inline bool kv_places_apart(const b2_paged_kv& kv) {
    struct Dim {
        __int128 step, n;
    };
    const __int128 k = (uintptr_t)kv.k, v = (uintptr_t)kv.v;
    Dim d[] = {{(__int128)2 * kv.page_stride, kv.n_pages}, {(__int128)2 * kv.pos_stride, kv.page_size},
               {(__int128)2 * kv.head_stride, kv.nkv}, {k < v ? v - k : k - v, 2}};
    std::sort(d, d + 4, [](const Dim& a, const Dim& b) { return a.step < b.step; });
    __int128 extent = 2 * kv.hd;
    for (const Dim& x : d) {
        if (x.n == 1) continue;
        if (x.step < extent) return false;
        extent += (x.n - 1) * x.step;
    }
    return true;
}

}  // namespace b2
