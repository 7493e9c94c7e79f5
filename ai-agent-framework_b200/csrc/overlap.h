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

// Whether a row of a meets a row of b.  Rows of one distance are taken modulo
// it (the halves of a pair of tables laid row beside row are apart); rows of
// different distances meet where their extents do.
inline bool rows_meet(const Region& a, const Region& b) {
    if (a.rows == 1) return regions_meet(a, b);
    if (b.rows == 1) return regions_meet(b, a);
    if (a.bytes <= 0 || b.bytes <= 0) return false;
    const __int128 pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    const __int128 ea = pa + (a.rows - 1) * a.stride + a.bytes, eb = pb + (b.rows - 1) * b.stride + b.bytes;
    if (ea <= pb || eb <= pa) return false;
    if (a.stride != b.stride) return true;
    const __int128 off = ((pb - pa) % a.stride + a.stride) % a.stride;  // b's rows behind the start of a's
    return off < a.bytes || off + b.bytes > a.stride;
}

// "<output> overlaps <input>" where an output meets an input or another output.
inline std::string outputs_overlap(const Region* in, int n_in, const Region* out, int n_out) {
    for (int i = 0; i < n_out; i++) {
        if (!out[i].p) continue;
        for (int j = 0; j < n_in; j++)
            if (in[j].p && rows_meet(out[i], in[j])) return std::string(out[i].name) + " overlaps " + in[j].name;
        for (int j = 0; j < i; j++)
            if (out[j].p && rows_meet(out[i], out[j])) return std::string(out[i].name) + " overlaps " + out[j].name;
    }
    return "";
}

// Whether the places of a cache (of `layers` layers) are apart: pages,
// positions, heads and layers, and k and v, each taken with its distance, from
// the smallest distance up; every distance has to pass the extent of the ones
// before it.  (Distances that interleave without meeting in any other way are
// refused too.)
inline bool kv_places_apart(const b2_paged_kv& kv, int layers = 1, int64_t layer_stride = 0) {
    struct Dim {
        __int128 step, n;
    };
    const __int128 k = (uintptr_t)kv.k, v = (uintptr_t)kv.v;
    Dim d[] = {{(__int128)2 * kv.page_stride, kv.n_pages}, {(__int128)2 * kv.pos_stride, kv.page_size},
               {(__int128)2 * kv.head_stride, kv.nkv}, {k < v ? v - k : k - v, 2}, {(__int128)2 * layer_stride, layers}};
    std::sort(d, d + 5, [](const Dim& a, const Dim& b) { return a.step < b.step; });
    __int128 extent = 2 * kv.hd;
    for (const Dim& x : d) {
        if (x.n == 1) continue;
        if (x.step < extent) return false;
        extent += (x.n - 1) * x.step;
    }
    return true;
}

// Rows that lie back to back are one run.
inline Region rows_of(const char* name, const void* p, __int128 bytes, __int128 rows, __int128 stride) {
    if (stride == bytes) return {name, p, bytes * rows};
    return {name, p, bytes, rows, stride};
}

// The pages of a cache's k or v, each with all that lies between its first and
// last element.
inline Region pages_of_cache(const char* name, const b2_paged_kv& kv, const void* p) {
    const __int128 page = 2 * ((__int128)(kv.page_size - 1) * kv.pos_stride + (__int128)(kv.nkv - 1) * kv.head_stride + kv.hd);
    return rows_of(name, p, page, kv.n_pages, (__int128)2 * kv.page_stride);
}

// "<output> overlaps <input>" where what an attention over shared prefixes
// writes shares memory with what it reads.
inline std::string attention_shared_overlap(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q,
                                            const int32_t* table, const int32_t* lens, const int32_t* req, int batch,
                                            const int32_t* starts, const int32_t* prefix, int n_groups, const void* out,
                                            const float* lse, const void* scratch, size_t scratch_bytes) {
    const __int128 es = o.dtype == 0 ? 4 : 2, row = es * o.nh * kv.hd, rows = batch;
    const Region in[] = {rows_of("q", q, row, rows, o.q_stride ? es * o.q_stride : row),
                         pages_of_cache("the cache's k", kv, kv.k), pages_of_cache("the cache's v", kv, kv.v),
                         rows_of("table", table, (__int128)4 * o.max_pages, o.n_req,
                                 (__int128)4 * (o.table_stride ? o.table_stride : o.max_pages)),
                         {"lens", lens, 4 * rows}, {"req", req, 4 * rows}, {"starts", starts, (__int128)4 * n_groups + 4},
                         {"prefix", prefix, (__int128)4 * n_groups}, {"slopes", o.slopes, (__int128)4 * o.nh}};
    const Region to[] = {rows_of("out", out, row, rows, o.out_stride ? es * o.out_stride : row),
                         {"lse", lse, 4 * rows * o.nh}, {"scratch", scratch, (__int128)scratch_bytes}};
    return outputs_overlap(in, 9, to, 3);
}

}  // namespace b2
