// The pages of a cache among rows that share them: block tables forked, pages
// copied, holders counted, the pages in use moved to the front of the pool.
//
// All whole-number work, bound by latency for the tables and by HBM for the
// copies.  Where the order of what is taken matters (new pages, the free list,
// the moves of a compaction) places come from sums over what lies before, so
// the results do not depend on timing; the holders are counted by atomic adds
// of whole numbers, whose order does not show.
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

// pages of `len` positions
__device__ __forceinline__ int pages_of(int len, int page_size) { return len <= 0 ? 0 : (int)(((unsigned)len - 1) / (unsigned)page_size) + 1; }

// The sum over the threads before this one, and over all (THREADS of a CTA).
template <int THREADS>
__device__ __forceinline__ int sum_before(int x, int* warps, int* all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += t;
    }
    __syncthreads();  // (`warps` may still be read)
    if (lane == 31) warps[warp] = inc;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) before += warps[w];
        total += warps[w];
    }
    *all = total;
    return before + inc - x;
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------

constexpr int kForkThreads = 512;
constexpr int kWalk = 4;             // table entries of a lane in flight
constexpr int kPiece = 32 * kWalk;   // those of one warp's turn

// Every CTA works out for itself which rows take a page (the words are few and
// stay in L2), so one launch does all; then the rows' entries, in pieces, go
// round the warps of the grid.  Bound by latency, four dependent loads and the
// sums: 6 us for 4 rows as for 128.
__global__ void __launch_bounds__(kForkThreads) page_fork_kernel(const __grid_constant__ PageForkArgs a) {
    extern __shared__ int fork_sm[];
    int* first = fork_sm;            // [n_src] the first new row of each old one
    int* taken = fork_sm + a.n_src;  // [n_req] the row's page among those taken; -1: it takes none
    __shared__ int warps[kForkThreads / 32];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, R = a.n_req, P = a.page_size;
    const int n_free = max(0, *a.n_free);
    for (int i = tid; i < a.n_src; i += kForkThreads) first[i] = R;
    __syncthreads();
    int bad = 0;
    for (int r = tid; r < R; r += kForkThreads) {
        const int p = a.parent[r];
        if (p >= a.n_src) bad |= B2_FORK_BAD_PARENT;
        else if (p >= 0) atomicMin(&first[p], r);
    }
    __syncthreads();
    const long long most = (long long)a.max_pages * P;
    int total = 0;
    for (int r0 = 0; r0 < R; r0 += kForkThreads) {
        const int r = r0 + tid;
        const int p = r < R ? a.parent[r] : -1;
        int takes = 0;
        if (p >= 0 && p < a.n_src) {
            const int len = a.lens[p];
            if (len < 0) bad |= B2_PLAN_BAD_LENGTH;
            else if (len > most) bad |= B2_PLAN_TABLE_FULL;
            else if (len % P) {
                const int page = a.table[(int64_t)p * a.table_stride + len / P];
                const bool known = a.refs && page >= 0 && page < a.n_pages;
                takes = first[p] != r || (known && a.refs[page] > 1);
            }
        }
        int all;
        const int at = sum_before<kForkThreads>(takes, warps, &all);
        if (r < R) taken[r] = takes ? total + at : -1;
        total += all;
    }
    int status = __syncthreads_or(bad & B2_FORK_BAD_PARENT) ? B2_FORK_BAD_PARENT : 0;
    if (__syncthreads_or(bad & B2_PLAN_BAD_LENGTH)) status |= B2_PLAN_BAD_LENGTH;
    if (__syncthreads_or(bad & B2_PLAN_TABLE_FULL)) status |= B2_PLAN_TABLE_FULL;
    if (total > n_free) status |= B2_PLAN_NO_PAGES;
    if (blockIdx.x == 0 && tid == 0) {
        a.info[0] = status;
        a.info[1] = status ? 0 : total;
        a.info[2] = a.info[3] = 0;
    }
    if (status) return;
    const int warp0 = (blockIdx.x * kForkThreads + tid) / 32, n_warps = gridDim.x * kForkThreads / 32;
    const int pieces = (a.max_pages - 1) / kPiece + 1;
    const long long items = (long long)R * pieces;
    for (long long it = warp0; it < items; it += n_warps) {
        const int c = (int)(it / R), r = (int)(it - (long long)c * R);
        const int p = a.parent[r], len = p >= 0 ? a.lens[p] : 0, n = pages_of(len, P);
        if (c == 0 && lane == 0) a.new_lens[r] = len;
        const int e0 = c * kPiece + lane;
        if (c * kPiece >= n) continue;
        const int32_t* src = a.table + (int64_t)p * a.table_stride;
        int32_t* dst = a.new_table + (int64_t)r * a.new_stride;
        const int swap = taken[r] >= 0 ? len / P : -1;
        int page[kWalk];
#pragma unroll
        for (int j = 0; j < kWalk; j++)
            if (e0 + 32 * j < n) page[j] = src[e0 + 32 * j];
#pragma unroll
        for (int j = 0; j < kWalk; j++) {
            const int e = e0 + 32 * j;
            if (e == swap) {
                const int t = taken[r], copy = a.free_pages[t];
                a.pairs[3 * t] = page[j];
                a.pairs[3 * t + 1] = copy;
                a.pairs[3 * t + 2] = len % P;
                page[j] = copy;
            }
            if (e < n) dst[e] = page[j];
        }
    }
}

// ---------------------------------------------------------------------------
// copy
// ---------------------------------------------------------------------------

struct PageCopyArgs {
    uint16_t *k, *v;
    const int32_t *pairs, *n_pairs;
    int64_t page_stride, pos_stride, head_stride, layer_stride;
    int n_pages, page_size, nkv, hc, layers, max_pairs;  // hc: 16-byte chunks of a head
    int dense;                                           // a position's heads, and positions, lie back to back
};

constexpr int kCopyThreads = 128;

// One CTA's turn: 16-byte chunks of one page's k or v in one layer, LOADS to a
// thread: 8, or 4 where a page is no more than 8 KB.  Bound by HBM: 1.17 GB read and
// written for pages of 32 KB take 186 us, 6.3 TB/s (4 loads: 189), 130 MB of half
// pages 25 us (27), 57 MB of pages of 4 KB 11.8 us (8 loads: 14.8).
template <int LOADS>
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const __grid_constant__ PageCopyArgs a) {
    pdl_trigger();
    pdl_wait();
    const int n = max(0, min(*a.n_pairs, a.max_pairs));
    constexpr int kCopyChunks = kCopyThreads * LOADS;
    const int per_pos = a.nkv * a.hc;
    const int turns = (int)(((int64_t)a.page_size * per_pos + kCopyChunks - 1) / kCopyChunks);
    const unsigned planes = 2u * (unsigned)a.layers;
    const int64_t items = (int64_t)n * planes * turns;
    const bool narrow = items <= 0x7fffffff;  // divisions of 32 bits where they do
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        int turn, pair;
        unsigned which;
        if (narrow) {
            const unsigned i = (unsigned)it, rest = i / (unsigned)turns;
            turn = (int)(i - rest * turns);
            pair = (int)(rest / planes);
            which = rest - (unsigned)pair * planes;
        } else {
            const int64_t rest = it / turns;
            turn = (int)(it - rest * turns);
            pair = (int)(rest / planes);
            which = (unsigned)(rest - (int64_t)pair * planes);
        }
        const int src = a.pairs[3 * (int64_t)pair], dst = a.pairs[3 * (int64_t)pair + 1];
        const int count = min(a.pairs[3 * (int64_t)pair + 2], a.page_size);
        if (src == dst || (unsigned)src >= (unsigned)a.n_pages || (unsigned)dst >= (unsigned)a.n_pages) continue;
        const int64_t chunks = (int64_t)max(count, 0) * per_pos;
        if ((int64_t)turn * kCopyChunks >= chunks) continue;
        uint16_t* base = (which & 1 ? a.v : a.k) + (int64_t)(which >> 1) * a.layer_stride;
        const uint16_t* from = base + src * a.page_stride;
        uint16_t* to = base + dst * a.page_stride;
        uint4 v[LOADS];
        int64_t off[LOADS];
#pragma unroll
        for (int j = 0; j < LOADS; j++) {
            const int64_t i = (int64_t)turn * kCopyChunks + j * kCopyThreads + threadIdx.x;
            off[j] = -1;
            if (i < chunks) {
                if (a.dense) {
                    off[j] = 8 * i;
                } else {
                    const int pos = (int)(i / per_pos), in = (int)(i - (int64_t)pos * per_pos), h = in / a.hc;
                    off[j] = pos * a.pos_stride + h * a.head_stride + (in - h * a.hc) * 8;
                }
                v[j] = *reinterpret_cast<const uint4*>(from + off[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < LOADS; j++)
            if (off[j] >= 0) *reinterpret_cast<uint4*>(to + off[j]) = v[j];
    }
}

// ---------------------------------------------------------------------------
// holders, free list
// ---------------------------------------------------------------------------

// f(page, its place) for the table entries that the lengths hold, a piece of a
// row at a time, by the warps from `warp` on in steps of `n_warps`.
template <typename A, typename F>
__device__ __forceinline__ void walk_table(const A& a, int warp, int n_warps, F f) {
    const int lane = threadIdx.x & 31, pieces = (a.max_pages - 1) / kPiece + 1;
    const long long items = (long long)a.n_req * pieces;
    for (long long it = warp; it < items; it += n_warps) {
        const int c = (int)(it / a.n_req), r = (int)(it - (long long)c * a.n_req);
        const int n = min(pages_of(a.lens[r], a.page_size), a.max_pages);
        auto* row = a.table + (int64_t)r * a.table_stride;
        int page[kWalk];
#pragma unroll
        for (int j = 0; j < kWalk; j++) {
            const int e = c * kPiece + 32 * j + lane;
            page[j] = e < n ? row[e] : -1;
        }
#pragma unroll
        for (int j = 0; j < kWalk; j++)
            if (page[j] >= 0) f(page[j], row + c * kPiece + 32 * j + lane);
    }
}

constexpr int kPoolThreads = 512;
constexpr int kPoolBlock = 4 * kPoolThreads;  // pages of one CTA

struct PoolArgs {
    const int32_t *table, *lens;
    int64_t table_stride;
    int32_t *refs, *free_pages, *n_free, *counts;
    int n_req, page_size, max_pages, n_pages;
};

__global__ void __launch_bounds__(kPoolThreads) pool_zero_kernel(const __grid_constant__ PoolArgs a) {
    pdl_trigger();
    pdl_wait();
    for (unsigned i = blockIdx.x * kPoolThreads + threadIdx.x; i < (unsigned)a.n_pages; i += gridDim.x * kPoolThreads) a.refs[i] = 0;
}

__global__ void __launch_bounds__(kPoolThreads) pool_count_kernel(const __grid_constant__ PoolArgs a) {
    pdl_trigger();
    pdl_wait();
    const int warp0 = (blockIdx.x * kPoolThreads + threadIdx.x) / 32, n_warps = gridDim.x * kPoolThreads / 32;
    walk_table(a, warp0, n_warps, [&](int page, const int32_t*) {
        if (page < a.n_pages) atomicAdd(&a.refs[page], 1);
    });
}

// The four launches in one, by a CTA that keeps the counts in its shared memory.
constexpr int kSmallThreads = 1024;
constexpr int kSmallPages = 4096;
constexpr int kSmallEntries = 4096;

__global__ void __launch_bounds__(kSmallThreads) pool_small_kernel(const __grid_constant__ PoolArgs a) {
    __shared__ int count[kSmallPages], warps[kSmallThreads / 32];
    pdl_trigger();
    const int tid = threadIdx.x, per = (a.n_pages + kSmallThreads - 1) / kSmallThreads;
    for (int i = tid; i < a.n_pages; i += kSmallThreads) count[i] = 0;
    pdl_wait();
    __syncthreads();
    walk_table(a, tid / 32, kSmallThreads / 32, [&](int page, const int32_t*) {
        if (page < a.n_pages) atomicAdd(&count[page], 1);
    });
    __syncthreads();
    for (int i = tid; i < a.n_pages; i += kSmallThreads) a.refs[i] = count[i];
    const int i0 = tid * per, i1 = min(a.n_pages, i0 + per);
    int n = 0, all;
    for (int i = i0; i < i1; i++) n += count[i] == 0;
    int at = sum_before<kSmallThreads>(n, warps, &all);
    for (int i = i0; i < i1; i++)
        if (count[i] == 0) a.free_pages[at++] = i;
    if (tid == 0) *a.n_free = all;
}

// how many pages of each block are free
__global__ void __launch_bounds__(kPoolThreads) pool_blocks_kernel(const int32_t* refs, int n_pages, int32_t* counts) {
    __shared__ int warps[kPoolThreads / 32];
    pdl_trigger();
    pdl_wait();
    int n = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const unsigned p = blockIdx.x * kPoolBlock + 4 * threadIdx.x + j;  // (the last block may pass 2^31)
        n += p < (unsigned)n_pages && refs[p] == 0;
    }
    int all;
    sum_before<kPoolThreads>(n, warps, &all);
    if (threadIdx.x == 0) counts[blockIdx.x] = all;
}

// the free pages of the blocks before this one, and of all
__device__ __forceinline__ int free_before(const int32_t* counts, int* warps, int* total) {
    int mine = 0, all = 0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += kPoolThreads) {
        all += counts[i];
        if (i < (int)blockIdx.x) mine += counts[i];
    }
    int before;
    sum_before<kPoolThreads>(mine, warps, &before);
    sum_before<kPoolThreads>(all, warps, total);
    return before;
}

__global__ void __launch_bounds__(kPoolThreads) pool_list_kernel(const __grid_constant__ PoolArgs a) {
    __shared__ int warps[kPoolThreads / 32];
    pdl_trigger();
    pdl_wait();
    int total;
    const int before = free_before(a.counts, warps, &total);
    const unsigned p0 = blockIdx.x * kPoolBlock + 4 * threadIdx.x, N = a.n_pages;
    int n = 0;
    bool free_[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        free_[j] = p0 + j < N && a.refs[p0 + j] == 0;
        n += free_[j];
    }
    int all;
    int at = before + sum_before<kPoolThreads>(n, warps, &all);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (free_[j]) a.free_pages[at++] = (int)(p0 + j);
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_free = total;
}

// ---------------------------------------------------------------------------
// compaction
// ---------------------------------------------------------------------------

struct CompactArgs {
    int32_t* table;
    const int32_t *lens, *refs;
    int64_t table_stride;
    int32_t *pairs, *info, *counts, *moves, *holes, *movers, *rank;
    int n_req, page_size, max_pages, n_pages, max_pairs;
};

// holes[i]: the i-th lowest free page below U; movers[i]: the i-th highest
// page in use at U or above, rank[movers[i]] = i.  Page p, with `before` free
// pages before it, into them; the free pages up to it.
__device__ __forceinline__ int place(const CompactArgs& a, int p, bool free_, int U, int before) {
    if (free_) {
        if (p < U) a.holes[before] = p;
        before++;
    } else if (p >= U) {
        const int i = U - 1 - (p - before);  // pages in use above p
        a.movers[i] = p;
        a.rank[p] = i;
    }
    if (p == U - 1) *a.moves = before;  // the holes below U
    return before;
}

__global__ void __launch_bounds__(kPoolThreads) compact_rank_kernel(const __grid_constant__ CompactArgs a) {
    __shared__ int warps[kPoolThreads / 32];
    pdl_trigger();
    pdl_wait();
    int n_free;
    int before = free_before(a.counts, warps, &n_free);
    const int U = a.n_pages - n_free;
    const unsigned p0 = blockIdx.x * kPoolBlock + 4 * threadIdx.x, N = a.n_pages;
    int n = 0;
    bool free_[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        free_[j] = p0 + j < N && a.refs[p0 + j] == 0;
        n += free_[j];
    }
    int all;
    before += sum_before<kPoolThreads>(n, warps, &all);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (p0 + j < N) before = place(a, (int)(p0 + j), free_[j], U, before);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.info[2] = U;
        if (U == 0) *a.moves = 0;
    }
}

// A table entry that is in use, given its new page if it has one.
__device__ __forceinline__ void moved(const CompactArgs& a, int page, int32_t* at, int U, int done) {
    if (page < U || page >= a.n_pages) return;
    const int refs = a.refs[page], i = __ldcg(a.rank + page);
    if (refs > 0 && i < done) *at = __ldcg(a.holes + i);
}

// The moves, and the table entries that they change, by n_threads threads.
__device__ __forceinline__ void apply(const CompactArgs& a, int tid, int n_threads, int U) {
    const int moves = __ldcg(a.moves), done = min(moves, a.max_pairs);
    for (int i = tid; i < done; i += n_threads) {
        a.pairs[3 * (int64_t)i] = __ldcg(a.movers + i);
        a.pairs[3 * (int64_t)i + 1] = __ldcg(a.holes + i);
        a.pairs[3 * (int64_t)i + 2] = a.page_size;
    }
    if (tid == 0) {
        a.info[0] = 0;
        a.info[1] = done;
        a.info[3] = done < moves ? __ldcg(a.movers + done) + 1 : U;
    }
    walk_table(a, tid / 32, n_threads / 32, [&](int page, int32_t* at) { moved(a, page, at, U, done); });
}

__global__ void __launch_bounds__(kPoolThreads) compact_apply_kernel(const __grid_constant__ CompactArgs a) {
    pdl_trigger();
    pdl_wait();
    apply(a, blockIdx.x * kPoolThreads + threadIdx.x, gridDim.x * kPoolThreads, a.info[2]);
}

int pool_blocks(int n_pages) { return (n_pages - 1) / kPoolBlock + 1; }
size_t words16(size_t n) { return (n + 3) & ~(size_t)3; }

// CTAs for the rows' entries: a warp for every kPiece of them
int entry_ctas(int n_req, int max_pages, int threads, int sms) {
    const long long items = (long long)n_req * ((max_pages - 1) / kPiece + 1);
    return (int)std::max<long long>(1, std::min<long long>(2048 / threads * sms, (items + threads / 32 - 1) / (threads / 32)));
}

}  // namespace

int launch_page_fork(const PageForkArgs& a, cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const size_t smem = sizeof(int) * ((size_t)a.n_src + a.n_req);
    cudaError_t e = cudaSuccess;
    if (smem > 47 * 1024)
        e = cudaFuncSetAttribute(page_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * sizeof(int) * kPlanMaxReq));
    if (e == cudaSuccess)
        e = launch_pdl(page_fork_kernel, dim3(std::min(entry_ctas(a.n_req, a.max_pages, kForkThreads, sms), sms)),
                       dim3(kForkThreads), smem, s, a);
    return e == cudaSuccess ? B2_OK : cuda_failed("page fork launch", e, err);
}

int launch_page_copy(const b2_paged_kv& kv, int layers, int64_t layer_stride, const int32_t* pairs, const int32_t* n_pairs,
                     int max_pairs, cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    PageCopyArgs a{};
    a.k = static_cast<uint16_t*>(kv.k);
    a.v = static_cast<uint16_t*>(kv.v);
    a.pairs = pairs;
    a.n_pairs = n_pairs;
    a.page_stride = kv.page_stride;
    a.pos_stride = kv.pos_stride;
    a.head_stride = kv.head_stride;
    a.layer_stride = layer_stride;
    a.n_pages = kv.n_pages;
    a.page_size = kv.page_size;
    a.nkv = kv.nkv;
    a.hc = kv.hd / 8;
    a.layers = layers;
    a.max_pairs = max_pairs;
    a.dense = kv.head_stride == kv.hd && kv.pos_stride == (int64_t)kv.nkv * kv.hd;
    const int64_t chunks = (int64_t)a.page_size * a.nkv * a.hc;
    const int loads = chunks <= 4 * kCopyThreads ? 4 : 8;
    const int64_t turns = (chunks + kCopyThreads * loads - 1) / (kCopyThreads * loads);
    const __int128 items = (__int128)max_pairs * 2 * layers * turns;
    const cudaError_t e = launch_pdl(loads == 4 ? page_copy_kernel<4> : page_copy_kernel<8>,
                                     dim3((unsigned)std::min<__int128>(items, 16 * sms)), dim3(kCopyThreads), 0, s, a);
    return e == cudaSuccess ? B2_OK : cuda_failed("page copy launch", e, err);
}

size_t page_pool_scratch(int n_pages) { return 4 * words16(pool_blocks(n_pages)); }

int launch_page_pool(const int32_t* table, int64_t table_stride, const int32_t* lens, int n_req, int page_size,
                     int max_pages, int32_t* refs, int n_pages, int32_t* free_pages, int32_t* n_free, void* scratch,
                     cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const PoolArgs a{table, lens, table_stride, refs, free_pages, n_free, static_cast<int32_t*>(scratch),
                     n_req, page_size, max_pages, n_pages};
    // (256 pages, 128 entries: 4.2 us, by four launches 6.2; 4096 pages, 4096 entries: 6.2 and 8.3; 8192 pages of
    // as many entries: 10.3 and 8.3)
    if (n_pages <= kSmallPages && (int64_t)n_req * max_pages <= kSmallEntries) {
        const cudaError_t e = launch_pdl(pool_small_kernel, dim3(1), dim3(kSmallThreads), 0, s, a);
        return e == cudaSuccess ? B2_OK : cuda_failed("page pool launch", e, err);
    }
    const int blocks = pool_blocks(n_pages);
    cudaError_t e = launch_pdl(pool_zero_kernel, dim3(std::min(4 * sms, (n_pages - 1) / kPoolThreads + 1)),
                               dim3(kPoolThreads), 0, s, a);
    if (e == cudaSuccess)
        e = launch_pdl(pool_count_kernel, dim3(entry_ctas(n_req, max_pages, kPoolThreads, sms)), dim3(kPoolThreads), 0, s, a);
    if (e == cudaSuccess)
        e = launch_pdl(pool_blocks_kernel, dim3(blocks), dim3(kPoolThreads), 0, s, (const int32_t*)refs, n_pages, a.counts);
    if (e == cudaSuccess) e = launch_pdl(pool_list_kernel, dim3(blocks), dim3(kPoolThreads), 0, s, a);
    return e == cudaSuccess ? B2_OK : cuda_failed("page pool launch", e, err);
}

size_t page_compact_scratch(int n_pages) { return 4 * (words16(pool_blocks(n_pages)) + 3 * words16(n_pages) + 4); }

int launch_page_compact(int32_t* table, int64_t table_stride, const int32_t* lens, int n_req, int page_size,
                        int max_pages, const int32_t* refs, int n_pages, int32_t* pairs, int max_pairs, int32_t* info,
                        void* scratch, cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const int blocks = pool_blocks(n_pages);
    CompactArgs a{};
    a.table = table;
    a.lens = lens;
    a.refs = refs;
    a.table_stride = table_stride;
    a.pairs = pairs;
    a.info = info;
    a.counts = static_cast<int32_t*>(scratch);
    a.holes = a.counts + words16(blocks);
    a.movers = a.holes + words16(n_pages);
    a.rank = a.movers + words16(n_pages);
    a.moves = a.rank + words16(n_pages);
    a.n_req = n_req;
    a.page_size = page_size;
    a.max_pages = max_pages;
    a.n_pages = n_pages;
    a.max_pairs = max_pairs;
    cudaError_t e = launch_pdl(pool_blocks_kernel, dim3(blocks), dim3(kPoolThreads), 0, s, refs, n_pages, a.counts);
    if (e == cudaSuccess) e = launch_pdl(compact_rank_kernel, dim3(blocks), dim3(kPoolThreads), 0, s, a);
    if (e == cudaSuccess)
        e = launch_pdl(compact_apply_kernel, dim3(entry_ctas(n_req, max_pages, kPoolThreads, sms)), dim3(kPoolThreads), 0, s, a);
    return e == cudaSuccess ? B2_OK : cuda_failed("page compaction launch", e, err);
}

}  // namespace b2
