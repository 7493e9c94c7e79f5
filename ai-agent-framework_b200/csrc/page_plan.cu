// Block tables and slot maps of a paged serving step, built from the
// requests' lengths on the device.
//
// Request r holds cached[r] positions in ceil(cached / P) pages and gets
// fresh[r] more tokens.  With the exclusive sums
//   start[r] = sum_{i<r} fresh[i],
//   taken[r] = sum_{i<r} (ceil((cached[i] + fresh[i]) / P) - ceil(cached[i] / P)),
// new page e of the step is free_pages[e] and goes to the request with
// taken[r] <= e < taken[r + 1], and token t (start[r] <= t < start[r + 1]) has
// position p = cached[r] + t - start[r] and slot table[r][p / P] * P + p % P.
//
// Every CTA computes both sums over all requests for itself: the lengths are
// 8 bytes a request and stay in L2, so one launch with no word between CTAs
// replaces a scan kernel, an expand kernel and their hand-off.  Whether the
// step fits (pages, table width, token rows) is known to every CTA before it
// writes, so a step that does not fit changes nothing in the table.
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

__device__ __forceinline__ int pages_of(int len, int P) { return len / P + (len % P != 0); }

// The last index r of a[0 .. n] (ascending, a[0] = 0) with a[r] <= x.
__device__ __forceinline__ int last_le(const int* a, int n, int x) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const __grid_constant__ PagePlanArgs a) {
    extern __shared__ int plan_sm[];
    int* start = plan_sm;                // [n_req + 1]
    int* taken = plan_sm + a.n_req + 1;  // [n_req + 1]
    __shared__ long long wsum[2][kPlanWarps];
    __shared__ int wbad[kPlanWarps];
    pdl_trigger();
    pdl_wait();
    const int R = a.n_req, P = a.page_size, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(R, tid * per), r1 = min(R, r0 + per);

    // this thread's requests: their tokens and pages (64-bit: the sums of bad lengths must not wrap)
    long long tok = 0, pg = 0;
    int bad = 0;
    for (int r = r0; r < r1; r++) {
        const int c = a.cached[r], f = a.fresh[r];
        if (c < 0 || f < 0) {
            bad |= B2_PLAN_BAD_LENGTH;
            continue;
        }
        const long long len = (long long)c + f;
        if (len > 0x7fffffffLL || (len + P - 1) / P > a.max_pages) {
            bad |= B2_PLAN_TABLE_FULL;
            continue;
        }
        tok += f;
        pg += pages_of((int)len, P) - pages_of(c, P);
    }
    long long it = tok, ip = pg;  // inclusive over the warp, then over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, it, o), p = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) {
            it += t;
            ip += p;
        }
    }
    if (lane == 31) {
        wsum[0][warp] = it;
        wsum[1][warp] = ip;
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    if (lane == 0) wbad[warp] = bad;
    __syncthreads();
    int status = 0;
    long long total_tok = 0, total_pg = 0;
#pragma unroll
    for (int w = 0; w < kPlanWarps; w++) {
        if (w == warp) {
            it += total_tok;
            ip += total_pg;
        }
        total_tok += wsum[0][w];
        total_pg += wsum[1][w];
        status |= wbad[w];
    }
    if (total_tok > a.max_tokens) status |= B2_PLAN_ROWS_FULL;
    if (total_pg > max(0, *a.n_free)) status |= B2_PLAN_NO_PAGES;
    const bool ok = status == 0;
    const int T = ok ? (int)total_tok : 0, N = ok ? (int)total_pg : 0;
    if (ok) {
        int t = (int)(it - tok), p = (int)(ip - pg);
        for (int r = r0; r < r1; r++) {
            start[r] = t;
            taken[r] = p;
            const int c = a.cached[r], f = a.fresh[r];
            t += f;
            p += pages_of(c + f, P) - pages_of(c, P);
        }
        if (tid == 0) {
            start[R] = T;
            taken[R] = N;
        }
    }
    __syncthreads();

    const int gtid = blockIdx.x * kPlanThreads + tid, gsize = gridDim.x * kPlanThreads;
    if (gtid == 0) {
        a.info[0] = status;
        a.info[1] = T;
        a.info[2] = N;
        a.info[3] = 0;
    }
    for (int r = gtid; r <= R; r += gsize) {
        a.starts[r] = ok ? start[r] : 0;
        if (r < R) a.lens[r] = ok ? a.cached[r] + a.fresh[r] : a.cached[r];
    }
    for (int e = gtid; e < N; e += gsize) {
        const int r = last_le(taken, R, e);
        a.table[(int64_t)r * a.table_stride + pages_of(a.cached[r], P) + (e - taken[r])] = a.free_pages[e];
    }
    for (int t = gtid; t < a.max_tokens; t += gsize) {
        int64_t slot = -1;
        int pos = 0, req = -1;
        if (t < T) {
            req = last_le(start, R, t);
            const int c = a.cached[req], have = pages_of(c, P);
            pos = c + (t - start[req]);
            const int idx = pos / P;
            // (a page of this step comes from the list: its table entry may be another CTA's to write)
            const int page = idx < have ? a.table[(int64_t)req * a.table_stride + idx] : a.free_pages[taken[req] + idx - have];
            if (page >= 0) slot = (int64_t)page * P + pos % P;
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
        a.token_req[t] = req;
    }
}

}  // namespace

int launch_page_plan(const PagePlanArgs& a, cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const int smem = (int)(2 * sizeof(int) * ((size_t)a.n_req + 1));
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(page_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(2 * sizeof(int) * (kPlanMaxReq + 1))) != cudaSuccess) {
        *err = "page plan: shared memory attribute";
        return B2_ERR_CUDA;
    }
    const long long work = std::max<long long>(a.max_tokens, a.n_req);
    const int grid = (int)std::max<long long>(1, std::min<long long>(2 * sms, (work + kPlanThreads - 1) / kPlanThreads));
    const cudaError_t e = launch_pdl(page_plan_kernel, dim3(grid), dim3(kPlanThreads), smem, s, a);
    if (e != cudaSuccess) {
        *err = std::string("page plan launch: ") + cudaGetErrorString(e);
        return B2_ERR_CUDA;
    }
    return B2_OK;
}

}  // namespace b2
