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
//
// Bound by latency: 3.1 us for 16 tokens (a launch, the lengths, a search, a
// page), 10.0 us for a million tokens of 2048 requests, of which the 17 MB
// written need 2.7 (the issue slots of the scan, the searches and the table's
// entries, one after another).
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

// Tokens of one lane, 32 apart, so that a warp's stores are whole lines: eight
// where there are enough to fill the machine (a million tokens: 10 us, 32 with
// one), one for a decode step (16 tokens: 3.1 us, 5.5 with four, one after
// another's search).
constexpr int kManyTokens = 8;

constexpr unsigned kSumMax = 0x7fffffffu;
// sums that stop at kSumMax (which no valid step reaches)
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, kSumMax); }

// n / P for 0 <= n < 2^31 (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994): with s = ceil(log2 P) and mul =
// floor(2^32 (2^s - P) / P) + 1, n / P = (mulhi(mul, n) + n) >> s.
__device__ __forceinline__ int div_page(const PagePlanArgs& a, int n) {
    return (int)((__umulhi(a.page_mul, (unsigned)n) + (unsigned)n) >> a.page_shift);
}
__device__ __forceinline__ int pages_of(const PagePlanArgs& a, int len) {
    const int q = div_page(a, len);
    return q + (q * a.page_size != len);
}

// The last index r of a[lo .. hi] (ascending, a[lo] <= x) with a[r] <= x.
__device__ __forceinline__ int last_le(const int* a, int lo, int hi, int x) {
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

template <int kPlanThreads, int J>
__global__ void __launch_bounds__(kPlanThreads) page_plan_kernel(const __grid_constant__ PagePlanArgs a) {
    constexpr int kPlanWarps = kPlanThreads / 32;
    extern __shared__ int plan_sm[];
    int* start = plan_sm;                // [n_req + 1]
    int* taken = plan_sm + a.n_req + 1;  // [n_req + 1]
    __shared__ unsigned wsum[2][kPlanWarps];
    __shared__ int wbad[kPlanWarps];
    pdl_trigger();
    pdl_wait();
    const int R = a.n_req, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (R + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int n_free = max(0, *a.n_free);

    // this thread's requests: their tokens and pages
    unsigned tok = 0, pg = 0;
    int bad = 0, c0 = 0, f0 = 0;  // (the first one's lengths stay at hand)
    const long long most = min(0x7fffffffLL, (long long)a.max_pages * a.page_size);
    constexpr int B = kPlanThreads > 512 ? 2 : 4;  // requests whose loads go out at once
    for (int r = r0; r < r1; r += B) {
        int c[B], f[B];
#pragma unroll
        for (int k = 0; k < B; k++) {
            c[k] = r + k < r1 ? a.cached[r + k] : 0;
            f[k] = r + k < r1 ? a.fresh[r + k] : 0;
        }
        if (r == r0) {
            c0 = c[0];
            f0 = f[0];
        }
#pragma unroll
        for (int k = 0; k < B; k++) {
            const long long len = (long long)c[k] + f[k];
            const bool neg = c[k] < 0 || f[k] < 0, wide = len > most;
            bad |= neg ? B2_PLAN_BAD_LENGTH : wide ? B2_PLAN_TABLE_FULL : 0;
            if (!neg && !wide) {
                tok = sat_add(tok, f[k]);
                pg = sat_add(pg, pages_of(a, (int)len) - pages_of(a, c[k]));
            }
        }
    }
    unsigned it = tok, ip = pg;  // inclusive over the warp, then over the CTA
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, it, o), p = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) {
            it = sat_add(it, t);
            ip = sat_add(ip, p);
        }
    }
    if (lane == 31) {
        wsum[0][warp] = it;
        wsum[1][warp] = ip;
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    if (lane == 0) wbad[warp] = bad;
    __syncthreads();
    // the warps before this one, and all of them: a scan by every warp
    unsigned wt = lane < kPlanWarps ? wsum[0][lane] : 0, wp = lane < kPlanWarps ? wsum[1][lane] : 0;
#pragma unroll
    for (int o = 1; o < kPlanWarps; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, wt, o), p = __shfl_up_sync(0xffffffffu, wp, o);
        if (lane >= o) {
            wt = sat_add(wt, t);
            wp = sat_add(wp, p);
        }
    }
    const unsigned total_tok = __shfl_sync(0xffffffffu, wt, kPlanWarps - 1);
    const unsigned total_pg = __shfl_sync(0xffffffffu, wp, kPlanWarps - 1);
    const unsigned bt = __shfl_sync(0xffffffffu, wt, max(warp - 1, 0));
    const unsigned bp = __shfl_sync(0xffffffffu, wp, max(warp - 1, 0));
    if (warp) {
        it = sat_add(it, bt);
        ip = sat_add(ip, bp);
    }
    int status = __reduce_or_sync(0xffffffffu, lane < kPlanWarps ? wbad[lane] : 0);
    if (total_tok > (unsigned)a.max_tokens || total_tok == kSumMax) status |= B2_PLAN_ROWS_FULL;
    if (total_pg > (unsigned)n_free || total_pg == kSumMax) status |= B2_PLAN_NO_PAGES;
    const bool ok = status == 0;
    const int T = ok ? (int)total_tok : 0, N = ok ? (int)total_pg : 0;
    if (ok) {
        int t = (int)(it - tok), p = (int)(ip - pg);
        for (int r = r0; r < r1; r++) {
            start[r] = t;
            taken[r] = p;
            const int c = r == r0 ? c0 : a.cached[r], f = r == r0 ? f0 : a.fresh[r];
            t += f;
            p += pages_of(a, c + f) - pages_of(a, c);
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
        const int r = last_le(taken, 0, R, e);
        a.table[(int64_t)r * a.table_stride + pages_of(a, a.cached[r]) + (e - taken[r])] = a.free_pages[e];
    }
    // a warp: J runs of 32 tokens (unsigned: the last run may pass 2^31)
    const unsigned cap = a.max_tokens, wstep = (unsigned)(gsize / 32) * (32 * J);
    for (unsigned t0 = (unsigned)(gtid / 32) * (32 * J); t0 < cap; t0 = t0 + wstep < t0 ? cap : t0 + wstep) {
        int lo = 0, hi = R;
        if (J > 1 && t0 < (unsigned)T) {  // the requests of its first and last token bound the others'
            const unsigned t = min(lane ? t0 + 32 * J - 1 : t0, (unsigned)T - 1);
            const int r = lane < 2 ? last_le(start, 0, R, (int)t) : 0;
            lo = __shfl_sync(0xffffffffu, r, 0);
            hi = __shfl_sync(0xffffffffu, r, 1);
        }
        int pos[J], req[J], in[J], page[J];
#pragma unroll
        for (int j = 0; j < J; j++) {
            const unsigned t = t0 + 32 * j + lane;
            pos[j] = in[j] = 0;
            req[j] = page[j] = -1;
            if (t < (unsigned)T) {
                const int r = last_le(start, lo, hi, (int)t), c = a.cached[r];
                pos[j] = c + ((int)t - start[r]);
                const int idx = div_page(a, pos[j]), have = pages_of(a, c);
                in[j] = pos[j] - idx * a.page_size;
                req[j] = r;
                // (a page of this step comes from the list: its table entry may be another CTA's to write)
                page[j] = *(idx < have ? a.table + ((int64_t)r * a.table_stride + idx)
                                       : a.free_pages + (taken[r] + idx - have));
            }
        }
        int64_t* slots = a.slots + t0 + lane;
        int32_t *positions = a.positions + t0 + lane, *token_req = a.token_req + t0 + lane;
#pragma unroll
        for (int j = 0; j < J; j++)
            if (t0 + 32 * j + lane < cap) {
                slots[32 * j] = page[j] >= 0 ? (int64_t)page[j] * a.page_size + in[j] : -1;
                positions[32 * j] = pos[j];
                token_req[32 * j] = req[j];
            }
    }
}

}  // namespace

template <int THREADS, int J>
static cudaError_t go_plan(const PagePlanArgs& a, int sms, cudaStream_t s) {
    const int smem = (int)(2 * sizeof(int) * ((size_t)a.n_req + 1));
    if (smem > 47 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(page_plan_kernel<THREADS, J>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(2 * sizeof(int) * (kPlanMaxReq + 1)));
        if (e != cudaSuccess) return e;
    }
    const long long work = std::max<long long>(((long long)a.max_tokens + J - 1) / J, a.n_req);
    const int grid = (int)std::max<long long>(1, std::min<long long>(1024 / THREADS * sms, (work + THREADS - 1) / THREADS));
    return launch_pdl(page_plan_kernel<THREADS, J>, dim3(grid), dim3(THREADS), smem, s, a);
}

int launch_page_plan(const PagePlanArgs& args, cudaStream_t s, std::string* err) {
    PagePlanArgs a = args;
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const unsigned P = (unsigned)a.page_size;
    int sh = 0;
    while ((1ull << sh) < P) sh++;
    a.page_shift = sh;
    a.page_mul = (unsigned)((((1ull << sh) - P) << 32) / P + 1);
    // every CTA scans all requests: more threads for many of them
    const bool many = a.max_tokens > 512 * sms;
    const cudaError_t e = a.n_req > 1024 ? (many ? go_plan<1024, kManyTokens>(a, sms, s) : go_plan<1024, 1>(a, sms, s))
                                         : (many ? go_plan<256, kManyTokens>(a, sms, s) : go_plan<256, 1>(a, sms, s));
    return e == cudaSuccess ? B2_OK : cuda_failed("page plan launch", e, err);
}

}  // namespace b2
