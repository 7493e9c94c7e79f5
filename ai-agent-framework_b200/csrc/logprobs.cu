// Log probabilities of given tokens, the entropy and the top alternatives of
// rows of logits.
//
// With m = max x and d = x - m:  S = sum e^d,  T = sum d e^d,
//   log p(i) = d_i - log S,   H = log S - T / S.
// (Both terms of H are >= 0, so nothing cancels.)  One pass keeps (m, S, T)
// per thread, rescaled when a thread's maximum grows:
//   m -> m':  S' = S e^(m - m'),  T' = e^(m - m') (T + (m - m') S).
//
// Top k without a second pass over the row.  The pass leaves, besides each
// thread's largest logit, the largest of every 32 that a thread took together
// (in shared memory, rounded up to bf16).  The k-th largest of the maxima of 64
// groups of threads (of all threads for k past 32) is a lower bound of the k-th largest logit; only the 32s
// whose maximum reaches it, a few more than k of them, are read again (from
// L2), and their candidates are ordered by counting.  Where very many reach it
// (a vocabulary masked with one value), the logits above the bound are taken
// first and the ties in index order from the start of the row.
//
// A row's slices go to the CTAs of a cluster, so that few rows still fill the
// machine (one row of 151936 fp32: 9.2 us on 8 CTAs); the lists and sums meet in
// the first CTA's hands over distributed shared memory.
//
// Bound by HBM for fp32 (2048 rows of 128256, 20 alternatives: 1.05 GB in 168
// us, 6.3 TB/s).  16-bit logits (bf16: 525 MB in 96 us, 5.5 TB/s) bring twice the
// exponentials a byte: the exponential units are 70 % busy, the issue slots 60
// %.  Measured and not kept there: part of the exponentials as polynomials on
// the multiplying units (108 us and more: registers cost warps), batches ahead
// in registers (103) or in shared memory (94, but no faster in calls back to
// back, where the card is at its 1000 W cap), 512 threads (109).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "logits_top.cuh"
#include "paged.h"

namespace b2 {
namespace {

namespace cg = cooperative_groups;

struct LogprobArgs {
    const void* x;
    int64_t ld;
    const int32_t* ids;
    float *logprob, *entropy, *top_logprob;
    int32_t* top_ids;
    int n, m, k, cluster, wide;
};

template <typename T, int VEC, int NT>
__global__ void __launch_bounds__(NT) logprob_kernel(const __grid_constant__ LogprobArgs a) {
    extern __shared__ __align__(16) uint8_t lp_raw[];
    LpShared<NT>& s = *reinterpret_cast<LpShared<NT>*>(lp_raw);
    constexpr int kWarps = LpShared<NT>::kWarps;
    pdl_trigger();
    pdl_wait();
    const int C = a.cluster, rank = C > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int64_t row = blockIdx.x / C;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nv = (a.n + VEC - 1) / VEC, per = (nv + C - 1) / C;
    const int v0 = min(nv, rank * per), v1 = min(nv, v0 + per);

    // the given tokens' logits, on their way during the pass
    constexpr int kIds = 2;
    float given[kIds];
#pragma unroll
    for (int j = 0; j < kIds; j++) {
        const int i = tid + j * NT;
        const int id = rank == 0 && i < a.m ? a.ids[row * a.m + i] : -1;
        given[j] = id >= 0 && id < a.n ? lf(x[id]) : __int_as_float(0x7fc00000);
    }

    Acc acc;
    const int ne = slice_pass<T, VEC, NT>(x, a.n, v0, v1, a.k > 0, acc, s);
    slice_sums(acc, a.k, s);
    if (a.k > 0) slice_top<T, VEC, NT>(x, a.n, v0, v1, a.k, acc.m, ne, s);

    if (C > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0) {
            if (warp == 0) {
                const Sums u = join_lanes(lane < C ? cl.map_shared_rank(&s, lane)->row : Sums{-INFINITY, 0.0f, 0.0f});
                __syncwarp();
                if (lane == 0) s.row = u;
            }
            // the C lists as one, with no empty places
            if (tid == 0) s.n_cand = 0;
            __syncthreads();
            for (int i = tid; i < C * a.k; i += NT) {
                const unsigned long long key = cl.map_shared_rank(&s, i / a.k)->top[i % a.k];
                if (key) s.cand[atomicAdd(&s.n_cand, 1)] = key;
            }
            __syncthreads();
            if (a.k > 0) order_top(s, s.n_cand, a.k);
            __syncthreads();
        }
        cl.sync();  // no CTA leaves while its lists are read
        if (rank) return;
    }
    const Sums r = s.row;
    const float lS = logf(r.S);
    const float z = r.m == -INFINITY ? 0.0f : r.m;
    auto lp = [&](float v) { return (v - z) - lS; };
    const float nan = __int_as_float(0x7fc00000);
    for (int i = tid, j = 0; i < a.m; i += NT, j++) {
        float v = nan;
        if (j < kIds) {
            v = j ? given[kIds - 1] : given[0];
        } else {
            const int id = a.ids[row * a.m + i];
            if (id >= 0 && id < a.n) v = lf(x[id]);
        }
        a.logprob[row * a.m + i] = r.m != -INFINITY ? lp(v) : nan;
    }
    if (tid == 0 && a.entropy) a.entropy[row] = lS - r.T / r.S * kLn2F;
    for (int i = tid; i < a.k; i += NT) {
        const unsigned long long key = s.top[i];
        a.top_ids[row * a.k + i] = key ? key_index(key) : -1;
        a.top_logprob[row * a.k + i] = key && r.m != -INFINITY ? lp(key_value(key)) : nan;
    }
}

template <typename T, int NT>
cudaError_t go_threads(const LogprobArgs& a, int rows, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    auto kern = a.wide ? logprob_kernel<T, W, NT> : logprob_kernel<T, 1, NT>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(LpShared<NT>));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * a.cluster));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = sizeof(LpShared<NT>);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)a.cluster, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T>
cudaError_t go(const LogprobArgs& a, int rows, cudaStream_t s) {
    return a.n <= kLpShortRow ? go_threads<T, 128>(a, rows, s) : go_threads<T, 256>(a, rows, s);
}

}  // namespace

int launch_logprobs(const void* logits, int dtype, int n, int rows, int64_t ld, const int32_t* ids, int m,
                    float* logprob, float* entropy, int k, int32_t* top_ids, float* top_logprob, cudaStream_t s,
                    std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const int es = dtype == 0 ? 4 : 2;
    LogprobArgs a{};
    a.x = logits;
    a.ld = ld;
    a.ids = ids;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprob = top_logprob;
    a.n = n;
    a.m = m;
    a.k = k;
    // 16-byte loads where every row starts on 16 bytes, else one logit a load
    // (2048 rows of 50257 bf16: 49 us 50264 apart, 58 back to back)
    a.wide = !((uintptr_t)logits & 15) && (rows == 1 || ld * es % 16 == 0);
    // CTAs per row: while the rows do not fill the machine and a slice keeps 4096 logits
    int c = 1;
    while (c < kLpMaxCluster && rows * 2LL * c <= sms && n / (2 * c) >= 4096) c *= 2;
    a.cluster = c;
    const cudaError_t e = dtype == 0   ? go<float>(a, rows, s)
                          : dtype == 1 ? go<__half>(a, rows, s)
                                       : go<__nv_bfloat16>(a, rows, s);
    return e == cudaSuccess ? B2_OK : cuda_failed("log probabilities launch", e, err);
}

}  // namespace b2
