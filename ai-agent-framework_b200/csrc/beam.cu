// The best continuations over a request's beams and the vocabulary, and rows
// of state brought into their order.
//
//   c(w, v) = scores[w] + x[w][v] - log Z_w,  log Z_w = m_w + log sum_v e^(x[w][v] - m_w)
//
// Within a beam the order is that of the logits, so no more than its k largest
// logits (k + 1 where one token is the end token, which is left out) can be
// among the request's k best.  The first launch makes one pass over every
// beam's row (logits_top.cuh, the pass of the log probabilities): log Z and
// that list.  The second takes a request's lists together: the k-th largest of
// a few entries off the top of each list bounds the k-th best candidate, and
// what reaches the bound is ordered by counting, in 64 bits.  Two beams' log Z
// are known to fp32 exponentials; where that leaves the order of two candidates open
// (a request in some 400), the CTA takes the two rows' log Z in 64 bits.
//
// Bound by the pass: 64 requests of 16 beams over 128256 bf16 logits, 263 MB, take 79 us
// with the histories' reordering (40 us of HBM; the pass 65, with exponential units and issue
// slots half busy, the lists 11, the histories 7, overlapped in part), or 138 where a request
// needs sums in 64 bits: 25 us a beam.  Beams that tie all need them: 16 with the same logits and
// scores 420 us, 64 1640.  4 beams of one request over 151936 fp32 16.5 us, launches all of it.
// A cluster for each request that shares the sums in 64 bits lost: 105 -> 115 us.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "logits_top.cuh"
#include "paged.h"

namespace b2 {
namespace {

namespace cg = cooperative_groups;

struct BeamArgs {
    const void* x;
    int64_t ld;
    const float* scores;
    int32_t *parent, *token;
    float *score, *eos_score;
    double* log_z;             // [rows], NaN: the row offers nothing
    unsigned long long* keys;  // [rows][k1], the row's largest logits in order (0: no more)
    int n, width, k, k1, eos, cluster, wide, sms;
};

// A beam's score, NaN where it offers nothing.
__device__ __forceinline__ float beam_score(const BeamArgs& a, int64_t row) {
    const float s = a.scores ? a.scores[row] : 0.0f;
    return fabsf(s) < INFINITY ? s : __int_as_float(0x7fc00000);
}

template <typename T, int VEC, int NT>
__global__ void __launch_bounds__(NT) beam_rows_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ __align__(16) uint8_t lp_raw[];
    LpShared<NT>& s = *reinterpret_cast<LpShared<NT>*>(lp_raw);
    pdl_wait();
    pdl_trigger();
    const int C = a.cluster, rank = C > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int64_t row = blockIdx.x / C;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float score = beam_score(a, row);
    const double nan = __longlong_as_double(0x7ff8000000000000LL);
    if (score != score) {  // an ended beam: its logits are not looked at
        if (rank == 0 && tid == 0) {
            a.log_z[row] = nan;
            if (a.eos_score) a.eos_score[row] = -INFINITY;
        }
        return;
    }
    const int nv = (a.n + VEC - 1) / VEC, per = (nv + C - 1) / C;
    const int v0 = min(nv, rank * per), v1 = min(nv, v0 + per);
    AccZ acc;
    const int ne = slice_pass<T, VEC, NT>(x, a.n, v0, v1, true, acc, s);
    slice_sums(acc, a.k1, s);
    slice_top<T, VEC, NT>(x, a.n, v0, v1, a.k1, acc.m, ne, s);
    if (C > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (rank == 0) {
            if (warp == 0) {
                const Sums u = AccZ::join(lane < C ? cl.map_shared_rank(&s, lane)->row : Sums{-INFINITY, 0.0f, 0.0f});
                __syncwarp();
                if (lane == 0) s.row = u;
            }
            if (tid == 0) s.n_cand = 0;
            __syncthreads();
            for (int i = tid; i < C * a.k1; i += NT) {
                const unsigned long long key = cl.map_shared_rank(&s, i / a.k1)->top[i % a.k1];
                if (key) s.cand[atomicAdd(&s.n_cand, 1)] = key;
            }
            __syncthreads();
            order_top(s, s.n_cand, a.k1);
            __syncthreads();
        }
        cl.sync();  // no CTA leaves while its lists are read
        if (rank) return;
    }
    const Sums r = s.row;
    const bool ok = fabsf(r.m) < INFINITY && r.S == r.S;
    const double z = ok ? (double)r.m + log((double)r.S + (double)r.T) : nan;
    for (int i = tid; i < a.k1; i += NT) a.keys[row * a.k1 + i] = s.top[i];
    if (tid == 0) {
        a.log_z[row] = z;
        if (a.eos_score) a.eos_score[row] = ok ? (float)((double)score + ((double)lf(x[a.eos]) - z)) : -INFINITY;
    }
}

constexpr int kMergeThreads = 512;
constexpr int kMergeHeads = 2 * kLogprobMaxTop;                  // entries that give the bound, at most

// How far the first launch's log Z may be off: fp32 terms off by 2 steps and
// sums by the roundings of those taken together are 2^-20, the rounding of d (d
// steps of a term e^d) adds less than that.  Candidates of two beams that are closer
// than twice this are told apart by log Z in 64 bits.
constexpr double kClose = 2.0 / (1 << 18);

// Candidates in order: score down, then place (row, then token) up.
struct Cand {
    double score;
    unsigned long long at;  // row of the request << 32 | token
    __device__ __forceinline__ bool before(const Cand& o) const {
        return score > o.score || (score == o.score && at < o.at);
    }
};

struct MergeShared {
    double base[kBeamMaxWidth];   // the beam's score, NaN: nothing from this beam
    double log_z[kBeamMaxWidth];
    double head[kMergeHeads];
    double part[kMergeThreads / 32];
    double pow2[32];              // 2^(j/32)
    double bound;
    int fine[kBeamMaxWidth];      // log_z is in 64 bits; 2: it has to be
    int live, n, again;
    Cand best[kLogprobMaxTop];      // in order
    Cand cand[1];                   // width x k1 of them
};

// e^x for x <= 0, off by 2^-49 of itself to -40 and 2^-45 to -700 (Tang's table method: x = (32 n + j) log(2) / 32 + r,
// e^x = 2^n 2^(j/32) e^r with e^r as its series to r^6 / 720, |r| <= log(2) / 64;
// pow2[j] = 2^(j/32)).  In 64 bits that is 12 operations; exp() took twice the time.
__device__ __forceinline__ double exp64(double x, const double* pow2) {
    x = fmax(x, -700.0);  // (adds nothing to a sum that holds 1)
    const double shift = 6755399441055744.0;  // 1.5 2^52: the sum's low bits are the rounded whole number
    const double t = fma(x, 32.0 * 1.4426950408889634, shift);
    const int k = __double2loint(t);
    const double r = fma(t - shift, -0.6931471805599453 / 32.0, x);
    double p = fma(r, 1.0 / 720.0, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    const double b = pow2[k & 31];
    p = fma(p * r, b, b);
    return __hiloint2double(__double2hiint(p) + ((k >> 5) << 20), __double2loint(p));
}

// log Z of a row whose largest logit is m in 64 bits, by the CTA: bound by the
// SM's 64-bit units, some 25 us for 128256 logits.
template <typename T>
__device__ double log_z64(const T* x, int n, bool wide, double m, double* part, const double* pow2) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double z[4] = {0, 0, 0, 0};
    constexpr int VEC = 16 / sizeof(T), U = 4;  // four 16-byte loads in flight (two rows of 128256 fp32 one by one: 113 us)
    const int chunks = wide ? n / VEC : 0;
    for (int c = tid; c < chunks; c += U * kMergeThreads) {
        LpPack<T, VEC> p[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c + u * kMergeThreads < chunks) p[u] = reinterpret_cast<const LpPack<T, VEC>*>(x)[c + u * kMergeThreads];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (c + u * kMergeThreads < chunks)
#pragma unroll
                for (int i = 0; i < VEC; i++) z[i & 3] += exp64((double)lf(p[u].v[i]) - m, pow2);
    }
    for (int i = chunks * VEC + tid; i < n; i += kMergeThreads) z[0] += exp64((double)lf(x[i]) - m, pow2);
    double s = (z[0] + z[1]) + (z[2] + z[3]);
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (lane == 0) part[warp] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < kMergeThreads / 32; w++) s += part[w];
    return m + log(s);
}

// One CTA a request.
template <typename T>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const __grid_constant__ BeamArgs a) {
    extern __shared__ __align__(16) uint8_t mg_raw[];
    MergeShared& s = *reinterpret_cast<MergeShared*>(mg_raw);
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, W = a.width, k = a.k, k1 = a.k1;
    const int64_t row0 = (int64_t)blockIdx.x * W, out = (int64_t)blockIdx.x * k;
    if (tid == 0) s.live = 0;
    __syncthreads();
    if (tid < W) {
        const double z = a.log_z[row0 + tid];
        s.log_z[tid] = z;
        s.base[tid] = z == z ? (double)beam_score(a, row0 + tid) : z;
        s.fine[tid] = 0;
        if (z == z) atomicAdd(&s.live, 1);
    }
    __syncthreads();
    // entry i of beam w; -inf where there is none
    auto entry = [&](int w, int i) {
        Cand c{-INFINITY, 0};
        const double b = s.base[w];
        if (b != b) return c;
        const unsigned long long key = a.keys[(row0 + w) * k1 + i];
        const int v = key_index(key);
        if (!key || v == a.eos) return c;
        c.score = b + ((double)key_value(key) - s.log_z[w]);
        c.at = (unsigned long long)w << 32 | (unsigned)v;
        return c;
    };
    // a lower bound of the k-th best: the k-th largest among the first few of every list
    // (one more of each where one of them may be the end token)
    const int deep = s.live ? min(k1, max((k + s.live - 1) / s.live + (a.eos >= 0), kMergeHeads / W)) : 0, heads = W * deep;
    double bound = -INFINITY;
    if (heads <= kMergeHeads) {
        if (tid < heads) s.head[tid] = entry(tid / deep, tid % deep).score;
        if (tid == 0) s.bound = -INFINITY;
        __syncthreads();
        constexpr int kHelp = kMergeThreads / kMergeHeads;  // lanes that count for one of them
        const int i = tid / kHelp;
        const double v = i < heads ? s.head[i] : 0.0;
        int above = 0;
        for (int j = tid % kHelp; j < heads; j += kHelp) above += s.head[j] > v || (s.head[j] == v && j < i);
#pragma unroll
        for (int o = 1; o < kHelp; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
        if (i < heads && above == k - 1) s.bound = v;
        __syncthreads();
        bound = s.bound - 2 * kClose;
    }
    while (true) {
        if (tid == 0) s.n = s.again = 0;
        __syncthreads();
        for (int i = tid; i < W * k1; i += kMergeThreads) {
            const Cand c = entry(i / k1, i % k1);
            if (c.score > -INFINITY && c.score >= bound) s.cand[atomicAdd(&s.n, 1)] = c;
        }
        __syncthreads();
        const int n = s.n;
        for (int i = tid; i < n; i += kMergeThreads) {
            const Cand c = s.cand[i];
            int above = 0;
            for (int j = 0; j < n; j++) above += s.cand[j].before(c);
            if (above < k) s.best[above] = c;
        }
        __syncthreads();
        // two beams too close for what is known of them: neighbours among the k best, and the k-th
        // with any that comes behind it (a beam's own next ones may lie between)
        auto close = [&](const Cand& x, const Cand& y) {
            const int u = (int)(x.at >> 32), v = (int)(y.at >> 32);
            if (u != v && x.score - y.score < kClose && (s.fine[u] != 1 || s.fine[v] != 1)) {
                atomicCAS(&s.fine[u], 0, 2);
                atomicCAS(&s.fine[v], 0, 2);
                s.again = 1;
            }
        };
        for (int i = tid; i < min(n, k) - 1; i += kMergeThreads) close(s.best[i], s.best[i + 1]);
        if (n > k) {
            const Cand last = s.best[k - 1];
            for (int i = tid; i < n; i += kMergeThreads)
                if (last.before(s.cand[i])) close(last, s.cand[i]);
        }
        __syncthreads();
        if (!s.again) break;
        if (tid < 32) s.pow2[tid] = exp2(tid / 32.0);
        __syncthreads();
        for (int w = 0; w < W; w++) {
            if (s.fine[w] != 2) continue;
            const double z = log_z64(static_cast<const T*>(a.x) + (row0 + w) * a.ld, a.n, a.wide,
                                     (double)key_value(a.keys[(row0 + w) * k1]), s.part, s.pow2);
            __syncthreads();
            if (tid == 0) {
                s.log_z[w] = z;
                s.fine[w] = 1;
            }
        }
        __syncthreads();
    }
    if (a.eos_score && tid < W && s.fine[tid])  // (a row has one log Z)
        a.eos_score[row0 + tid] =
            (float)(s.base[tid] + ((double)lf(static_cast<const T*>(a.x)[(row0 + tid) * a.ld + a.eos]) - s.log_z[tid]));
    const int n = min(s.n, k);
    for (int i = tid; i < k; i += kMergeThreads) {
        const Cand c = i < n ? s.best[i] : Cand{-INFINITY, 0};
        a.parent[out + i] = i < n ? (int)(row0 + (int)(c.at >> 32)) : -1;
        a.token[out + i] = i < n ? (int)(c.at & 0xffffffffu) : -1;
        a.score[out + i] = (float)c.score;
    }
}

constexpr size_t kPlainSmem = 48 * 1024;  // shared memory that a launch may ask for as it is

template <typename T, int NT>
cudaError_t go_rows(const BeamArgs& a, int rows, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    auto kern = a.wide ? beam_rows_kernel<T, W, NT> : beam_rows_kernel<T, 1, NT>;
    static_assert(sizeof(LpShared<NT>) <= kPlainSmem, "no attribute to set");
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

// 128 threads instead of 256 also where the CTAs of 256, 6 an SM, would go round
// once and by up to a third again, and those of 128 fit at once (rows of 128256
// bf16, 256 and 128 threads: 880 rows 70 and 72 us, 896 rows 80 and 72, 1184 rows 91
// and 82, 1760 rows 113 and 124).  Not with fp32, 5 an SM: 960 rows of 50000 60 and 70.
template <typename T>
bool small_ctas(const BeamArgs& a, int rows) {
    const int round = 6 * a.sms;
    return a.n <= kLpShortRow || (sizeof(T) == 2 && rows > round && 3LL * rows <= 4LL * round);
}

template <typename T>
cudaError_t go(const BeamArgs& a, int rows, cudaStream_t s) {
    cudaError_t e = small_ctas<T>(a, rows) ? go_rows<T, 128>(a, rows, s) : go_rows<T, 256>(a, rows, s);
    if (e != cudaSuccess) return e;
    auto kern = beam_merge_kernel<T>;
    const size_t smem = sizeof(MergeShared) + (size_t)a.width * a.k1 * sizeof(Cand);
    // (the limit is the kernel's, not the call's: always the most, so that no thread lowers it under another's launch)
    constexpr int most = sizeof(MergeShared) + kBeamMaxWidth * (kLogprobMaxTop + 1) * sizeof(Cand);
    if (smem > kPlainSmem) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3(rows / a.width), dim3(kMergeThreads), smem, s, a);
}

// entries of a row's list: one more where one of them may be the end token
int list_len(int n, int k) { return std::min(n, k + 1); }

// ---------------------------------------------------------------------------

struct ReorderArgs {
    const uint32_t* src;
    uint32_t* dst;
    const int32_t *parent, *lens, *token;
    int32_t* new_lens;
    int64_t src_stride, dst_stride, words, chunks;  // chunks of kReorderWords words in a row
    int n_src, n_dst, wide;
};

constexpr int kReorderThreads = 128;
constexpr int kReorderWords = 4 * kReorderThreads * 4;  // words of one CTA's turn: four 16-byte loads a thread

__global__ void __launch_bounds__(kReorderThreads) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x;
    const int64_t items = a.chunks * a.n_dst;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int r = (int)(it / a.chunks);
        const int64_t c0 = (it - (int64_t)r * a.chunks) * kReorderWords;
        const int p = a.parent[r];
        const bool live = p >= 0 && p < a.n_src;
        const int64_t len = !live ? 0 : a.lens ? min((int64_t)max(a.lens[p], 0), a.words) : a.words;
        const uint32_t* src = a.src + (live ? p : 0) * a.src_stride;
        uint32_t* dst = a.dst + r * a.dst_stride;
        const bool put = live && a.token && len < a.words;
        if (c0 == 0 && tid == 0) {
            if (a.new_lens) a.new_lens[r] = (int)min(len + (put ? 1 : 0), (int64_t)0x7fffffff);
            if (put) dst[len] = (uint32_t)a.token[r];
        }
        const int64_t c1 = min(len, c0 + kReorderWords);
        if (a.wide) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t i = c0 + 4 * (tid + j * kReorderThreads);
                if (i + 4 <= c1) v[j] = *reinterpret_cast<const uint4*>(src + i);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t i = c0 + 4 * (tid + j * kReorderThreads);
                if (i + 4 <= c1) *reinterpret_cast<uint4*>(dst + i) = v[j];
                else
                    for (int64_t x = i; x < c1; x++) dst[x] = src[x];
            }
        } else {
            for (int64_t i = c0 + tid; i < c1; i += kReorderThreads) dst[i] = src[i];
        }
    }
}

}  // namespace

size_t beam_select_scratch(int n, int rows, int k) {
    return (size_t)rows * (8 + 8 * (size_t)list_len(n, k));
}

int launch_beam_select(const void* logits, int dtype, int n, int n_groups, int width, int64_t ld, const float* scores,
                       int k, int eos, int32_t* parent, int32_t* token, float* score, float* eos_score, void* scratch,
                       cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    const int es = dtype == 0 ? 4 : 2, rows = n_groups * width;
    BeamArgs a{};
    a.x = logits;
    a.ld = ld;
    a.scores = scores;
    a.parent = parent;
    a.token = token;
    a.score = score;
    a.eos_score = eos >= 0 ? eos_score : nullptr;
    a.log_z = static_cast<double*>(scratch);
    a.keys = reinterpret_cast<unsigned long long*>(a.log_z + rows);
    a.n = n;
    a.width = width;
    a.k = k;
    a.k1 = eos >= 0 ? list_len(n, k) : k;
    a.eos = eos >= 0 ? eos : -1;
    a.wide = !((uintptr_t)logits & 15) && (rows == 1 || ld * es % 16 == 0);
    // CTAs per row: while the rows do not fill the machine and a slice keeps 4096 logits
    int c = 1;
    while (c < kLpMaxCluster && rows * 2LL * c <= sms && n / (2 * c) >= 4096) c *= 2;
    a.cluster = c;
    a.sms = sms;
    const cudaError_t e = dtype == 0   ? go<float>(a, rows, s)
                          : dtype == 1 ? go<__half>(a, rows, s)
                                       : go<__nv_bfloat16>(a, rows, s);
    return e == cudaSuccess ? B2_OK : cuda_failed("beam selection launch", e, err);
}

int launch_beam_reorder(const void* src, int n_src, int64_t src_stride, void* dst, int n_dst, int64_t dst_stride,
                        int64_t words, const int32_t* parent, const int32_t* lens, const int32_t* token,
                        int32_t* new_lens, cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    ReorderArgs a{};
    a.src = static_cast<const uint32_t*>(src);
    a.dst = static_cast<uint32_t*>(dst);
    a.parent = parent;
    a.lens = lens;
    a.token = token;
    a.new_lens = new_lens;
    a.src_stride = src_stride;
    a.dst_stride = dst_stride;
    a.words = words;
    a.chunks = std::max<int64_t>(1, (words + kReorderWords - 1) / kReorderWords);
    a.n_src = n_src;
    a.n_dst = n_dst;
    a.wide = !(((uintptr_t)src | (uintptr_t)dst) & 15) && src_stride % 4 == 0 && dst_stride % 4 == 0;
    const int64_t items = a.chunks * n_dst;
    const cudaError_t e = launch_pdl(beam_reorder_kernel, dim3((unsigned)std::min<int64_t>(items, 16LL * sms)),
                                     dim3(kReorderThreads), 0, s, a);
    return e == cudaSuccess ? B2_OK : cuda_failed("beam reorder launch", e, err);
}

}  // namespace b2
