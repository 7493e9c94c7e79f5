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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpBatch = 32;                     // logits a thread takes together
constexpr int kLpEntries = 16;                   // maxima kept by a thread; longer slices: of several batches each
constexpr int kLpGroups = 64;                    // groups of threads whose maxima give the bound (k up to half of them)
constexpr int kLpList = 256;                     // batches at the bound, at most, for their candidates to be taken directly
constexpr int kLpMaxCluster = 8;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kLn2F = 0.6931471805599453f;

struct LogprobArgs {
    const void* x;
    int64_t ld;
    const int32_t* ids;
    float *logprob, *entropy, *top_logprob;
    int32_t* top_ids;
    int n, m, k, cluster, wide;
};

__device__ __forceinline__ float lf(float x) { return x; }
__device__ __forceinline__ float lf(__half x) { return __half2float(x); }
__device__ __forceinline__ float lf(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float lex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Order of the alternatives: value down (-0 equals 0), then index up.
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
    uint32_t b = __float_as_uint(x + 0.0f);
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)b << 32) | (uint32_t)~i;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)~(uint32_t)k; }

// the warp's maximum (a NaN loses)
__device__ __forceinline__ float max_lanes(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

struct Sums {
    float m, S, T;  // T in units of log 2: sum (x - m) log2(e) e^(x - m)
};

// t with its maximum raised to m
__device__ __forceinline__ Sums raise(Sums t, float m) {
    const float d = max_nan((t.m - (m == -INFINITY ? 0.0f : m)) * kLog2eF, -150.0f), f = lex2(d);
    return Sums{m, t.S * f, f * fmaf(d, t.S, t.T)};
}
// the warp's sums, in every lane
__device__ __forceinline__ Sums join_lanes(Sums t) {
    t = raise(t, max_lanes(t.m));
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        t.S += __shfl_xor_sync(0xffffffffu, t.S, o);
        t.T += __shfl_xor_sync(0xffffffffu, t.T, o);
    }
    return t;
}

// A thread's sums, S and T as pairs (even and odd elements)
struct Acc {
    float m = -INFINITY;
    unsigned long long S = 0, T = 0;

    // the maximum grows to at least bm; returns the reference
    __device__ __forceinline__ float grow(float bm) {
        const float nm = fmaxf(m, bm);
        const float z = nm == -INFINITY ? 0.0f : nm;
        const float df = max_nan((m - z) * kLog2eF, -150.0f), g = lex2(df);
        const unsigned long long g2 = f2_pack(g, g);
        T = f2_mul(g2, f2_fma(f2_pack(df, df), S, T));
        S = f2_mul(S, g2);
        m = nm;
        return z;
    }
    // two elements, x - z in `d`; `clamp`: they may be far below z, or -inf
    template <bool CLAMP>
    __device__ __forceinline__ void add(unsigned long long d) {
        unsigned long long t = f2_mul(d, f2_pack(kLog2eF, kLog2eF));
        float2 u = f2_unpack(t);
        if (CLAMP) {  // (e^d is 0 there, and 0 * inf would not be)
            u.x = max_nan(u.x, -150.0f);
            u.y = max_nan(u.y, -150.0f);
            t = f2_pack(u.x, u.y);
        }
        const unsigned long long e = f2_pack(lex2(u.x), lex2(u.y));
        S = f2_add(S, e);
        T = f2_fma(t, e, T);
    }
    __device__ __forceinline__ Sums sums() const {
        const float2 s = f2_unpack(S), t = f2_unpack(T);
        return Sums{m, s.x + s.y, t.x + t.y};
    }
};

// 16-bit logits two at a time: the larger (a NaN loses), the larger (a NaN
// stays), and as floats
template <typename T>
struct Two;
template <>
struct Two<__nv_bfloat16> {
    using V = __nv_bfloat162;
    static __device__ __forceinline__ V of(uint32_t u) { return *reinterpret_cast<const V*>(&u); }
    static __device__ __forceinline__ V both(float x) { return __bfloat162bfloat162(__float2bfloat16_rd(x)); }
    static __device__ __forceinline__ float2 floats(V v) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
};
template <>
struct Two<__half> {
    using V = __half2;
    static __device__ __forceinline__ V of(uint32_t u) { return *reinterpret_cast<const V*>(&u); }
    static __device__ __forceinline__ V both(float x) { return __half2half2(__float2half_rd(x)); }
    static __device__ __forceinline__ float2 floats(V v) { return __half22float2(v); }
};

// Threads of a CTA: 256, or 128 for rows of up to kLpShortRow logits, whose
// fixed steps weigh more than their reading (4096 rows of 1000 fp32: 31 us with
// 256, 19 with 128; of 16384 bf16: 47 and 41; of 32000: 69 both; 2048 of 128256:
// 96 and 109).
constexpr int kLpShortRow = 24576;

template <int NT>
struct LpShared {
    static constexpr int kWarps = NT / 32;
    static constexpr int kRound = NT * 8;         // logits one collecting round may add
    static constexpr int kCap = kRound + 1024;    // candidates held at once

    Sums part[kWarps];
    Sums row;                                // this CTA's slice
    __align__(16) float gmax[NT];
    float thr;
    int n_cand, n_list;
    int list[kLpList];
    int wcount[kWarps];
    __nv_bfloat16 ent[kLpEntries][NT];
    unsigned long long top[kLogprobMaxTop];  // this CTA's list, in order
    unsigned long long cand[kCap];
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) LpPack {
    T v[VEC];
};

// The k largest of s.cand[0 .. cnt) into s.top in order (zeros past cnt).
template <int NT>
__device__ void order_top(LpShared<NT>& s, int cnt, int k) {
    for (int i = threadIdx.x; i < k; i += NT)
        if (i >= cnt) s.top[i] = 0;
    for (int i = threadIdx.x; i < cnt; i += NT) {
        const unsigned long long key = s.cand[i];
        int above = 0;
        for (int j = 0; j < cnt; j++) above += s.cand[j] > key;
        if (above < k) s.top[above] = key;
    }
    __syncthreads();
}

// N chunks of VEC logits added to the sums; returns their maximum.
template <typename T, int VEC, int N>
__device__ __forceinline__ float add_chunks(const LpPack<T, VEC> (&p)[N], Acc& t) {
    if constexpr (sizeof(T) == 2 && VEC == 8) {
        using W = Two<T>;
        typename W::V v[N * 4];
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[u * 4 + i] = W::of(reinterpret_cast<const uint32_t*>(p[u].v)[i]);
        typename W::V mx = v[0];
#pragma unroll
        for (int i = 1; i < N * 4; i++) mx = __hmax2(mx, v[i]);
        const float2 f = W::floats(mx);
        const float bm = fmaxf(f.x, f.y), z = t.grow(bm);
        // logits that add nothing are raised to where they still add nothing (-inf among them)
        const typename W::V low = W::both(z - fmaxf(256.0f, fabsf(z) * 0.015625f));
        const unsigned long long z2 = f2_pack(-z, -z);
        if (W::floats(low).x > -INFINITY) {
#pragma unroll
            for (int i = 0; i < N * 4; i++) {
                const float2 x = W::floats(__hmax2_nan(v[i], low));
                t.template add<false>(f2_add(f2_pack(x.x, x.y), z2));
            }
        } else {  // the largest so far is next to the type's lowest value
#pragma unroll
            for (int i = 0; i < N * 4; i++) {
                const float2 x = W::floats(v[i]);
                t.template add<true>(f2_add(f2_pack(x.x, x.y), z2));
            }
        }
        return bm;
    } else {
        float f[N * VEC];
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int i = 0; i < VEC; i++) f[u * VEC + i] = lf(p[u].v[i]);
        float bm = f[0];
#pragma unroll
        for (int i = 1; i < N * VEC; i++) bm = fmaxf(bm, f[i]);
        const float z = t.grow(bm);
        const unsigned long long z2 = f2_pack(-z, -z);
#pragma unroll
        for (int i = 0; i < N * VEC; i += 2)
            t.template add<true>(f2_add(f2_pack(f[i], i + 1 < N * VEC ? f[i + 1] : -INFINITY), z2));
        return bm;
    }
}

// How a thread's chunks (its i-th is v0 + tid + i NT) fall to its
// entries: entry e has the chunks from e * len() on.
template <int VEC, int NT>
struct Entries {
    static constexpr int U = kLpBatch / VEC;  // chunks of a batch
    int agg;                                  // batches of an entry

    __device__ __forceinline__ Entries(int v0, int v1) {
        const int per = (v1 - v0 + NT - 1) / NT, batches = (per + U - 1) / U;
        agg = max(1, (batches + kLpEntries - 1) / kLpEntries);
    }
    __device__ __forceinline__ int len() const { return U * agg; }
};

// One CTA: the slice [v0, v1) of a row in chunks of VEC logits (the last one
// cut at n).  Returns how many entries this thread wrote.
template <typename T, int VEC, int NT>
__device__ __forceinline__ int slice_pass(const T* x, int n, int v0, int v1, bool keep, Acc& t, LpShared<NT>& s) {
    constexpr int U = Entries<VEC, NT>::U;
    using P = LpPack<T, VEC>;
    const Entries<VEC, NT> en(v0, v1);
    const int full = min(v1, n / VEC);  // chunks without a cut
    int left = en.agg, e = 0;
    float em = -INFINITY;
    auto put = [&]() { s.ent[e][threadIdx.x] = __float2bfloat16_ru(em); };
    int v = v0 + (int)threadIdx.x;
    constexpr int S = U * NT, B = S - NT;
    auto load = [&](P (&p)[U], int at) {
#pragma unroll
        for (int u = 0; u < U; u++) p[u] = *reinterpret_cast<const P*>(x + (int64_t)(at + u * NT) * VEC);
    };
    auto work = [&](const P (&p)[U]) {
        em = fmaxf(em, add_chunks<T, VEC, U>(p, t));
        if (keep && --left == 0) {
            put();
            e++;
            left = en.agg;
            em = -INFINITY;
        }
    };
    // (prefetching the next batch costs more in warps than it gains: 96 -> 103 us)
    for (; v + B < full; v += S) {
        P p[U];
        load(p, v);
        work(p);
    }
    const int tail = v;
    for (; v < full; v += NT) {
        const P p[1] = {*reinterpret_cast<const P*>(x + (int64_t)v * VEC)};
        em = fmaxf(em, add_chunks<T, VEC, 1>(p, t));
    }
    for (; v < v1; v += NT)  // the cut chunk
        for (int i = v * VEC; i < n; i++) {
            const LpPack<T, 1> p[1] = {{x[i]}};
            em = fmaxf(em, add_chunks<T, 1, 1>(p, t));
        }
    if (keep && (left != en.agg || v != tail)) {  // the last entry is a short one
        put();
        e++;
    }
    return e;
}

// The CTA's sums into s.part, and the k-th largest of kLpGroups maxima into s.thr.
template <int NT>
__device__ __forceinline__ void slice_sums(const Acc& acc, int k, LpShared<NT>& s) {
    constexpr int kWarps = LpShared<NT>::kWarps;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = k <= kLpGroups / 2 ? kLpGroups : NT, gl = NT / groups;  // lanes of a group
    if (tid == 0) s.n_cand = s.n_list = 0;
    if (k > 1) {
        float g = acc.m;
        for (int o = 1; o < gl; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (tid % gl == 0) s.gmax[tid / gl] = g;
    }
    const Sums t = join_lanes(acc.sums());
    if (lane == 0) s.part[warp] = t;
    __syncthreads();
    if (k == 1 && tid == 0) {
        float m = s.part[0].m;
#pragma unroll
        for (int w = 1; w < kWarps; w++) m = fmaxf(m, s.part[w].m);
        s.thr = m;
    }
    if (k > 1 && tid < groups) {
        const float g = s.gmax[tid];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < groups; j += 4) {
            const float4 o = *reinterpret_cast<const float4*>(s.gmax + j);
            above += (o.x > g || (o.x == g && j < tid)) + (o.y > g || (o.y == g && j + 1 < tid)) +
                     (o.z > g || (o.z == g && j + 2 < tid)) + (o.w > g || (o.w == g && j + 3 < tid));
        }
        if (above == k - 1) s.thr = g;
    }
    if (warp == kWarps - 1) {
        const Sums u = join_lanes(lane < kWarps ? s.part[lane] : Sums{-INFINITY, 0.0f, 0.0f});
        if (lane == 0) s.row = u;
    }
    __syncthreads();
}

// The k largest of the slice into s.top, from the thread's maximum and its
// `ne` entries.
template <typename T, int VEC, int NT>
__device__ __forceinline__ void slice_top(const T* x, int n, int v0, int v1, int k, float mine, int ne, LpShared<NT>& s) {
    constexpr int kWarps = LpShared<NT>::kWarps, kRound = LpShared<NT>::kRound, kCap = LpShared<NT>::kCap;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Entries<VEC, NT> en(v0, v1);
    const float thr = s.thr;
    auto list = [&](bool ties) {  // the entries that reach the bound (or pass it), as first chunks
        for (int e = 0; e < ne; e++) {
            const float m = __bfloat162float(s.ent[e][tid]);
            if (ties ? m >= thr : m > thr) {
                const int at = atomicAdd(&s.n_list, 1);
                if (at < kLpList) s.list[at] = tid + e * en.len() * NT;
            }
        }
        __syncthreads();
        return s.n_list <= kLpList;
    };
    const bool plain = list(true) && thr > -INFINITY;
    bool few = plain;
    if (!plain) {
        __syncthreads();
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        few = list(false);
    }
    unsigned long long bound = 0;  // after a cut of the list: keys at or under it are out
    auto push = [&](unsigned long long key) {
        if (key <= bound) return;
        const int at = atomicAdd(&s.n_cand, 1);
        if (at < kCap) s.cand[at] = key;
    };
    auto take = [&](int v) {
        if (v >= v1) return;
        const int i0 = v * VEC;
        if (i0 + VEC <= n) {
            const LpPack<T, VEC> p = *reinterpret_cast<const LpPack<T, VEC>*>(x + i0);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float f = lf(p.v[i]);
                if (plain ? f >= thr : f > thr) {
                    push(key_of(f, i0 + i));
                }
            }
        } else {
            for (int i = i0; i < n; i++) {
                const float f = lf(x[i]);
                if (plain ? f >= thr : f > thr) {
                    push(key_of(f, i));
                }
            }
        }
    };
    if (few) {  // their chunks, one to a thread
        for (int i = tid; i < s.n_list * en.len(); i += NT) {
            const int q = i / en.len();
            take(v0 + s.list[q] + (i - q * en.len()) * NT);
        }
        __syncthreads();
        if (s.n_cand > kCap) {  // they hold more candidates than the list
            __syncthreads();
            if (tid == 0) s.n_cand = 0;
            __syncthreads();
            few = false;
        }
    }
    if (!few) {  // chunk by chunk, the list cut to the k largest whenever the next might not fit
        for (int v = v0; v < v1; v += NT) {
            if (plain ? mine >= thr : mine > thr) take(v + tid);
            __syncthreads();
            const int cnt = s.n_cand;
            if (cnt > kCap - kRound) {
                order_top(s, cnt, k);
                for (int i = tid; i < k; i += NT) s.cand[i] = s.top[i];
                bound = s.top[k - 1];
                if (tid == 0) s.n_cand = k;
            }
            __syncthreads();
        }
    }
    const int cnt0 = s.n_cand;
    order_top(s, cnt0, k);
    if (!plain) {  // ties at the bound, in index order
        const int i1 = min(n, v1 * VEC);
        int cnt = min(cnt0, k);
        for (int base = v0 * VEC; base < i1 && cnt < k; base += NT) {
            const int i = base + tid;
            const bool tie = i < i1 && lf(x[i]) == thr;
            const unsigned bal = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) s.wcount[warp] = __popc(bal);
            __syncthreads();
            int at = cnt + __popc(bal & ((1u << lane) - 1)), all = 0;
            for (int w = 0; w < kWarps; w++) {
                if (w < warp) at += s.wcount[w];
                all += s.wcount[w];
            }
            if (tie && at < k) s.top[at] = key_of(thr, i);
            cnt = min(k, cnt + all);
            __syncthreads();
        }
    }
}

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
