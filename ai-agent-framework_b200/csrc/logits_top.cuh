// One pass over a slice of a row of logits by a CTA: running maximum and sums,
// and the k largest logits in order (logprobs.cu says how they are found).
// Used by the log probabilities and by the beam search's selection.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

constexpr int kLpBatch = 32;                     // logits a thread takes together
constexpr int kLpEntries = 16;                   // maxima kept by a thread; longer slices: of several batches each
constexpr int kLpGroups = 64;                    // groups of threads whose maxima give the bound (twice as many for k past half)
constexpr int kLpList = 256;                     // batches at the bound, at most, for their candidates to be taken directly
constexpr int kLpMaxCluster = 8;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kLn2F = 0.6931471805599453f;

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
    float m, S, T;  // T in units of log 2: sum (x - m) log2(e) e^(x - m); of an AccZ: what S leaves of its sum
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
    static constexpr bool kClamp = true;  // (e^d is multiplied by d, which may be -inf)
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
    // two elements, x - z in `d`, the i-th two of those taken together; `clamp`: they may be far below z, or -inf
    template <bool CLAMP>
    __device__ __forceinline__ void add(unsigned long long d, int) {
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
    __device__ __forceinline__ void flush() {}
    __device__ __forceinline__ Sums sums() const {
        const float2 s = f2_unpack(S), t = f2_unpack(T);
        return Sums{m, s.x + s.y, t.x + t.y};
    }
    static __device__ __forceinline__ Sums join(Sums t) { return join_lanes(t); }
};

// a + b, and what its rounding leaves (a + b = s + rest exactly, Knuth's two-sum)
__device__ __forceinline__ float two_sum(float a, float b, float& rest) {
    const float s = __fadd_rn(a, b), bb = __fsub_rn(s, a);
    rest = __fadd_rn(__fsub_rn(a, __fsub_rn(s, bb)), __fsub_rn(b, bb));
    return s;
}

// A thread's S alone, closer: elements taken together are summed on their own,
// in four chains, and that sum enters S with what the rounding leaves kept, from
// thread to thread too, so a large element meets a handful of roundings instead
// of one with every later element, and what is small beside it is not lost: the
// log of a sum of 1 and little more is that little to its own precision.
struct AccZ {
    static constexpr bool kClamp = false;
    float m = -INFINITY, S = 0.0f, rest = 0.0f;
    unsigned long long part[4] = {0, 0, 0, 0};

    __device__ __forceinline__ float grow(float bm) {
        const float nm = fmaxf(m, bm);
        const float z = nm == -INFINITY ? 0.0f : nm;
        const float g = lex2(max_nan((m - z) * kLog2eF, -150.0f));
        S *= g;
        rest *= g;
        m = nm;
        return z;
    }
    template <bool CLAMP>
    __device__ __forceinline__ void add(unsigned long long d, int i) {
        float2 u = f2_unpack(f2_mul(d, f2_pack(kLog2eF, kLog2eF)));
        if (CLAMP) {
            u.x = max_nan(u.x, -150.0f);
            u.y = max_nan(u.y, -150.0f);
        }
        const unsigned long long e = f2_pack(lex2(u.x), lex2(u.y));
        part[i & 3] = i < 4 ? e : f2_add(part[i & 3], e);
    }
    __device__ __forceinline__ void flush() {
        const float2 p = f2_unpack(f2_add(f2_add(part[0], part[1]), f2_add(part[2], part[3])));
        float left;
        S = two_sum(S, p.x + p.y, left);
        rest += left;
        part[0] = part[1] = part[2] = part[3] = 0;
    }
    __device__ __forceinline__ Sums sums() const { return Sums{m, S, rest}; }
    // the warp's sum, in every lane (its rest may differ there in the last bits)
    static __device__ __forceinline__ Sums join(Sums t) {
        const float nm = max_lanes(t.m), f = lex2(max_nan((t.m - (nm == -INFINITY ? 0.0f : nm)) * kLog2eF, -150.0f));
        const float p = __fmul_rn(t.S, f);
        t = Sums{nm, p, fmaf(t.T, f, fmaf(t.S, f, -p))};
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            float left;
            t.S = two_sum(t.S, __shfl_xor_sync(0xffffffffu, t.S, o), left);
            t.T += __shfl_xor_sync(0xffffffffu, t.T, o) + left;
        }
        return t;
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
    unsigned long long top[kLogprobMaxTop + 1];  // this CTA's list, in order (beams: one more, for the end token)
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
template <typename T, int VEC, int N, typename A>
__device__ __forceinline__ float add_chunks(const LpPack<T, VEC> (&p)[N], A& t) {
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
        const unsigned long long z2 = f2_pack(-z, -z);
        // logits that add nothing are raised to where they still add nothing (-inf among them)
        const typename W::V low = W::both(z - fmaxf(256.0f, fabsf(z) * 0.015625f));
        if (A::kClamp && W::floats(low).x > -INFINITY) {
#pragma unroll
            for (int i = 0; i < N * 4; i++) {
                const float2 x = W::floats(__hmax2_nan(v[i], low));
                t.template add<false>(f2_add(f2_pack(x.x, x.y), z2), i);
            }
        } else {  // the largest so far is next to the type's lowest value
#pragma unroll
            for (int i = 0; i < N * 4; i++) {
                const float2 x = W::floats(v[i]);
                t.template add<A::kClamp>(f2_add(f2_pack(x.x, x.y), z2), i);
            }
        }
        t.flush();
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
            t.template add<A::kClamp>(f2_add(f2_pack(f[i], i + 1 < N * VEC ? f[i + 1] : -INFINITY), z2), i / 2);
        t.flush();
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
template <typename T, int VEC, int NT, typename A>
__device__ __forceinline__ int slice_pass(const T* x, int n, int v0, int v1, bool keep, A& t, LpShared<NT>& s) {
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
        em = fmaxf(em, add_chunks<T, VEC, U, A>(p, t));
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
        em = fmaxf(em, add_chunks<T, VEC, 1, A>(p, t));
    }
    for (; v < v1; v += NT)  // the cut chunk
        for (int i = v * VEC; i < n; i++) {
            const LpPack<T, 1> p[1] = {{x[i]}};
            em = fmaxf(em, add_chunks<T, 1, 1, A>(p, t));
        }
    if (keep && (left != en.agg || v != tail)) {  // the last entry is a short one
        put();
        e++;
    }
    return e;
}

// The CTA's sums into s.part, and the k-th largest of kLpGroups maxima into s.thr.
template <int NT, typename A>
__device__ __forceinline__ void slice_sums(const A& acc, int k, LpShared<NT>& s) {
    constexpr int kWarps = LpShared<NT>::kWarps;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = k <= kLpGroups / 2 ? kLpGroups : 2 * kLpGroups, gl = NT / groups;  // lanes of a group
    if (tid == 0) s.n_cand = s.n_list = 0;
    if (k > 1) {
        float g = acc.m;
        for (int o = 1; o < gl; o <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
        if (tid % gl == 0) s.gmax[tid / gl] = g;
    }
    const Sums t = A::join(acc.sums());
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
        const Sums u = A::join(lane < kWarps ? s.part[lane] : Sums{-INFINITY, 0.0f, 0.0f});
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

}  // namespace
}  // namespace b2
