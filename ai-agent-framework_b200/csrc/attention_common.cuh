// What the attentions over a paged cache have in common: a row's visible
// positions, 16-byte copies, numbers as sums of 16-bit terms, shares of a line
// of units.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "dev.cuh"

namespace b2 {
namespace {

constexpr long long kMaxLen = 0x7fffffffLL - 63;  // so that a step's positions are ints
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 16384.0f;  // probabilities enter P V times 2^14

// A row's sequence: table row, visible positions [lo, len).  len 0: nothing.
struct Seq {
    int tr, lo, len;
    bool bad;  // the length passes the table, or the row has none
};

// Lengths, requests and table entries are usually the work of the launches
// just before (a page plan on the same stream, whose grid may still run when
// this one's CTAs start), so they take no read-only loads: plain ones behind
// pdl_wait, and with EARLY, ahead of it, loads from L2, where the words of a
// grid that has ended are.
template <bool EARLY>
__device__ __forceinline__ int word(const int32_t* p) {
    return EARLY ? __ldcg(p) : *p;
}

template <bool EARLY = false, typename A>
__device__ __forceinline__ Seq seq_of(const A& a, int b) {
    Seq s;
    s.tr = a.req ? word<EARLY>(a.req + b) : b;
    const long long len = (long long)word<EARLY>(a.lens + b) + a.len_add;
    const bool none = s.tr < 0 || len <= 0;
    s.bad = !none && (s.tr >= a.n_req || len > (long long)a.max_pages * a.page_size || len > kMaxLen);
    s.len = none || s.bad ? 0 : (int)len;
    s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
    return s;
}

__device__ __forceinline__ void cp16(uint32_t smem, const void* gmem, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename C>
struct Cvt;
template <>
struct Cvt<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b, float2& back) {
        const __half2 h = __floats2half2_rn(a, b);
        back = __half22float2(h);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    // d += a b
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // d = a b
    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};
template <>
struct Cvt<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b, float2& back) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        back = __bfloat1622float2(h);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    // d += a b
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    // d = a b
    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};

// (a, b) as N packed terms, each the rounding of what the ones before left
template <typename C, int N>
__device__ __forceinline__ void split_terms(float a, float b, uint32_t* t) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        float2 f;
        t[i] = Cvt<C>::pack(a, b, f);
        a -= f.x;
        b -= f.y;
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (x * y + add) / z, none negative, exact; in 32 bits where they do (a 64-bit
// division is some 100 instructions)
__device__ __forceinline__ long long mul_div(long long x, long long y, long long z, int add = 0) {
    const long long p = x * y + add;
    return (p | z) <= 0xffffffffLL ? (long long)((unsigned)p / (unsigned)z) : p / z;
}

}  // namespace
}  // namespace b2
