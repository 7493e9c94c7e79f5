// Attention of one query row per sequence over a paged KV cache, split over
// the cache's length and joined.
//
//   s_j = scale * q . k_j;  s_j <- cap * tanh(s_j / cap) (cap > 0);
//   s_j <- s_j + slope_h * (j - (len - 1)) (slopes given);
//   out = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M) over the positions
//   max(0, len - window) <= j < len;  lse = M + log of the sum.
//
// HBM-bound: every visible K and V row is read from the page that holds it once
// for each block of query heads that share it, 8 or 16 of them; the blocks of a
// larger group walk the rows side by side, so HBM gives them once and L2 the
// other times.
//
// Split.  The sequences of the batch, one after another, are a line of units,
// a unit being one step of 16 or 32 positions.  Group g of G takes the units
// [g W / G, (g + 1) W / G), and its workers, one warp for every (KV head, block
// of query heads), walk that share side by side.  Ragged batches thus load
// every SM equally without the host knowing a length, and a launch captured in
// a graph follows the lengths it finds; and the heads of a position, neighbours
// in memory, are read at about the same time (head dimension 112, 8 KV heads:
// heads apart in time cost 1.3 times the bytes in half-used 128-byte lines).
// Each sequence starts with kOverhead empty units, the price of starting and
// ending it in steps, so that a group with many short ones gets fewer bytes.
// A worker whose share starts or ends inside a sequence writes that piece's
// unnormalised (o, m, l) to the scratch: at most two pieces a worker, so the
// scratch does not grow with the lengths.  A second launch joins the pieces of
// the sequences that were cut and fills the rows that see nothing.
//
// A warp streams its positions through a cp.async ring of its own and meets no
// other warp: the ring runs on into the next sequence while one ends.
// The products are S^T = K Q^T and O^T = V^T P^T on mma.m16n8k16: 16 positions
// (or dimensions) by 8 query heads, so a group of up to 8 heads fills the tile
// (16 heads: two of them on the same K and V fragments), and P^T is S^T's
// accumulator transposed by movmatrix.  With the heads as the 16 rows instead,
// half of every product, exponential and rescaling of a group of 8 would be of
// rows that do not exist; the 128-row tcgen05 tile would be 94 % empty.
//
// Rounding.  K and V enter the products as they are.  q (fp32) is scaled per
// row by a power of two and split into 2 terms for an fp16 cache (22 bits) or
// 3 for a bf16 cache (24 bits); the probabilities, times 2^14 so that small
// ones keep their bits in fp16, into 2 terms (3 where the output is fp32 and
// the cache bf16).  A step's P V is summed on its own and added in fp32: the
// tensor cores' accumulation cuts instead of rounding, which over a long row
// would pull the output towards zero.  Sums, maxima and outputs are fp32,
// rounded once at the end.
//
// Measured (8 KV heads of 128, HBM copies run at 6.5 TB/s): 8 x 32K, fp32 rows,
// 32 heads: 159 us, 6.7 TB/s; 64 sequences of 16 .. 16384, bf16, 64 heads: 111 us,
// 5.8 TB/s, the ragged ends and 4 us of joining being the rest; 1 x 4K: 11.5 us,
// two launches and a chain of dependent loads (lengths, pages, K and V, pieces).
// Rows of one sequence (a prompt's) are rows like any other: each reads its
// positions for itself (2048 rows of one prompt, 64 heads, bf16: 1057 us, 8.6 GB
// asked for, mostly of L2).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

constexpr int kOverhead = 4;    // units' worth of starting and ending a sequence
constexpr int kMinUnits = 2;    // a group's share, at least (overhead counted)
constexpr long long kMaxLen = 0x7fffffffLL - 63;  // so that a step's positions are ints
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinRows = 1024;  // rows of one joining CTA, at most
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 16384.0f;  // probabilities enter P V times 2^14

struct PagedArgs {
    const void* q;
    const uint16_t *k, *v;
    const int32_t *table, *lens, *req;
    void* out;
    float* lse;
    float* part;   // [workers][2][heads][hd + 2]: o, m (log2 units), l
    const float* slopes;
    int64_t q_stride, out_stride, table_stride, page_stride, pos_stride, head_stride;
    int batch, nh, nkv, grp, heads, rt, hd, page_size, page_shift, n_pages, max_pages, n_req;
    int len_add, window, groups, sms;
    // heads: query heads of one unit (8 or 16); rt: blocks of that many in a group;
    // page_shift: log2 of the page size, or -1
    int q_pairs;   // q's rows can be read two elements at a time
    float scale, softcap;
};

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

template <bool EARLY = false>
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
    Seq s;
    s.tr = a.req ? word<EARLY>(a.req + b) : b;
    const long long len = (long long)word<EARLY>(a.lens + b) + a.len_add;
    const bool none = s.tr < 0 || len <= 0;
    s.bad = !none && (s.tr >= a.n_req || len > (long long)a.max_pages * a.page_size || len > kMaxLen);
    s.len = none || s.bad ? 0 : (int)len;
    s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
    return s;
}

// steps of sequence s, positions [lo, len), of `step` positions (16 or 32)
__device__ __forceinline__ int steps_of(const Seq& s, int step) {
    const int sh = step == 16 ? 4 : 5;
    return s.len == 0 ? 0 : ((s.len - 1) >> sh) - (s.lo >> sh) + 1;
}
// units of sequence s: its steps behind the overhead
__device__ __forceinline__ int units_of(const Seq& s, int step) {
    return s.len == 0 ? 0 : steps_of(s, step) + kOverhead;
}

__device__ __forceinline__ void cp16(uint32_t smem, const void* gmem, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t* r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
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

__device__ __forceinline__ float2 pair_of(const float* p, bool pairs) {
    return pairs ? *reinterpret_cast<const float2*>(p) : make_float2(p[0], p[1]);
}
__device__ __forceinline__ float2 pair_of(const __half* p, bool pairs) {
    return pairs ? __half22float2(*reinterpret_cast<const __half2*>(p)) : make_float2(__half2float(p[0]), __half2float(p[1]));
}
__device__ __forceinline__ float2 pair_of(const __nv_bfloat16* p, bool pairs) {
    return pairs ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p))
                 : make_float2(__bfloat162float(p[0]), __bfloat162float(p[1]));
}

// (x * y + add) / z, none negative, exact; in 32 bits where they do (a 64-bit
// division is some 100 instructions)
__device__ __forceinline__ long long mul_div(long long x, long long y, long long z, int add = 0) {
    const long long p = x * y + add;
    return (p | z) <= 0xffffffffLL ? (long long)((unsigned)p / (unsigned)z) : p / z;
}

// How many groups share W units; group g has the units from mul_div(g, W, G) on.
__device__ __forceinline__ long long groups_for(const PagedArgs& a, long long W) {
    return max(1LL, min((long long)a.groups, mul_div(W, 1, kMinUnits)));
}

// A worker's place in its units: step `step` of the `ns` of row b, up to `end`
// of which are its share; `left` units of its share lie behind this row.
template <int STEP>
struct Cursor {
    Seq sq;
    int b, ns, step, end;
    long long left;

    // takes this row's part of `left` units, from unit x of the row on
    __device__ __forceinline__ void enter(int x) {
        const long long take = min((long long)(ns + kOverhead - x), left);
        left -= take;
        step = max(0, x - kOverhead);
        end = max(0, (int)(x + take) - kOverhead);
    }
    // on to the worker's next step; false when there is none
    __device__ __forceinline__ bool settle(const PagedArgs& a) {
        while (step >= end) {
            if (left <= 0) return false;
            do {
                sq = seq_of(a, ++b);
                ns = steps_of(sq, STEP);
            } while (ns == 0);
            enter(0);
        }
        return true;
    }
};

template <int HD, int NG>
struct Sm {
    // 32 positions a step, as two products side by side, hide each other's
    // latencies (8 x 32K of head dimension 64: 131 us with 16, 94 with 32); with
    // head dimension 256 or 16 query heads the registers are better kept for two
    // warps a scheduler (32K x 16 of 16 heads: 69 us with 32, 61 with 16).
    static constexpr int kSub = HD > 128 || NG > 1 ? 1 : 2;
    static constexpr int kStep = 16 * kSub;
    // The copies in flight are what the ring holds beyond the step at work.
    // 64 KB an SM is enough for the full rate, and more is worse: the SMs then
    // get unequal shares of the bandwidth (8 x 32K with 128 KB: 178 us, the first
    // SM done after 132, the last after 175; with 64 KB 162 us).
    static constexpr int kStages = 2;
    static constexpr int kWarps = 4;
    static constexpr int kCtas = HD > 128 ? 1 : HD == 128 && NG == 1 ? 1 : 2;  // of an SM
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kRow = HD * 2;
    static constexpr int kStage = 2 * kStep * kRow;  // a warp's K and V rows of one step
    static constexpr int kWarp = kStages * kStage;
    static constexpr int kTotal = kWarps * kWarp;
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// T: the type of q and out; C: the cache's; QT, PT: terms of q and of the
// probabilities; NG: blocks of 8 query heads.
template <int HD, typename T, typename C, int QT, int PT, int NG>
__global__ void __launch_bounds__(Sm<HD, NG>::kThreads) paged_split_kernel(const __grid_constant__ PagedArgs a) {
    using SM = Sm<HD, NG>;
    constexpr int KS = HD / 16, ST = SM::kStages, SUB = SM::kSub, STEP = SM::kStep, kHeads = 8 * NG;
    constexpr int kWarps = SM::kWarps, kThreads = SM::kThreads;
    extern __shared__ __align__(1024) uint8_t psm[];
    __shared__ long long wsum[kWarps];
    __shared__ long long chunk[kThreads];  // units before the end of each thread's sequences
    pdl_wait();
    pdl_trigger();  // (behind the wait, in every thread: the joining launch reads the lengths before its own)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gi = lane >> 2, ti = lane & 3;
    const int hd = a.hd, hc = hd / 8, rpb = a.nkv * a.rt;
    uint8_t* const ring = psm + warp * SM::kWarp;

    // columns past hd stay zero: the copies never write them
    if (hd < HD)
        for (int i = lane; i < SM::kWarp / 16; i += 32) *reinterpret_cast<uint4*>(ring + 16 * i) = make_uint4(0, 0, 0, 0);

    // the units before each sequence, by a scan over the lengths
    const int per = (a.batch + kThreads - 1) / kThreads;
    {
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        long long inc = 0;
        for (int b = b0; b < b1; b++) inc += units_of(seq_of(a, b), STEP);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++)
            if (w < warp) inc += wsum[w];
        chunk[tid] = inc;
    }
    __syncthreads();
    const long long W = chunk[kThreads - 1];
    const long long G = groups_for(a, W);
    const int worker = warp * gridDim.x + blockIdx.x;  // neighbours on different SMs
    const int group = worker / rpb, hr = worker - group * rpb;
    if (group >= G || W == 0) return;
    const long long u0 = mul_div(group, W, G), u1 = mul_div(group + 1, W, G);
    Cursor<STEP> ld;
    {
        int c = 0;  // the thread whose sequences hold u0
#pragma unroll
        for (int j = 0; j < kThreads / 32; j++) c += __popc(__ballot_sync(0xffffffffu, chunk[j * 32 + lane] <= u0));
        long long base = c ? chunk[c - 1] : 0;
        int b = c * per;
        while (true) {
            ld.sq = seq_of(a, b);
            const int n = units_of(ld.sq, STEP);
            if (u0 < base + n) break;
            base += n;
            b++;
        }
        ld.b = b;
        ld.ns = steps_of(ld.sq, STEP);
        ld.left = u1 - u0;
        ld.enter((int)(u0 - base));
    }
    const int h = hr / a.rt, row0 = (hr - h * a.rt) * kHeads;  // KV head, first query head of the group
    const int heads = min(kHeads, a.grp - row0), head0 = h * a.grp + row0;
    const int64_t h_off = (int64_t)h * a.head_stride;
    bool more = ld.settle(a);  // the loading side has a step
    if (!more) return;         // (overhead alone)
    Cursor<STEP> cu = ld;

    const uint32_t ring_s = smem_u32(ring);
    // ldmatrix places of this lane in a stage, K as A (positions x dims) and V^T as
    // A (dims x positions): chunk 2 i + c of row r is at (place of chunk c) ^ 32 i
    const int k_row = lane & 15, k_c = lane >> 4;
    const int v_row = (lane & 7) + ((lane >> 4) & 1) * 8, v_c = (lane >> 3) & 1;
    const uint32_t k_at = k_row * SM::kRow + ((k_c ^ (k_row & 7)) << 4), v_at = v_row * SM::kRow + ((v_c ^ (v_row & 7)) << 4);
    // copies: row r0 + j LR, chunk c of each; chunk c of row r goes to c ^ (r & 7)
    constexpr int LR = 32 / (HD / 8);  // rows one warp copy covers
    const int c_c = lane % (HD / 8), c_r = lane / (HD / 8);
    const uint32_t c_at = c_r * SM::kRow + ((c_c ^ c_r) << 4);
    const bool c_in = c_c < hc, one_page = a.page_size % 16 == 0;
    const int64_t v_off = a.v - a.k;

    // The loading side: fetch looks up the page of this lane's row (lane & 15)
    // of a step two steps before issue copies the step's rows.
    struct Place {
        int64_t off;  // the row's place in its page; -1: a position that is not seen
        int page;
        bool live, full;  // a step; all of it seen, every 16 rows in one page
    };
    auto fetch = [&]() {
        Place f{-1, -1, more, false};
        if (more) {
            const int first = (ld.sq.lo / STEP + ld.step) * STEP, p = first + (lane & (STEP - 1));
            f.full = one_page && first >= ld.sq.lo && first + STEP <= ld.sq.len;
            if (p >= ld.sq.lo && p < ld.sq.len) {
                const int pg = a.page_shift >= 0 ? p >> a.page_shift : p / a.page_size;
                f.page = a.table[(int64_t)ld.sq.tr * a.table_stride + pg];
                f.off = (int64_t)(p - pg * a.page_size) * a.pos_stride + h_off;
            }
            ld.step++;
            more = ld.settle(a);
        }
        return f;
    };
    uint32_t bad_slots = 0;
    auto issue = [&](int slot, const Place& f) {
        if (f.live) {
            const bool seen = f.off >= 0;
            const bool ok = seen && (unsigned)f.page < (unsigned)a.n_pages;
            const uint32_t bad = __ballot_sync(0xffffffffu, seen && !ok);
            bad_slots = (bad_slots & ~(1u << slot)) | (bad ? 1u << slot : 0u);
            const uint32_t kt = ring_s + slot * SM::kStage + c_at;
            const int64_t off = ok ? f.page * a.page_stride + f.off : -1;
            if (f.full && !bad) {  // 16 rows follow each other by pos_stride
                const int64_t at0 = c_r * a.pos_stride + c_c * 8, next = LR * a.pos_stride;
#pragma unroll
                for (int sub = 0; sub < SUB; sub++) {
                    const uint16_t* k = a.k + (__shfl_sync(0xffffffffu, off, 16 * sub) + at0);
                    if (c_in) {
#pragma unroll
                        for (int j = 0; j < 16 / LR; j++) {
                            const uint32_t at = (kt ^ (((j * LR) & 7) << 4)) + (16 * sub + j * LR) * SM::kRow;
                            cp16(at, k, true);
                            cp16(at + STEP * SM::kRow, k + v_off, true);
                            k += next;
                        }
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < STEP / LR; j++) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, c_r + j * LR);
                    const uint32_t at = (kt ^ (((j * LR) & 7) << 4)) + j * LR * SM::kRow;
                    if (c_in) {
                        const uint16_t* k = a.k + ((o < 0 ? 0 : o) + c_c * 8);
                        cp16(at, k, o >= 0);
                        cp16(at + STEP * SM::kRow, k + v_off, o >= 0);
                    }
                }
            }
        }
        cp_async_commit();
    };
    Place f0 = fetch(), f1 = fetch();
#pragma unroll 1
    for (int i = 0; i < ST - 1; i++) {
        const Place f2 = fetch();
        issue(i, f0);
        f0 = f1;
        f1 = f2;
    }

    int slot = 0;
    while (true) {
        // a sequence begins
        const int first = cu.step, lo = cu.sq.lo, len = cu.sq.len;
        uint32_t qf[NG][KS][QT][2];  // B fragments: head gi, dims 16 kk + 2 ti + {0, 1} and + 8
        float ks[NG][2], sl[NG][2];  // heads 2 ti, 2 ti + 1 of each block: score factor, slope
        const float cap = a.softcap;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const bool v = 8 * g + gi < heads, pairs = a.q_pairs;
            const T* q0 = static_cast<const T*>(a.q) + (int64_t)cu.b * a.q_stride +
                          (int64_t)(head0 + (v ? 8 * g + gi : 0)) * hd;
            float x[KS][4];
#pragma unroll
            for (int kk = 0; kk < KS; kk++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int c = 16 * kk + 2 * ti + 8 * j;
                    const float2 t = v && c < hd ? pair_of(q0 + c, pairs) : make_float2(0.0f, 0.0f);
                    x[kk][2 * j] = t.x;
                    x[kk][2 * j + 1] = t.y;
                }
            float up = 1.0f, factor = a.scale;
            if (QT > 1) {  // the row's largest element to [2^10, 2^11); a single term is q itself
                float m = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KS; kk++)
#pragma unroll
                    for (int j = 0; j < 4; j++) m = fmaxf(m, fabsf(x[kk][j]));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                // (the exponent field is enough: subnormal rows count as 2^-127; down to
                // -117 for the largest finite row, so that both factors stay normal)
                const int e = m < INFINITY ? min(100, 137 - (int)(__float_as_uint(m) >> 23)) : 0;
                up = __int_as_float((127 + e) << 23);
                factor *= __int_as_float((127 - e) << 23);
            }
#pragma unroll
            for (int kk = 0; kk < KS; kk++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    uint32_t w[QT];
                    split_terms<C, QT>(x[kk][2 * j] * up, x[kk][2 * j + 1] * up, w);
#pragma unroll
                    for (int i = 0; i < QT; i++) qf[g][kk][i][j] = w[i];
                }
            factor = cap > 0.0f ? factor / cap : factor * kLog2e;  // scores in log2 units
#pragma unroll
            for (int j = 0; j < 2; j++) {
                ks[g][j] = __shfl_sync(0xffffffffu, factor, 4 * (2 * ti + j));
                const int head = 8 * g + 2 * ti + j;
                sl[g][j] = a.slopes && head < heads ? __ldg(a.slopes + head0 + head) * kLog2e : 0.0f;
            }
        }

        unsigned long long o[NG][KS][2];  // dims 16 i + gi and + 8; heads 2 ti, 2 ti + 1 as a pair
        float m[NG][2], l[NG][2];
#pragma unroll
        for (int g = 0; g < NG; g++) {
#pragma unroll
            for (int i = 0; i < KS; i++) o[g][i][0] = o[g][i][1] = 0;
            m[g][0] = m[g][1] = -INFINITY;
            l[g][0] = l[g][1] = 0.0f;
        }
        bool bad = false;

#pragma unroll 1
        for (; cu.step < cu.end; cu.step++) {
            const Place f2 = fetch();
            issue(slot == 0 ? ST - 1 : slot - 1, f0);
            f0 = f1;
            f1 = f2;
            cp_wait<ST - 1>();
            __syncwarp();
            const uint32_t kt = ring_s + slot * SM::kStage, vt = kt + STEP * SM::kRow;
            bad |= (bad_slots >> slot) & 1;
            slot = slot == ST - 1 ? 0 : slot + 1;
            const int p0 = (lo / STEP + cu.step) * STEP;
            // one accumulator per term of q: short chains, and the terms below the
            // first stay out of a score that an infinite key made infinite (0 * inf)
            float st[SUB][NG][QT][4], sp[SUB][NG][4];
#pragma unroll
            for (int kk = 0; kk < KS; kk++)
#pragma unroll
                for (int sub = 0; sub < SUB; sub++) {
                    uint32_t ak[4];
                    ldsm(((kt + k_at) ^ (kk * 32)) + sub * 16 * SM::kRow, ak);
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int t = 0; t < QT; t++) {
                            // (fp32 rows: the first term is summed 64 dimensions at a time, the sums
                            // added in fp32, which rounds where the tensor cores' accumulation cuts)
                            const bool parts = QT > 1 && t == 0 && kk >= 4;
                            float* d = parts ? sp[sub][g] : st[sub][g][t];
                            if (kk == 0 || (parts && kk % 4 == 0)) Cvt<C>::mma0(d, ak, qf[g][kk][t][0], qf[g][kk][t][1]);
                            else Cvt<C>::mma(d, ak, qf[g][kk][t][0], qf[g][kk][t][1]);
                            if (parts && (kk % 4 == 3 || kk == KS - 1)) {
#pragma unroll
                                for (int j = 0; j < 4; j++) st[sub][g][0][j] += sp[sub][g][j];
                            }
                        }
                }
            uint32_t pb[SUB][NG][PT][2];
            unsigned long long fo2[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) {
                // positions p0 + 16 sub + gi (values 0, 1) and + 8 (2, 3); heads 2 ti, 2 ti + 1
                float s[SUB][4];
#pragma unroll
                for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float top = st[sub][g][0][j];
                        float low = 0.0f;
#pragma unroll
                        for (int t = QT - 1; t > 0; t--) low += st[sub][g][t][j];
                        s[sub][j] = (QT > 1 && fabsf(top) == INFINITY ? top : top + low) * ks[g][j & 1];
                    }
                if (cap > 0.0f) {
#pragma unroll
                    for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                        for (int j = 0; j < 4; j++) s[sub][j] = (cap * kLog2e) * tanhf(s[sub][j]);
                }
                if (a.slopes) {
#pragma unroll
                    for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            s[sub][j] = fmaf(sl[g][j & 1], (float)(p0 + 16 * sub + gi + (j & 2) * 4 - (len - 1)), s[sub][j]);
                }
                if (p0 < lo || p0 + STEP > len) {
#pragma unroll
                    for (int sub = 0; sub < SUB; sub++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int p = p0 + 16 * sub + gi + (j & 2) * 4;
                            if (p < lo || p >= len) s[sub][j] = -INFINITY;
                        }
                }
                float fo[2], z[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float r = fmaxf(s[0][j], s[0][j + 2]);
#pragma unroll
                    for (int sub = 1; sub < SUB; sub++) r = fmaxf(r, fmaxf(s[sub][j], s[sub][j + 2]));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 4));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 8));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 16));
                    const float n = fmaxf(m[g][j], r);
                    z[j] = n == -INFINITY ? 0.0f : n;  // (a row whose scores are all -inf so far keeps weight zero)
                    fo[j] = ex2(m[g][j] - z[j]);
                    m[g][j] = n;
                    l[g][j] *= fo[j];
                }
                fo2[g] = f2_pack(fo[0], fo[1]);
#pragma unroll
                for (int sub = 0; sub < SUB; sub++) {
                    float p[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) p[j] = ex2(s[sub][j] - z[j & 1]) * kPScale;
                    l[g][0] += p[0] + p[2];
                    l[g][1] += p[1] + p[3];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        uint32_t t[PT];
                        split_terms<C, PT>(p[2 * j], p[2 * j + 1], t);
#pragma unroll
                        for (int x = 0; x < PT; x++) pb[sub][g][x][j] = transpose8x8(t[x]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < KS; i++) {
                float t[NG][4];
#pragma unroll
                for (int sub = 0; sub < SUB; sub++) {
                    uint32_t av[4];
                    ldsm_t(((vt + v_at) ^ (i * 32)) + sub * 16 * SM::kRow, av);
#pragma unroll
                    for (int g = 0; g < NG; g++)
#pragma unroll
                        for (int x = PT - 1; x >= 0; x--) {
                            if (sub == 0 && x == PT - 1) Cvt<C>::mma0(t[g], av, pb[sub][g][x][0], pb[sub][g][x][1]);
                            else Cvt<C>::mma(t[g], av, pb[sub][g][x][0], pb[sub][g][x][1]);
                        }
                }
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    o[g][i][0] = f2_fma(o[g][i][0], fo2[g], f2_pack(t[g][0], t[g][1]));
                    o[g][i][1] = f2_fma(o[g][i][1], fo2[g], f2_pack(t[g][2], t[g][3]));
                }
            }
            __syncwarp();  // the slot is refilled by the next step's issue
        }

        const bool from_start = first == 0, to_end = cu.end == cu.ns, whole = from_start && to_end;
        auto val = [&](int g, int i, int half, int j) {
            const float2 x = f2_unpack(o[g][i][half]);
            return j ? x.y : x.x;
        };
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float x = l[g][j], y = m[g][j];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (bad) x = y = __int_as_float(0x7fc00000);  // a page that is not there
                const int head = 8 * g + 2 * ti + j;
                if (head >= heads) continue;
                if (whole) {
                    const float inv = x == 0.0f ? 0.0f : 1.0f / x;
                    T* out = static_cast<T*>(a.out) + (int64_t)cu.b * a.out_stride + (int64_t)(head0 + head) * hd;
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        const int d = 16 * i + gi;
                        if (d < hd) out[d] = (T)(val(g, i, 0, j) * inv);
                        if (d + 8 < hd) out[d + 8] = (T)(val(g, i, 1, j) * inv);
                    }
                    if (a.lse && gi == 0)
                        a.lse[(int64_t)cu.b * a.nh + head0 + head] = x == 0.0f ? -INFINITY : (y + (log2f(x) - 14.0f)) * kLn2;
                } else {
                    float* part = a.part + ((int64_t)(2 * worker + (from_start ? 1 : 0)) * kHeads + head) * (hd + 2);
#pragma unroll
                    for (int i = 0; i < KS; i++) {
                        const int d = 16 * i + gi;
                        if (d < hd) part[d] = val(g, i, 0, j);
                        if (d + 8 < hd) part[d + 8] = val(g, i, 1, j);
                    }
                    if (gi == 0) *reinterpret_cast<float2*>(part + hd) = make_float2(y, x);
                }
            }
        if (!cu.settle(a)) break;
    }
    cp_wait<0>();
}

// CTAs (rows, blockIdx.y): each has a run of neighbouring rows (one row while
// there are no more rows than CTAs), the y shares taking the query heads in
// turn: join the pieces of a row that was cut, and fill a row that sees nothing
// (zeros, lse -inf) or whose length passes its table (NaN).  The 8 warps are 8 /
// PW heads times PW shares of the pieces; a lane holds ND pairs of a head (hd <=
// 64 ND).  PW = 8 is for few heads, one to a CTA, PW = 1 for many.  Which groups
// hold a row's pieces follows from the lengths, worked out while the split
// kernel still runs: every CTA walks all lengths once, so their number is
// bounded (16 sequences of 2001 among 65536 rows: 7.5 ms with a CTA for each
// row, 0.71 with 8 an SM; the same among 1024: 43 us, 50 with 4 an SM, which
// puts two of them in one CTA; 20000 short rows: 218 us, 258 with 16 an SM).
template <typename T, int ND, int PW>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedArgs a, int step) {
    __shared__ __align__(8) float red[kJoinWarps][kPagedMaxHd + 2];
    __shared__ long long sums[2][kJoinWarps];
    struct Todo {
        int row, first, last, kind;  // the row's groups; what it is
    };
    enum { kCut, kEmpty, kBad };
    __shared__ Todo todo[kJoinRows];
    __shared__ int n_todo;
    pdl_trigger();
    if (threadIdx.x == 0) n_todo = 0;
    const int rpb = a.nkv * a.rt, hd = a.hd, nh = a.nh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = warp % PW;
    constexpr int rw = kJoinWarps / PW;
    const float nan = __int_as_float(0x7fc00000);
    const unsigned rows = a.batch, run = rows / gridDim.x, more = rows - run * gridDim.x;
    const unsigned b0 = blockIdx.x * run + min(blockIdx.x, more), b1 = b0 + run + (blockIdx.x < more);
    // (the lengths' writer has ended: the split kernel waited for it before it let this one start)
    long long before = 0, all = 0;  // units before row b0, and of all rows
    for (unsigned i = tid; i < rows; i += kJoinThreads) {
        const int n = units_of(seq_of<true>(a, i), step);
        all += n;
        if (i < b0) before += n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        before += __shfl_xor_sync(0xffffffffu, before, o);
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    if (lane == 0) {
        sums[0][warp] = before;
        sums[1][warp] = all;
    }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < kJoinWarps; w++) {
        before += sums[0][w];
        all += sums[1][w];
    }
    // a head's place among the workers: KV head, block of its group, row of the block
    const int64_t ps = (int64_t)a.heads * (hd + 2);  // floats of a piece; a group's are 2 rpb pieces apart
    auto place = [&](int head) {
        const int h = head / a.grp, in = head - h * a.grp, blk = in / a.heads;
        return a.part + (int64_t)2 * (h * a.rt + blk) * ps + (in - blk * a.heads) * (hd + 2);
    };
    const int first0 = blockIdx.y * rw;
    const float* const base0 = place(first0 + warp / PW);  // (worked out before the wait)

#pragma unroll 1
    for (unsigned at = b0; at < b1; at += kJoinThreads) {
        // a row to a thread: its units, those before it, its groups
        const unsigned b = at + tid;
        Seq sq{};
        if (b < b1) sq = seq_of<true>(a, b);
        const int n = units_of(sq, step);
        long long end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += t;
        }
        __syncthreads();  // (the sums were read)
        if (lane == 31) sums[0][warp] = end;
        __syncthreads();
        long long rows_units = 0;
#pragma unroll
        for (int w = 0; w < kJoinWarps; w++) {
            if (w < warp) end += sums[0][w];
            rows_units += sums[0][w];
        }
        if (b < b1) {
            Todo t{(int)b, 0, 0, sq.bad ? kBad : kEmpty};
            if (sq.len) {  // the group of unit u: floor(((u + 1) G - 1) / W)
                const long long G = groups_for(a, all), u = before + end - n;
                t.first = (int)mul_div(u + kOverhead + 1, G, all, -1);
                t.last = (int)mul_div(u + n, G, all, -1);
                t.kind = kCut;
            }
            if (t.kind != kCut || t.first != t.last) todo[atomicAdd(&n_todo, 1)] = t;
        }
        before += rows_units;
    }
    __syncthreads();
    pdl_wait();
#pragma unroll 1
    for (int e = 0; e < n_todo; e++) {
        const Todo t = todo[e];
        const float* base = base0;
        // (once where PW > 1)
#pragma unroll 1
        for (int first = first0; first < nh; first += gridDim.y * rw, base = place(first + warp / PW)) {
            const int head = first + warp / PW;
            const bool live = head < nh;
            constexpr int NP = ND <= 2 ? 8 : 4;  // pieces in flight
            float2 o[ND];
            float M = -INFINITY, L = 0.0f;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < ND; j++) o[j] = make_float2(0.0f, 0.0f);
            if (live && t.kind == kCut) {
                for (int i0 = t.first + share; i0 <= t.last; i0 += NP * PW) {
                    float2 ml[NP], x[NP][ND];
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        const int i = i0 + k * PW;
                        const float* p = base + (2 * (int64_t)i * rpb + (i == t.first ? 1 : 0)) * ps;
                        ml[k] = i <= t.last ? *reinterpret_cast<const float2*>(p + hd) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                        for (int j = 0; j < ND; j++) {
                            const int d = 2 * lane + 64 * j;
                            x[k][j] = i <= t.last && d < hd ? *reinterpret_cast<const float2*>(p + d) : make_float2(0.0f, 0.0f);
                        }
                    }
                    float N = M;
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        bad |= ml[k].x != ml[k].x;
                        N = fmaxf(N, ml[k].x);
                    }
                    const float z = N == -INFINITY ? 0.0f : N, f = ex2(M - z);
                    M = N;
                    L *= f;
#pragma unroll
                    for (int j = 0; j < ND; j++) {
                        o[j].x *= f;
                        o[j].y *= f;
                    }
#pragma unroll
                    for (int k = 0; k < NP; k++) {
                        const float w = ex2(ml[k].x - z);
                        L = fmaf(ml[k].y, w, L);
#pragma unroll
                        for (int j = 0; j < ND; j++) {
                            o[j].x = fmaf(x[k][j].x, w, o[j].x);
                            o[j].y = fmaf(x[k][j].y, w, o[j].y);
                        }
                    }
                }
                if (bad) M = L = nan;
            }
            if constexpr (PW > 1) {  // the shares of a head meet in its first warp
#pragma unroll
                for (int j = 0; j < ND; j++)
                    if (2 * lane + 64 * j < hd) *reinterpret_cast<float2*>(&red[warp][2 * lane + 64 * j]) = o[j];
                if (lane == 0) *reinterpret_cast<float2*>(&red[warp][kPagedMaxHd]) = make_float2(M, L);
                __syncthreads();
                if (share == 0) {
                    float N = M;
                    bool any = M != M;
                    for (int w = 1; w < PW; w++) {
                        const float m = red[warp + w][kPagedMaxHd];
                        any |= m != m;
                        N = fmaxf(N, m);
                    }
                    const float z = N == -INFINITY ? 0.0f : N, f = ex2(M - z);
                    L *= f;
#pragma unroll
                    for (int j = 0; j < ND; j++) {
                        o[j].x *= f;
                        o[j].y *= f;
                    }
                    for (int w = 1; w < PW; w++) {
                        const float2 ml = *reinterpret_cast<const float2*>(&red[warp + w][kPagedMaxHd]);
                        const float g = ex2(ml.x - z);
                        L = fmaf(ml.y, g, L);
#pragma unroll
                        for (int j = 0; j < ND; j++)
                            if (2 * lane + 64 * j < hd) {
                                const float2 x = *reinterpret_cast<const float2*>(&red[warp + w][2 * lane + 64 * j]);
                                o[j].x = fmaf(x.x, g, o[j].x);
                                o[j].y = fmaf(x.y, g, o[j].y);
                            }
                    }
                    M = any ? nan : N;
                    if (any) L = nan;
                }
                __syncthreads();
            }
            if (live && share == 0) {
                if (t.kind == kBad) M = L = nan;
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                T* out = static_cast<T*>(a.out) + (int64_t)t.row * a.out_stride + (int64_t)head * hd;
#pragma unroll
                for (int j = 0; j < ND; j++) {
                    const int d = 2 * lane + 64 * j;
                    if (d < hd) {
                        out[d] = (T)(o[j].x * inv);
                        out[d + 1] = (T)(o[j].y * inv);
                    }
                }
                if (a.lse && lane == 0)
                    a.lse[(int64_t)t.row * nh + head] = L == 0.0f ? -INFINITY : (M + (log2f(L) - 14.0f)) * kLn2;
            }
            if (PW > 1) break;
        }
    }
}

constexpr int kMaxPagedDevices = 64;

template <int HD, typename T, typename C, int QT, int PT, int NG>
cudaError_t go(const PagedArgs& a, cudaStream_t s) {
    static std::atomic<bool> attr[kMaxPagedDevices] = {};  // the attribute belongs to a device
    using SM = Sm<HD, NG>;
    constexpr int smem = SM::kTotal;
    auto kern = paged_split_kernel<HD, T, C, QT, PT, NG>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxPagedDevices || !attr[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxPagedDevices) attr[dev] = true;
    }
    e = launch_pdl(kern, dim3((a.groups * a.nkv * a.rt + SM::kWarps - 1) / SM::kWarps), dim3(SM::kThreads), smem, s, a);
    if (e != cudaSuccess) return e;
    // few heads in all: a CTA for each, its pieces over the 8 warps; many: a warp
    // for each, a CTA for each row while there are up to 8 an SM of them
    if ((long long)a.batch * a.nh <= 2 * a.sms)
        return launch_pdl(paged_join_kernel<T, HD / 64, kJoinWarps>, dim3(a.batch, a.nh), dim3(kJoinThreads), 0, s, a,
                          SM::kStep);
    const int ctas = std::min(a.batch, std::max(8 * a.sms, (a.batch - 1) / kJoinRows + 1));
    const int y = std::max(1, std::min((a.nh + kJoinWarps - 1) / kJoinWarps, 4 * a.sms / ctas));
    return launch_pdl(paged_join_kernel<T, HD / 64, 1>, dim3(ctas, y), dim3(kJoinThreads), 0, s, a, SM::kStep);
}

// Query heads of one unit: 16 for groups past 8, so that one pass over K and V
// serves them (32K x 16 of 16 heads of 128: 68 us with two units of 8, 57 with
// one of 16), up to head dimension 128.  Past that the fragments of q and O of
// 16 heads are more than the registers hold, and two units, whose rows meet in
// L2, are faster (16K x 16 of 16 heads of 256, 16-bit rows: 79 us; 88 with one).
int unit_heads(int hd, int grp) { return grp > 8 && hd <= 128 ? 16 : 8; }

template <int HD, typename T, typename C, int QT, int PT>
cudaError_t go_heads(const PagedArgs& a, cudaStream_t s) {
    if constexpr (HD <= 128) {
        if (a.heads == 16) return go<HD, T, C, QT, PT, 2>(a, s);
    }
    return go<HD, T, C, QT, PT, 1>(a, s);
}

template <int HD>
cudaError_t go_hd(const PagedArgs& a, int dtype, int cache, cudaStream_t s) {
    if (dtype == 0)
        return cache == 1 ? go_heads<HD, float, __half, 2, 2>(a, s) : go_heads<HD, float, __nv_bfloat16, 3, 3>(a, s);
    return cache == 1 ? go_heads<HD, __half, __half, 1, 2>(a, s) : go_heads<HD, __nv_bfloat16, __nv_bfloat16, 1, 2>(a, s);
}

// Groups of rpb workers each: as many as fit the machine at once.
template <int HD, int NG>
int groups_in(int rpb, int sms) {
    return std::max(1, Sm<HD, NG>::kCtas * Sm<HD, NG>::kWarps * sms / rpb);
}
int groups_of(int hd, int heads, int rpb, int sms) {
    const bool two = heads == 16;
    if (hd <= 64) return two ? groups_in<64, 2>(rpb, sms) : groups_in<64, 1>(rpb, sms);
    if (hd <= 128) return two ? groups_in<128, 2>(rpb, sms) : groups_in<128, 1>(rpb, sms);
    return groups_in<256, 1>(rpb, sms);
}

size_t part_bytes(int hd, int heads, int rpb, int sms) {
    return (size_t)groups_of(hd, heads, rpb, sms) * rpb * 2 * heads * (hd + 2) * sizeof(float);
}

}  // namespace

size_t attention_paged_scratch(int batch, int nh, int nkv, int hd, int sms) {
    const int grp = nh / nkv, heads = unit_heads(hd, grp);
    (void)batch;  // (the pieces are the workers', whatever the batch)
    return part_bytes(hd, heads, nkv * ((grp + heads - 1) / heads), sms);
}

int launch_attention_paged(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q, const int32_t* table,
                           const int32_t* lens, const int32_t* req, int batch, void* out, float* lse, void* scratch,
                           cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    PagedArgs a{};
    a.q = q;
    a.k = static_cast<const uint16_t*>(kv.k);
    a.v = static_cast<const uint16_t*>(kv.v);
    a.table = table;
    a.lens = lens;
    a.req = req;
    a.out = out;
    a.lse = lse;
    a.part = static_cast<float*>(scratch);
    a.grp = o.nh / kv.nkv;
    a.heads = unit_heads(kv.hd, a.grp);
    a.rt = (a.grp + a.heads - 1) / a.heads;
    a.slopes = o.slopes;
    const int64_t qd = (int64_t)o.nh * kv.hd;
    a.q_stride = o.q_stride ? o.q_stride : qd;
    a.out_stride = o.out_stride ? o.out_stride : qd;
    a.table_stride = o.table_stride ? o.table_stride : o.max_pages;
    a.page_stride = kv.page_stride;
    a.pos_stride = kv.pos_stride;
    a.head_stride = kv.head_stride;
    a.batch = batch;
    a.nh = o.nh;
    a.nkv = kv.nkv;
    a.hd = kv.hd;
    a.page_size = kv.page_size;
    a.page_shift = (kv.page_size & (kv.page_size - 1)) ? -1 : __builtin_ctz(kv.page_size);
    a.n_pages = kv.n_pages;
    a.max_pages = o.max_pages;
    a.n_req = o.n_req;
    a.len_add = o.len_add;
    a.window = o.window;
    a.groups = groups_of(kv.hd, a.heads, kv.nkv * a.rt, sms);
    a.sms = sms;
    const int es = o.dtype == 0 ? 4 : 2;
    a.q_pairs = a.q_stride % 2 == 0 && !(reinterpret_cast<uintptr_t>(q) & (2 * es - 1));
    a.scale = o.scale > 0.0f ? o.scale : (float)(1.0 / sqrt((double)kv.hd));
    a.softcap = o.softcap;
    const cudaError_t e = kv.hd <= 64    ? go_hd<64>(a, o.dtype, kv.dtype, s)
                          : kv.hd <= 128 ? go_hd<128>(a, o.dtype, kv.dtype, s)
                                         : go_hd<256>(a, o.dtype, kv.dtype, s);
    return e == cudaSuccess ? B2_OK : cuda_failed("paged attention launch", e, err);
}

}  // namespace b2
