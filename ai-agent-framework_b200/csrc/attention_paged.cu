// Attention of one query row per sequence over a paged KV cache, split over
// the cache's length and joined.
//
//   s_j = scale * q . k_j;  s_j <- cap * tanh(s_j / cap) (cap > 0);
//   s_j <- s_j + slope_h * (j - (len - 1)) (slopes given);
//   out = sum_j e^(s_j - M) v_j / sum_j e^(s_j - M) over the positions
//   max(0, len - window) <= j < len;  lse = M + log of the sum.
//
// HBM-bound: every visible K and V row is read once, from the page that holds
// it, whatever the number of query heads that share it.
//
// Split.  The work of the whole batch is one line of units, a unit being one
// step of kStep positions of one (sequence, KV head, block of query heads),
// and worker w of G, a warp, takes the units [w W / G, (w + 1) W / G).  Ragged
// batches thus load every SM equally without the host knowing a length, and
// a launch captured in a graph follows the lengths it finds.  Each row of
// units starts with kOverhead empty ones, the price of starting and ending a
// row in steps, so that a worker with many short sequences gets fewer bytes.
// A worker whose share starts or ends inside a row writes that piece's
// unnormalised (o, m, l) to the scratch: at most two pieces a worker, so the
// scratch does not grow with the lengths.  A second launch joins the pieces of
// the rows that were cut and fills the rows that see nothing.
//
// A warp streams its positions through a cp.async ring of its own and meets no
// other warp: the ring runs on into the next row's K and V while a row ends.
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
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreadsP = 32 * kWarps;
constexpr int kStep = 16;       // positions of one unit
constexpr int kOverhead = 4;    // units' worth of starting and ending a row
constexpr int kMinUnits = 6;    // a worker's share, at least (overhead counted)
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
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
    int2* desc;    // [batch * nkv * rt]: first and last worker of each row of units
    const float* slopes;
    int64_t q_stride, out_stride, table_stride, page_stride, pos_stride, head_stride;
    int batch, nh, nkv, grp, heads, rt, hd, page_size, page_shift, n_pages, max_pages, n_req, len_add, window, workers, sms;
    int q_pairs;   // q's rows can be read two elements at a time
    float scale, softcap;
};
// heads: query heads of one unit (8 or 16); rt: blocks of that many in a group.
// page_shift: log2 of the page size, or -1.

// A row's sequence: table row, visible positions [lo, len).  len 0: nothing.
struct Seq {
    int tr, lo, len;
    bool bad;  // the length passes the table
};

__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int b) {
    Seq s;
    s.tr = a.req ? __ldg(a.req + b) : b;
    const long long len = (long long)__ldg(a.lens + b) + a.len_add;
    const bool none = s.tr < 0 || len <= 0;
    s.bad = !none && (s.tr >= a.n_req || len > (long long)a.max_pages * a.page_size || len > 0x7fffffffLL);
    s.len = none || s.bad ? 0 : (int)len;
    s.lo = a.window > 0 ? max(0, s.len - a.window) : 0;
    return s;
}

__device__ __forceinline__ int steps_of(const Seq& s) { return s.len == 0 ? 0 : (s.len - 1) / kStep - s.lo / kStep + 1; }
// units of one row of sequence s: its steps behind the overhead
__device__ __forceinline__ int units_of(const Seq& s) { return s.len == 0 ? 0 : steps_of(s) + kOverhead; }

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
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
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
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
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

// x * y / z, exact; in 32 bits where they do (a 64-bit division is some 100 instructions)
__device__ __forceinline__ long long mul_div(long long x, long long y, long long z) {
    const long long p = x * y;
    return p <= 0xffffffffLL ? (long long)((unsigned)p / (unsigned)z) : p / z;
}

// A worker's place in its units: step `step` of `ns` of row `hr` of sequence
// b, `left` units after this row's, of which this row's share ends at `end`.
struct Cursor {
    Seq sq;
    int b, hr, ns, step, end;
    long long left;  // units of the worker behind this row

    // takes the row's share of `left` units from unit x of the row on
    __device__ __forceinline__ void enter(int x) {
        const int row = ns + kOverhead;
        const long long take = min((long long)(row - x), left);
        left -= take;
        step = max(0, x - kOverhead);
        end = max(0, (int)(x + take) - kOverhead);
    }
    __device__ __forceinline__ bool done() const { return step >= end; }
    // on to the worker's next step; false when there is none
    __device__ __forceinline__ bool settle(const PagedArgs& a, int rpb) {
        while (step >= end) {
            if (left <= 0) return false;
            if (++hr == rpb) {
                hr = 0;
                do {
                    sq = seq_of(a, ++b);
                    ns = steps_of(sq);
                } while (ns == 0);
            }
            enter(0);
        }
        return true;
    }
};

template <int HD>
struct Sm {
    static constexpr int kRow = HD * 2;
    static constexpr int kStages = HD == 64 ? 6 : 3;
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
__global__ void __launch_bounds__(kThreadsP) paged_split_kernel(const __grid_constant__ PagedArgs a) {
    using SM = Sm<HD>;
    constexpr int KS = HD / 16, ST = SM::kStages, kHeads = 8 * NG;
    extern __shared__ __align__(1024) uint8_t psm[];
    __shared__ long long wsum[kWarps];
    __shared__ long long chunk[kThreadsP];  // units before the end of each thread's sequences
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gi = lane >> 2, ti = lane & 3;
    const int hd = a.hd, hc = hd / 8, rpb = a.nkv * a.rt;
    uint8_t* const ring = psm + warp * SM::kWarp;

    // columns past hd stay zero: the copies never write them
    if (hd < HD)
        for (int i = lane; i < SM::kWarp / 16; i += 32) *reinterpret_cast<uint4*>(ring + 16 * i) = make_uint4(0, 0, 0, 0);

    // the units before each sequence, by a scan over the lengths
    const int per = (a.batch + kThreadsP - 1) / kThreadsP;
    {
        const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
        long long inc = 0;
        for (int b = b0; b < b1; b++) inc += units_of(seq_of(a, b));
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
        chunk[tid] = inc * rpb;
    }
    __syncthreads();
    const long long W = chunk[kThreadsP - 1];
    const long long G = max(1LL, min((long long)a.workers, mul_div(W, 1, kMinUnits)));
    const int worker = warp * gridDim.x + blockIdx.x;  // neighbours on different SMs
    if (worker >= G || W == 0) return;
    const long long u0 = mul_div(worker, W, G), u1 = mul_div(worker + 1, W, G);
    Cursor ld;
    {
        int c = 0;  // the thread whose sequences hold u0
#pragma unroll
        for (int j = 0; j < kThreadsP / 32; j++) c += __popc(__ballot_sync(0xffffffffu, chunk[j * 32 + lane] <= u0));
        long long base = c ? chunk[c - 1] : 0;
        int b = c * per;
        while (true) {
            ld.sq = seq_of(a, b);
            const long long n = (long long)units_of(ld.sq) * rpb;
            if (u0 < base + n) break;
            base += n;
            b++;
        }
        ld.b = b;
        ld.ns = steps_of(ld.sq);
        const int row = ld.ns + kOverhead;
        ld.hr = (int)mul_div(u0 - base, 1, row);
        ld.left = u1 - u0;
        ld.enter((int)((u0 - base) - (long long)ld.hr * row));
    }
    bool more = ld.settle(a, rpb);  // the loading side has a step
    if (!more) return;              // (overhead alone)
    Cursor cu = ld;

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
    const bool c_in = c_c < hc, one_page = a.page_size % kStep == 0;
    const int64_t v_off = a.v - a.k;

    // The loading side: fetch looks up the page of this lane's row (lane & 15)
    // of a step two steps before issue copies the step's rows.
    struct Place {
        int64_t off;  // the row's place in its page; -1: a position that is not seen
        int page;
        bool live, full;  // a step; all of it seen and in one page
    };
    auto fetch = [&]() {
        Place f{-1, -1, more, false};
        if (more) {
            const int first = (ld.sq.lo / kStep + ld.step) * kStep, p = first + (lane & (kStep - 1));
            f.full = one_page && first >= ld.sq.lo && first + kStep <= ld.sq.len;
            if (p >= ld.sq.lo && p < ld.sq.len) {
                const int pg = a.page_shift >= 0 ? p >> a.page_shift : p / a.page_size;
                f.page = __ldg(a.table + (int64_t)ld.sq.tr * a.table_stride + pg);
                f.off = (int64_t)(p - pg * a.page_size) * a.pos_stride + (int64_t)(ld.hr / a.rt) * a.head_stride;
            }
            ld.step++;
            more = ld.settle(a, rpb);
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
            if (f.full && !bad) {  // the rows follow each other by pos_stride
                const uint16_t* k = a.k + (__shfl_sync(0xffffffffu, off, 0) + c_r * a.pos_stride + c_c * 8);
                const int64_t next = LR * a.pos_stride;
                if (c_in) {
#pragma unroll
                    for (int j = 0; j < kStep / LR; j++) {
                        const uint32_t at = (kt ^ (((j * LR) & 7) << 4)) + j * LR * SM::kRow;
                        cp16(at, k, true);
                        cp16(at + kStep * SM::kRow, k + v_off, true);
                        k += next;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < kStep / LR; j++) {
                    const int64_t o = __shfl_sync(0xffffffffu, off, c_r + j * LR);
                    const uint32_t at = (kt ^ (((j * LR) & 7) << 4)) + j * LR * SM::kRow;
                    if (c_in) {
                        const uint16_t* k = a.k + ((o < 0 ? 0 : o) + c_c * 8);
                        cp16(at, k, o >= 0);
                        cp16(at + kStep * SM::kRow, k + v_off, o >= 0);
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
        // a row begins
        const int h = cu.hr / a.rt, row0 = (cu.hr - h * a.rt) * kHeads;  // KV head, first query head of the group
        const int heads = min(kHeads, a.grp - row0), head0 = h * a.grp + row0;
        const int first = cu.step, lo = cu.sq.lo, len = cu.sq.len;
        uint32_t qf[NG][KS][QT][2];  // B fragments: head gi, dims 16 kk + 2 ti + {0, 1} and + 8
        float ks[NG][2], sl[NG][2];  // heads 2 ti, 2 ti + 1 of each block: score factor, slope
        const float cap = a.softcap;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const bool v = 8 * g + gi < heads, pairs = a.q_pairs;
            const T* q0 = static_cast<const T*>(a.q) + (int64_t)cu.b * a.q_stride + (int64_t)(head0 + (v ? 8 * g + gi : 0)) * hd;
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
                // (the exponent field is enough: subnormal rows count as 2^-127)
                const int e = m < 3.0e38f ? min(100, max(-100, 137 - (int)(__float_as_uint(m) >> 23))) : 0;
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
                sl[g][j] = a.slopes && 8 * g + 2 * ti + j < heads ? __ldg(a.slopes + head0 + 8 * g + 2 * ti + j) * kLog2e : 0.0f;
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
            const uint32_t kt = ring_s + slot * SM::kStage, vt = kt + kStep * SM::kRow;
            bad |= (bad_slots >> slot) & 1;
            slot = slot == ST - 1 ? 0 : slot + 1;
            const int p0 = (lo / kStep + cu.step) * kStep;
            // one accumulator per term of q: short chains, and the terms below the
            // first stay out of a score that an infinite key made infinite (0 * inf)
            float st[NG][QT][4];
#pragma unroll
            for (int kk = 0; kk < KS; kk++) {
                uint32_t ak[4];
                ldsm((kt + k_at) ^ (kk * 32), ak);
#pragma unroll
                for (int g = 0; g < NG; g++)
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        if (kk == 0) Cvt<C>::mma0(st[g][t], ak, qf[g][kk][t][0], qf[g][kk][t][1]);
                        else Cvt<C>::mma(st[g][t], ak, qf[g][kk][t][0], qf[g][kk][t][1]);
                    }
            }
            uint32_t pb[NG][PT][2];
            unsigned long long fo2[NG];
#pragma unroll
            for (int g = 0; g < NG; g++) {
                // positions p0 + gi (values 0, 1) and + 8 (2, 3); heads 2 ti, 2 ti + 1
                float s[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float top = st[g][0][j];
                    float low = 0.0f;
#pragma unroll
                    for (int t = QT - 1; t > 0; t--) low += st[g][t][j];
                    s[j] = (QT > 1 && fabsf(top) == INFINITY ? top : top + low) * ks[g][j & 1];
                }
                if (cap > 0.0f) {
#pragma unroll
                    for (int j = 0; j < 4; j++) s[j] = (cap * kLog2e) * tanhf(s[j]);
                }
                if (a.slopes) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s[j] = fmaf(sl[g][j & 1], (float)(p0 + gi + (j & 2) * 4 - (len - 1)), s[j]);
                }
                if (p0 < lo || p0 + kStep > len) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int p = p0 + gi + (j & 2) * 4;
                        if (p < lo || p >= len) s[j] = -INFINITY;
                    }
                }
                float p[4], fo[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float r = fmaxf(s[j], s[j + 2]);
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 4));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 8));
                    r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, 16));
                    const float n = fmaxf(m[g][j], r);
                    const float z = n == -INFINITY ? 0.0f : n;  // (a row whose scores are all -inf so far keeps weight zero)
                    fo[j] = ex2(m[g][j] - z);
                    m[g][j] = n;
                    p[j] = ex2(s[j] - z) * kPScale;
                    p[j + 2] = ex2(s[j + 2] - z) * kPScale;
                    l[g][j] = fmaf(l[g][j], fo[j], p[j] + p[j + 2]);
                }
                fo2[g] = f2_pack(fo[0], fo[1]);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    uint32_t t[PT];
                    split_terms<C, PT>(p[2 * j], p[2 * j + 1], t);
#pragma unroll
                    for (int x = 0; x < PT; x++) pb[g][x][j] = transpose8x8(t[x]);
                }
            }
#pragma unroll
            for (int i = 0; i < KS; i++) {
                uint32_t av[4];
                ldsm_t((vt + v_at) ^ (i * 32), av);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    float t[4];
                    Cvt<C>::mma0(t, av, pb[g][PT - 1][0], pb[g][PT - 1][1]);
#pragma unroll
                    for (int x = PT - 2; x >= 0; x--) Cvt<C>::mma(t, av, pb[g][x][0], pb[g][x][1]);
                    o[g][i][0] = f2_fma(o[g][i][0], fo2[g], f2_pack(t[0], t[1]));
                    o[g][i][1] = f2_fma(o[g][i][1], fo2[g], f2_pack(t[2], t[3]));
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
        if (to_end && lane == 0) {
            // the worker that holds the row's first step: floor(((u + 1) G - 1) / W) of its unit u
            int c0 = worker;
            if (!from_start) c0 = (int)(((u1 - cu.left - cu.ns + 1) * G - 1) / W);
            a.desc[(int64_t)cu.b * rpb + cu.hr] = make_int2(c0, worker);
        }
        if (!cu.settle(a, rpb)) break;
    }
    cp_wait<0>();
}

// One CTA per row of units, or per query head of it (blockIdx.y): joins the
// pieces of a row that was cut, and fills a row that sees nothing (zeros, lse
// -inf) or whose length passes its table (NaN).  The 8 warps are 8 / pw heads
// times pw shares of the pieces; a lane holds ND pairs of a head (hd <= 64 ND).
template <typename T, int ND>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedArgs a, int pw) {
    __shared__ __align__(8) float red[kJoinWarps][kPagedMaxHd + 2];
    pdl_trigger();
    pdl_wait();
    const int rpb = a.nkv * a.rt, b = blockIdx.x / rpb, hr = blockIdx.x - b * rpb, hd = a.hd;
    const int h = hr / a.rt, row0 = (hr - h * a.rt) * a.heads, rows = min(a.heads, a.grp - row0), head0 = h * a.grp + row0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rw = kJoinWarps / pw, share = warp % pw;
    const float nan = __int_as_float(0x7fc00000);
    int2 c = a.desc[blockIdx.x];  // (not read before sq says that it was written)
    const Seq sq = seq_of(a, b);
    if (sq.len && c.x == c.y) return;
    for (int rb = blockIdx.y * rw; rb < rows; rb += gridDim.y * rw) {
        const int r = rb + warp / pw;
        const bool live = r < rows;
        constexpr int NP = 4;  // pieces in flight
        float2 o[ND];
        float M = -INFINITY, L = 0.0f;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < ND; j++) o[j] = make_float2(0.0f, 0.0f);
        if (live && sq.len) {
            const float* base = a.part + (int64_t)r * (hd + 2);
            const int64_t ps = (int64_t)a.heads * (hd + 2);
            for (int i0 = c.x + share; i0 <= c.y; i0 += NP * pw) {
                float2 ml[NP], x[NP][ND];
#pragma unroll
                for (int k = 0; k < NP; k++) {
                    const int i = i0 + k * pw;
                    const float* p = base + (2 * (int64_t)i + (i == c.x ? 1 : 0)) * ps;
                    ml[k] = i <= c.y ? *reinterpret_cast<const float2*>(p + hd) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                    for (int j = 0; j < ND; j++) {
                        const int d = 2 * lane + 64 * j;
                        x[k][j] = i <= c.y && d < hd ? *reinterpret_cast<const float2*>(p + d) : make_float2(0.0f, 0.0f);
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
        if (pw > 1) {  // the shares of a head meet in its first warp
#pragma unroll
            for (int j = 0; j < ND; j++)
                if (2 * lane + 64 * j < hd) *reinterpret_cast<float2*>(&red[warp][2 * lane + 64 * j]) = o[j];
            if (lane == 0) *reinterpret_cast<float2*>(&red[warp][kPagedMaxHd]) = make_float2(M, L);
            __syncthreads();
            if (share == 0) {
                float N = M;
                bool any = M != M;
                for (int w = 1; w < pw; w++) {
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
                for (int w = 1; w < pw; w++) {
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
            if (sq.bad) M = L = nan;
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            T* out = static_cast<T*>(a.out) + (int64_t)b * a.out_stride + (int64_t)(head0 + r) * hd;
#pragma unroll
            for (int j = 0; j < ND; j++) {
                const int d = 2 * lane + 64 * j;
                if (d < hd) {
                    out[d] = (T)(o[j].x * inv);
                    out[d + 1] = (T)(o[j].y * inv);
                }
            }
            if (a.lse && lane == 0)
                a.lse[(int64_t)b * a.nh + head0 + r] = L == 0.0f ? -INFINITY : (M + (log2f(L) - 14.0f)) * kLn2;
        }
    }
}

constexpr int kMaxPagedDevices = 64;

template <int HD, typename T, typename C, int QT, int PT, int NG>
cudaError_t go(const PagedArgs& a, cudaStream_t s) {
    static std::atomic<bool> attr[kMaxPagedDevices] = {};  // the attribute belongs to a device
    constexpr int smem = Sm<HD>::kTotal;
    auto kern = paged_split_kernel<HD, T, C, QT, PT, NG>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxPagedDevices || !attr[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxPagedDevices) attr[dev] = true;
    }
    e = launch_pdl(kern, dim3(a.workers / kWarps), dim3(kThreadsP), smem, s, a);
    if (e != cudaSuccess) return e;
    // few rows: a CTA per query head, its pieces over the 8 warps; many: a warp per head
    const int rows = a.batch * a.nkv * a.rt, heads = std::min(a.grp, a.heads);
    return rows * heads <= 2 * a.sms
               ? launch_pdl(paged_join_kernel<T, HD / 64>, dim3(rows, heads), dim3(kJoinThreads), 0, s, a, kJoinWarps)
               : launch_pdl(paged_join_kernel<T, HD / 64>, dim3(rows, 1), dim3(kJoinThreads), 0, s, a, 1);
}

// Query heads of one unit: 16 for groups past 8, so that K and V are read
// once for all of them, while the fragments of q and O fit the registers.
int unit_heads(int hd, int grp, int dtype) { return grp > 8 && (hd <= 128 || dtype != 0) ? 16 : 8; }

template <int HD, typename T, typename C, int QT, int PT>
cudaError_t go_heads(const PagedArgs& a, cudaStream_t s) {
    if constexpr (HD <= 128 || QT == 1) {
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

// Warps that fit the machine at once: two CTAs an SM, one for head dimensions
// past 128 (their rings take most of the shared memory).
int paged_workers(int hd, int sms) { return (hd > 128 ? 1 : 2) * kWarps * sms; }

size_t part_bytes(int hd, int heads, int sms) { return (size_t)paged_workers(hd, sms) * 2 * heads * (hd + 2) * sizeof(float); }

}  // namespace

size_t attention_paged_scratch(int batch, int nh, int nkv, int hd, int sms) {
    // (the type of q is not known here: the larger of the two unit sizes)
    const int grp = nh / nkv, heads = grp > 8 ? 16 : 8;
    return part_bytes(hd, heads, sms) + (size_t)batch * nkv * ((grp + 7) / 8) * sizeof(int2);
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
    a.heads = unit_heads(kv.hd, a.grp, o.dtype);
    a.rt = (a.grp + a.heads - 1) / a.heads;
    a.desc = reinterpret_cast<int2*>(static_cast<uint8_t*>(scratch) + part_bytes(kv.hd, a.heads, sms));
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
    a.workers = paged_workers(kv.hd, sms);
    a.sms = sms;
    const int es = o.dtype == 0 ? 4 : 2;
    a.q_pairs = a.q_stride % 2 == 0 && !(reinterpret_cast<uintptr_t>(q) & (2 * es - 1));
    a.scale = o.scale > 0.0f ? o.scale : (float)(1.0 / sqrt((double)kv.hd));
    a.softcap = o.softcap;
    const cudaError_t e = kv.hd <= 64    ? go_hd<64>(a, o.dtype, kv.dtype, s)
                          : kv.hd <= 128 ? go_hd<128>(a, o.dtype, kv.dtype, s)
                                         : go_hd<256>(a, o.dtype, kv.dtype, s);
    if (e != cudaSuccess) {
        *err = std::string("paged attention launch: ") + cudaGetErrorString(e);
        return B2_ERR_CUDA;
    }
    return B2_OK;
}

}  // namespace b2
