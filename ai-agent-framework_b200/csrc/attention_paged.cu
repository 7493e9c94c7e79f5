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
// tile of kTile positions of one (sequence, KV head, block of 16 query
// heads), and CTA c of G takes the units [c W / G, (c + 1) W / G).  Ragged
// batches thus load every SM equally without the host knowing a length, and
// a launch captured in a graph follows the lengths it finds.  A CTA whose
// share starts or ends inside a (sequence, head) writes that piece's
// unnormalised (o, m, l) to the scratch: at most two pieces a CTA, so the
// scratch does not grow with the lengths.  A second launch joins the pieces of
// the (sequence, head)s that were cut and fills the rows that see nothing.
//
// One CTA is 4 warps; each warp streams its own 16 positions of every tile
// through its own cp.async ring (no barrier between warps until a piece
// ends).  S = Q K^T and O = P V are mma.m16n8k16 with the group's query heads
// as the 16 rows: the tensor work is a small part of the time the bytes need,
// so the 128-row tcgen05 tile, which a group of 8 heads would leave 94 %
// empty, has nothing to give here.
//
// Rounding.  K and V enter the products as they are.  q (fp32) is scaled per
// row by a power of two and split into 2 terms for an fp16 cache (22 bits) or
// 3 for a bf16 cache (24 bits); the probabilities, times 2^14 so that small
// ones keep their bits in fp16, into 2 terms (3 where the output is fp32 and
// the cache bf16).  Sums, maxima and outputs are fp32, rounded once at the end.
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
constexpr int kStep = 16;             // positions of one warp step
constexpr int kTile = kWarps * kStep; // positions of one unit
constexpr int kRows = 16;             // query heads of one unit (rows of the mma)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 14.0f;      // probabilities are kept times 2^14

struct PagedArgs {
    const void* q;
    const uint16_t *k, *v;
    const int32_t *table, *lens, *req;
    void* out;
    float* lse;
    float* part;   // [G][2][kRows][hd + 2]
    int2* desc;    // [batch * nkv * rt]: first and last CTA of each unit row
    const float* slopes;
    int64_t q_stride, out_stride, table_stride, page_stride, pos_stride, head_stride;
    int batch, nh, nkv, grp, rt, hd, page_size, n_pages, max_pages, n_req, len_add, window, grid;
    float scale, softcap;
};

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

__device__ __forceinline__ int tiles_of(const Seq& s) { return s.len == 0 ? 0 : (s.len - 1) / kTile - s.lo / kTile + 1; }

template <int HD>
__device__ __forceinline__ uint32_t sw(int r, int c) {
    return (uint32_t)(r * (HD * 2) + ((c ^ (r & 7)) << 4));
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
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

template <int HD, int QT>
struct Sm {
    static constexpr int kRow = HD * 2;
    static constexpr int kStages = HD == 64 ? 6 : 3;
    static constexpr int kStage = 2 * kStep * kRow;              // a warp's K and V rows of one tile
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kQ = kRows * kRow;                      // one term of q
    static constexpr int kTotal = kRing + QT * kQ + kRows * 4;   // + the rows' 2^-e
    static_assert(kWarps * kRows * (HD + 2) * 4 <= kRing, "the warps' merge fits over the ring");
};

// T: the type of q and out; C: the cache's; QT, PT: terms of q and of the
// probabilities.
template <int HD, typename T, typename C, int QT, int PT>
__global__ void __launch_bounds__(kThreadsP) paged_split_kernel(const __grid_constant__ PagedArgs a) {
    using SM = Sm<HD, QT>;
    constexpr int KS = HD / 16, NT = HD / 8, ST = SM::kStages;
    extern __shared__ __align__(1024) uint8_t psm[];
    __shared__ long long wsum[kWarps];
    __shared__ int sh_b;
    __shared__ long long sh_base;
    uint8_t* qs = psm + SM::kRing;
    float* qscale = reinterpret_cast<float*>(qs + QT * SM::kQ);
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gi = lane >> 2, ti = lane & 3;
    const int hd = a.hd, hc = hd / 8, rpb = a.nkv * a.rt;

    // columns past hd stay zero: the copies never write them
    if (hd < HD)
        for (int i = tid; i < SM::kRing / 16; i += kThreadsP) *reinterpret_cast<uint4*>(psm + 16 * i) = make_uint4(0, 0, 0, 0);

    // this CTA's units: the tiles of the sequences before each, by a scan
    const int per = (a.batch + kThreadsP - 1) / kThreadsP;
    const int b0 = min(a.batch, tid * per), b1 = min(a.batch, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; b++) mine += tiles_of(seq_of(a, b));
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        if (w == warp) inc += total;
        total += wsum[w];
    }
    const long long W = total * rpb;
    const long long G = min((long long)a.grid, W);
    const int cta = blockIdx.x;
    if (cta >= G) return;
    long long u = cta * W / G;
    const long long u1 = (cta + 1) * W / G;
    {
        long long base = (inc - mine) * rpb;
        if (u >= base && u < inc * rpb) {
            for (int b = b0; b < b1; b++) {
                const long long n = (long long)tiles_of(seq_of(a, b)) * rpb;
                if (u < base + n) {
                    sh_b = b;
                    sh_base = base;
                    break;
                }
                base += n;
            }
        }
    }
    __syncthreads();
    int b = sh_b;
    Seq sq = seq_of(a, b);
    int nt = tiles_of(sq);
    int hr = (int)((u - sh_base) / nt), tile = (int)((u - sh_base) - (long long)hr * nt);

    uint8_t* ring = psm + warp * ST * SM::kStage;
    const uint32_t ring_s = smem_u32(ring), qs_s = smem_u32(qs);
    const int a_row = (lane & 7) + ((lane >> 3) & 1) * 8, a_kc = (lane >> 4) & 1;
    const int bk_row = (lane & 7) + ((lane >> 4) & 1) * 8, bk_kc = (lane >> 3) & 1;
    const int bv_row = (lane & 7) + ((lane >> 3) & 1) * 8, bv_dc = (lane >> 4) & 1;

    while (u < u1) {
        const int h = hr / a.rt, row0 = (hr - h * a.rt) * kRows;  // KV head, first query head of the group
        const int rows = min(kRows, a.grp - row0);
        const int n = (int)min((long long)(nt - tile), u1 - u);
        const bool from_start = tile == 0, to_end = tile + n == nt;
        const int head0 = h * a.grp + row0;
        const int t_first = sq.lo / kTile + tile;  // absolute tile
        const int32_t* trow = a.table + (int64_t)sq.tr * a.table_stride;
        bool bad = false;

        // page of this lane's row (lane & 15) of tile i: -1 for a position that is not seen
        auto fetch = [&](int i) {
            const int p = (t_first + i) * kTile + warp * kStep + (lane & 15);
            int id = -1;
            if (i < n && p >= sq.lo && p < sq.len) {
                id = __ldg(trow + p / a.page_size);
                if (id < 0 || id >= a.n_pages) {
                    bad = true;
                    id = -1;
                }
            }
            return id;
        };
        auto issue = [&](int i, int id) {
            if (i < n) {
                const int p = (t_first + i) * kTile + warp * kStep + (lane & 15);
                const int64_t off = id < 0 ? 0 : id * a.page_stride + (p % a.page_size) * a.pos_stride + h * a.head_stride;
                const uint32_t kt = ring_s + (i % ST) * SM::kStage, vt = kt + kStep * SM::kRow;
                constexpr int LR = HD / 8 <= 32 ? 32 / (HD / 8) : 1;  // rows one warp copy covers
                const int c = lane % (HD / 8), r0 = lane / (HD / 8);
#pragma unroll
                for (int j = 0; j < kStep / LR; j++) {
                    const int r = r0 + j * LR;
                    const int64_t o = __shfl_sync(0xffffffffu, off, r) + c * 8;
                    const bool ok = __shfl_sync(0xffffffffu, id, r) >= 0;
                    if (c < hc) {
                        cp16(kt + sw<HD>(r, c), a.k + o, ok);
                        cp16(vt + sw<HD>(r, c), a.v + o, ok);
                    }
                }
            }
            cp_async_commit();
        };
        int id = fetch(0);
#pragma unroll 1
        for (int i = 0; i < ST - 1; i++) {
            const int nx = fetch(i + 1);
            issue(i, id);
            id = nx;
        }

        // q: warp w takes rows w, w + 4, ...
        for (int r = warp; r < kRows; r += kWarps) {
            const T* qr = static_cast<const T*>(a.q) + (int64_t)b * a.q_stride + (int64_t)(head0 + r) * hd;
            float x[HD / 32];
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < HD / 64; j++) {
                const int c = 2 * (lane + 32 * j);
                x[2 * j] = x[2 * j + 1] = 0.0f;
                if (r < rows && c < hd) {
                    x[2 * j] = (float)qr[c];
                    x[2 * j + 1] = (float)qr[c + 1];
                }
                mx = fmaxf(mx, fmaxf(fabsf(x[2 * j]), fabsf(x[2 * j + 1])));
            }
            float back = 1.0f;
            if (QT > 1) {  // the largest element to [2^10, 2^11); one term is q itself
                mx = warp_max(mx);
                const int e = mx > 0.0f && mx < 3.0e38f ? min(100, max(-100, 10 - ilogbf(mx))) : 0;
                const float f = __int_as_float((127 + e) << 23);
                back = __int_as_float((127 - e) << 23);
#pragma unroll
                for (int j = 0; j < HD / 32; j++) x[j] *= f;
            }
#pragma unroll
            for (int j = 0; j < HD / 64; j++) {
                const int c = 2 * (lane + 32 * j);
                uint32_t t[QT];
                split_terms<C, QT>(x[2 * j], x[2 * j + 1], t);
                const uint32_t off = sw<HD>(r, c / 8) + (c % 8) * 2;
#pragma unroll
                for (int i = 0; i < QT; i++) *reinterpret_cast<uint32_t*>(qs + i * SM::kQ + off) = t[i];
            }
            if (lane == 0) qscale[r] = back * a.scale;
        }
        __syncthreads();
        const float sc0 = qscale[gi], sc1 = qscale[gi + 8];
        float sl0 = 0.0f, sl1 = 0.0f;
        if (a.slopes) {
            if (gi < rows) sl0 = __ldg(a.slopes + head0 + gi);
            if (gi + 8 < rows) sl1 = __ldg(a.slopes + head0 + gi + 8);
        }

        float o[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;  // rows gi, gi + 8

#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const int nx = fetch(i + ST);
            issue(i + ST - 1, id);
            id = nx;
            cp_wait<ST - 1>();
            __syncwarp();
            const uint32_t kt = ring_s + (i % ST) * SM::kStage, vt = kt + kStep * SM::kRow;
            const int p0 = (t_first + i) * kTile + warp * kStep;
            if (p0 < sq.len && p0 + kStep > sq.lo) {
                // one accumulator pair per term of q: short chains, and the terms below the
                // first stay out of a score that an infinite key made infinite (0 * inf)
                float s0[QT][4], s1[QT][4];
#pragma unroll
                for (int t = 0; t < QT; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s0[t][j] = s1[t][j] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < KS; kk++) {
                    uint32_t bk[4];
                    ldsm(kt + sw<HD>(bk_row, 2 * kk + bk_kc), bk);
#pragma unroll
                    for (int t = 0; t < QT; t++) {
                        uint32_t aq[4];
                        ldsm(qs_s + t * SM::kQ + sw<HD>(a_row, 2 * kk + a_kc), aq);
                        Cvt<C>::mma(s0[t], aq, bk[0], bk[1]);
                        Cvt<C>::mma(s1[t], aq, bk[2], bk[3]);
                    }
                }
                // rows gi (values 0, 1) and gi + 8 (2, 3); positions p0 + 2 ti + {0, 1} (s0), + 8 (s1)
                float s[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float top = j < 4 ? s0[0][j] : s1[0][j - 4];
                    float low = 0.0f;
#pragma unroll
                    for (int t = QT - 1; t > 0; t--) low += j < 4 ? s0[t][j] : s1[t][j - 4];
                    s[j] = (QT > 1 && fabsf(top) == INFINITY ? top : top + low) * ((j & 2) ? sc1 : sc0);
                }
                if (a.softcap > 0.0f) {
#pragma unroll
                    for (int j = 0; j < 8; j++) s[j] = a.softcap * tanhf(s[j] / a.softcap);
                }
                const int pj = p0 + 2 * ti;
                if (a.slopes) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        s[j] = fmaf((j & 2) ? sl1 : sl0, (float)(pj + (j & 1) + (j & 4) * 2 - (sq.len - 1)), s[j]);
                }
                if (p0 < sq.lo || p0 + kStep > sq.len) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int p = pj + (j & 1) + (j & 4) * 2;
                        if (p < sq.lo || p >= sq.len) s[j] = -INFINITY;
                    }
                }
                float r0 = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[4], s[5])), r1 = fmaxf(fmaxf(s[2], s[3]), fmaxf(s[6], s[7]));
                r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, 1));
                r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, 1));
                r0 = fmaxf(r0, __shfl_xor_sync(0xffffffffu, r0, 2));
                r1 = fmaxf(r1, __shfl_xor_sync(0xffffffffu, r1, 2));
                const float n0 = fmaxf(m0, r0), n1 = fmaxf(m1, r1);
                // (a row whose scores are all -inf so far keeps weight zero)
                const float z0 = n0 == -INFINITY ? 0.0f : n0, z1 = n1 == -INFINITY ? 0.0f : n1;
                const float f0 = ex2((m0 - z0) * kLog2e), f1 = ex2((m1 - z1) * kLog2e);
                m0 = n0;
                m1 = n1;
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = ex2(fmaf(s[j] - ((j & 2) ? z1 : z0), kLog2e, kPShift));
                l0 = fmaf(l0, f0, (p[0] + p[1]) + (p[4] + p[5]));
                l1 = fmaf(l1, f1, (p[2] + p[3]) + (p[6] + p[7]));
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    o[j][0] *= f0;
                    o[j][1] *= f0;
                    o[j][2] *= f1;
                    o[j][3] *= f1;
                }
                uint32_t pa[PT][4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t t[PT];
                    split_terms<C, PT>(p[2 * j], p[2 * j + 1], t);
#pragma unroll
                    for (int x = 0; x < PT; x++) pa[x][j] = t[x];
                }
#pragma unroll
                for (int j = 0; j < NT / 2; j++) {
                    uint32_t bv[4];
                    ldsm_t(vt + sw<HD>(bv_row, 2 * j + bv_dc), bv);
#pragma unroll
                    for (int x = 0; x < PT; x++) {
                        Cvt<C>::mma(o[2 * j], pa[x], bv[0], bv[1]);
                        Cvt<C>::mma(o[2 * j + 1], pa[x], bv[2], bv[3]);
                    }
                }
            }
            __syncwarp();  // the slot is refilled by the next step's issue
        }
        cp_wait<0>();
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if (__any_sync(0xffffffffu, bad)) m0 = m1 = l0 = l1 = __int_as_float(0x7fc00000);  // a page that is not there

        // the warps' pieces meet over the ring: [warp][16][HD + 2]
        __syncthreads();
        float* mw = reinterpret_cast<float*>(psm);
        float* wr = mw + warp * kRows * (HD + 2);
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int d = j * 8 + 2 * ti;
            wr[gi * (HD + 2) + d] = o[j][0];
            wr[gi * (HD + 2) + d + 1] = o[j][1];
            wr[(gi + 8) * (HD + 2) + d] = o[j][2];
            wr[(gi + 8) * (HD + 2) + d + 1] = o[j][3];
        }
        if (ti == 0) {
            wr[gi * (HD + 2) + HD] = m0;
            wr[gi * (HD + 2) + HD + 1] = l0;
            wr[(gi + 8) * (HD + 2) + HD] = m1;
            wr[(gi + 8) * (HD + 2) + HD + 1] = l1;
        }
        __syncthreads();
        const bool whole = from_start && to_end;
        float* part = a.part + (int64_t)(2 * cta + (from_start ? 1 : 0)) * kRows * (hd + 2);
        for (int i = tid; i < rows * (hd + 1); i += kThreadsP) {
            const int r = i / (hd + 1), d = i - r * (hd + 1);  // d == hd: the row's m and l
            float M = -INFINITY;
            bool nan = false;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float m = mw[(w * kRows + r) * (HD + 2) + HD];
                nan |= m != m;
                M = fmaxf(M, m);
            }
            float val = 0.0f, L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float* pw = mw + (w * kRows + r) * (HD + 2);
                const float f = pw[HD] == -INFINITY ? 0.0f : ex2((pw[HD] - M) * kLog2e);
                if (d < hd) val = fmaf(pw[d], f, val);
                L = fmaf(pw[HD + 1], f, L);
            }
            if (nan) M = L = val = __int_as_float(0x7fc00000);
            if (!whole) {
                part[r * (hd + 2) + d] = d < hd ? val : M;
                if (d == hd) part[r * (hd + 2) + hd + 1] = L;
            } else if (d < hd) {
                static_cast<T*>(a.out)[(int64_t)b * a.out_stride + (int64_t)(head0 + r) * hd + d] =
                    (T)(L == 0.0f ? 0.0f : val / L);
            } else if (a.lse) {
                a.lse[(int64_t)b * a.nh + head0 + r] = L == 0.0f ? -INFINITY : M + (log2f(L) - kPShift) * 0.6931471805599453f;
            }
        }
        if (to_end && tid == 0) {
            const long long first = u - tile;  // the unit row's first unit, and the CTA that holds it
            a.desc[(int64_t)b * rpb + hr] = make_int2((int)(((first + 1) * G - 1) / W), cta);
        }
        __syncthreads();
        if (hd < HD && u + n < u1) {  // the merge wrote over the ring's zero columns
            for (int i = tid; i < SM::kRing / 16; i += kThreadsP)
                *reinterpret_cast<uint4*>(psm + 16 * i) = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }

        u += n;
        tile = 0;
        if (to_end && ++hr == rpb) {
            hr = 0;
            while (u < u1) {
                sq = seq_of(a, ++b);
                nt = tiles_of(sq);
                if (nt) break;
            }
        }
    }
}

// One CTA per (sequence, query head): joins the pieces of a row that was cut,
// and fills a row that sees nothing (zeros, lse -inf) or whose length passes
// its table (NaN).
template <typename T>
__global__ void __launch_bounds__(kThreadsP) paged_join_kernel(const __grid_constant__ PagedArgs a) {
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x / a.nh, head = blockIdx.x - b * a.nh, hd = a.hd;
    const Seq sq = seq_of(a, b);
    T* out = static_cast<T*>(a.out) + (int64_t)b * a.out_stride + (int64_t)head * hd;
    float* lse = a.lse ? a.lse + (int64_t)b * a.nh + head : nullptr;
    if (sq.len == 0) {
        const float nan = __int_as_float(0x7fc00000);
        for (int d = threadIdx.x; d < hd; d += kThreadsP) out[d] = (T)(sq.bad ? nan : 0.0f);
        if (lse && threadIdx.x == 0) *lse = sq.bad ? nan : -INFINITY;
        return;
    }
    const int h = head / a.grp, rg = head - h * a.grp, hr = h * a.rt + rg / kRows;
    const int2 c = a.desc[(int64_t)b * a.nkv * a.rt + hr];
    if (c.x == c.y) return;
    const float* row = a.part + (int64_t)(rg % kRows) * (hd + 2);
    const int64_t ps = (int64_t)kRows * (hd + 2);
    auto piece = [&](int i) { return row + (2 * (int64_t)i + (i == c.x ? 1 : 0)) * ps; };
    float M = -INFINITY;
    bool nan = false;
    for (int i = c.x; i <= c.y; i++) {
        const float m = piece(i)[hd];
        nan |= m != m;
        M = fmaxf(M, m);
    }
    float L = 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int d0 = threadIdx.x, d1 = threadIdx.x + kThreadsP;
    for (int i = c.x; i <= c.y; i++) {
        const float* p = piece(i);
        const float f = p[hd] == -INFINITY ? 0.0f : ex2((p[hd] - M) * kLog2e);
        L = fmaf(p[hd + 1], f, L);
        if (d0 < hd) o0 = fmaf(p[d0], f, o0);
        if (d1 < hd) o1 = fmaf(p[d1], f, o1);
    }
    if (nan) M = L = o0 = o1 = __int_as_float(0x7fc00000);
    if (d0 < hd) out[d0] = (T)(L == 0.0f ? 0.0f : o0 / L);
    if (d1 < hd) out[d1] = (T)(L == 0.0f ? 0.0f : o1 / L);
    if (lse && threadIdx.x == 0) *lse = L == 0.0f ? -INFINITY : M + (log2f(L) - kPShift) * 0.6931471805599453f;
}

constexpr int kMaxPagedDevices = 64;

template <int HD, typename T, typename C, int QT, int PT>
cudaError_t go(const PagedArgs& a, cudaStream_t s) {
    static std::atomic<bool> attr[kMaxPagedDevices] = {};  // the attribute belongs to a device
    constexpr int smem = Sm<HD, QT>::kTotal;
    auto kern = paged_split_kernel<HD, T, C, QT, PT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxPagedDevices || !attr[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxPagedDevices) attr[dev] = true;
    }
    e = launch_pdl(kern, dim3(a.grid), dim3(kThreadsP), smem, s, a);
    if (e != cudaSuccess) return e;
    return launch_pdl(paged_join_kernel<T>, dim3(a.batch * a.nh), dim3(kThreadsP), 0, s, a);
}

template <int HD>
cudaError_t go_hd(const PagedArgs& a, int dtype, int cache, cudaStream_t s) {
    if (dtype == 0)
        return cache == 1 ? go<HD, float, __half, 2, 2>(a, s) : go<HD, float, __nv_bfloat16, 3, 3>(a, s);
    return cache == 1 ? go<HD, __half, __half, 1, 2>(a, s) : go<HD, __nv_bfloat16, __nv_bfloat16, 1, 2>(a, s);
}

// CTAs that fit the machine at once: two an SM, one for head dimensions past
// 128 (their rings take most of the shared memory)
int paged_grid(int hd, int sms) { return hd > 128 ? sms : 2 * sms; }

size_t part_bytes(int hd, int sms) { return (size_t)paged_grid(hd, sms) * 2 * kRows * (hd + 2) * sizeof(float); }

}  // namespace

size_t attention_paged_scratch(int batch, int nh, int nkv, int hd, int sms) {
    const int rt = (nh / nkv + kRows - 1) / kRows;
    return part_bytes(hd, sms) + (size_t)batch * nkv * rt * sizeof(int2);
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
    a.desc = reinterpret_cast<int2*>(static_cast<uint8_t*>(scratch) + part_bytes(kv.hd, sms));
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
    a.grp = o.nh / kv.nkv;
    a.rt = (a.grp + kRows - 1) / kRows;
    a.hd = kv.hd;
    a.page_size = kv.page_size;
    a.n_pages = kv.n_pages;
    a.max_pages = o.max_pages;
    a.n_req = o.n_req;
    a.len_add = o.len_add;
    a.window = o.window;
    a.grid = paged_grid(kv.hd, sms);
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
