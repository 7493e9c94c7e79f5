// Attention of rows that share a prefix of a paged KV cache: what b2_attention_paged
// computes (attention_paged.cu has the formulas), with the positions that the
// rows of a group have in common read once for all of them.
//
// Items.  A group's shared positions times up to 128 (row, query head) pairs of
// one KV head are an item, and so are the positions of one row behind its
// prefix, times its own heads.  A tile is 128 positions of an item:
//   S = Q K^T (128 x 128),  m = max s, p = e^(s - m), l = sum p,  T = P V,
// each tile with a maximum of its own, so tiles do not wait for one another; O
// and L take them up in fp32 registers,
//   M' = max(M, m),  O <- O e^(M - M') + T e^(m - M').
// Items need not share a maximum either, so a row's pieces (shared, own, and
// those of an item that was cut) meet in one joining launch.
//
// What bounds it: of 64 rows behind 32K shared positions (64 heads on 8 of 128, bf16)
// 70 GFLOP would take 42 us of the tensor cores; the chain of a tile
// (scores, exponentials, values, one tile's tensor memory waiting for the next) takes
// 3600 clocks for products of 1650 (two terms of P), so 166 us.
//
// Split.  The items of the batch, one after another, are a line of units, a
// tile being one (and an item's start another).  Share s of G takes the units
// [s W / G, (s + 1) W / G) for every KV head side by side, so the machine is
// evenly loaded whatever the lengths, the host knows none of them, and a graph
// follows the lengths that it finds.  A first launch lays the line, by one CTA.
//
// One CTA an SM, its roles warp by warp:
//   16-17  K and V rows into a ring of tiles in the 128-byte swizzle that the
//          products read: by TMA where pages are multiples of 8 positions, by
//          cp.async row by row elsewhere and at the ends of what is seen
//   18     the share's pieces of the items, laid out ahead for the others, and Q
//          by TMA, whose 16-bit terms the first launch has made
//   19     tcgen05.mma, one thread: S = Q K^T of tile j + 1, then T = P V of tile
//          j, P being read from tensor memory
//   0-7    two warpgroups taking tiles in turn: S out of tensor memory, a row to
//          a thread, the exponentials, P back over S
//   8-15   O, a half of the dimensions each four: T out of tensor memory, added in
//          fp32 (the tensor cores' own accumulation cuts instead of rounding, which
//          over a long row pulls towards zero); at an item's end the result or the piece
//
// Rounding.  K and V as they are; fp32 rows scaled per row by a power of two and
// split into 2 fp16 or 3 bf16 terms, and their probabilities times 2^14 into as
// many (22 bits or more: what fp32 results need).  16-bit rows as they are, their
// probabilities in 2 terms, 22 bits of fp16 or 16 of bf16, as row by row: with one
// term, 12 % faster, weights that round to the same side move the result by up to
// a step.  Sums, maxima and O in fp32, rounded once.
//
// Measured (B200, graphs, all three launches): 8 requests of 8 beams over up to 32K, 32 heads
// on 8 of 128, fp32 rows 102 us (row by row 389); 64 rows behind 32K, 64 heads on 8,
// bf16 166 (1010); a prompt of 2048 tokens, the same heads 149 (1064).
//
// A value that one row of an item sees and another does not meets a weight of 0
// there, and 0 times infinity or NaN is NaN: a row whose result is not finite is
// computed again by the joining launch, alone, from its own positions.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "attention_common.cuh"
#include "dev.cuh"
#include "paged.h"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace b2 {
namespace {

constexpr int kTile = 128;       // positions of a tile, rows of a product
constexpr int kItemUnits = 1;    // units' worth of starting an item
constexpr int kMinShare = 3;     // a share's units, at least
constexpr int kPlanThreads = 1024;
constexpr int kPlanItems = 2 * kPlanThreads;  // items whose units stay in shared memory,
constexpr int kLineGroups = 2048;               // and groups
constexpr int kNoLimit = 0x7fffffff;

struct Item {
    long long u0;      // units before it
    int row0, rows;    // its rows
    int lo, hi;        // positions
    int tr, limit;     // table row; positions from limit on are not its own (kNoLimit: a row's own positions)
};
static_assert(sizeof(Item) == 32, "two 16-byte loads");

struct Line {
    long long units;
    int items, shares;
    int dead;  // a wait of the tiles' launch gave up: every row becomes NaN
};

// Where a share starts: item, its unit, units of the share.
struct Share {
    int item, at;
    long long units;
};

struct SharedArgs {
    const void* q;
    const uint16_t *k, *v;
    const int32_t *table, *lens, *req, *starts, *prefix;
    void* out;
    float* lse;
    const float* slopes;
    int64_t q_stride, out_stride, table_stride, page_stride, pos_stride, head_stride;
    int batch, nh, nkv, grp, hd, page_size, n_pages, max_pages, n_req, len_add, window, n_groups;
    int hb, blocks, rows;  // query heads of an item, such blocks of a group of heads, rows of an item
    int shares;            // at most
    int q_wide, out_wide;  // 16-byte accesses
    int terms;             // of Q that the first launch makes; 0: the products read q as it is
    int box;               // positions of a box of the tensor maps (16 or 8); 0: pages that they cannot tell
    int flat;              // pages follow one another as their positions do: one dimension; 2: boxes of whole heads
    float scale, softcap;
    uint32_t page_mul;  // division by the page size
    int page_shift;
    // scratch
    Line* line;
    Share* share;  // [shares]
    uint16_t* term;  // [terms][batch][nh][hd] Q, scaled per row, as 16-bit terms
    float* factor;   // [batch][nh] what a product with them is times for a score
    int* redo;     // [batch]
    int4* row;     // [batch] {first visible position, length, shared item, own item}: -1 none, -2 a row of NaN
    Item* item;    // [2 batch]
    float* whole;  // [2][batch][nh][hd + 4] results of whole items of rows that have two: o, m (log2 units), l
    float* part;   // [CTAs][2][128][hd + 4] pieces of items that were cut
};

// n / page_size for 0 <= n < 2^31 (Granlund and Montgomery, "Division by
// invariant integers using multiplication", 1994): with s = ceil(log2 P) and mul
// = floor(2^32 (2^s - P) / P) + 1, n / P = (mulhi(mul, n) + n) >> s.
__device__ __forceinline__ int page_of(const SharedArgs& a, int n) {
    return (int)((__umulhi(a.page_mul, (unsigned)n) + (unsigned)n) >> a.page_shift);
}

// tiles start on multiples of 16 positions
__device__ __forceinline__ int base_of(const Item& it) { return it.lo & ~15; }
__device__ __forceinline__ int tiles_of(const Item& it) { return (it.hi - base_of(it) - 1) / kTile + 1; }  // (it.hi > it.lo, up to 2^31 - 64)

// The last i of a[0 .. n) (ascending, a[0] <= x) with a[i] <= x.
template <typename F>
__device__ __forceinline__ int last_at(int n, F&& le) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (le(mid)) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---------------------------------------------------------------------------
// the line of items, by one CTA
// ---------------------------------------------------------------------------

// Rows of one turn, RPT to a thread, and the 127 behind them that its items may
// reach into.
template <int RPT>
struct LineShared {
    static constexpr int kRows = RPT * kPlanThreads;
    int lo[kRows + kTile], hi[kRows + kTile];  // a row's positions among its group's shared ones
    int len[kRows + kTile], tr[kRows + kTile];  // len -1: a row of NaN
    int group[kRows + kTile];
    int owner[kTile + kRows];                  // the item that starts at a row, also of the 128 rows before
    int starts[kLineGroups + 1], prefix[kLineGroups];
    long long w_units[kPlanThreads / 32], u_item[kPlanItems];
    int w_items[kPlanThreads / 32];
};

template <int RPT>
__device__ __forceinline__ void lay_line(const SharedArgs& a) {
    using LS = LineShared<RPT>;
    extern __shared__ __align__(16) uint8_t line_raw[];
    LS& s = *reinterpret_cast<LS*>(line_raw);
    constexpr int W = kPlanThreads / 32, N = LS::kRows;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, R = a.rows;
    const bool near = a.n_groups <= kLineGroups;  // the groups are in shared memory
    if (near) {
        for (int i = tid; i <= a.n_groups; i += kPlanThreads) s.starts[i] = a.starts[i];
        for (int i = tid; i < a.n_groups; i += kPlanThreads) s.prefix[i] = a.prefix[i];
    }
    auto start_of = [&](int g) { return near ? s.starts[g] : a.starts[g]; };
    // (at most the longest length there is: kNoLimit marks a row's own positions)
    auto prefix_of = [&](int g) { return (int)min((long long)max(near ? s.prefix[g] : a.prefix[g], 0), kMaxLen); };

    int items = 0;
    long long units = 0;
    for (int base = 0; base < a.batch; base += N) {
        Seq sq[RPT + 1];
#pragma unroll
        for (int u = 0; u <= RPT; u++) {  // (their words, on their way together)
            const int i = tid + u * kPlanThreads;
            sq[u] = Seq{};
            if (i < N + R - 1 && base + i < a.batch) sq[u] = seq_of(a, base + i);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u <= RPT; u++) {
            const int i = tid + u * kPlanThreads, b = base + i;
            if (i >= N + R - 1) continue;
            int g = -1, prefix = 0;
            if (b < a.batch) {
                g = last_at(a.n_groups, [&](int x) { return start_of(x) <= b; });
                if (start_of(g) > b || start_of(g + 1) <= b) g = -1;
                else prefix = prefix_of(g);
            }
            s.lo[i] = sq[u].lo;
            s.hi[i] = min(sq[u].len, prefix);
            s.len[i] = sq[u].bad ? -1 : sq[u].len;
            s.tr[i] = sq[u].tr;
            s.group[i] = g;
        }
        __syncthreads();
        // this thread's rows: their items and units
        Item sh[RPT], own[RPT];
        int n = 0, first[RPT];  // first: the row's group's first row
        long long u = 0;
#pragma unroll
        for (int k = 0; k < RPT; k++) {
            const int i = tid * RPT + k, b = base + i;
            sh[k] = own[k] = Item{};
            first[k] = b;
            if (b >= a.batch) continue;
            const int g = s.group[i];
            int prefix = 0;
            if (g >= 0) {
                first[k] = max(start_of(g), 0);
                prefix = prefix_of(g);
                if ((b - first[k]) % R == 0) {
                    Item x{};
                    x.row0 = b;
                    x.rows = min(R, min(start_of(g + 1), a.batch) - b);
                    x.lo = kNoLimit;
                    x.tr = -1;
                    x.limit = prefix;
#pragma unroll 4
                    for (int r = 0; r < x.rows; r++)
                        if (s.hi[i + r] > s.lo[i + r]) {
                            if (x.tr < 0) x.tr = s.tr[i + r];
                            x.lo = min(x.lo, s.lo[i + r]);
                            x.hi = max(x.hi, s.hi[i + r]);
                        }
                    sh[k] = x;
                }
            }
            own[k] = Item{0, b, 1, max(s.lo[i], prefix), max(s.len[i], 0), s.tr[i], kNoLimit};
            a.redo[b] = 0;
            if (sh[k].hi > sh[k].lo) {
                n++;
                u += tiles_of(sh[k]) + kItemUnits;
            }
            if (own[k].hi > own[k].lo) {
                n++;
                u += tiles_of(own[k]) + kItemUnits;
            }
        }
        int ni = n;
        long long nu = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, ni, o);
            const long long y = __shfl_up_sync(0xffffffffu, nu, o);
            if (lane >= o) {
                ni += x;
                nu += y;
            }
        }
        if (lane == 31) {
            s.w_items[warp] = ni;
            s.w_units[warp] = nu;
        }
        if (tid < kTile) s.owner[tid] = base ? s.owner[N + tid] : -1;
        __syncthreads();
        // the warps before this one, and all of them: a scan by every warp
        int wi = lane < W ? s.w_items[lane] : 0;
        long long wu = lane < W ? s.w_units[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, wi, o);
            const long long y = __shfl_up_sync(0xffffffffu, wu, o);
            if (lane >= o) {
                wi += x;
                wu += y;
            }
        }
        int at = items + ni - n + (warp ? __shfl_sync(0xffffffffu, wi, max(warp - 1, 0)) : 0);
        long long u0 = units + nu - u + (warp ? __shfl_sync(0xffffffffu, wu, max(warp - 1, 0)) : 0);
        items += __shfl_sync(0xffffffffu, wi, 31);
        units += __shfl_sync(0xffffffffu, wu, 31);
        int i_own[RPT];
        auto put = [&](Item& x) {
            if (x.hi <= x.lo) return -1;
            x.u0 = u0;
            u0 += tiles_of(x) + kItemUnits;
            a.item[at] = x;
            if (at < kPlanItems) s.u_item[at] = x.u0;
            return at++;
        };
#pragma unroll
        for (int k = 0; k < RPT; k++) {
            s.owner[kTile + tid * RPT + k] = put(sh[k]);
            i_own[k] = put(own[k]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RPT; k++) {
            const int i = tid * RPT + k, b = base + i;
            if (b >= a.batch) continue;
            int mine = -1;
            if (s.hi[i] > s.lo[i]) {  // (the item starts at most 127 rows before)
                const int o = first[k] + (b - first[k]) / R * R - base + kTile;
                mine = o >= 0 ? s.owner[o] : -1;
            }
            a.row[b] = s.len[i] < 0 ? make_int4(0, 0, -2, -2) : make_int4(s.lo[i], s.len[i], mine, i_own[k]);
        }
        __syncthreads();
    }
    const int G = (int)max(1LL, min((long long)a.shares, units / kMinShare));
    if (tid == 0) *a.line = Line{units, items, G, 0};
    if (units == 0) {
        for (int i = tid; i < a.shares; i += kPlanThreads) a.share[i] = Share{0, 0, 0};
        return;
    }
    for (int i = G + tid; i < a.shares; i += kPlanThreads) a.share[i] = Share{0, 0, 0};
    for (int h = tid; h < G; h += kPlanThreads) {
        const long long u = mul_div(h, units, G);
        const int i = last_at(items, [&](int x) { return (items <= kPlanItems ? s.u_item[x] : a.item[x].u0) <= u; });
        const long long at = u - (items <= kPlanItems ? s.u_item[i] : a.item[i].u0);
        a.share[h] = Share{i, (int)at, mul_div(h + 1, units, G) - u};
    }
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// 4 elements from p on
__device__ __forceinline__ float4 load4(const float* p, bool wide) {
    return wide ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
}
template <typename T>
__device__ __forceinline__ float4 load4(const T* p, bool wide) {
    alignas(8) T t[4];
    if (wide) *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p);
    else
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = p[i];
    return make_float4(to_float(t[0]), to_float(t[1]), to_float(t[2]), to_float(t[3]));
}

// The power of two that takes a row's largest element to [2^10, 2^11), the row
// four elements a lane.  The exponent field is enough: subnormal rows count as
// 2^-127; from -117 for the largest finite row to 100, so that 2^e and 2^-e are normal.
__device__ __forceinline__ int row_exponent(float4 x) {
    const float mx = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));  // (none negative: ordered as their bits)
    return top < 0x7f800000u ? min(100, 137 - (int)(top >> 23)) : 0;
}
__device__ __forceinline__ float pow2f(int e) { return __int_as_float((127 + e) << 23); }

// A warp's rows of Q, one after another: largest element to [2^10, 2^11), then
// 16-bit terms.  (A single term is q itself, copied for its alignment.)
template <typename T, typename C, int QT>
__device__ __forceinline__ void make_terms(const SharedArgs& a, long long first, long long step) {
    const int lane = threadIdx.x & 31, d = 4 * lane;
    const long long rows = (long long)a.batch * a.nh;
    const bool in = d < a.hd;
    constexpr int U = 4;
    for (long long r0 = first; r0 < rows; r0 += U * step) {
        float4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = r0 + u * step;
            x[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (r < rows && in) {
                const int b = (int)(r / a.nh), head = (int)(r - (long long)b * a.nh);
                x[u] = load4(static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)head * a.hd + d, a.q_wide);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long r = r0 + u * step;
            if (r >= rows) break;
            if (QT > 1) {
                const int e = row_exponent(x[u]);
                const float up = pow2f(e), f = a.scale * pow2f(-e);
                if (lane == 0) a.factor[r] = a.softcap > 0.0f ? f / a.softcap : f * kLog2e;
                x[u] = make_float4(x[u].x * up, x[u].y * up, x[u].z * up, x[u].w * up);
            }
            uint32_t w0[QT], w1[QT];
            split_terms<C, QT>(x[u].x, x[u].y, w0);
            split_terms<C, QT>(x[u].z, x[u].w, w1);
            if (in)
#pragma unroll
                for (int k = 0; k < QT; k++) *reinterpret_cast<uint2*>(a.term + (k * rows + r) * a.hd + d) = make_uint2(w0[k], w1[k]);
        }
    }
}

// The first launch: the line by one CTA, Q's terms by the others.
template <typename T, typename C, int QT, int RPT>
__global__ void __launch_bounds__(kPlanThreads) shared_line_kernel(const __grid_constant__ SharedArgs a) {
    pdl_trigger();
    pdl_wait();
    if (blockIdx.x == 0) lay_line<RPT>(a);
    else make_terms<T, C, QT>(a, (blockIdx.x - 1) * (kPlanThreads / 32) + threadIdx.x / 32, (gridDim.x - 1) * (kPlanThreads / 32));
}

// ---------------------------------------------------------------------------
// the products
// ---------------------------------------------------------------------------

constexpr int kSoftWarps = 8, kSumWarps = 8;  // then two warps that copy, one that plans and brings Q, one that multiplies
constexpr int kCopyWarp = kSoftWarps + kSumWarps, kCopyWarps = 2, kQWarp = kCopyWarp + kCopyWarps, kMmaWarp = kQWarp + 1;
constexpr int kSharedThreads = 32 * (kMmaWarp + 1);
constexpr int kSharedSmemMax = 232448;
constexpr int kPieces = 4;  // pieces known ahead
constexpr int kGroup = 16;  // positions that one step of the products takes; tiles start on multiples
// registers of a thread: 96 at the launch, of which the last four warps give some to the others
constexpr int kSoftRegs = 112, kSumRegs = 96, kLastRegs = 64;
static_assert(kSharedThreads == 640 && 256 * kSoftRegs + 256 * kSumRegs + 128 * kLastRegs <= 640 * 96, "register split");

template <int HD, int QT, int PT>
struct Tm {
    static constexpr int kTileBytes = kTile * HD * 2;  // K or V rows of a tile, and one term of Q
    static constexpr int kQBufs = QT == 1 ? 2 : 1;
    static constexpr int kQ = kQBufs * QT * kTileBytes;
    static constexpr int kFixed = 1024 + 19456;  // alignment, then barriers and small tables
    static constexpr int kFit = (kSharedSmemMax - kFixed - kQ) / kTileBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    // V's tiles share the barriers of the two P that they are multiplied with
    static constexpr int kStagesV = kStages >= 4 ? 2 : 1, kStagesK = kStages - kStagesV > 4 ? 4 : kStages - kStagesV;
    // copies that a copying thread leaves in flight behind the one it has just issued
    static constexpr int kAhead = kStages - 2 > 4 ? 4 : kStages - 2;
    static_assert(kStages >= 3, "three tiles must fit");
    static constexpr int kTotal = kFixed + kQ + (kStagesK + kStagesV) * kTileBytes;
    // tensor memory: two S, three where they fit beside two T (P over it, a third term behind it), then T.
    // (Three S and one T for 128 dimensions: 64 rows behind 32K 166 -> 153 us, a prompt 149 -> 150, but 897
    // rows of 32 requests, 8 / 2 heads of 96, capped, 69 -> 80, and 692 fp32 rows, pages of 100, 242 -> 256.)
    static constexpr int kSCols = PT == 3 ? 192 : 128;
    static constexpr int kSBufs = 3 * kSCols + 2 * HD <= 512 ? 3 : 2;
    static constexpr int kTBufs = kSBufs * kSCols + 2 * HD <= 512 ? 2 : 1;
    static_assert(kSBufs * kSCols + kTBufs * HD <= 512, "tensor memory plan");
};

// Tiles [t0, t1) of an item, as the planning warp lays them out for the others.
struct Piece {
    int row0, rows, lo, hi, tr, t0, t1;
    int kind;  // of the bits below
    __device__ __forceinline__ int start(int t) const { return (lo & ~15) + t * kTile; }
};
constexpr int kPieceStart = 1, kPieceWhole = 2, kPieceOwn = 4, kPieceLast = 8;  // kPieceLast: no piece, the share is done

struct SmallShared {
    uint64_t k_full[4], k_empty[4], q_full[2], q_empty[2];
    uint64_t s_full[3];  // S of tiles j, j + 1, j + 2 (and where there are two K, their places are free)
    uint64_t ready[3];   // their P, V and a place for T
    uint64_t t_full[2];  // their T (and V's places are free)
    uint64_t piece_full[kPieces], piece_empty[kPieces];
    uint32_t tmem;
    int dead;                    // a wait gave up
    alignas(16) uint32_t bad[8][4];          // positions of a tile whose page does not exist
    Piece piece[kPieces];
    int4 row[kPieces][kTile];    // of a row of the product: first and end position, length, 1 + (all of the row: 2); 0: no row
    float2 stats[8][kTile];      // m (log2 units) and l of a tile's rows; the exponentials are up to 4 tiles ahead of O
    float factor[kPieces][kTile];  // what an accumulator of S is times for a score
};
static_assert(sizeof(SmallShared) <= 19456, "");

// Waits for a barrier's phase; by a warp, one answer for all lanes.  A wait that
// does not end (some 0.1 s at least, 4 s where every try sleeps a microsecond)
// gives up: `dead` is set, and the call's rows become NaN.  Small, as it stands
// in every role: what the roles run per tile has to stay in the SM's instruction
// cache (with the clock in this loop, and copies and pages unrolled, the GPC's
// was 65 % busy and everything four times as slow).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* dead) {
#pragma unroll 1
    for (int n = 0; n < (1 << 22); n++)
        if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    *dead = 1;
    return false;
}

// K and V tiles: 8 positions by 64 dimensions are 1024 bytes in the 128-byte
// swizzle, a position a line of 128; the 64-dimension blocks of 8 positions
// follow one another, then the next 8 positions.  The byte of dimension 8 c
// (c: its 16-byte chunk) of position row:
template <int BL>
__device__ __forceinline__ uint32_t kv_at(int row, int c) {
    return (row >> 3) * (BL * 1024) + (c >> 3) * 1024 + (row & 7) * 128 + (((c & 7) ^ (row & 7)) << 4);
}
// K as the second operand: 8 positions are BL * 1024 bytes on (stride).  V: its
// rows are the products' K, so that is again the stride, and the blocks of
// dimensions are 1024 apart (leading).
template <int BL>
__device__ __forceinline__ uint64_t kv_desc() {
    return ((uint64_t)(1024u >> 4) << 16) | ((uint64_t)((BL * 1024u) >> 4) << 32) | ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

__device__ __forceinline__ uint64_t desc_of(uint32_t lo, uint32_t hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}

template <typename C>
__device__ __forceinline__ uint32_t idesc(int n, bool v) {
    const uint32_t type = std::is_same<C, __half>::value ? 0u : 1u;
    return (1u << 4) | (type << 7) | (type << 10) | ((v ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// 16 columns of this thread's lane, on their way until tmem_wait16 of the same
// registers.
__device__ __forceinline__ void tmem_get16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// (the registers pass through, so that nothing reads them before)
__device__ __forceinline__ void tmem_wait16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}

// 16 bytes from global to shared memory where `go`; `valid` false: zeros.  No
// branch, so that a run of them is issued back to back.
__device__ __forceinline__ void cp16_if(uint32_t smem, const void* gmem, bool valid, bool go) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\t"
        "@p cp.async.cg.shared.global [%0], [%1], 16, %2;\n\t}" ::"r"(smem),
        "l"(gmem), "r"(valid ? 16 : 0), "r"((uint32_t)go)
        : "memory");
}

// The same of a map over all positions of a pool, 8 by 8: all dimensions of a
// head, positions from 8 * eight on.
__device__ __forceinline__ void tma_eights(uint32_t smem, const CUtensorMap* map, int eight, int head, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], [%5];" ::
            "r"(smem),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(eight), "r"(head), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// A box of a tensor map to shared memory: of a cache's, 64 dimensions from x on,
// one head, kGroup or 8 positions from pos on, one page; of Q's, 64 dimensions,
// an item's heads, its rows, one term.
__device__ __forceinline__ void tma_rows(uint32_t smem, const CUtensorMap* map, int x, int head, int pos, int page, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(smem),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(pos), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// tanh; its error is times the cap in a score.  16-bit rows: 1 - 2 / (1 + e^2x), off by
// 2^-23, so 2^-17 in a score at a cap of 50 (tanhf in its place: 37 -> 40 us for 16
// ragged requests); fp32 rows: to the last bits.
template <bool EXACT>
__device__ __forceinline__ float tanh_of(float x) {
    return EXACT ? tanhf(x) : 1.0f - __fdividef(2.0f, 1.0f + ex2(x * (2.0f * kLog2e)));
}

// One lane of a converged warp, chosen so that the compiler knows of it: the
// products' descriptors live in the warp's uniform registers.  (With lane == 0
// in place of this and unrolled loops, one product of eight got its
// predecessor's descriptor.)
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Where a warp is in the pieces.
struct Pieces {
    int n = 0;  // pieces taken
    // the next one (of its slot), or null: no more, or a wait gave up
    __device__ __forceinline__ const Piece* next(SmallShared& s) {
        const int slot = n % kPieces;
        if (!warp_wait(&s.piece_full[slot], (n / kPieces) & 1, &s.dead)) return nullptr;
        n++;
        return s.piece[slot].kind & kPieceLast ? nullptr : &s.piece[slot];
    }
    // the warp is done with the one taken last
    __device__ __forceinline__ void done(SmallShared& s) const {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&s.piece_empty[(n - 1) % kPieces]);
    }
};

template <int HD, typename T, typename C, int QT, int PT>
__global__ void __launch_bounds__(kSharedThreads, 1)
    shared_tiles_kernel(const __grid_constant__ SharedArgs a, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q) {
    using TM = Tm<HD, QT, PT>;
    constexpr int NK = TM::kStagesK, NV = TM::kStagesV, NS = TM::kSBufs, NT = TM::kTBufs, QB = TM::kQBufs;
    extern __shared__ __align__(1024) uint8_t ssm_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ssm_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const q_sm = base;
    uint8_t* const ring = base + TM::kQ;
    SmallShared& s = *reinterpret_cast<SmallShared*>(ring + (NK + NV) * TM::kTileBytes);
    volatile int* dead = &s.dead;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int heads = a.nkv * a.blocks;
    const int share = blockIdx.x / heads, hr = blockIdx.x - share * heads;
    const int h = hr / a.blocks, blk = hr - h * a.blocks;  // KV head, block of its query heads
    const int head0 = h * a.grp + blk * a.hb, hn = min(a.hb, a.grp - blk * a.hb);
    const int hd = a.hd;

    if (tid == 0) {
        const int copies = a.box ? 1 : kCopyWarps;
        for (int i = 0; i < 4; i++) {
            mbar_init(&s.k_full[i], copies);
            mbar_init(&s.k_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s.q_full[i], 1);
            mbar_init(&s.q_empty[i], 1);
            mbar_init(&s.t_full[i], 1);
        }
        for (int i = 0; i < NS; i++) {
            mbar_init(&s.s_full[i], 1);
            mbar_init(&s.ready[i], 4 + kSumWarps + copies);
        }
        for (int i = 0; i < kPieces; i++) {
            mbar_init(&s.piece_full[i], 1);
            mbar_init(&s.piece_empty[i], kSoftWarps + kSumWarps + kCopyWarps + 1);
        }
        s.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // columns past hd stay zero: the copies never write them
    if (hd < HD) {
        for (int i = tid; i < (TM::kQ + (NK + NV) * TM::kTileBytes) / 16; i += kSharedThreads)
            *reinterpret_cast<uint4*>(base + 16 * i) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s.tmem;
    pdl_wait();
    pdl_trigger();

    if (warp < kSoftWarps) {
        // ------------------------------------------------------------ exponentials
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int wg = warp >> 2, quad = warp & 3, m = quad * 32 + lane;
        const uint32_t s_row = tmem + ((uint32_t)(quad * 32) << 16);
        const float cap = a.softcap;
        const bool plain = !(cap > 0.0f) && !a.slopes;
        float slope = 0.0f;
        if (a.slopes && m % a.hb < hn) slope = a.slopes[head0 + m % a.hb] * kLog2e;
        const float f_all = cap > 0.0f ? a.scale / cap : a.scale * kLog2e;
        int j = 0, sb = 0, lap = 0;
        auto next_s = [&]() {
            if (++sb == NS) {
                sb = 0;
                lap ^= 1;
            }
        };
        Pieces pieces;
        while (const Piece* p = pieces.next(s)) {
            const int slot = (pieces.n - 1) % kPieces;
            const int4 row = s.row[slot][m];
            const int start = p->start(0), it_hi = p->hi, t1 = p->t1;
            const bool busy = __any_sync(0xffffffffu, row.w != 0);
            bool ok = true;
            for (int t = p->t0; t < t1; t++, j++, next_s()) {
                if ((j & 1) != wg) continue;
                const uint32_t s_col = s_row + sb * TM::kSCols;
                if (!warp_wait(&s.s_full[sb], lap, dead)) {
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (busy) {
                    const int p0 = start + t * kTile, c0 = row.x - p0, c1 = row.y - p0;
                    const int chunks = (min(kTile, it_hi - p0) + 31) / 32;
                    const bool mask = __any_sync(0xffffffffu, c0 > 0 || c1 < 32 * chunks);
                    float f = QT == 1 ? f_all : s.factor[slot][m];
                    if (!plain) {  // cap and slope
#pragma unroll 1
                        for (int c = 0; c < 32 * chunks; c += 16) {
                            uint32_t r[16];
                            tmem_ld16(s_col + c, r);
                            const float p1 = (float)(p0 - (row.z - 1) + c);
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                float x = __uint_as_float(r[i]) * f;
                                if (cap > 0.0f) x = (cap * kLog2e) * tanh_of<std::is_same<T, float>::value>(x);
                                r[i] = __float_as_uint(fmaf(slope, p1 + (float)i, x));
                            }
                            tmem_st16(s_col + c, r);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        f = 1.0f;
                    }
                    if (mask) {  // the scores that are not seen to -inf
#pragma unroll 1
                        for (int c = 0; c < 32 * chunks; c += 16) {
                            const int lo = min(max(c0 - c, 0), 16), hi = min(max(c1 - c, 0), 16);
                            const uint32_t seen = hi > lo ? ((1u << hi) - 1) & ~((1u << lo) - 1) : 0;
                            if (__all_sync(0xffffffffu, seen == 0xffff)) continue;
                            uint32_t r[16];
                            tmem_ld16(s_col + c, r);
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (!(seen >> i & 1)) r[i] = 0xff800000u;
                            tmem_st16(s_col + c, r);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    }
                    // 16 columns on their way while 16 are worked on, in loops that the instruction
                    // cache next to the scheduler holds
                    uint32_t ra[16], rb[16];
                    float x0 = -INFINITY, x1 = -INFINITY;
                    auto largest = [&](const uint32_t* r) {
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            x0 = fmaxf(fmaxf(x0, __uint_as_float(r[i])), __uint_as_float(r[i + 1]));
                            x1 = fmaxf(fmaxf(x1, __uint_as_float(r[i + 2])), __uint_as_float(r[i + 3]));
                        }
                    };
                    const uint32_t end = s_col + 32 * chunks;
                    tmem_get16(s_col, ra);
#pragma unroll 1
                    for (uint32_t c = s_col; c < end; c += 32) {
                        tmem_wait16(ra);
                        tmem_get16(c + 16, rb);
                        largest(ra);
                        tmem_wait16(rb);
                        tmem_get16(c + 32 < end ? c + 32 : s_col, ra);  // (at the end, the first columns again)
                        largest(rb);
                    }
                    const float mx = fmaxf(x0, x1);
                    const float top = mx == -INFINITY ? -INFINITY : mx * f, z = 14.0f - (top == -INFINITY ? 0.0f : top);
                    const unsigned long long f2 = f2_pack(f, f), z2 = f2_pack(z, z);
                    unsigned long long l2 = 0, l3 = 0;
                    auto weigh = [&](const uint32_t* r, uint32_t to, uint32_t third) {
                        uint32_t w[PT][8];
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float2 d = f2_unpack(f2_fma(f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), f2, z2));
                            const float e0 = ex2(d.x), e1 = ex2(d.y);
                            if (i & 1) l2 = f2_add(l2, f2_pack(e0, e1));
                            else l3 = f2_add(l3, f2_pack(e0, e1));
                            uint32_t x[PT];
                            split_terms<C, PT>(e0, e1, x);
#pragma unroll
                            for (int k = 0; k < PT; k++) w[k][i] = x[k];
                        }
                        tmem_st8(to, w[0]);
                        if (PT > 1) tmem_st8(to + 8, w[PT > 1 ? 1 : 0]);
                        if (PT == 3) tmem_st8(third, w[PT - 1]);
                    };
#pragma unroll 1
                    for (uint32_t c = s_col, th = s_col + 128; c < end; c += 32, th += 16) {
                        tmem_wait16(ra);
                        tmem_get16(c + 16, rb);
                        weigh(ra, c, th);
                        tmem_wait16(rb);
                        if (c + 32 < end) tmem_get16(c + 32, ra);
                        weigh(rb, c + 16, th + 8);
                    }
                    l2 = f2_add(l2, l3);
                    const float2 ls = f2_unpack(l2);
                    float l = ls.x + ls.y;
                    const uint32_t* bad = s.bad[j & 7];
                    const uint4 any = *reinterpret_cast<const uint4*>(bad);
                    if (any.x | any.y | any.z | any.w) {
#pragma unroll 1
                        for (int c = max(c0, 0); c < min(c1, kTile); c++)
                            if ((bad[c >> 5] >> (c & 31)) & 1) l = __int_as_float(0x7fc00000);
                    }
                    s.stats[j & 7][m] = make_float2(top, l);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.ready[sb]);
            }
            if (!ok) break;
            pieces.done(s);
        }
    } else if (warp < kSoftWarps + kSumWarps) {
        // ------------------------------------------------------------ O
        constexpr int HC = HD / 2;  // columns of a warp
        const int half = (warp - kSoftWarps) >> 2, quad = warp & 3, m = quad * 32 + lane;
        const uint32_t t_col = tmem + ((uint32_t)(quad * 32) << 16) + NS * TM::kSCols + half * HC;
        const int rr = m / a.hb, head = head0 + m - rr * a.hb;
        const int d0 = half * HC, dn = min(HC, hd - d0);  // this warp's dimensions
        if (lane == 0)  // (T's places are free)
            for (int i = 0; i < NT; i++) mbar_arrive(&s.ready[i]);
        int j = 0, freed = NT % NS;  // freed: the tile that gets this one's place for T, of those `ready` knows
        bool ok = true;
        auto release = [&]() {  // T has been read
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&s.ready[freed]);
            if (++freed == NS) freed = 0;
        };
        Pieces pieces;
        while (const Piece* p = pieces.next(s)) {
            const int4 row = s.row[(pieces.n - 1) % kPieces][m];
            const bool busy = __any_sync(0xffffffffu, row.w != 0);
            unsigned long long o[HC / 2];
            float M = -INFINITY, L = 0.0f;
#pragma unroll
            for (int i = 0; i < HC / 2; i++) o[i] = 0;
            const int t1 = p->t1;
#pragma unroll 1
            for (int t = p->t0; t < t1; t++, j++) {
                const int buf = j % NT;
                ok = ok && warp_wait(&s.t_full[j & 1], (j >> 1) & 1, dead);
                if (!ok) continue;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (busy) {
                    const float2 st = s.stats[j & 7][m];
                    const float n = fmaxf(M, st.x), z = n == -INFINITY ? 0.0f : n;
                    const float fo = ex2(M - z), ft = ex2(st.x - z);
                    M = n;
                    L = fmaf(L, fo, st.y * ft);
                    const unsigned long long fo2 = f2_pack(fo, fo), ft2 = f2_pack(ft, ft);
                    const uint32_t from = t_col + buf * HD;
#pragma unroll
                    for (int c = 0; c < HC; c += 16) {
                        uint32_t r[16];
                        tmem_ld16(from + c, r);
                        if (c + 16 >= HC) release();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const unsigned long long x = f2_pack(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                            o[c / 2 + i] = f2_fma(o[c / 2 + i], fo2, f2_mul(x, ft2));
                        }
                    }
                } else {
                    release();
                }
            }
            const int b = p->row0 + rr, kind = p->kind;
            pieces.done(s);
            if (!row.w || dn <= 0) continue;
            if ((kind & kPieceWhole) && (row.w & 2)) {  // all that the row sees
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                T* out = static_cast<T*>(a.out) + (int64_t)b * a.out_stride + (int64_t)head * hd + d0;
                bool odd = false;  // not finite
#pragma unroll
                for (int i = 0; i < HC / 8; i++) {
                    if (8 * i >= dn) break;
                    alignas(16) T y[8];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float2 x = f2_unpack(o[4 * i + k]);
                        const float u = x.x * inv, v = x.y * inv;
                        odd |= u - u != 0.0f || v - v != 0.0f;
                        y[2 * k] = (T)u;
                        y[2 * k + 1] = (T)v;
                    }
                    if (a.out_wide) {
#pragma unroll
                        for (int k = 0; k < (int)sizeof(T) / 2; k++)
                            reinterpret_cast<uint4*>(out + 8 * i)[k] = reinterpret_cast<const uint4*>(y)[k];
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; k++) out[8 * i + k] = y[k];
                    }
                }
                if (a.lse && half == 0) a.lse[(int64_t)b * a.nh + head] = L == 0.0f ? -INFINITY : (M + (log2f(L) - 14.0f)) * kLn2;
                if (odd) a.redo[b] = 1;
            } else {
                const int64_t width = hd + 4;
                float* to = kind & kPieceWhole
                                ? a.whole + (((int64_t)(kind & kPieceOwn ? 1 : 0) * a.batch + b) * a.nh + head) * width
                                : a.part + (((int64_t)blockIdx.x * 2 + (kind & kPieceStart ? 1 : 0)) * kTile + m) * width;
#pragma unroll
                for (int i = 0; i < HC / 4; i++) {
                    if (4 * i >= dn) break;
                    const float2 x = f2_unpack(o[2 * i]), y = f2_unpack(o[2 * i + 1]);
                    *reinterpret_cast<float4*>(to + d0 + 4 * i) = make_float4(x.x, x.y, y.x, y.y);
                }
                if (half == 0) *reinterpret_cast<float2*>(to + hd) = make_float2(M, L);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLastRegs));
        asm volatile("fence.proxy.async;" ::: "memory");  // what the launches before wrote, for the TMA copies
        if (warp < kQWarp) {
            // -------------------------------------------------------- K and V
            const int lw = warp - kCopyWarp, hc = hd / 8;
            const uint32_t ring_k = smem_u32(ring), ring_v = ring_k + NK * TM::kTileBytes;
            int j = 0;
            Pieces pieces;
            const Piece* p = pieces.next(s);
            int t = p ? p->t0 : 0;
            bool ok = true;
            auto page_at = [&](const Piece* q, int pos) { return a.table[(int64_t)q->tr * a.table_stride + page_of(a, pos)]; };
            auto place = [&](int pos) { return pos - page_of(a, pos) * a.page_size; };  // in its page
            if (a.box) {
                // K by the first warp, V by the second.  Groups of `box` positions that lie in one
                // page: seen whole, a tensor map's box each; in part, or in no page, row by row.
                // The products take 16 positions at a time, so rows of V up to there that nobody
                // sees are zeros.
                const int G = a.box, groups = kTile / G;
                const bool value = lw != 0;
                const CUtensorMap* map = value ? &map_v : &map_k;
                const uint16_t* src = value ? a.v : a.k;
                const int slots = value ? NV : NK;
                const uint32_t ring_s = value ? ring_v : ring_k;
                int slot = 0;
                constexpr int BL = HD / 64;  // boxes of a group
                const uint32_t all = (1u << groups) - 1;
                const int r0 = lane * G;
                // the piece: first position of its next tile, seen positions, table row; this lane's place in it
                int p0 = 0, p_lo = 0, p_hi = 0;
                const int32_t* row = nullptr;
                auto enter = [&]() {
                    if (!p) return;
                    t = p->t1 - p->t0;
                    p0 = p->start(p->t0);
                    p_lo = p->lo;
                    p_hi = p->hi;
                    row = a.table + (int64_t)p->tr * a.table_stride;
                };
                auto look = [&]() {  // this lane's group: its page (any position of it that is seen names it)
                    const int lo = max(p_lo - p0, r0);
                    if (lane >= groups || lo >= r0 + G || lo >= p_hi - p0) return -1;
                    return row[page_of(a, p0 + lo)];
                };
                enter();
                int nx = p ? look() : -1;
#pragma unroll 1
                while (p) {
                    const int page = nx, lo_t = p_lo - p0, hi_t = min(kTile, p_hi - p0), in = r0 < hi_t ? place(p0 + r0) : 0;
                    if (--t == 0) {
                        pieces.done(s);
                        p = pieces.next(s);
                        enter();
                    } else {
                        p0 += kTile;
                    }
                    if (p) nx = look();  // (the next tile's pages, on their way meanwhile)
                    const bool there = (unsigned)page < (unsigned)a.n_pages;
                    const bool whole = lane < groups && there && r0 >= lo_t && r0 + G <= hi_t;
                    const int where = a.flat ? page * a.page_size + in : in;
                    const uint32_t by_box = __ballot_sync(0xffffffffu, whole);
                    uint32_t rest = 0, bits = 0;
                    if (by_box != all) {
                        rest = __ballot_sync(0xffffffffu, lane < groups && !whole && r0 < ((hi_t + kGroup - 1) & ~(kGroup - 1)));
                        // positions seen whose page is not there
                        const int lo = max(lo_t, r0), hi = min(hi_t, r0 + G);
                        const bool gone = lane < groups && lo < hi && !there;
                        const uint32_t mine = gone ? ((1u << (hi - lo)) - 1) << (lo & 31) : 0;
#pragma unroll 1
                        for (int i = 0; i < 4; i++) {
                            const uint32_t b = __reduce_or_sync(0xffffffffu, (lo >> 5) == i ? mine : 0);
                            if (lane == i) bits = b;
                        }
                    }
                    if (!value && lane < 4) s.bad[j & 7][lane] = bits;
                    // the tile's place is free once the one before in it was multiplied
                    const int was = j - slots;
                    if (was >= 0)
                        ok = ok && (value      ? warp_wait(&s.t_full[was & 1], (was >> 1) & 1, dead)
                                    : NK == 2 ? warp_wait(&s.s_full[was % NS], (was / NS) & 1, dead)
                                              : warp_wait(&s.k_empty[slot], (was / NK) & 1, dead));
                    if (!ok) break;
                    uint64_t* bar = value ? &s.ready[j % NS] : &s.k_full[slot];
                    const uint32_t to = __shfl_sync(0xffffffffu, ring_s + slot * TM::kTileBytes, 0);
                    __syncwarp();  // (the lanes' s.bad before the arrival that the exponentials wait for)
                    const bool one = elected();
                    if (one) {
                        const uint32_t bytes = __popc(by_box) * G * 128 * BL;
                        if (rest) mbar_expect_tx(bar, bytes);
                        else mbar_arrive_expect_tx(bar, bytes);
                    }
                    __syncwarp();
                    if (a.flat == 2) {
                        if (whole) tma_eights(to + lane * (G * 128 * BL), map, where >> 3, h, bar);
                    } else if (whole) {
#pragma unroll 1
                        for (int r = 0, x = 0; r < G; x++) {  // (a box: of 8 positions where there are blocks)
                            tma_rows(to + lane * (G * 128 * BL) + r * (128 * BL) + x * 1024, map, 64 * x, h, where + r, a.flat ? 0 : page, bar);
                            if (x == BL - 1) {
                                r += BL == 1 ? G : 8;
                                x = -1;
                            }
                        }
                    }
                    __syncwarp();
                    if (rest) {
                        while (rest) {
                            const int g = __ffs(rest) - 1;
                            rest &= rest - 1;
                            const int pg = __shfl_sync(0xffffffffu, page, g), at = __shfl_sync(0xffffffffu, in, g);
                            const bool in_pool = (unsigned)pg < (unsigned)a.n_pages;
                            const uint16_t* from = src + (in_pool ? pg * a.page_stride + at * a.pos_stride : 0) + h * a.head_stride;
#pragma unroll 2
                            for (int i = lane; i < G * hc; i += 32) {
                                const int r = i / hc, c = i - r * hc, rt = g * G + r;
                                const bool seen = in_pool && rt >= lo_t && rt < hi_t;
                                cp16_if(to + kv_at<BL>(rt, c), seen ? from + r * a.pos_stride + c * 8 : src, seen, seen || value);
                            }
                        }
                        cp_async_commit();
                        cp_wait<0>();
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar);
                    }
                    if (++slot == slots) slot = 0;
                    j++;
                }
            } else {
                // Pages of any size and place: row by row, half of the tile's rows to a warp.
                constexpr int RW = kTile / kCopyWarps;
                constexpr int CH = HD / 8, LR = 32 / CH;  // chunks of a row, rows of a warp's copy
                const int row0 = lw * RW + lane, c = lane % CH, r0 = lane / CH;
                const uint32_t at0 = ring_k + kv_at<HD / 64>(lw * RW, 0);
                const int64_t h_off = (int64_t)h * a.head_stride + c * 8;
                int issued[2] = {0, 0}, told[2] = {0, 0};  // tiles of K, of V, and those that the products know of
                int waiting = 0;                           // stages issued that they do not know of,
                uint32_t kinds = 0;                        // and what these are (V: 1), the last in bit 0
                bool have = false;
                auto tell = [&](int leave) {  // all but the last `leave` stages have landed
                    fence_proxy_async();
                    __syncwarp();
                    for (; waiting > leave; waiting--) {
                        const bool v = (kinds >> (waiting - 1)) & 1;
                        const int n = v ? told[1]++ : told[0]++;
                        if (lane == 0) mbar_arrive(v ? &s.ready[n % NS] : &s.k_full[n % NK]);
                    }
                };
                // this lane's rows of a tile: their offset; -1: none there; -2: nor needed
                struct Place {
                    int64_t off[RW / 32];
                };
                struct Look {  // looked up, not yet used
                    int page[RW / 32], pos, lo, hi;
                };
                auto look = [&](const Piece* q, int tt) {
                    Look f;
                    const int p0 = q->start(tt);
                    f.lo = q->lo - p0;
                    f.hi = min(kTile, q->hi - p0);
                    f.pos = p0 + row0;
#pragma unroll
                    for (int i = 0; i < RW / 32; i++) {
                        const int r = row0 + 32 * i;
                        f.page[i] = r >= f.lo && r < f.hi ? page_at(q, f.pos + 32 * i) : -1;
                    }
                    return f;
                };
                auto issue = [&](const uint16_t* src, const Place& f, bool value) {
                    const int n = value ? issued[1]++ : issued[0]++, slots = value ? NV : NK, slot = n % slots, was = n - slots;
                    if (was >= 0) {
                        uint64_t* bar = value ? &s.t_full[was & 1] : NK == 2 ? &s.s_full[was % NS] : &s.k_empty[slot];
                        const uint32_t parity = (value ? was >> 1 : NK == 2 ? was / NS : was / NK) & 1;
                        if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
                            cp_wait<0>();  // (what frees it may wait for what is on its way)
                            tell(0);
                            ok = ok && warp_wait(bar, parity, dead);
                        }
                    }
                    if (!ok) return;
                    const uint32_t to = at0 + (slot + (value ? NK : 0)) * TM::kTileBytes;
                    constexpr int U = 4;  // copies whose places are worked out together
#pragma unroll
                    for (int i0 = 0; i0 < RW / LR; i0 += U) {
                        int64_t o[U];
#pragma unroll
                        for (int u = 0; u < U; u++) o[u] = __shfl_sync(0xffffffffu, f.off[(i0 + u) * LR / 32], ((i0 + u) * LR + r0) & 31);
#pragma unroll
                        for (int u = 0; u < U; u++) {
                            const int r = (i0 + u) * LR + r0;
                            const uint32_t at = to + kv_at<HD / 64>(r, c);  // (lw * RW is a multiple of 8)
                            cp16_if(at, src + (o[u] < 0 ? 0 : o[u] + h_off), o[u] >= 0, c < hc && (o[u] >= 0 || (value && o[u] == -1)));
                        }
                    }
                    cp_async_commit();
                    kinds = kinds << 1 | (value ? 1 : 0);
                    if (++waiting > TM::kAhead) {
                        cp_wait<TM::kAhead>();
                        tell(TM::kAhead);
                    }
                };
                Place v{};
                Look nx{};
                if (p) nx = look(p, t);
                while (ok && p) {
                    const Look now = nx;
                    if (++t == p->t1) {
                        pieces.done(s);
                        // (the piece that comes may wait for what is on its way)
                        if (!__all_sync(0xffffffffu, mbar_try_wait(&s.piece_full[pieces.n % kPieces], (pieces.n / kPieces) & 1))) {
                            cp_wait<0>();
                            tell(0);
                        }
                        p = pieces.next(s);
                        t = p ? p->t0 : 0;
                    }
                    if (p) nx = look(p, t);
                    Place f;
#pragma unroll
                    for (int i = 0; i < RW / 32; i++) {
                        const int r = row0 + 32 * i;
                        f.off[i] = r < ((now.hi + kGroup - 1) & ~(kGroup - 1)) ? -1 : -2;
                        const bool in = r >= now.lo && r < now.hi, there = in && (unsigned)now.page[i] < (unsigned)a.n_pages;
                        if (there) f.off[i] = now.page[i] * a.page_stride + (int64_t)place(now.pos + 32 * i) * a.pos_stride;
                        const uint32_t bad = __ballot_sync(0xffffffffu, in && !there);
                        if (lane == 0) s.bad[j & 7][lw * (RW / 32) + i] = bad;
                    }
                    issue(a.k, f, false);
                    if (ok && have) issue(a.v, v, true);
                    v = f;
                    have = true;
                    j++;
                }
                if (ok && have) issue(a.v, v, true);
                cp_wait<0>();
                if (ok) tell(0);
            }
        } else if (warp == kQWarp) {
            // -------------------------------------------------------- pieces and Q
            const Share mine = share < a.shares ? a.share[share] : Share{0, 0, 0};
            const int items = a.line->items;
            long long left = mine.units;  // units of this share that are left
            int next = mine.item, at = mine.at;
            Item ahead{};
            auto load = [&]() {
                if (next < items) {
                    const int4* from = reinterpret_cast<const int4*>(a.item + next);
                    reinterpret_cast<int4*>(&ahead)[0] = from[0];
                    reinterpret_cast<int4*>(&ahead)[1] = from[1];
                }
            };
            if (left > 0) load();
            bool ok = true;
            // lays out piece n; false: there is none
            auto plan = [&](int n) {
                const int slot = n % kPieces;
                if (n >= kPieces) ok = ok && warp_wait(&s.piece_empty[slot], (n / kPieces - 1) & 1, dead);
                if (!ok) return false;
                Piece p{};
                p.kind = kPieceLast;
                int limit = 0;
                while (left > 0 && next < items) {
                    const Item it = ahead;
                    next++;
                    load();
                    const int tiles = tiles_of(it), x = at, take = (int)min((long long)(tiles + kItemUnits - x), left);
                    left -= take;
                    at = 0;
                    p.t0 = max(0, x - kItemUnits);
                    p.t1 = max(0, x + take - kItemUnits);
                    if (p.t1 == p.t0) continue;
                    p.row0 = it.row0;
                    p.rows = it.rows;
                    p.lo = it.lo;
                    p.hi = it.hi;
                    p.tr = it.tr;
                    limit = it.limit;
                    p.kind = (p.t0 == 0 ? kPieceStart : 0) | (p.t0 == 0 && p.t1 == tiles ? kPieceWhole : 0) |
                             (it.limit == kNoLimit ? kPieceOwn : 0);
                    break;
                }
                if (!(p.kind & kPieceLast)) {
#pragma unroll
                    for (int i = 0; i < kTile / 32; i++) {
                        const int m = 32 * i + lane, rr = m / a.hb;
                        int4 w = make_int4(0, 0, 0, 0);
                        if (rr < p.rows && m - rr * a.hb < hn) {
                            const int4 r = a.row[p.row0 + rr];
                            const bool all = (p.kind & kPieceOwn ? r.z : r.w) < 0;
                            w = make_int4(max(r.x, p.lo), min(r.y, limit), r.y, all ? 3 : 1);
                            if (QT > 1) s.factor[slot][m] = a.factor[(int64_t)(p.row0 + rr) * a.nh + head0 + m - rr * a.hb];
                        }
                        s.row[slot][m] = w;
                    }
                }
                if (lane == 0) s.piece[slot] = p;
                __syncwarp();
                if (lane == 0) mbar_arrive(&s.piece_full[slot]);
                return !(p.kind & kPieceLast);
            };
            auto bring = [&](int n) {  // Q of piece n: rows that are not the item's come along, and are not looked at
                if (n >= QB) ok = ok && warp_wait(&s.q_empty[n % QB], (n / QB - 1) & 1, dead);
                if (!ok) return;
                uint64_t* bar = &s.q_full[n % QB];
                const uint32_t to = smem_u32(q_sm) + (n % QB) * QT * TM::kTileBytes;
                const int row0 = s.piece[n % kPieces].row0;
                if (elected()) {
                    mbar_arrive_expect_tx(bar, a.hb * a.rows * 128 * (HD / 64) * QT);
#pragma unroll
                    for (int x = 0; x < QT; x++)
#pragma unroll
                        for (int k = 0; k < HD / 64; k++)
                            tma_rows(to + x * TM::kTileBytes + k * (kTile * 128), &map_q, 64 * k, head0, row0, x, bar);
                }
                __syncwarp();
            };
            bool more = plan(0);
            for (int n = 0; ok && more; n++) {
                more = plan(n + 1);
                if (ok) bring(n);
            }
        } else {
            // -------------------------------------------------------- products
            // (values that go into descriptors are shuffled from lane 0, which keeps them, and
            // the sums with constants below, in the warp's uniform registers)
            auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
            const uint32_t ring_k = smem_u32(ring) >> 4, ring_v = ring_k + NK * (TM::kTileBytes >> 4), q_s = smem_u32(q_sm) >> 4;
            constexpr int BL = HD / 64;
            const uint32_t hi_q = (uint32_t)(sw128_desc(0) >> 32), lo_q = (uint32_t)sw128_desc(0);
            const uint32_t hi_kv = (uint32_t)(kv_desc<BL>() >> 32), lo_kv = (uint32_t)kv_desc<BL>();
            const int ks = (hd + 15) / 16;
            const uint32_t id_v = uniform(idesc<C>(ks * 16, true)), id_k = uniform(idesc<C>(0, false));
            const uint32_t tm = uniform(tmem);
            constexpr int LAG = NS - 1;  // S is this many tiles ahead of T
            int j = 0, was[LAG] = {};    // was: positions of the tiles between, in 16s, the oldest first
            int sb = 0;                  // S's place
            int vb = 0, v_lap = 0;       // and that of the next tile whose T is made
            int k_slot = 0, k_lap = 0;
            bool ok = true, k_there = false;  // k_there: the next tile's K was waited for
            auto values = [&](int jj, bool more) {  // T = P V of tile jj
                // (K first: it is there as a rule, and every wait takes its time)
                k_there = more && (LAG == 1 || a.box);
                if (k_there) ok = ok && warp_wait(&s.k_full[k_slot], k_lap & 1, dead);
                ok = ok && warp_wait(&s.ready[vb], v_lap, dead);
                if (!ok) return;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t b = uniform(jj & 1), n = uniform(was[0]);
                const uint32_t v = lo_kv + ring_v + (NV == 2 ? b : 0) * (TM::kTileBytes >> 4);
                const uint32_t pc = tm + uniform(vb) * TM::kSCols, tc = tm + NS * TM::kSCols + (NT == 2 ? b : 0) * HD;
                if (elected()) {
                    if (n == kTile / 16) {
#pragma unroll
                        for (int x = PT - 1; x >= 0; x--)  // (small terms first)
#pragma unroll
                            for (int k = 0; k < kTile / 16; k++)
                                mma_f16_ts(tc, pc + (x == 2 ? 128 + 8 * k : 16 * k + 8 * x), desc_of(v + k * ((2 * BL * 1024) >> 4), hi_kv), id_v,
                                           x < PT - 1 || k > 0);
                    } else {
                        uint32_t acc = 0;
#pragma unroll 1
                        for (int x = PT - 1; x >= 0; x--)
#pragma unroll 1
                            for (uint32_t k = 0; k < n; k++) {
                                mma_f16_ts(tc, pc + (x == 2 ? 128 + 8 * k : 16 * k + 8 * x), desc_of(v + k * ((2 * BL * 1024) >> 4), hi_kv), id_v, acc);
                                acc = 1;
                            }
                    }
                    mma_commit(&s.t_full[jj & 1]);
                }
                __syncwarp();
                if (++vb == NS) {
                    vb = 0;
                    v_lap ^= 1;
                }
                for (int i = 0; i + 1 < LAG; i++) was[i] = was[i + 1];
            };
            Pieces pieces;
            while (const Piece* p = pieces.next(s)) {
                const int n = pieces.n - 1, start = p->start(0), hi = p->hi, t0 = p->t0, t1 = p->t1;
                pieces.done(s);
                const uint32_t q = uniform(lo_q + q_s + (n % QB) * QT * (TM::kTileBytes >> 4));
                ok = ok && warp_wait(&s.q_full[n % QB], (n / QB) & 1, dead);
#pragma unroll 1
                for (int t = t0; t < t1 && ok; t++, j++) {
                    const int n16 = (min(kTile, hi - (start + t * kTile)) + 15) / 16;
                    if (!k_there) ok = ok && warp_wait(&s.k_full[k_slot], k_lap & 1, dead);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t ksl = uniform(k_slot), id = uniform(id_k | (uint32_t)(2 * n16) << 17);
                    const uint32_t k_sm = lo_kv + ring_k + ksl * (TM::kTileBytes >> 4), sc = tm + uniform(sb) * TM::kSCols;
                    if (elected()) {
                        if (ks == HD / 16) {
#pragma unroll
                            for (int x = QT - 1; x >= 0; x--)
#pragma unroll
                                for (int k = 0; k < HD / 16; k++) {
                                    const uint32_t in = (uint32_t)(k >> 2) * ((kTile * 128) >> 4) + (k & 3) * 2;
                                    mma_f16(sc, desc_of(q + x * (TM::kTileBytes >> 4) + in, hi_q),
                                            desc_of(k_sm + (k >> 2) * (1024 >> 4) + (k & 3) * 2, hi_kv), id, x < QT - 1 || k > 0);
                                }
                        } else {
                            uint32_t acc = 0;
#pragma unroll 1
                            for (int x = QT - 1; x >= 0; x--)
#pragma unroll 1
                                for (int k = 0; k < ks; k++) {
                                    const uint32_t in = (uint32_t)(k >> 2) * ((kTile * 128) >> 4) + (k & 3) * 2;
                                    mma_f16(sc, desc_of(q + x * (TM::kTileBytes >> 4) + in, hi_q),
                                            desc_of(k_sm + (uint32_t)(k >> 2) * (1024 >> 4) + (k & 3) * 2, hi_kv), id, acc);
                                    acc = 1;
                                }
                        }
                        mma_commit(&s.s_full[sb]);
                        if (NK != 2) mma_commit(&s.k_empty[k_slot]);
                        if (t == t1 - 1) mma_commit(&s.q_empty[n % QB]);
                    }
                    __syncwarp();
                    if (++k_slot == NK) {
                        k_slot = 0;
                        k_lap++;
                    }
                    if (++sb == NS) sb = 0;
                    if (j >= LAG) values(j - LAG, t + 1 < t1);
                    if (j == 0) was[0] = n16;
                    else was[LAG - 1] = n16;
                }
                if (!ok) break;
            }
            for (int i = max(0, j - LAG); ok && i < j; i++) values(i, false);
        }
    }
    if (*dead) {
        a.line->dead = 1;
        for (int i = 0; i < 1000; i++) __nanosleep(1000);  // (copies of a share that gave up may still be on their way here)
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------------------
// joining
// ---------------------------------------------------------------------------

constexpr int kSharedJoinThreads = 256;

// o, M (log2 units), L of a row's head, four dimensions a lane
struct Sum {
    float4 o;
    float M, L;
    __device__ __forceinline__ void add(float4 x, float m, float l) {
        const float n = fmaxf(M, m), z = n == -INFINITY ? 0.0f : n, f = ex2(M - z), g = ex2(m - z);
        M = n;
        L = fmaf(L, f, l * g);
        o.x = fmaf(o.x, f, x.x * g);
        o.y = fmaf(o.y, f, x.y * g);
        o.z = fmaf(o.z, f, x.z * g);
        o.w = fmaf(o.w, f, x.w * g);
    }
};

// A row's head by one warp, from its own positions: 32 scores at a time, a
// position to a lane, then the values, four dimensions to a lane.
template <typename T, typename C>
__device__ __noinline__ Sum row_alone(const SharedArgs& a, int b, int head) {
    const int lane = threadIdx.x & 31, hd = a.hd, d = 4 * lane;
    const Seq sq = seq_of(a, b);
    const int64_t h_off = (int64_t)(head / a.grp) * a.head_stride;
    const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.q_stride + (int64_t)head * hd;
    const float slope = a.slopes ? a.slopes[head] : 0.0f;
    float up = 1.0f, scale = a.scale;
    if (std::is_same<T, float>::value) {  // as the products take it
        const int e = row_exponent(d < hd ? load4(q + d, a.q_wide) : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        up = pow2f(e);
        scale *= pow2f(-e);
    }
    Sum r{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
    bool bad = false;
    for (int p0 = sq.lo; p0 < sq.len; p0 += 32) {
        const int pos = p0 + lane;
        int64_t off = -1;
        float x = -INFINITY;
        if (pos < sq.len) {
            const int pg = page_of(a, pos), page = a.table[(int64_t)sq.tr * a.table_stride + pg];
            if ((unsigned)page < (unsigned)a.n_pages) {
                off = page * a.page_stride + (int64_t)(pos - pg * a.page_size) * a.pos_stride + h_off;
                const C* k = reinterpret_cast<const C*>(a.k) + off;
                float dot = 0.0f;
                for (int i = 0; i < hd; i++) dot = fmaf(to_float(q[i]) * up, to_float(k[i]), dot);
                x = dot * scale;
                if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
                x = fmaf(slope, (float)(pos - (sq.len - 1)), x) * kLog2e;
            } else {
                bad = true;
            }
        }
        float m = x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float n = fmaxf(r.M, m), z = n == -INFINITY ? 0.0f : n, f = ex2(r.M - z);
        const float e = pos < sq.len ? ex2(x - z + 14.0f) : 0.0f;
        r.M = n;
        float l = e;
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        r.L = fmaf(r.L, f, l);
        r.o = make_float4(r.o.x * f, r.o.y * f, r.o.z * f, r.o.w * f);
        for (int j = 0; j < min(32, sq.len - p0); j++) {
            const int64_t at = __shfl_sync(0xffffffffu, off, j);
            const float w = __shfl_sync(0xffffffffu, e, j);
            if (at >= 0 && d < hd) {
                const C* v = reinterpret_cast<const C*>(a.v) + at + d;
                r.o.x = fmaf(w, to_float(v[0]), r.o.x);
                r.o.y = fmaf(w, to_float(v[1]), r.o.y);
                r.o.z = fmaf(w, to_float(v[2]), r.o.z);
                r.o.w = fmaf(w, to_float(v[3]), r.o.w);
            }
        }
    }
    if (__any_sync(0xffffffffu, bad)) r.L = __int_as_float(0x7fc00000);
    return r;
}

// CTAs (rows in turn, heads in turn): which of its rows there is something to
// join of, a row to a thread; then a warp for each of their heads.
template <typename T, typename C>
__global__ void __launch_bounds__(kSharedJoinThreads) shared_join_kernel(const __grid_constant__ SharedArgs a) {
    struct Todo {
        int b, kind;               // kind: 0 pieces, 1 by itself, 2 NaN
        int first[2], last[2], base[2];  // the shares of its items, its place among the item's (row, head) pairs
    };
    __shared__ Todo todo[kSharedJoinThreads];
    __shared__ int n_todo;
    constexpr int kWarps = kSharedJoinThreads / 32;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hd = a.hd, d = 4 * lane;
    const Line line = *a.line;
    const int64_t width = hd + 4;
    const int mine = (a.batch - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // rows of this CTA
#pragma unroll 1
    for (int r0 = 0; r0 < mine; r0 += kSharedJoinThreads) {
        if (tid == 0) n_todo = 0;
        __syncthreads();
        if (r0 + tid < mine) {
            Todo t{};
            t.b = (int)(blockIdx.x + (int64_t)(r0 + tid) * gridDim.x);
            const int4 row = a.row[t.b];
            const int redo = a.redo[t.b];
            bool cut = false;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int i = k ? row.w : row.z;
                t.last[k] = -1;
                if (i < 0) continue;
                const Item it = a.item[i];
                const long long u = it.u0 + kItemUnits;
                t.first[k] = (int)mul_div(u + 1, line.shares, line.units, -1);
                t.last[k] = (int)mul_div(u + tiles_of(it), line.shares, line.units, -1);
                t.base[k] = (t.b - it.row0) * a.hb;
                cut |= t.first[k] != t.last[k];
            }
            t.kind = row.z == -2 || line.dead ? 2 : redo ? 1 : 0;
            // (a row of one item that was not cut is written already)
            if (t.kind || cut || (row.z >= 0) == (row.w >= 0)) todo[atomicAdd(&n_todo, 1)] = t;
        }
        __syncthreads();
        const int heads = (a.nh + (int)gridDim.y - 1) / (int)gridDim.y, h0 = blockIdx.y * heads, h1 = min(a.nh, h0 + heads);
#pragma unroll 1
        for (int x = warp; x < n_todo * heads; x += kWarps) {
            const int e = x / heads, head = h0 + x - e * heads;
            if (head >= h1) continue;
            const Todo t = todo[e];
            Sum r{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
            bool alone = t.kind == 1;
            if (t.kind == 0) {
                const int h = head / a.grp, in = head - h * a.grp, blk = in / a.hb, hh = in - blk * a.hb;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    constexpr int N = 4;  // pieces in flight
                    for (int i0 = t.first[k]; i0 <= t.last[k]; i0 += N) {
                        float4 v[N];
                        float2 ml[N];
#pragma unroll
                        for (int n = 0; n < N; n++) {
                            const int i = i0 + n;
                            const float* from =
                                t.first[k] == t.last[k]
                                    ? a.whole + (((int64_t)k * a.batch + t.b) * a.nh + head) * width
                                    : a.part + (((int64_t)(i * a.nkv * a.blocks + h * a.blocks + blk) * 2 + (i == t.first[k] ? 1 : 0)) * kTile +
                                                t.base[k] + hh) * width;
                            v[n] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            ml[n] = make_float2(-INFINITY, 0.0f);
                            if (i <= t.last[k]) {
                                ml[n] = *reinterpret_cast<const float2*>(from + hd);
                                if (d < hd) v[n] = *reinterpret_cast<const float4*>(from + d);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < N; n++) r.add(v[n], ml[n].x, ml[n].y);
                    }
                }
                const float f = r.L == 0.0f ? 0.0f : (r.o.x + r.o.y + r.o.z + r.o.w) / r.L;
                alone = __any_sync(0xffffffffu, d < hd && f - f != 0.0f);
            }
            if (alone) r = row_alone<T, C>(a, t.b, head);
            if (t.kind == 2) r.L = __int_as_float(0x7fc00000);
            const float inv = r.L == 0.0f ? 0.0f : 1.0f / r.L;
            T* out = static_cast<T*>(a.out) + (int64_t)t.b * a.out_stride + (int64_t)head * hd;
            if (d < hd) {
                out[d] = (T)(r.o.x * inv);
                out[d + 1] = (T)(r.o.y * inv);
                out[d + 2] = (T)(r.o.z * inv);
                out[d + 3] = (T)(r.o.w * inv);
            }
            if (a.lse && lane == 0)
                a.lse[(int64_t)t.b * a.nh + head] = r.L == 0.0f ? -INFINITY : (r.M + (log2f(r.L) - 14.0f)) * kLn2;
        }
        __syncthreads();
    }
}

constexpr int kMaxSharedDevices = 64;

cudaError_t launch_line(void (*kern)(SharedArgs), int smem, int ctas, const SharedArgs& a, cudaStream_t s) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return e == cudaSuccess ? launch_pdl(kern, dim3(ctas), dim3(kPlanThreads), smem, s, a) : e;
}

template <int HD, typename T, typename C, int QT, int PT>
cudaError_t go(const SharedArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq, int sms, cudaStream_t s) {
    static std::atomic<bool> attr[kMaxSharedDevices] = {};  // the attribute belongs to a device
    constexpr int smem = Tm<HD, QT, PT>::kTotal;
    auto kern = shared_tiles_kernel<HD, T, C, QT, PT>;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxSharedDevices || !attr[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxSharedDevices) attr[dev] = true;
    }
    const long long q_rows = a.terms ? (long long)a.batch * a.nh : 0;  // (a warp takes four at a time)
    const int ctas = 1 + (int)std::min<long long>(2 * sms - 1, (q_rows + kPlanThreads / 8 - 1) / (kPlanThreads / 8));
    // (a row to a thread; four where there are more: 2048 rows 9 us, 14 in two turns)
    if (a.batch <= kPlanThreads) {
        e = launch_line(shared_line_kernel<T, C, QT, 1>, (int)sizeof(LineShared<1>), ctas, a, s);
    } else {
        e = launch_line(shared_line_kernel<T, C, QT, 4>, (int)sizeof(LineShared<4>), ctas, a, s);
    }
    if (e != cudaSuccess) return e;
    e = launch_pdl(kern, dim3((unsigned)(a.shares * a.nkv * a.blocks)), dim3(kSharedThreads), smem, s, a, mk, mv, mq);
    if (e != cudaSuccess) return e;
    const int rows = std::min(a.batch, 4 * sms);
    const int y = std::max(1, std::min((a.nh + 7) / 8, 16 * sms / rows));
    return launch_pdl(shared_join_kernel<T, C>, dim3(rows, y), dim3(kSharedJoinThreads), 0, s, a);
}

template <int HD>
cudaError_t go_hd(const SharedArgs& a, int dtype, int cache, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mq,
                  int sms, cudaStream_t s) {
    if (dtype == 0)
        return cache == 1 ? go<HD, float, __half, 2, 2>(a, mk, mv, mq, sms, s) : go<HD, float, __nv_bfloat16, 3, 3>(a, mk, mv, mq, sms, s);
    return cache == 1 ? go<HD, __half, __half, 1, 2>(a, mk, mv, mq, sms, s)
                      : go<HD, __nv_bfloat16, __nv_bfloat16, 1, 2>(a, mk, mv, mq, sms, s);
}

// The positions of a tensor map's box: 16, or 8, where pages are multiples of
// it; 0 where the cache's sizes or strides are not what a map takes.
int box_of(const b2_paged_kv& kv) {
    const int64_t top = (int64_t)1 << 38;  // (strides below 2^40 bytes)
    const bool apart = (kv.nkv == 1 || kv.head_stride > 0) && kv.pos_stride > 0 && (kv.n_pages == 1 || kv.page_stride > 0);
    if (!apart || kv.head_stride >= top || kv.pos_stride >= top || kv.page_stride >= top) return 0;
    return kv.page_size % 16 == 0 ? 16 : kv.page_size % 8 == 0 ? 8 : 0;
}

// A map of 16-bit elements in the 128-byte swizzle: n elements, strides (in
// elements) from the second dimension on, and the box of each dimension.
template <int R>
bool make_map(CUtensorMap* m, int dtype, const void* at, const int64_t (&n)[R], const int64_t (&stride)[R - 1], const int (&box)[R]) {
    const auto enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint64_t dims[R], strides[R - 1];
    cuuint32_t boxes[R], steps[R];
    for (int i = 0; i < R; i++) {
        dims[i] = (cuuint64_t)n[i];
        boxes[i] = (cuuint32_t)box[i];
        steps[i] = 1;
        if (i) strides[i - 1] = (cuuint64_t)std::max<int64_t>(16, 2 * stride[i - 1]);
    }
    return enc(m, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, R, const_cast<void*>(at), dims,
               strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether the cache's pages follow one another as their positions do (1), and
// then whether a box may take whole heads (2).
int flat_of(const b2_paged_kv& kv) {
    if (kv.page_stride != kv.page_size * kv.pos_stride || (int64_t)kv.page_size * kv.n_pages >= ((int64_t)1 << 31)) return 0;
    return kv.hd % 64 == 0 ? 2 : 1;
}

// A cache's k or v.  Boxes of 64 dimensions (those past hd read as zero), one
// head, `box` positions (8 where a head has two blocks) of one page; or of whole
// heads, positions 8 by 8.
bool make_map(CUtensorMap* m, const b2_paged_kv& kv, const void* at, int box, int flat) {
    const int64_t all = (int64_t)kv.page_size * kv.n_pages;
    if (flat == 2)
        return make_map<5>(m, kv.dtype, at, {64, 8, kv.hd / 64, all / 8, kv.nkv}, {kv.pos_stride, 64, 8 * kv.pos_stride, kv.head_stride},
                           {64, 8, kv.hd / 64, box / 8, 1});
    const int rows = kv.hd <= 64 ? box : 8;
    if (flat) return make_map<4>(m, kv.dtype, at, {kv.hd, kv.nkv, all, 1}, {kv.head_stride, kv.pos_stride, 8}, {64, 1, rows, 1});
    return make_map<4>(m, kv.dtype, at, {kv.hd, kv.nkv, kv.page_size, kv.n_pages}, {kv.head_stride, kv.pos_stride, kv.page_stride},
                       {64, 1, rows, 1});
}

// How a group of query heads falls to items, and the shares of the machine.
struct Shape {
    int hb, blocks, rows, shares;
    Shape(int nh, int nkv, int sms) {
        const int grp = nh / nkv;
        hb = std::min(grp, kTile);
        blocks = (grp + hb - 1) / hb;
        rows = kTile / hb;
        shares = std::max(1, sms / (nkv * blocks));
    }
};

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// The scratch of `batch` rows; where its parts start, if a is given.
size_t layout(int batch, int nh, int nkv, int hd, int sms, uint8_t* base, SharedArgs* a) {
    const Shape sh(nh, nkv, sms);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = base + at;
        at += up16(bytes);
        return p;
    };
    uint8_t* line = take(sizeof(Line));
    uint8_t* share = take(sizeof(Share) * (size_t)sh.shares);
    uint8_t* redo = take(4 * (size_t)batch);
    uint8_t* row = take(16 * (size_t)batch);
    uint8_t* item = take(2 * sizeof(Item) * (size_t)batch);
    uint8_t* factor = take(4 * (size_t)batch * nh);
    uint8_t* term = take((size_t)6 * batch * nh * hd);  // (three terms at most)
    uint8_t* whole = take((size_t)2 * batch * nh * (hd + 4) * 4);
    uint8_t* part = take((size_t)sh.shares * nkv * sh.blocks * 2 * kTile * (hd + 4) * 4);
    if (a) {
        a->line = reinterpret_cast<Line*>(line);
        a->share = reinterpret_cast<Share*>(share);
        a->factor = reinterpret_cast<float*>(factor);
        a->term = reinterpret_cast<uint16_t*>(term);
        a->redo = reinterpret_cast<int*>(redo);
        a->row = reinterpret_cast<int4*>(row);
        a->item = reinterpret_cast<Item*>(item);
        a->whole = reinterpret_cast<float*>(whole);
        a->part = reinterpret_cast<float*>(part);
    }
    return at;
}

}  // namespace

// When to read what the rows of a group have in common once, and when row by row
// (attention_paged.cu).  The three launches here take 22-30 us however little
// there is to do; row by row costs 10-13 us and then the bytes of all rows, most
// of them from L2, at 8 TB/s (or, with more than 8 query heads to a KV head, the
// products' time).  The two meet where the rows' positions times max(heads to a
// KV head, 8) x KV heads x dimensions come to some 2^28 (134 MB at 8 heads), in us:
//   heads, dims, type     rows   positions   of 2^28   row by row   shared
//   32 / 8, 128, fp32     1 x 4   2080        1/4       14.4         28.8
//   64 / 8, 128, bf16     1 x 16  2080        1         28.7         29.4
//   32 / 8, 128, fp32     1 x 64   544        1         28.8         32.9
//   64 / 1, 128, bf16     4 x 4   2080        1         29.6         28.8
//   32 / 8, 128, fp32     8 x 8   2080        4         75.9         45.2
//   64 / 8, 128, bf16     1 x 16  8224        4         70.9         37.0
// Positions: the window, or what the table has room for, since the lengths are on
// the device (16 requests of 1 to 8 rows, window 4096 of 9336, 14 / 2 heads of 64: 22.6
// and 39; 139 rows of one sequence, window 3: 10.3 and 22.5).
// Where groups have fewer than two rows on average there is too little to share,
// however they lie: rows that share nothing take 1.5 to 1.9 times as long in the
// tiles (64 x 1 rows of 2080 positions, 64 / 8 heads: 100 and 146; 81 rows in 43 groups,
// 28 / 4 heads of 64, fp32: 29 and 55), and a prompt of 512 tokens beside 520 tokens of
// rows of 500 is 262 and 300 (by itself in tiles 43).  Groups without rows count, so a
// prompt of 300 in a table of 256 requests takes 65 where tiles would take 41.
bool row_by_row(const b2_paged_kv& kv, const b2_paged_attn_opts& o, int batch, int n_groups) {
    const double room = (double)o.max_pages * kv.page_size;
    const double positions = batch * (o.window > 0 ? std::min(room, (double)o.window) : room);
    return kv.hd > 128 || batch < 2LL * n_groups || positions * std::max(o.nh, 8 * kv.nkv) * kv.hd <= (double)(1 << 28);
}

size_t attention_shared_scratch(int batch, int nh, int nkv, int hd, int sms) {
    const size_t rows = attention_paged_scratch(batch, nh, nkv, hd, sms);
    return hd > 128 ? rows : std::max(rows, layout(batch, nh, nkv, hd, sms, nullptr, nullptr));
}

int launch_attention_shared(const b2_paged_kv& kv, const b2_paged_attn_opts& o, const void* q, const int32_t* table,
                            const int32_t* lens, const int32_t* req, int batch, const int32_t* starts,
                            const int32_t* prefix, int n_groups, void* out, float* lse, void* scratch, cudaStream_t s,
                            std::string* err) {
    if (row_by_row(kv, o, batch, n_groups)) return launch_attention_paged(kv, o, q, table, lens, req, batch, out, lse, scratch, s, err);
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    SharedArgs a{};
    a.q = q;
    a.k = static_cast<const uint16_t*>(kv.k);
    a.v = static_cast<const uint16_t*>(kv.v);
    a.table = table;
    a.lens = lens;
    a.req = req;
    a.starts = starts;
    a.prefix = prefix;
    a.out = out;
    a.lse = lse;
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
    a.hd = kv.hd;
    a.page_size = kv.page_size;
    while ((1ull << a.page_shift) < (unsigned)kv.page_size) a.page_shift++;
    a.page_mul = (uint32_t)((((1ull << a.page_shift) - kv.page_size) << 32) / kv.page_size + 1);
    a.n_pages = kv.n_pages;
    a.max_pages = o.max_pages;
    a.n_req = o.n_req;
    a.len_add = o.len_add;
    a.window = o.window;
    a.n_groups = n_groups;
    const Shape sh(o.nh, kv.nkv, sms);
    a.hb = sh.hb;
    a.blocks = sh.blocks;
    a.rows = sh.rows;
    a.shares = sh.shares;
    const int es = o.dtype == 0 ? 4 : 2;
    a.q_wide = !(reinterpret_cast<uintptr_t>(q) & 15) && a.q_stride * es % 16 == 0;
    a.out_wide = !(reinterpret_cast<uintptr_t>(out) & 15) && a.out_stride * es % 16 == 0;
    a.scale = o.scale > 0.0f ? o.scale : (float)(1.0 / sqrt((double)kv.hd));
    a.softcap = o.softcap;
    a.terms = o.dtype == 0 ? (kv.dtype == 1 ? 2 : 3) : a.q_wide && a.q_stride < ((int64_t)1 << 38) ? 0 : 1;
    layout(batch, o.nh, kv.nkv, kv.hd, sms, static_cast<uint8_t*>(scratch), &a);
    CUtensorMap mk{}, mv{}, mq{};
    const bool q_map =
        a.terms ? make_map<4>(&mq, kv.dtype, a.term, {kv.hd, o.nh, batch, a.terms}, {kv.hd, qd, qd * batch}, {64, a.hb, a.rows, 1})
                : make_map<4>(&mq, kv.dtype, q, {kv.hd, o.nh, batch, 1}, {kv.hd, a.q_stride, 8}, {64, a.hb, a.rows, 1});
    if (!q_map) {
        *err = "shared attention: no tensor map of q";
        return B2_ERR_CUDA;
    }
    a.box = box_of(kv);
    a.flat = flat_of(kv);
    if (a.box && !(make_map(&mk, kv, kv.k, a.box, a.flat) && make_map(&mv, kv, kv.v, a.box, a.flat))) a.box = 0;
    const cudaError_t e = kv.hd <= 64 ? go_hd<64>(a, o.dtype, kv.dtype, mk, mv, mq, sms, s)
                                      : go_hd<128>(a, o.dtype, kv.dtype, mk, mv, mq, sms, s);
    return e == cudaSuccess ? B2_OK : cuda_failed("shared attention launch", e, err);
}

}  // namespace b2
