// Rotary positions on the rows of a step, written to the paged KV cache.
//
// Pair i of a head turns by the angle position * freq[i]:
//   (a, b) -> scale * (a cos - b sin, a sin + b cos),
// (a, b) = elements (2i, 2i + 1) (interleaved) or (i, i + rot_dim / 2) (half);
// elements from rot_dim on stay as they are.
//
// The angle is kept as a fraction of a turn in 64-bit fixed point: with
// F = frac(freq / 2 pi) * 2^64, position * F mod 2^64 is the wrapped angle to
// 2^-53 * position of a turn, so a far position costs one integer product
// where the product in fp32 would lose the angle (at 10^6 positions its
// rounding is 0.03 radians).  The wrapped angle is then split into a quarter
// turn and a remainder of at most an eighth, so sin and cos see an argument
// that fp32 holds to 2^-27 of a turn.  They are computed once a token and
// pair, in shared memory, for all heads.
//
// HBM-bound: every q, k and v element is read once and written once (32768
// rows of 64 + 16 heads of 128, bf16: 1.34 GB in 203 us, 6.6 TB/s; 16 rows: 2.5
// us, a launch and three dependent loads).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "dev.cuh"
#include "paged.h"

namespace b2 {
namespace {

// (32768 rows back to back: 219 us; 226 with 256, 266 with 512: a CTA waits for its sines first)
constexpr int kRopeThreads = 128;

struct RopeArgs {
    const double* freqs;
    const int32_t* positions;
    const int64_t* slots;  // null: k_out
    const void *q, *k, *v;
    void *q_out, *k_out, *v_out;
    int64_t q_stride, k_stride, v_stride, qo_stride, ko_stride;
    // the cache: page of slot / P, row of slot % P
    int64_t page_stride, pos_stride, head_stride;
    int64_t n_slots;
    int page_size;
    int n_tok, nh, nkv, hd, rot, half_layout;
    float scale;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f(const T* p, float* f) {
    const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = to_f(x.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_f(T* p, const float* f) {
    Pack<T, N> x;
#pragma unroll
    for (int i = 0; i < N; i++) x.v[i] = from_f<T>(f[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = x;
}

// cos and sin of pos * freq, times scale
__device__ __forceinline__ float2 turn(double freq, int pos, float scale) {
    double t = freq * 0.15915494309189533577;  // turns per position
    t -= floor(t);
    const unsigned long long F = __double2ull_rz(t * 18446744073709551616.0);
    const unsigned long long u = (unsigned long long)(long long)pos * F;
    const unsigned q = (unsigned)((u + (1ull << 61)) >> 62);  // nearest quarter turn
    const long long r = (long long)(u - ((unsigned long long)q << 62));
    float s, c;
    sincospif((float)r * 1.0842021724855044e-19f, &s, &c);  // r / 2^63 half turns, at most a quarter of one
    if (q & 1) {
        const float x = c;
        c = -s;
        s = x;
    }
    if (q & 2) {
        c = -c;
        s = -s;
    }
    return make_float2(c * scale, s * scale);
}

// Units of one head of `rot` rotated elements out of hd, VEC elements wide:
// interleaved: hd / VEC chunks, each within or past rot; half: rot / 2 / VEC
// pairs of chunks, then the chunks past rot.  VEC = 1 is the form for odd
// sizes and unaligned rows (a unit is then one pair, or one element past rot).
template <typename T, typename C, int VEC>
__device__ __forceinline__ void rope_unit(const T* src, C* dst, int u, const float2* cs, int hd, int rot, int half_layout) {
    if (half_layout) {
        const int h = rot / 2, np = h / VEC;
        if (u < np) {
            float a[VEC], b[VEC];
            load_f<T, VEC>(src + u * VEC, a);
            load_f<T, VEC>(src + h + u * VEC, b);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float2 w = cs[u * VEC + i];
                const float x = a[i], y = b[i];
                a[i] = x * w.x - y * w.y;
                b[i] = x * w.y + y * w.x;
            }
            store_f<C, VEC>(dst + u * VEC, a);
            store_f<C, VEC>(dst + h + u * VEC, b);
            return;
        }
        u = (rot / VEC) + (u - np);
    } else if (VEC == 1) {
        if (u < rot / 2) {
            const float2 w = cs[u];
            const float x = to_f(src[2 * u]), y = to_f(src[2 * u + 1]);
            dst[2 * u] = from_f<C>(x * w.x - y * w.y);
            dst[2 * u + 1] = from_f<C>(x * w.y + y * w.x);
            return;
        }
        u = rot + (u - rot / 2);
    }
    float a[VEC];
    load_f<T, VEC>(src + u * VEC, a);
    if (!half_layout && VEC > 1 && u * VEC < rot) {
#pragma unroll
        for (int i = 0; i + 1 < VEC; i += 2) {
            const float2 w = cs[(u * VEC + i) / 2];
            const float x = a[i], y = a[i + 1];
            a[i] = x * w.x - y * w.y;
            a[i + 1] = x * w.y + y * w.x;
        }
    }
    store_f<C, VEC>(dst + u * VEC, a);
}

// One CTA = one token's heads [blockIdx.y share]; T: the rows' type, C: the
// cache's (or k_out's) type.
template <typename T, typename C, int VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ float2 cs[kPagedMaxHd / 2];
    pdl_trigger();
    pdl_wait();
    const int64_t t = blockIdx.x;
    const int half = a.rot / 2, tid = threadIdx.x;
    const int pos = a.positions[t];
    for (int i = tid; i < half; i += kRopeThreads) cs[i] = turn(a.freqs[i], pos, a.scale);
    __syncthreads();
    C* kd = nullptr;
    C* vd = nullptr;
    int64_t kh = a.head_stride;
    if (a.slots) {
        const int64_t slot = a.slots[t];
        if (slot >= 0 && slot < a.n_slots) {
            const int64_t page = slot / a.page_size;
            const int64_t off = page * a.page_stride + (slot - page * a.page_size) * a.pos_stride;
            kd = static_cast<C*>(a.k_out) + off;
            vd = static_cast<C*>(a.v_out) + off;
        }
    } else if (a.k_out) {
        kd = static_cast<C*>(a.k_out) + t * a.ko_stride;
        kh = a.hd;
    }
    const int upr = a.half_layout || VEC == 1 ? half / VEC + (a.hd - a.rot) / VEC : a.hd / VEC;  // units of a rotated head
    const int upv = a.hd / VEC;
    const int nq = a.q ? a.nh * upr : 0, nk = kd ? a.nkv * upr : 0, nv = vd ? a.nkv * upv : 0;
    const int n = nq + nk + nv;
    for (int i = blockIdx.y * kRopeThreads + tid; i < n; i += gridDim.y * kRopeThreads) {
        if (i < nq) {
            const int h = i / upr, u = i - h * upr;
            rope_unit<T, T, VEC>(static_cast<const T*>(a.q) + t * a.q_stride + h * a.hd,
                                 static_cast<T*>(a.q_out) + t * a.qo_stride + h * a.hd, u, cs, a.hd, a.rot, a.half_layout);
        } else if (i < nq + nk) {
            const int j = i - nq, h = j / upr, u = j - h * upr;
            rope_unit<T, C, VEC>(static_cast<const T*>(a.k) + t * a.k_stride + h * a.hd, kd + h * kh, u, cs, a.hd, a.rot,
                                 a.half_layout);
        } else {
            const int j = i - nq - nk, h = j / upv, u = j - h * upv;
            float f[VEC];
            load_f<T, VEC>(static_cast<const T*>(a.v) + t * a.v_stride + h * a.hd + u * VEC, f);
            store_f<C, VEC>(vd + h * kh + u * VEC, f);
        }
    }
}

template <typename T, typename C>
cudaError_t go(const RopeArgs& a, bool wide, int sms, cudaStream_t s) {
    constexpr int W = 16 / sizeof(T);
    const int units = (a.nh + 2 * a.nkv) * a.hd / (wide ? W : 1);
    // a token's heads over several CTAs while the grid is small
    const int split = std::max(1, std::min((units + kRopeThreads - 1) / kRopeThreads, 2 * sms / std::max(1, a.n_tok)));
    const dim3 grid(a.n_tok, split);
    return wide ? launch_pdl(rope_kernel<T, C, W>, grid, dim3(kRopeThreads), 0, s, a)
                : launch_pdl(rope_kernel<T, C, 1>, grid, dim3(kRopeThreads), 0, s, a);
}

}  // namespace

int launch_rope(const b2_rope_rows& d, const b2_paged_kv* kv, const double* freqs, const int32_t* positions,
                const int64_t* slots, int n_tok, const void* q, const void* k, const void* v, void* q_out, void* k_out,
                cudaStream_t s, std::string* err) {
    const int sms = current_sms(err);
    if (!sms) return B2_ERR_CUDA;
    RopeArgs a{};
    a.freqs = freqs;
    a.positions = positions;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = q_out;
    a.k_out = k_out;
    const int64_t qd = (int64_t)d.nh * d.hd, kd = (int64_t)d.nkv * d.hd;
    a.q_stride = d.q_stride ? d.q_stride : qd;
    a.k_stride = d.k_stride ? d.k_stride : kd;
    a.v_stride = d.v_stride ? d.v_stride : kd;
    a.qo_stride = d.q_out_stride ? d.q_out_stride : qd;
    a.ko_stride = d.k_out_stride ? d.k_out_stride : kd;
    a.page_size = 1;
    if (kv) {
        a.slots = slots;
        a.k_out = kv->k;
        a.v_out = kv->v;
        a.page_size = kv->page_size;
        a.n_slots = (int64_t)kv->n_pages * kv->page_size;
        a.page_stride = kv->page_stride;
        a.pos_stride = kv->pos_stride;
        a.head_stride = kv->head_stride;
    }
    a.n_tok = n_tok;
    a.nh = q ? d.nh : 0;
    a.nkv = k ? d.nkv : 0;
    a.hd = d.hd;
    a.rot = d.rot_dim;
    a.half_layout = d.layout == B2_ROPE_HALF;
    a.scale = d.scale;
    // 16-byte rows, and rotated parts that whole 16-byte chunks cover: the
    // wide form; anything else element by element, the unrotated elements and v
    // too (32768 rows of 64 q, k and v heads of 96, half layout, bf16: 461 us
    // with 32 of them rotated, 1533 with 24)
    const int es = d.dtype == 0 ? 4 : 2, w = 16 / es;
    auto aligned = [&](const void* p, int64_t stride) { return !p || (!((uintptr_t)p & 15) && stride * es % 16 == 0); };
    const bool wide = d.hd % w == 0 && d.rot_dim % w == 0 && (!a.half_layout || d.rot_dim / 2 % w == 0) &&
                      aligned(q, a.q_stride) && aligned(k, a.k_stride) && aligned(v, a.v_stride) &&
                      aligned(q_out, a.qo_stride) && (kv || aligned(k_out, a.ko_stride));
    cudaError_t e;
    const int ct = kv ? kv->dtype : d.dtype;
    if (d.dtype == 0)
        e = ct == 0 ? go<float, float>(a, wide, sms, s)
            : ct == 1 ? go<float, __half>(a, wide, sms, s) : go<float, __nv_bfloat16>(a, wide, sms, s);
    else if (d.dtype == 1)
        e = go<__half, __half>(a, wide, sms, s);
    else
        e = go<__nv_bfloat16, __nv_bfloat16>(a, wide, sms, s);
    return e == cudaSuccess ? B2_OK : cuda_failed("rope launch", e, err);
}

}  // namespace b2
