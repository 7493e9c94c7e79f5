// Host side of the paged serving operators: rotary frequencies, the SM count
// and the check of a pointer's device.
#include "paged.h"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace b2 {

int current_sms(std::string* err) {
    constexpr int kMaxDevices = 64;
    static std::atomic<int> sms[kMaxDevices];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) {
        cudaGetLastError();
        *err = "no CUDA device";
        return 0;
    }
    int n = dev < kMaxDevices ? sms[dev].load(std::memory_order_relaxed) : 0;
    if (n) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        *err = "no CUDA device";
        return 0;
    }
    if (dev < kMaxDevices) sms[dev].store(n, std::memory_order_relaxed);
    return n;
}

int check_alignment(const DevicePtr* p, int n, std::string* err) {
    for (int i = 0; i < n; i++)
        if (reinterpret_cast<uintptr_t>(p[i].p) & (p[i].align - 1)) {
            *err = std::string(p[i].name) + " must be " + std::to_string(p[i].align) + "-byte aligned";
            return B2_ERR_BAD_ARG;
        }
    return B2_OK;
}

int check_device_pointers(const DevicePtr* p, int n, std::string* err) {
    int dev = -1;
    cudaError_t e = cudaGetDevice(&dev);
    for (int i = 0; i < n && e == cudaSuccess; i++) {
        if (!p[i].p) continue;
        cudaPointerAttributes at{};
        e = cudaPointerGetAttributes(&at, p[i].p);
        if (e != cudaSuccess) break;
        if (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev)) continue;
        *err = p[i].name;
        if (at.type == cudaMemoryTypeDevice)
            *err += " is on device " + std::to_string(at.device) + ", the current device is " + std::to_string(dev);
        else
            *err += " is not device memory";
        return B2_ERR_BAD_ARG;
    }
    return e == cudaSuccess ? B2_OK : cuda_failed("no CUDA device", e, err);
}

int cuda_failed(const char* what, cudaError_t e, std::string* err) {
    cudaGetLastError();  // reported here: not again to the caller's next CUDA call
    *err = std::string(what) + ": " + cudaGetErrorString(e);
    return B2_ERR_CUDA;
}

}  // namespace b2

// Frequencies in radians per position and the factor on cos and sin.  i is
// the pair, rot the rotated width, base = theta^(-2 i / rot):
//   none   base
//   linear base / factor
//   bands  a pair that turns n = orig_ctx * base / 2 pi times over the
//          original context keeps its frequency for n >= high, is divided by
//          factor for n <= low, and is blended linearly in n between
//   yarn   the same blend, linear in the pair's number between the pairs that
//          turn `high` times (rounded down) and `low` times (rounded up); cos
//          and sin are scaled by 0.1 log(factor) + 1
int b2_rope_freqs_impl(const b2_rope_opts& o, double* freqs, float* scale) {
    const int rot = o.rot_dim;
    const double two_pi = 6.283185307179586476925;
    const double low = o.low > 0 ? o.low : 1.0;
    const double high = o.high > 0 ? o.high : (o.scaling == B2_ROPE_SCALE_YARN ? 32.0 : 4.0);
    if (!(high > low)) return B2_ERR_BAD_ARG;
    auto pair = [&](double turns) { return rot * std::log(o.orig_ctx / (turns * two_pi)) / (2 * std::log(o.theta)); };
    double lo = 0, hi = 0;
    if (o.scaling == B2_ROPE_SCALE_YARN) {
        lo = std::max(std::floor(pair(high)), 0.0);
        hi = std::min(std::ceil(pair(low)), rot - 1.0);
    }
    for (int i = 0; i < rot / 2; i++) {
        const double base = std::pow(o.theta, -2.0 * i / rot);
        double keep = 1.0;
        if (o.scaling == B2_ROPE_SCALE_LINEAR) keep = 0.0;
        if (o.scaling == B2_ROPE_SCALE_BANDS) keep = (o.orig_ctx * base / two_pi - low) / (high - low);
        if (o.scaling == B2_ROPE_SCALE_YARN) keep = 1.0 - (i - lo) / std::max(hi - lo, 1e-3);
        keep = std::min(1.0, std::max(0.0, keep));
        freqs[i] = o.scaling == B2_ROPE_SCALE_NONE ? base : base * (keep + (1.0 - keep) / o.factor);
    }
    if (scale) *scale = o.scaling == B2_ROPE_SCALE_YARN ? (float)(0.1 * std::log(o.factor) + 1.0) : 1.0f;
    return B2_OK;
}
