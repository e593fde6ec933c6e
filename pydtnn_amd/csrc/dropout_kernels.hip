// Dropout whose mask is a function of (seed, offset, index): nothing is stored, the backward pass draws it again.
//
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011) with the seed as
// its key and (call, offset) as its counter gives 128 bits a call.  An element takes 16 of them, so one call serves
// eight elements, and is kept when its number is not below threshold = rate * 2^16 rounded to a whole number.
//
// Bound by memory: a thread loads eight elements, computes its call's ten rounds while they are on their way and stores eight.
// 51 million in float32 take 73 us, 5.6 TB/s, what a copy takes; 262144 take 2.7 us, a launch.
#include <cmath>
#include "../../include/pydtnn_hip.h"
#include "conv_internal.h"
#include "dtypes.h"

namespace {

constexpr int kT = 256;
constexpr int kPerCall = 8;

// The four words of one call.
__device__ __forceinline__ uint4 philox(uint64_t call, uint64_t offset, uint64_t seed)
{
    uint32_t c0 = (uint32_t)call, c1 = (uint32_t)(call >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

template <typename T>
__global__ void __launch_bounds__(kT) dropout_kernel(const T* x, T* y, long total, uint32_t threshold, wide_t<T> scale,
                                                     uint64_t seed, uint64_t offset, const int64_t* offset_dev)
{
    const long call = (long)blockIdx.x * kT + threadIdx.x;
    const long first = call * kPerCall;
    if (first >= total) return;
    if (offset_dev) offset += (uint64_t)*offset_dev;
    const uint4 w = philox((uint64_t)call, offset, seed);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    auto one = [&](int j, T v) {
        const uint32_t u = (j & 1) ? word[j / 2] >> 16 : word[j / 2] & 0xffffu;
        return u >= threshold ? (T)((wide_t<T>)v * scale) : (T)0.0f;
    };
    if (first + kPerCall <= total) {      // accesses of 16 bytes, wherever the tensors start
        T p[kPerCall];
        __builtin_memcpy(p, x + first, sizeof(p));
#pragma unroll
        for (int j = 0; j < kPerCall; ++j) p[j] = one(j, p[j]);
        __builtin_memcpy(y + first, p, sizeof(p));
    } else {
#pragma unroll
        for (int j = 0; j < kPerCall; ++j)
            if (first + j < total) y[first + j] = one(j, x[first + j]);
    }
}

}  // namespace

extern "C" {

int pydtnn_hip_dropout(int dtype, const void* x, void* y, long total, double rate, uint64_t seed, uint64_t offset,
                       const int64_t* offset_dev, void* stream)
{
    if (!x || !y || total <= 0 || !(rate >= 0.0 && rate <= 1.0)) return PYDTNN_HIP_ERR_INVALID;
    const long blocks = (total + (long)kT * kPerCall - 1) / ((long)kT * kPerCall);
    if (blocks * kT >= (1l << 32)) return PYDTNN_HIP_ERR_UNSUPPORTED;   // a launch counts its threads in 32 bits
    const uint32_t threshold = (uint32_t)std::nearbyint(rate * 65536.0);
    const double scale = threshold >= 65536u ? 0.0 : 65536.0 / (65536.0 - threshold);
    const hipStream_t st = convint::as_stream(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((dropout_kernel<T>), dim3((unsigned)blocks), dim3(kT), 0, st, (const T*)x, (T*)y, total, threshold,
                           (wide_t<T>)scale, seed, offset, offset_dev);
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    });
}

}  // extern "C"
