// Element types of the kernels that are not float32 only.
#pragma once
#include "common.h"

// Values of the `dtype` arguments of include/pydtnn_hip.h.
enum { kDtypeF32 = 0, kDtypeF64 = 1, kDtypeF16 = 2, kDtypeBF16 = 3 };

// What sums, statistics and per-channel vectors of a T tensor are held in: 32 bits, or 64 for double.
template <typename T>
struct Wide {
    using type = float;
};
template <>
struct Wide<double> {
    using type = double;
};
template <typename T>
using wide_t = typename Wide<T>::type;

// V consecutive elements, aligned for accesses of up to 16 bytes.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
    T v[V];
};

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Calls f with a value of the element type that `dtype` names; anything else is an invalid argument.
template <typename F>
static inline int with_dtype(int dtype, F f)
{
    switch (dtype) {
        case kDtypeF32: return f(float());
        case kDtypeF64: return f(double());
        case kDtypeF16: return f((_Float16)0);
        case kDtypeBF16: return f((__bf16)0.0f);
        default: return PYDTNN_HIP_ERR_INVALID;
    }
}
