// Matrix product in e4m3 with a scale for each block of 128, for FC layers that serve:
//   y[m][n] = act( sum over blocks b of 2^(ex[m][b] + ew[n][b]) * sum over the block of qx[m][k] qw[n][k]  + bias[n] )
// The scale of a block of 128 consecutive k of a row is the smallest power of two 2^e with amax <= 448 * 2^e, 448 being
// the largest e4m3 value, e in [-127, 127].  A power of two is what the matrix instructions and the conversions from e4m3
// multiply by themselves, so a block costs no instruction beside its product, and dividing by it rounds nothing: what is
// rounded is each value to e4m3, once, to the nearest (to even between two), and the sums.
//
// Two instructions take the products, by the type of the result:
//   16-bit results: v_mfma_scale_f32_16x16x128_f8f6f4, twice the rate of the 16-bit instructions.  It adds its products in
//       eights, each aligned to the largest of the eight with 13 bits below that one's leading bit (measured with powers of
//       two; eights are then added in 32 bits): a relative error of 1e-5 of a sum of like signs, a fortieth of the half
//       step that a float16 result is rounded by.
//   float32 results: the operands are converted to bfloat16 with their scales, which is exact, and go through
//       v_mfma_f32_16x16x32_bf16, which keeps 24 bits of everything it adds.
//
// Layout: q is (rows, k to a multiple of 128), zeros behind k; scales is (rows, blocks to a multiple of 4), one byte e + 127
// each, 127 behind the last block, so that a lane fetches the scales of four blocks as one word.
// A block that holds an infinity or a NaN is NaN throughout, with scale 1.
#include "../../include/pydtnn_hip.h"
#include "conv_internal.h"
#include "dtypes.h"

namespace {

constexpr int kT = 256;
constexpr int kWave = 64;
constexpr int kBlock = 128;

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

struct Fp8Shape {
    long m, n, k;
    int blocks, words;      // blocks of 128 of a row, words of four scales of a row
};

// Biased exponent of the scale of a block from the bits of its largest magnitude; 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_byte(uint32_t amax)
{
    const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 0 ? 0 : e;
}

// One wave takes four blocks of a row, 16 lanes a block, eight elements a lane.
template <typename T, bool PACKED>
__global__ void __launch_bounds__(kT) quantize_fp8_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                          uint32_t* __restrict__ scales, long rows, long k, int blocks,
                                                          int words)
{
    const long item = (long)blockIdx.x * (kT / kWave) + threadIdx.x / kWave;
    if (item >= rows * words) return;
    const long row = item / words;
    const int lane = threadIdx.x % kWave;
    const long c = (item % words) * 4 * kBlock + lane * 8;
    float v[8];
    if (PACKED && c + 8 <= k) {
        const Pack<T, 8> p = *reinterpret_cast<const Pack<T, 8>*>(x + row * k + c);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)p.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < k ? (float)x[row * k + c + j] : 0.0f;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o, kWave));
    const bool finite = amax < 0x7f800000u;
    const bool real = c / kBlock < blocks;
    const int byte = finite && real ? scale_byte(amax) : 127;
    const float inverse = __uint_as_float((uint32_t)(254 - byte) << 23);      // 2^-(byte - 127), byte <= 247
    if (real) {
        uint2 out;
        if (finite) {
            int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, 0, false);
            int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inverse, v[5] * inverse, 0, false);
            a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, a, true);
            b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inverse, v[7] * inverse, b, true);
            out = make_uint2((uint32_t)a, (uint32_t)b);
        } else {
            out = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
        }
        *reinterpret_cast<uint2*>(q + row * blocks * kBlock + c) = out;
    }
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) word |= (uint32_t)__shfl(byte, b * 16, kWave) << (8 * b);
    if (lane == 0) scales[item] = word;
}

// acc += the product of one block: 32 bytes a lane of each operand, lane l those of row l % 16, with the scale bytes of
// those rows in the low byte of `we` and `xe`.  Both operands take the bytes of a block in the same order, which is all
// that a sum over the block asks for.
template <bool EXACT>
__device__ __forceinline__ v4f block_product(v8i w, int we, v8i x, int xe, v4f acc)
{
    if (!EXACT) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, acc, 0, 0, 0, we, 0, xe);
    const float wf = __int_as_float((we & 255) << 23), xf = __int_as_float((xe & 255) << 23);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        v8b a, b;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const v2b a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i + j], wf, false);
            const v2b a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i + j], wf, true);
            const v2b b0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i + j], xf, false);
            const v2b b1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i + j], xf, true);
            a[4 * j] = a0[0], a[4 * j + 1] = a0[1], a[4 * j + 2] = a1[0], a[4 * j + 3] = a1[1];
            b[4 * j] = b0[0], b[4 * j + 1] = b0[1], b[4 * j + 2] = b1[0], b[4 * j + 3] = b1[1];
        }
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
    }
    return acc;
}

// One wave computes 16 n by 16 m.  The weights are the first operand, so that a lane ends with four consecutive n of one m.
template <typename T>
__global__ void __launch_bounds__(kT) matmul_fp8_kernel(const uint8_t* __restrict__ xq, const uint32_t* __restrict__ xs,
                                                        const uint8_t* __restrict__ wq, const uint32_t* __restrict__ ws,
                                                        const float* __restrict__ bias, T* __restrict__ y, Fp8Shape s,
                                                        int relu)
{
    const int lane = threadIdx.x % kWave, row = lane % 16, part = lane / 16;
    const long n0 = (long)blockIdx.x * 64 + threadIdx.x / kWave * 16, m0 = (long)blockIdx.y * 16;
    const long wr = min(n0 + row, s.n - 1), xr = min(m0 + row, s.m - 1);
    const long kp = (long)s.blocks * kBlock;
    const v4i* wp = reinterpret_cast<const v4i*>(wq + wr * kp + part * 32);
    const v4i* xp = reinterpret_cast<const v4i*>(xq + xr * kp + part * 32);
    v4f acc = {0, 0, 0, 0};
    for (int b = 0; b < s.blocks; ++b) {
        const v4i w0 = wp[b * 8], w1 = wp[b * 8 + 1], x0 = xp[b * 8], x1 = xp[b * 8 + 1];
        const v8i wv = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
        const v8i xv = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
        const int we = (int)(ws[wr * s.words + b / 4] >> (b % 4 * 8)), xe = (int)(xs[xr * s.words + b / 4] >> (b % 4 * 8));
        acc = block_product<sizeof(T) == 4>(wv, we, xv, xe, acc);
    }
    const long m = m0 + row;
    if (m >= s.m) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long n = n0 + part * 4 + i;
        if (n >= s.n) return;
        float v = acc[i] + (bias ? bias[n] : 0.0f);
        if (relu) v = v > 0.0f ? v : 0.0f;
        y[m * s.n + n] = (T)v;
    }
}

bool shape_of(Fp8Shape* s, long m, long n, long k)
{
    if (m <= 0 || n <= 0 || k <= 0) return false;
    *s = Fp8Shape{m, n, k, (int)((k + kBlock - 1) / kBlock), (int)((k + 4 * kBlock - 1) / (4 * kBlock))};
    return true;
}

size_t q_bytes(const Fp8Shape& s) { return (size_t)s.m * s.blocks * kBlock; }

template <typename F>
int with_fp8_input(int dtype, F f)
{
    switch (dtype) {
        case kDtypeF32: return f(float());
        case kDtypeF16: return f((_Float16)0);
        case kDtypeBF16: return f((__bf16)0.0f);
        default: return PYDTNN_HIP_ERR_INVALID;
    }
}

template <typename T>
int quantize(const T* x, long rows, long k, uint8_t* q, uint8_t* scales, hipStream_t st)
{
    Fp8Shape s;
    if (!shape_of(&s, rows, 1, k)) return PYDTNN_HIP_ERR_INVALID;
    const long blocks = (rows * s.words + kT / kWave - 1) / (kT / kWave);
    if (blocks * kT >= (1l << 32)) return PYDTNN_HIP_ERR_UNSUPPORTED;     // a launch counts its threads in 32 bits
    if (aligned16(x) && k % 8 == 0)
        hipLaunchKernelGGL((quantize_fp8_kernel<T, true>), dim3((unsigned)blocks), dim3(kT), 0, st, x, q, (uint32_t*)scales,
                           rows, k, s.blocks, s.words);
    else
        hipLaunchKernelGGL((quantize_fp8_kernel<T, false>), dim3((unsigned)blocks), dim3(kT), 0, st, x, q, (uint32_t*)scales,
                           rows, k, s.blocks, s.words);
    HIP_RETURN_IF_LAUNCH_FAILED();
    return PYDTNN_HIP_OK;
}

constexpr long kMost = 1l << 30;      // rows and columns are counted in 32 bits

}  // namespace

extern "C" {

int pydtnn_hip_quantize_fp8(int dtype, const void* x, long rows, long k, uint8_t* q, uint8_t* scales, void* stream)
{
    if (!x || !q || !scales) return PYDTNN_HIP_ERR_INVALID;
    if (!aligned16(q) || ((uintptr_t)scales & 3)) return PYDTNN_HIP_ERR_INVALID;
    if (rows > kMost || k > kMost) return PYDTNN_HIP_ERR_UNSUPPORTED;
    return with_fp8_input(dtype, [&](auto t) {
        using T = decltype(t);
        return quantize<T>((const T*)x, rows, k, q, scales, convint::as_stream(stream));
    });
}

size_t pydtnn_hip_matmul_fp8_workspace_bytes(long m, long n, long k)
{
    Fp8Shape s;
    if (!shape_of(&s, m, n, k) || m > kMost || n > kMost || k > kMost) return 0;
    return q_bytes(s) + (size_t)m * s.words * 4;
}

int pydtnn_hip_matmul_fp8(int dtype, const void* x, long m, long k, const uint8_t* wq, const uint8_t* wscales, long n,
                          const float* bias, int relu, void* y, void* workspace, size_t workspace_bytes, void* stream)
{
    Fp8Shape s;
    if (!x || !wq || !wscales || !y || !shape_of(&s, m, n, k)) return PYDTNN_HIP_ERR_INVALID;
    if (!aligned16(wq) || ((uintptr_t)wscales & 3)) return PYDTNN_HIP_ERR_INVALID;
    if (m > kMost || n > kMost || k > kMost || (m + 15) / 16 > 65535) return PYDTNN_HIP_ERR_UNSUPPORTED;
    if (!workspace || !aligned16(workspace) || workspace_bytes < pydtnn_hip_matmul_fp8_workspace_bytes(m, n, k))
        return PYDTNN_HIP_ERR_WORKSPACE;
    return with_fp8_input(dtype, [&](auto t) {
        using T = decltype(t);
        const hipStream_t st = convint::as_stream(stream);
        uint8_t* xq = static_cast<uint8_t*>(workspace);
        uint8_t* xs = xq + q_bytes(s);
        const int rc = quantize<T>((const T*)x, m, k, xq, xs, st);
        if (rc != PYDTNN_HIP_OK) return rc;
        hipLaunchKernelGGL((matmul_fp8_kernel<T>), dim3((unsigned)((n + 63) / 64), (unsigned)((m + 15) / 16)), dim3(kT), 0, st,
                           xq, (const uint32_t*)xs, wq, (const uint32_t*)wscales, bias, (T*)y, s, relu);
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    });
}

}  // extern "C"
