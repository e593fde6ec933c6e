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
//       step that a float16 result is rounded by.  4096 x 4096 x 4096 in bfloat16 lies 2.0e-4 of its norm from sums of 24 bits
//       rounded alike, and 1.66e-3 from the result in 64 bits, as those do: that is its own rounding.
//   float32 results: the operands are converted to bfloat16 with their scales, which is exact, and go through
//       v_mfma_f32_16x16x32_bf16, which keeps 24 bits of everything it adds (4096 x 4096 x 4096: 126 us, 68 in bfloat16).
//
// Layout: q is (rows, k to a multiple of 128), zeros behind k; scales is (rows, blocks to a multiple of 4), one byte e + 127
// each, 127 behind the last block, so that a lane fetches the scales of four blocks as one word.
// A block that holds an infinity or a NaN is NaN throughout, with scale 1.
//
// Times below, unless they are the product's alone, are of whole calls in a replayed graph, inputs from three sets in turn.  Rows of
// a thousand calls without a graph take less where a call is long (4096 x 4096 x 4096 in bfloat16 68 us, 72 in the graph; 16 x 25088 x
// 4096 32 and 35) and more where it is short, by what a call costs the host (1 x 4096 x 1000 10 and 6).
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

struct Eight {
    uint2 q;
    int byte;
};

// Eight elements c .. c + 7 of a row, by one of the 16 lanes that have a block: their e4m3 values and the block's scale byte.
template <typename T>
__device__ __forceinline__ Eight quantize_eight(const T* __restrict__ row, long c, long k)
{
    float v[8];
    if (c + 8 <= k) {
        T p[8];
        // loads of 16 bytes wherever the row starts (4096 x 4097 in float32: 14.6 us, 33.5 an element at a time)
        __builtin_memcpy(p, row + c, sizeof(p));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)p[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < k ? (float)row[c + j] : 0.0f;
    }
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o, kWave));
    Eight e;
    if (amax < 0x7f800000u) {
        e.byte = scale_byte(amax);
        const float inverse = __uint_as_float((uint32_t)(254 - e.byte) << 23);      // 2^-(byte - 127), byte <= 247
        int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inverse, v[1] * inverse, 0, false);
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inverse, v[5] * inverse, 0, false);
        a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inverse, v[3] * inverse, a, true);
        b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inverse, v[7] * inverse, b, true);
        e.q = make_uint2((uint32_t)a, (uint32_t)b);
    } else {      // an infinity or a NaN
        e.byte = 127;
        e.q = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
    }
    return e;
}

// One wave takes four blocks of a row, 16 lanes a block.
template <typename T>
__global__ void __launch_bounds__(kT) quantize_fp8_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                          uint32_t* __restrict__ scales, long rows, long k, int blocks,
                                                          int words)
{
    const long item = (long)blockIdx.x * (kT / kWave) + threadIdx.x / kWave;
    if (item >= rows * words) return;
    const long row = item / words;
    const int lane = threadIdx.x % kWave;
    const long c = (item % words) * 4 * kBlock + lane * 8;
    Eight e = quantize_eight<T>(x + row * k, c, k);
    if (c / kBlock < blocks) *reinterpret_cast<uint2*>(q + row * blocks * kBlock + c) = e.q;
    else e.byte = 127;
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) word |= (uint32_t)__shfl(e.byte, b * 16, kWave) << (8 * b);
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

// bias, ReLU and the one rounding to the type of the result
template <typename T>
__device__ __forceinline__ T finish(float v, const float* bias, long n, int relu)
{
    if (bias) v += bias[n];
    if (relu) v = v > 0.0f ? v : 0.0f;
    return (T)v;
}

// Four consecutive n of one m.
template <typename T>
__device__ __forceinline__ void store_four(T* y, long m, long n, const Fp8Shape& s, v4f v, const float* bias, int relu)
{
    T* to = y + m * s.n + n;
    if (n + 4 <= s.n && s.n % 4 == 0 && ((uintptr_t)y & (4 * sizeof(T) - 1)) == 0) {
        Pack<T, 4> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out.v[i] = finish<T>(v[i], bias, n + i, relu);
        *reinterpret_cast<Pack<T, 4>*>(to) = out;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < s.n) to[i] = finish<T>(v[i], bias, n + i, relu);
}

// A buffer resource over rows from `base`: what is read behind the last byte is zero.
typedef __amdgpu_buffer_rsrc_t Rows;
__device__ __forceinline__ Rows rows_of(const void* base, long bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(uint32_t)min(bytes, 0xffffffffl), 0x00020000);
}

// The same as the four words that inline assembly takes.
typedef v4i RowsWords;
__device__ __forceinline__ RowsWords rows_words(const void* base, long bytes)
{
    return RowsWords{(int)(uint32_t)(uintptr_t)base, (int)((uintptr_t)base >> 32), (int)(uint32_t)min(bytes, 0xffffffffl),
                     0x00020000};
}

// ---------------------------------------------------------------------------------------------- few rows
// Up to 16 rows of x: bound by reading the weights, each of which is used for those rows only.  A workgroup takes 16 rows
// of the weights; its waves take the words of four blocks in turn, with the next word's operands on their way while
// the present one's are multiplied, and join their sums in local memory, in the order of the waves.  The weights are the
// first operand, so that a lane ends with four consecutive n of one m.
//
// Where local memory holds all of x (kFewLocal bytes), every workgroup quantises it for itself, while its first weights
// are on their way: one launch instead of two (1 x 4096 x 1000 in float32: 5.8 us, 7.4 with two).  Otherwise x comes quantised.
// 16 x 4096 x 1000 in float32 takes 9 us, 12 in tiles; 8 x 4096 x 4096 9.5 and 13; 16 x 25088 x 4096 35 and 38, where the
// weights arrive at 3.6 TB/s beside as many bytes of x from the second-level cache.
constexpr int kFewWaves = 8, kFewLocal = 32 * 1024;

__device__ __forceinline__ v8i join(v4i a, v4i b)
{
    return v8i{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A word of four blocks of 16 rows: a lane's two pieces of each block, and the four scale bytes.  Blocks behind the last are
// not used: of buffers that one is read again, since an offset beyond a buffer's end would be outside its range check; local
// memory holds something there.
struct WordOfBlocks {
    v4i q[4][2];
    int e;

    // `at`: a lane's offset in bytes, of its row and piece; `scale_at`: that of its row's scales; `last`: a row's last block
    __device__ __forceinline__ void load(Rows rows, int at, Rows scales, int scale_at, int word, int last)
    {
        e = __builtin_amdgcn_raw_buffer_load_b32(scales, scale_at, word * 4, 0);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int from = min(word * 4 + b, last) * kBlock;
            q[b][0] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rows, at, from, 0));
            q[b][1] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rows, at + 64, from, 0));
        }
    }
    __device__ __forceinline__ void load(const uint8_t* row, const uint8_t* scales, int word)
    {
        e = *reinterpret_cast<const int*>(scales + word * 4);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            q[b][0] = *reinterpret_cast<const v4i*>(row + (word * 4 + b) * kBlock);
            q[b][1] = *reinterpret_cast<const v4i*>(row + (word * 4 + b) * kBlock + 64);
        }
    }
};

template <typename T, int DEPTH, bool LOCAL>
__global__ void __launch_bounds__(kFewWaves* kWave) matmul_fp8_few_kernel(const T* __restrict__ x,
                                                                          const uint8_t* __restrict__ xq,
                                                                          const uint32_t* __restrict__ xs,
                                                                          const uint8_t* __restrict__ wq,
                                                                          const uint32_t* __restrict__ ws,
                                                                          const float* __restrict__ bias, T* __restrict__ y,
                                                                          Fp8Shape s, int relu)
{
    constexpr bool EXACT = sizeof(T) == 4;
    __shared__ v4f part[kFewWaves][kWave];
    // a row of x and its scale words; 16 bytes more than its values, so that rows start on different banks
    __shared__ __attribute__((aligned(16))) uint8_t local[LOCAL ? kFewLocal + 4 * kBlock : 16];      // (the last word's end)
    const int lane = threadIdx.x % kWave, row = lane % 16, piece = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long n0 = (long)blockIdx.x * 16, kp = (long)s.blocks * kBlock;
    const Rows wrows = rows_of(wq + n0 * kp, (s.n - n0) * kp), wscales = rows_of(ws + n0 * s.words, (s.n - n0) * s.words * 4);
    const int at = (int)(row * kp) + piece * 16, scale_at = row * s.words * 4;
    v4f acc = {0, 0, 0, 0};
    // The wave's words are wave, wave + kFewWaves, ...; DEPTH - 1 of them are on their way while one is multiplied.  They stand
    // in places of their own in turn: a copy from one place to another would wait for its loads.
    const int mine = s.words > wave ? (s.words - wave + kFewWaves - 1) / kFewWaves : 0;
    auto word_of = [&](int i) { return wave + i * kFewWaves; };
    WordOfBlocks w[DEPTH], v[LOCAL ? 1 : DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d)
        if (d < mine) w[d].load(wrows, at, wscales, scale_at, word_of(d), s.blocks - 1);
    const long stride = kp + 16 + (s.words * 4 + 15) / 16 * 16;
    // rows behind the last are that one again in local memory, zeros otherwise
    const uint8_t* xlocal = local + min((long)row, s.m - 1) * stride;
    const Rows xrows = rows_of(xq, LOCAL ? 0 : s.m * kp), xscales = rows_of(xs, LOCAL ? 0 : s.m * s.words * 4);
    if constexpr (LOCAL) {
        for (int item = wave; item < s.m * s.words; item += kFewWaves) {
            const int r = item / s.words, word = item % s.words, c = word * 4 * kBlock + lane * 8;
            const Eight e = quantize_eight<T>(x + (long)r * s.k, c, s.k);
            if (c < kp) {
                *reinterpret_cast<uint2*>(local + r * stride + c) = e.q;
                if (lane % 16 == 0) local[r * stride + kp + 16 + c / kBlock] = (uint8_t)e.byte;
            }
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int d = 0; d < DEPTH - 1; ++d)
            if (d < mine) v[d].load(xrows, at, xscales, scale_at, word_of(d), s.blocks - 1);
    }
    for (int done = 0; done < mine; done += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (done + d >= mine) break;
            const int ahead = word_of(done + d + DEPTH - 1), word = word_of(done + d);
            const bool more = done + d + DEPTH - 1 < mine;
            if (more) w[(d + DEPTH - 1) % DEPTH].load(wrows, at, wscales, scale_at, ahead, s.blocks - 1);
            if constexpr (LOCAL) v[0].load(xlocal + piece * 16, xlocal + kp + 16, word);
            else if (more) v[(d + DEPTH - 1) % DEPTH].load(xrows, at, xscales, scale_at, ahead, s.blocks - 1);
            const WordOfBlocks& here = v[LOCAL ? 0 : d];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (word * 4 + b >= s.blocks) break;
                acc = block_product<EXACT>(join(w[d].q[b][0], w[d].q[b][1]), w[d].e >> (8 * b),
                                           join(here.q[b][0], here.q[b][1]), here.e >> (8 * b), acc);
            }
        }
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    v4f sum = part[0][lane];
#pragma unroll
    for (int k = 1; k < kFewWaves; ++k) sum += part[k][lane];
    const long n = n0 + piece * 4;
    if (row < s.m && n < s.n) store_four(y, (long)row, n, s, sum, bias, relu);
}

// ---------------------------------------------------------------------------------------------- tiles
// A workgroup of WN x WM waves computes BN rows of the weights by BM rows of x.  A step is one block of 128 k: its BN + BM
// rows of 128 bytes go to local memory by loads that write there directly, STAGES - 1 steps ahead of their use.  The
// eight 16-byte pieces of a row r stand at place piece ^ (r % 8), so that the sixteen rows that a fragment reads at once fall
// on different banks; the loads' lanes pick their pieces accordingly, and since a lane's two pieces of a block are any two,
// as long as both operands take the same, a lane takes pieces p and p + 4.
// m0 is set here and nowhere else; the compiler warns that it reserves it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// Loads that write local memory directly: 16 bytes, or 4, a lane, to `to` + lane * 16 (4).  As the builtin the compiler lets
// every later read of local memory wait for them, whatever it reads: no load would be under way beside the products (4096 x
// 4096 x 4096: 75 us that way).  There is no output register; what waits for them is wait_loads and the barrier behind it.
__device__ __forceinline__ void load_quads(uint32_t to, uint32_t at, RowsWords rows, int offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(at), "s"(rows), "s"(offset) : "memory", "m0");
}
__device__ __forceinline__ void load_words(uint32_t to, uint32_t at, RowsWords rows, int offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 ::"s"(to), "v"(at), "s"(rows), "s"(offset) : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t local_address(const void* p)
{
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Waits for all but the last N loads, and for this wave's reads of local memory, whose place the other waves' loads take next.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// Writes a tile through local memory, so that whole lines of rows go out: lanes hold four n of 16 different m each (the tile of
// 4096 x 4096 x 4096 that way took 62 us without a single load, of which 27 were its products).  The 16-byte pieces of row m
// stand at place piece ^ (m % 16), or less where a row has fewer pieces.
template <typename T, int BN, int BM, int TN, int TM, int WAVES>
__device__ __forceinline__ void store_tile(uint8_t* lds, const v4f (&acc)[TN][TM], int wn, int wm, T* __restrict__ y, long m0,
                                           long n0, const Fp8Shape& s, const float* __restrict__ bias, int relu)
{
    constexpr int PER = 16 / (int)sizeof(T), PIECES = BN / PER;      // elements of a piece, pieces of a row
    constexpr int TURNS = PIECES < 16 ? PIECES : 16;
    const int lane = threadIdx.x % kWave, row = lane % 16, piece = lane / 16;
    auto place = [&](int m, int n) { return lds + m * BN * sizeof(T) + ((n / PER) ^ (m % TURNS)) * 16; };
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const int n = (wn * TN + i) * 16 + piece * 4;
        v4f b = {0, 0, 0, 0};
        if (bias) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (n0 + n + k < s.n) b[k] = bias[n0 + n + k];
        }
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int m = (wm * TM + j) * 16 + row;
            Pack<T, 4> out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v = acc[i][j][k] + b[k];
                if (relu) v = v > 0.0f ? v : 0.0f;
                out.v[k] = (T)v;
            }
            *reinterpret_cast<Pack<T, 4>*>(place(m, n) + n % PER * sizeof(T)) = out;
        }
    }
    __syncthreads();
    const bool whole = s.n % PER == 0 && ((uintptr_t)y & 15) == 0;
#pragma unroll 4
    for (int at = threadIdx.x; at < BM * PIECES; at += WAVES * kWave) {
        const int m = at / PIECES, n = at % PIECES * PER;
        if (m0 + m >= s.m || n0 + n >= s.n) continue;
        const Pack<T, PER> v = *reinterpret_cast<const Pack<T, PER>*>(place(m, n));
        T* to = y + (m0 + m) * s.n + n0 + n;
        if (whole) {
            // past the caches: the workgroups of a launch store all at once (4096 x 4096 in bfloat16: 13 us, plain stores 19)
            typedef uint32_t quad __attribute__((ext_vector_type(4)));
            __builtin_nontemporal_store(*reinterpret_cast<const quad*>(&v), reinterpret_cast<quad*>(to));
        } else {
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (n0 + n + k < s.n) to[k] = v.v[k];
        }
    }
}

template <typename T, bool EXACT, int BN, int BM, int WN, int WM, int STAGES>
__global__ void __launch_bounds__(WN* WM* kWave, STAGES * (BN + BM) * kBlock > 80 * 1024 ? 1 : 2)
    matmul_fp8_tile_kernel(const uint8_t* __restrict__ xq, const uint32_t* __restrict__ xs, const uint8_t* __restrict__ wq,
                           const uint32_t* __restrict__ ws, const float* __restrict__ bias, T* __restrict__ y,
                           float* __restrict__ partial, Fp8Shape s, int relu, int tiles_n, int tiles_m, int splits)
{
    constexpr int WAVES = WN * WM, TN = BN / WN / 16, TM = BM / WM / 16;
    constexpr int WLOADS = BN / 8 / WAVES, LOADS = (BN + BM) / 8 / WAVES;     // loads of a wave and step: eight rows each
    constexpr int STAGE = (BN + BM) * kBlock;
    constexpr int CHUNKS = (BN + BM) / 64;      // scale words: 64 rows to a load
    constexpr int EACH = (CHUNKS + WAVES - 1) / WAVES;
    __shared__ __attribute__((aligned(128))) uint8_t lds[STAGES * STAGE];
    __shared__ uint32_t scale[2][BN + BM];

    // Consecutive workgroups go to the eight dies in turn; a die's tiles are consecutive, in bands of four tiles of n, so that
    // its second-level cache holds what they share.
    const long tiles = (long)tiles_n * tiles_m * splits, share = (tiles + 7) / 8;
    const long place = (long)(blockIdx.x % 8) * share + blockIdx.x / 8;
    if (blockIdx.x / 8 >= share || place >= tiles) return;
    const int split = (int)(place % splits);
    const long tile = place / splits;
    const int band = (int)(tile / (4l * tiles_m)), in_band = (int)(tile % (4l * tiles_m));
    const int band_n = min(4, tiles_n - band * 4);
    const long n0 = (band * 4l + in_band % band_n) * BN, m0 = (long)(in_band / band_n) * BM;

    const int words = (s.words + splits - 1) / splits;      // of a split
    const int first = split * words * 4, last = min((split + 1) * words * 4, s.blocks);

    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int row = lane % 16, piece = lane / 16, wn = wave % WN, wm = wave / WN;
    const long kp = (long)s.blocks * kBlock;
    const RowsWords wres = rows_words(wq + n0 * kp, (s.n - n0) * kp), xres = rows_words(xq + m0 * kp, (s.m - m0) * kp);
    uint32_t from[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (wave + (i < WLOADS ? i : i - WLOADS) * WAVES) * 8 + lane / 8;
        from[i] = (uint32_t)(r * kp) + (uint32_t)(((lane % 8) ^ (lane / 8)) * 16);
    }
    // the scale words of W's rows, then of x's, 64 rows to a load; where all of those are behind the last, one row is left
    // to read, since an offset beyond a buffer's end would be outside its range check
    RowsWords scale_from[EACH];
    const uint32_t scale_at = (uint32_t)(lane * s.words * 4);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const int chunk = wave + e * WAVES;
        const bool of_w = chunk < BN / 64;
        const long r = of_w ? n0 + chunk * 64 : m0 + (chunk - BN / 64) * 64, left = (of_w ? s.n : s.m) - r;
        scale_from[e] = rows_words((of_w ? ws : xs) + (left > 0 ? r : 0) * s.words, max(left, 1l) * s.words * 4);
    }
    const uint32_t lds_at = local_address(lds), scales_at = local_address(scale);
    auto load_rows = [&](int step, int stage, int i) {
        const int group = i < WLOADS ? wave + i * WAVES : BN / 8 + wave + (i - WLOADS) * WAVES;
        load_quads(lds_at + stage * STAGE + group * 1024, from[i], i < WLOADS ? wres : xres, step * kBlock);
    };
    // with the first of four steps, their scales; two words' scales have a place each
    auto load_scales = [&](int step) {
        if (step % 4 == 0) {
#pragma unroll
            for (int e = 0; e < EACH; ++e)
                if (CHUNKS % WAVES == 0 || wave + e * WAVES < CHUNKS)
                    load_words(scales_at + (step / 4 & 1) * (BN + BM) * 4 + (wave + e * WAVES) * 256, scale_at, scale_from[e],
                               step / 4 * 4);
        }
    };

    int we[TN] = {}, xe[TM] = {};
    v4f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j) acc[i][j] = v4f{0, 0, 0, 0};

    if (first < last) {
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t)
            if (first + t < last) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) load_rows(first + t, t, i);
                load_scales(first + t);
            }
    }
    const uint32_t mine = (uint32_t)((row * kBlock) + ((piece ^ (row % 8)) * 16));
    const uint32_t wbase = (uint32_t)(wn * TN * 16 * kBlock) + mine, xbase = (uint32_t)((BN + wm * TM * 16) * kBlock) + mine;
    int stage = 0;
    for (int step = first; step < last; ++step) {
        // this step's loads are the oldest; while later steps' follow them, those may stay under way
        if (STAGES > 2 && step + STAGES - 2 < last) wait_loads<(STAGES - 2) * LOADS>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");      // no access moves across the barrier
        const int coming = step + STAGES - 1, coming_stage = stage == 0 ? STAGES - 1 : stage - 1;
        if (coming < last) load_scales(coming);
        const uint8_t* here = lds + stage * STAGE;
        if (step % 4 == 0) {
            const uint32_t* words_here = scale[step / 4 & 1];
#pragma unroll
            for (int i = 0; i < TN; ++i) we[i] = (int)words_here[(wn * TN + i) * 16 + row];
#pragma unroll
            for (int j = 0; j < TM; ++j) xe[j] = (int)words_here[BN + (wm * TM + j) * 16 + row];
        } else {
#pragma unroll
            for (int i = 0; i < TN; ++i) we[i] = (int)((uint32_t)we[i] >> 8);
#pragma unroll
            for (int j = 0; j < TM; ++j) xe[j] = (int)((uint32_t)xe[j] >> 8);
        }
        v8i x[TM];
#pragma unroll
        for (int j = 0; j < TM; ++j)
            x[j] = join(*reinterpret_cast<const v4i*>(here + xbase + j * 16 * kBlock),
                        *reinterpret_cast<const v4i*>(here + (xbase ^ 64u) + j * 16 * kBlock));
        auto weights = [&](int i) {
            return join(*reinterpret_cast<const v4i*>(here + wbase + i * 16 * kBlock),
                        *reinterpret_cast<const v4i*>(here + (wbase ^ 64u) + i * 16 * kBlock));
        };
        v8i w = weights(0);
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const v8i after = weights(i + 1 < TN ? i + 1 : i);
            // a coming step's loads, a few at a time over the first half of the products
            if (coming < last) {
#pragma unroll
                for (int l = i * 2 * LOADS / TN; l < (i + 1) * 2 * LOADS / TN && l < LOADS; ++l)
                    load_rows(coming, coming_stage, l);
            }
#pragma unroll
            for (int j = 0; j < TM; ++j) acc[i][j] = block_product<EXACT>(w, we[i], x[j], xe[j], acc[i][j]);
            w = after;
        }
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }

    if (splits == 1) {
        store_tile<T, BN, BM, TN, TM, WAVES>(lds, acc, wn, wm, y, m0, n0, s, bias, relu);
    } else if constexpr (BN == 64) {      // (larger tiles are enough by themselves)
        store_tile<float, BN, BM, TN, TM, WAVES>(lds, acc, wn, wm, partial + split * s.m * s.n, m0, n0, s, nullptr, 0);
    }
}

// The sum of the splits' results, in order.
template <typename T>
__global__ void __launch_bounds__(kT) join_splits_kernel(const float* __restrict__ partial, const float* __restrict__ bias,
                                                         T* __restrict__ y, long m, long n, int splits, int relu)
{
    const long i = (long)blockIdx.x * kT + threadIdx.x;
    if (i >= m * n) return;
    float v = partial[i];
    for (int k = 1; k < splits; ++k) v += partial[k * m * n + i];
    y[i] = finish<T>(v, bias, i % n, relu);
}

bool shape_of(Fp8Shape* s, long m, long n, long k)
{
    if (m <= 0 || n <= 0 || k <= 0) return false;
    *s = Fp8Shape{m, n, k, (int)((k + kBlock - 1) / kBlock), (int)((k + 4 * kBlock - 1) / (4 * kBlock))};
    return true;
}

size_t q_bytes(const Fp8Shape& s) { return (size_t)s.m * s.blocks * kBlock; }
size_t scale_bytes(const Fp8Shape& s) { return ((size_t)s.m * s.words * 4 + 15) / 16 * 16; }

constexpr long kFewRows = 16;
constexpr int kSplitsMost = 16;

// Tiles of `size` by `size`: the largest that are about enough for 256 compute units.  In bfloat16, quantising x included:
// 4096 x 4096 x 4096 72 us with 256 by 256, 79 with 128 by 128, 123 with 64 by 64; 1024 x 4096 x 4096 35 with 128, 57 with
// 256, 37 with 64; 512 x 4096 x 4096 23 with 64, 33 with 128.  Where tiles of 64 are too few, k is cut into `splits` pieces of
// at least two words of four blocks, a workgroup each, as far as there are units for them (777 x 2049 x 1003 in float16: 15 us
// with 208 workgroups, 20 with twice as many, whose results have to be joined; 64 x 25088 x 4096: 37 and 41).
struct Tiling {
    int size, splits;
};

Tiling tiling_of(const Fp8Shape& s, bool exact)
{
    auto tiles = [&](long size) { return ((s.m + size - 1) / size) * ((s.n + size - 1) / size); };
    Tiling t = {64, 1};
    if (!exact && tiles(256) >= 192) t.size = 256;
    else if (tiles(128) >= 192) t.size = 128;
    const long count = tiles(t.size);
    if (t.size == 64) {
        long splits = 256 / count;
        if (splits > s.words / 2) splits = s.words / 2;
        if (splits > kSplitsMost) splits = kSplitsMost;
        if (splits > 1) t.splits = (int)splits;
    }
    return t;
}

// Whether a workgroup of the few rows' kernel holds all of x: values, scales and 16 bytes a row.
bool few_local(const Fp8Shape& s)
{
    return s.m <= kFewRows && s.m * ((long)s.blocks * kBlock + 16 + (s.words * 4 + 15) / 16 * 16) <= kFewLocal;
}

size_t partial_bytes(const Fp8Shape& s, bool exact)
{
    if (s.m <= kFewRows) return 0;
    const Tiling t = tiling_of(s, exact);
    return t.splits > 1 ? (size_t)t.splits * s.m * s.n * 4 : 0;
}

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
    hipLaunchKernelGGL((quantize_fp8_kernel<T>), dim3((unsigned)blocks), dim3(kT), 0, st, x, q, (uint32_t*)scales, rows, k,
                       s.blocks, s.words);
    HIP_RETURN_IF_LAUNCH_FAILED();
    return PYDTNN_HIP_OK;
}

template <typename T, bool EXACT, int BN, int BM, int WN, int WM, int STAGES>
int launch_tiles(const uint8_t* xq, const uint8_t* xs, const uint8_t* wq, const uint8_t* ws, const float* bias, T* y,
                 float* partial, const Fp8Shape& s, int relu, int splits, hipStream_t st)
{
    const long tiles_n = (s.n + BN - 1) / BN, tiles_m = (s.m + BM - 1) / BM;
    const long blocks = (tiles_n * tiles_m * splits + 7) / 8 * 8;
    if (blocks * WN * WM * kWave >= (1l << 32)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((matmul_fp8_tile_kernel<T, EXACT, BN, BM, WN, WM, STAGES>), dim3((unsigned)blocks),
                       dim3(WN * WM * kWave), 0, st, xq, (const uint32_t*)xs, wq, (const uint32_t*)ws, bias, y, partial,
                       s, relu, (int)tiles_n, (int)tiles_m, splits);
    HIP_RETURN_IF_LAUNCH_FAILED();
    if (splits == 1) return PYDTNN_HIP_OK;
    const long join = (s.m * s.n + kT - 1) / kT;
    if (join * kT >= (1l << 32)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((join_splits_kernel<T>), dim3((unsigned)join), dim3(kT), 0, st, partial, bias, y, s.m, s.n, splits,
                       relu);
    HIP_RETURN_IF_LAUNCH_FAILED();
    return PYDTNN_HIP_OK;
}

template <typename T>
int product(const T* x, const uint8_t* xq, const uint8_t* xs, const uint8_t* wq, const uint8_t* ws, const float* bias, T* y,
            float* partial, const Fp8Shape& s, int relu, hipStream_t st)
{
    constexpr bool EXACT = sizeof(T) == 4;
    if (s.m <= kFewRows) {
        const long blocks = (s.n + 15) / 16;
        if (blocks * kFewWaves * kWave >= (1l << 32)) return PYDTNN_HIP_ERR_UNSUPPORTED;
        auto few = [&](auto local) {
            hipLaunchKernelGGL((matmul_fp8_few_kernel<T, 2, decltype(local)::value>), dim3((unsigned)blocks),
                               dim3(kFewWaves * kWave), 0, st, x, xq, (const uint32_t*)xs, wq, (const uint32_t*)ws, bias, y, s,
                               relu);
        };
        if (few_local(s)) few(std::true_type());
        else few(std::false_type());
        HIP_RETURN_IF_LAUNCH_FAILED();
        return PYDTNN_HIP_OK;
    }
    const Tiling t = tiling_of(s, EXACT);
    if constexpr (!EXACT)
        if (t.size == 256)
            return launch_tiles<T, EXACT, 256, 256, 2, 4, 2>(xq, xs, wq, ws, bias, y, partial, s, relu, t.splits, st);
    if (t.size == 128)
        return launch_tiles<T, EXACT, 128, 128, 2, 2, 2>(xq, xs, wq, ws, bias, y, partial, s, relu, t.splits, st);
    return launch_tiles<T, EXACT, 64, 64, 2, 2, 4>(xq, xs, wq, ws, bias, y, partial, s, relu, t.splits, st);
}

constexpr long kMost = 1l << 30, kMostK = 1l << 23;      // rows are counted, and a tile's rows addressed, in 32 bits

bool too_large(long m, long n, long k) { return m > kMost || n > kMost || k > kMostK; }

}  // namespace

extern "C" {

int pydtnn_hip_quantize_fp8(int dtype, const void* x, long rows, long k, uint8_t* q, uint8_t* scales, void* stream)
{
    if (!x || !q || !scales) return PYDTNN_HIP_ERR_INVALID;
    if (!aligned16(q) || ((uintptr_t)scales & 3)) return PYDTNN_HIP_ERR_INVALID;
    if (too_large(rows, 1, k)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    return with_fp8_input(dtype, [&](auto t) {
        using T = decltype(t);
        return quantize<T>((const T*)x, rows, k, q, scales, convint::as_stream(stream));
    });
}

size_t pydtnn_hip_matmul_fp8_workspace_bytes(int dtype, long m, long n, long k)
{
    Fp8Shape s;
    if (!shape_of(&s, m, n, k) || too_large(m, n, k)) return 0;
    return few_local(s) ? 0 : q_bytes(s) + scale_bytes(s) + partial_bytes(s, dtype == kDtypeF32);
}

int pydtnn_hip_matmul_fp8(int dtype, const void* x, long m, long k, const uint8_t* wq, const uint8_t* wscales, long n,
                          const float* bias, int relu, void* y, void* workspace, size_t workspace_bytes, void* stream)
{
    Fp8Shape s;
    if (!x || !wq || !wscales || !y || !shape_of(&s, m, n, k)) return PYDTNN_HIP_ERR_INVALID;
    if (!aligned16(wq) || ((uintptr_t)wscales & 3)) return PYDTNN_HIP_ERR_INVALID;
    if (too_large(m, n, k)) return PYDTNN_HIP_ERR_UNSUPPORTED;
    if (dtype == kDtypeF64) return PYDTNN_HIP_ERR_INVALID;
    const size_t need = pydtnn_hip_matmul_fp8_workspace_bytes(dtype, m, n, k);
    if (need && (!workspace || !aligned16(workspace) || workspace_bytes < need)) return PYDTNN_HIP_ERR_WORKSPACE;
    return with_fp8_input(dtype, [&](auto t) {
        using T = decltype(t);
        const hipStream_t st = convint::as_stream(stream);
        uint8_t* xq = static_cast<uint8_t*>(workspace);
        uint8_t* xs = need ? xq + q_bytes(s) : nullptr;
        float* partial = need ? reinterpret_cast<float*>(xs + scale_bytes(s)) : nullptr;
        const int rc = need ? quantize<T>((const T*)x, m, k, xq, xs, st) : PYDTNN_HIP_OK;
        if (rc != PYDTNN_HIP_OK) return rc;
        return product<T>((const T*)x, xq, xs, wq, wscales, bias, (T*)y, partial, s, relu, st);
    });
}

}  // extern "C"
