// Root-mean-square norm with the residual's addition and an 8-bit output with scales, and its gradients.
//
//   h = x + residual,   rstd = 1 / sqrt(mean(h^2) + eps),   y = (h * gamma) * rstd
//   q, scale: y in 8 bits with one scale per row, per group of columns, or e8m0 scales per 32 columns (MX)
//
// Memory bound: a row is read once, kept in registers in fp32, and every output is written once.  h is stored before the
// reduction (it does not depend on it), so what stays in registers is h * gamma alone, and because
// max|y| = max|h * gamma| * rstd the sum of squares and the largest magnitude of a row come out of one reduction.
//
// gradients, with hat = h * rstd and g = dy * gamma:   dx = rstd * (g - hat * mean(g * hat)) + dh,   dgamma = sum over rows of dy * hat
// One pass as well: a block walks rows and owns the same columns in each, so dgamma is summed in its registers; the blocks'
// partial sums go through the caller's workspace and are added in block order (no atomics: the result does not depend on timing).
#include <algorithm>

#include "partial_sum.cuh"

namespace ascb200 {
namespace {

// ---- rows in chunks of eight elements ------------------------------------------------------------------------------------
template <typename T>
struct Raw8;
template <>
struct Raw8<__half> {
    uint4 v;
};
template <>
struct Raw8<__nv_bfloat16> {
    uint4 v;
};
template <>
struct Raw8<float> {
    uint4 v, w;
};

// Two fp32 operations per instruction, each rounded to nearest.  The kernels move seven to eight bytes per element, so at the memory's rate an
// SM has about 30 instruction slots per element: with unpacked arithmetic and a test per chunk for the row's end (31 instructions) the forward
// pass took 145 us for 16383 x 7168 bf16 with residual and int8 codes; so, 131 us, and 124 (6.6 TB/s) since y and its code come from one product.
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, w, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// (not the read-only path: an output may be the row's own input)
__device__ __forceinline__ uint4 ld_v4(const void* p)
{
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

// One element where `inside`, else zero: a predicated load, so that the eight of a chunk go out back to back.
template <int BYTES>
__device__ __forceinline__ uint32_t ld_element(const void* p, bool inside)
{
    uint32_t r = 0u;
    if constexpr (BYTES == 4)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u32 %0, [%1];\n\t}" : "+r"(r) : "l"(p), "r"(static_cast<uint32_t>(inside)));
    else
        asm volatile("{\n\t.reg .pred q;\n\t.reg .u16 h;\n\tmov.u16 h, 0;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}"
                     : "=r"(r) : "l"(p), "r"(static_cast<uint32_t>(inside)));
    return r;
}

// How a thread's i-th eight columns lie; a warp owns 256 neighbouring columns in either case.
//   kVec       neighbours, one 16-byte access: every row of every tensor starts on 16 bytes and k is a multiple of 8;
//   kPairs     16-bit rows else, where all tensors' rows have the same parity: pairs, 64 columns apart, that start on 4 bytes (in a row that does
//              not, the pairs begin one column to the left: the first pair then has only its second column);
//   kElements  single elements, 32 columns apart, so that a warp's accesses are contiguous whatever the alignment.
// (us, bf16 with residual and int8 codes, 65536 x 511: neighbouring columns one by one 174, kElements 71, kPairs 57, and the aligned 65536 x 512
// 38; gradients of 8192 x 4095 / 4096: kElements 117, kPairs 69, kVec 50.)
enum Mode : int { kElements = 0, kVec = 1, kPairs = 2 };
// `shift`: kPairs, 1 where the row's pairs begin to the left of its first column.  The column may then be -1.
template <int MODE>
__device__ __forceinline__ int first_column(int threads, int t, int i, int shift)
{
    if constexpr (MODE == kVec) return (t + i * threads) * 8;
    else if constexpr (MODE == kPairs) return (i * threads + (t & ~31)) * 8 + 2 * (t & 31) - shift;
    else return (i * threads + (t & ~31)) * 8 + (t & 31);
}
template <int MODE>
__device__ __forceinline__ int column(int c, int j)  // the j-th of the eight that start at c
{
    return MODE == kVec ? c + j : MODE == kPairs ? c + 64 * (j >> 1) + (j & 1) : c + 32 * j;
}
__device__ __forceinline__ bool in_row(int col, int k) { return static_cast<unsigned>(col) < static_cast<unsigned>(k); }
template <int MODE>
__device__ __forceinline__ int row_shift(const void* row) { return MODE == kPairs ? static_cast<int>(reinterpret_cast<uintptr_t>(row) >> 1) & 1 : 0; }
// kPairs: whether all of the warp's pairs are whole; the same for its lanes.
__device__ __forceinline__ bool whole_pairs(int c, int k)
{
    const int warp_first = c - 2 * (threadIdx.x & 31);
    return warp_first >= 0 && warp_first + 256 <= k;
}

// kPairs: which pairs of a row (by their first column) are read as a whole.  The pair that begins at -1 holds the element before the row, the one
// that begins at k - 1 the element behind it: these belong to the neighbouring rows, or to what lies between rows, and are thrown
// away, except before the first row and behind the last, where they would not belong to the tensor.
struct PairRange {
    int first, last;
};
template <int MODE>
__device__ __forceinline__ PairRange pair_range(long long row, int m, int k)
{
    if constexpr (MODE != kPairs) return {0, 0};
    return {row == 0 ? 0 : -1, row == m - 1 ? k - 2 : k - 1};
}

// The eight elements at column c < k; elements outside the row are not touched and read as zero (kPairs: see finish_chunk).
template <typename T, int MODE>
__device__ __forceinline__ void load_chunk(const T* row, int c, int k, const PairRange& range, Raw8<T>& r)
{
    if constexpr (MODE == kVec) {
        r.v = ld_v4(row + c);
        if constexpr (sizeof(T) == 4) r.w = ld_v4(row + c + 4);
    } else if constexpr (MODE == kPairs) {
        uint32_t u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = ld_element<4>(row + c + 64 * j, static_cast<unsigned>(c + 64 * j - range.first) <= static_cast<unsigned>(range.last - range.first) && range.last >= range.first);
        r.v = make_uint4(u[0], u[1], u[2], u[3]);
    } else {
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = ld_element<sizeof(T)>(row + column<MODE>(c, j), in_row(column<MODE>(c, j), k));
        if constexpr (sizeof(T) == 4) {
            r.v = make_uint4(u[0], u[1], u[2], u[3]);
            r.w = make_uint4(u[4], u[5], u[6], u[7]);
        } else {
            r.v = make_uint4(u[0] | (u[1] << 16), u[2] | (u[3] << 16), u[4] | (u[5] << 16), u[6] | (u[7] << 16));
        }
    }
}
// Before the first use of a loaded chunk.  kPairs, where the warp has a pair that the row only half owns: takes the other half out, and fetches the
// element of a pair that was not read.  (Here and not at the load, which would then be waited for.)
template <typename T, int MODE>
__device__ __forceinline__ void finish_chunk(const T* row, int c, int k, const PairRange& range, Raw8<T>& r)
{
    if constexpr (MODE == kPairs) {
        if (whole_pairs(c, k)) return;
        uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
        const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = c + 64 * j;
            if (col == -1) u[j] = range.first == 0 ? (k > 0 ? static_cast<uint32_t>(e[0]) << 16 : 0u) : u[j] & 0xFFFF0000u;
            if (col == k - 1 && col >= 0) u[j] = range.last < col ? static_cast<uint32_t>(e[col]) : u[j] & 0xFFFFu;
        }
        r.v = make_uint4(u[0], u[1], u[2], u[3]);
    }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float2 (&f)[4])
{
    f[0] = make_float2(__uint_as_float(r.v.x), __uint_as_float(r.v.y)), f[1] = make_float2(__uint_as_float(r.v.z), __uint_as_float(r.v.w));
    f[2] = make_float2(__uint_as_float(r.w.x), __uint_as_float(r.w.y)), f[3] = make_float2(__uint_as_float(r.w.z), __uint_as_float(r.w.w));
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float2 (&f)[4])
{
    const __half2* h = reinterpret_cast<const __half2*>(&r.v);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __half22float2(h[j]);
}
__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float2 (&f)[4])
{
    const uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = make_float2(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xFFFF0000u));
}
// One rounding, to the output type; halves saturate at +-65504 like every fp16 output of the library, NaN is kept.
__device__ __forceinline__ uint32_t pack2(float a, float b, __half)
{
    uint32_t v;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(b), "f"(a));
    return v;
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T, int MODE>
__device__ __forceinline__ void store_chunk(T* row, int c, int k, const float2 (&f)[4])
{
    if constexpr (sizeof(T) == 4) {
        if constexpr (MODE == kVec) {
            *reinterpret_cast<float4*>(row + c) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
            *reinterpret_cast<float4*>(row + c + 4) = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (in_row(column<MODE>(c, j), k)) row[column<MODE>(c, j)] = j & 1 ? f[j / 2].y : f[j / 2].x;
        }
    } else {
        const uint4 v = make_uint4(pack2(f[0].x, f[0].y, T()), pack2(f[1].x, f[1].y, T()), pack2(f[2].x, f[2].y, T()), pack2(f[3].x, f[3].y, T()));
        if constexpr (MODE == kVec) {
            *reinterpret_cast<uint4*>(row + c) = v;
        } else {
            const uint32_t u[4] = {v.x, v.y, v.z, v.w};
            if constexpr (MODE == kPairs) {
                if (whole_pairs(c, k)) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(row + c + 64 * j) = u[j];
                    return;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (in_row(column<MODE>(c, j), k)) reinterpret_cast<uint16_t*>(row)[column<MODE>(c, j)] = static_cast<uint16_t>(u[j >> 1] >> (16 * (j & 1)));
        }
    }
}
// gamma: NULL (ones), fp32, or the rows' type.
template <typename T, int MODE>
__device__ __forceinline__ void load_gamma(const void* __restrict__ gamma, int gamma_f32, int c, int k, float2 (&g)[4])
{
    if (!gamma) {
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = both(1.0f);
    } else if (sizeof(T) == 4 || gamma_f32) {
        const float* src = static_cast<const float*>(gamma);
        if constexpr (MODE == kVec) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(src + c)), b = __ldg(reinterpret_cast<const float4*>(src + c) + 1);
            g[0] = make_float2(a.x, a.y), g[1] = make_float2(a.z, a.w), g[2] = make_float2(b.x, b.y), g[3] = make_float2(b.z, b.w);
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = in_row(column<MODE>(c, j), k) ? __ldg(src + column<MODE>(c, j)) : 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) g[j] = make_float2(v[2 * j], v[2 * j + 1]);
        }
    } else {
        Raw8<T> r;
        if constexpr (MODE == kVec) r.v = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(gamma) + c));
        else {
            const uint16_t* src = static_cast<const uint16_t*>(gamma);  // (its pairs need not lie like the rows')
            uint32_t u[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j] = in_row(column<MODE>(c, j), k) ? __ldg(src + column<MODE>(c, j)) : 0u;
            r.v = make_uint4(u[0] | (u[1] << 16), u[2] | (u[3] << 16), u[4] | (u[5] << 16), u[6] | (u[7] << 16));
        }
        unpack8(r, g);
    }
}

__device__ __forceinline__ float max_nan(float a, float b)  // a NaN stays
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float max_abs(float m, float2 v)  // m >= 0
{
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(v.x), "f"(v.y));
    return r;
}
// Largest of a warp's non-negative floats: their bit patterns are in the same order, and a NaN's is above infinity's.
__device__ __forceinline__ float warp_max_abs(float v) { return __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v))); }

// Sum and (of non-negative values) maximum over the threads of a row (TPR at most: a warp, or the block); `red` holds one entry per warp and is not used again before
// the next barrier.
template <int TPR, bool MAX = true>
__device__ __forceinline__ void row_reduce(float& s, float& mx, float2* red)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    if (MAX) mx = warp_max_abs(mx);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;  // a power of two
        const int w = threadIdx.x >> 5, l = threadIdx.x & (W - 1);
        if ((threadIdx.x & 31) == 0) red[w] = make_float2(s, mx);
        __syncthreads();
        const float2 v = l < static_cast<int>(blockDim.x >> 5) ? red[l] : make_float2(0.0f, 0.0f);
        s = v.x;
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
        if (MAX) mx = warp_max_abs(v.y);
    }
}

struct NormArgs {
    const void* x;
    const void* residual;
    const void* gamma;
    void* sum;
    void* y;
    void* q;
    void* scale;
    float* rstd;
    long long ldx, ld_residual, ld_sum, ldy, ldq;
    int m, k;
    int gamma_f32;
    int q_s8;         // 8-bit output: int8, else e4m3
    int scale_mode;   // ASCB200_SCALE_*
    int group_lanes;  // PER_GROUP / MX: lanes (of eight columns) per group, a power of two up to 32
    float eps, inv_k;
};

// Largest magnitude that a code stands for, in units of the scale.
constexpr float kTopS8 = 127.0f, kTopE4M3 = 448.0f;

// scale = amax / top and its reciprocal, each within a unit in the last place.  A scale under the smallest normal number counts as zero:
// its reciprocal would not be finite, and codes times scale are then below 2^-117 anyway.  NaN stays NaN.  An infinite scale (of an infinite gamma,
// or a product beyond fp32) makes e4m3 codes 0 and NaN by y / inf, and int8 codes 0 as where the scale is NaN.
__device__ __forceinline__ void scale_of(float amax, bool s8, float& scale, float& inv)
{
    const float s = amax * (s8 ? 1.0f / kTopS8 : 1.0f / kTopE4M3);
    const bool none = s < 1.1754943508222875e-38f;
    scale = none ? 0.0f : s;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    inv = none ? 0.0f : s8 && s == __builtin_huge_valf() ? __uint_as_float(0x7FC00000u) : r;
}
// MX: the shared exponent floor(log2 amax) - 8 (the exponent of the largest e4m3 power of two), biased by 127; 255 marks a block
// that holds an infinity or a NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(float amax, float& inv)
{
    const uint32_t e = (__float_as_uint(amax) >> 23) & 0xFFu;
    if (e == 255u) {
        inv = __uint_as_float(0x7FC00000u);
        return 255u;
    }
    const uint32_t byte = e > 8u ? e - 8u : 0u;
    inv = __uint_as_float(byte == 0u ? 0x7F000000u : (254u - byte) << 23);  // 2^(127 - byte)
    return byte;
}

__device__ __forceinline__ uint32_t e4m3x2_of(float2 v)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
    return r;
}
// Low bytes of four words.
__device__ __forceinline__ uint32_t pack_bytes(float2 a, float2 b)
{
    const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
}
// Eight codes of y * mul (mul: the reciprocals of the scales).  int8: |y * mul| is at most 127 and a bit, so adding 1.5 * 2^23 in the
// same instruction rounds it once, to the nearest even integer, which is then the sum's low byte in two's complement; values whose
// scale is NaN give 0.
template <int MODE>
__device__ __forceinline__ void store_codes(uint8_t* row, int c, int k, bool s8, const float2 (&y)[4], const float2 (&mul)[4])
{
    uint32_t a, b;
    if (s8) {
        const float2 magic = both(12582912.0f);
        float2 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = fma2(y[j], mul[j], magic);
            if constexpr (MODE == kElements) {  // the eight values may have different scales
                if (mul[j].x != mul[j].x) v[j].x = 0.0f;
                if (mul[j].y != mul[j].y) v[j].y = 0.0f;
            }
        }
        a = pack_bytes(v[0], v[1]), b = pack_bytes(v[2], v[3]);
        if (MODE != kElements && mul[0].x != mul[0].x) a = b = 0u;
    } else {
        a = e4m3x2_of(mul2(y[0], mul[0])) | (e4m3x2_of(mul2(y[1], mul[1])) << 16);
        b = e4m3x2_of(mul2(y[2], mul[2])) | (e4m3x2_of(mul2(y[3], mul[3])) << 16);
    }
    if constexpr (MODE == kVec) {
        *reinterpret_cast<uint2*>(row + c) = make_uint2(a, b);
    } else {
        if constexpr (MODE == kPairs) {
            if (whole_pairs(c, k)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<uint16_t*>(row + c + 64 * j) = static_cast<uint16_t>((j < 2 ? a : b) >> (16 * (j & 1)));
                return;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (in_row(column<MODE>(c, j), k)) row[column<MODE>(c, j)] = static_cast<uint8_t>((j < 4 ? a : b) >> (8 * (j & 3)));
    }
}

// One row per warp (TPR = 32; blocks of 128 threads hold four rows) or per block (of up to TPR threads).  Thread t owns chunks t, t + threads, ...
template <typename T, int TPR, int NCHUNK, int MODE, bool RES>
__global__ void __launch_bounds__(TPR > 32 ? TPR : 128)
rms_norm_kernel(const NormArgs p)
{
    __shared__ float2 red[32];
    grid_dependency_wait();
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x & 31, threads = TPR > 32 ? blockDim.x : 32;
    const long long row = TPR > 32 ? blockIdx.x : blockIdx.x * 4ll + (threadIdx.x >> 5);
    if (row >= p.m) return;  // whole warps; never with a block per row
    const int k = p.k;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const int shift = row_shift<MODE>(x);
    const PairRange range = pair_range<MODE>(row, p.m, k);
    const T* r = RES ? static_cast<const T*>(p.residual) + row * p.ld_residual : nullptr;
    Raw8<T> xr[NCHUNK], rr[RES ? NCHUNK : 1];
#pragma unroll
    for (int i = 0; i < NCHUNK; ++i) {
        const int c = first_column<MODE>(threads, t, i, shift);
        if (c < k) {
            load_chunk<T, MODE>(x, c, k, range, xr[i]);
            if constexpr (RES) load_chunk<T, MODE>(r, c, k, range, rr[i]);
        }
    }
    constexpr bool EARLY = NCHUNK == 1;  // gamma is requested with the row: where few rows leave latency to count
    float2 early[4];
    if constexpr (EARLY) {
        const int c = first_column<MODE>(threads, t, 0, shift);
        if (c < k) load_gamma<T, MODE>(p.gamma, p.gamma_f32, c, k, early);
    }
    float2 hg[NCHUNK][4], ss2 = both(0.0f);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NCHUNK; ++i) {
        const int c = first_column<MODE>(threads, t, i, shift);
        if (c < k) {
            float2 g[4];
            finish_chunk<T, MODE>(x, c, k, range, xr[i]);
            unpack8(xr[i], hg[i]);
            if constexpr (RES) {
                float2 v[4];
                finish_chunk<T, MODE>(r, c, k, range, rr[i]);
                unpack8(rr[i], v);
#pragma unroll
                for (int j = 0; j < 4; ++j) hg[i][j] = add2(hg[i][j], v[j]);
            }
            if (p.sum) store_chunk<T, MODE>(static_cast<T*>(p.sum) + row * p.ld_sum, c, k, hg[i]);
            if constexpr (!EARLY) load_gamma<T, MODE>(p.gamma, p.gamma_f32, c, k, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (EARLY) g[j] = early[j];
                ss2 = fma2(hg[i][j], hg[i][j], ss2);
                hg[i][j] = mul2(hg[i][j], g[j]);
                amax = max_abs(amax, hg[i][j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) hg[i][j] = both(0.0f);
        }
    }
    float ss = ss2.x + ss2.y;
    row_reduce<TPR>(ss, amax, red);
    const float rstd = rsqrtf(fmaf(ss, p.inv_k, p.eps));  // within two units in the last place; correctly rounded division and root took 40 instructions per warp
    if (p.rstd && t == 0) p.rstd[row] = rstd;
    if (p.y) {
        T* y = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i) {
            const int c = first_column<MODE>(threads, t, i, shift);
            if (c < k) {
                float2 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = mul2(hg[i][j], both(rstd));
                store_chunk<T, MODE>(y, c, k, v);
            }
        }
    }
    if (!p.q) return;
    uint8_t* q = static_cast<uint8_t*>(p.q) + row * p.ldq;
    const bool s8 = p.q_s8 != 0;
    if (p.scale_mode == ASCB200_SCALE_PER_TOKEN) {
        float scale, inv;
        scale_of(amax * rstd, s8, scale, inv);
        if (t == 0) static_cast<float*>(p.scale)[row] = scale;
        // y / scale in one product, unless its factor leaves fp32 (rows of |y| under 1e-30)
        float once = rstd * inv;
        if (once > 3.0e38f) {
            once = inv;
#pragma unroll
            for (int i = 0; i < NCHUNK; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) hg[i][j] = mul2(hg[i][j], both(rstd));
        }
        const float2 mul[4] = {both(once), both(once), both(once), both(once)};
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i) {
            const int c = first_column<MODE>(threads, t, i, shift);
            if (c < k) store_codes<MODE>(q, c, k, s8, hg[i], mul);
        }
        return;
    }
    const int lanes = p.group_lanes;
    const int group_bits = 31 - __clz(lanes * 8);  // columns per group: a power of two
    const long long group0 = row * ((k + lanes * 8 - 1) >> group_bits);
    auto scale_group = [&](float g, int col, bool writes) {  // the group's largest magnitude -> its scale, stored, and the reciprocal
        float r;
        if (p.scale_mode == ASCB200_SCALE_MX) {
            const uint32_t byte = mx_scale_byte(g, r);
            if (writes) static_cast<uint8_t*>(p.scale)[group0 + (col >> group_bits)] = static_cast<uint8_t>(byte);
        } else {
            float scale;
            scale_of(g, s8, scale, r);
            if (writes) static_cast<float*>(p.scale)[group0 + (col >> group_bits)] = scale;
        }
        return r;
    };
#pragma unroll
    for (int i = 0; i < NCHUNK; ++i) {
        const int c = first_column<MODE>(threads, t, i, shift);
        float2 y[4], mul[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = mul2(hg[i][j], both(rstd));
        // the whole warp takes part in a group's maximum, columns past the row's end with zeros
        if constexpr (MODE == kVec) {  // a group is `lanes` neighbouring lanes
            float g = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) g = max_abs(g, y[j]);
            for (int o = 1; o < lanes; o <<= 1) g = max_nan(g, __shfl_xor_sync(0xFFFFFFFFu, g, o));
            const float r = scale_group(g, c, (c / 8 & (lanes - 1)) == 0 && c < k);
#pragma unroll
            for (int j = 0; j < 4; ++j) mul[j] = both(r);
        } else if constexpr (MODE == kElements) {  // a group is one, two, four or eight of the warp's 32-column runs
            float g[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = warp_max_abs(fabsf(j & 1 ? y[j / 2].y : y[j / 2].x));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                if (o * 4 >= lanes) break;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (!(j & o)) g[j] = g[j ^ o] = max_nan(g[j], g[j ^ o]);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = scale_group(g[j], c + j * 32, (t & 31) == 0 && (j * 4 & (lanes - 1)) == 0 && c + j * 32 < k);
#pragma unroll
            for (int j = 0; j < 4; ++j) mul[j] = make_float2(g[2 * j], g[2 * j + 1]);
        }
        if (c < k) store_codes<MODE>(q, c, k, s8, y, mul);
    }
}

constexpr int kMaxNormK = 32768;

template <typename T, int MODE, bool RES>
int launch_norm(const NormArgs& p, int sms, cudaStream_t st)
{
    const int chunks = (p.k + (MODE == kPairs) + 7) / 8;  // pairs may begin one column early
#define ASCB200_NORM_WARP(NC) ASCB200_CUDA(launch_pdl(rms_norm_kernel<T, 32, NC, MODE, RES>, static_cast<unsigned>((p.m + 3ll) / 4), 128, 0, st, p))
#define ASCB200_NORM_BLOCK(TPR, NC) ASCB200_CUDA(launch_pdl(rms_norm_kernel<T, TPR, NC, MODE, RES>, p.m, (chunks + 32 * NC - 1) / (32 * NC) * 32, 0, st, p))
    // While all rows fit the machine at once with one chunk per thread: that, so that a row's loads are all in flight (us, bf16 with residual and e4m3
    // codes, rows x k: 1 x 4096 1.6, 300 x 1024 2.3 against 3.4 with four chunks per lane, 1200 x 1024 3.3 against 4.8, 300 x 4096 3.3
    // against 4.1).  More rows: two to four chunks per thread, whose reductions cost less per element (600 x 4096 4.3 against 4.8,
    // 5000 x 4096 24.8 against 30.7, 5000 x 8192 47 against 85).  A block has just the threads that its chunks take (9912 x 9216 without residual
    // 77 -> 55, with 107 -> 99; 9912 x 2100 29 -> 23).
    // Without a residual there are few bytes per instruction, so more chunks per thread pay: four up to 512 chunks (9912 x 4096 28.4 -> 23.6 us, but
    // with residual 44.0 -> 44.7, 9912 x 4095 by pairs 51.8 -> 58.7), six per lane of a warp up to 192 (20000 x 1200 23.0 -> 15.8; with
    // residual 27.2 -> 27.5, by pairs 37.7 -> 57).
    constexpr bool LIGHT = !RES && MODE == kVec;
    if (chunks > 32 && chunks <= 1024 && static_cast<long long>(p.m) * chunks <= 1536ll * sms) {
        if (chunks <= 128) ASCB200_NORM_BLOCK(128, 1);
        else if (chunks <= 256) ASCB200_NORM_BLOCK(256, 1);
        else if (chunks <= 512) ASCB200_NORM_BLOCK(512, 1);
        else ASCB200_NORM_BLOCK(1024, 1);
        return ASCB200_OK;
    }
    if (chunks <= 32) ASCB200_NORM_WARP(1);
    else if (chunks <= 64) ASCB200_NORM_WARP(2);
    else if (chunks <= 128) ASCB200_NORM_WARP(4);
    else if (LIGHT && chunks <= 192) ASCB200_NORM_WARP((LIGHT ? 6 : 4));
    else if (!LIGHT && chunks <= 512) ASCB200_NORM_BLOCK(256, (LIGHT ? 4 : 2));
    else if (chunks <= 1024) ASCB200_NORM_BLOCK(256, 4);
    else if (chunks <= 2048) ASCB200_NORM_BLOCK(512, 4);
    else ASCB200_NORM_BLOCK(1024, 4);
#undef ASCB200_NORM_WARP
#undef ASCB200_NORM_BLOCK
    return ASCB200_OK;
}

bool is_float_type(int dtype) { return dtype == ASCB200_F32 || dtype == ASCB200_F16 || dtype == ASCB200_BF16; }
int float_bytes(int dtype) { return dtype == ASCB200_F32 ? 4 : 2; }

// A matrix of rows `ld` elements apart: 0 stands for packed rows.  Returns false for a leading dimension under the row's length.
bool resolve_ld(int64_t& ld, int k)
{
    if (ld == 0) ld = k;
    return ld >= k;
}
bool element_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
bool rows_aligned(const void* p, int64_t ld, int bytes, int to) { return !p || (aligned_to(p, to) && (ld * bytes) % to == 0); }

// Where elements of `bytes` lie to pairs of them: the parity of the first row's place and of the leading dimension.  kPairs needs the same of
// every tensor, so that their rows' pairs begin at the same column; absent tensors agree with all.
struct PairPlace {
    int first = -1, step = -1;
    bool same = true;
    void add(const void* p, int64_t ld, int bytes)
    {
        if (!p) return;
        const int f = static_cast<int>((reinterpret_cast<uintptr_t>(p) / bytes) & 1), s = static_cast<int>(ld & 1);
        same = same && (first < 0 || (first == f && step == s));
        first = f, step = s;
    }
};
template <typename T, bool RES>
int launch_norm_mode(const NormArgs& p, int mode, int sms, cudaStream_t st)
{
    if (mode == kVec) return launch_norm<T, kVec, RES>(p, sms, st);
    if constexpr (sizeof(T) == 2)
        if (mode == kPairs) return launch_norm<T, kPairs, RES>(p, sms, st);
    return launch_norm<T, kElements, RES>(p, sms, st);
}
template <typename T>
int launch_norm_type(const NormArgs& p, int mode, int sms, cudaStream_t st)
{
    return p.residual ? launch_norm_mode<T, true>(p, mode, sms, st) : launch_norm_mode<T, false>(p, mode, sms, st);
}

int run_rms_norm(const ascb200_rms_norm_desc* desc, cudaStream_t stream)
{
    DeviceState* st = current_state();
    if (!st) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_rms_norm_desc d = *desc;
    if (d.m < 0 || d.k <= 0 || !(d.eps >= 0.0f)) return ASCB200_EINVAL;
    if (!is_float_type(d.dtype)) return ASCB200_EUNSUPPORTED;
    if (d.gamma_dev && d.gamma_dtype != d.dtype && d.gamma_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    if (d.reserved[0] != 0 || d.reserved[1] != 0) return ASCB200_EINVAL;
    if (!resolve_ld(d.ldx, d.k) || !resolve_ld(d.ld_residual, d.k) || !resolve_ld(d.ld_sum, d.k) || !resolve_ld(d.ldy, d.k) || !resolve_ld(d.ldq, d.k)) return ASCB200_EINVAL;
    NormArgs p = {};
    if (d.q_dev) {
        if (d.q_dtype != ASCB200_S8 && d.q_dtype != ASCB200_FP8_E4M3) return ASCB200_EUNSUPPORTED;
        if (!d.scale_dev && d.m > 0) return ASCB200_EINVAL;
        int group = 256;
        if (d.scale_mode == ASCB200_SCALE_PER_TOKEN) {
            if (d.group_size != 0) return ASCB200_EINVAL;
        } else if (d.scale_mode == ASCB200_SCALE_PER_GROUP) {
            group = d.group_size;
            if (group != 32 && group != 64 && group != 128 && group != 256) return ASCB200_EUNSUPPORTED;
        } else if (d.scale_mode == ASCB200_SCALE_MX) {
            if (d.q_dtype != ASCB200_FP8_E4M3) return ASCB200_EUNSUPPORTED;
            if (d.group_size != 0 && d.group_size != 32) return ASCB200_EINVAL;
            group = 32;
        } else {
            return ASCB200_EINVAL;
        }
        p.group_lanes = group / 8;
        if (d.scale_mode != ASCB200_SCALE_MX && !element_aligned(d.scale_dev, 4)) return ASCB200_EALIGN;
    } else {
        if (!d.y_dev && d.m > 0) return ASCB200_EINVAL;  // nothing that depends on the norm would be written
        p.group_lanes = 32;
    }
    if (d.k > kMaxNormK) return ASCB200_ETOOBIG;
    if (d.m == 0) return ASCB200_OK;
    if (!d.x_dev) return ASCB200_EINVAL;
    // in place only row by row, and not two outputs in one
    if (d.sum_dev && d.sum_dev == d.y_dev) return ASCB200_EINVAL;
    auto same_rows = [](const void* out, int64_t ld_out, const void* in, int64_t ld_in) { return !out || out != in || ld_out == ld_in; };
    if (!same_rows(d.sum_dev, d.ld_sum, d.x_dev, d.ldx) || !same_rows(d.sum_dev, d.ld_sum, d.residual_dev, d.ld_residual) || !same_rows(d.y_dev, d.ldy, d.x_dev, d.ldx) ||
        !same_rows(d.y_dev, d.ldy, d.residual_dev, d.ld_residual))
        return ASCB200_EINVAL;
    const int esz = float_bytes(d.dtype), gsz = float_bytes(d.gamma_dtype);
    if (!element_aligned(d.x_dev, esz) || !element_aligned(d.residual_dev, esz) || !element_aligned(d.sum_dev, esz) || !element_aligned(d.y_dev, esz) ||
        (d.gamma_dev && !element_aligned(d.gamma_dev, gsz)) || !element_aligned(d.rstd_dev, 4))
        return ASCB200_EALIGN;
    p.x = d.x_dev, p.residual = d.residual_dev, p.gamma = d.gamma_dev, p.sum = d.sum_dev, p.y = d.y_dev, p.q = d.q_dev, p.scale = d.scale_dev;
    p.rstd = d.rstd_dev;
    p.ldx = d.ldx, p.ld_residual = d.ld_residual, p.ld_sum = d.ld_sum, p.ldy = d.ldy, p.ldq = d.ldq;
    p.m = d.m, p.k = d.k, p.gamma_f32 = d.gamma_dtype == ASCB200_F32, p.q_s8 = d.q_dtype == ASCB200_S8, p.scale_mode = d.scale_mode, p.eps = d.eps, p.inv_k = 1.0f / static_cast<float>(d.k);
    const bool vec = d.k % 8 == 0 && rows_aligned(d.x_dev, d.ldx, esz, 16) && rows_aligned(d.residual_dev, d.ld_residual, esz, 16) &&
                     rows_aligned(d.sum_dev, d.ld_sum, esz, 16) && rows_aligned(d.y_dev, d.ldy, esz, 16) && rows_aligned(d.q_dev, d.ldq, 1, 8) &&
                     (!d.gamma_dev || aligned_to(d.gamma_dev, 16));
    PairPlace pairs;
    pairs.add(d.x_dev, d.ldx, esz), pairs.add(d.residual_dev, d.ld_residual, esz), pairs.add(d.sum_dev, d.ld_sum, esz), pairs.add(d.y_dev, d.ldy, esz);
    pairs.add(d.q_dev, d.ldq, 1);
    // (groups of columns end inside pairs that begin one column early; and the longest rows would take a column more than a block has threads for)
    const int mode = vec ? kVec : esz == 2 && pairs.same && d.k < kMaxNormK && (!d.q_dev || d.scale_mode == ASCB200_SCALE_PER_TOKEN) ? kPairs : kElements;
    const int sms = st->sm_count;
    switch (d.dtype) {
        case ASCB200_F16: return launch_norm_type<__half>(p, mode, sms, stream);
        case ASCB200_BF16: return launch_norm_type<__nv_bfloat16>(p, mode, sms, stream);
        default: return launch_norm_type<float>(p, mode, sms, stream);
    }
}

// ---- gradients -----------------------------------------------------------------------------------------------------------------
struct NormGradArgs {
    const void* dy;
    const void* h;
    const float* rstd;
    const void* gamma;
    const void* dh;
    void* dx;
    float* partial;  // [blocks][k], or nullptr
    void* dgamma;    // a single block writes it itself
    int dgamma_dtype;
    long long ld_dy, ldh, ld_dh, ld_dx;
    int m, k;
    int gamma_f32;
};

// Blocks that have to fit an SM: 64 registers per thread with one chunk of a 16-bit row, else 128.
constexpr int grad_blocks_per_sm(int tpr, int nchunk, int bytes)
{
    return bytes == 4 ? (nchunk == 2 && tpr > 32 && tpr < 512 ? 512 / tpr : 1) : tpr == 32 ? 2 : nchunk == 1 ? 1024 / tpr : 512 / tpr;
}

// The rows to come wait in shared memory: every thread copies its own columns of dy, h and dh there (cp.async: no registers, and no barrier, since
// nobody else reads them) and takes them up STAGES - 1 rows later; STAGES by what an SM has for its blocks.  16-bit rows up to 16384.  With
// two chunks per thread that beats one whose next row waits in registers (us, bf16, m x k: 8192 x 4096 with dh 53.8 -> 49.6, 16384 x 2048 46.1 -> 40.2,
// 30000 x 1024 with dh 54.0 -> 45.7, 9107 x 8192 102 -> 77, 9107 x 12288 197 -> 117, 7000 x 16384 with dh 205 -> 151: 6.1 TB/s; one chunk per
// thread by ring 59 for the first); not where the copies have four bytes, but for long rows (pairs: 6100 x 1427 with dh 21.4 -> 27, 9107 x 9252
// 262 -> 182), and not for fp32 (two stages: 9107 x 4096 88.5 -> 121).
constexpr int kGradRing = 200 * 1024;
constexpr int grad_threads(int tpr) { return tpr > 32 ? tpr : 256; }
constexpr int grad_stage_bytes(int tpr, int nchunk, int bytes) { return grad_threads(tpr) * nchunk * 8 * bytes * 3; }
constexpr int grad_resident(int tpr, int nchunk)  // blocks per SM that the grid is made for
{
    return tpr == 32 ? 4 : nchunk > 1 ? (tpr >= 512 ? 1 : 512 / tpr) : tpr == 128 ? 6 : tpr == 256 ? 4 : 2;
}
constexpr int grad_stages(int tpr, int nchunk, int bytes, int mode)
{
    const int n = kGradRing / (grad_resident(tpr, nchunk) * grad_stage_bytes(tpr, nchunk, bytes));
    return bytes == 4 || mode == kElements || (mode == kPairs && (tpr < 512 || nchunk < 2)) || n < 2 ? 0 : n > 4 ? 4 : n;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool inside)  // zeros where not inside
{
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(inside ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(inside ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_end_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// kPairs: the element whose address a copy of the pair at `col` is given.  A copy that brings nothing is not to leave the row far behind, but needs an
// address on four bytes all the same: pairs start there, so any element of the pair's parity has one, the row itself only where its pairs begin with it.
constexpr int pair_source(int col, bool inside) { return inside ? col : col & 1; }
static_assert(pair_source(-1, false) == 1 && pair_source(63, false) == 1 && pair_source(64, false) == 0 && pair_source(63, true) == 63 && pair_source(-1, true) == -1,
              "a whole number of pairs from the pair's own place");

// One chunk to or from its place: words of 16 bytes (kVec) or four (kPairs), those of the block's threads side by side.
template <typename T, int MODE>
__device__ __forceinline__ void copy_chunk(uint32_t place, const T* row, int c, int k, const PairRange& range, int threads)
{
    constexpr int WORDS = static_cast<int>(sizeof(T)) * 2;  // of four bytes
    if constexpr (MODE == kVec) {
#pragma unroll
        for (int j = 0; j < WORDS / 4; ++j) copy_async<16>(place + (j * threads + threadIdx.x) * 16, row + c + j * 16 / sizeof(T), true);
    } else {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) {
            const int col = c + 64 * j;
            const bool inside = range.last >= range.first && static_cast<unsigned>(col - range.first) <= static_cast<unsigned>(range.last - range.first);
            copy_async<4>(place + (j * threads + threadIdx.x) * 4, row + pair_source(col, inside), inside);
        }
    }
}
template <typename T, int MODE>
__device__ __forceinline__ void take_chunk(const uint8_t* place, int threads, Raw8<T>& r)
{
    constexpr int WORDS = static_cast<int>(sizeof(T)) * 2;
    if constexpr (MODE == kVec) {
        const uint4* at = reinterpret_cast<const uint4*>(place) + threadIdx.x;
        r.v = at[0];
        if constexpr (WORDS == 8) r.w = at[threads];
    } else {
        const uint32_t* at = reinterpret_cast<const uint32_t*>(place) + threadIdx.x;
        r.v = make_uint4(at[0], at[threads], at[2 * threads], at[3 * threads]);
    }
}

// TPR threads per row as above; a block holds ROWS rows at a time (blocks of 256 threads for warp rows).  Up to two chunks per thread keep gamma,
// dy * gamma and hat in registers from the reduction to the output; more chunks unpack dy and h twice (and read gamma twice, without the ring).
template <typename T, int TPR, int NCHUNK, int MODE>
__global__ void __launch_bounds__(grad_threads(TPR), grad_blocks_per_sm(TPR, NCHUNK, sizeof(T)))
rms_norm_grad_kernel(const NormGradArgs p)
{
    constexpr int ROWS = TPR > 32 ? 1 : 8, THREADS = grad_threads(TPR);
    constexpr int STAGES = grad_stages(TPR, NCHUNK, sizeof(T), MODE);
    constexpr bool RING = STAGES > 0;
    constexpr bool AHEAD = !RING && MODE != kElements && NCHUNK * sizeof(T) <= 4;  // the next row is requested before this one is worked on
    constexpr bool KEEP = NCHUNK == 1 || (NCHUNK == 2 && TPR > 32);
    constexpr bool KEEP_GAMMA = KEEP || (RING && TPR > 32);
    constexpr int HELD = KEEP ? NCHUNK : 1;
    constexpr int CHUNK_BYTES = THREADS * 8 * sizeof(T), ARRAY_BYTES = NCHUNK * CHUNK_BYTES, STAGE_BYTES = 3 * ARRAY_BYTES;
    __shared__ float2 red[2][32];
    extern __shared__ uint4 dynamic_smem[];  // the ring: [STAGES][dy, h, dh][NCHUNK][THREADS] chunks; warp rows, at the end: [8][TPR * NCHUNK * 8] sums
    uint8_t* ring = reinterpret_cast<uint8_t*>(dynamic_smem);
    grid_dependency_wait();
    const int t = TPR > 32 ? threadIdx.x : threadIdx.x & 31;
    const int sub = TPR > 32 ? 0 : threadIdx.x >> 5;
    const int k = p.k;
    const float inv_k = __frcp_rn(static_cast<float>(k));
    const long long step = static_cast<long long>(gridDim.x) * ROWS;
    long long row = static_cast<long long>(blockIdx.x) * ROWS + sub;
    const T* dy = static_cast<const T*>(p.dy);
    const T* h = static_cast<const T*>(p.h);
    const T* dh = static_cast<const T*>(p.dh);
    // A thread's columns are the same in all of its rows: kPairs' shift too, since the rows are an even number apart (see grad_blocks).
    const int shift = row_shift<MODE>(dy + row * p.ld_dy);
    float2 acc[NCHUNK][4], gamma[KEEP_GAMMA ? NCHUNK : 1][4], hat[HELD][4], g[HELD][4];
#pragma unroll
    for (int i = 0; i < NCHUNK; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = both(0.0f);
        if constexpr (KEEP_GAMMA) {
            const int c = first_column<MODE>(TPR, t, i, shift);
            if (c < k) load_gamma<T, MODE>(p.gamma, p.gamma_f32, c, k, gamma[i]);
        }
    }
    auto request = [&](long long to_come, int stage) {  // a row into the ring
        if (to_come < p.m) {
            const PairRange range = pair_range<MODE>(to_come, p.m, k);
            const uint32_t place = static_cast<uint32_t>(__cvta_generic_to_shared(ring)) + stage * STAGE_BYTES;
#pragma unroll
            for (int i = 0; i < NCHUNK; ++i) {
                const int c = first_column<MODE>(TPR, t, i, shift);
                if (c < k) {
                    copy_chunk<T, MODE>(place + i * CHUNK_BYTES, dy + to_come * p.ld_dy, c, k, range, THREADS);
                    copy_chunk<T, MODE>(place + ARRAY_BYTES + i * CHUNK_BYTES, h + to_come * p.ldh, c, k, range, THREADS);
                    if (dh) copy_chunk<T, MODE>(place + 2 * ARRAY_BYTES + i * CHUNK_BYTES, dh + to_come * p.ld_dh, c, k, range, THREADS);
                }
            }
        }
        copies_end_group();
    };
    if constexpr (RING) {
#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) request(row + s * step, s);
    }
    float next_rstd = row < p.m ? __ldg(p.rstd + row) : 0.0f;
    int parity = 0, stage = 0;
    constexpr int RAW = RING ? 1 : NCHUNK;
    struct Row {
        Raw8<T> dy[RAW], h[RAW], dh[RAW];
    };
    Row raw, next;
    auto load = [&](long long to_come, Row& to) {
        if (to_come >= p.m) return;
        const PairRange range = pair_range<MODE>(to_come, p.m, k);
#pragma unroll
        for (int i = 0; i < RAW; ++i) {
            const int c = first_column<MODE>(TPR, t, i, shift);
            if (c < k) {
                load_chunk<T, MODE>(dy + to_come * p.ld_dy, c, k, range, to.dy[i]);
                load_chunk<T, MODE>(h + to_come * p.ldh, c, k, range, to.h[i]);
                if (dh) load_chunk<T, MODE>(dh + to_come * p.ld_dh, c, k, range, to.dh[i]);
            }
        }
    };
    if constexpr (AHEAD) load(row, next);
    for (; row < p.m; row += step, parity ^= 1) {
        const PairRange range = pair_range<MODE>(row, p.m, k);
        const float2 rstd = both(next_rstd);
        if (row + step < p.m) next_rstd = __ldg(p.rstd + row + step);
        const uint8_t* place = ring + stage * STAGE_BYTES;
        if constexpr (RING) {
            copies_wait_but<RING ? STAGES - 2 : 0>();
            // the place that the row before has left: its thread has read it for the last time
            request(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        } else if constexpr (AHEAD) {
            raw = next;
            load(row + step, next);
        } else {
            load(row, raw);
        }
        // chunk i of dy (0), h (1) or dh (2)
        auto take = [&](int which, int i, int c, float2 (&f)[4]) {
            Raw8<T>& r = which == 0 ? raw.dy[RING ? 0 : i] : which == 1 ? raw.h[RING ? 0 : i] : raw.dh[RING ? 0 : i];
            if constexpr (RING) take_chunk<T, MODE>(place + which * ARRAY_BYTES + i * CHUNK_BYTES, THREADS, r);
            finish_chunk<T, MODE>(which == 0 ? dy + row * p.ld_dy : which == 1 ? h + row * p.ldh : dh + row * p.ld_dh, c, k, range, r);
            unpack8(r, f);
        };
        float2 dot2 = both(0.0f);
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i) {
            const int c = first_column<MODE>(TPR, t, i, shift);
            const int held = KEEP ? i : 0, gi = KEEP_GAMMA ? i : 0;
            if (c < k) {
                float2 a[4];
                take(0, i, c, a);
                take(1, i, c, hat[held]);
                if constexpr (!KEEP_GAMMA) load_gamma<T, MODE>(p.gamma, p.gamma_f32, c, k, gamma[0]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    hat[held][j] = mul2(hat[held][j], rstd);
                    acc[i][j] = fma2(a[j], hat[held][j], acc[i][j]);
                    g[held][j] = mul2(a[j], gamma[gi][j]);
                    dot2 = fma2(g[held][j], hat[held][j], dot2);
                }
            }
        }
        float dot = dot2.x + dot2.y, none = 0.0f;
        row_reduce<TPR, false>(dot, none, red[parity]);
        const float2 minus_mean = both(-dot * inv_k);
        T* dx = static_cast<T*>(p.dx) + row * p.ld_dx;
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i) {
            const int c = first_column<MODE>(TPR, t, i, shift);
            const int held = KEEP ? i : 0;
            if (c < k) {
                float2 e[4];
                const int gi = KEEP_GAMMA ? i : 0;
                if constexpr (!KEEP) {
                    float2 a[4];
                    take(0, i, c, a);
                    take(1, i, c, hat[held]);
                    if constexpr (!KEEP_GAMMA) load_gamma<T, MODE>(p.gamma, p.gamma_f32, c, k, gamma[0]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) hat[held][j] = mul2(hat[held][j], rstd), g[held][j] = mul2(a[j], gamma[gi][j]);
                }
                if (dh) {
                    take(2, i, c, e);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) e[j] = both(0.0f);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) e[j] = fma2(fma2(hat[held][j], minus_mean, g[held][j]), rstd, e[j]);
                store_chunk<T, MODE>(dx, c, k, e);
            }
        }
    }
    if (!p.partial) return;
    float* out = p.partial + static_cast<size_t>(blockIdx.x) * k;
    auto put = [&](int col, float v) {
        if (gridDim.x > 1) out[col] = v;
        else if (p.dgamma_dtype == ASCB200_F32) static_cast<float*>(p.dgamma)[col] = v;
        else static_cast<T*>(p.dgamma)[col] = rounded<T>(v);
    };
    if constexpr (TPR > 32) {
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int col = column<MODE>(first_column<MODE>(TPR, t, i, shift), j);
                if (in_row(col, k)) put(col, j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x);
            }
    } else {
        constexpr int W = TPR * NCHUNK * 8;
        float* warp_acc = reinterpret_cast<float*>(dynamic_smem);
        if constexpr (RING) copies_wait_but<0>();  // (the last groups are empty)
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NCHUNK; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int col = column<MODE>(first_column<MODE>(TPR, t, i, shift), j);
                if (in_row(col, k)) warp_acc[sub * W + col] = j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x;
            }
        __syncthreads();
        for (int col = threadIdx.x; col < k; col += 256) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < ROWS; ++w) v += warp_acc[w * W + col];
            put(col, v);
        }
    }
}

// Blocks of the gradient kernel, at most: rows of the workspace.  By m and k alone, since a caller asks for the workspace's size without a device: what the
// 148 SMs of a B200 hold at once (see grad_resident).  Measured with half / these / twice as many (us, bf16 with dh): 30000 x 512 25.9 / 28.4 / 34.2, 30000 x
// 1024 61 / 46 / 52, 16384 x 2048 57 / 51 / 59, 8192 x 4096 62 / 50 / 59, 9107 x 8192 134 / 94 / 104, 1000 x 1024 9.3 / 9.5 / 9.6.
int grad_blocks(int m, int k)
{
    const int chunks = (k + 7) / 8;
    const long long most = chunks <= 64 ? 592 : chunks <= 128 ? 888 : chunks <= 256 ? 592 : chunks <= 512 ? 296 : 148;
    const long long rows = chunks <= 64 ? (m + 7ll) / 8 : m;
    const int blocks = static_cast<int>(std::min(most, std::min(rows, std::max(148ll, rows / 4))));  // four rows at a time before a second block per SM
    return blocks > 1 ? blocks & ~1 : blocks;
}

template <typename T, int TPR, int NCHUNK, int MODE>
int launch_norm_grad_as(const NormGradArgs& p, cudaStream_t st, int* blocks)
{
    constexpr int ring = grad_stages(TPR, NCHUNK, sizeof(T), MODE) * grad_stage_bytes(TPR, NCHUNK, sizeof(T)), sums = TPR > 32 ? 0 : 8 * TPR * NCHUNK * 8 * 4;
    constexpr int smem = ring > sums ? ring : sums;
    if constexpr (smem > 46 * 1024) {  // beyond what a launch may take unasked
        static bool configured[16] = {};
        int dev = 0;
        ASCB200_CUDA(cudaGetDevice(&dev));
        if (!configured[dev & 15]) {
            ASCB200_CUDA(cudaFuncSetAttribute(rms_norm_grad_kernel<T, TPR, NCHUNK, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            configured[dev & 15] = true;
        }
    }
    *blocks = grad_blocks(p.m, p.k);
    ASCB200_CUDA(launch_pdl(rms_norm_grad_kernel<T, TPR, NCHUNK, MODE>, *blocks, TPR > 32 ? TPR : 256, smem, st, p));
    return ASCB200_OK;
}
template <typename T, int MODE>
int launch_norm_grad(const NormGradArgs& p, cudaStream_t st, int* blocks)
{
    const int chunks = (p.k + 7) / 8;
    if (chunks <= 32) return launch_norm_grad_as<T, 32, 1, MODE>(p, st, blocks);
    if (chunks <= 64) return launch_norm_grad_as<T, 32, 2, MODE>(p, st, blocks);
    if constexpr (MODE == kElements && sizeof(T) == 4) {
        // Single fp32 elements of many rows: two chunks per thread leave two blocks per SM instead of one (us: 23233 x 2635 228 -> 166, 9107 x 4095 with dh
        // 128 -> 115, 20000 x 2047 109 -> 95; but 1000 x 1111 6.3 -> 8.5, and 9107 x 4096 by 16 bytes 89 -> 95).
        if (p.m >= 4096 && chunks > 128 && chunks <= 256) return launch_norm_grad_as<T, 128, 2, MODE>(p, st, blocks);
        if (p.m >= 4096 && chunks > 256 && chunks <= 512) return launch_norm_grad_as<T, 256, 2, MODE>(p, st, blocks);
    }
    if constexpr (MODE != kVec || sizeof(T) == 4) {
        if (chunks <= 128) return launch_norm_grad_as<T, 128, 1, MODE>(p, st, blocks);
        if (chunks <= 256) return launch_norm_grad_as<T, 256, 1, MODE>(p, st, blocks);
        if (chunks <= 512) return launch_norm_grad_as<T, 512, 1, MODE>(p, st, blocks);
    } else {
        if (chunks <= 128) return launch_norm_grad_as<T, 64, 2, MODE>(p, st, blocks);
        if (chunks <= 256) return launch_norm_grad_as<T, 128, 2, MODE>(p, st, blocks);
        if (chunks <= 512) return launch_norm_grad_as<T, 256, 2, MODE>(p, st, blocks);
    }
    if (chunks <= 1024) return launch_norm_grad_as<T, 512, 2, MODE>(p, st, blocks);
    if (chunks <= 2048) return launch_norm_grad_as<T, 512, 4, MODE>(p, st, blocks);
    return launch_norm_grad_as<T, 1024, 4, MODE>(p, st, blocks);
}

template <typename T>
int launch_norm_grad_mode(const NormGradArgs& p, int mode, cudaStream_t st, int* blocks)
{
    if (mode == kVec) return launch_norm_grad<T, kVec>(p, st, blocks);
    if constexpr (sizeof(T) == 2)
        if (mode == kPairs) return launch_norm_grad<T, kPairs>(p, st, blocks);
    return launch_norm_grad<T, kElements>(p, st, blocks);
}

size_t grad_workspace(int m, int k) { return m <= 0 || k <= 0 ? 0 : static_cast<size_t>(grad_blocks(m, k)) * k * sizeof(float); }

int run_rms_norm_grad(const ascb200_rms_norm_grad_desc* desc, cudaStream_t stream)
{
    if (!current_state()) return ASCB200_ENODEV;
    if (!desc) return ASCB200_EINVAL;
    ascb200_rms_norm_grad_desc d = *desc;
    if (d.m < 0 || d.k <= 0 || d.reserved != 0) return ASCB200_EINVAL;
    if (!is_float_type(d.dtype)) return ASCB200_EUNSUPPORTED;
    if (d.gamma_dev && d.gamma_dtype != d.dtype && d.gamma_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    if (d.dgamma_dev && d.dgamma_dtype != d.dtype && d.dgamma_dtype != ASCB200_F32) return ASCB200_EUNSUPPORTED;
    if (!resolve_ld(d.ld_dy, d.k) || !resolve_ld(d.ldh, d.k) || !resolve_ld(d.ld_dh, d.k) || !resolve_ld(d.ld_dx, d.k)) return ASCB200_EINVAL;
    if (d.k > kMaxNormK) return ASCB200_ETOOBIG;
    const int esz = float_bytes(d.dtype);
    if (d.dgamma_dev && !element_aligned(d.dgamma_dev, float_bytes(d.dgamma_dtype))) return ASCB200_EALIGN;
    if (d.m == 0) {
        if (d.dgamma_dev) ASCB200_CUDA(cudaMemsetAsync(d.dgamma_dev, 0, static_cast<size_t>(d.k) * float_bytes(d.dgamma_dtype), stream));
        return ASCB200_OK;
    }
    if (!d.dy_dev || !d.h_dev || !d.rstd_dev || !d.dx_dev) return ASCB200_EINVAL;
    if ((d.dx_dev == d.dy_dev && d.ld_dx != d.ld_dy) || (d.dx_dev == d.h_dev && d.ld_dx != d.ldh) || (d.dx_dev == d.dh_dev && d.ld_dx != d.ld_dh)) return ASCB200_EINVAL;
    if (!element_aligned(d.dy_dev, esz) || !element_aligned(d.h_dev, esz) || !element_aligned(d.dh_dev, esz) || !element_aligned(d.dx_dev, esz) ||
        !element_aligned(d.rstd_dev, 4) || (d.gamma_dev && !element_aligned(d.gamma_dev, float_bytes(d.gamma_dtype))))
        return ASCB200_EALIGN;
    if (d.dgamma_dev) {
        if (!d.workspace_dev || d.workspace_bytes < grad_workspace(d.m, d.k)) return ASCB200_EINVAL;
        if (!aligned_to(d.workspace_dev, 16)) return ASCB200_EALIGN;
    }
    NormGradArgs p = {};
    p.dy = d.dy_dev, p.h = d.h_dev, p.rstd = d.rstd_dev, p.gamma = d.gamma_dev, p.dh = d.dh_dev, p.dx = d.dx_dev;
    p.partial = d.dgamma_dev ? static_cast<float*>(d.workspace_dev) : nullptr;
    p.ld_dy = d.ld_dy, p.ldh = d.ldh, p.ld_dh = d.ld_dh, p.ld_dx = d.ld_dx, p.m = d.m, p.k = d.k, p.gamma_f32 = d.gamma_dtype == ASCB200_F32;
    const bool vec = d.k % 8 == 0 && rows_aligned(d.dy_dev, d.ld_dy, esz, 16) && rows_aligned(d.h_dev, d.ldh, esz, 16) && rows_aligned(d.dh_dev, d.ld_dh, esz, 16) &&
                     rows_aligned(d.dx_dev, d.ld_dx, esz, 16) && (!d.gamma_dev || aligned_to(d.gamma_dev, 16));
    PairPlace pairs;
    pairs.add(d.dy_dev, d.ld_dy, esz), pairs.add(d.h_dev, d.ldh, esz), pairs.add(d.dh_dev, d.ld_dh, esz), pairs.add(d.dx_dev, d.ld_dx, esz);
    // (k % 8: the early column must not change the number of chunks, by which the blocks are counted)
    const int mode = vec ? kVec : esz == 2 && pairs.same && d.k % 8 != 0 ? kPairs : kElements;
    p.dgamma = d.dgamma_dev, p.dgamma_dtype = d.dgamma_dtype;
    int blocks = 0, rc;
    switch (d.dtype) {
        case ASCB200_F16: rc = launch_norm_grad_mode<__half>(p, mode, stream, &blocks); break;
        case ASCB200_BF16: rc = launch_norm_grad_mode<__nv_bfloat16>(p, mode, stream, &blocks); break;
        default: rc = launch_norm_grad_mode<float>(p, mode, stream, &blocks);
    }
    if (rc != ASCB200_OK || !d.dgamma_dev || blocks == 1) return rc;
    return sum_partials(p.partial, d.dgamma_dev, d.dgamma_dtype, blocks, d.k, stream);
}

}  // namespace
}  // namespace ascb200

extern "C" {

int ascb200_rms_norm(const ascb200_rms_norm_desc* desc, void* stream) { return ascb200::run_rms_norm(desc, static_cast<cudaStream_t>(stream)); }

size_t ascb200_rms_norm_grad_workspace_bytes(int32_t m, int32_t k) { return ascb200::grad_workspace(m, k); }

int ascb200_rms_norm_grad(const ascb200_rms_norm_grad_desc* desc, void* stream)
{
    return ascb200::run_rms_norm_grad(desc, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
