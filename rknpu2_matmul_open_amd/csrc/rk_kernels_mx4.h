// What the MX4 kernels share: loads and stores of eight values of any type, the block's scale and its codes.
#ifndef RK_KERNELS_MX4_H
#define RK_KERNELS_MX4_H

#include "rk_kernels_common.h"
#include "rk_mx4_shim.h"

typedef int v8i __attribute__((ext_vector_type(8)));

namespace {

// 16 bytes at any address: the memory path takes them in one access whatever their alignment.
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));
typedef int v2i_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint16_t u16_any __attribute__((aligned(1)));

// A launch holds fewer than 2^32 threads: of more, all but what is left modulo 2^32 never run, without an error.  Longer ones are cut into
// pieces of so many workgroups of 256.
constexpr int64_t MX_TOO_MANY_THREADS = INT64_C(1) << 32, MX_MOST_GROUPS = MX_TOO_MANY_THREADS / 2 / 256;

template <int TYPE> struct MxType;
template <> struct MxType<RKH_MX4_F32> { using T = float; };
template <> struct MxType<RKH_MX4_F16> { using T = _Float16; };
template <> struct MxType<RKH_MX4_BF16> { using T = __bf16; };

// Calls f with the tag of a run-time type.
template <class F> __host__ __device__ __forceinline__ void mx_with_type(int type, F&& f) {
    if (type == RKH_MX4_F32) f(std::integral_constant<int, RKH_MX4_F32>{});
    else if (type == RKH_MX4_F16) f(std::integral_constant<int, RKH_MX4_F16>{});
    else f(std::integral_constant<int, RKH_MX4_BF16>{});
}

template <int TYPE> __device__ __forceinline__ float mx_load1(const void* p, size_t i) {
    return (float)static_cast<const typename MxType<TYPE>::T*>(p)[i];
}
template <int TYPE> __device__ __forceinline__ void mx_store1(void* p, size_t i, float v) {
    static_cast<typename MxType<TYPE>::T*>(p)[i] = (typename MxType<TYPE>::T)v;
}

// Eight values as they lie in memory, so that a caller can put other loads between fetching and converting them.
template <int TYPE> struct MxRaw { v4i w[TYPE == RKH_MX4_F32 ? 2 : 1]; };
template <int TYPE> __device__ __forceinline__ MxRaw<TYPE> mx_fetch8(const void* p, size_t i) {
    MxRaw<TYPE> r;
    const uint8_t* at = static_cast<const uint8_t*>(p) + i * sizeof(typename MxType<TYPE>::T);
    r.w[0] = *reinterpret_cast<const v4i_any*>(at);
    if constexpr (TYPE == RKH_MX4_F32) r.w[1] = *reinterpret_cast<const v4i_any*>(at + 16);
    return r;
}
// ... of which only `count` exist; the others read as zero.
template <int TYPE> __device__ __forceinline__ MxRaw<TYPE> mx_fetch_some(const void* p, size_t i, int count) {
    using T = typename MxType<TYPE>::T;
    typedef T v8 __attribute__((ext_vector_type(8)));
    v8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? static_cast<const T*>(p)[i + e] : (T)0.0f;
    return __builtin_bit_cast(MxRaw<TYPE>, v);
}
template <int TYPE> __device__ __forceinline__ void mx_unpack(const MxRaw<TYPE>& r, float (&v)[8]) {
    typedef typename MxType<TYPE>::T v8 __attribute__((ext_vector_type(8)));
    const v8 x = __builtin_bit_cast(v8, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
}
template <int TYPE> __device__ __forceinline__ void mx_load8(const void* p, size_t i, int count, float (&v)[8]) {
    if (count >= 8) mx_unpack<TYPE>(mx_fetch8<TYPE>(p, i), v);
    else mx_unpack<TYPE>(mx_fetch_some<TYPE>(p, i, count), v);
}
// N (4 or 8) values to consecutive places, one rounding to nearest.
template <int TYPE, int N> __device__ __forceinline__ void mx_store(void* p, size_t i, const float* v) {
    using T = typename MxType<TYPE>::T;
    typedef T vec __attribute__((ext_vector_type(N)));
    vec x;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = (T)v[e];
    uint8_t* at = static_cast<uint8_t*>(p) + i * sizeof(T);
    if constexpr (sizeof(x) == 8) {
        *reinterpret_cast<v2i_any*>(at) = __builtin_bit_cast(v2i, x);
    } else if constexpr (sizeof(x) == 16) {
        *reinterpret_cast<v4i_any*>(at) = __builtin_bit_cast(v4i, x);
    } else {
        struct Two { v4i a, b; };
        const Two t = __builtin_bit_cast(Two, x);
        *reinterpret_cast<v4i_any*>(at) = t.a;
        *reinterpret_cast<v4i_any*>(at + 16) = t.b;
    }
}

// The scale byte of a block whose largest magnitude has the bits `top`: 2^(floor(log2 largest) - 2) with a bias of 127, so that
// the largest value becomes 4 .. 8 times the scale (and saturates at 6); no smaller than 2^-127, which zeros take too.
// A block with an Inf or a NaN is NaN as a whole.
__device__ __forceinline__ uint32_t mx_scale(uint32_t top) {
    const int e = (int)(top >> 23);
    return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// What its values are multiplied with ahead of the conversion: the scale's reciprocal, a power of two and therefore exact (only
// values that become zero anyway can lose bits); 0 for NaN blocks, whose codes then need mx_codes(.., true).
__device__ __forceinline__ float mx_factor(uint32_t scale) { return __uint_as_float((254u - min(scale, 254u)) << 23); }

__device__ __forceinline__ uint32_t mx_top(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
    return top;
}
// Eight codes: nearest e2m1 value, ties to an even code, saturating (v_cvt_scalef32_pk_fp4_f32 with a scale of one).
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], uint32_t scale) {
    const float f = mx_factor(scale);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * f, v[1] * f, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * f, v[3] * f, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * f, v[5] * f, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * f, v[7] * f, 1.0f, 3);
    return scale == 255u ? 0u : w;
}

// Largest of a block's maxima over the four lanes that hold eight values each.
__device__ __forceinline__ uint32_t mx_top_of_quad(uint32_t top) {
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true)); // lanes 1 0 3 2
    return max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true)); // lanes 2 3 0 1
}

// ---- norms.  The sum of squares of a row has one order wherever it is made: eight values of a lane one after the other, 64 lanes
// as a butterfly -- a segment of 512 values --, segments one after the other.
__device__ __forceinline__ float mx_squares(const float (&v)[8], float sum) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
    return sum;
}
__device__ __forceinline__ float mx_segment_sum(float x) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off);
    return x;
}
__device__ __forceinline__ float mx_sum_of_segments(const float* part, int segments) {
    float sum = part[0];
    for (int s = 1; s < segments; ++s) sum += part[s];
    return sum;
}
__device__ __forceinline__ float mx_norm_factor(float sum, int D, float eps) { return 1.0f / sqrtf(sum / (float)D + eps); }
__device__ __forceinline__ void mx_normed(float (&v)[8], float factor, bool weighted, const float (&weight)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = weighted ? v[e] * factor * weight[e] : v[e] * factor;
}

// Byte offsets of block b of row m in operand blocks.
__device__ __forceinline__ size_t mx_code_at(int m, int b, int K4) {
    return ((size_t)(m >> 4) * K4 * 4 + (b >> 2)) * 1024 + (m & 15) * 16 + (b & 3) * 256;
}
__device__ __forceinline__ size_t mx_scale_at(int m, int b, int K4) {
    return ((size_t)(m >> 4) * K4 + (b >> 4)) * 256 + (m & 15) * 4 + (b & 3) * 64 + ((b >> 2) & 3);
}

// Logical column of place p of a weight matrix of N columns (2F: gate / up pairs), or -1: padding.
__device__ __forceinline__ int mx_column(int p, int N, int gate_up) {
    const int in32 = p & 31, col = 8 * ((in32 >> 2) & 3) + 4 * (in32 >> 4) + (in32 & 3);
    if (!gate_up) return (p & ~31) + col < N ? (p & ~31) + col : -1;
    const int F = N / 2, n = (p >> 6) * 32 + col;
    return n < F ? n + (p & 32 ? F : 0) : -1;
}

} // namespace

#endif // RK_KERNELS_MX4_H
