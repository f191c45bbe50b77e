// What the kernels of group-scaled 4-bit (G4) layers share: codes to operands, scales, and stores of results.
#ifndef RK_KERNELS_G4_H
#define RK_KERNELS_G4_H

#include "rk_g4_shim.h"
#include "rk_kernels_mx4.h"

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));

namespace rkk {
// rk_kernels_g4_tile*.hip, by internal groups in a piece (compiling all of them in one unit takes minutes)
struct G4Route { // tiles of 32 rm rows x 128 places
    int rm, parts, mblocks, nblocks;
};
int launch_g4_tiles1(hipStream_t st, const rkh_g4_args& g, const G4Route& r);
int launch_g4_tiles2(hipStream_t st, const rkh_g4_args& g, const G4Route& r);
int launch_g4_tiles4(hipStream_t st, const rkh_g4_args& g, const G4Route& r);
} // namespace rkk

namespace {

// The scale of a scale dword.
__device__ __forceinline__ float g4_scale(uint32_t d, int type) {
    return type == RKH_MX4_BF16 ? __uint_as_float(d & 0xffff0000u) : (float)__builtin_bit_cast(_Float16, (uint16_t)(d >> 16));
}

// code - zero as halves, exactly.  A code under the exponent of 1024 is the half 1024 + code, four bits further up 1024 + 16 code (a known way from
// integers to floating point): one addition, or one multiplication and addition, of neighbours in a dword.  9 instructions for eight weights.
struct G4Zero {
    v2h low, high; // -(1024 + zero), -(64 + zero)
    __device__ __forceinline__ void of(uint32_t scale_dword) {
        const uint32_t one = (scale_dword & 0xffffu) | 0x8000u;
        low = __builtin_bit_cast(v2h, one | one << 16);
        high = low + v2h{960, 960};
    }
};
// The exponents, in a vector register: as a constant they would be a literal, and masking and joining two instructions.
__device__ __forceinline__ uint32_t g4_exponents() {
    uint32_t v;
    asm("v_mov_b32 %0, 0x64006400" : "=v"(v));
    return v;
}
// The eight weights of a dword, in their order.
__device__ __forceinline__ v4i g4_halves(uint32_t w, const G4Zero& zero, uint32_t exponents) {
    const auto low = [&](uint32_t u) { return __builtin_bit_cast(int, __builtin_bit_cast(v2h, (u & 0x000f000fu) | exponents) + zero.low); };
    const auto high = [&](uint32_t u) {
        const v2h sixteenth = {0.0625f, 0.0625f};
        return __builtin_bit_cast(int, __builtin_elementwise_fma(__builtin_bit_cast(v2h, (u & 0x00f000f0u) | exponents), sixteenth, zero.high));
    };
    return v4i{low(w), high(w), low(w >> 8), high(w >> 8)};
}
// Codes as bf16, the zero point not taken off: a byte 0..15 is the e4m3 number code * 2^-9, which the conversion scales by 2^9.  7 instructions for
// eight.  The order is k0 k4 k1 k5 k2 k6 k3 k7; g4_turned_rows gives activations the same.
__device__ __forceinline__ v4i g4_codes(uint32_t w) {
    const int even = (int)(w & 0x0f0f0f0fu), odd = (int)((w >> 4) & 0x0f0f0f0fu);
    return v4i{__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(even, 512.0f, true)),
               __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, false)), __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(odd, 512.0f, true))};
}
__device__ __forceinline__ v4i g4_turned_rows(const v4i& x) {
    return v4i{(int)__builtin_amdgcn_perm((uint32_t)x.z, (uint32_t)x.x, 0x05040100u), (int)__builtin_amdgcn_perm((uint32_t)x.z, (uint32_t)x.x, 0x07060302u),
               (int)__builtin_amdgcn_perm((uint32_t)x.w, (uint32_t)x.y, 0x05040100u), (int)__builtin_amdgcn_perm((uint32_t)x.w, (uint32_t)x.y, 0x07060302u)};
}

// Column of place 16 block + c of a matrix, in SwiGLU's case that of the half j = block & 1.
__host__ __device__ __forceinline__ int64_t g4_column(int64_t block, int c, bool gate_up) {
    const int64_t unit = block >> 2;
    const int b = (int)(block >> 1) & 1, j = (int)block & 1;
    return gate_up ? unit * 32 + 16 * b + c : unit * 64 + 32 * b + 2 * c + j;
}

// The result of row m and column n.
__device__ __forceinline__ void g4_put(const rkh_g4_args& g, int m, int64_t n, float v) {
    if (n >= g.N) return;
    mx_with_type(g.out_type, [&](auto t) { mx_store1<decltype(t)::value>(g.C, (size_t)m * g.ldc + n, v); });
}

} // namespace

#endif // RK_KERNELS_G4_H
