// MX4 rows: quantization, reading back, staging as operand blocks, and the packing of weights.
// All of them are bound by memory; nothing is kept between values but a block's largest magnitude.
#include <algorithm>

#include "rk_kernels_mx4.h"

namespace {

// ---- MX4 rows from values --------------------------------------------------------
// Four lanes per block, eight values each: a wave reads and writes whole lines whatever the type.  The rows' blocks are
// counted through from `first`, so that short rows fill the workgroups, too.
constexpr int QUANT_UNITS = 4; // blocks of a quad of lanes; their loads go out together

// DENSE: the values follow one another, and rows are whole blocks.  (As two branches of one kernel the loads waited for each other:
// 4096 x 14336 bf16 49 us.)
template <int TYPE, bool DENSE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* x, uint8_t* codes, uint8_t* scales, int64_t rows, int K, int64_t ldx) {
    const int KB = (K + 31) / 32, part = threadIdx.x & 3;
    const int64_t blocks = rows * KB, first = (int64_t)blockIdx.x * (64 * QUANT_UNITS);
    const int mine = threadIdx.x >> 2, live = (int)min(blocks - first, (int64_t)(64 * QUANT_UNITS)); // units of this workgroup
    const int64_t row0 = DENSE ? 0 : first / KB;
    const unsigned rest = (unsigned)(first - row0 * KB);
    MxRaw<TYPE> raw[QUANT_UNITS];
#pragma unroll
    for (int u = 0; u < QUANT_UNITS; ++u) {
        const int unit = u * 64 + mine;
        if constexpr (DENSE) {
            // (beyond the end: the last block again, which is not stored)
            raw[u] = mx_fetch8<TYPE>(x, (first + min(unit, live - 1)) * 32 + part * 8);
        } else {
            const unsigned t = rest + min(unit, live - 1), r = t / (unsigned)KB;
            const int k = (int)(t - r * KB) * 32 + part * 8;
            const size_t i = (row0 + r) * ldx + k;
            if (k + 8 <= K) raw[u] = mx_fetch8<TYPE>(x, i);
            else raw[u] = mx_fetch_some<TYPE>(x, i, K - k);
        }
    }
#pragma unroll
    for (int u = 0; u < QUANT_UNITS; ++u) {
        const int unit = u * 64 + mine;
        float v[8];
        mx_unpack<TYPE>(raw[u], v);
        const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(v)));
        if (unit >= live) continue;
        *reinterpret_cast<u32_any*>(codes + (first + unit) * 16 + part * 4) = mx_codes(v, scale);
        if (part == 0) scales[first + unit] = (uint8_t)scale;
    }
}

// ---- and back --------------------------------------------------------------------
__device__ __forceinline__ float mx_value(uint32_t code) { // e2m1: sign, two bits of exponent, one of mantissa
    const uint32_t e = (code >> 1) & 3, m = code & 1;
    const float size = e ? __uint_as_float(((e + 126) << 23) | (m << 22)) : 0.5f * (float)m;
    return code & 8 ? -size : size;
}

// A lane makes 16 bytes of a row, so that a wave stores 1 KiB in a row.  STREAM: with streaming stores, for results that the caches would not
// hold: written the usual way, 32 bytes apart, the 235 MB of 4096 x 14336 fp32 values were still on their way to memory when the next launch read its
// rows (quantization and reading back together 87 -> 68 us; streaming stores of half lines, 16 bytes of every 32: 124).
constexpr size_t STREAM_FROM = (size_t)64 << 20; // a quarter of the memory-side cache

template <int TYPE, bool STREAM>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, void* y, int64_t rows, int K, int64_t ldy) {
    constexpr int V = TYPE == RKH_MX4_F32 ? 4 : 8, LANES = 32 / V; // values of a lane, lanes of a block
    constexpr int PASSES = 64 * QUANT_UNITS * LANES / 256;
    const int KB = (K + 31) / 32, part = threadIdx.x % LANES, mine = threadIdx.x / LANES;
    const int64_t blocks = rows * KB, first = (int64_t)blockIdx.x * (64 * QUANT_UNITS);
    const int live = (int)min(blocks - first, (int64_t)(64 * QUANT_UNITS));
    const bool dense = K % 32 == 0 && (ldy == K || rows == 1);
    const int64_t row0 = dense ? 0 : first / KB;
    const unsigned rest = (unsigned)(first - row0 * KB);
    uint32_t w[PASSES], s[PASSES];
#pragma unroll
    for (int u = 0; u < PASSES; ++u) { // (beyond the end: the last block again, which is not stored)
        const int64_t at = first + min(u * (256 / LANES) + mine, live - 1);
        if constexpr (V == 4) w[u] = *reinterpret_cast<const u16_any*>(codes + at * 16 + part * 2);
        else w[u] = *reinterpret_cast<const u32_any*>(codes + at * 16 + part * 4);
        s[u] = scales[at];
    }
#pragma unroll
    for (int u = 0; u < PASSES; ++u) {
        const int unit = u * (256 / LANES) + mine;
        if (unit >= live) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = s[u] == 255u ? __uint_as_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(mx_value((w[u] >> (4 * e)) & 15u), (int)s[u] - 127);
        size_t i;
        int count = V;
        if (dense) {
            i = (size_t)(first + unit) * 32 + part * V;
        } else {
            const unsigned t = rest + unit, r = t / (unsigned)KB;
            const int k = (int)(t - r * KB) * 32 + part * V;
            i = (row0 + r) * ldy + k;
            count = K - k;
        }
        if (count >= V) {
            using T = typename MxType<TYPE>::T;
            typedef T vec __attribute__((ext_vector_type(V)));
            vec x;
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = (T)v[e];
            v4i_any* to = reinterpret_cast<v4i_any*>(static_cast<uint8_t*>(y) + i * sizeof(T));
            if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(v4i, x), to);
            else *to = __builtin_bit_cast(v4i, x);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e < count) mx_store1<TYPE>(y, i + e, v[e]);
        }
    }
}

// ---- operand blocks from values --------------------------------------------------
// A workgroup makes four pieces of 16 rows x 128 k, which share their scale dwords.  A wave reads 512 values of a row at a time, whole lines, eight per
// lane; codes and scales meet in LDS, from which the pieces are stored as they lie, 1 KiB in a row.  (Read in the operands' order, 16 rows at a time:
// 4096 x 4096 bf16 11.3 - 14.4 us, 2048 x 4096 fp16 5.4; a launch of a few rows is 1.9 - 2.8 us either way.)
template <int TYPE>
__global__ __launch_bounds__(256) void mx4_stage_kernel(const void* x, uint8_t* codes, uint8_t* scales, int rows, int K, int64_t ldx) {
    constexpr int QUARTER = 256 + 16, PIECE = 1024 + 64; // (padded: the 16 blocks of a wave's row fall on different banks)
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * PIECE];
    __shared__ __attribute__((aligned(16))) uint8_t lds_scales[256];
    const int K4 = (int)rkh_mx4_k4(K);
    const int lane = lane_id(), wave = wave_id(), rb = blockIdx.x / K4, k4 = blockIdx.x - rb * K4;
    const int k = k4 * 512 + lane * 8, block = lane >> 2;
    MxRaw<TYPE> raw[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int m = rb * 16 + wave * 4 + c;
        const size_t i = (size_t)m * ldx + k;
        if (m < rows && k + 8 <= K) raw[c] = mx_fetch8<TYPE>(x, i);
        else raw[c] = mx_fetch_some<TYPE>(x, i, m < rows ? K - k : 0);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int r = wave * 4 + c;
        float v[8];
        mx_unpack<TYPE>(raw[c], v);
        const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(v)));
        *reinterpret_cast<uint32_t*>(lds + (block >> 2) * PIECE + (block & 3) * QUARTER + r * 16 + (lane & 3) * 4) = mx_codes(v, scale);
        if ((lane & 3) == 0) lds_scales[(r + 16 * (block & 3)) * 4 + (block >> 2)] = (uint8_t)scale;
    }
    __syncthreads();
    const v4i piece = *reinterpret_cast<const v4i*>(lds + wave * PIECE + (lane >> 4) * QUARTER + (lane & 15) * 16);
    *reinterpret_cast<v4i*>(codes + ((size_t)blockIdx.x * 4 + wave) * 1024 + lane * 16) = piece;
    if (wave == 0) reinterpret_cast<uint32_t*>(scales)[(size_t)blockIdx.x * 64 + lane] = reinterpret_cast<const uint32_t*>(lds_scales)[lane];
}

// ---- weights ---------------------------------------------------------------------
// One thread per 16 bytes of operand blocks, then per scale byte; places without a column, and blocks beyond K, are zero.
__global__ __launch_bounds__(256) void mx4_pack_kernel(const uint8_t* codes, const uint8_t* scales, uint8_t* dst, uint8_t* dst_scales, int K, int N,
                                                       int gate_up, size_t first, size_t pieces, size_t bytes) {
    const int KB = (K + 31) / 32, K4 = (int)rkh_mx4_k4(K);
    const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < pieces) {
        const size_t piece = i >> 6;
        const int lane = (int)(i & 63), rb = (int)(piece / (K4 * 4)), b = (int)(piece - (size_t)rb * K4 * 4) * 4 + (lane >> 4);
        const int n = mx_column(rb * 16 + (lane & 15), N, gate_up);
        v4i w = {0, 0, 0, 0};
        if (n >= 0 && b < KB) w = *reinterpret_cast<const v4i_any*>(codes + ((size_t)n * KB + b) * 16);
        *reinterpret_cast<v4i*>(dst + i * 16) = w;
    }
    if (i < bytes) {
        const size_t group = i >> 8;
        const int lane = (int)(i >> 2) & 63, rb = (int)(group / K4), b = (int)(group - (size_t)rb * K4) * 16 + (int)(i & 3) * 4 + (lane >> 4);
        const int n = mx_column(rb * 16 + (lane & 15), N, gate_up);
        dst_scales[i] = n >= 0 && b < KB ? scales[(size_t)n * KB + b] : 0;
    }
}

} // namespace

extern "C" {

int rkh_mx4_quantize(void* stream, int type, int64_t rows, int K, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales) {
    if (!rows) return RKH_OK;
    const int64_t KB = (K + 31) / 32, most = MX_MOST_GROUPS * 64 * QUANT_UNITS / KB; // rows of a launch
    mx_with_type(type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        const auto kernel = K % 32 == 0 && (ldx == K || rows == 1) ? mx4_quantize_kernel<TYPE, true> : mx4_quantize_kernel<TYPE, false>;
        for (int64_t first = 0; first < rows; first += most) {
            const int64_t some = std::min(most, rows - first), groups = (some * KB + 64 * QUANT_UNITS - 1) / (64 * QUANT_UNITS);
            mark((hipStream_t)stream, "mx4_quantize_kernel");
            hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream,
                               static_cast<const typename MxType<TYPE>::T*>(x) + first * ldx, codes + first * KB * 16, scales + first * KB, some, K, ldx);
        }
    });
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

int rkh_mx4_dequantize(void* stream, int type, int64_t rows, int K, const uint8_t* codes, const uint8_t* scales, void* y, int64_t ldy) {
    if (!rows) return RKH_OK;
    const int64_t KB = (K + 31) / 32, most = MX_MOST_GROUPS * 64 * QUANT_UNITS / KB;
    mx_with_type(type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        using T = typename MxType<TYPE>::T;
        const bool streams = (size_t)rows * K * sizeof(T) > STREAM_FROM;
        const auto kernel = streams ? mx4_dequantize_kernel<TYPE, true> : mx4_dequantize_kernel<TYPE, false>;
        for (int64_t first = 0; first < rows; first += most) {
            const int64_t some = std::min(most, rows - first), groups = (some * KB + 64 * QUANT_UNITS - 1) / (64 * QUANT_UNITS);
            mark((hipStream_t)stream, "mx4_dequantize_kernel");
            hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream, codes + first * KB * 16, scales + first * KB,
                               static_cast<T*>(y) + first * ldy, some, K, ldy);
        }
    });
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

int rkh_mx4_stage(void* stream, int type, int rows, int K, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales) {
    if (!rows) return RKH_OK;
    const int64_t K4 = rkh_mx4_k4(K), most = MX_MOST_GROUPS / K4 * 16;
    mx_with_type(type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        for (int64_t first = 0; first < rows; first += most) {
            const int64_t some = std::min(most, rows - first), groups = (some + 15) / 16 * K4;
            mark((hipStream_t)stream, "mx4_stage_kernel");
            hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_stage_kernel<TYPE>), dim3((unsigned)groups), dim3(256), 0, (hipStream_t)stream,
                               static_cast<const typename MxType<TYPE>::T*>(x) + first * ldx, codes + rkh_mx4_code_bytes(first, K),
                               scales + rkh_mx4_scale_bytes(first, K), (int)some, K, ldx);
        }
    });
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

int rkh_mx4_pack(void* stream, const uint8_t* codes, const uint8_t* scales, int K, int N, int gate_up, uint8_t* dst, uint8_t* dst_scales) {
    const int64_t columns = rkh_mx4_columns(N, gate_up);
    const size_t pieces = rkh_mx4_code_bytes(columns, K) / 16, bytes = rkh_mx4_scale_bytes(columns, K);
    const int64_t groups = (int64_t)((std::max(pieces, bytes) + 255) / 256);
    for (int64_t first = 0; first < groups; first += MX_MOST_GROUPS)
        hipLaunchKernelGGL(mx4_pack_kernel, dim3((unsigned)std::min(MX_MOST_GROUPS, groups - first)), dim3(256), 0, (hipStream_t)stream, codes, scales, dst,
                           dst_scales, K, N, gate_up, (size_t)first * 256, pieces, bytes);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

} // extern "C"
