// The norms around a block: z = rms(branch) * w_b, r' = a r + b gate z, y = rms(r') * w, one row per workgroup.
// Bound by memory for many rows (4096 x 4096, fp32 stream, bf16 branch, gate and y: 55 us, 235 MB at 4.3 TB/s), by the round trips of one
// workgroup for few: everything that a row needs is loaded at once, weights and gate included, and the row lives in registers between its two
// sums of squares (one row of 4096: 4.4 us, with weights and gate loaded where they are used 5.4).
#include <algorithm>

#include "rk_kernels_mx4.h"

namespace {

constexpr int NORM_MAX_THREADS = 1024;
constexpr int NORM_SEGMENTS = 2 * NORM_MAX_THREADS / 64; // of 512 values, that registers hold

__device__ __forceinline__ void norm_load(int type, const void* p, size_t i, int count, float (&v)[8]) {
    mx_with_type(type, [&](auto t) { mx_load8<decltype(t)::value>(p, i, count, v); });
}
__device__ __forceinline__ void norm_store(int type, void* p, size_t i, int count, const float (&v)[8]) {
    mx_with_type(type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        if (count >= 8) {
            mx_store<TYPE, 8>(p, i, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < count) mx_store1<TYPE>(p, i + e, v[e]);
        }
    });
}

// r' of eight values, from z and the stream's
__device__ __forceinline__ void norm_join(const rkh_block_norm_args& a, const float (&z)[8], const float (&gate)[8], float (&r)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = fmaf(a.residual_scale, r[e], a.branch_scale * (a.gate ? z[e] * gate[e] : z[e]));
}
// the normed values to wherever they go
__device__ __forceinline__ void norm_out(const rkh_block_norm_args& a, int m, int k, const float (&r)[8]) {
    const int count = a.D - k;
    if (a.y && count > 0) norm_store(a.y_type, a.y, (size_t)m * a.ld_y + k, count, r);
    if (a.q) { // (values beyond D are zeros; a block's four lanes come here together)
        const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(r)));
        const int b = k >> 5, K4 = (int)rkh_mx4_k4(a.D);
        if (b * 32 < a.D) {
            *reinterpret_cast<uint32_t*>(a.q + mx_code_at(m, b, K4) + (k & 31) / 2) = mx_codes(r, scale);
            if ((k & 31) == 0) a.q_scale[mx_scale_at(m, b, K4)] = (uint8_t)scale;
        }
    }
}

// CHUNKS pieces of eight values per thread.
template <int CHUNKS>
__global__ __launch_bounds__(NORM_MAX_THREADS) void block_norm_kernel(rkh_block_norm_args a) {
    __shared__ float part[2][NORM_SEGMENTS];
    const int m = a.first + (int)blockIdx.x, waves = blockDim.x >> 6, segments = (a.D + 511) / 512;
    float r[CHUNKS][8], z[CHUNKS][8], gate[CHUNKS][8], wb[CHUNKS][8], w[CHUNKS][8];
    const auto at = [&](int c) { return (c * (int)blockDim.x + (int)threadIdx.x) * 8; };
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int k = at(c), count = a.D - k;
        norm_load(a.stream_type, a.stream, (size_t)m * a.ld_stream + k, count, r[c]);
        if (a.branch) norm_load(a.branch_type, a.branch, (size_t)m * a.ld_branch + k, count, z[c]);
        if (a.gate) norm_load(a.gate_type, a.gate, (size_t)m * a.gate_row_stride + k, count, gate[c]);
        if (a.branch_weight) mx_load8<RKH_MX4_F32>(a.branch_weight, k, count, wb[c]);
        if (a.weight) mx_load8<RKH_MX4_F32>(a.weight, k, count, w[c]);
    }
    // the factor of the values' norm: one part per segment, chunk c of wave v holds segment c * waves + v
    const auto factor_of = [&](const float (&v)[CHUNKS][8], float* sums) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const float sum = mx_segment_sum(mx_squares(v[c], 0.0f));
            if (lane_id() == 0) sums[c * waves + wave_id()] = sum;
        }
        __syncthreads();
        return mx_norm_factor(mx_sum_of_segments(sums, segments), a.D, a.eps);
    };
    if (a.branch) {
        if (a.branch_weight) {
            const float factor = factor_of(z, part[0]);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) mx_normed(z[c], factor, true, wb[c]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) norm_join(a, z[c], gate[c], r[c]);
    }
    if (a.stream_out) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (at(c) < a.D) norm_store(a.stream_type, a.stream_out, (size_t)m * a.ld_stream_out + at(c), a.D - at(c), r[c]);
    }
    if (!a.y && !a.q) return;
    const float factor = factor_of(r, part[1]);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        mx_normed(r[c], factor, a.weight != nullptr, w[c]);
        norm_out(a, m, at(c), r[c]);
    }
}

// Rows that do not fit into registers are read up to three times; nothing is written before the last pass, so that the
// stream may be updated in place here, too.
__global__ __launch_bounds__(NORM_MAX_THREADS) void block_norm_long_kernel(rkh_block_norm_args a) {
    extern __shared__ float parts[]; // one per segment
    const int m = a.first + (int)blockIdx.x, step = blockDim.x * 8, segments = (a.D + 511) / 512;
    const auto factor_of = [&](auto&& values) {
        __syncthreads(); // (the parts are read no more)
        for (int k = threadIdx.x * 8; k < segments * 512; k += step) {
            float v[8];
            values(k, v);
            const float sum = mx_segment_sum(mx_squares(v, 0.0f));
            if (lane_id() == 0) parts[k >> 9] = sum;
        }
        __syncthreads();
        return mx_norm_factor(mx_sum_of_segments(parts, segments), a.D, a.eps);
    };
    const auto branch = [&](int k, float (&z)[8]) { norm_load(a.branch_type, a.branch, (size_t)m * a.ld_branch + k, a.D - k, z); };
    const float branch_factor = a.branch && a.branch_weight ? factor_of(branch) : 1.0f;
    const auto joined = [&](int k, float (&r)[8]) {
        norm_load(a.stream_type, a.stream, (size_t)m * a.ld_stream + k, a.D - k, r);
        if (!a.branch) return;
        float z[8], w[8], gate[8];
        branch(k, z);
        if (a.branch_weight) {
            mx_load8<RKH_MX4_F32>(a.branch_weight, k, a.D - k, w);
            mx_normed(z, branch_factor, true, w);
        }
        if (a.gate) norm_load(a.gate_type, a.gate, (size_t)m * a.gate_row_stride + k, a.D - k, gate);
        norm_join(a, z, gate, r);
    };
    const float factor = a.y || a.q ? factor_of(joined) : 1.0f;
    for (int k = threadIdx.x * 8; k < rkh_align_up(a.D, 32); k += step) { // (whole blocks: their lanes stay together)
        float r[8], w[8];
        joined(k, r);
        if (a.stream_out && k < a.D) norm_store(a.stream_type, a.stream_out, (size_t)m * a.ld_stream_out + k, a.D - k, r);
        if (!a.y && !a.q) continue;
        if (a.weight) mx_load8<RKH_MX4_F32>(a.weight, k, a.D - k, w);
        mx_normed(r, factor, a.weight != nullptr, w);
        norm_out(a, m, k, r);
    }
}

} // namespace

extern "C" int rkh_block_norm(void* stream, const rkh_block_norm_args* args) {
    rkh_block_norm_args a = *args;
    const int64_t segments = (a.D + 511) / 512; // a wave's pieces
    const int chunks = segments <= NORM_MAX_THREADS / 64 ? 1 : 2;
    const bool in_registers = segments <= NORM_SEGMENTS;
    const int64_t threads = in_registers ? (segments + chunks - 1) / chunks * 64 : NORM_MAX_THREADS;
    // a launch holds fewer than 2^32 threads: more rows take several
    const int64_t most = (INT64_C(1) << 31) / threads;
    for (int64_t first = 0; first < args->rows; first += most) {
        a.first = (int)first;
        const dim3 rows((unsigned)std::min<int64_t>(most, args->rows - first));
        mark((hipStream_t)stream, "block_norm_kernel");
        if (!in_registers) // (one float per segment: 16 KiB for the longest rows there are)
            hipLaunchKernelGGL(block_norm_long_kernel, rows, dim3((unsigned)threads), (size_t)segments * 4, (hipStream_t)stream, a);
        else if (chunks == 1)
            hipLaunchKernelGGL(block_norm_kernel<1>, rows, dim3((unsigned)threads), 0, (hipStream_t)stream, a);
        else
            hipLaunchKernelGGL(block_norm_kernel<2>, rows, dim3((unsigned)threads), 0, (hipStream_t)stream, a);
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}
