// The norms around a block: z = rms(branch) * w_b, r' = a r + b gate z, y = rms(r') * w, one row per workgroup.
// Bound by memory: every value is read and written once.  A row lives in registers between its two sums of squares.
#include "rk_kernels_mx4.h"

namespace {

constexpr int NORM_MAX_WAVES = 16;

// Sum over the workgroup, the same in every thread.  The waves' sums are added in order; `part` takes turns between calls.
__device__ __forceinline__ float norm_sum(float x, float* part) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) x += __shfl_xor(x, off);
    const int waves = blockDim.x >> 6;
    if (waves == 1) return x;
    if (lane_id() == 0) part[wave_id()] = x;
    __syncthreads();
    float sum = part[0];
    for (int w = 1; w < waves; ++w) sum += part[w];
    return sum;
}
__device__ __forceinline__ float norm_factor(float sum, int D, float eps) { return 1.0f / sqrtf(sum / (float)D + eps); }

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

// z of eight values of the branch, without the gate
__device__ __forceinline__ void norm_branch(const rkh_block_norm_args& a, int k, int count, float factor, float (&v)[8]) {
    if (!a.branch_weight) return;
    float w[8];
    mx_load8<RKH_MX4_F32>(a.branch_weight, k, count, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * factor * w[e];
}
// r' of eight values, from z and the stream's
__device__ __forceinline__ void norm_join(const rkh_block_norm_args& a, int m, int k, int count, const float (&z)[8], float (&r)[8]) {
    float g[8];
    if (a.gate) norm_load(a.gate_type, a.gate, (size_t)m * a.gate_row_stride + k, count, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float gated = a.gate ? z[e] * g[e] : z[e];
        r[e] = fmaf(a.residual_scale, r[e], a.branch_scale * gated);
    }
}
__device__ __forceinline__ float norm_squares(const float (&v)[8], float sum) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
    return sum;
}
// the normed values to wherever they go
__device__ __forceinline__ void norm_out(const rkh_block_norm_args& a, int m, int k, int count, float factor, float (&r)[8]) {
    if (a.weight) {
        float w[8];
        mx_load8<RKH_MX4_F32>(a.weight, k, count, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = r[e] * factor * w[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] *= factor;
    }
    if (a.y && count > 0) norm_store(a.y_type, a.y, (size_t)m * a.ld_y + k, count, r);
    if (a.q) { // (values beyond D are zeros; a block's four lanes come here together)
        const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(r)));
        const int b = k >> 5;
        if (b * 32 < a.D) {
            *reinterpret_cast<uint32_t*>(a.q + mx_code_at(m, b, (int)rkh_mx4_k4(a.D)) + (k & 31) / 2) = mx_codes(r, scale);
            if ((k & 31) == 0) a.q_scale[mx_scale_at(m, b, (int)rkh_mx4_k4(a.D))] = (uint8_t)scale;
        }
    }
}

// CHUNKS pieces of eight values per thread.
template <int CHUNKS>
__global__ __launch_bounds__(1024) void block_norm_kernel(rkh_block_norm_args a) {
    __shared__ float part[2][NORM_MAX_WAVES];
    const int m = blockIdx.x, t = threadIdx.x, step = blockDim.x * 8;
    float r[CHUNKS][8], z[CHUNKS][8];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
        const int k = c * step + t * 8;
        norm_load(a.stream_type, a.stream, (size_t)m * a.ld_stream + k, a.D - k, r[c]);
        if (a.branch) norm_load(a.branch_type, a.branch, (size_t)m * a.ld_branch + k, a.D - k, z[c]);
    }
    if (a.branch) {
        float factor = 1.0f;
        if (a.branch_weight) {
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) sum = norm_squares(z[c], sum);
            factor = norm_factor(norm_sum(sum, part[0]), a.D, a.eps);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int k = c * step + t * 8;
            norm_branch(a, k, a.D - k, factor, z[c]);
            norm_join(a, m, k, a.D - k, z[c], r[c]);
        }
    }
    if (a.stream_out) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int k = c * step + t * 8;
            if (k < a.D) norm_store(a.stream_type, a.stream_out, (size_t)m * a.ld_stream_out + k, a.D - k, r[c]);
        }
    }
    if (!a.y && !a.q) return;
    float sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) sum = norm_squares(r[c], sum);
    const float factor = norm_factor(norm_sum(sum, part[1]), a.D, a.eps);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) norm_out(a, m, c * step + t * 8, a.D - c * step - t * 8, factor, r[c]);
}

// Rows that do not fit into registers are read up to three times; nothing is written before the last pass, so that the
// stream may be updated in place here, too.
__global__ __launch_bounds__(1024) void block_norm_long_kernel(rkh_block_norm_args a) {
    __shared__ float part[2][NORM_MAX_WAVES];
    const int m = blockIdx.x, step = blockDim.x * 8;
    float branch_factor = 1.0f;
    if (a.branch && a.branch_weight) {
        float sum = 0.0f;
        for (int k = threadIdx.x * 8; k < a.D; k += step) {
            float z[8];
            norm_load(a.branch_type, a.branch, (size_t)m * a.ld_branch + k, a.D - k, z);
            sum = norm_squares(z, sum);
        }
        branch_factor = norm_factor(norm_sum(sum, part[0]), a.D, a.eps);
    }
    const auto joined = [&](int k, float (&r)[8]) {
        norm_load(a.stream_type, a.stream, (size_t)m * a.ld_stream + k, a.D - k, r);
        if (a.branch) {
            float z[8];
            norm_load(a.branch_type, a.branch, (size_t)m * a.ld_branch + k, a.D - k, z);
            norm_branch(a, k, a.D - k, branch_factor, z);
            norm_join(a, m, k, a.D - k, z, r);
        }
    };
    float factor = 1.0f;
    if (a.y || a.q) {
        float sum = 0.0f;
        for (int k = threadIdx.x * 8; k < a.D; k += step) {
            float r[8];
            joined(k, r);
            sum = norm_squares(r, sum);
        }
        factor = norm_factor(norm_sum(sum, part[1]), a.D, a.eps);
    }
    for (int k = threadIdx.x * 8; k < rkh_align_up(a.D, 32); k += step) { // (whole blocks: their lanes stay together)
        float r[8];
        joined(k, r);
        if (a.stream_out && k < a.D) norm_store(a.stream_type, a.stream_out, (size_t)m * a.ld_stream_out + k, a.D - k, r);
        if (a.y || a.q) norm_out(a, m, k, a.D - k, factor, r);
    }
}

} // namespace

extern "C" int rkh_block_norm(void* stream, const rkh_block_norm_args* args) {
    const rkh_block_norm_args& a = *args;
    if (!a.rows) return RKH_OK;
    const int64_t pieces = rkh_align_up(a.D, 32) / 8; // of eight values
    // two pieces per thread once a row fills four waves
    const int chunks = pieces <= 256 ? 1 : 2;
    int threads = (int)rkh_align_up((pieces + chunks - 1) / chunks, 64);
    mark((hipStream_t)stream, "block_norm_kernel");
    if (threads > 1024) hipLaunchKernelGGL(block_norm_long_kernel, dim3(a.rows), dim3(1024), 0, (hipStream_t)stream, a);
    else if (chunks == 1) hipLaunchKernelGGL(block_norm_kernel<1>, dim3(a.rows), dim3(threads), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL(block_norm_kernel<2>, dim3(a.rows), dim3(threads), 0, (hipStream_t)stream, a);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}
