// Products of MX4 operands (v_mfma_scale_f32_16x16x128_f8f6f4, fp32 sums): mx4_few_kernel for decode-sized M, bound by the
// weights' bytes; mx4_tile_kernel for more rows, bound by the matrix pipes; mx4_join_kernel, the sum of partial tiles.
//
// The weights are the FIRST operand: lane (r, q) = (l % 16, l / 16) of a 16 x 16 accumulator owns activation row r and four of the
// tile's weight rows, which the packing has made the consecutive columns 8 q + 4 h .. + 3 of a block of 32 (h: the first or the
// second tile of the block).
#ifndef RK_KERNELS_MX4_GEMM_H
#define RK_KERNELS_MX4_GEMM_H

#include <algorithm>

#include "rk_kernels_mx4.h"

namespace rkk {
// rk_kernels_mx4_swiglu.hip, which holds the kernels of gate / up weights (compiling all of them in one unit takes over two minutes)
int launch_mx4_swiglu(hipStream_t st, const rkh_mx4_gemm_args& g);
} // namespace rkk

namespace {

typedef __attribute__((address_space(3))) uint8_t* mx_lds_ptr;

// sum += W * A over 128 k; the scales are byte STEP of the lanes' dwords.
template <int STEP> __device__ __forceinline__ v4f mx_mfma(const v4i& w, const v4i& a, const v4f& sum, uint32_t ws, uint32_t as) {
    const v8i w8 = {w.x, w.y, w.z, w.w, 0, 0, 0, 0}, a8 = {a.x, a.y, a.z, a.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, sum, 4, 4, STEP, (int)ws, STEP, (int)as);
}

// The same as an asm statement, for the tiles: the sums stay in one place (of products that it knows the compiler moved 256 sums
// between registers and spilled others).  What the compiler then does not order: a vector instruction that writes an operand has
// to be two wait states ahead of the product -- here LDS reads alone write them --, and one that reads a sum waits for the last
// products, at the end of the loop.
// ACC: the sum is in the accumulation half of the registers.  (256 of them take all of it; with none to spare the compiler kept
// some on the move, so a few live in the other half.)
template <int STEP, bool ACC> __device__ __forceinline__ void mx_mfma_in_place(const v4i& w, const v4i& a, v4f& sum, uint32_t ws, uint32_t as) {
    if constexpr (ACC)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%c5,%c5,0] op_sel_hi:[%c6,%c6,0] cbsz:4 blgp:4"
                     : "+a"(sum) : "v"(w), "v"(a), "v"(ws), "v"(as), "n"(STEP & 1), "n"(STEP >> 1));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%c5,%c5,0] op_sel_hi:[%c6,%c6,0] cbsz:4 blgp:4"
                     : "+v"(sum) : "v"(w), "v"(a), "v"(ws), "v"(as), "n"(STEP & 1), "n"(STEP >> 1));
}
// ... of which there is no sum yet
template <int STEP, bool ACC> __device__ __forceinline__ void mx_mfma_first(const v4i& w, const v4i& a, v4f& sum, uint32_t ws, uint32_t as) {
    if constexpr (ACC)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel:[%c5,%c5,0] op_sel_hi:[%c6,%c6,0] cbsz:4 blgp:4"
                     : "=&a"(sum) : "v"(w), "v"(a), "v"(ws), "v"(as), "n"(STEP & 1), "n"(STEP >> 1));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel:[%c5,%c5,0] op_sel_hi:[%c6,%c6,0] cbsz:4 blgp:4"
                     : "=&v"(sum) : "v"(w), "v"(a), "v"(ws), "v"(as), "n"(STEP & 1), "n"(STEP >> 1));
}
// The sum as it is at this point, where it is: what keeps the compiler from fetching all sums ahead of the first one's store, and
// from putting anything but products between two of them.
template <bool ACC> __device__ __forceinline__ void mx_settled(v4f& sum) {
    if constexpr (ACC) asm volatile("" : "+a"(sum));
    else asm volatile("" : "+v"(sum));
}

// gate / (1 + exp(-gate)) * up.  exp(x) = 2^(x log2 e): the product's rounded-off part goes in as a factor of its own, so that the
// error does not grow with x (a few 2^-24); quotient and power by the hardware's reciprocal and exponential, an ulp each.  (The polynomial
// and the correctly rounded division of the int4 layers' SwiGLU are their interface's bits; in the epilogue of a 256 x 256 tile they took 7 us.)
__device__ __forceinline__ float mx_silu(float gate, float up) {
    constexpr float L = 1.44269504088896f, L_REST = 1.92596299e-8f, LN2 = 0.693147180559945f; // log2 e = L + L_REST
    const float t = -gate * L, rest = fmaf(-gate, L_REST, fmaf(-gate, L, -t));
    const float power = __builtin_amdgcn_exp2f(t) * (fabsf(gate) < 128.0f ? fmaf(rest, LN2, 1.0f) : 1.0f); // (beyond: 0 or infinity)
    // (of a quarter: the reciprocal gives zero for what is 2^126 or more, where gate * reciprocal is still a normal number)
    return 0.25f * gate * __builtin_amdgcn_rcpf(fmaf(0.25f, power, 0.25f)) * up;
}

// N (4 or 8) consecutive values to where `to` points, of which `count` exist.  (Instructions that are not yet in the cache cost small
// calls more than those that run: the part of a row's end is a loop.)
template <int TYPE, int N> __device__ __forceinline__ void mx_put(void* to, int count, float (&v)[N]) {
    if (count >= N) {
        mx_store<TYPE, N>(to, 0, v);
    } else {
#pragma unroll 1
        for (int e = 0; e < count; ++e) {
            mx_store1<TYPE>(to, e, v[0]);
#pragma unroll
            for (int i = 0; i + 1 < N; ++i) v[i] = v[i + 1];
        }
    }
}
template <int N> __device__ __forceinline__ void mx_put(const rkh_mx4_gemm_args& g, int m, int n, float (&v)[N]) {
    mx_with_type(g.out_type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        mx_put<TYPE, N>(static_cast<typename MxType<TYPE>::T*>(g.C) + (size_t)m * g.ldc + n, g.N - n, v);
    });
}

// A block of 32 middle columns as MX4: the lane's eight values of row m, the block shared with lanes 16, 32 and 48 on.
__device__ __forceinline__ void mx_put_rows(const rkh_mx4_gemm_args& g, int m, int block, bool live, const float (&v)[8], int lane) {
    uint32_t top = mx_top(v);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const uint32_t scale = mx_scale(top);
    if (!live) return;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.C) + mx_code_at(m, block, (int)rkh_mx4_k4(g.N)) + (lane >> 4) * 4) = mx_codes(v, scale);
    if (lane < 16) g.c_scale[mx_scale_at(m, block, (int)rkh_mx4_k4(g.N))] = (uint8_t)scale;
}

// ---- few rows ----------------------------------------------------------------------
// One workgroup multiplies all rows with 16 * CN places; its waves split K in groups of 512 and are summed through LDS.  Every weight
// byte is loaded once, straight into registers, NG groups of a wave together: all of its share unless K is very long.
// FUSED: the rows are given as values, and every workgroup quantizes them for itself (2: norms them first), behind its first weights'
// loads: those wait to leave for as long as the stream takes, the last of them almost to its end.  (Waves of their own that quantize have their
// loads behind everyone's weights: 1 x 4096 -> 14336 7.6 -> 11.3 us.  A launch in front costs 3.)
__host__ __device__ constexpr int few_row_bytes(int K4) { return K4 * (256 + 16 + 4); } // codes, scales, sums of squares

struct MxFewRows { // the workgroup's rows in LDS
    uint8_t* codes;  // block b of row r: 16 bytes at (b * M + r) * 16
    uint8_t* scales; // a lane's four of a group: one dword
    float* squares;  // [row][segment of 512]
    int M, K4;
    __device__ MxFewRows(uint8_t* lds, int rows, int k4)
        : codes(lds), scales(lds + k4 * rows * 256), squares(reinterpret_cast<float*>(scales + k4 * rows * 16)), M(rows), K4(k4) {}
    __device__ __forceinline__ void put(int r, int piece, const float (&v)[8]) const { // (four lanes of a block together)
        const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(v)));
        const int b = piece >> 2;
        *reinterpret_cast<uint32_t*>(codes + (b * M + r) * 16 + (piece & 3) * 4) = mx_codes(v, scale);
        if ((piece & 3) == 0) scales[(((b >> 4) * M + r) * 4 + (b & 3)) * 4 + ((b >> 2) & 3)] = (uint8_t)scale;
    }
};

// Quantizes the rows into `to` with `threads` threads; `between` runs behind the first loads.  A wave's 64 pieces of eight values are a segment of one
// row.  K is a multiple of eight.  PIECES: of a thread, that are fetched ahead.
template <int TYPE, int PIECES, bool NORM, class Between>
__device__ __forceinline__ void mx_few_quantize(const rkh_mx4_gemm_args& g, const MxFewRows& to, int threads, Between&& between) {
    const int per_row = to.K4 * 64, total = per_row * to.M, t = threadIdx.x;
    const auto row_of = [&](int i) { return to.M == 1 ? 0 : (int)((unsigned)i / (unsigned)per_row); };
    const auto fetch = [&](int i) {
        const int r = row_of(i), k = (i - r * per_row) * 8;
        MxRaw<TYPE> raw = {};
        if (i < total && k < g.K) raw = mx_fetch8<TYPE>(g.x, (size_t)r * g.ldx + k);
        return raw;
    };
    const auto weight_of = [&](int i) {
        const int k = (i - row_of(i) * per_row) * 8;
        MxRaw<RKH_MX4_F32> raw = {};
        if (i < total && k < g.K) raw = mx_fetch8<RKH_MX4_F32>(g.x_weight, k);
        return raw;
    };
    MxRaw<TYPE> raw[PIECES];
    MxRaw<RKH_MX4_F32> weight[PIECES];
#pragma unroll
    for (int u = 0; u < PIECES; ++u) raw[u] = fetch(t + u * threads);
    if (NORM && g.x_weight) {
#pragma unroll
        for (int u = 0; u < PIECES; ++u) weight[u] = weight_of(t + u * threads);
    }
    // (a wave's share of the rows would queue behind the weights of those that are ahead of it, and all wait for the last)
    asm volatile("s_barrier" ::: "memory");
    between();
    const auto each = [&](auto&& f) { // f(piece, values, its place among those fetched ahead or -1)
        static_for<PIECES>([&](auto u) {
            if (t + u() * threads >= total) return;
            float v[8];
            mx_unpack<TYPE>(raw[u()], v);
            f(t + u() * threads, v, u);
        });
#pragma unroll 1
        for (int i = t + PIECES * threads; i < total; i += threads) {
            float v[8];
            mx_unpack<TYPE>(fetch(i), v);
            f(i, v, std::integral_constant<int, -1>{});
        }
    };
    if constexpr (NORM) {
        each([&](int i, float (&v)[8], auto) {
            const float sum = mx_segment_sum(mx_squares(v, 0.0f));
            if (lane_id() == 0) to.squares[i >> 6] = sum;
        });
        __syncthreads();
        each([&](int i, float (&v)[8], auto ahead) {
            constexpr int U = decltype(ahead)::value;
            const int r = row_of(i);
            const float factor = mx_norm_factor(mx_sum_of_segments(to.squares + r * to.K4, to.K4), g.K, g.x_eps);
            float w[8];
            if (g.x_weight) {
                if constexpr (U >= 0) mx_unpack<RKH_MX4_F32>(weight[U], w);
                else mx_unpack<RKH_MX4_F32>(weight_of(i), w);
            }
            mx_normed(v, factor, g.x_weight != nullptr, w);
            to.put(r, i - r * per_row, v);
        });
    } else {
        each([&](int i, float (&v)[8], auto) {
            const int r = row_of(i);
            to.put(r, i - r * per_row, v);
        });
    }
    __syncthreads();
}

// (Leading scalar arguments arrive in registers; the structure takes a round trip to memory, which its users here can wait for.
// FUSED: a_scale is the rows' stride.)
// X: the rows' type.
template <int RM, int CN, int NG, int MAX_WAVES, bool SWIGLU, int FUSED, int X>
__global__ __launch_bounds__(MAX_WAVES * 64, RM == 1 ? 4 : 1) void mx4_few_kernel(const uint8_t* W, const uint8_t* w_scale, const void* rows, const uint8_t* a_scale, int M, int N,
                                                                                 int K, int per_wave, int workgroups, int waves, rkh_mx4_gemm_args g) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    static_assert(!SWIGLU || CN == 4, "gate and up halves of a block of 32 columns");
    static_assert(!FUSED || RM == 1, "rows as given: up to 16");
    g.M = M, g.N = N, g.K = K;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    const int KS = (int)rkh_mx4_ks(K), K4 = (int)rkh_mx4_k4(K);
    const int col0 = xcd_remap(blockIdx.x, workgroups) * CN; // first of the workgroup's operands of weights
    const int cols = (int)rkh_mx4_columns(SWIGLU ? 2 * N : N, SWIGLU) / 16;
    const int first = wave * per_wave, last = min(first + per_wave, K4); // groups of 512 k

    v4i w[NG][4][CN], a[NG][4][RM];
    uint32_t ws[NG][CN], as[NG][RM];
    // (groups beyond the last: that one again, multiplied with nothing.  Pieces beyond K: the activations' are zeros, any weights will do)
    const auto load = [&](int from, auto s0, auto s1) { // steps s0 .. s1 - 1 of each group, the scales behind the last
        static_for<NG>([&](auto p_tag) {
            constexpr int P = decltype(p_tag)::value;
            const int group = min(from + P, K4 - 1);
#pragma unroll
            for (int s = s0(); s < s1(); ++s) {
#pragma unroll
                for (int j = 0; j < CN; ++j)
                    w[P][s][j] = *reinterpret_cast<const v4i*>(W + ((size_t)min(col0 + j, cols - 1) * K4 + group) * 4096 + (group * 4 + s < KS ? s * 1024 : 0) + lane * 16);
                if constexpr (!FUSED) {
#pragma unroll
                    for (int i = 0; i < RM; ++i)
                        a[P][s][i] = *reinterpret_cast<const v4i*>(static_cast<const uint8_t*>(rows) + ((size_t)min(i, (M - 1) >> 4) * K4 + group) * 4096 + s * 1024 + lane * 16);
                }
            }
            if constexpr (s1() == 4) {
#pragma unroll
                for (int j = 0; j < CN; ++j) ws[P][j] = reinterpret_cast<const uint32_t*>(w_scale)[((size_t)min(col0 + j, cols - 1) * K4 + group) * 64 + lane];
                if constexpr (!FUSED) {
#pragma unroll
                    for (int i = 0; i < RM; ++i) as[P][i] = reinterpret_cast<const uint32_t*>(a_scale)[((size_t)min(i, (M - 1) >> 4) * K4 + group) * 64 + lane];
                }
            }
        });
        __builtin_amdgcn_sched_barrier(0);
    };
    using S0 = std::integral_constant<int, 0>;
    using S4 = std::integral_constant<int, 4>;
    // what goes out ahead of the rows' quantization: half of the weights where they are many
    using Ahead = std::integral_constant<int, CN * NG >= 4 ? 2 : 4>;
    v4f* sums = reinterpret_cast<v4f*>(lds);
    const MxFewRows staged(lds + waves * RM * CN * 1024, M, K4);
    if constexpr (FUSED) {
        g.x = rows;
        g.ldx = (int64_t)reinterpret_cast<intptr_t>(a_scale);
        mx_few_quantize<X, CN == 4 ? 1 : 2, FUSED == 2>(g, staged, waves * 64, [&]() { load(first, S0{}, Ahead{}); });
        if constexpr (Ahead::value < 4) load(first, Ahead{}, S4{});
    } else {
        load(first, S0{}, S4{});
    }

    v4f acc[RM][CN];
#pragma unroll
    for (int t = 0; t < RM * CN; ++t) acc[t / CN][t % CN] = v4f{0, 0, 0, 0};
    const bool live = (lane & 15) < M;
    for (int from = first;;) {
        static_for<NG>([&](auto p_tag) {
            constexpr int P = decltype(p_tag)::value;
            const int group = from + P;
            if (group >= last) return;
            if constexpr (FUSED) as[P][0] = live ? *reinterpret_cast<const uint32_t*>(staged.scales + ((group * M + (lane & 15)) * 4 + (lane >> 4)) * 4) : 0;
            static_for<4>([&](auto s_tag) {
                constexpr int S = decltype(s_tag)::value;
                if constexpr (FUSED)
                    a[P][S][0] = live ? *reinterpret_cast<const v4i*>(staged.codes + (((group * 4 + S) * 4 + (lane >> 4)) * M + (lane & 15)) * 16) : v4i{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < CN; ++j) acc[i][j] = mx_mfma<S>(w[P][S][j], a[P][S][i], acc[i][j], ws[P][j], as[P][i]);
            });
        });
        from += NG;
        if (from >= last) break;
        load(from, S0{}, S4{});
    }

    // the waves' sums, added in order: thread (tile, lane) takes the tile's place `lane`
#pragma unroll
    for (int t = 0; t < RM * CN; ++t) sums[(wave * RM * CN + t) * 64 + lane] = acc[t / CN][t % CN];
    __syncthreads();
    if constexpr (!SWIGLU) {
        for (int t = wave; t < RM * CN; t += waves) {
            v4f s = sums[t * 64 + lane];
            for (int o = 1; o < waves; ++o) s += sums[(o * RM * CN + t) * 64 + lane];
            const int m = t / CN * 16 + (lane & 15), col = col0 + t % CN;
            float v[4] = {s.x, s.y, s.z, s.w};
            if (m < M && col < cols) mx_put<4>(g, m, (col >> 1) * 32 + 8 * (lane >> 4) + 4 * (col & 1), v);
        }
    } else {
        for (int i = wave; i < RM; i += waves) {
            v4f s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = sums[(i * 4 + j) * 64 + lane];
                for (int o = 1; o < waves; ++o) s[j] += sums[((o * RM + i) * 4 + j) * 64 + lane];
            }
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = mx_silu(s[e >> 2][e & 3], s[2 + (e >> 2)][e & 3]);
            const int m = i * 16 + (lane & 15), block = col0 / 4;
            if (g.out_type == RKH_MX4_ROWS) mx_put_rows(g, m, block, m < M, v, lane);
            else if (m < M) mx_put<8>(g, m, block * 32 + 8 * (lane >> 4), v);
        }
    }
}

// ---- tiles ---------------------------------------------------------------------------
// Tiles of 32 RM rows x 32 CN places by four waves (two by two), RM x CN accumulators each.  A step is 128 k: every operand of the tile is 1 KiB,
// copied global -> LDS directly (no registers) D steps ahead, and read into registers one step ahead of its products.  Four steps
// are a group, whose scales are 256 bytes per operand, copied two groups ahead.  K ends with a group: pieces beyond it are zeros.
//
// The copies are inline assembly (they write no register; the compiler, which would put every LDS read behind ALL copies in
// flight, does not see them), and what orders them is explicit:
//  * the copies of step s + D are issued in step s, into the buffer of step s - 1 (the ring has D + 1): its last reads were issued in step
//    s - 2 and waited for by the products of step s - 1, ahead of the barrier that ended it;
//  * step s reads the operands of step s + 1; the wait in front of the barrier that ends step s - 1 has left no copy of that step in
//    flight (vector memory loads complete in order, wait_for() counts what was issued since);
//  * the scales of group g + 2, issued in the second step of group g, overwrite those of group g, which were read in the last
//    step of group g - 1 and waited for by the products of the first step of group g, ahead of the barrier that ended it.
// Copies beyond the part's K bring its last step again, for the count; nothing reads them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is set and clobbered on purpose below
// 16 bytes per lane from base + off, lane-contiguous to LDS address `to`.  (A load to LDS needs a wait state behind a write of M0.)
__device__ __forceinline__ void mx_copy(const uint8_t* base, unsigned off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop

// HALVES: groups that the ring holds.
template <int RM, int CN, int HALVES> struct MxTile {
    static constexpr int AB = 2 * RM, WB = 2 * CN;               // operands of a step
    static constexpr int COPIES = (AB + WB) / 4;                 // 1 KiB copies of a wave per step
    static constexpr int SCALE_COPIES = (AB + WB) / 4;           // 1 KiB copies of four operands' scales, of all waves
    static constexpr int SC = (SCALE_COPIES + 3) / 4;            // ... of a wave per group
    static constexpr int D = 4 * HALVES - 1;                     // look-ahead
    static constexpr int BUF = (AB + WB) * 1024, SBUF = (AB + WB) * 256;
    static constexpr int SCALES_OFF = 4 * HALVES * BUF, LDS = SCALES_OFF + 2 * SBUF;
    static_assert(RM % 2 == 0 && CN % 2 == 0 && (HALVES == 1 || HALVES == 2) && LDS <= 160 * 1024, "");
    // The copies of step t + 2 of a group have landed: what a wave has issued in the D - 2 steps up to step t.  FIRST: no group is ahead of this one; the
    // prologue issues its scales earlier than a group would.
    static constexpr int wait_for(int t, bool first) {
        int n = 0;
        for (int s = 0; s < D - 2; ++s) n += COPIES + ((t - s + 8) % 4 == 1 && (!first || t - s >= 0) ? SC : 0);
        return n;
    }
    // All of it counted out over the first groups: whatever a step reads has landed behind the wait that ends the step before.
    static constexpr bool covers() {
        constexpr int STEPS = 16;
        int issued = 0, step_at[STEPS + 16] = {}, scales_at[STEPS / 4 + 4] = {};
        scales_at[0] = issued += SC;
        for (int s = 0; s < D; ++s) {
            if (s == 2) scales_at[1] = issued += SC;
            step_at[s] = issued += COPIES;
        }
        int landed = issued - (D - 2) * COPIES;
        if (step_at[1] > landed || scales_at[1] > landed) return false;
        for (int t = 0; t < STEPS; ++t) {
            if (t % 4 == 1) scales_at[t / 4 + 2] = issued += SC;
            step_at[t + D] = issued += COPIES;
            landed = issued - wait_for(t % 4, t < 4);
            if (step_at[t + 2] > landed || ((t + 1) % 4 == 3 && scales_at[t / 4 + 1] > landed)) return false;
        }
        return true;
    }
};

// Where a tile lies: column sweeps over groups of row blocks, so that concurrently running tiles share weights in L2.
__device__ __forceinline__ void mx_place(unsigned tile, unsigned mblocks, unsigned nblocks, int& mblk, int& nblk) {
    constexpr unsigned GM = 4;
    const unsigned per_group = GM * nblocks, grp = tile / per_group, first_m = grp * GM, gm = min(mblocks - first_m, GM);
    const unsigned in_group = tile - grp * per_group, col = in_group / gm;
    mblk = __builtin_amdgcn_readfirstlane((int)(first_m + in_group - col * gm));
    nblk = __builtin_amdgcn_readfirstlane((int)col);
}

// The jobs of a launch: tiles, or parts of them where K is split (all tiles' first parts, then all second ones, ..).  `halves`: from tile `skip` on every
// tile is two jobs, its upper and its lower half of rows.
struct MxJobs {
    int mblocks, nblocks, parts; // of whole tiles
    int jobs, skip;
    bool halves;
    __device__ __forceinline__ void place(int job, int& mblk, int& nblk, int& kpart) const {
        const unsigned j = (unsigned)xcd_remap(job, jobs);
        // (quotients of uniform values come out of vector registers)
        if (halves) {
            mx_place(skip + (j >> 1), mblocks, nblocks, mblk, nblk);
            mblk = 2 * mblk + (j & 1), kpart = 0;
        } else {
            const unsigned tiles = (unsigned)mblocks * nblocks;
            kpart = parts == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)(j / tiles));
            mx_place(j - kpart * tiles, mblocks, nblocks, mblk, nblk);
        }
    }
    __device__ __forceinline__ unsigned partial(int job) const { // [tile][part] of a split job's sums
        const unsigned j = (unsigned)xcd_remap(job, jobs), tiles = (unsigned)mblocks * nblocks;
        return (j % tiles) * parts + j / tiles;
    }
};

// Multiplies jobs job, job + stride, ...  Their steps follow one another: the copies that run ahead of a tile's end are the next
// tile's first, and land while the tile is converted and stored.
template <int RM, int CN, int HALVES, bool SWIGLU, int OUT>
__device__ __forceinline__ void mx_tiles(const rkh_mx4_gemm_args& g, uint8_t* lds, const MxJobs& of, int job, int stride) {
    using S = MxTile<RM, CN, HALVES>;
    static_assert(!SWIGLU || CN % 4 == 0, "gate and up halves of blocks of 32 columns in one wave");
    static_assert(S::covers(), "a step would read what has not landed");
    constexpr auto in_acc = [](int i) { return RM * CN < 64 || i < RM - 1; };
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), wm = wave & 1, wn = wave >> 1;
    const int K4 = (int)rkh_mx4_k4(g.K);
    const int cols = (int)rkh_mx4_columns(SWIGLU ? 2 * g.N : g.N, SWIGLU) / 16, rows = (g.M + 15) / 16; // operands that exist

    // ---- sources: wave-uniform base pointers and a lane offset that advances with K.  Two streams, of steps and of groups of scales, each
    // with the job that it has come to.
    const uint32_t base = (uint32_t)(uintptr_t)(mx_lds_ptr)lds;
    const uint32_t a_to = base + wave * (RM / 2) * 1024, w_to = base + (S::AB + wave * (CN / 2)) * 1024;
    const auto part_of = [&](int kpart, int& g0, int& groups) {
        g0 = of.parts == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)((unsigned)(K4 * kpart) / of.parts));
        groups = (of.parts == 1 ? K4 : __builtin_amdgcn_readfirstlane((int)((unsigned)(K4 * (kpart + 1)) / of.parts))) - g0;
    };
    const uint8_t *a_src[RM / 2], *w_src[CN / 2];
    unsigned k_off = lane * 16, k_step = 1024;
    int mblk_next = 0, nblk_next = 0, groups_next = 0; // of the job that the copies have come to
    const auto steps_of = [&](int j) {
        int kpart, g0;
        of.place(j, mblk_next, nblk_next, kpart);
        part_of(kpart, g0, groups_next);
        const int mblk = mblk_next, nblk = nblk_next;
#pragma unroll
        for (int c = 0; c < RM / 2; ++c) a_src[c] = g.A + ((size_t)min(mblk * S::AB + wave * (RM / 2) + c, rows - 1) * K4 + g0) * 4096;
#pragma unroll
        for (int c = 0; c < CN / 2; ++c) w_src[c] = g.W + ((size_t)min(nblk * S::WB + wave * (CN / 2) + c, cols - 1) * K4 + g0) * 4096;
        k_off = lane * 16;
    };
    // copy x of a group's scales brings those of operands 4 x .. 4 x + 3 of the tile (activations first)
    const uint8_t* s_src[S::SC];
    unsigned s_off[S::SC];
    int s_job = job, s_left = 0; // groups that are still to come of s_job
    const auto scales_of = [&](int j) {
        int mblk, nblk, kpart, g0;
        of.place(j, mblk, nblk, kpart);
        part_of(kpart, g0, s_left);
#pragma unroll
        for (int c = 0; c < S::SC; ++c) {
            const int x = (c * 4 + wave) % S::SCALE_COPIES, op = x * 4 + (lane >> 4);
            static_assert(S::AB % 4 == 0, "a copy's operands are of one kind");
            const bool is_a = x * 4 < S::AB;
            const int first_op = is_a ? mblk * S::AB : nblk * S::WB, limit = (is_a ? rows : cols) - 1;
            const int at = min(first_op, limit);
            s_src[c] = (is_a ? g.a_scale : g.w_scale) + ((size_t)at * K4 + g0) * 256;
            s_off[c] = (unsigned)(min(first_op + op - (is_a ? 0 : S::AB), limit) - at) * (unsigned)K4 * 256 + (lane & 15) * 16;
        }
    };

    v4f acc[RM][CN];
    v4i a[RM], w[2][CN];
    uint32_t as[RM], ws[CN];
    // places in LDS, from the half of the ring that the group lies in and the half of the scales'
    uint32_t half = 0, s_half = 0;
    const auto other = [&](uint32_t h) { return HALVES == 2 ? (uint32_t)(4 * S::BUF) - h : h; };
    const uint8_t* a_at = lds + wm * RM * 1024 + lane * 16;
    const uint8_t* w_at = lds + (S::AB + wn * CN) * 1024 + lane * 16;
    const uint8_t* as_at = lds + S::SCALES_OFF + wm * RM * 256 + lane * 4;
    const uint8_t* ws_at = lds + S::SCALES_OFF + (S::AB + wn * CN) * 256 + lane * 4;

    const auto copy = [&](uint32_t to, auto buf_tag, auto c_tag) {
        constexpr int B = decltype(buf_tag)::value % 4, C = decltype(c_tag)::value;
        if constexpr (C < RM / 2) mx_copy(a_src[C], k_off, a_to + to + B * S::BUF + C * 1024);
        else mx_copy(w_src[C - RM / 2], k_off, w_to + to + B * S::BUF + (C - RM / 2) * 1024);
        if constexpr (C == S::COPIES - 1) k_off += k_step;
    };
    const auto copy_scales = [&](uint32_t to) {
        if (s_left == 0 && s_job + stride < of.jobs) scales_of(s_job += stride);
#pragma unroll
        for (int c = 0; c < S::SC; ++c) {
            mx_copy(s_src[c], s_off[c], base + S::SCALES_OFF + to + (c * 4 + wave) % S::SCALE_COPIES * 1024);
            s_off[c] += s_left > 1 ? 256 : 0;
        }
        s_left -= s_left > 0 ? 1 : 0;
    };
    const auto read_a = [&](uint32_t from, auto t_tag, auto i_tag) {
        constexpr int B = decltype(t_tag)::value % 4, I = decltype(i_tag)::value;
        a[I] = *reinterpret_cast<const v4i*>(a_at + from + B * S::BUF + I * 1024);
    };
    const auto read_w = [&](uint32_t from, auto t_tag, auto j_tag) {
        constexpr int T = decltype(t_tag)::value, B = T % 4, J = decltype(j_tag)::value;
        w[T & 1][J] = *reinterpret_cast<const v4i*>(w_at + from + B * S::BUF + J * 1024);
    };
    const auto read_as = [&](uint32_t from, int i) { as[i] = *reinterpret_cast<const uint32_t*>(as_at + from + i * 256); };
    const auto read_ws = [&](uint32_t from, int j) { ws[j] = *reinterpret_cast<const uint32_t*>(ws_at + from + j * 256); };

    // ---- prologue
    using C0 = std::integral_constant<int, 0>;
    steps_of(job);
    scales_of(job);
    int mblk = mblk_next, nblk = nblk_next, groups = groups_next;
    int c_job = job, c_left = groups * 4; // steps that are still to be copied of c_job
    const auto copied = [&](int n) { // n steps more (never past a tile's last): the next ones are the next tile's, or nobody's
        c_left -= n;
        if (c_left == 0) {
            if (c_job + stride < of.jobs) {
                steps_of(c_job += stride);
                c_left = groups_next * 4;
            } else { // (the last step again, for the count of loads)
                k_off -= k_step;
                k_step = 0;
            }
        }
    };
    copy_scales(0);
    static_for<2>([&](auto b) { static_for<S::COPIES>([&](auto c) { copy(0, b, c); }); });
    copy_scales(S::SBUF);
    static_for<S::D - 2>([&](auto b) {
        constexpr int B = decltype(b)::value + 2;
        if constexpr (B == 4) copied(4);
        static_for<S::COPIES>([&](auto c) { copy(B / 4 * 4 * S::BUF, std::integral_constant<int, B>{}, c); });
    });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S::D - 2) * S::COPIES) : "memory"); // steps 0 and 1, both groups of scales
    static_for<RM>([&](auto i) { read_a(0, C0{}, i); });
    static_for<CN>([&](auto j) { read_w(0, C0{}, j); });
#pragma unroll
    for (int i = 0; i < RM; ++i) read_as(0, i);
#pragma unroll
    for (int j = 0; j < CN; ++j) read_ws(0, j);

    const auto step = [&](auto t_tag, auto fresh_tag) { // FRESH: the sums start here
        constexpr int T = decltype(t_tag)::value, MF = RM * CN;
        using Next = std::integral_constant<int, T + 1>;
        const uint32_t from = T == 3 ? other(half) : half, to = T == 0 ? other(half) : half, s_from = S::SBUF - s_half;
        constexpr int COPIES = S::COPIES, ITEMS = CN + COPIES, BOTH = COPIES < CN ? COPIES : CN;
        if constexpr (T == 1) {
            copied(4); // (the fourth of a group in the step before)
            copy_scales(s_half);
        }
        static_for<MF>([&](auto x_tag) {
            // (rows there and back, so that one operand stays; the last one forth, whose scales are then replaced in order)
            constexpr int X = decltype(x_tag)::value, I = X / CN, J = (I & 1) && I < RM - 1 ? CN - 1 - X % CN : X % CN;
            if constexpr (decltype(fresh_tag)::value && T == 0) mx_mfma_first<T, in_acc(I)>(w[T & 1][J], a[I], acc[I][J], ws[J], as[I]);
            else mx_mfma_in_place<T, in_acc(I)>(w[T & 1][J], a[I], acc[I][J], ws[J], as[I]);
            constexpr int FROM = X * ITEMS / MF, TO = (X + 1) * ITEMS / MF;
            static_for<TO - FROM>([&](auto z_tag) { // copies and reads of weights in turn while there are both
                constexpr int Z = FROM + decltype(z_tag)::value;
                if constexpr (Z < 2 * BOTH ? (Z & 1) == 0 : COPIES > CN)
                    copy(to, std::integral_constant<int, T + S::D>{}, std::integral_constant<int, Z < 2 * BOTH ? Z / 2 : Z - CN>{});
                else read_w(from, Next{}, std::integral_constant<int, Z < 2 * BOTH ? Z / 2 : Z - COPIES>{});
            });
            // what its last product has used is replaced by the next step's
            if constexpr (X % CN == CN - 1) read_a(from, Next{}, std::integral_constant<int, I>{});
            if constexpr (T == 3 && X % CN == CN - 1) read_as(s_from, I);
            if constexpr (T == 3 && I == RM - 1) read_ws(s_from, J);
            __builtin_amdgcn_sched_barrier(0);
        });
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::wait_for(T, decltype(fresh_tag)::value)) : "memory");
    };
    for (;;) {
        const auto group = [&](auto fresh_tag) {
            static_for<4>([&](auto t) { step(t, fresh_tag); });
            half = other(half);
            s_half = S::SBUF - s_half;
        };
        group(std::true_type{});
        for (int n = 1; n < groups; ++n) group(std::false_type{});
        // the last products have to be through
        asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");

        const int m0 = (mblk * 2 + wm) * RM * 16, m_first = m0 + (lane & 15), col_first = (nblk * 2 + wn) * CN;
        if (of.parts > 1) { // partial tile in accumulator order: [tile][part][wave][tile of 16 x 16][lane]
            v4f* to = reinterpret_cast<v4f*>(g.scratch) + ((size_t)of.partial(job) * 4 + wave) * (RM * CN * 64) + lane;
            static_for<RM * CN>([&](auto t) {
                mx_settled<in_acc(t() / CN)>(acc[t() / CN][t() % CN]);
                to[t() * 64] = acc[t() / CN][t() % CN];
            });
        } else {
            constexpr int W = SWIGLU ? 4 : 2; // accumulators of a block of 32 columns
            const int n0 = col_first / W * 32 + 8 * (lane >> 4);
            using T = typename MxType<OUT == RKH_MX4_ROWS ? RKH_MX4_F32 : OUT>::T;
            T* row = static_cast<T*>(g.C) + (size_t)m_first * g.ldc + n0;
            const size_t rows16 = (size_t)16 * g.ldc;
            static_for<RM * CN / W>([&](auto t) {
                constexpr int i = t() / (CN / W), j = t() % (CN / W) * W;
                const int m = m_first + i * 16, n = n0 + j / W * 32;
                float v[8];
#pragma unroll
                for (int x = 0; x < W; ++x) mx_settled<in_acc(i)>(acc[i][j + x]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = acc[i][j + (e >> 2)][e & 3];
                    if constexpr (SWIGLU) v[e] = mx_silu(v[e], acc[i][(j + 2 + (e >> 2)) % CN][e & 3]);
                }
                if constexpr (OUT == RKH_MX4_ROWS) {
                    mx_put_rows(g, m, n >> 5, m < g.M && (n & ~31) < g.N, v, lane);
                } else {
                    if (m < g.M) mx_put<OUT, 8>(row + j / W * 32, g.N - n, v);
                    if constexpr (j + W == CN) row += rows16;
                }
            });
        }
        job += stride;
        if (job >= of.jobs) break;
        mblk = mblk_next, nblk = nblk_next, groups = groups_next; // (copies are less than a tile ahead)
    }
    // a load to LDS must not outlive the workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int RM, int CN, int HALVES, bool SWIGLU, int OUT>
__global__ __launch_bounds__(256) void mx4_tile_kernel(rkh_mx4_gemm_args g, int mblocks, int nblocks, int parts) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    mx_tiles<RM, CN, HALVES, SWIGLU, OUT>(g, lds, MxJobs{mblocks, nblocks, parts, mblocks * nblocks * parts, 0, false}, blockIdx.x, gridDim.x);
}

// Whole tiles of 256 x 256 by one workgroup per compute unit, one after the other; what would be a last round for half of them or fewer goes as tiles of
// 128 x 256, one each.
template <bool SWIGLU, int OUT>
__global__ __launch_bounds__(256) void mx4_big_kernel(rkh_mx4_gemm_args g, int mblocks, int nblocks, int big) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int rest = mblocks * nblocks - big;
    if ((int)blockIdx.x < big) mx_tiles<8, 8, 1, SWIGLU, OUT>(g, lds, MxJobs{mblocks, nblocks, 1, big, 0, false}, blockIdx.x, gridDim.x);
    if ((int)blockIdx.x < 2 * rest) {
        __syncthreads();
        mx_tiles<4, 8, 1, SWIGLU, OUT>(g, lds, MxJobs{mblocks, nblocks, 1, 2 * rest, big, true}, blockIdx.x, 2 * rest);
    }
}

// Sum of the parts of a tile, in their order, and the epilogue.  One wave per 16 rows x 32 columns (SwiGLU: x 32 of the middle).
template <int RM, int CN, bool SWIGLU>
__global__ __launch_bounds__(256) void mx4_join_kernel(rkh_mx4_gemm_args g, int mblocks, int nblocks, int parts) {
    constexpr int W = SWIGLU ? 4 : 2, UNITS = 4 * RM * CN / W; // of a tile
    const int lane = lane_id(), unit = (blockIdx.x * 4 + wave_id());
    const int tile = unit / UNITS, in_tile = unit - tile * UNITS;
    if (tile >= mblocks * nblocks) return;
    const int wave = in_tile / (RM * CN / W), u = in_tile % (RM * CN / W), i = u / (CN / W), j = u % (CN / W) * W;
    int mblk, nblk;
    mx_place(tile, mblocks, nblocks, mblk, nblk);
    const int m = ((mblk * 2 + (wave & 1)) * RM + i) * 16 + (lane & 15), col = (nblk * 2 + (wave >> 1)) * CN + j;

    const v4f* from = reinterpret_cast<const v4f*>(g.scratch) + ((size_t)tile * parts * 4 + wave) * (RM * CN * 64) + (i * CN + j) * 64 + lane;
    v4f s[W];
#pragma unroll
    for (int x = 0; x < W; ++x) s[x] = from[x * 64];
    for (int p = 1; p < parts; ++p) {
        from += 4 * RM * CN * 64;
#pragma unroll
        for (int x = 0; x < W; ++x) s[x] += from[x * 64];
    }
    float v[8];
    if constexpr (SWIGLU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mx_silu(s[e >> 2][e & 3], s[2 + (e >> 2)][e & 3]);
        const int block = col / 4;
        const bool live = m < g.M && block * 32 < g.N;
        if (g.out_type == RKH_MX4_ROWS) mx_put_rows(g, m, block, live, v, lane);
        else if (live) mx_put<8>(g, m, block * 32 + 8 * (lane >> 4), v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s[e >> 2][e & 3];
        if (m < g.M) mx_put<8>(g, m, col * 16 + 8 * (lane >> 4), v);
    }
}

// ---- which kernel ------------------------------------------------------------------
struct MxRoute {
    bool few;
    int rm, cn, parts, mblocks, nblocks; // few: 16 rm rows, 16 cn places of a workgroup
};

constexpr int MX_ROWS = 4;  // rows that the few-row kernel quantizes itself
constexpr int MX_CUS = 256; // compute units that a launch is cut for

// The shapes of tiles, what a group of 512 k takes in each when every compute unit has one, and a tile's conversion, us: from 4096 x 4096 x 4096
// (256 x 256: 32 us), 2048 x 4096 x 4096 (128 x 256, halves of the former: 19.9; 256 x 128 takes the same and had no sizes of its own), 1024 x 4096 x
// 4096 (128 x 128: 11.7), 512 x 4096 x 14336 (128 x 64: 20.7, 64 x 128: 21.0), 256 x 4096 x 4096 (64 x 64: 6.3).
struct MxShape { int rm, cn; float group, end; };
constexpr MxShape MX_SHAPES[] = {{8, 8, 3.4f, 1.8f}, {4, 4, 1.05f, 0.5f}, {2, 4, 0.63f, 0.3f}, {4, 2, 0.62f, 0.3f}, {2, 2, 0.4f, 0.2f}};
constexpr float MX_HALF_GROUP = 2.0f;                     // of 128 x 256
constexpr float MX_TILES_US = 3.0f, MX_JOIN_US = 3.0f, MX_JOIN_RATE = 4.5e6f; // a launch of tiles; of their sum, and its bytes per us
constexpr float MX_FEW_US = 1.0f, MX_FEW_RATE[] = {5.0e6f, 4.5e6f, 3.2e6f};    // 16, 32, 64 rows: 31 MB of weights 6.3, 6.9, 9.6 us

// The kernel that is expected to take the least time.  Where both sides of a choice were measured, us: 64 x 14336 x 4096 few rows 10.1, tiles of 64 x 64
// 7.5; 64 x 4096 x 14336 9.7 and 11.5; 128 x 11008 x 4096 tiles of 64 x 64 9.6, 128 x 64 8.2, 128 x 128 11.2; 128 x 4096 x 14336 64 x 64 13.2, K in two
// parts 12.1; 512 x 14336 x 4096 256 x 256 18.9, 128 x 128 19.4, 64 x 128 27.6; 128 x 4096 -> 2 x 14336 128 x 128 16.5, 64 x 128 17.9, 256 x 128 21.8.
MxRoute mx_route(int M, int N, int K, int swiglu) {
    const int64_t cols = rkh_mx4_columns(swiglu ? 2 * (int64_t)N : N, swiglu) / 16, K4 = rkh_mx4_k4(K);
    MxRoute best{};
    float least = FLT_MAX;
    if (M <= (swiglu ? 32 : 64)) {
        const int size = M <= 16 ? 0 : M <= 32 ? 1 : 2;
        best.few = true;
        best.rm = 1 << size;
        best.cn = swiglu ? 4 : size == 1 && cols > 4 * MX_CUS ? 2 : 1; // (32 x 65536 x 2048 17.7 -> 14.6 us; 1 x 65536 x 4096 the other way, 21.3 -> 22.7)
        best.parts = best.mblocks = 1;
        best.nblocks = (int)((cols + best.cn - 1) / best.cn);
        least = MX_FEW_US + (float)cols * 16 * K4 * 512 * 17 / 32 / MX_FEW_RATE[size];
    }
    if (M <= 16) return best;
    for (const MxShape& s : MX_SHAPES) {
        if (swiglu && s.cn % 4) continue;
        MxRoute r{};
        r.rm = s.rm, r.cn = s.cn, r.parts = 1;
        r.mblocks = (M + 32 * s.rm - 1) / (32 * s.rm);
        r.nblocks = (int)((cols + 2 * s.cn - 1) / (2 * s.cn));
        const int64_t tiles = (int64_t)r.mblocks * r.nblocks, left = tiles % MX_CUS;
        const float round = K4 * s.group + s.end;
        float us = MX_TILES_US + (tiles - left) / MX_CUS * round;
        if (left) us += s.cn == 8 && left <= MX_CUS / 2 ? K4 * MX_HALF_GROUP + s.end / 2 : round;
        if (us < least) least = us, best = r;
        // K in parts where the tiles leave compute units without one
        for (int64_t parts = 2; s.cn < 8 && parts <= K4 / 4 && tiles * parts <= MX_CUS; ++parts) {
            us = MX_TILES_US + (K4 + parts - 1) / parts * s.group + s.end + MX_JOIN_US + (float)M * cols * 16 * 8 * parts / MX_JOIN_RATE;
            if (us < least) least = us, best = r, best.parts = (int)parts;
        }
    }
    return best;
}
size_t mx_scratch(const MxRoute& r) { return r.few || r.parts == 1 ? 0 : (size_t)r.mblocks * r.nblocks * r.parts * r.rm * r.cn * 4096; }

// More than 64 KiB of LDS for a kernel, once per device; `opted_in` is the kernel's own.
int mx_allow_lds(const void* kernel, std::atomic<bool> (&opted_in)[64], int bytes) {
    int dev = 0;
    RKH_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64) return RKH_ERR_RUNTIME;
    if (!opted_in[dev].load(std::memory_order_acquire)) {
        RKH_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        opted_in[dev].store(true, std::memory_order_release);
    }
    return RKH_OK;
}

template <int RM, int CN, int NG, int MAX_WAVES, bool SWIGLU, int FUSED, int X>
int launch_few_as(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r, int per, int waves) {
    const int K4 = (int)rkh_mx4_k4(g.K);
    if ((int64_t)r.nblocks * waves * 64 >= MX_TOO_MANY_THREADS) return RKH_ERR_RUNTIME;
    const size_t bytes = (size_t)waves * RM * CN * 1024 + (FUSED ? (size_t)few_row_bytes(K4) * g.M : 0);
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(&mx4_few_kernel<RM, CN, NG, MAX_WAVES, SWIGLU, FUSED, X>), opted_in, 160 * 1024)) return rc;
    mark(st, "mx4_few_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_few_kernel<RM, CN, NG, MAX_WAVES, SWIGLU, FUSED, X>), dim3(r.nblocks), dim3(waves * 64), bytes, st, g.W,
                       g.w_scale, FUSED ? g.x : g.A, FUSED ? reinterpret_cast<const uint8_t*>((intptr_t)g.ldx) : g.a_scale, g.M, g.N, g.K, per, r.nblocks, waves, g);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}
template <int RM, int CN, int MAX_WAVES, bool SWIGLU, int FUSED> int launch_few(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    const int K4 = (int)rkh_mx4_k4(g.K), per = (K4 + MAX_WAVES - 1) / MAX_WAVES, waves = (K4 + per - 1) / per;
    int rc = RKH_OK;
    const auto as = [&](auto x) {
        constexpr int X = decltype(x)::value;
        if constexpr (RM * CN == 1) {
            if (per > 1) {
                rc = launch_few_as<RM, CN, 2, MAX_WAVES, SWIGLU, FUSED, X>(st, g, r, per, waves);
                return;
            }
        }
        rc = launch_few_as<RM, CN, 1, MAX_WAVES, SWIGLU, FUSED, X>(st, g, r, per, waves);
    };
    if constexpr (FUSED) mx_with_type(g.x_type, as);
    else as(std::integral_constant<int, RKH_MX4_F32>{});
    return rc;
}

template <int RM, int CN, int HALVES, bool SWIGLU, int OUT> int launch_tiles(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    constexpr int LDS = MxTile<RM, CN, HALVES>::LDS;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(&mx4_tile_kernel<RM, CN, HALVES, SWIGLU, OUT>), opted_in, LDS)) return rc;
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
    if (tiles * r.parts * 256 >= MX_TOO_MANY_THREADS) return RKH_ERR_RUNTIME;
    mark(st, "mx4_tile_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_tile_kernel<RM, CN, HALVES, SWIGLU, OUT>), dim3((unsigned)(tiles * r.parts)), dim3(256), LDS, st, g, r.mblocks,
                       r.nblocks, r.parts);
    RKH_CHECK(hipGetLastError());
    if (r.parts > 1) {
        mark(st, "mx4_join_kernel");
        hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_join_kernel<RM, CN, SWIGLU>), dim3((unsigned)(tiles * RM * CN / (SWIGLU ? 4 : 2))), dim3(256), 0, st, g,
                           r.mblocks, r.nblocks, r.parts);
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}

template <bool SWIGLU, int OUT> int launch_big(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    constexpr int LDS = MxTile<8, 8, 1>::LDS;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(&mx4_big_kernel<SWIGLU, OUT>), opted_in, LDS)) return rc;
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks, left = tiles % MX_CUS, big = left <= MX_CUS / 2 ? tiles - left : tiles;
    if (tiles > 0x3fffffff) return RKH_ERR_RUNTIME;
    mark(st, "mx4_big_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_big_kernel<SWIGLU, OUT>), dim3((unsigned)(big ? std::min<int64_t>(big, MX_CUS) : 2 * left)), dim3(256), LDS,
                       st, g, r.mblocks, r.nblocks, (int)big);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

template <bool SWIGLU, int OUT> int launch_shape(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    if (r.rm == 8) return launch_big<SWIGLU, OUT>(st, g, r);
    if constexpr (!SWIGLU) {
        if (r.cn == 2) return r.rm == 4 ? launch_tiles<4, 2, 2, SWIGLU, OUT>(st, g, r) : launch_tiles<2, 2, 2, SWIGLU, OUT>(st, g, r);
    }
    return r.rm == 4 ? launch_tiles<4, 4, 1, SWIGLU, OUT>(st, g, r) : launch_tiles<2, 4, 2, SWIGLU, OUT>(st, g, r);
}

template <bool SWIGLU> int launch(hipStream_t st, const rkh_mx4_gemm_args& g) {
    MxRoute r = mx_route(g.M, g.N, g.K, SWIGLU);
    if (r.few) {
        if (!g.A) {
            if constexpr (SWIGLU) return g.x_norm ? launch_few<1, 4, 8, true, 2>(st, g, r) : launch_few<1, 4, 8, true, 1>(st, g, r);
            else return launch_few<1, 1, 16, false, 1>(st, g, r);
        }
        if constexpr (SWIGLU) {
            if (r.rm == 1) return launch_few<1, 4, 8, true, 0>(st, g, r);
            return launch_few<2, 4, 8, true, 0>(st, g, r);
        } else {
            if (r.rm == 1) return launch_few<1, 1, 16, false, 0>(st, g, r);
            if (r.rm == 2) return r.cn == 1 ? launch_few<2, 1, 16, false, 0>(st, g, r) : launch_few<2, 2, 8, false, 0>(st, g, r);
            return launch_few<4, 1, 8, false, 0>(st, g, r);
        }
    }
    if (mx_scratch(r) > (g.scratch ? g.scratch_bytes : 0)) r.parts = 1;
    // (partial tiles have no type)
    switch (r.parts > 1 ? RKH_MX4_F32 : g.out_type) {
    case RKH_MX4_F16: return launch_shape<SWIGLU, RKH_MX4_F16>(st, g, r);
    case RKH_MX4_BF16: return launch_shape<SWIGLU, RKH_MX4_BF16>(st, g, r);
    case RKH_MX4_ROWS:
        if constexpr (SWIGLU) return launch_shape<SWIGLU, RKH_MX4_ROWS>(st, g, r);
        return RKH_ERR_RUNTIME;
    default: return launch_shape<SWIGLU, RKH_MX4_F32>(st, g, r);
    }
}

} // namespace

#endif // RK_KERNELS_MX4_GEMM_H
