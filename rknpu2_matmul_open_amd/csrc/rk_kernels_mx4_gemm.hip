// Products of MX4 operands (v_mfma_scale_f32_16x16x128_f8f6f4, fp32 sums): mx4_few_kernel for decode-sized M, bound by the
// weights' bytes; mx4_tile_kernel for more rows, bound by the matrix pipes; mx4_join_kernel, the sum of partial tiles.
//
// The weights are the FIRST operand: lane (r, q) = (l % 16, l / 16) of a 16 x 16 accumulator owns activation row r and four of the
// tile's weight rows, which the packing has made the consecutive columns 8 q + 4 h .. + 3 of a block of 32 (h: the first or the
// second tile of the block).
#include "rk_kernels_mx4.h"

namespace {

typedef __attribute__((address_space(3))) uint8_t* mx_lds_ptr;

// sum += W * A over 128 k; the scales are byte STEP of the lanes' dwords.
template <int STEP> __device__ __forceinline__ v4f mx_mfma(const v4i& w, const v4i& a, const v4f& sum, uint32_t ws, uint32_t as) {
    const v8i w8 = {w.x, w.y, w.z, w.w, 0, 0, 0, 0}, a8 = {a.x, a.y, a.z, a.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, sum, 4, 4, STEP, (int)ws, STEP, (int)as);
}

__device__ __forceinline__ float mx_silu(float gate, float up) { return __fmul_rn(silu_poly(gate), up); }

// N (4 or 8) consecutive columns from n on of row m, of which those below `end` exist.
template <int N> __device__ __forceinline__ void mx_put(const rkh_mx4_gemm_args& g, int m, int n, int end, const float* v) {
    mx_with_type(g.out_type, [&](auto t) {
        constexpr int TYPE = decltype(t)::value;
        const size_t at = (size_t)m * g.ldc + n;
        if (n + N <= end) {
            mx_store<TYPE, N>(g.C, at, v);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (n + e < end) mx_store1<TYPE>(g.C, at + e, v[e]);
        }
    });
}

// A block of 32 middle columns as MX4: the lane's eight values of row m, the block shared with lanes 16, 32 and 48 on.
__device__ __forceinline__ void mx_put_rows(const rkh_mx4_gemm_args& g, int m, int block, bool live, const float (&v)[8], int lane) {
    uint32_t top = mx_top(v);
    top = max(top, (uint32_t)__shfl_xor((int)top, 16));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32));
    const uint32_t scale = mx_scale(top);
    if (!live) return;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.C) + mx_code_at(m, block, (int)rkh_mx4_ks(g.N)) + (lane >> 4) * 4) = mx_codes(v, scale);
    if (lane < 16) g.c_scale[mx_scale_at(m, block, (int)rkh_mx4_k4(g.N))] = (uint8_t)scale;
}

// ---- few rows ----------------------------------------------------------------------
// One workgroup multiplies all rows with 16 * CN places; its waves split K in groups of 512 and are summed through LDS.  Every weight
// byte is loaded once, straight into registers, a group (CN * 4 KiB per wave) ahead of its products.
// FUSED: the rows are given as values, and every workgroup quantizes them for itself while its first weights are on their way.
constexpr int FEW_FUSED_LDS = 64 * 1024;

template <int RM, int CN, int MAX_WAVES, bool SWIGLU, bool FUSED>
__global__ __launch_bounds__(MAX_WAVES * 64) void mx4_few_kernel(rkh_mx4_gemm_args g, int per_wave) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    static_assert(!SWIGLU || CN == 4, "gate and up halves of a block of 32 columns");
    static_assert(!FUSED || RM == 1, "rows as given: up to 16");
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), waves = blockDim.x >> 6;
    const int KS = (int)rkh_mx4_ks(g.K), K4 = (int)rkh_mx4_k4(g.K);
    const int col0 = xcd_remap(blockIdx.x, gridDim.x) * CN; // first of the workgroup's operands of weights
    const int cols = (int)rkh_mx4_columns(SWIGLU ? 2 * g.N : g.N, SWIGLU) / 16;
    const int rblocks = (g.M + 15) / 16;
    const int first = wave * per_wave, last = min(first + per_wave, K4); // groups of 512 k

    v4i w[4][CN];
    uint32_t ws[CN];
    const auto load_w = [&](int group) {
#pragma unroll
        for (int j = 0; j < CN; ++j) {
            const int col = min(col0 + j, cols - 1);
            const uint8_t* src = g.W + ((size_t)col * KS + group * 4) * 1024 + lane * 16;
#pragma unroll
            for (int s = 0; s < 4; ++s) w[s][j] = *reinterpret_cast<const v4i*>(src + (group * 4 + s < KS ? s * 1024 : 0));
            ws[j] = reinterpret_cast<const uint32_t*>(g.w_scale)[((size_t)col * K4 + group) * 64 + lane];
        }
    };

    if constexpr (FUSED) {
        // Blocks b of row r: 16 bytes at (b * M + r) * 16; their scales behind them, so that a lane's four of a group are a dword.
        uint8_t* lds_scales = lds + (size_t)KS * 4 * g.M * 16;
        mx_with_type(g.x_type, [&](auto t) {
            constexpr int TYPE = decltype(t)::value;
            const int per_row = KS * 16, total = per_row * g.M; // pieces of eight values
            const auto fetch = [&](int i) {
                const int r = i / per_row, k = (i - r * per_row) * 8;
                const size_t at = (size_t)r * g.ldx + k;
                return k + 8 <= g.K ? mx_fetch8<TYPE>(g.x, at) : mx_fetch_some<TYPE>(g.x, at, g.K - k);
            };
            const auto put = [&](int i, const MxRaw<TYPE>& raw) {
                const int r = i / per_row, piece = i - r * per_row, b = piece >> 2;
                float v[8];
                mx_unpack<TYPE>(raw, v);
                const uint32_t scale = mx_scale(mx_top_of_quad(mx_top(v)));
                *reinterpret_cast<uint32_t*>(lds + ((size_t)b * g.M + r) * 16 + (piece & 3) * 4) = mx_codes(v, scale);
                if ((piece & 3) == 0) lds_scales[(((b >> 4) * g.M + r) * 4 + (b & 3)) * 4 + ((b >> 2) & 3)] = (uint8_t)scale;
            };
            int i = threadIdx.x;
            MxRaw<TYPE> raw = {};
            if (i < total) raw = fetch(i);
            if (first < last) load_w(first);
            for (; i < total; i += blockDim.x) {
                MxRaw<TYPE> next = {};
                if (i + (int)blockDim.x < total) next = fetch(i + blockDim.x);
                put(i, raw);
                raw = next;
            }
        });
        __syncthreads();
    } else {
        if (first < last) load_w(first);
    }

    v4f acc[RM][CN];
#pragma unroll
    for (int t = 0; t < RM * CN; ++t) acc[t / CN][t % CN] = v4f{0, 0, 0, 0};
    for (int group = first; group < last; ++group) {
        v4i a[4][RM];
        uint32_t as[RM];
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            if constexpr (FUSED) {
                const int r = lane & 15, q = lane >> 4;
                const bool live = r < g.M;
                const uint8_t* lds_scales = lds + (size_t)KS * 4 * g.M * 16;
                as[i] = live ? *reinterpret_cast<const uint32_t*>(lds_scales + ((group * g.M + r) * 4 + q) * 4) : 0;
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    a[s][i] = live && group * 4 + s < KS ? *reinterpret_cast<const v4i*>(lds + ((size_t)((group * 4 + s) * 4 + q) * g.M + r) * 16) : v4i{0, 0, 0, 0};
            } else {
                const int rb = min(i, rblocks - 1);
                const uint8_t* src = g.A + ((size_t)rb * KS + group * 4) * 1024 + lane * 16;
#pragma unroll
                for (int s = 0; s < 4; ++s) a[s][i] = *reinterpret_cast<const v4i*>(src + (group * 4 + s < KS ? s * 1024 : 0));
                as[i] = reinterpret_cast<const uint32_t*>(g.a_scale)[((size_t)rb * K4 + group) * 64 + lane];
            }
        }
        v4i wc[4][CN];
        uint32_t wsc[CN];
#pragma unroll
        for (int j = 0; j < CN; ++j) {
#pragma unroll
            for (int s = 0; s < 4; ++s) wc[s][j] = w[s][j];
            wsc[j] = ws[j];
        }
        if (group + 1 < last) load_w(group + 1);
        static_for<4>([&](auto s_tag) {
            constexpr int S = decltype(s_tag)::value;
            if (group * 4 + S < KS) {
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < CN; ++j) acc[i][j] = mx_mfma<S>(wc[S][j], a[S][i], acc[i][j], wsc[j], as[i]);
            }
        });
    }

    // the waves' sums, added in order: thread (tile, lane) takes the tile's place `lane`
    v4f* sums = reinterpret_cast<v4f*>(lds);
    if constexpr (FUSED) __syncthreads();
#pragma unroll
    for (int t = 0; t < RM * CN; ++t) sums[(wave * RM * CN + t) * 64 + lane] = acc[t / CN][t % CN];
    __syncthreads();
    if constexpr (!SWIGLU) {
        for (int t = wave; t < RM * CN; t += waves) {
            v4f s = sums[t * 64 + lane];
            for (int o = 1; o < waves; ++o) s += sums[(o * RM * CN + t) * 64 + lane];
            const int m = t / CN * 16 + (lane & 15), col = col0 + t % CN;
            const float v[4] = {s.x, s.y, s.z, s.w};
            if (m < g.M && col < cols) mx_put<4>(g, m, (col >> 1) * 32 + 8 * (lane >> 4) + 4 * (col & 1), g.N, v);
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
            if (g.out_type == RKH_MX4_ROWS) mx_put_rows(g, m, block, m < g.M, v, lane);
            else if (m < g.M) mx_put<8>(g, m, block * 32 + 8 * (lane >> 4), g.N, v);
        }
    }
}

// ---- tiles ---------------------------------------------------------------------------
// Tiles of 32 RM rows x 32 CN places by four waves (two by two), RM x CN accumulators each.  A step is 128 k: every operand of the tile is 1 KiB,
// copied global -> LDS directly (no registers) NBUF - 1 steps ahead, and read into registers one step ahead of its products.
// The scales of four steps are 256 bytes per operand, copied two groups ahead and read one step ahead.
//
// The copies are inline assembly (they write no register; the compiler, which would put every LDS read behind ALL copies in
// flight, does not see them), and what orders them is explicit:
//  * the copies of step s + NBUF - 1 are issued in step s, into the buffer of step s - 1: its last reads were issued in step
//    s - 2 and waited for by the first products of step s - 1, ahead of the barrier that ended it;
//  * step s reads the operands of step s + 1; the wait in front of the barrier that ends step s - 1 has left no copy of that step in
//    flight (vector memory loads complete in order, wait_for() counts what was issued since);
//  * the scales of group g + 2, issued in the first step of group g, overwrite those of group g, which were read in the last
//    step of group g - 1.
// Copies beyond the part's K bring its last step again, for the count; nothing reads them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is set and clobbered on purpose below
// 16 bytes per lane from base + off, lane-contiguous to LDS address `to`.  (A load to LDS needs a wait state behind a write of M0.)
__device__ __forceinline__ void mx_copy(const uint8_t* base, unsigned off, uint32_t to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int RM, int CN, int NBUF> struct MxTile {
    static constexpr int AB = 2 * RM, WB = 2 * CN;               // operands of a step
    static constexpr int COPIES = (AB + WB) / 4;                 // 1 KiB copies of a wave per step
    static constexpr int SCALE_COPIES = (AB + WB) / 4;           // 1 KiB copies of four operands' scales, of all waves
    static constexpr int SC = (SCALE_COPIES + 3) / 4;            // ... of a wave per group
    static constexpr int D = NBUF - 1, UNR = 8;                  // look-ahead; steps of an unrolled trip
    static constexpr int BUF = (AB + WB) * 1024, SBUF = (AB + WB) * 256;
    static constexpr int SCALES_OFF = NBUF * BUF, LDS = SCALES_OFF + 2 * SBUF;
    static_assert(RM % 2 == 0 && CN % 2 == 0 && UNR % NBUF == 0 && LDS <= 160 * 1024, "");
    // loads of a wave issued in the last `steps` steps up to step t of a trip
    static constexpr int issued(int t, int steps) {
        int n = 0;
        for (int s = 0; s < steps; ++s) n += COPIES + ((t - s + 8) % 4 == 0 ? SC : 0);
        return n;
    }
    static constexpr int wait_for(int t) { return issued(t, D - 2); } // the copies of step t + 2 have landed
    static_assert(D >= 3 && D - 2 <= 5, "a group's scales are older than what wait_for leaves in flight");
};

template <int RM, int CN, int NBUF, bool SWIGLU>
__global__ __launch_bounds__(256) void mx4_tile_kernel(rkh_mx4_gemm_args g, int mblocks, int nblocks, int parts) {
    using S = MxTile<RM, CN, NBUF>;
    static_assert(!SWIGLU || CN % 4 == 0, "gate and up halves of blocks of 32 columns in one wave");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), wm = wave & 1, wn = wave >> 1;
    const int KS = (int)rkh_mx4_ks(g.K), K4 = (int)rkh_mx4_k4(g.K);
    const int cols = (int)rkh_mx4_columns(SWIGLU ? 2 * g.N : g.N, SWIGLU) / 16, rows = (g.M + 15) / 16; // operands that exist

    // column sweeps over groups of row blocks, so that concurrently running tiles share weights in L2
    constexpr unsigned GM = 4;
    const unsigned tiles = mblocks * nblocks, job = xcd_remap(blockIdx.x, tiles * parts);
    const unsigned kpart = job / tiles, tile = job - kpart * tiles;
    const unsigned per_group = GM * nblocks, grp = tile / per_group, first_m = grp * GM, gm = min(mblocks - first_m, GM);
    const unsigned in_group = tile - grp * per_group, nblk = in_group / gm, mblk = first_m + in_group - nblk * gm;

    const int g0 = (int)((size_t)K4 * kpart / parts), g1 = (int)((size_t)K4 * (kpart + 1) / parts); // groups of 512 k
    const int ks0 = g0 * 4, steps = min(g1 * 4, KS) - ks0, groups = g1 - g0;

    // ---- sources: wave-uniform base pointers and a lane offset that advances with K
    const uint8_t *a_src[RM / 2], *w_src[CN / 2];
#pragma unroll
    for (int c = 0; c < RM / 2; ++c) a_src[c] = g.A + ((size_t)min((int)mblk * S::AB + wave * (RM / 2) + c, rows - 1) * KS + ks0) * 1024;
#pragma unroll
    for (int c = 0; c < CN / 2; ++c) w_src[c] = g.W + ((size_t)min((int)nblk * S::WB + wave * (CN / 2) + c, cols - 1) * KS + ks0) * 1024;
    const uint32_t base = (uint32_t)(uintptr_t)(mx_lds_ptr)lds;
    const uint32_t a_to = base + wave * (RM / 2) * 1024, w_to = base + (S::AB + wave * (CN / 2)) * 1024;
    // scales: copy x brings those of operands 4 x .. 4 x + 3 of the tile (activations first)
    const uint8_t* s_src[S::SC];
    unsigned s_off[S::SC];
    uint32_t s_to[S::SC];
#pragma unroll
    for (int c = 0; c < S::SC; ++c) {
        const int x = (c * 4 + wave) % S::SCALE_COPIES, op = x * 4 + (lane >> 4);
        static_assert(S::AB % 4 == 0, "a copy's operands are of one kind");
        const bool is_a = x * 4 < S::AB;
        const int first_op = is_a ? (int)mblk * S::AB : (int)nblk * S::WB, limit = (is_a ? rows : cols) - 1;
        const int at = min(first_op, limit);
        s_src[c] = (is_a ? g.a_scale : g.w_scale) + ((size_t)at * K4 + g0) * 256;
        s_off[c] = (unsigned)(min(first_op + op - (is_a ? 0 : S::AB), limit) - at) * (unsigned)K4 * 256 + (lane & 15) * 16;
        s_to[c] = base + S::SCALES_OFF + x * 1024;
    }

    v4f acc[RM][CN];
    v4i a[2][RM], w[2][CN];
    uint32_t as[2][RM], ws[2][CN];
    const uint8_t* a_at = lds + wm * RM * 1024 + lane * 16;
    const uint8_t* w_at = lds + (S::AB + wn * CN) * 1024 + lane * 16;
    const uint8_t* as_at = lds + S::SCALES_OFF + wm * RM * 256 + lane * 4;
    const uint8_t* ws_at = lds + S::SCALES_OFF + (S::AB + wn * CN) * 256 + lane * 4;

    int ahead = 0; // next step to copy
    unsigned k_off = lane * 16;
    const auto copy = [&](auto buf_tag, auto c_tag) {
        constexpr int B = decltype(buf_tag)::value % NBUF, C = decltype(c_tag)::value;
        if constexpr (C < RM / 2) mx_copy(a_src[C], k_off, a_to + B * S::BUF + C * 1024);
        else mx_copy(w_src[C - RM / 2], k_off, w_to + B * S::BUF + (C - RM / 2) * 1024);
        if constexpr (C == S::COPIES - 1) {
            ++ahead;
            k_off += ahead < steps ? 1024u : 0u;
        }
    };
    int s_ahead = 0; // next group whose scales are to be copied
    const auto copy_scales = [&](auto half_tag) {
#pragma unroll
        for (int c = 0; c < S::SC; ++c) mx_copy(s_src[c], s_off[c] + (unsigned)min(s_ahead, groups - 1) * 256, s_to[c] + decltype(half_tag)::value * S::SBUF);
        ++s_ahead;
    };
    // item Y of what step T reads for the next one: weights, activations, then (from the first step of a group) scales
    const auto read = [&](auto t_tag, auto y_tag) {
        constexpr int T = decltype(t_tag)::value, Y = decltype(y_tag)::value, B = T % NBUF, P = T & 1, H = (T / 4) & 1;
        if constexpr (Y < CN) w[P][Y] = *reinterpret_cast<const v4i*>(w_at + B * S::BUF + Y * 1024);
        else if constexpr (Y < CN + RM) a[P][Y - CN] = *reinterpret_cast<const v4i*>(a_at + B * S::BUF + (Y - CN) * 1024);
        else if constexpr (Y < 2 * CN + RM) ws[H][Y - CN - RM] = *reinterpret_cast<const uint32_t*>(ws_at + H * S::SBUF + (Y - CN - RM) * 256);
        else as[H][Y - 2 * CN - RM] = *reinterpret_cast<const uint32_t*>(as_at + H * S::SBUF + (Y - 2 * CN - RM) * 256);
    };

    // ---- prologue
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    copy_scales(C0{});
    static_for<2>([&](auto b) { static_for<S::COPIES>([&](auto c) { copy(b, c); }); });
    copy_scales(C1{});
    static_for<S::D - 2>([&](auto b) { static_for<S::COPIES>([&](auto c) { copy(std::integral_constant<int, decltype(b)::value + 2>{}, c); }); });
#pragma unroll
    for (int t = 0; t < RM * CN; ++t) acc[t / CN][t % CN] = v4f{0, 0, 0, 0};
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S::D - 2) * S::COPIES) : "memory"); // steps 0 and 1, both groups of scales
    static_for<2 * (RM + CN)>([&](auto y) { read(C0{}, y); });

    const auto step = [&](auto t_tag) {
        constexpr int T = decltype(t_tag)::value, P = T & 1, H = (T / 4) & 1, MF = RM * CN;
        using Next = std::integral_constant<int, (T + 1) % S::UNR>;
        constexpr int READS = (RM + CN) * (T % 4 == 3 ? 2 : 1), COPIES = S::COPIES, ITEMS = READS + COPIES;
        if constexpr (T % 4 == 0) copy_scales(std::integral_constant<int, H>{});
        static_for<MF>([&](auto x_tag) {
            constexpr int X = decltype(x_tag)::value, I = X / CN, J = I & 1 ? CN - 1 - X % CN : X % CN;
            acc[I][J] = mx_mfma<T % 4>(w[P][J], a[P][I], acc[I][J], ws[H][J], as[H][I]);
            constexpr int FROM = X * ITEMS / MF, TO = (X + 1) * ITEMS / MF;
            static_for<TO - FROM>([&](auto z_tag) {
                constexpr int Z = FROM + decltype(z_tag)::value;
                // copies and reads in turn while there are copies
                if constexpr (Z < 2 * COPIES && (Z & 1) == 0) copy(std::integral_constant<int, T + S::D>{}, std::integral_constant<int, Z / 2>{});
                else read(Next{}, std::integral_constant<int, (Z < 2 * COPIES ? Z / 2 : Z - COPIES)>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::wait_for(T)) : "memory");
    };
    for (int s = 0; s < steps; s += S::UNR)
        static_while<S::UNR>([&](auto t) {
            if (s + decltype(t)::value >= steps) return false;
            step(t);
            return true;
        });
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // a load to LDS must not outlive the workgroup

    // ---- epilogue
    const int m_first = ((int)mblk * 2 + wm) * RM * 16 + (lane & 15), col_first = ((int)nblk * 2 + wn) * CN;
    if (parts > 1) { // partial tile in accumulator order: [tile][part][wave][tile of 16 x 16][lane]
        v4f* to = reinterpret_cast<v4f*>(g.scratch) + (((size_t)tile * parts + kpart) * 4 + wave) * (RM * CN * 64) + lane;
#pragma unroll
        for (int t = 0; t < RM * CN; ++t) to[t * 64] = acc[t / CN][t % CN];
        return;
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int m = m_first + i * 16;
        if constexpr (SWIGLU) {
#pragma unroll
            for (int j = 0; j < CN; j += 4) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = mx_silu(acc[i][j + (e >> 2)][e & 3], acc[i][j + 2 + (e >> 2)][e & 3]);
                const int block = (col_first + j) / 4;
                const bool live = m < g.M && block * 32 < g.N;
                if (g.out_type == RKH_MX4_ROWS) mx_put_rows(g, m, block, live, v, lane);
                else if (live) mx_put<8>(g, m, block * 32 + 8 * (lane >> 4), g.N, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < CN; j += 2) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][j + (e >> 2)][e & 3];
                if (m < g.M) mx_put<8>(g, m, (col_first + j) * 16 + 8 * (lane >> 4), g.N, v);
            }
        }
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
    constexpr unsigned GM = 4;
    const unsigned per_group = GM * nblocks, grp = tile / per_group, first_m = grp * GM, gm = min(mblocks - first_m, GM);
    const unsigned in_group = tile - grp * per_group, nblk = in_group / gm, mblk = first_m + in_group - nblk * gm;
    const int m = (((int)mblk * 2 + (wave & 1)) * RM + i) * 16 + (lane & 15), col = ((int)nblk * 2 + (wave >> 1)) * CN + j;

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
        else if (live) mx_put<8>(g, m, block * 32 + 8 * (lane >> 4), g.N, v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s[e >> 2][e & 3];
        if (m < g.M) mx_put<8>(g, m, col * 16 + 8 * (lane >> 4), g.N, v);
    }
}

// ---- which kernel ------------------------------------------------------------------
struct MxRoute {
    bool few;
    int rm, cn, parts, mblocks, nblocks; // few: 16 rm rows, 16 cn places of a workgroup
};

constexpr int MX_CUS = 256; // compute units that a launch is cut for

MxRoute mx_route(int M, int N, int K, int swiglu) {
    const int64_t cols = rkh_mx4_columns(swiglu ? 2 * (int64_t)N : N, swiglu) / 16, K4 = rkh_mx4_k4(K);
    MxRoute r{};
    r.parts = 1;
    if (M <= (swiglu ? 32 : 64)) {
        r.few = true;
        r.rm = M <= 16 ? 1 : M <= 32 ? 2 : 4;
        r.cn = swiglu ? 4 : cols <= 4 * MX_CUS || r.rm == 4 ? 1 : 2;
        r.mblocks = 1;
        r.nblocks = (int)((cols + r.cn - 1) / r.cn);
        return r;
    }
    static constexpr int SHAPES[][2] = {{8, 4}, {4, 4}, {2, 4}};
    for (const auto& s : SHAPES) {
        r.rm = s[0], r.cn = s[1];
        r.mblocks = (M + 32 * r.rm - 1) / (32 * r.rm);
        r.nblocks = (int)((cols + 2 * r.cn - 1) / (2 * r.cn));
        if ((int64_t)r.mblocks * r.nblocks >= MX_CUS * 3 / 4) break;
    }
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
    if (tiles < MX_CUS * 3 / 4) {
        int64_t parts = MX_CUS / tiles;
        if (parts > K4 / 2) parts = K4 / 2;
        r.parts = parts < 1 ? 1 : (int)parts;
    }
    return r;
}
size_t mx_scratch(const MxRoute& r) { return r.few || r.parts == 1 ? 0 : (size_t)r.mblocks * r.nblocks * r.parts * r.rm * r.cn * 4096; }

template <int RM, int CN, int MAX_WAVES, bool SWIGLU, bool FUSED>
int launch_few(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    const int K4 = (int)rkh_mx4_k4(g.K), per = (K4 + MAX_WAVES - 1) / MAX_WAVES, waves = (K4 + per - 1) / per;
    const size_t sums = (size_t)waves * RM * CN * 1024, rows = FUSED ? (size_t)rkh_mx4_ks(g.K) * 4 * g.M * 16 + (size_t)K4 * g.M * 16 : 0;
    const size_t bytes = sums > rows ? sums : rows;
    static std::atomic<int> ready{0};
    if (!ready.load()) {
        RKH_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&mx4_few_kernel<RM, CN, MAX_WAVES, SWIGLU, FUSED>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
        ready.store(1);
    }
    mark(st, "mx4_few_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_few_kernel<RM, CN, MAX_WAVES, SWIGLU, FUSED>), dim3(r.nblocks), dim3(waves * 64), bytes, st, g, per);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

template <int RM, int CN, int NBUF, bool SWIGLU> int launch_tiles(hipStream_t st, const rkh_mx4_gemm_args& g, const MxRoute& r) {
    constexpr int LDS = MxTile<RM, CN, NBUF>::LDS;
    static std::atomic<int> ready{0};
    if (!ready.load()) {
        RKH_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(&mx4_tile_kernel<RM, CN, NBUF, SWIGLU>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        ready.store(1);
    }
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
    if (tiles * r.parts > 0x7fffffff) return RKH_ERR_RUNTIME;
    mark(st, "mx4_tile_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(mx4_tile_kernel<RM, CN, NBUF, SWIGLU>), dim3((unsigned)(tiles * r.parts)), dim3(256), LDS, st, g, r.mblocks,
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

template <bool SWIGLU> int launch(hipStream_t st, const rkh_mx4_gemm_args& g) {
    MxRoute r = mx_route(g.M, g.N, g.K, SWIGLU);
    if (r.few) {
        if (!g.A) {
            if constexpr (SWIGLU) return launch_few<1, 4, 8, true, true>(st, g, r);
            else return r.cn == 1 ? launch_few<1, 1, 16, false, true>(st, g, r) : launch_few<1, 2, 16, false, true>(st, g, r);
        }
        if constexpr (SWIGLU) {
            if (r.rm == 1) return launch_few<1, 4, 8, true, false>(st, g, r);
            return launch_few<2, 4, 8, true, false>(st, g, r);
        } else {
            if (r.rm == 1) return r.cn == 1 ? launch_few<1, 1, 16, false, false>(st, g, r) : launch_few<1, 2, 16, false, false>(st, g, r);
            if (r.rm == 2) return r.cn == 1 ? launch_few<2, 1, 16, false, false>(st, g, r) : launch_few<2, 2, 8, false, false>(st, g, r);
            return launch_few<4, 1, 8, false, false>(st, g, r);
        }
    }
    if (mx_scratch(r) > (g.scratch ? g.scratch_bytes : 0)) r.parts = 1;
    if (r.rm == 8) return launch_tiles<8, 4, 4, SWIGLU>(st, g, r);
    return r.rm == 4 ? launch_tiles<4, 4, 4, SWIGLU>(st, g, r) : launch_tiles<2, 4, 8, SWIGLU>(st, g, r);
}

} // namespace

extern "C" {

int rkh_mx4_gemm(void* stream, const rkh_mx4_gemm_args* args) {
    if (!args->M || !args->N) return RKH_OK;
    if (!args->A && !rkh_mx4_takes_rows(args->M, args->N, args->K, args->swiglu)) return RKH_ERR_RUNTIME;
    return args->swiglu ? launch<true>((hipStream_t)stream, *args) : launch<false>((hipStream_t)stream, *args);
}
int rkh_mx4_takes_rows(int M, int N, int K, int swiglu) {
    (void)N, (void)swiglu;
    return M <= 4 && rkh_mx4_ks(K) * 4 * M * 16 + rkh_mx4_k4(K) * M * 16 <= FEW_FUSED_LDS;
}
void rkh_mx4_route(int M, int N, int K, int swiglu, int* kernel, int* rows, int* columns, int* parts) {
    const MxRoute r = mx_route(M, N, K, swiglu);
    *kernel = r.few ? 0 : 1;
    *rows = r.few ? 16 * r.rm : 32 * r.rm;
    *columns = r.few ? 16 * r.cn : 32 * r.cn;
    *parts = r.parts;
}
size_t rkh_mx4_scratch_bytes(int M, int N, int K, int swiglu) { return mx_scratch(mx_route(M, N, K, swiglu)); }

} // extern "C"
