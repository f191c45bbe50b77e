// Group-scaled 4-bit (G4) layers: weights laid out, rows staged for the tiles, products of few rows, and which kernel takes a product.
//
// C[m, n] = sum over groups of scale[n, g] * (sum over k in g of (code - zero) * x[m, k]).  Codes and code - zero are small integers and exact in 16 bits, so the
// matrix cores' products with 16-bit activations are exact and their sums have 32 bits; the scales multiply sums, and no weight is rounded.  What is multiplied:
//   fp16 rows, as many as there are: code - zero.
//   bf16 rows, up to 16: the code; the zero point times the group's sum of activations is taken off the group's sum.  Both have 32 bits, so the roundings of terms
//   (code + zero) |x| stay, also where code and zero are equal.
//   bf16 rows, more: code - zero, with the row as halves (g4_stage_kernel), which is the row itself down to 2^-31 of its largest value.
#include <algorithm>

#include "rk_kernels_g4.h"

namespace {

// ---- weights -----------------------------------------------------------------------
// One workgroup for up to PACK_PIECES pieces of 16 places, a thread for a dword of each: rows are read 256 bytes at a time.  14336 x 4096: 20 us (a byte and a division at a time: 99).
constexpr int PACK_PIECES = 4;
__global__ __launch_bounds__(256) void g4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int K, int N, int group, int groups, int gpb,
                                                      int gate_up, uint32_t* dst, uint32_t* dst_scales, size_t first) {
    typedef uint32_t word_any __attribute__((aligned(1)));
    const int KB = (int)rkh_g4_kb(K), spans = (KB + PACK_PIECES - 1) / PACK_PIECES, half_rows = (K + 1) / 2, F = gate_up ? N / 2 : N, tid = threadIdx.x;
    const int64_t block = (int64_t)((first + blockIdx.x) / spans);
    const int kb0 = (int)(first + blockIdx.x - (size_t)block * spans) * PACK_PIECES;
    const auto column = [&](int c) -> int64_t { // in the matrix given, or -1
        const int64_t n = g4_column(block, c, gate_up != 0);
        return n < F ? n + (gate_up && (block & 1) ? F : 0) : -1;
    };
    const int lane = tid >> 2, step = tid & 3, c = lane & 15;
    const int64_t n = column(c);
    const uint8_t* row = codes + (size_t)max(n, (int64_t)0) * half_rows;
    uint32_t raw[PACK_PIECES];
#pragma unroll
    for (int p = 0; p < PACK_PIECES; ++p) {
        const int k = (kb0 + p) * 128 + step * 32 + (lane >> 4) * 8;
        raw[p] = 0;
        if (n < 0 || k >= K) continue;
        if (k + 8 <= K) {
            raw[p] = *reinterpret_cast<const word_any*>(row + (k >> 1));
        } else {
            for (int t = 0; t < K - k; ++t) raw[p] |= (uint32_t)(row[(k + t) >> 1] >> (4 * (t & 1)) & 15) << (4 * t); // (k is even)
        }
    }
#pragma unroll
    for (int p = 0; p < PACK_PIECES; ++p) {
        if (kb0 + p >= KB) break;
        const auto gather = [](uint32_t w) { // the low halves of four bytes one behind the other
            w &= 0x0f0f0f0fu;
            w = (w | w >> 4) & 0x00ff00ffu;
            return (w | w >> 8) & 0xffffu;
        };
        dst[((size_t)block * KB + kb0 + p) * 256 + tid] = gather(raw[p]) | gather(raw[p] >> 4) << 16;
    }
    for (int i = tid; i < 16 * gpb * min(PACK_PIECES, KB - kb0); i += 256) {
        const int at = i / gpb, kb = kb0 + (at >> 4), k = kb * 128 + (i - at * gpb) * (128 / gpb);
        const int64_t n = column(at & 15);
        uint32_t d = 0x6400u;
        if (n >= 0 && k < K) {
            const size_t from = (size_t)n * groups + k / group;
            d = (uint32_t)scales[from] << 16 | (0x6400u + (zeros ? zeros[from] : 8u));
        }
        dst_scales[((size_t)block * KB + kb0) * 16 * gpb + i] = d;
    }
}

// ---- rows for the tiles ---------------------------------------------------------------
// One workgroup per row, or a wave (ROWS = 4) where rows are short: 2457 x 768 with SwiGLU behind it 21.6 -> 19.1 us.
// bf16: the row's largest finite magnitude is moved to 2^14 .. 2^15.  A half's smallest step is 2^-24, where the eight bits of a value of 2^-17 end, so all that is 2^-31 of the
// largest or more stays as it is.  What is smaller is rounded to a multiple of 2^-24, by 2^-25 or 2^-39 of the largest at most.  (As bf16, code - zero would take
// twice the instructions, which are what tiles are bound by.)  Infinities and NaN stay what they are.
template <bool BF16, int ROWS>
__global__ __launch_bounds__(256) void g4_stage_kernel(const uint16_t* x, int64_t ldx, int M, int K, uint16_t* staged, int* exponents, int first) {
    constexpr int THREADS = 256 / ROWS, STRIDE = THREADS * 8; // of a row
    const int tid = threadIdx.x % THREADS, m = first + blockIdx.x * ROWS + threadIdx.x / THREADS, Kp = (int)rkh_g4_kb(K) * 128;
    if (m >= M) return; // (whole waves, and the last workgroup where a row has one)
    const uint16_t* row = x + (size_t)m * ldx;
    uint16_t* to = staged + (size_t)m * Kp;
    const auto fetch = [&](int k) { return k + 8 <= K ? mx_fetch8<RKH_MX4_F16>(row, k) : mx_fetch_some<RKH_MX4_F16>(row, k, K - k); };
    if constexpr (!BF16) {
        for (int k = tid * 8; k < Kp; k += STRIDE) *reinterpret_cast<v4i*>(to + k) = fetch(k).w[0];
    } else {
        constexpr int AHEAD = 4; // 32 values a thread in registers; what is beyond is read twice
        v4i raw[AHEAD];
        uint32_t top = 0;
        const auto look = [&](const v4i& r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t lo = (uint32_t)r[e] << 16 & 0x7fff0000u, hi = (uint32_t)r[e] & 0x7fff0000u;
                if (lo < 0x7f800000u) top = max(top, lo);
                if (hi < 0x7f800000u) top = max(top, hi);
            }
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = tid * 8 + u * STRIDE;
            raw[u] = k < Kp ? fetch(k).w[0] : v4i{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) look(raw[u]);
        for (int k = tid * 8 + AHEAD * STRIDE; k < Kp; k += STRIDE) look(fetch(k).w[0]);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
        if constexpr (ROWS == 1) {
            __shared__ uint32_t part[4];
            if (lane_id() == 0) part[wave_id()] = top;
            __syncthreads();
            top = max(max(part[0], part[1]), max(part[2], part[3]));
        }
        // 2^e: from the exponent of the largest to 14 (of numbers below the normal ones the largest has 127 places to go at least)
        const int e = top ? 14 + 127 - (int)max(top >> 23, 1u) : 0;
        if (tid == 0) exponents[m] = -e;
        const auto put = [&](int k, const v4i& r) {
            v8h h;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                h[2 * i] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float((uint32_t)r[i] << 16), e);
                h[2 * i + 1] = (_Float16)__builtin_amdgcn_ldexpf(__uint_as_float((uint32_t)r[i] & 0xffff0000u), e);
            }
            *reinterpret_cast<v8h*>(to + k) = h;
        };
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (tid * 8 + u * STRIDE < Kp) put(tid * 8 + u * STRIDE, raw[u]);
        for (int k = tid * 8 + AHEAD * STRIDE; k < Kp; k += STRIDE) put(k, fetch(k).w[0]);
    }
}

// ---- few rows ------------------------------------------------------------------------
// One workgroup multiplies up to 16 rows with 16 CN places; its waves split K into pieces of 128 and are summed through LDS.  Codes go straight into
// registers, once; so do activations, which every workgroup reads for itself.
// ROWS (1, 4, 8 or 16): up to so many rows.  A wave loads a row's 512 values together and turns them into operands through LDS of its own.  0: up to 16 rows,
// loaded as the operands lie.
// One row is bound by the weights' way from HBM (1 x 14336 x 4096 7.2 us where caches help, 7.8 to 8.1 where they do not: 3.8 TB/s, where a launch that only reads takes 5.9),
// more rows by the activations' from L2 as well (8 x 4096 x 14336 8.9, 11.1).
// fp16 rows are multiplied with code - zero.  bf16 rows with the code, and the zero point times the group's sum of activations, which a product with ones gives, is taken off
// a group's sum: bf16 has no packed additions, so that code - zero takes 17 instructions for eight weights by way of fp32, not 7, and one row x 14336 x 4096
// 8.7 us and not 7.8, SwiGLU of it 15.2 and not 13.1, 8 x 4096 x 14336 11.6 and not 11.1.
constexpr int FEW_PITCH = 1024 + 16; // bytes of a row of 512 values in LDS
constexpr int few_area(int rows, int cn) { return rows * FEW_PITCH > cn * 1024 ? rows * FEW_PITCH : cn * 1024; }

template <int TYPE, int CN, int GPB, int ROWS, bool SWIGLU, bool LONG, int NP, int MAX_WAVES>
__global__ __launch_bounds__(MAX_WAVES * 64) void g4_few_kernel(const uint8_t* W, const uint32_t* scales, const uint16_t* x, int64_t ldx, int M, int K,
                                                                int per_wave, int workgroups, int waves, rkh_g4_args g) {
    constexpr bool HALVES = TYPE == RKH_MX4_F16;
    constexpr int ONE = 0x3f803f80; // two of bf16
    constexpr int STEPS = 4 / GPB; // 32-k steps of a group
    static_assert(!SWIGLU || CN % 2 == 0, "gate and up halves");
    static_assert(!ROWS || NP % 4 == 0, "rows are loaded 512 values at a time");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c = lane & 15, q = lane >> 4;
    const int KB = (int)rkh_g4_kb(K);
    const int block0 = xcd_remap(blockIdx.x, workgroups) * CN;
    const int first = wave * per_wave, last = min(first + per_wave, KB);
    const int row = min(c, M - 1); // (operand rows beyond M: the last one again, whose results nobody takes)
    typedef uint32_t words __attribute__((ext_vector_type(GPB)));

    struct Batch {
        v4i w[NP][CN], x[ROWS ? ROWS * NP / 4 : NP * 4];
        words s[NP][CN];
    };
    // (What lies beyond K, eight at least, is loaded from a row's last eight values and dropped where it is used: a branch here would wait for the activations
    // ahead of the codes' loads.)
    const auto fetch = [&](int m, int k) { return mx_fetch8<TYPE>(x, (size_t)m * ldx + min(k, K - 8)).w[0]; };
    const auto within = [&](const v4i& v, int k) { return k < K ? HALVES ? v : g4_turned_rows(v) : v4i{0, 0, 0, 0}; };
    // Where K ends within eight values: the last eight to their places, by four values, by two and by one.  (A 64-bit shift by a register reads a pair of registers
    // for the amount; where that is the last one a wave has, it reads v0 instead: rows of 4140 values were shifted by the lane's number.  audit_waits looks for these.)
    const auto moved = [&](v4i v, int k) {
        const int beyond = k < K ? max(k + 8 - K, 0) : 0;
        const bool four = beyond & 4, two = beyond & 2;
        v = v4i{four ? v.z : v.x, four ? v.w : v.y, four ? 0 : v.z, four ? 0 : v.w};
        v = v4i{two ? v.y : v.x, two ? v.z : v.y, two ? v.w : v.z, two ? 0 : v.w};
        const uint32_t bits = (beyond & 1) * 16;
        return v4i{(int)__builtin_amdgcn_alignbit((uint32_t)v.y, (uint32_t)v.x, bits), (int)__builtin_amdgcn_alignbit((uint32_t)v.z, (uint32_t)v.y, bits),
                   (int)__builtin_amdgcn_alignbit((uint32_t)v.w, (uint32_t)v.z, bits), (int)((uint32_t)v.w >> bits)};
    };
    const auto load = [&](Batch& b, int from) { // (pieces beyond the last: that one again, which is not multiplied)
        if constexpr (ROWS) {
#pragma unroll
            for (int m = 0; m < ROWS * NP / 4; ++m) b.x[m] = fetch(min(m % ROWS, M - 1), (from + m / ROWS * 4) * 128 + lane * 8);
        } else {
#pragma unroll
            for (int i = 0; i < NP * 4; ++i) b.x[i] = fetch(row, from * 128 + i * 32 + q * 8);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int kb = min(from + p, KB - 1);
#pragma unroll
            for (int j = 0; j < CN; ++j) {
                b.w[p][j] = *reinterpret_cast<const v4i*>(W + ((size_t)(block0 + j) * KB + kb) * 1024 + lane * 16);
                b.s[p][j] = *reinterpret_cast<const words*>(scales + (((size_t)(block0 + j) * KB + kb) * 16 + c) * GPB);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto product = [](const v4i& rows, const v4i& codes, const v4f& sum) {
        if constexpr (TYPE == RKH_MX4_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, rows), __builtin_bit_cast(v8h, codes), sum, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, rows), __builtin_bit_cast(v8b, codes), sum, 0, 0, 0);
    };
    const uint32_t exponents = g4_exponents();
    v4f acc[CN];
#pragma unroll
    for (int j = 0; j < CN; ++j) acc[j] = v4f{0, 0, 0, 0};
    constexpr int AREA = few_area(ROWS, CN); // a wave's part of LDS: its activations, and in the end its sums
    uint8_t* own = lds + wave * AREA;
    const auto multiply = [&](const Batch& b, int from) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            if (from + p >= last) break;
            if constexpr (ROWS) {
                if (p % 4 == 0) {
                    __builtin_amdgcn_wave_barrier(); // (a wave's LDS operations complete in order)
#pragma unroll
                    for (int m = 0; m < ROWS; ++m)
                        *reinterpret_cast<v4i*>(own + m * FEW_PITCH + lane * 16) = within(b.x[p / 4 * ROWS + m], (from + p) * 128 + lane * 8);
                    __builtin_amdgcn_wave_barrier();
                }
            }
#pragma unroll
            for (int n = 0; n < GPB; ++n) {
                v4i a[4];
#pragma unroll
                for (int i = n * STEPS; i < (n + 1) * STEPS; ++i) {
                    if constexpr (ROWS) a[i] = *reinterpret_cast<const v4i*>(own + row * FEW_PITCH + (p & 3) * 256 + i * 64 + q * 16);
                    else a[i] = within(b.x[p * 4 + i], (from + p) * 128 + i * 32 + q * 8);
                }
                v4f sum = {0, 0, 0, 0};
                if constexpr (!HALVES) {
#pragma unroll
                    for (int i = n * STEPS; i < (n + 1) * STEPS; ++i) sum = product(a[i], v4i{ONE, ONE, ONE, ONE}, sum);
                }
#pragma unroll
                for (int j = 0; j < CN; ++j) {
                    const uint32_t d = b.s[p][j][n];
                    const float s = g4_scale(d, g.scale_type);
                    v4f part = {0, 0, 0, 0};
                    if constexpr (HALVES) {
                        G4Zero zero;
                        zero.of(d);
#pragma unroll
                        for (int i = n * STEPS; i < (n + 1) * STEPS; ++i) part = product(a[i], g4_halves((uint32_t)b.w[p][j][i], zero, exponents), part);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(part[e], s, acc[j][e]);
                    } else {
                        const float zero = (float)(d & 0xffu);
#pragma unroll
                        for (int i = n * STEPS; i < (n + 1) * STEPS; ++i) part = product(a[i], g4_codes((uint32_t)b.w[p][j][i]), part);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(fmaf(-zero, sum[e], part[e]), s, acc[j][e]);
                    }
                }
            }
        }
    };
    // LONG: a wave has more pieces than it loads together.  (One batch of registers: other waves' loads are on their way meanwhile.  With the next batch's loads
    // ahead of the products, which leaves room for half of the waves, 1 x 11008 x 14336 took 23.6 us, this way 17.7, and 8 x 4096 x 14336 10.3, 8.9.  Written
    // as a loop where there is one batch, the kernel has ten registers more: SwiGLU of 1 x 14336 x 4096 13.2 -> 14.1.)
    for (int from = first;;) {
        Batch b;
        load(b, from);
        if (ROWS < 16 && K % 8 && (from + NP) * 128 > K) { // (of sixteen rows it costs the loads' order 1.4 us of 12.3: those are staged)
            if constexpr (ROWS) {
#pragma unroll
                for (int m = 0; m < ROWS * NP / 4; ++m) b.x[m] = moved(b.x[m], (from + m / ROWS * 4) * 128 + lane * 8);
            } else {
#pragma unroll
                for (int i = 0; i < NP * 4; ++i) b.x[i] = moved(b.x[i], from * 128 + i * 32 + q * 8);
            }
        }
        multiply(b, from);
        if (!LONG || (from += NP) >= last) break;
    }

    // the waves' sums, added in order: a thread takes one result (SwiGLU: both halves of one)
#pragma unroll
    for (int j = 0; j < CN; ++j) *reinterpret_cast<v4f*>(own + j * 1024 + lane * 16) = acc[j];
    __syncthreads();
    const auto total = [&](int i) {
        const float* from = reinterpret_cast<const float*>(lds) + i;
        float s = *from;
#pragma unroll 4
        for (int o = 1; o < waves; ++o) s += from[o * (AREA / 4)];
        return s;
    };
    for (int i = threadIdx.x; i < (SWIGLU ? CN / 2 : CN) * 256; i += waves * 64) {
        const int m = (i >> 6 & 3) * 4 + (i & 3), at = SWIGLU ? (i >> 8) * 512 + (i & 255) : i;
        if (m >= M) continue;
        const int ex = g.exponents ? g.exponents[m] : 0;
        const float a = __builtin_amdgcn_ldexpf(total(at), ex);
        const float v = SWIGLU ? mx_silu(a, __builtin_amdgcn_ldexpf(total(at + 256), ex)) : a;
        g4_put(g, m, g4_column(block0 + (at >> 8), i >> 2 & 15, SWIGLU), v);
    }
}

constexpr int FEW_ROWS = 16;
constexpr int G4_CUS = 256; // compute units that a launch is cut for

// What a workgroup of the few-row kernel takes.  Where both sides were measured (fp16, one scale in 128, the weights of four layers in turn, us):
//   rows at a time as they are in LDS, or as operands (ROWS 0) with 64 columns a workgroup, where there are columns for that: 16 rows x 8192 columns x K = 4096
//   10.7 and 7.8, x 8192 13.5 and 13.7; x 11008 columns x 14336 33.3 and 27.8; 8 rows x 14336 x 8192 14.9 and 13.0, x 8192 x 8192 9.1 and 11.6; 4 rows x 14336
//   x 14336 26.0 and 22.8, x 8192 12.2 and 12.5;
//   waves, where there are more workgroups than compute units and several share one: 8 rows x 8192 x 8192 16 waves 10.2, 8 9.1, 4 10.8; 16 rows x 6144 x 14336
//   8 waves 21.5, 4 18.0; 4 rows x 8192 x 14336 16 waves 12.1, 8 13.1; 1 row of it with groups of 32 18.6,
//   16.1; where there are not: 8 rows x 4096 x 14336 16 waves 8.8, 8 9.4, 4 10.8;
//   columns of four rows: x 14336 x 4096 16 columns 9.0, 32 8.3, x 4096 x 4096 4.4 and 4.7;
//   K in parts, which takes a second launch: 8 x 4096 x 14336 8.8 -> 12 at best.
struct FewShape {
    int rows, cn, most; // LDS rows of a wave (0: none), blocks of 16 places, most waves
};
// (more than eight waves leave 128 registers for a lane, which is too few for two blocks or many groups and rows at once)
FewShape few_shape(int M, int64_t blocks, int KB, int gpb, bool swiglu) {
    if ((M > 4 && blocks >= 640) || (M > 8 && blocks >= 512 && KB <= 32) || (M > 1 && blocks >= 768 && KB > 64)) return {0, 4, gpb == 4 ? 8 : 16};
    const int rows = M == 1 ? 1 : M <= 4 ? 4 : M <= 8 ? 8 : 16;
    const int cn = swiglu || (rows == 4 && blocks >= 768 && KB <= 32) ? 2 : 1;
    const bool shared = blocks / cn > G4_CUS;
    return {rows, cn, rows == 16 ? shared ? 4 : 8 : cn == 2 || (shared && (rows == 8 || gpb == 4)) || (rows == 8 && gpb == 4) ? 8 : 16};
}

// ... and its waves: pieces of K that one loads together, and has in all.
struct FewPlan {
    FewShape shape;
    int together, per, waves;
};
FewPlan few_plan(int M, int64_t blocks, int KB, int gpb, bool swiglu) {
    const FewShape shape = few_shape(M, blocks, KB, gpb, swiglu);
    // pieces of a wave: up to four (as operands: two) that are loaded together, eight waves where they go round, and as many as there are waves for
    const int together = shape.rows ? 4 : 2, per = std::max((KB + shape.most - 1) / shape.most, std::min(together, (KB + 7) / 8));
    return {shape, together, per, (KB + per - 1) / per};
}

template <int TYPE, int CN, int GPB, int ROWS, bool SWIGLU, bool LONG, int NP, int MAX_WAVES> int launch_few(hipStream_t st, const rkh_g4_args& g, const FewPlan& plan) {
    const int per = plan.per, waves = plan.waves;
    const int64_t workgroups = rkh_g4_places(SWIGLU ? 2 * (int64_t)g.N : g.N, SWIGLU) / (16 * CN);
    if (workgroups * waves * 64 >= MX_TOO_MANY_THREADS) return RKH_ERR_RUNTIME;
    constexpr size_t BYTES = few_area(ROWS, CN); // of a wave
    static_assert(MAX_WAVES * BYTES <= 160 * 1024, "");
    const auto kernel = g4_few_kernel<TYPE, CN, GPB, ROWS, SWIGLU, LONG, NP, MAX_WAVES>;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(kernel), opted_in, 160 * 1024)) return rc;
    mark(st, "g4_few_kernel");
    hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups), dim3(waves * 64), waves * BYTES, st, g.W, g.w_scale, static_cast<const uint16_t*>(g.x), g.ldx, g.M, g.K,
                       per, (int)workgroups, waves, g);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}
template <int TYPE, int GPB, bool SWIGLU> int launch_few(hipStream_t st, const rkh_g4_args& g) {
    const FewPlan plan = few_plan(g.M, rkh_g4_places(SWIGLU ? 2 * (int64_t)g.N : g.N, SWIGLU) / 16, (int)rkh_g4_kb(g.K), GPB, SWIGLU);
    const FewShape& shape = plan.shape;
    const auto go = [&](auto is_long) {
        constexpr bool LONG = decltype(is_long)::value;
        if (!shape.rows) return launch_few<TYPE, 4, GPB, 0, SWIGLU, LONG, 2, GPB == 4 ? 8 : 16>(st, g, plan);
        constexpr int CN = SWIGLU ? 2 : 1, MOST = SWIGLU ? 8 : 16;
        if (shape.rows == 1) return launch_few<TYPE, CN, GPB, 1, SWIGLU, LONG, 4, MOST>(st, g, plan);
        if constexpr (!SWIGLU && !LONG) {
            if (shape.cn == 2) return launch_few<TYPE, 2, GPB, 4, SWIGLU, LONG, 4, 8>(st, g, plan);
        }
        if (shape.rows == 4) return launch_few<TYPE, CN, GPB, 4, SWIGLU, LONG, 4, MOST>(st, g, plan);
        if (shape.rows == 8) return launch_few<TYPE, CN, GPB, 8, SWIGLU, LONG, 4, GPB == 4 ? 8 : MOST>(st, g, plan);
        return launch_few<TYPE, CN, GPB, 16, SWIGLU, LONG, 4, 8>(st, g, plan);
    };
    return plan.per > plan.together ? go(std::true_type{}) : go(std::false_type{});
}
template <int TYPE> int launch_few(hipStream_t st, const rkh_g4_args& g) {
    if (g.swiglu) return g.gpb == 1 ? launch_few<TYPE, 1, true>(st, g) : g.gpb == 2 ? launch_few<TYPE, 2, true>(st, g) : launch_few<TYPE, 4, true>(st, g);
    return g.gpb == 1 ? launch_few<TYPE, 1, false>(st, g) : g.gpb == 2 ? launch_few<TYPE, 2, false>(st, g) : launch_few<TYPE, 4, false>(st, g);
}

// ---- which kernel ------------------------------------------------------------------
// Tiles of 32 rm rows x 128 places: us of a step of 128 k where up to half of the compute units have a tile, where all have one, and, for tiles of which two share a
// unit, where few and where all have two.  (What all units do at once they do slower.)  From products of K = 4096 and groups of 128, us, with 32, 64, 128 and 256 rows:
//   128 x 8192 15.7 19.7 28.5;  x 11008 23.7 20.3 28.7;  x 28672 49.8 39.9 39.4;  256 x 4096 15.7 19.5 29.3 48;  x 5504 23.9 20.3 29.6;  x 8192 27.4 22.8 29.7 48.1;
//   512 x 8192 51.6 40.5 39.8 48.8;  x 11008 72.1 57.2 67.6 54.2;  x 14336 87.5 73.2 73.3 61.3;  1024 x 14336 170 132 147 123;  2048 x 8192 - 149 154 133.
//   And of K = 1024: 1000 x 4096 - 15.1 14.6 18.5;  4096 x 4096 - 49.6 52.0 45.5.
//   With groups of 32: 256 x 4096 x 4096 19.2 26.3 42.1 73.7;  512 x 16384 x 4096 110 89 91 85;  1600 x 1280 x 1536 14.0 12.7 19.7 32.9;  of 64: 17.1 21.5 32.0 55.6;
//   100 79 78 73;  12.6 11.7 16.1 26.0.
struct G4Shape { int rm; float few, all, some_two, all_two; int share; float launch, round; }; // launch, round: what a launch has beside its steps, and what another round has
constexpr G4Shape G4_SHAPES[3][4] = {// one, two and four groups in a step
                                     {{8, 1.31f, 1.90f, 0, 0, 1, 7.0f, 5.0f},
                                      {4, 0.75f, 1.09f, 0, 0, 1, 5.0f, 3.5f},
                                      {2, 0.465f, 0.575f, 0.90f, 1.105f, 2, 4.6f, 2.0f},
                                      {1, 0.33f, 0.36f, 0.61f, 0.73f, 2, 4.0f, 1.0f}},
                                     {{8, 1.53f, 2.07f, 0, 0, 1, 7.0f, 5.0f},
                                      {4, 0.85f, 1.09f, 0, 0, 1, 5.0f, 3.5f},
                                      {2, 0.53f, 0.61f, 0.92f, 1.13f, 2, 4.6f, 2.0f},
                                      {1, 0.38f, 0.41f, 0.66f, 0.76f, 2, 4.0f, 1.0f}},
                                     {{8, 2.10f, 2.44f, 0, 0, 1, 7.0f, 5.0f},
                                      {4, 1.16f, 1.31f, 0, 0, 1, 5.0f, 3.5f},
                                      {2, 0.68f, 0.72f, 1.08f, 1.33f, 2, 4.6f, 2.0f},
                                      {1, 0.44f, 0.475f, 0.70f, 0.83f, 2, 4.0f, 1.0f}}};
constexpr float G4_JOIN_US = 2.4f, G4_JOIN_RATE = 1.2e7f; // a launch that adds parts, and its bytes per us
constexpr int G4_MOST_PARTS = 16;

float g4_steps_us(const G4Shape& s, int64_t tiles, int64_t steps) {
    const int64_t round = (int64_t)G4_CUS * s.share, whole = tiles / round, rest = tiles % round;
    const auto step = [&](int64_t n) {
        return n <= G4_CUS ? s.few + (s.all - s.few) * std::max(0.0f, n * 2.0f / G4_CUS - 1) : s.some_two + (s.all_two - s.some_two) * ((float)n / G4_CUS - 1);
    };
    return s.launch + steps * (whole * (whole ? step(round) : 0) + (rest ? step(rest) : 0)) + s.round * (whole + (rest > 0) - 1);
}

// The tiles that are expected to take the least time.  (K in parts, us: 64 x 4096 x 4096 32 rows in four parts 9.7, in one 15.3; 128 x 4096 x 4096 in two 12.6.)
rkk::G4Route g4_route(int M, int N, int K, int gpb, int swiglu) {
    const int64_t places = rkh_g4_places(swiglu ? 2 * (int64_t)N : N, swiglu), KB = rkh_g4_kb(K);
    rkk::G4Route best{};
    float least = FLT_MAX;
    for (const G4Shape& s : G4_SHAPES[gpb / 2]) {
        if (s.rm > 1 && M <= 16 * s.rm) continue; // (half of the rows would be none)
        rkk::G4Route r{};
        r.rm = s.rm, r.parts = 1;
        r.mblocks = (M + 32 * s.rm - 1) / (32 * s.rm);
        r.nblocks = (int)((places + 127) / 128);
        const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
        float us = g4_steps_us(s, tiles, KB);
        if (us < least) least = us, best = r;
        for (int64_t parts = 2; parts <= KB / 2 && parts <= G4_MOST_PARTS && tiles * parts <= G4_CUS; ++parts) {
            us = g4_steps_us(s, tiles * parts, (KB + parts - 1) / parts) + G4_JOIN_US + (float)M * places * 8 * parts / G4_JOIN_RATE;
            if (us < least) least = us, best = r, best.parts = (int)parts;
        }
    }
    return best;
}
size_t g4_scratch(const rkk::G4Route& r) { return r.parts == 1 ? 0 : (size_t)r.mblocks * r.nblocks * r.parts * r.rm * 32 * 128 * 4; }

} // namespace

extern "C" {

int rkh_g4_pack(void* stream, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int K, int N, int group, int gate_up, uint8_t* dst,
                uint32_t* dst_scales) {
    const int64_t places = rkh_g4_places(N, gate_up);
    const int gpb = rkh_g4_gpb(group);
    const int64_t workgroups = places / 16 * ((rkh_g4_kb(K) + PACK_PIECES - 1) / PACK_PIECES);
    for (int64_t first = 0; first < workgroups; first += MX_MOST_GROUPS)
        hipLaunchKernelGGL(g4_pack_kernel, dim3((unsigned)std::min(MX_MOST_GROUPS, workgroups - first)), dim3(256), 0, (hipStream_t)stream, codes, scales, zeros, K,
                           N, group, (int)(((int64_t)K + group - 1) / group), gpb, gate_up, reinterpret_cast<uint32_t*>(dst), dst_scales, (size_t)first);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

int rkh_g4_run(void* stream, const rkh_g4_args* args) {
    if (!args->M || !args->N) return RKH_OK;
    const hipStream_t st = (hipStream_t)stream;
    rkh_g4_args g = *args;
    // few rows are taken as they are when they are whole pieces of eight values, or eight rows at most and values at least; tiles copy fp16 rows to LDS that are whole pieces of 128, 16-byte
    // aligned and less than 2^32 bytes of a tile apart
    const bool few = g.M <= FEW_ROWS;
    const bool as_is = few ? g.K % 8 == 0 || (g.K >= 8 && g.M <= 8)
                           : g.x_type == RKH_MX4_F16 && g.K % 128 == 0 && g.ldx % 8 == 0 && g.ldx <= 1 << 22 && reinterpret_cast<uintptr_t>(g.x) % 16 == 0;
    if (as_is) {
        g.exponents = nullptr;
    } else {
        const int rows = rkh_g4_kb(g.K) <= 16 ? 4 : 1; // of a workgroup
        const int64_t most = (INT64_C(1) << 31) / 256 * rows;
        for (int64_t first = 0; first < g.M; first += most) {
            const dim3 grid((unsigned)((std::min<int64_t>(most, g.M - first) + rows - 1) / rows));
            mark(st, "g4_stage_kernel");
            const auto kernel = g.x_type == RKH_MX4_F16 ? rows == 4 ? g4_stage_kernel<false, 4> : g4_stage_kernel<false, 1> : rows == 4 ? g4_stage_kernel<true, 4> : g4_stage_kernel<true, 1>;
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, static_cast<const uint16_t*>(g.x), g.ldx, g.M, g.K, g.staged, g.exponents, (int)first);
            RKH_CHECK(hipGetLastError());
        }
        if (g.x_type == RKH_MX4_F16) g.exponents = nullptr;
        g.x_type = RKH_MX4_F16;
        g.x = g.staged;
        g.ldx = rkh_g4_kb(g.K) * 128;
        if (few) g.K = (int)g.ldx; // (zeros there, in the rows as in the codes)
    }
    if (few) return g.x_type == RKH_MX4_F16 ? launch_few<RKH_MX4_F16>(st, g) : launch_few<RKH_MX4_BF16>(st, g);
    rkk::G4Route r = g4_route(g.M, g.N, g.K, g.gpb, g.swiglu);
    if (g4_scratch(r) > (g.scratch ? g.scratch_bytes : 0)) r.parts = 1;
    return g.gpb == 1 ? rkk::launch_g4_tiles1(st, g, r) : g.gpb == 2 ? rkk::launch_g4_tiles2(st, g, r) : rkk::launch_g4_tiles4(st, g, r);
}
void rkh_g4_route(int M, int N, int K, int gpb, int swiglu, int* kernel, int* rows, int* columns, int* parts) {
    if (M <= FEW_ROWS) {
        *kernel = 0, *rows = 16, *parts = 1;
        *columns = 16 * few_shape(M, rkh_g4_places(swiglu ? 2 * (int64_t)N : N, swiglu) / 16, (int)rkh_g4_kb(K), gpb, swiglu).cn;
        return;
    }
    const rkk::G4Route r = g4_route(M, N, K, gpb, swiglu);
    *kernel = 1, *rows = 32 * r.rm, *columns = 128, *parts = r.parts;
}
void rkh_g4_few_route(int M, int N, int K, int gpb, int swiglu, int* rows, int* columns, int* waves, int* again) {
    const FewPlan plan = few_plan(M, rkh_g4_places(swiglu ? 2 * (int64_t)N : N, swiglu) / 16, (int)rkh_g4_kb(K), gpb, swiglu != 0);
    *rows = plan.shape.rows, *columns = 16 * plan.shape.cn, *waves = plan.waves, *again = plan.per > plan.together;
}
size_t rkh_g4_scratch_bytes(int M, int N, int K, int gpb, int swiglu) { return M <= FEW_ROWS ? 0 : g4_scratch(g4_route(M, N, K, gpb, swiglu)); }
// (g4_route: a part for each compute unit at most, tiles no larger than the rows ask for)
size_t rkh_g4_scratch_most(int max_rows, int K) {
    return max_rows > FEW_ROWS && rkh_g4_kb(K) >= 4 ? (size_t)G4_CUS * 32 * 128 * 4 * (max_rows > 128 ? 8 : max_rows > 64 ? 4 : max_rows > 32 ? 2 : 1) : 0;
}

} // extern "C"
