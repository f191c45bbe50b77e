// Group-scaled 4-bit (G4) layers: weights laid out, rows staged for the tiles, products of few rows, and which kernel takes a product.
//
// C[m, n] = sum over groups of scale[n, g] * (sum over k in g of (code - zero) * x[m, k]).  code - zero is a small integer and exact in 16 bits, so the
// matrix cores' products with 16-bit activations are exact and their sums have 32 bits; the scales multiply sums, and no weight is rounded.
#include <algorithm>

#include "rk_kernels_g4.h"

namespace {

// ---- weights -----------------------------------------------------------------------
// One thread per dword of codes, then per scale dword.
__global__ __launch_bounds__(256) void g4_pack_kernel(const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int K, int N, int group, int gpb,
                                                      int gate_up, uint32_t* dst, uint32_t* dst_scales, size_t first, size_t words, size_t scale_words) {
    const size_t i = first + (size_t)blockIdx.x * 256 + threadIdx.x;
    const int KB = (int)rkh_g4_kb(K), half_rows = (K + 1) / 2, F = gate_up ? N / 2 : N;
    const auto column = [&](int64_t block, int c) -> int64_t { // in the matrix given, or -1
        const int64_t n = g4_column(block, c, gate_up != 0);
        return n < F ? n + (gate_up && (block & 1) ? F : 0) : -1;
    };
    if (i < words) {
        const size_t piece = i >> 8;
        const int lane = (int)(i >> 2) & 63, step = (int)i & 3;
        const int64_t block = (int64_t)(piece / KB), n = column(block, lane & 15);
        const int k = (int)(piece - (size_t)block * KB) * 128 + step * 32 + (lane >> 4) * 8;
        uint32_t w = 0;
        if (n >= 0) {
            const uint8_t* row = codes + (size_t)n * half_rows;
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (k + t >= K) break;
                const uint32_t code = (row[(k + t) >> 1] >> (4 * (t & 1))) & 15u; // (k is even)
                w |= code << (t & 1 ? 16 + 2 * (t - 1) : 2 * t);
            }
        }
        dst[i] = w;
    }
    if (i < scale_words) {
        const int64_t places = rkh_g4_places(N, gate_up);
        const int g = (int)(i % gpb);
        const size_t at = i / gpb;
        const int64_t kb = (int64_t)(at / places), place = (int64_t)(at - (size_t)kb * places), n = column(place >> 4, (int)place & 15);
        const int64_t k = kb * 128 + g * (128 / gpb);
        uint32_t d = 0x6400u;
        if (n >= 0 && k < K) {
            const size_t from = (size_t)n * ((K + group - 1) / group) + k / group;
            d = (uint32_t)scales[from] << 16 | (0x6400u + (zeros ? zeros[from] : 8u));
        }
        dst_scales[i] = d;
    }
}

// ---- rows for the tiles ---------------------------------------------------------------
// One workgroup per row.  bf16: the row's largest finite magnitude is moved to 2^14 .. 2^15, where eight bits fit a half down to 2^-38 of it (what is
// smaller than that is rounded to a multiple of 2^-39 of it); infinities and NaN stay what they are.
template <bool BF16>
__global__ __launch_bounds__(256) void g4_stage_kernel(const uint16_t* x, int64_t ldx, int K, uint16_t* staged, int* exponents, int first) {
    __shared__ uint32_t part[4];
    const int m = first + blockIdx.x, Kp = (int)rkh_g4_kb(K) * 128;
    const uint16_t* row = x + (size_t)m * ldx;
    uint16_t* to = staged + (size_t)m * Kp;
    const auto fetch = [&](int k) { return k + 8 <= K ? mx_fetch8<RKH_MX4_F16>(row, k) : mx_fetch_some<RKH_MX4_F16>(row, k, K - k); };
    if constexpr (!BF16) {
        for (int k = threadIdx.x * 8; k < Kp; k += 2048) *reinterpret_cast<v4i*>(to + k) = fetch(k).w[0];
    } else {
        constexpr int AHEAD = 4; // 8192 values in registers; what is beyond is read twice
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
            const int k = threadIdx.x * 8 + u * 2048;
            raw[u] = k < Kp ? fetch(k).w[0] : v4i{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) look(raw[u]);
        for (int k = threadIdx.x * 8 + AHEAD * 2048; k < Kp; k += 2048) look(fetch(k).w[0]);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
        if (lane_id() == 0) part[wave_id()] = top;
        __syncthreads();
        top = max(max(part[0], part[1]), max(part[2], part[3]));
        // 2^e: from the exponent of the largest to 14 (of numbers below the normal ones the largest has 127 places to go at least)
        const int e = top ? 14 + 127 - (int)max(top >> 23, 1u) : 0;
        if (threadIdx.x == 0) exponents[m] = -e;
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
            if ((int)threadIdx.x * 8 + u * 2048 < Kp) put(threadIdx.x * 8 + u * 2048, raw[u]);
        for (int k = threadIdx.x * 8 + AHEAD * 2048; k < Kp; k += 2048) put(k, fetch(k).w[0]);
    }
}

// ---- few rows ------------------------------------------------------------------------
// One workgroup multiplies up to 16 rows with 16 CN places; its waves split K into pieces of 128 and are summed through LDS.  Codes go straight into
// registers, once; so do activations, which every workgroup reads for itself.
// BOUNCE: up to four rows.  A wave loads a row's 512 values together and turns them into operands through LDS of its own; more rows are
// loaded as the operands lie.
// fp16: products with code - zero.  bf16: products with the code, and the zero point times the group's sum of activations, which a product with ones
// gives, is taken off the sum.
constexpr int FEW_PITCH = 1024 + 16; // bytes of a row of 512 values in LDS

template <int TYPE, int CN, int GPB, bool BOUNCE, bool SWIGLU, int NP, int MAX_WAVES>
__global__ __launch_bounds__(MAX_WAVES * 64) void g4_few_kernel(const uint8_t* W, const uint32_t* scales, const uint16_t* x, int64_t ldx, int M, int K,
                                                                int per_wave, int workgroups, int waves, rkh_g4_args g) {
    constexpr bool F16 = TYPE == RKH_MX4_F16;
    constexpr int STEPS = 4 / GPB; // 32-k steps of a group
    static_assert(!SWIGLU || CN == 2, "a gate and an up half");
    static_assert(!BOUNCE || NP % 4 == 0, "rows are loaded 512 values at a time");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), c = lane & 15, q = lane >> 4;
    const int KB = (int)rkh_g4_kb(K);
    const int64_t places = rkh_g4_places(SWIGLU ? 2 * (int64_t)g.N : g.N, SWIGLU);
    const int block0 = xcd_remap(blockIdx.x, workgroups) * CN;
    const int first = wave * per_wave, last = min(first + per_wave, KB);
    const int row = min(c, M - 1); // (operand rows beyond M: the last one again, whose results nobody takes)
    typedef uint32_t words __attribute__((ext_vector_type(GPB)));

    const auto fetch = [&](int m, int k) -> v4i { // (K is a multiple of eight)
        const v4i v = mx_fetch8<TYPE>(x, (size_t)m * ldx + (k < K ? k : 0)).w[0];
        return k < K ? v : v4i{0, 0, 0, 0};
    };
    v4f acc[CN];
#pragma unroll
    for (int j = 0; j < CN; ++j) acc[j] = v4f{0, 0, 0, 0};
    uint8_t* own = lds + wave * (4 * FEW_PITCH);

    for (int from = first; from < last; from += NP) {
        v4i w[NP][CN], rows[BOUNCE ? NP : NP * 4]; // BOUNCE: [512 values][row]
        words sd[NP][CN];
        // everything that the pieces need (of pieces beyond the last: that one again, which is not multiplied)
#pragma unroll
        for (int i = 0; i < (BOUNCE ? NP : NP * 4); ++i) {
            if constexpr (!BOUNCE) rows[i] = fetch(row, from * 128 + i * 32 + q * 8);
            else if ((i & 3) < M) rows[i] = fetch(i & 3, (from + (i & ~3)) * 128 + lane * 8);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int kb = min(from + p, KB - 1);
#pragma unroll
            for (int j = 0; j < CN; ++j) {
                w[p][j] = *reinterpret_cast<const v4i*>(W + ((size_t)(block0 + j) * KB + kb) * 1024 + lane * 16);
                sd[p][j] = *reinterpret_cast<const words*>(scales + ((size_t)kb * places + (block0 + j) * 16 + c) * GPB);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            if (from + p >= last) break;
            if constexpr (BOUNCE) {
                if (p % 4 == 0) {
                    __builtin_amdgcn_wave_barrier(); // (a wave's LDS operations complete in order)
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        if (m < M) *reinterpret_cast<v4i*>(own + m * FEW_PITCH + lane * 16) = F16 ? rows[p + m] : g4_turned_rows(rows[p + m]);
                    __builtin_amdgcn_wave_barrier();
                }
            }
            v4i a[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (BOUNCE) a[i] = *reinterpret_cast<const v4i*>(own + row * FEW_PITCH + (p & 3) * 256 + i * 64 + q * 16);
                else a[i] = F16 ? rows[p * 4 + i] : g4_turned_rows(rows[p * 4 + i]);
            }
#pragma unroll
            for (int n = 0; n < GPB; ++n) {
                if constexpr (F16) {
#pragma unroll
                    for (int j = 0; j < CN; ++j) {
                        G4Zero z;
                        z.of(sd[p][j][n]);
                        v4f part = {0, 0, 0, 0};
#pragma unroll
                        for (int i = n * STEPS; i < (n + 1) * STEPS; ++i)
                            part = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a[i]), g4_halves((uint32_t)w[p][j][i], z), part, 0, 0, 0);
                        const float s = g4_scale(sd[p][j][n], g.scale_type);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(part[e], s, acc[j][e]);
                    }
                } else {
                    constexpr int ONES = 0x3f803f80;
                    const v8b ones = __builtin_bit_cast(v8b, (v4i{ONES, ONES, ONES, ONES}));
                    v4f sum = {0, 0, 0, 0};
#pragma unroll
                    for (int i = n * STEPS; i < (n + 1) * STEPS; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a[i]), ones, sum, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < CN; ++j) {
                        v4f part = {0, 0, 0, 0};
#pragma unroll
                        for (int i = n * STEPS; i < (n + 1) * STEPS; ++i)
                            part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a[i]), g4_codes_bf16((uint32_t)w[p][j][i]), part, 0, 0, 0);
                        const float s = g4_scale(sd[p][j][n], g.scale_type), zero = (float)(sd[p][j][n] & 0xffu);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][e] = fmaf(fmaf(-zero, sum[e], part[e]), s, acc[j][e]);
                    }
                }
            }
        }
    }

    // the waves' sums, added in order
    v4f* sums = reinterpret_cast<v4f*>(lds + (BOUNCE ? waves * 4 * FEW_PITCH : 0));
#pragma unroll
    for (int j = 0; j < CN; ++j) sums[(wave * CN + j) * 64 + lane] = acc[j];
    __syncthreads();
    if (wave != 0) return;
    v4f s[CN];
#pragma unroll
    for (int j = 0; j < CN; ++j) {
        s[j] = sums[j * 64 + lane];
        for (int o = 1; o < waves; ++o) s[j] += sums[(o * CN + j) * 64 + lane];
    }
    const int64_t n = g4_column(block0, c, SWIGLU);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int m = 4 * q + e;
        if (m >= M) break;
        float v[CN];
#pragma unroll
        for (int j = 0; j < CN; ++j) v[j] = g.exponents ? __builtin_amdgcn_ldexpf(s[j][e], g.exponents[m]) : s[j][e];
        if constexpr (SWIGLU) {
            const float y[1] = {mx_silu(v[0], v[1])};
            g4_put<1>(g, m, n, y);
        } else {
            g4_put<CN>(g, m, n, v);
        }
    }
}

constexpr int FEW_ROWS = 16;

template <int TYPE, int CN, int GPB, bool BOUNCE, bool SWIGLU, int NP, int MAX_WAVES> int launch_few(hipStream_t st, const rkh_g4_args& g, int per) {
    const int KB = (int)rkh_g4_kb(g.K), waves = (KB + per - 1) / per;
    const int64_t workgroups = rkh_g4_places(SWIGLU ? 2 * (int64_t)g.N : g.N, SWIGLU) / (16 * CN);
    if (workgroups * waves * 64 >= MX_TOO_MANY_THREADS) return RKH_ERR_RUNTIME;
    const size_t bytes = (size_t)waves * (CN * 1024 + (BOUNCE ? 4 * FEW_PITCH : 0));
    const auto kernel = g4_few_kernel<TYPE, CN, GPB, BOUNCE, SWIGLU, NP, MAX_WAVES>;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(kernel), opted_in, 160 * 1024)) return rc;
    mark(st, "g4_few_kernel");
    hipLaunchKernelGGL(kernel, dim3((unsigned)workgroups), dim3(waves * 64), bytes, st, g.W, g.w_scale, static_cast<const uint16_t*>(g.x), g.ldx, g.M, g.K, per,
                       (int)workgroups, waves, g);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}
template <int TYPE, int GPB> int launch_few(hipStream_t st, const rkh_g4_args& g) {
    const int KB = (int)rkh_g4_kb(g.K);
    const auto per = [&](int waves, int np) { return std::max((KB + waves - 1) / waves, std::min(np, (KB + 3) / 4)); }; // pieces of a wave
    if (g.swiglu) return g.M <= 4 ? launch_few<TYPE, 2, GPB, true, true, 4, 8>(st, g, per(8, 4)) : launch_few<TYPE, 2, GPB, false, true, 2, 8>(st, g, per(8, 4));
    return g.M <= 4 ? launch_few<TYPE, 1, GPB, true, false, 4, 16>(st, g, per(16, 4)) : launch_few<TYPE, 1, GPB, false, false, 2, 16>(st, g, per(16, 4));
}
template <int TYPE> int launch_few(hipStream_t st, const rkh_g4_args& g) {
    return g.gpb == 1 ? launch_few<TYPE, 1>(st, g) : g.gpb == 2 ? launch_few<TYPE, 2>(st, g) : launch_few<TYPE, 4>(st, g);
}

// ---- which kernel ------------------------------------------------------------------
constexpr int G4_CUS = 256; // compute units that a launch is cut for
// Tiles of 64 rm rows x 128 places: what a step of 128 k takes in each, us
struct G4Shape { int rm; float step, end; };
constexpr G4Shape G4_SHAPES[] = {{4, 1.3f, 3.0f}, {2, 0.8f, 2.0f}, {1, 0.5f, 1.5f}};
constexpr float G4_TILES_US = 3.0f, G4_JOIN_US = 3.0f, G4_JOIN_RATE = 4.5e6f;
constexpr int G4_MOST_PARTS = 16;

rkk::G4Route g4_route(int M, int N, int K, int gpb, int swiglu) {
    (void)gpb;
    const int64_t places = rkh_g4_places(swiglu ? 2 * (int64_t)N : N, swiglu), KB = rkh_g4_kb(K);
    rkk::G4Route best{};
    float least = FLT_MAX;
    for (const G4Shape& s : G4_SHAPES) {
        if (s.rm > 1 && M <= 32 * s.rm) continue; // (half of the rows would be none)
        rkk::G4Route r{};
        r.rm = s.rm, r.parts = 1;
        r.mblocks = (M + 64 * s.rm - 1) / (64 * s.rm);
        r.nblocks = (int)((places + 127) / 128);
        const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
        float us = G4_TILES_US + (tiles + G4_CUS - 1) / G4_CUS * (KB * s.step + s.end);
        if (us < least) least = us, best = r;
        for (int64_t parts = 2; parts <= KB / 2 && parts <= G4_MOST_PARTS && tiles * parts <= G4_CUS; ++parts) {
            us = G4_TILES_US + (KB + parts - 1) / parts * s.step + s.end + G4_JOIN_US + (float)M * places * 8 * parts / G4_JOIN_RATE;
            if (us < least) least = us, best = r, best.parts = (int)parts;
        }
    }
    return best;
}
size_t g4_scratch(const rkk::G4Route& r) { return r.parts == 1 ? 0 : (size_t)r.mblocks * r.nblocks * r.parts * r.rm * 64 * 128 * 4; }

} // namespace

extern "C" {

int rkh_g4_pack(void* stream, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, int K, int N, int group, int gate_up, uint8_t* dst,
                uint32_t* dst_scales) {
    const int64_t places = rkh_g4_places(N, gate_up);
    const int gpb = rkh_g4_gpb(group);
    const size_t words = rkh_g4_code_bytes(places, K) / 4, scale_words = rkh_g4_scale_bytes(places, K, gpb) / 4;
    const int64_t groups = (int64_t)((std::max(words, scale_words) + 255) / 256);
    for (int64_t first = 0; first < groups; first += MX_MOST_GROUPS)
        hipLaunchKernelGGL(g4_pack_kernel, dim3((unsigned)std::min(MX_MOST_GROUPS, groups - first)), dim3(256), 0, (hipStream_t)stream, codes, scales, zeros, K,
                           N, group, gpb, gate_up, reinterpret_cast<uint32_t*>(dst), dst_scales, (size_t)first * 256, words, scale_words);
    RKH_CHECK(hipGetLastError());
    return RKH_OK;
}

int rkh_g4_run(void* stream, const rkh_g4_args* args) {
    if (!args->M || !args->N) return RKH_OK;
    const hipStream_t st = (hipStream_t)stream;
    rkh_g4_args g = *args;
    // few rows are taken as they are when they are whole pieces of eight values; tiles copy fp16 rows to LDS that are whole pieces of 128, 16-byte
    // aligned and less than 2^32 bytes of a tile apart
    const bool few = g.M <= FEW_ROWS;
    const bool as_is = few ? g.K % 8 == 0
                           : g.x_type == RKH_MX4_F16 && g.K % 128 == 0 && g.ldx % 8 == 0 && g.ldx <= 1 << 22 && reinterpret_cast<uintptr_t>(g.x) % 16 == 0;
    if (as_is) {
        g.exponents = nullptr;
    } else {
        const int64_t most = (INT64_C(1) << 31) / 256;
        for (int64_t first = 0; first < g.M; first += most) {
            const dim3 rows((unsigned)std::min<int64_t>(most, g.M - first));
            mark(st, "g4_stage_kernel");
            const auto kernel = g.x_type == RKH_MX4_F16 ? g4_stage_kernel<false> : g4_stage_kernel<true>;
            hipLaunchKernelGGL(kernel, rows, dim3(256), 0, st, static_cast<const uint16_t*>(g.x), g.ldx, g.K, g.staged, g.exponents, (int)first);
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
        *kernel = 0, *rows = 16, *columns = swiglu ? 32 : 16, *parts = 1;
        return;
    }
    const rkk::G4Route r = g4_route(M, N, K, gpb, swiglu);
    *kernel = 1, *rows = 64 * r.rm, *columns = 128, *parts = r.parts;
}
size_t rkh_g4_scratch_bytes(int M, int N, int K, int gpb, int swiglu) { return M <= FEW_ROWS ? 0 : g4_scratch(g4_route(M, N, K, gpb, swiglu)); }
// (g4_route: a part for each compute unit at most, tiles no larger than the rows ask for)
size_t rkh_g4_scratch_most(int max_rows, int K) {
    return max_rows > FEW_ROWS && rkh_g4_kb(K) >= 4 ? (size_t)G4_CUS * 64 * 128 * 4 * (max_rows > 128 ? 4 : max_rows > 64 ? 2 : 1) : 0;
}

} // extern "C"
