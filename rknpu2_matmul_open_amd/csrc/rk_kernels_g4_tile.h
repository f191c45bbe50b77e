// Tiles of G4 products.
//
// Many rows: 256 rows x 128 places by four waves (two by two), each 4 x 2 accumulators of 32 x 32.  Bound by power, and by what one wave has to issue: about
// 2950 clocks a step, 2090 of them products; variants with 2800 took no less time, as the clock fell.  4096 x 14336 x 4096 429 us, 1.12 PFLOP/s (a library's
// product of halves of this size, which has no codes to turn into halves, 417); 512 rows of SwiGLU with groups of 64 130 us, 0.92.
//
// A step is 128 k.  Its activations (rows of 256 bytes), codes and scales are copied global -> LDS directly, two steps ahead of the products and one
// ahead of the LDS reads:
//  * a wave's activations of a step live in registers, 8 RM operands that both of its 32-place halves j multiply.  An operand's last product
//    is one of half 1; behind it, it is replaced by the next step's;
//  * codes become halves (code - zero) one operand at a time, before the half's first products: the first four operands have registers for each half, and
//    the other four take those of the other half behind its last products;
//  * a group's products start from zero, and its sum goes into the accumulators, times the scale, while the next group's run.
// In half-time of step s (between the halves) a wave waits for its copies of step s + 1 and for its LDS reads, and meets the others: from
// there on LDS holds step s + 1 for all, and nobody reads step s any more, whose place the copies of step s + 2 take.
//
// Places in LDS: a row's 128 bytes of 64 k are eight pieces of 16 bytes, of which piece c lies at place c ^ (row / 2 & 7); sixteen lanes then read
// sixteen rows from all 64 banks, and a copy still fetches whole 128-byte lines.
#ifndef RK_KERNELS_G4_TILE_H
#define RK_KERNELS_G4_TILE_H

#include <algorithm>

#include "rk_kernels_g4.h"

namespace {

template <int GPB> struct G4Tile {
    static constexpr int RM = 4, ROWS = 64 * RM, HALF = ROWS * 128; // HALF: bytes of 64 k
    static constexpr int W_OFF = 2 * HALF, S_OFF = W_OFF + 8192, S_COPIES = GPB == 4 ? 2 : 1, BUF = S_OFF + S_COPIES * 1024, LDS = 2 * BUF;
    // copies of a wave and step: activations, codes, scales; and the statements that issue them, two at a time but the last
    static constexpr int XC = 4 * RM, COPIES = XC + 3, PAIRS = XC / 2 + 2;
    static constexpr int copies(int statements) { return statements < PAIRS ? 2 * statements : COPIES; }
    static_assert(LDS <= 160 * 1024, "");
};

// What a step issues, as asm statements: they stay where they are written (of plain operations the compiler collects a step's sums, and its halves, in a
// few places, and moves sums between the halves of the registers).  What it then does not order: a vector instruction that writes an operand has to be
// two wait states ahead of the product; one that reads a sum eleven behind it, and a product in between counts for eight of them, which it
// takes to issue behind another one.
__device__ __forceinline__ void g4_product(const v4i& a, const v4i& w, v16f& sum) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(sum) : "a"(a), "v"(w));
}
__device__ __forceinline__ void g4_product_first(const v4i& a, const v4i& w, v16f& sum) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(sum) : "a"(a), "v"(w));
}
__device__ __forceinline__ void g4_add_scaled(float& acc, float sum, float scale) { asm volatile("v_fmac_f32_e32 %0, %1, %2" : "+v"(acc) : "v"(sum), "v"(scale)); }
// Pair R of g4_halves; `magic` is g4_exponents.  (One statement: between two of them the compiler puts a wait state for a hazard that these
// instructions do not have.)  R = 2 leaves the codes, shifted by eight bits, in `upper` for R = 3.
template <int R> __device__ __forceinline__ uint32_t g4_pair_here(uint32_t w, const G4Zero& z, uint32_t magic, uint32_t& upper) {
    uint32_t v;
    if constexpr (R == 0)
        asm volatile("v_and_or_b32 %0, %1, %2, %3\n\tv_pk_add_f16 %0, %0, %4" : "=&v"(v) : "v"(w), "s"(0x000f000fu), "v"(magic), "v"(z.low));
    else if constexpr (R == 2)
        asm volatile("v_lshrrev_b32 %1, 8, %2\n\tv_and_or_b32 %0, %1, %3, %4\n\tv_pk_add_f16 %0, %0, %5"
                     : "=&v"(v), "=&v"(upper) : "v"(w), "s"(0x000f000fu), "v"(magic), "v"(z.low));
    else // (times 1/16)
        asm volatile("v_and_or_b32 %0, %1, %2, %3\n\tv_pk_fma_f16 %0, %0, %4, %5"
                     : "=&v"(v) : "v"(R == 1 ? w : upper), "s"(0x00f000f0u), "v"(magic), "s"(0x2c002c00u), "v"(z.high));
    return v;
}

// The same for the four pairs of a dword, for a wave that has nothing to wait for in between.
__device__ __forceinline__ v4i g4_dword_here(uint32_t w, const G4Zero& z, uint32_t magic) {
    uint32_t v0, v1, v2, v3, upper;
    asm volatile("v_and_or_b32 %0, %5, %6, %8\n\tv_and_or_b32 %1, %5, %7, %8\n\tv_lshrrev_b32 %4, 8, %5\n\tv_pk_add_f16 %0, %0, %9\n\tv_pk_fma_f16 %1, %1, %11, %10\n\t"
                 "v_and_or_b32 %2, %4, %6, %8\n\tv_and_or_b32 %3, %4, %7, %8\n\tv_pk_add_f16 %2, %2, %9\n\tv_pk_fma_f16 %3, %3, %11, %10"
                 : "=&v"(v0), "=&v"(v1), "=&v"(v2), "=&v"(v3), "=&v"(upper)
                 : "v"(w), "s"(0x000f000fu), "s"(0x00f000f0u), "v"(magic), "v"(z.low), "v"(z.high), "s"(0x2c002c00u));
    return v4i{(int)v0, (int)v1, (int)v2, (int)v3};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is set and clobbered on purpose below
// mx_copy to `to` + `more`, which M0 takes as the sum that it is.
__device__ __forceinline__ void g4_copy(const uint8_t* base, unsigned off, uint32_t to, uint32_t more) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to), "s"(more) : "memory", "m0", "scc");
}
template <int MORE> __device__ __forceinline__ void g4_copy(const uint8_t* base, unsigned off, uint32_t to) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(to), "n"(MORE) : "memory", "m0", "scc");
}
// mx_copy_two
__device__ __forceinline__ void g4_copy_two(const uint8_t* base, const uint8_t* base2, unsigned off, uint32_t to, uint32_t more) {
    asm volatile("s_add_u32 m0, %3, %4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n\tglobal_load_lds_dwordx4 %0, %2 offset:1024" ::"v"(off), "s"(base), "s"(base2),
                 "s"(to), "s"(more) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

// What a launch of tiles covers, and the numbers that its workgroups would divide by.  (With divisions, of 64 bits among them, a workgroup of 32 rows had its
// first address after 2000 clocks and not after 1200, and 32 x 4096 x 4096 took 11.8 us, now 10.4.)
struct G4Grid {
    int mblocks, nblocks, parts;
    int blocks;                   // of 16 places
    int each, more;               // pieces of K of a part; the first `more` have one more
    MxDivider tiles, group, last; // .. by tiles, by those of a group of row blocks, by the row blocks of the last group
    static constexpr int GROUP = 4; // row blocks that are swept together

    static G4Grid of(const rkk::G4Route& r, const rkh_g4_args& g) {
        const int KB = (int)rkh_g4_kb(g.K), left = r.mblocks % GROUP;
        return {r.mblocks, r.nblocks, r.parts, (int)(rkh_g4_places(g.swiglu ? 2 * (int64_t)g.N : g.N, g.swiglu) / 16), KB / r.parts, KB % r.parts,
                MxDivider::of((uint32_t)(r.mblocks * r.nblocks)), MxDivider::of((uint32_t)(GROUP * r.nblocks)), MxDivider::of((uint32_t)(left ? left : GROUP))};
    }
    // Where a tile lies: column sweeps over groups of row blocks, so that concurrently running tiles share weights in L2.
    __device__ __forceinline__ void place(unsigned tile, int& mblk, int& nblk) const {
        const unsigned grp = group.divide(tile), first_m = grp * GROUP, in_group = tile - grp * GROUP * nblocks;
        const bool whole = mblocks - first_m >= GROUP;
        const unsigned of_last = last.divide(in_group), col = whole ? in_group / GROUP : of_last;
        mblk = __builtin_amdgcn_readfirstlane((int)(first_m + in_group - col * (whole ? (unsigned)GROUP : mblocks - first_m)));
        nblk = __builtin_amdgcn_readfirstlane((int)col);
    }
    __device__ __forceinline__ void job(unsigned at, unsigned& tile, int& part) const {
        const unsigned in_order = (unsigned)xcd_remap((int)at, mblocks * nblocks * parts);
        part = __builtin_amdgcn_readfirstlane((int)tiles.divide(in_order));
        tile = in_order - part * mblocks * nblocks;
    }
    __device__ __forceinline__ int begin(int part) const { return part * each + min(part, more); }
    __device__ __forceinline__ int KB() const { return begin(parts); }
};
// The exponents of four rows from `first` on.  (All of them are fetched ahead of the first store, behind which a load would wait: 1622 x 1335 x 1536 of bf16 32.7 us
// with a load a row, now 26.3.)
template <bool EXPONENTS> __device__ __forceinline__ v4i g4_exponents4(const rkh_g4_args& g, int first) {
    if constexpr (EXPONENTS) return *reinterpret_cast<const v4i*>(g.exponents + first);
    else return v4i{0, 0, 0, 0};
}
// Four rows from `first` on of a lane's two columns (SwiGLU: of both halves of one) from accumulators of 32 x 32 to results; n: the first column.
template <int OUT, bool SWIGLU, bool EXPONENTS>
__device__ __forceinline__ void g4_finish4(const rkh_g4_args& g, int first, int64_t n, const float* s0, const float* s1, const v4i& exponents) {
    using T = typename MxType<OUT>::T;
    typedef T pair __attribute__((ext_vector_type(2)));
    typedef pair pair_any __attribute__((aligned(sizeof(T))));
    T* to = static_cast<T*>(g.C) + (size_t)first * g.ldc + n;
    const int live = n < g.N ? g.M - first : 0;
    const bool both = n + 1 < g.N;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e < live) {
            float a = s0[e], b = s1[e];
            if constexpr (EXPONENTS) a = __builtin_amdgcn_ldexpf(a, exponents[e]), b = __builtin_amdgcn_ldexpf(b, exponents[e]);
            if constexpr (SWIGLU) *to = (T)mx_silu(a, b);
            else if (both) *reinterpret_cast<pair_any*>(to) = pair{(T)a, (T)b};
            else *to = (T)a;
        }
        to += g.ldc;
    }
}
template <bool SWIGLU, class F> __device__ __forceinline__ void g4_with_finish(const rkh_g4_args& g, F&& f) {
    mx_with_type(g.out_type, [&](auto t) {
        constexpr int OUT = decltype(t)::value;
        const auto go = [&](auto with) {
            constexpr bool EXPONENTS = decltype(with)::value;
            f([&](int first) { return g4_exponents4<EXPONENTS>(g, first); },
              [&](int first, int64_t n, const float* s0, const float* s1, const v4i& exponents) { g4_finish4<OUT, SWIGLU, EXPONENTS>(g, first, n, s0, s1, exponents); });
        };
        if (g.exponents) go(std::true_type{});
        else go(std::false_type{});
    });
}
// A lane's first column of the 64 places from `unit` on.
template <bool SWIGLU> __device__ __forceinline__ int64_t g4_lane_column(int64_t unit, int lane) { return SWIGLU ? unit * 32 + (lane & 31) : unit * 64 + 2 * (lane & 31); }

template <int GPB, bool SWIGLU>
__global__ __launch_bounds__(256) void g4_tile_kernel(G4Grid t, rkh_g4_args g) {
    using S = G4Tile<GPB>;
    constexpr int RM = S::RM;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id()), wm = wave & 1, wn = wave >> 1;
    const int parts = t.parts, KB = t.KB();
    unsigned tile;
    int part, mblk, nblk;
    t.job(blockIdx.x, tile, part);
    t.place(tile, mblk, nblk);
    const int kb0 = t.begin(part), kb1 = t.begin(part + 1);

    // ---- copies.  Wave-uniform addresses that advance by a step, lane offsets that stay.
    const uint32_t base = (uint32_t)(uintptr_t)(mx_lds_ptr)lds;
    const int m0 = mblk * S::ROWS;
    // (a bias of 1024: offsets of the second copies of pairs are 1024 less, see mx_copy_two)
    const uint8_t* x_src = static_cast<const uint8_t*>(g.x) + ((size_t)m0 * g.ldx + (size_t)kb0 * 128) * 2 - 1024;
    unsigned x_off[2 * RM]; // of eight rows' 128 bytes; rows beyond M: the last one again
#pragma unroll
    for (int r = 0; r < 2 * RM; ++r) {
        const int row = min(m0 + (wave * 2 * RM + r) * 8 + (lane >> 3), g.M - 1) - m0;
        x_off[r] = (unsigned)row * (unsigned)g.ldx * 2 + ((lane & 7) ^ ((r & 1) * 4 + (lane >> 4))) * 16 + (r & 1 ? 0 : 1024);
    }
    const uint8_t* w_src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) w_src[i] = g.W + ((size_t)min(nblk * 8 + wave * 2 + i, t.blocks - 1) * KB + kb0) * 1024 - i * 1024;
    // (waves copy the same scales, or the same half of them, to one place: of each block of 16 places a piece of 64 GPB bytes)
    const unsigned s_lane = (GPB == 4 ? (wave & 1) * 1024 : 0) + lane * 16, s_at_tile = s_lane % (512 * GPB);
    const uint8_t* s_src = reinterpret_cast<const uint8_t*>(g.w_scale) + ((size_t)nblk * 8 * KB + kb0) * (64 * GPB);
    const unsigned s_off = (unsigned)min((int)(s_at_tile / (64 * GPB)), t.blocks - 1 - nblk * 8) * (unsigned)KB * (64 * GPB) + s_at_tile % (64 * GPB);
    int ahead = kb1 - kb0; // steps that are still to be copied
    const auto copy = [&](uint32_t to, auto p_tag) {
        constexpr int P = decltype(p_tag)::value;
        if constexpr (P < S::XC / 2) {
            constexpr int SUB = P / RM, R = P % RM * 2;
            mx_copy_two(x_src + SUB * 128, x_off[R], x_src + SUB * 128, x_off[R + 1], base + to + SUB * S::HALF + (wave * 2 * RM + R) * 1024);
        } else if constexpr (P == S::XC / 2) {
            mx_copy_two(w_src[0], lane * 16, w_src[1], lane * 16, base + to + S::W_OFF + wave * 2048);
        } else {
            mx_copy(s_src, s_off, base + to + S::S_OFF + (GPB == 4 ? (wave & 1) * 1024 : 0));
        }
    };
    const auto copied = [&]() { // (behind the last step: that one again, which nobody reads)
        if (--ahead > 0) {
            x_src += 256;
            w_src[0] += 1024, w_src[1] += 1024;
            s_src += 64 * GPB;
        }
    };

    // ---- LDS reads
    uint32_t a_at[4]; // step s of a row's 64 k: s % 4
#pragma unroll
    for (int s = 0; s < 4; ++s) a_at[s] = (wm * RM * 32 + (lane & 31)) * 128 + (((2 * s + (lane >> 5)) ^ (lane >> 1 & 7)) * 16);
    const uint32_t w_at = S::W_OFF + wn * 4096 + (lane >> 4 & 1) * 2048 + (lane & 15) * 16 + (lane >> 5) * 256;
    const uint32_t s_at = S::S_OFF + (wn * 64 + (lane >> 4 & 1) * 32 + (lane & 15)) * GPB * 4; // [block][c][gpb], as copied
    v4i a[RM][8], w[12]; // (of half 0: 0 .. 3 and 8 .. 11, of half 1: 4 .. 11)
    v4i raw[2][2];
    typedef uint32_t words __attribute__((ext_vector_type(GPB)));
    words sd[2];
    float scale[2][GPB];
    const auto read_a = [&](uint32_t from, auto i_tag, auto s_tag) {
        constexpr int I = decltype(i_tag)::value, ST = decltype(s_tag)::value;
        a[I][ST] = *reinterpret_cast<const v4i*>(lds + from + a_at[ST & 3] + (ST >> 2) * S::HALF + I * 4096);
    };
    const auto read_w = [&](uint32_t from, auto j_tag) {
        constexpr int J = decltype(j_tag)::value;
        raw[J][0] = *reinterpret_cast<const v4i*>(lds + from + w_at + J * 1024);
        raw[J][1] = *reinterpret_cast<const v4i*>(lds + from + w_at + J * 1024 + 512);
    };
    const auto read_s = [&](uint32_t from, auto j_tag) {
        constexpr int J = decltype(j_tag)::value;
        sd[J] = *reinterpret_cast<const words*>(lds + from + s_at + J * 64 * GPB);
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;

    // ---- codes to operands: pair x (0..31) of a half's eight operands
    G4Zero zero[2][GPB];
    uint32_t magic, upper[2] = {0, 0};
    asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
    const auto decode = [&](auto j_tag, auto x_tag) {
        constexpr int J = decltype(j_tag)::value, X = decltype(x_tag)::value, ST = X / 4, R = X % 4;
        w[ST < 4 ? 4 * J + ST : 4 + ST][R] = (int)g4_pair_here<R>((uint32_t)raw[J][ST & 1][ST >> 1], zero[J][ST * GPB / 8], magic, upper[J]);
    };
    const auto zeros_of = [&](auto j_tag) {
        constexpr int J = decltype(j_tag)::value;
#pragma unroll
        for (int n = 0; n < GPB; ++n) zero[J][n].of(sd[J][n]);
    };
    const auto scale_of = [&](auto j_tag) {
        constexpr int J = decltype(j_tag)::value;
#pragma unroll
        for (int n = 0; n < GPB; ++n) scale[J][n] = g4_scale(sd[J][n], g.scale_type);
    };

    // ---- steps.  Slot t is product t of the step and what is issued behind it.  What goes where is spread so that a slot has five or six instructions
    // beside its product, which are what the product's 32 clocks have room for.
    constexpr int L = 8 / GPB, GROUPS = 2 * RM * GPB, SLOTS = 16 * RM, MID = 8 * RM; // products of a group, groups and slots of a step
    // half J's codes, in slots from the start of the other half's last chain: operands 0 .. 3, then 4 .. 7
    constexpr int CODES_FROM = -17, CODES_THEN = 5, CODES_TO = 14;
    // copies go out from half-time on, evenly, those of half-time's step + 2 ending some slots ahead of the next one; EARLY of the statements behind a step's end
    constexpr int COPY_SLOTS = 44, EARLY = S::PAIRS * MID / COPY_SLOTS;
    constexpr int READS = 18; // slots that operands of half the rows are read in

    // ---- prologue
    static_for<S::PAIRS>([&](auto p) { copy(0, p); });
    copied();
    static_for<EARLY>([&](auto p) { copy(S::BUF, p); });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::copies(EARLY)) : "memory");
    static_for<RM>([&](auto i) { static_for<8>([&](auto s) { read_a(0, i, s); }); });
    read_w(0, I0{}), read_w(0, I1{});
    read_s(0, I0{}), read_s(0, I1{});
    zeros_of(I0{});
    static_for<32>([&](auto x) { decode(I0{}, x); });

    float acc[RM][2][16];
    v16f sum[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
        for (int i = 0; i < RM; ++i) acc[i][0][e] = acc[i][1][e] = 0;
        sum[0][e] = sum[1][e] = 0;
    }
#pragma unroll
    for (int n = 0; n < GPB; ++n) scale[0][n] = scale[1][n] = 0;

    const auto fold = [&](auto g_tag, auto from_tag, auto to_tag) { // elements of group G's sum into the accumulators
        constexpr int G = decltype(g_tag)::value, C = G / GPB, I = C % RM, J = C / RM;
#pragma unroll
        for (int e = from_tag(); e < to_tag(); ++e) g4_add_scaled(acc[I][J][e], sum[G & 1][e], scale[J][G % GPB]);
    };
    const auto decode_some = [&](auto j_tag, auto at_tag) {
        constexpr int AT = decltype(at_tag)::value;
        if constexpr (AT >= CODES_FROM && AT < CODES_TO) {
            if constexpr (AT == CODES_FROM) zeros_of(j_tag);
            constexpr bool FIRST = AT < CODES_THEN;
            constexpr int FROM = FIRST ? CODES_FROM : CODES_THEN, N = (FIRST ? CODES_THEN : CODES_TO) - FROM, O = FIRST ? 0 : 16;
            constexpr int X0 = O + 16 * (AT - FROM) / N, X1 = O + 16 * (AT + 1 - FROM) / N;
            static_for<X1 - X0>([&](auto x) { decode(j_tag, std::integral_constant<int, X0 + decltype(x)::value>{}); });
        }
    };
    uint32_t here = 0; // of the step that is multiplied
    for (int kb = kb0; kb < kb1; ++kb) {
        const uint32_t next = S::BUF - here;
        static_for<SLOTS>([&](auto t_tag) {
            constexpr int T = decltype(t_tag)::value, C = T / 8, ST = T % 8, I = C % RM, G = T / L;
            if constexpr (T == MID) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            constexpr int J = C / RM, W = ST < 4 ? 4 * J + ST : 4 + ST;
            if constexpr (T % L == 0) g4_product_first(a[I][ST], w[W], sum[G & 1]);
            else g4_product(a[I][ST], w[W], sum[G & 1]);
            // the sum of a group from two slots behind its last product up to where its registers are wanted again
            constexpr int U = T + SLOTS - L - 1, F = U / L % GROUPS, O = U % L;
            if constexpr (O < L - 1) fold(std::integral_constant<int, F>{}, std::integral_constant<int, 16 * O / (L - 1)>{}, std::integral_constant<int, 16 * (O + 1) / (L - 1)>{});
            if constexpr (T == 0) scale_of(I0{});
            if constexpr (T == 8) scale_of(I1{});
            // (a step's slots are both the ones from its own start and the last ones from the step before)
            decode_some(I1{}, std::integral_constant<int, T - (MID - 8)>{});
            decode_some(I0{}, std::integral_constant<int, T < 8 ? T + 8 : T - (SLOTS - 8)>{});
            if constexpr (T == MID) read_s(next, I0{}), read_w(next, I0{});
            if constexpr (T == MID + 7) read_s(next, I1{}), read_w(next, I1{});
            // operands of rows 0 and 1 behind the barrier, of 2 and 3 early in the next step
            constexpr int N0 = T >= MID + 7 ? T - MID - 7 : T >= 7 && T < 7 + READS ? T - 7 : READS, R = T >= MID ? 0 : 16;
            if constexpr (N0 < READS) {
                constexpr int R0 = R + 16 * N0 / READS, R1 = R + 16 * (N0 + 1) / READS;
                static_for<R1 - R0>([&](auto r) {
                    constexpr int X = R0 + decltype(r)::value;
                    read_a(T >= MID ? next : here, std::integral_constant<int, X / 8>{}, std::integral_constant<int, X % 8>{});
                });
            }
            constexpr int H = T >= MID ? T - MID : T + MID; // (SLOTS = 2 MID)
            if constexpr (H < COPY_SLOTS) {
                constexpr int P0 = S::PAIRS * H / COPY_SLOTS, P1 = S::PAIRS * (H + 1) / COPY_SLOTS;
                static_for<P1 - P0>([&](auto p) { copy(T >= MID ? here : next, std::integral_constant<int, P0 + decltype(p)::value>{}); });
            }
            if constexpr (H == COPY_SLOTS - 1) copied();
            __builtin_amdgcn_sched_barrier(0);
        });
        here = next;
    }
    asm volatile("s_nop 7\n\ts_nop 7" ::: "memory"); // (the last product has to be through)
    fold(std::integral_constant<int, GROUPS - 1>{}, I0{}, std::integral_constant<int, 16>{});
    // a load to LDS must not outlive the workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    if (parts > 1) { // partial tile in accumulator order: [tile][part][wave][i][j][quarter of 16][lane]
        v4f* to = reinterpret_cast<v4f*>(g.scratch) + (((size_t)tile * parts + part) * 4 + wave) * (RM * 2 * 4 * 64) + lane;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    to[((i * 2 + j) * 4 + e) * 64] = v4f{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
    } else {
        const int64_t n = g4_lane_column<SWIGLU>((int64_t)nblk * 2 + wn, lane);
        const auto first = [&](int x) { return m0 + (wm * RM + x / 4) * 32 + 8 * (x % 4) + 4 * (lane >> 5); };
        g4_with_finish<SWIGLU>(g, [&](auto&& exponents4, auto&& finish4) {
            v4i exponents[RM * 4];
#pragma unroll
            for (int x = 0; x < RM * 4; ++x) exponents[x] = exponents4(first(x));
#pragma unroll
            for (int x = 0; x < RM * 4; ++x) finish4(first(x), n, &acc[x / 4][0][x % 4 * 4], &acc[x / 4][1][x % 4 * 4], exponents[x]);
        });
    }
}

// Sum of the parts of a tile, in their order, and the results.  One wave per quarter of 32 rows x 64 places.
template <bool SWIGLU>
__global__ __launch_bounds__(256) void g4_join_kernel(G4Grid t, rkh_g4_args g) {
    constexpr int RM = G4Tile<1>::RM;
    const int lane = lane_id(), e = wave_id();
    const unsigned tile = blockIdx.x / (4 * RM), in_tile = blockIdx.x % (4 * RM), wave = in_tile / RM, i = in_tile % RM;
    const int parts = t.parts;
    int mblk, nblk;
    t.place(tile, mblk, nblk);
    constexpr size_t step = 4 * RM * 512;
    const v4f* from = reinterpret_cast<const v4f*>(g.scratch) + tile * parts * step + (wave * RM + i) * 512 + e * 64 + lane;
    v4f s0 = from[0], s1 = from[256];
#pragma unroll 4
    for (int p = 1; p < parts; ++p) s0 += from[p * step], s1 += from[p * step + 256];
    const float a[4] = {s0.x, s0.y, s0.z, s0.w}, b[4] = {s1.x, s1.y, s1.z, s1.w};
    const int64_t n = g4_lane_column<SWIGLU>((int64_t)nblk * 2 + (wave >> 1), lane);
    const int first = ((mblk * 2 + (int)(wave & 1)) * RM + i) * 32 + 8 * e + 4 * (lane >> 5);
    g4_with_finish<SWIGLU>(g, [&](auto&& exponents4, auto&& finish4) { finish4(first, n, a, b, exponents4(first)); });
}

template <int GPB, bool SWIGLU> int launch_big_tiles(hipStream_t st, const rkh_g4_args& g, const rkk::G4Route& r) {
    constexpr int LDS = G4Tile<GPB>::LDS, RM = G4Tile<GPB>::RM;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(&g4_tile_kernel<GPB, SWIGLU>), opted_in, LDS)) return rc;
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
    if (tiles * r.parts * 256 >= MX_TOO_MANY_THREADS || (r.parts > 1 && tiles * RM * 4 * 256 >= MX_TOO_MANY_THREADS)) return RKH_ERR_RUNTIME;
    const G4Grid t = G4Grid::of(r, g);
    mark(st, "g4_tile_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(g4_tile_kernel<GPB, SWIGLU>), dim3((unsigned)(tiles * r.parts)), dim3(256), LDS, st, t, g);
    RKH_CHECK(hipGetLastError());
    if (r.parts > 1) {
        mark(st, "g4_join_kernel");
        hipLaunchKernelGGL(HIP_KERNEL_NAME(g4_join_kernel<SWIGLU>), dim3((unsigned)(tiles * RM * 4)), dim3(256), 0, st, t, g);
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}

// ---- tiles of few rows -----------------------------------------------------------------
// 32 RM rows x 128 places by four waves, each all of the rows and 32 places: nobody makes the same codes into halves twice, which is what tiles of few rows are
// bound by (128 x 128 x 128 two by two 2020 clocks, this way 1100 - 1700), for twice the reads of activations.  A wave issues some 150 instructions a step of 32
// rows, one in five clocks at best, and eight of them are products: 128 x 8192 x 4096 in 32 rows 15.2 us, in 64 rows 19.7, x 11008 23.7 and 19.9.  Without codes made into
// halves 32 rows x 8192 took 13.2 of 18.4, without LDS reads 16.3, without copies 15.4, without sums added 16.3 (all before the last steps).  Neither more steps under
// way nor codes spread over more of the products change it.
//  * A step's activations live in registers as above, each replaced by the next step's behind its product; the next step's codes become halves in
//    registers of their own, so that two steps make one turn of the loop.
//  * At the start of step s a wave waits for its copies of step s + 1 and for its LDS reads, and meets the others: nobody reads step s any more, and the
//    copies of step s + BUFFERS take its place.  Steps are short, and memory answers after a microsecond: as many are under way as LDS holds.
template <int RM, int GPB> struct G4Rows {
    static constexpr int ROWS = 32 * RM, HALF = ROWS * 128, W_OFF = 2 * HALF, S_OFF = W_OFF + 8192, S_COPIES = GPB == 4 ? 2 : 1, BUF = S_OFF + S_COPIES * 1024,
                         BUFFERS = RM == 1 ? 4 : 3, LDS = BUFFERS * BUF;
    static constexpr int COPIES = 2 * RM + 3; // of a wave and step: activations, codes, scales
    static_assert(LDS <= 160 * 1024, "");
};

// Four rows from `first` on of a lane's column n to results.  (SwiGLU: lanes 16 .. 31 and 48 .. 63 hold what goes with the gates of the 16 before.)
template <int OUT, bool SWIGLU, bool EXPONENTS>
__device__ __forceinline__ void g4_rows_finish4(const rkh_g4_args& g, int first, int64_t n, int lane, const float* s, const v4i& exponents) {
    using T = typename MxType<OUT>::T;
    T* to = static_cast<T*>(g.C) + (size_t)first * g.ldc + n;
    const int live = n < g.N && (!SWIGLU || !(lane & 16)) ? g.M - first : 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = s[e];
        if constexpr (EXPONENTS) v = __builtin_amdgcn_ldexpf(v, exponents[e]);
        if constexpr (SWIGLU) v = mx_silu(v, __shfl_xor(v, 16));
        if (e < live) *to = (T)v;
        to += g.ldc;
    }
}
template <bool SWIGLU, class F> __device__ __forceinline__ void g4_with_rows_finish(const rkh_g4_args& g, int block0, int lane, F&& f) {
    const int64_t n = g4_column(block0 + (lane >> 4 & 1), lane & 15, SWIGLU);
    mx_with_type(g.out_type, [&](auto t) {
        constexpr int OUT = decltype(t)::value;
        const auto go = [&](auto with) {
            constexpr bool EXPONENTS = decltype(with)::value;
            f([&](int first) { return g4_exponents4<EXPONENTS>(g, first); },
              [&](int first, const float* s, const v4i& exponents) { g4_rows_finish4<OUT, SWIGLU, EXPONENTS>(g, first, n, lane, s, exponents); });
        };
        if (g.exponents) go(std::true_type{});
        else go(std::false_type{});
    });
}

template <int RM, int GPB, bool SWIGLU>
__global__ __launch_bounds__(256) void g4_rows_tile_kernel(G4Grid t, rkh_g4_args g) {
    using S = G4Rows<RM, GPB>;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(wave_id());
    const int parts = t.parts, KB = t.KB();
    unsigned tile;
    int part, mblk, nblk;
    t.job(blockIdx.x, tile, part);
    t.place(tile, mblk, nblk);
    const int kb0 = t.begin(part), kb1 = t.begin(part + 1);

    // ---- copies
    const uint32_t base = (uint32_t)(uintptr_t)(mx_lds_ptr)lds;
    const int m0 = mblk * S::ROWS;
    const uint8_t* x_src = static_cast<const uint8_t*>(g.x) + ((size_t)m0 * g.ldx + (size_t)kb0 * 128) * 2;
    const uint8_t* x_src2 = x_src + 128;
    unsigned x_off[RM]; // of eight rows' 128 bytes; rows beyond M: the last one again
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const int row = min(m0 + (wave * RM + r) * 8 + (lane >> 3), g.M - 1) - m0;
        x_off[r] = (unsigned)row * (unsigned)g.ldx * 2 + ((lane & 7) ^ (((wave * RM + r) & 1) * 4 + (lane >> 4))) * 16;
    }
    const uint8_t* w_src[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) w_src[i] = g.W + ((size_t)min(nblk * 8 + wave * 2 + i, t.blocks - 1) * KB + kb0) * 1024 - i * 1024;
    const unsigned s_lane = (GPB == 4 ? (wave & 1) * 1024 : 0) + lane * 16, s_at_tile = s_lane % (512 * GPB);
    const uint8_t* s_src = reinterpret_cast<const uint8_t*>(g.w_scale) + ((size_t)nblk * 8 * KB + kb0) * (64 * GPB);
    const unsigned s_first = (unsigned)min((int)(s_at_tile / (64 * GPB)), t.blocks - 1 - nblk * 8) * (unsigned)KB * (64 * GPB) + s_at_tile % (64 * GPB);
    unsigned w_off = lane * 16, s_off = s_first;
    const uint32_t x_to = base + wave * RM * 1024, w_to = base + S::W_OFF + wave * 2048, s_to = base + S::S_OFF + (GPB == 4 ? (wave & 1) * 1024 : 0);
    int ahead = kb1 - kb0; // steps that are still to be copied
    const auto copy = [&](uint32_t to, auto p_tag) { // statement P: activations of eight rows, 64 k and 64 k; codes; scales
        constexpr int P = decltype(p_tag)::value;
        if constexpr (P < RM) {
            g4_copy<P * 1024>(x_src, x_off[P], to + x_to);
            g4_copy<S::HALF + P * 1024>(x_src2, x_off[P], to + x_to);
        } else if constexpr (P == RM) {
            g4_copy_two(w_src[0], w_src[1], w_off, to, w_to);
        } else {
            g4_copy(s_src, s_off, to, s_to);
        }
    };
    // (a wave issues an instruction every five clocks, scalar ones among them: lanes' offsets advance, not addresses)
    const auto copied = [&]() { // (behind the last step: that one again, which nobody reads)
        const bool more = --ahead > 0;
        const unsigned x_by = more ? 256 : 0, w_by = more ? 1024 : 0, s_by = more ? 64 * GPB : 0;
#pragma unroll
        for (int r = 0; r < RM; ++r) x_off[r] += x_by;
        w_off += w_by;
        s_off += s_by;
    };

    // ---- LDS reads
    uint32_t a_at[4]; // step s of a row's 64 k: s % 4
#pragma unroll
    for (int s = 0; s < 4; ++s) a_at[s] = (lane & 31) * 128 + (((2 * s + (lane >> 5)) ^ (lane >> 1 & 7)) * 16);
    const uint32_t w_at = S::W_OFF + wave * 2048 + (lane >> 4 & 1) * 1024 + (lane & 15) * 16 + (lane >> 5) * 256;
    const uint32_t s_at = S::S_OFF + (wave * 32 + (lane & 31)) * GPB * 4;
    v4i a[RM][8], w[2][8], raw[2];
    typedef uint32_t words __attribute__((ext_vector_type(GPB)));
    words sd;
    float scale[2][GPB];
    const auto read_a = [&](uint32_t from, auto i_tag, auto s_tag) {
        constexpr int I = decltype(i_tag)::value, ST = decltype(s_tag)::value;
        a[I][ST] = *reinterpret_cast<const v4i*>(lds + from + a_at[ST & 3] + (ST >> 2) * S::HALF + I * 4096);
    };
    const auto read_w = [&](uint32_t from) {
        raw[0] = *reinterpret_cast<const v4i*>(lds + from + w_at);
        raw[1] = *reinterpret_cast<const v4i*>(lds + from + w_at + 512);
        sd = *reinterpret_cast<const words*>(lds + from + s_at);
    };

    // ---- codes to operands: pair x (0 .. 31) of a step's eight
    G4Zero zero[GPB];
    uint32_t magic, upper = 0;
    asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(magic));
    const auto decode = [&](auto p_tag, auto x_tag) {
        constexpr int P = decltype(p_tag)::value, X = decltype(x_tag)::value, ST = X / 4, R = X % 4;
        if constexpr (X == 0) {
#pragma unroll
            for (int n = 0; n < GPB; ++n) zero[n].of(sd[n]);
        }
        w[P][ST][R] = (int)g4_pair_here<R>((uint32_t)raw[ST & 1][ST >> 1], zero[ST * GPB / 8], magic, upper);
    };
    const auto decode_dword = [&](auto p_tag, auto st_tag) {
        constexpr int P = decltype(p_tag)::value, ST = decltype(st_tag)::value;
        if constexpr (ST == 0) {
#pragma unroll
            for (int n = 0; n < GPB; ++n) zero[n].of(sd[n]);
        }
        w[P][ST] = g4_dword_here((uint32_t)raw[ST & 1][ST >> 1], zero[ST * GPB / 8], magic);
    };
    const auto scale_of = [&](auto p_tag) {
        constexpr int P = decltype(p_tag)::value;
#pragma unroll
        for (int n = 0; n < GPB; ++n) scale[P][n] = g4_scale(sd[n], g.scale_type);
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;

    // ---- prologue
    static_for<S::BUFFERS>([&](auto b) {
        static_for<RM + 2>([&](auto p) { copy(decltype(b)::value * S::BUF, p); });
        copied();
    });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S::BUFFERS - 1) * S::COPIES) : "memory");
    static_for<RM>([&](auto i) { static_for<8>([&](auto s) { read_a(0, i, s); }); });
    read_w(0);
    static_for<32>([&](auto x) { decode(I0{}, x); });
    scale_of(I0{});

    float acc[RM][16];
    v16f sum[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
        for (int i = 0; i < RM; ++i) acc[i][e] = 0;
        sum[0][e] = sum[1][e] = 0;
    }
#pragma unroll
    for (int n = 0; n < GPB; ++n) scale[1][n] = 0;

    constexpr int L = 8 / GPB, GROUPS = RM * GPB, SLOTS = 8 * RM; // products of a group, groups and slots of a step
    constexpr int CODES_FROM = RM == 1 ? 4 : 6;                   // (codes are read in slot 0)
    const auto fold = [&](auto p_tag, auto g_tag, auto from_tag, auto to_tag) { // elements of the sum of group G of a step of parity P into the accumulators
        constexpr int P = decltype(p_tag)::value, G = decltype(g_tag)::value;
#pragma unroll
        for (int e = from_tag(); e < to_tag(); ++e) g4_add_scaled(acc[G / GPB][e], sum[(P * GROUPS + G) & 1][e], scale[P][G % GPB]);
    };
    uint32_t next = S::BUF, here = 0; // of the next step and this one
    const auto step = [&](auto p_tag) {
        constexpr int P = decltype(p_tag)::value;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S::BUFFERS - 2) * S::COPIES) : "memory");
        static_for<SLOTS>([&](auto t_tag) {
            constexpr int T = decltype(t_tag)::value, ST = T % 8, I = T / 8, G = P * GROUPS + T / L;
            if constexpr (T % L == 0) g4_product_first(a[I][ST], w[P][ST], sum[G & 1]);
            else g4_product(a[I][ST], w[P][ST], sum[G & 1]);
            // the sum of a group from two slots behind its last product up to where its registers are wanted again
            constexpr int U = T + 2 * SLOTS - L - 1, O = U % L, F = (P * GROUPS + U / L) % (2 * GROUPS);
            if constexpr (O < L - 1)
                fold(std::integral_constant<int, F / GROUPS>{}, std::integral_constant<int, F % GROUPS>{}, std::integral_constant<int, 16 * O / (L - 1)>{},
                     std::integral_constant<int, 16 * (O + 1) / (L - 1)>{});
            if constexpr (T == 0) read_w(next);
            if constexpr (RM <= 2 && T >= CODES_FROM) {
                constexpr int N = SLOTS - CODES_FROM, X0 = 8 * (T - CODES_FROM) / N, X1 = 8 * (T + 1 - CODES_FROM) / N;
                static_for<X1 - X0>([&](auto x) { decode_dword(std::integral_constant<int, 1 - P>{}, std::integral_constant<int, X0 + decltype(x)::value>{}); });
            } else if constexpr (T >= CODES_FROM) {
                constexpr int N = SLOTS - CODES_FROM, X0 = 32 * (T - CODES_FROM) / N, X1 = 32 * (T + 1 - CODES_FROM) / N;
                static_for<X1 - X0>([&](auto x) { decode(std::integral_constant<int, 1 - P>{}, std::integral_constant<int, X0 + decltype(x)::value>{}); });
            }
            read_a(next, std::integral_constant<int, I>{}, std::integral_constant<int, ST>{});
            if constexpr (T == SLOTS - 1) scale_of(std::integral_constant<int, 1 - P>{}); // (the step before has been added with its own)
            constexpr int P0 = (RM + 2) * T / SLOTS, P1 = (RM + 2) * (T + 1) / SLOTS;
            static_for<P1 - P0>([&](auto p) { copy(here, std::integral_constant<int, P0 + decltype(p)::value>{}); });
            __builtin_amdgcn_sched_barrier(0);
        });
        copied();
        here = next;
        next = next == (S::BUFFERS - 1) * S::BUF ? 0 : next + S::BUF;
    };
    const auto last = [&](auto p_tag) {
        asm volatile("s_nop 7\n\ts_nop 7" ::: "memory"); // (the last product has to be through)
        fold(p_tag, std::integral_constant<int, GROUPS - 1>{}, I0{}, std::integral_constant<int, 16>{});
    };
    int left = kb1 - kb0;
    for (; left >= 2; left -= 2) {
        step(I0{});
        step(I1{});
    }
    if (left) {
        step(I0{});
        last(I0{});
    } else {
        last(I1{});
    }
    // a load to LDS must not outlive the workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    if (parts > 1) { // partial tile in accumulator order: [tile][part][wave][i][quarter of 16][lane]
        v4f* to = reinterpret_cast<v4f*>(g.scratch) + (((size_t)tile * parts + part) * 4 + wave) * (RM * 4 * 64) + lane;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) to[(i * 4 + e) * 64] = v4f{acc[i][4 * e], acc[i][4 * e + 1], acc[i][4 * e + 2], acc[i][4 * e + 3]};
    } else {
        const auto first = [&](int x) { return m0 + x / 4 * 32 + 8 * (x % 4) + 4 * (lane >> 5); };
        g4_with_rows_finish<SWIGLU>(g, nblk * 8 + wave * 2, lane, [&](auto&& exponents4, auto&& finish4) {
            v4i exponents[RM * 4];
#pragma unroll
            for (int x = 0; x < RM * 4; ++x) exponents[x] = exponents4(first(x));
#pragma unroll
            for (int x = 0; x < RM * 4; ++x) finish4(first(x), &acc[x / 4][x % 4 * 4], exponents[x]);
        });
    }
}

// Sum of the parts, in their order, and the results.  One workgroup per 32 rows x 32 places, one wave per quarter of its accumulator.
template <bool SWIGLU> __global__ __launch_bounds__(256) void g4_rows_join_kernel(G4Grid t, int rm_bits, rkh_g4_args g) {
    const int lane = lane_id(), e = wave_id();
    const unsigned rm = 1u << rm_bits, tile = blockIdx.x >> (2 + rm_bits), wave = blockIdx.x >> rm_bits & 3, i = blockIdx.x & (rm - 1);
    const int parts = t.parts;
    int mblk, nblk;
    t.place(tile, mblk, nblk);
    const size_t step = (size_t)rm * 1024;
    const v4f* from = reinterpret_cast<const v4f*>(g.scratch) + tile * parts * step + (wave * rm + i) * 256 + e * 64 + lane;
    v4f s = from[0];
#pragma unroll 4
    for (int p = 1; p < parts; ++p) s += from[p * step];
    const float v[4] = {s.x, s.y, s.z, s.w};
    const int first = (mblk * rm + (int)i) * 32 + 8 * e + 4 * (lane >> 5);
    g4_with_rows_finish<SWIGLU>(g, nblk * 8 + wave * 2, lane, [&](auto&& exponents4, auto&& finish4) { finish4(first, v, exponents4(first)); });
}

template <int RM, int GPB, bool SWIGLU> int launch_rows_tiles(hipStream_t st, const rkh_g4_args& g, const rkk::G4Route& r) {
    constexpr int LDS = G4Rows<RM, GPB>::LDS;
    static std::atomic<bool> opted_in[64] = {};
    if (const int rc = mx_allow_lds(reinterpret_cast<const void*>(&g4_rows_tile_kernel<RM, GPB, SWIGLU>), opted_in, LDS)) return rc;
    const int64_t tiles = (int64_t)r.mblocks * r.nblocks;
    if (tiles * r.parts * 256 >= MX_TOO_MANY_THREADS || (r.parts > 1 && tiles * RM * 4 * 256 >= MX_TOO_MANY_THREADS)) return RKH_ERR_RUNTIME;
    const G4Grid t = G4Grid::of(r, g);
    mark(st, "g4_rows_tile_kernel");
    hipLaunchKernelGGL(HIP_KERNEL_NAME(g4_rows_tile_kernel<RM, GPB, SWIGLU>), dim3((unsigned)(tiles * r.parts)), dim3(256), LDS, st, t, g);
    RKH_CHECK(hipGetLastError());
    if (r.parts > 1) {
        mark(st, "g4_rows_join_kernel");
        hipLaunchKernelGGL(HIP_KERNEL_NAME(g4_rows_join_kernel<SWIGLU>), dim3((unsigned)(tiles * RM * 4)), dim3(256), 0, st, t, RM / 2, g);
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}

template <int GPB, bool SWIGLU> int launch_tiles(hipStream_t st, const rkh_g4_args& g, const rkk::G4Route& r) {
    switch (r.rm) {
    case 8: return launch_big_tiles<GPB, SWIGLU>(st, g, r);
    case 4: return launch_rows_tiles<4, GPB, SWIGLU>(st, g, r);
    case 2: return launch_rows_tiles<2, GPB, SWIGLU>(st, g, r);
    default: return launch_rows_tiles<1, GPB, SWIGLU>(st, g, r);
    }
}
template <int GPB> int launch_tiles(hipStream_t st, const rkh_g4_args& g, const rkk::G4Route& r) {
    return g.swiglu ? launch_tiles<GPB, true>(st, g, r) : launch_tiles<GPB, false>(st, g, r);
}

} // namespace

#endif // RK_KERNELS_G4_TILE_H
