// The norm of attention heads and their rotation by position: z = rms(x) * w, pairs of z turned by position * inv_freq, one pass over the rows.
//
// Bound by memory for many rows, by one workgroup's round trips for few.  A thread keeps its place in its head through some rows, so that weights and
// addresses are fetched and made once; it holds both values of the pairs that it turns, so that nothing is exchanged but the sum of squares.  The rows' cosines
// and sines, which all heads share, are made in LDS while the rows are on their way.
// 8192 rows of 40 heads of 128 (bf16, norm): 34 us, 4.9 TB/s; two rows a workgroup 38, one 51; with half of the values a thread, and heads dealt out one by one, 52 us.
// 8192 rows of 20 heads of 90, 60 of them turned: bf16 18.8 us, fp32 30.3; a pair a time 31.3 and 35.6.
#include <algorithm>

#include "rk_heads_shim.h"
#include "rk_kernels_mx4.h"

namespace {

constexpr int HEADS_MOST_THREADS = 256;

// Places for a row's cosines, and its sines: those of the units' pairs one behind the other.
__host__ __device__ constexpr int heads_table(int R) { return (R / 2 + 7) & ~7; }

// Sum over aligned groups of `lanes` lanes, a power of two; every lane of a group gets the same bits.
__device__ __forceinline__ float heads_sum(float x, int lanes) {
    const auto add = [&](auto ctrl) { x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, true)); };
    if (lanes > 1) add(std::integral_constant<int, 0xB1>{});  // lanes 1 0 3 2
    if (lanes > 2) add(std::integral_constant<int, 0x4E>{});  // lanes 2 3 0 1
    if (lanes > 4) add(std::integral_constant<int, 0x141>{}); // 7 .. 0 of eight
    if (lanes > 8) add(std::integral_constant<int, 0x140>{}); // 15 .. 0 of sixteen
    if (lanes > 16) x += __shfl_xor(x, 16);
    if (lanes > 32) x += __shfl_xor(x, 32);
    return x;
}

// PAIRS (8, 4 or 1) pairs of neighbouring indices a unit, UNITS units a thread, 2^lane_bits threads a head, heads_each heads and ROWS rows a workgroup.
// The first units are turned: PAIRS pairs, from pair PAIRS u on; the others are 2 PAIRS of the values behind R.
// RAGGED: what is turned, or the rest, is not in whole units.  The last unit of either begins earlier, so that it is whole, and keeps only what it does not share
// with the one before; where there is no one before, it reaches beyond and keeps only its own.
template <int TYPE, int PAIRS, int UNITS, int ROWS, bool NEIGHBOURS, bool RAGGED>
__global__ __launch_bounds__(HEADS_MOST_THREADS) void heads_kernel(rkh_heads_args a, int lane_bits, int heads_each, int chunks, MxDivider by_chunks, MxDivider by_turns) {
    using T = typename MxType<TYPE>::T;
    typedef T vec __attribute__((ext_vector_type(PAIRS)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    extern __shared__ __attribute__((aligned(16))) float turns[]; // [row][cos of a pair .., sin of a pair ..]
    const int block = (int)by_chunks.divide(blockIdx.x), chunk = (int)blockIdx.x - block * chunks;
    const int row0 = a.first + block * ROWS, P = a.R / 2, table = heads_table(a.R);
    const int lanes = 1 << lane_bits, lane = (int)threadIdx.x & (lanes - 1), slot = (int)threadIdx.x >> lane_bits, head = chunk * heads_each + slot, heads = a.q_heads + a.k_heads;
    const bool live = slot < heads_each && head < heads, is_q = head < a.q_heads;

    // where a thread's units are: places of the first and the second PAIRS values, and which of those it keeps
    int at[UNITS][2], from_e[UNITS][2], to_e[UNITS][2], turn[UNITS];
    bool turned[UNITS], shares[UNITS][2]; // (whether all of the PAIRS values are of its kind)
    const int turned_units = (P + PAIRS - 1) / PAIRS;
    const auto first_pair = [&](int unit) { return RAGGED ? max(0, min(unit * PAIRS, P - PAIRS)) : unit * PAIRS; };
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int unit = lane + u * lanes;
        turned[u] = unit < turned_units;
        turn[u] = turned[u] ? unit * PAIRS : 0;
        if (turned[u]) {
            const int pair = first_pair(unit), own = unit * PAIRS - pair, end = min(P - pair, PAIRS); // first, first and last kept of the unit
            at[u][0] = NEIGHBOURS ? 2 * pair : pair;
            at[u][1] = NEIGHBOURS ? at[u][0] + PAIRS : P + pair;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                from_e[u][s] = NEIGHBOURS ? 2 * own - s * PAIRS : own;
                to_e[u][s] = NEIGHBOURS ? 2 * end - s * PAIRS : end;
            }
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int first = a.R + PAIRS * (2 * (unit - turned_units) + s);
                at[u][s] = RAGGED ? min(first, a.D - PAIRS) : first;
                from_e[u][s] = first - at[u][s]; // (PAIRS and more: nothing)
                to_e[u][s] = first < a.D ? PAIRS : 0;
            }
        }
        // (what does not exist is read where something does, and dropped)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            shares[u][s] = turned[u] ? P >= PAIRS : at[u][s] >= a.R;
            if (!live || at[u][s] + PAIRS > a.D) at[u][s] = to_e[u][s] = 0;
        }
    }
    const auto keeps = [&](int u, int s, int e) { return RAGGED ? e >= from_e[u][s] && e < to_e[u][s] : to_e[u][s] > 0; };
    const int h = live ? is_q ? head : head - a.q_heads : 0;
    const bool from_q = live ? is_q : a.q_heads > 0;
    const int64_t row_stride = from_q ? a.q_row : a.k_row, out_stride = from_q ? a.q_out_row : a.k_out_row;
    const T* from = static_cast<const T*>(from_q ? a.q : a.k) + h * (from_q ? a.q_head : a.k_head);
    T* to = static_cast<T*>(from_q ? a.q_out : a.k_out) + h * (from_q ? a.q_out_head : a.k_out_head);

    vec x[ROWS][UNITS][2]; // (rows beyond the last: that one again)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const T* p = from + (int64_t)min(row0 + r, a.rows - 1) * row_stride;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s) x[r][u][s] = *reinterpret_cast<const vec_any*>(p + at[u][s]);
    }
    typedef float fvec __attribute__((ext_vector_type(PAIRS)));
    typedef fvec fvec_any __attribute__((aligned(4)));
    fvec weight[UNITS][2];
    const float* w = from_q ? a.q_weight : a.k_weight;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int s = 0; s < 2; ++s) weight[u][s] = w ? *reinterpret_cast<const fvec_any*>(w + at[u][s]) : fvec(1.0f);

    // angles in turns, reduced in 64 bits: what is left, -1/2 .. 1/2, has no use for more than 32
    const int turns_of_row = turned_units * PAIRS;
    for (int i = threadIdx.x; i < min(ROWS, a.rows - row0) * turns_of_row; i += blockDim.x) {
        const int row = ROWS == 1 ? 0 : (int)by_turns.divide(i), at_row = i - row * turns_of_row;
        const int p = RAGGED ? min(first_pair(at_row / PAIRS) + at_row % PAIRS, P - 1) : at_row;
        const int axis = (int)(a.axis_of[p >> 4] >> (2 * (p & 15))) & 3;
        const double angle = (double)a.positions[axis * a.position_axis + row0 + row] * (double)a.inv_freq[p] * 0.15915494309189533577;
        float sine, cosine;
        sincospif((float)(2.0 * (angle - rint(angle))), &sine, &cosine);
        turns[row * 2 * table + at_row] = cosine * a.rotation_scale;
        turns[row * 2 * table + table + at_row] = sine * a.rotation_scale;
    }
    __syncthreads();

#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        if (row0 + r >= a.rows) break;
        if constexpr (RAGGED && PAIRS > 1) { // all of the row has been read before any of it is written
            typedef int words __attribute__((ext_vector_type(PAIRS * sizeof(T) / 4)));
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                words first = __builtin_bit_cast(words, x[r][u][0]), second = __builtin_bit_cast(words, x[r][u][1]);
                asm volatile("" : "+v"(first), "+v"(second));
                x[r][u][0] = __builtin_bit_cast(vec, first), x[r][u][1] = __builtin_bit_cast(vec, second);
            }
        }
        float v[UNITS][2][PAIRS], sum = 0;
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    v[u][s][e] = (float)x[r][u][s][e];
                    const float counted = keeps(u, s, e) ? v[u][s][e] : 0.0f;
                    sum = fmaf(counted, counted, sum);
                }
        if (a.norm) {
            const float factor = mx_norm_factor(heads_sum(sum, lanes), a.D, a.eps);
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int e = 0; e < PAIRS; ++e) v[u][s][e] = v[u][s][e] * factor * weight[u][s][e];
        }
        T* row_to = to + (int64_t)(row0 + r) * out_stride;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            if (turned[u]) {
                const float* cosine = turns + r * 2 * table + turn[u];
                const float* sine = cosine + table;
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    // neighbours: the unit's values one after the other, pair e at 2 e and 2 e + 1
                    float& first = NEIGHBOURS ? v[u][2 * e / PAIRS][2 * e % PAIRS] : v[u][0][e];
                    float& second = NEIGHBOURS ? v[u][(2 * e + 1) / PAIRS][(2 * e + 1) % PAIRS] : v[u][1][e];
                    const float p = first, q = second;
                    first = fmaf(p, cosine[e], -(q * sine[e]));
                    second = fmaf(q, cosine[e], p * sine[e]);
                }
            }
            vec y[2];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) y[s][e] = (T)v[u][s][e];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                T* p = row_to + at[u][s];
                // (ragged: streaming stores of parts of lines take three times as long; values that two units share are stored twice, the same)
                if constexpr (!RAGGED) {
                    if (to_e[u][s] > 0) __builtin_nontemporal_store(y[s], reinterpret_cast<vec_any*>(p));
                } else if (to_e[u][s] <= 0 || from_e[u][s] >= PAIRS) {
                } else if (shares[u][s]) {
                    *reinterpret_cast<vec_any*>(p) = y[s];
                } else {
#pragma unroll
                    for (int e = 0; e < PAIRS; ++e)
                        if (keeps(u, s, e)) p[e] = y[s][e];
                }
            }
        }
    }
}

} // namespace

extern "C" int rkh_heads(void* stream, const rkh_heads_args* args) {
    rkh_heads_args a = *args;
    const hipStream_t st = (hipStream_t)stream;
    // 16 bytes of each half at a time, of both for the shortest heads, or single pairs
    const int pairs = a.type != RKH_MX4_F32 && a.D >= 16 ? 8 : a.D >= 8 ? 4 : 1;
    const bool ragged = a.R % (2 * pairs) || (a.D - a.R) % (2 * pairs);
    const int units = (a.R / 2 + pairs - 1) / pairs + (a.D - a.R + 2 * pairs - 1) / (2 * pairs);
    int lane_bits = 0;
    while (1 << lane_bits < units && lane_bits < 6) ++lane_bits;
    const int lanes = 1 << lane_bits;
    const int per_lane = (units + lanes - 1) / lanes; // (two for ragged heads of nearly 512 values)
    const int heads = a.q_heads + a.k_heads, most_heads = HEADS_MOST_THREADS / lanes, chunks = (heads + most_heads - 1) / most_heads;
    const int heads_each = (heads + chunks - 1) / chunks, threads = (int)rkh_align_up((int64_t)heads_each * lanes, 64);
    // several rows a workgroup where that leaves enough of them (one row / four: 256 rows of 40 heads of 128 in bf16 4.2 / 5.5 us, 1000 rows 8.5 / 7.5; 1521
    // rows of 20 heads of 96 in fp32 12.1 / 7.4)
    const bool many = per_lane == 1 && (int64_t)a.rows * chunks >= 1024;
    const int rows_each = many ? 4 : 1;
    const MxDivider by_chunks = MxDivider::of(chunks), by_turns = MxDivider::of(std::max(1, (a.R / 2 + pairs - 1) / pairs * pairs));
    const size_t lds = (size_t)rows_each * 2 * heads_table(a.R) * 4;
    const int64_t most = std::max<int64_t>(1, (INT64_C(1) << 31) / threads / chunks) * rows_each; // rows of a launch, which holds fewer than 2^32 threads
    for (int64_t first = 0; first < args->rows; first += most) {
        a.first = (int)first;
        a.rows = (int)std::min<int64_t>(args->rows, first + most);
        const dim3 grid((unsigned)((a.rows - first + rows_each - 1) / rows_each * chunks));
        mark(st, "heads_kernel");
        mx_with_type(a.type, [&](auto t) {
            constexpr int TYPE = decltype(t)::value, WIDE = TYPE == RKH_MX4_F32 ? 4 : 8;
            const auto go = [&](auto n, auto rg) {
                constexpr bool N = decltype(n)::value, RG = decltype(rg)::value;
                const auto kernel = pairs == 8      ? many ? heads_kernel<TYPE, WIDE, 1, 4, N, RG> : heads_kernel<TYPE, WIDE, 1, 1, N, RG>
                                    : pairs == 1    ? many ? heads_kernel<TYPE, 1, 1, 4, N, true> : heads_kernel<TYPE, 1, 1, 1, N, true>
                                    : per_lane == 1 ? many ? heads_kernel<TYPE, 4, 1, 4, N, RG> : heads_kernel<TYPE, 4, 1, 1, N, RG>
                                                    : heads_kernel<TYPE, 4, 2, 1, N, true>;
                hipLaunchKernelGGL(kernel, grid, dim3((unsigned)threads), lds, st, a, lane_bits, heads_each, chunks, by_chunks, by_turns);
            };
            if (a.neighbours) ragged ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
            else ragged ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
        });
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}
