// The norm of attention heads and their rotation by position: z = rms(x) * w, pairs of z turned by position * inv_freq, one pass over the rows.
//
// Bound by memory for many rows, by one workgroup's round trips for few.  A workgroup takes some rows: it first makes their cosines and sines,
// which all heads share, in LDS; then groups of lanes take a head each.  A lane holds both values of the pairs that it turns, so nothing is
// exchanged but the sum of squares.
#include <algorithm>

#include "rk_heads_shim.h"
#include "rk_kernels_mx4.h"

namespace {

constexpr int HEADS_THREADS = 256;

// PAIRS (4 or 1) pairs of neighbouring indices a unit, UNITS units a lane, LANES lanes a head.
// Unit u < R / 2 / PAIRS: pairs PAIRS u .., the rest of the units 2 PAIRS of the values behind R.
template <int TYPE, int PAIRS, int UNITS, int AT_ONCE, bool NEIGHBOURS>
__global__ __launch_bounds__(HEADS_THREADS) void heads_kernel(rkh_heads_args a, int lanes, int rows_each) {
    using T = typename MxType<TYPE>::T;
    typedef T vec __attribute__((ext_vector_type(PAIRS)));
    typedef vec vec_any __attribute__((aligned(sizeof(T))));
    extern __shared__ __attribute__((aligned(16))) float turns[]; // [row][cos of a pair .., sin of a pair ..]
    const int row0 = a.first + (int)blockIdx.x * rows_each, rows = min(rows_each, a.rows - row0), P = a.R / 2;
    const int P4 = (P + 3) & ~3; // (16-byte places for units of four)
    const int heads = a.q_heads + a.k_heads, lane = threadIdx.x % lanes, groups = HEADS_THREADS / lanes;

    // what a lane's units are: places of the first and the second PAIRS values, and how many of each exist
    int first_at[UNITS], second_at[UNITS], pair[UNITS];
    bool turned[UNITS], any[UNITS], both[UNITS];
    const int turned_units = P / PAIRS;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int unit = lane + u * lanes;
        turned[u] = unit < turned_units;
        pair[u] = turned[u] ? unit * PAIRS : 0;
        if (turned[u]) {
            first_at[u] = NEIGHBOURS ? 2 * PAIRS * unit : PAIRS * unit;
            second_at[u] = NEIGHBOURS ? first_at[u] + PAIRS : P + PAIRS * unit;
        } else {
            first_at[u] = a.R + 2 * PAIRS * (unit - turned_units);
            second_at[u] = first_at[u] + PAIRS;
        }
        any[u] = first_at[u] < a.D; // (units of four end with the head)
        both[u] = any[u] && second_at[u] < a.D;
    }

    // items: heads of the rows, dealt to the groups; AT_ONCE of a group are loaded together
    struct Item { int row, head; };
    const auto next = [&](Item& i) {
        i.head += groups;
        while (i.head >= heads) i.head -= heads, ++i.row;
    };
    const auto base = [&](const Item& i, const void* q, const void* k, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head) {
        const bool is_q = i.head < a.q_heads;
        const int64_t at = is_q ? (int64_t)(row0 + i.row) * q_row + i.head * q_head : (int64_t)(row0 + i.row) * k_row + (i.head - a.q_heads) * k_head;
        return static_cast<T*>(const_cast<void*>(is_q ? q : k)) + at;
    };
    vec x[AT_ONCE][UNITS][2] = {};
    const auto load = [&](Item i) {
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            if (i.row < rows) {
                const T* p = base(i, a.q, a.k, a.q_row, a.q_head, a.k_row, a.k_head);
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    if (any[u]) x[n][u][0] = *reinterpret_cast<const vec_any*>(p + first_at[u]);
                    if (both[u]) x[n][u][1] = *reinterpret_cast<const vec_any*>(p + second_at[u]);
                }
            }
            next(i);
        }
    };
    Item item{0, (int)threadIdx.x / lanes};
    while (item.head >= heads) item.head -= heads, ++item.row;
    load(item);

    float q_weight[UNITS][2][PAIRS], k_weight[UNITS][2][PAIRS];
    if (a.norm) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    const bool is = h ? both[u] : any[u];
                    const int at = (h ? second_at[u] : first_at[u]) + e;
                    q_weight[u][h][e] = is && a.q_weight && a.q_heads ? a.q_weight[at] : 1.0f;
                    k_weight[u][h][e] = is && a.k_weight && a.k_heads ? a.k_weight[at] : 1.0f;
                }
    }

    // angles in turns, reduced in 64 bits: what is left, -1/2 .. 1/2, has no use for more than 32
    for (int i = threadIdx.x; i < rows * P; i += HEADS_THREADS) {
        const int row = i / P, p = i - row * P;
        const int axis = (int)(a.axis_of[p >> 4] >> (2 * (p & 15))) & 3;
        const double angle = (double)a.positions[axis * a.position_axis + row0 + row] * (double)a.inv_freq[p] * 0.15915494309189533577;
        float sine, cosine;
        sincospif((float)(2.0 * (angle - rint(angle))), &sine, &cosine);
        turns[row * 2 * P4 + p] = cosine * a.rotation_scale;
        turns[row * 2 * P4 + P4 + p] = sine * a.rotation_scale;
    }
    __syncthreads();

    while (item.row < rows) {
        Item i = item;
#pragma unroll
        for (int n = 0; n < AT_ONCE; ++n) {
            // (lanes of a group stay together; what a group beyond the last item reduces is nobody's)
            float v[UNITS][2][PAIRS], sum = 0;
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < PAIRS; ++e) {
                        v[u][h][e] = (h ? both[u] : any[u]) ? (float)x[n][u][h][e] : 0.0f;
                        sum = fmaf(v[u][h][e], v[u][h][e], sum);
                    }
            const bool is_q = i.head < a.q_heads;
            if (a.norm) {
                for (int off = 1; off < lanes; off <<= 1) sum += __shfl_xor(sum, off);
                const float factor = mx_norm_factor(sum, a.D, a.eps);
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < PAIRS; ++e) v[u][h][e] = v[u][h][e] * factor * (is_q ? q_weight[u][h][e] : k_weight[u][h][e]);
            }
            if (i.row < rows) {
                T* to = base(i, a.q_out, a.k_out, a.q_out_row, a.q_out_head, a.k_out_row, a.k_out_head);
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    if (turned[u]) {
                        const float* cosine = turns + i.row * 2 * P4 + pair[u];
                        const float* sine = cosine + P4;
                        float c[PAIRS], s[PAIRS];
#pragma unroll
                        for (int e = 0; e < PAIRS; ++e) c[e] = cosine[e], s[e] = sine[e];
#pragma unroll
                        for (int e = 0; e < PAIRS; ++e) {
                            // neighbours: the unit's values one after the other, pair e at 2 e and 2 e + 1
                            float& first = NEIGHBOURS ? v[u][2 * e / PAIRS][2 * e % PAIRS] : v[u][0][e];
                            float& second = NEIGHBOURS ? v[u][(2 * e + 1) / PAIRS][(2 * e + 1) % PAIRS] : v[u][1][e];
                            const float p = first, q = second;
                            first = fmaf(p, c[e], -(q * s[e]));
                            second = fmaf(q, c[e], p * s[e]);
                        }
                    }
                    vec y[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < PAIRS; ++e) y[h][e] = (T)v[u][h][e];
                    if (any[u]) *reinterpret_cast<vec_any*>(to + first_at[u]) = y[0];
                    if (both[u]) *reinterpret_cast<vec_any*>(to + second_at[u]) = y[1];
                }
            }
            next(i);
        }
        item = i;
        load(item);
    }
}

} // namespace

extern "C" int rkh_heads(void* stream, const rkh_heads_args* args) {
    rkh_heads_args a = *args;
    const hipStream_t st = (hipStream_t)stream;
    // four pairs at a time where they come in fours, and so do the values behind them; one otherwise
    const bool fours = a.D % 8 == 0 && a.R % 8 == 0;
    const int units = fours ? a.D / 8 : a.R / 2 + (a.D - a.R + 1) / 2;
    int lanes = 1;
    while (lanes < units && lanes < 64) lanes *= 2;
    const int per_lane = (units + lanes - 1) / lanes;
    const int heads = a.q_heads + a.k_heads;
    const int rows_each = std::max<int64_t>(1, std::min<int64_t>(8, 2048 / ((int64_t)heads * lanes)));
    const size_t lds = (size_t)rows_each * 2 * ((a.R / 2 + 3) & ~3) * 4;
    const int64_t most = (INT64_C(1) << 31) / HEADS_THREADS * rows_each; // rows of a launch
    for (int64_t first = 0; first < args->rows; first += most) {
        a.first = (int)first;
        a.rows = (int)std::min<int64_t>(args->rows, first + most);
        const dim3 grid((unsigned)((a.rows - first + rows_each - 1) / rows_each));
        mark(st, "heads_kernel");
        mx_with_type(a.type, [&](auto t) {
            constexpr int TYPE = decltype(t)::value;
            const auto go = [&](auto n) {
                constexpr bool N = decltype(n)::value;
                const auto kernel = fours           ? heads_kernel<TYPE, 4, 1, 4, N>
                                    : per_lane == 1 ? heads_kernel<TYPE, 1, 1, 4, N>
                                    : per_lane == 2 ? heads_kernel<TYPE, 1, 2, 2, N>
                                                    : heads_kernel<TYPE, 1, 4, 1, N>;
                hipLaunchKernelGGL(kernel, grid, dim3(HEADS_THREADS), lds, st, a, lanes, rows_each);
            };
            if (a.neighbours) go(std::true_type{});
            else go(std::false_type{});
        });
        RKH_CHECK(hipGetLastError());
    }
    return RKH_OK;
}
