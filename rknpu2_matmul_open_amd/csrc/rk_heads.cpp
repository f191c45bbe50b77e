// The norm and rotation of attention heads (include/rk_npu_heads.h).  No counterpart in the reference.
#include <climits>
#include <cstring>

#include "rk_heads_shim.h"
#include "rk_host.h"
#include "rk_npu_heads.h"
#include "rk_values.h"

using namespace rkhost;

namespace {

// A tensor of rows x heads x D values, as rows of one pitch: the stride further apart is the pitch, the other one fills it.
struct Heads {
    const void* p;
    int64_t rows, heads, D, row, head;
    int type;
    bool empty() const { return !rows || !heads; }
    bool rows_hold_heads() const { return rows == 1 || (heads > 1 ? head : D) <= row; }
    int64_t pitch() const { return rows == 1 && heads == 1 ? 0 : heads == 1 ? row : rows == 1 ? head : rows_hold_heads() ? row : head; }
    int64_t outer() const { return heads == 1 ? rows : rows == 1 ? heads : rows_hold_heads() ? rows : heads; }
    int64_t width() const { return heads == 1 || rows == 1 ? D : rows_hold_heads() ? (heads - 1) * head + D : (rows - 1) * row + D; }
    bool valid() const {
        if (empty()) return true;
        const int64_t most = INT64_C(1) << 40, all = INT64_C(1) << 56;
        if (!p || reinterpret_cast<uintptr_t>(p) % type_bytes(type) || (rows > 1 && (row < D || row > most)) || (heads > 1 && (head < D || head > most))) return false;
        // neither the inner extent nor the whole may leave 2^56 values: looked at ahead of the products, which 64 bits need not hold otherwise
        if ((rows > 1 && row > all / rows) || (heads > 1 && head > all / heads)) return false;
        return outer() == 1 || (pitch() >= width() && pitch() <= all / outer());
    }
    Span span() const { return empty() ? Span() : Span(p, outer(), pitch() * type_bytes(type), width() * type_bytes(type)); }
    bool is(const Heads& o) const { return p == o.p && (rows == 1 || row == o.row) && (heads == 1 || head == o.head); }
};

} // namespace

extern "C" {

void rk_npu_heads_args_init(rk_npu_heads_args* args, int rows, int head_dim) {
    if (!args) return;
    *args = rk_npu_heads_args{};
    args->struct_size = sizeof(*args);
    args->rows = rows;
    args->head_dim = args->rotary_dim = head_dim;
    args->norm = args->axes = 1;
    args->eps = 1e-6f;
    args->rotation_scale = 1.0f;
}

int rk_npu_heads_norm_rotate_device(rk_npu_ctx* ctx, const rk_npu_heads_args* a) {
    if (!ctx || !a || a->struct_size != sizeof(*a)) return RK_NPU_ERR_PARAM;
    const int D = a->head_dim, R = a->rotary_dim;
    if (a->rows < 0 || a->rows > INT_MAX - 15 || D < 1 || D > RKH_HEADS_MOST_DIM || a->q_heads < 0 || a->k_heads < 0 || a->q_heads > 1 << 20 || a->k_heads > 1 << 20 || !valid_type(a->type) ||
        R < 0 || R > D || R % 2 || a->axes < 1 || a->axes > 4)
        return RK_NPU_ERR_PARAM;
    if (a->norm ? !(a->eps >= 0.0f) : (a->q_weight || a->k_weight)) return RK_NPU_ERR_PARAM;
    const Heads q{a->q, a->rows, a->q_heads, D, a->q_row, a->q_head, a->type}, k{a->k, a->rows, a->k_heads, D, a->k_row, a->k_head, a->type},
        q_out{a->q_out, a->rows, a->q_heads, D, a->q_out_row, a->q_out_head, a->type}, k_out{a->k_out, a->rows, a->k_heads, D, a->k_out_row, a->k_out_head, a->type};
    if (!q.valid() || !k.valid() || !q_out.valid() || !k_out.valid()) return RK_NPU_ERR_PARAM;
    if (reinterpret_cast<uintptr_t>(a->q_weight) % 4 || reinterpret_cast<uintptr_t>(a->k_weight) % 4) return RK_NPU_ERR_PARAM;
    rkh_heads_args h{};
    const bool some = a->rows && (a->q_heads || a->k_heads);
    if (R) {
        if (some && (!a->positions || !a->inv_freq)) return RK_NPU_ERR_PARAM;
        if (reinterpret_cast<uintptr_t>(a->positions) % 4 || reinterpret_cast<uintptr_t>(a->inv_freq) % 4 || a->position_axis < 0 || a->position_axis > INT64_C(1) << 40)
            return RK_NPU_ERR_PARAM;
        for (int i = 0; a->pair_axis && i < R / 2; ++i) {
            if (a->pair_axis[i] >= a->axes) return RK_NPU_ERR_PARAM;
            h.axis_of[i / 16] |= (uint32_t)a->pair_axis[i] << (2 * (i % 16));
        }
    }
    const Span positions = R ? Span(a->positions, a->axes, a->position_axis * 4, a->rows * INT64_C(4)) : Span();
    const Span vectors[] = {Span(a->norm && a->q_heads ? a->q_weight : nullptr, 1, 0, D * 4), Span(a->norm && a->k_heads ? a->k_weight : nullptr, 1, 0, D * 4),
                            Span(R ? a->inv_freq : nullptr, 1, 0, R * 2)};
    const Span outs[] = {q_out.span(), k_out.span()};
    if (outs[0].meets(outs[1])) return RK_NPU_ERR_PARAM;
    for (const Span& out : outs) {
        if (out.meets(positions)) return RK_NPU_ERR_PARAM;
        for (const Span& in : vectors)
            if (out.meets(in)) return RK_NPU_ERR_PARAM;
    }
    if (outs[0].meets(k.span()) || outs[1].meets(q.span()) || (!q_out.is(q) && outs[0].meets(q.span())) || (!k_out.is(k) && outs[1].meets(k.span())))
        return RK_NPU_ERR_PARAM;
    if (!some) return RK_NPU_OK;
    h.rows = a->rows;
    h.D = D;
    h.R = R;
    h.q_heads = a->q_heads;
    h.k_heads = a->k_heads;
    h.type = a->type;
    h.norm = a->norm ? 1 : 0;
    h.neighbours = a->neighbours ? 1 : 0;
    h.eps = a->eps;
    h.rotation_scale = a->rotation_scale;
    h.q_weight = a->q_weight;
    h.k_weight = a->k_weight;
    h.inv_freq = a->inv_freq;
    h.q = a->q;
    h.k = a->k;
    h.q_out = a->q_out;
    h.k_out = a->k_out;
    h.q_row = a->q_row, h.q_head = a->q_head, h.k_row = a->k_row, h.k_head = a->k_head;
    h.q_out_row = a->q_out_row, h.q_out_head = a->q_out_head, h.k_out_row = a->k_out_row, h.k_out_head = a->k_out_head;
    h.positions = a->positions;
    h.position_axis = a->position_axis;
    const OnDevice device(ctx->device);
    if (!device) return RK_NPU_ERR_SUBMIT;
    std::lock_guard<std::mutex> submit(ctx->submit_mutex);
    return map_error(rkh_heads(ctx->stream, &h));
}

} // extern "C"
