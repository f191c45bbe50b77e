// Microscaled 4-bit linear layers, the norms around them, and the FFN block that runs both (include/rk_npu_mx4.h).
// No counterpart in the reference.
#include <algorithm>
#include <climits>
#include <new>

#include "rk_host.h"
#include "rk_mx4_shim.h"
#include "rk_npu_mx4.h"
#include "rk_rows.h"

using namespace rkhost;

struct rk_npu_mx4_weights {
    Owner owner;
    rk_npu_mx4_weight_config config{};
    DeviceBuffer codes, scales; // operand blocks
};

struct rk_npu_mx4_workspace {
    Owner owner;
    int rows = 0, K = 0, N = 0;
    DeviceBuffer codes, scales; // operand blocks of the staged rows
    DeviceBuffer scratch;       // partial tiles
    int staged = 0;             // rows that run_staged multiplies
    std::atomic_flag busy = ATOMIC_FLAG_INIT;
};

namespace {

bool valid_type(int type) { return type >= RK_NPU_MX4_F32 && type <= RK_NPU_MX4_BF16; }
int64_t type_bytes(int type) { return type == RK_NPU_MX4_F32 ? 4 : 2; }
bool valid_length(int K) { return K > 0 && K <= INT32_MAX / 1024; }

Span values(const void* p, int type, int64_t rows, int64_t ld, int64_t width) {
    return Span(p, rows, ld * type_bytes(type), width * type_bytes(type));
}
// Pointer and stride of rows of values: aligned to the type, no row on the next one, and all of it addressable.
bool valid_rows(const void* p, int type, int64_t rows, int64_t ld, int64_t width) {
    if (rows == 0) return valid_type(type); // (an empty tensor may have no address)
    return valid_type(type) && p && reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0 && ld >= width && ld <= (INT64_C(1) << 40) &&
           ld <= (INT64_C(1) << 56) / rows;
}

rk_npu_mx4_weights* create_weights(rk_npu_iommu_domain* domain, const rk_npu_mx4_weight_config* config, const uint8_t* codes, const uint8_t* scales,
                                   bool on_host) {
    if (!domain || !domain->ctx || !config || !codes || !scales || !valid_length(config->K) || config->N < 1 || config->N > INT_MAX - 127 ||
        (config->gate_up && config->N % 2))
        return nullptr;
    std::unique_ptr<rk_npu_mx4_weights> w(new (std::nothrow) rk_npu_mx4_weights());
    if (!w) return nullptr;
    const int K = config->K, N = config->N, gate_up = config->gate_up ? 1 : 0;
    w->owner.bind(domain);
    w->config = {K, N, gate_up};
    rk_npu_ctx* ctx = domain->ctx;
    std::lock_guard<std::mutex> lock(ctx->submit_mutex);
    const size_t blocks = (size_t)N * ((K + 31) / 32);
    DeviceBuffer raw, raw_scales;
    if (on_host) {
        if (upload(w->owner, raw, codes, blocks * 16) || upload(w->owner, raw_scales, scales, blocks)) return nullptr;
        codes = raw.as<>();
        scales = raw_scales.as<>();
    }
    const int64_t columns = rkh_mx4_columns(N, gate_up);
    if (w->codes.alloc(w->owner, rkh_mx4_code_bytes(columns, K), false) || w->scales.alloc(w->owner, rkh_mx4_scale_bytes(columns, K), false) ||
        rkh_mx4_pack(ctx->stream, codes, scales, K, N, gate_up, w->codes.as<>(), w->scales.as<>()) || rkh_sync(ctx->stream))
        return nullptr;
    return w.release();
}

// Checks that go with a product whatever its rows come from.
int check_pair(const rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, bool gate_up) {
    if (!ws || !w) return RK_NPU_ERR_PARAM;
    if (!w->owner.same(ws->owner)) return RK_NPU_ERR_DOMAIN;
    if (w->config.K != ws->K || w->config.N > ws->N || (w->config.gate_up != 0) != gate_up) return RK_NPU_ERR_PARAM;
    return RK_NPU_OK;
}
int check_rows(const rk_npu_mx4_workspace* ws, int rows, int type, const void* A, int64_t lda) {
    return rows < 0 || rows > ws->rows || !valid_rows(A, type, rows, lda, ws->K) ? RK_NPU_ERR_PARAM : RK_NPU_OK;
}

rkh_mx4_gemm_args product(const rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, int rows) {
    rkh_mx4_gemm_args g{};
    g.A = ws->codes.as<>();
    g.a_scale = ws->scales.as<>();
    g.W = w->codes.as<>();
    g.w_scale = w->scales.as<>();
    g.M = rows;
    g.K = ws->K;
    g.N = w->config.gate_up ? w->config.N / 2 : w->config.N;
    g.swiglu = w->config.gate_up;
    g.scratch = ws->scratch.as<float>();
    g.scratch_bytes = ws->scratch.bytes();
    return g;
}
// Quantization and product: one launch where the kernel takes the rows itself.
int enqueue(rk_npu_mx4_workspace* ws, rkh_mx4_gemm_args g, int type, const void* A, int64_t lda) {
    void* stream = ws->owner.ctx->stream;
    if (rkh_mx4_takes_rows(g.M, g.N, g.K, g.swiglu)) {
        g.A = nullptr;
        g.x = A;
        g.ldx = lda;
        g.x_type = type;
        return map_error(rkh_mx4_gemm(stream, &g));
    }
    const int rc = rkh_mx4_stage(stream, type, g.M, g.K, A, lda, ws->codes.as<>(), ws->scales.as<>());
    return map_error(rc ? rc : rkh_mx4_gemm(stream, &g));
}

int run(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, bool swiglu, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C,
        int64_t ldc) {
    int rc = check_pair(ws, w, swiglu);
    if (!rc) rc = check_rows(ws, rows, a_type, A, lda);
    if (rc) return rc;
    rkh_mx4_gemm_args g = product(ws, w, rows);
    if (!valid_rows(C, c_type, rows, ldc, g.N) || values(A, a_type, rows, lda, ws->K).meets(values(C, c_type, rows, ldc, g.N))) return RK_NPU_ERR_PARAM;
    BusyLock lock(ws->busy);
    if (!lock) return RK_NPU_ERR_BUSY;
    std::lock_guard<std::mutex> submit(ws->owner.ctx->submit_mutex);
    ws->staged = 0;
    if (!rows) return RK_NPU_OK;
    g.out_type = c_type;
    g.C = C;
    g.ldc = ldc;
    return enqueue(ws, g, a_type, A, lda);
}

// The pair of products of an FFN, apart from their rows.
int check_ffn(const rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* gate_up, const rk_npu_mx4_workspace* down_ws, const rk_npu_mx4_weights* down) {
    if (ws == down_ws) return RK_NPU_ERR_PARAM;
    int rc = check_pair(ws, gate_up, true);
    if (!rc) rc = check_pair(down_ws, down, false);
    if (rc) return rc;
    if (!ws->owner.same(down_ws->owner)) return RK_NPU_ERR_DOMAIN;
    return gate_up->config.N / 2 == down->config.K ? RK_NPU_OK : RK_NPU_ERR_PARAM;
}
// gate / up with SwiGLU into down_ws, the first product's arguments given
void to_middle(rkh_mx4_gemm_args& g, const rk_npu_mx4_workspace* down_ws) {
    g.out_type = RKH_MX4_ROWS;
    g.C = down_ws->codes.as<>();
    g.c_scale = down_ws->scales.as<>();
}

// Range checks of a norm's arguments; `branch`: whether there is one for the gate to go with.
int check_norm(const rk_npu_block_norm_args* a, bool branch) {
    if (!a || a->struct_size != sizeof(*a) || a->rows < 0 || a->D < 1 || a->D > INT32_MAX / 1024) return RK_NPU_ERR_PARAM;
    const int64_t rows = a->rows, D = a->D;
    if (!valid_rows(a->residual, a->residual_type, rows, a->residual_ld, D) || (a->branch && !valid_rows(a->branch, a->branch_type, rows, a->branch_ld, D)) ||
        (a->residual_out && !valid_rows(a->residual_out, a->residual_type, rows, a->residual_out_ld, D)) ||
        (a->y && !valid_rows(a->y, a->y_type, rows, a->y_ld, D)))
        return RK_NPU_ERR_PARAM;
    if (a->gate && (!branch || !valid_rows(a->gate, a->gate_type, a->gate_ld ? rows : 1, a->gate_ld ? a->gate_ld : D, D)))
        return RK_NPU_ERR_PARAM;
    if ((a->branch_weight && !branch) || reinterpret_cast<uintptr_t>(a->branch_weight) % 4 || reinterpret_cast<uintptr_t>(a->weight) % 4) return RK_NPU_ERR_PARAM;
    if (!(a->eps >= 0.0f)) return RK_NPU_ERR_PARAM;
    return RK_NPU_OK;
}
// No output on an input or on another output, but the stream on itself.  `branch`: the FFN's, an output.
bool norm_overlaps(const rk_npu_block_norm_args* a, const void* branch, const float* next_weight) {
    const int64_t rows = a->rows, D = a->D;
    const Span residual = values(a->residual, a->residual_type, rows, a->residual_ld, D), out = values(a->residual_out, a->residual_type, rows, a->residual_out_ld, D),
               y = values(a->y, a->y_type, rows, a->y_ld, D);
    const Span written = values(branch, a->branch_type, rows, a->branch_ld, D);
    const Span inputs[] = {values(a->branch, a->branch_type, rows, a->branch_ld, D),
                           values(a->gate, a->gate_type, a->gate_ld ? rows : 1, a->gate_ld ? a->gate_ld : D, D),
                           Span(a->branch_weight, 1, 0, D * 4), Span(a->weight, 1, 0, D * 4), Span(next_weight, 1, 0, D * 4)};
    for (const Span& in : inputs)
        if (out.meets(in) || y.meets(in) || written.meets(in)) return true;
    if (written.meets(residual) || written.meets(out) || written.meets(y)) return true;
    const bool in_place = a->residual_out == a->residual && a->residual_out_ld == a->residual_ld;
    return y.meets(out) || y.meets(residual) || (!in_place && out.meets(residual));
}
rkh_block_norm_args norm_args(const rk_npu_block_norm_args* a) {
    rkh_block_norm_args n{};
    n.rows = a->rows;
    n.D = a->D;
    n.stream_type = a->residual_type;
    n.branch_type = a->branch_type;
    n.gate_type = a->gate_type;
    n.y_type = a->y_type;
    n.eps = a->eps;
    n.residual_scale = a->residual_scale;
    n.branch_scale = a->branch_scale;
    n.stream = a->residual;
    n.branch = a->branch;
    n.gate = a->gate;
    n.branch_weight = a->branch_weight;
    n.weight = a->weight;
    n.stream_out = a->residual_out;
    n.y = a->y;
    n.ld_stream = a->residual_ld;
    n.ld_branch = a->branch_ld;
    n.gate_row_stride = a->gate_ld;
    n.ld_stream_out = a->residual_out_ld;
    n.ld_y = a->y_ld;
    return n;
}

} // namespace

extern "C" {

int rk_npu_mx4_quantize_device(rk_npu_ctx* ctx, int type, int64_t rows, int K, const void* x, int64_t ldx, uint8_t* codes, uint8_t* scales) {
    if (!ctx || rows < 0 || rows > INT64_C(1) << 40 || !valid_length(K) || !valid_rows(x, type, rows, ldx, K) ||
        (rows && (!codes || !scales)))
        return RK_NPU_ERR_PARAM;
    const int64_t blocks = (K + 31) / 32;
    const Span in = values(x, type, rows, ldx, K), c(codes, rows, blocks * 16, blocks * 16), s(scales, rows, blocks, blocks);
    if (rows * blocks > (INT64_C(1) << 38) || c.meets(in) || s.meets(in) || c.meets(s)) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::mutex> submit(ctx->submit_mutex);
    return map_error(rkh_mx4_quantize(ctx->stream, type, rows, K, x, ldx, codes, scales));
}

int rk_npu_mx4_dequantize_device(rk_npu_ctx* ctx, int type, int64_t rows, int K, const uint8_t* codes, const uint8_t* scales, void* y, int64_t ldy) {
    if (!ctx || rows < 0 || rows > INT64_C(1) << 40 || !valid_length(K) || !valid_rows(y, type, rows, ldy, K) ||
        (rows && (!codes || !scales)))
        return RK_NPU_ERR_PARAM;
    const int64_t blocks = (K + 31) / 32;
    const Span out = values(y, type, rows, ldy, K), c(codes, rows, blocks * 16, blocks * 16), s(scales, rows, blocks, blocks);
    if (rows * blocks > (INT64_C(1) << 38) || c.meets(out) || s.meets(out)) return RK_NPU_ERR_PARAM;
    std::lock_guard<std::mutex> submit(ctx->submit_mutex);
    return map_error(rkh_mx4_dequantize(ctx->stream, type, rows, K, codes, scales, y, ldy));
}

rk_npu_mx4_weights* rk_npu_mx4_weights_create(rk_npu_iommu_domain* domain, const rk_npu_mx4_weight_config* config, const uint8_t* codes,
                                              const uint8_t* scales) {
    return create_weights(domain, config, codes, scales, true);
}
rk_npu_mx4_weights* rk_npu_mx4_weights_create_device(rk_npu_iommu_domain* domain, const rk_npu_mx4_weight_config* config, const uint8_t* codes,
                                                     const uint8_t* scales) {
    return create_weights(domain, config, codes, scales, false);
}
void rk_npu_mx4_weights_free(rk_npu_mx4_weights* weights) { delete weights; }
int rk_npu_mx4_weights_query(const rk_npu_mx4_weights* weights, rk_npu_mx4_weight_config* config, uint64_t* device_bytes) {
    if (!weights) return RK_NPU_ERR_PARAM;
    if (config) *config = weights->config;
    if (device_bytes) *device_bytes = weights->codes.bytes() + weights->scales.bytes();
    return RK_NPU_OK;
}

rk_npu_mx4_workspace* rk_npu_mx4_workspace_create(rk_npu_iommu_domain* domain, int max_rows, int K, int N) {
    if (!domain || !domain->ctx || max_rows < 1 || max_rows > INT_MAX - 255 || !valid_length(K) || N < 1 || N > INT_MAX - 127) return nullptr;
    std::unique_ptr<rk_npu_mx4_workspace> ws(new (std::nothrow) rk_npu_mx4_workspace());
    if (!ws) return nullptr;
    ws->owner.bind(domain);
    ws->rows = max_rows;
    ws->K = K;
    ws->N = N;
    // what any of the calls may ask for, so that a result does not depend on the workspace's sizes
    const size_t scratch = rkh_mx4_scratch_most(max_rows, K);
    std::lock_guard<std::mutex> lock(domain->ctx->submit_mutex);
    // (zeros: blocks beyond K are read and never written by the SwiGLU epilogue)
    if (ws->codes.alloc(ws->owner, rkh_mx4_code_bytes(max_rows, K), true) || ws->scales.alloc(ws->owner, rkh_mx4_scale_bytes(max_rows, K), true) ||
        (scratch && ws->scratch.alloc(ws->owner, scratch, false)) || rkh_sync(domain->ctx->stream))
        return nullptr;
    return ws.release();
}
void rk_npu_mx4_workspace_free(rk_npu_mx4_workspace* workspace) { delete workspace; }

int rk_npu_mx4_run_device(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C,
                          int64_t ldc) {
    return run(ws, w, false, rows, a_type, A, lda, c_type, C, ldc);
}
int rk_npu_mx4_run_swiglu_device(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, int rows, int a_type, const void* A, int64_t lda, int c_type,
                                 void* C, int64_t ldc) {
    return run(ws, w, true, rows, a_type, A, lda, c_type, C, ldc);
}

int rk_npu_mx4_stage_device(rk_npu_mx4_workspace* ws, int rows, int a_type, const void* A, int64_t lda) {
    if (!ws) return RK_NPU_ERR_PARAM;
    int rc = check_rows(ws, rows, a_type, A, lda);
    if (rc) return rc;
    BusyLock lock(ws->busy);
    if (!lock) return RK_NPU_ERR_BUSY;
    std::lock_guard<std::mutex> submit(ws->owner.ctx->submit_mutex);
    rc = map_error(rkh_mx4_stage(ws->owner.ctx->stream, a_type, rows, ws->K, A, lda, ws->codes.as<>(), ws->scales.as<>()));
    ws->staged = rc ? 0 : rows;
    return rc;
}
int rk_npu_mx4_run_staged_device(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* w, int c_type, void* C, int64_t ldc) {
    int rc = check_pair(ws, w, w && w->config.gate_up);
    if (rc) return rc;
    BusyLock lock(ws->busy);
    if (!lock) return RK_NPU_ERR_BUSY;
    rkh_mx4_gemm_args g = product(ws, w, ws->staged);
    if (!ws->staged || !valid_rows(C, c_type, g.M, ldc, g.N)) return RK_NPU_ERR_PARAM;
    g.out_type = c_type;
    g.C = C;
    g.ldc = ldc;
    std::lock_guard<std::mutex> submit(ws->owner.ctx->submit_mutex);
    return map_error(rkh_mx4_gemm(ws->owner.ctx->stream, &g));
}

int rk_npu_mx4_run_ffn_device(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* gate_up, rk_npu_mx4_workspace* down_ws, const rk_npu_mx4_weights* down,
                              int rows, int a_type, const void* A, int64_t lda, int c_type, void* C, int64_t ldc) {
    int rc = check_ffn(ws, gate_up, down_ws, down);
    if (!rc) rc = check_rows(ws, rows, a_type, A, lda);
    if (rc) return rc;
    if (rows > down_ws->rows || !valid_rows(C, c_type, rows, ldc, down->config.N) ||
        values(A, a_type, rows, lda, ws->K).meets(values(C, c_type, rows, ldc, down->config.N)))
        return RK_NPU_ERR_PARAM;
    BusyLock lock(ws->busy), down_lock(down_ws->busy);
    if (!lock || !down_lock) return RK_NPU_ERR_BUSY;
    std::lock_guard<std::mutex> submit(ws->owner.ctx->submit_mutex);
    ws->staged = down_ws->staged = 0;
    if (!rows) return RK_NPU_OK;
    rkh_mx4_gemm_args g = product(ws, gate_up, rows), d = product(down_ws, down, rows);
    to_middle(g, down_ws);
    rc = enqueue(ws, g, a_type, A, lda);
    if (rc) return rc;
    d.out_type = c_type;
    d.C = C;
    d.ldc = ldc;
    return map_error(rkh_mx4_gemm(ws->owner.ctx->stream, &d));
}

void rk_npu_block_norm_args_init(rk_npu_block_norm_args* args, int rows, int D) {
    if (!args) return;
    *args = rk_npu_block_norm_args{};
    args->struct_size = sizeof(*args);
    args->rows = rows;
    args->D = D;
    args->eps = 1e-6f;
    args->residual_scale = args->branch_scale = 1.0f;
}

int rk_npu_block_norm_device(rk_npu_ctx* ctx, const rk_npu_block_norm_args* a) {
    if (!ctx || !a) return RK_NPU_ERR_PARAM;
    int rc = check_norm(a, a->branch != nullptr);
    if (rc) return rc;
    rk_npu_mx4_workspace* ws = a->staged;
    if ((a->rows && !a->residual_out && !a->y && !ws) || norm_overlaps(a, nullptr, nullptr)) return RK_NPU_ERR_PARAM;
    if (ws && (ws->owner.ctx != ctx || ws->owner.ctx_id != ctx->id)) return RK_NPU_ERR_DOMAIN;
    if (ws && (a->D != ws->K || a->rows > ws->rows)) return RK_NPU_ERR_PARAM;
    std::atomic_flag none = ATOMIC_FLAG_INIT;
    BusyLock lock(ws ? ws->busy : none);
    if (!lock) return RK_NPU_ERR_BUSY;
    rkh_block_norm_args n = norm_args(a);
    if (ws) {
        n.q = ws->codes.as<>();
        n.q_scale = ws->scales.as<>();
    }
    std::lock_guard<std::mutex> submit(ctx->submit_mutex);
    rc = map_error(rkh_block_norm(ctx->stream, &n));
    if (ws) ws->staged = rc ? 0 : a->rows;
    return rc;
}

int rk_npu_mx4_run_ffn_block_device(rk_npu_mx4_workspace* ws, const rk_npu_mx4_weights* gate_up, rk_npu_mx4_workspace* down_ws,
                                    const rk_npu_mx4_weights* down, const rk_npu_block_norm_args* a, void* branch, const float* next_weight) {
    int rc = check_ffn(ws, gate_up, down_ws, down);
    if (!rc) rc = check_norm(a, true);
    if (rc) return rc;
    if (a->branch || a->staged || (a->rows && !a->residual_out && !a->y) || !valid_rows(branch, a->branch_type, a->rows, a->branch_ld, a->D) ||
        a->D != ws->K || a->D != down->config.N || a->rows > ws->rows || a->rows > down_ws->rows || reinterpret_cast<uintptr_t>(next_weight) % 4 || norm_overlaps(a, branch, next_weight))
        return RK_NPU_ERR_PARAM;
    BusyLock lock(ws->busy), down_lock(down_ws->busy);
    if (!lock || !down_lock) return RK_NPU_ERR_BUSY;
    rk_npu_ctx* ctx = ws->owner.ctx;
    std::lock_guard<std::mutex> submit(ctx->submit_mutex);
    ws->staged = down_ws->staged = 0;
    if (!a->rows) return RK_NPU_OK;
    rkh_mx4_gemm_args g = product(ws, gate_up, a->rows), d = product(down_ws, down, a->rows);
    to_middle(g, down_ws);
    d.out_type = a->branch_type;
    d.C = branch;
    d.ldc = a->branch_ld;
    rkh_block_norm_args after = norm_args(a);
    after.branch = branch;
    after.weight = next_weight;
    if (rkh_mx4_takes_rows(g.M, g.N, g.K, 1)) { // h is made where it is multiplied
        g.A = nullptr;
        g.x = a->residual;
        g.ldx = a->residual_ld;
        g.x_type = a->residual_type;
        g.x_norm = 1;
        g.x_weight = a->weight;
        g.x_eps = a->eps;
    } else {
        rkh_block_norm_args before{}; // h, straight to the first product's rows
        before.rows = a->rows;
        before.D = a->D;
        before.stream_type = a->residual_type;
        before.eps = a->eps;
        before.stream = a->residual;
        before.ld_stream = a->residual_ld;
        before.weight = a->weight;
        before.q = ws->codes.as<>();
        before.q_scale = ws->scales.as<>();
        rc = rkh_block_norm(ctx->stream, &before);
    }
    if (!rc) rc = rkh_mx4_gemm(ctx->stream, &g);
    if (!rc) rc = rkh_mx4_gemm(ctx->stream, &d);
    if (!rc) rc = rkh_block_norm(ctx->stream, &after);
    return map_error(rc);
}

} // extern "C"
