// Linear layers on group-scaled 4-bit weights (include/rk_npu_g4.h).  No counterpart in the reference.
#include <climits>
#include <new>

#include "rk_g4_shim.h"
#include "rk_host.h"
#include "rk_npu_g4.h"
#include "rk_values.h"

using namespace rkhost;

struct rk_npu_g4_weights {
    Owner owner;
    rk_npu_g4_weight_config config{};
    DeviceBuffer codes, scales; // as the kernels read them
};

struct rk_npu_g4_workspace {
    Owner owner;
    int rows = 0, K = 0, N = 0;
    DeviceBuffer staged, exponents; // rows that a product does not take as they are
    DeviceBuffer scratch;           // partial tiles
    std::atomic_flag busy = ATOMIC_FLAG_INIT;
};

namespace {

bool half_type(int type) { return type == RK_NPU_MX4_F16 || type == RK_NPU_MX4_BF16; }

rk_npu_g4_weights* create_weights(rk_npu_iommu_domain* domain, const rk_npu_g4_weight_config* config, const uint8_t* codes, const void* scales,
                                  const uint8_t* zeros, bool on_host) {
    if (!domain || !domain->ctx || !config || !codes || !scales || reinterpret_cast<uintptr_t>(scales) % 2 || !valid_length(config->K) || config->N < 1 ||
        config->N > INT_MAX - 127 || config->group < 32 || config->group % 32 || !half_type(config->scale_type) || (config->gate_up && config->N % 2))
        return nullptr;
    std::unique_ptr<rk_npu_g4_weights> w(new (std::nothrow) rk_npu_g4_weights());
    if (!w) return nullptr;
    const int K = config->K, N = config->N, gate_up = config->gate_up ? 1 : 0;
    w->owner.bind(domain);
    w->config = *config;
    w->config.gate_up = gate_up;
    rk_npu_ctx* ctx = domain->ctx;
    const OnDevice device(ctx->device);
    if (!device) return nullptr;
    std::lock_guard<std::mutex> lock(ctx->submit_mutex);
    const size_t groups = (size_t)N * (((int64_t)K + config->group - 1) / config->group);
    DeviceBuffer raw, raw_scales, raw_zeros;
    if (on_host) {
        if (upload(w->owner, raw, codes, (size_t)N * ((K + 1) / 2)) || upload(w->owner, raw_scales, scales, groups * 2) ||
            (zeros && upload(w->owner, raw_zeros, zeros, groups)))
            return nullptr;
        codes = raw.as<>();
        scales = raw_scales.as<>();
        if (zeros) zeros = raw_zeros.as<>();
    }
    const int64_t places = rkh_g4_places(N, gate_up);
    // (one scale per row: groups that are whole pieces)
    const int group = config->group >= K ? (int)rkh_align_up(K, 128) : config->group;
    if (w->codes.alloc(w->owner, rkh_g4_code_bytes(places, K), false) ||
        w->scales.alloc(w->owner, rkh_g4_scale_bytes(places, K, rkh_g4_gpb(group)), false) ||
        rkh_g4_pack(ctx->stream, codes, static_cast<const uint16_t*>(scales), zeros, K, N, group, gate_up, w->codes.as<>(), w->scales.as<uint32_t>()) ||
        rkh_sync(ctx->stream))
        return nullptr;
    return w.release();
}

int run(rk_npu_g4_workspace* ws, const rk_npu_g4_weights* w, bool swiglu, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C, int64_t ldc) {
    if (!ws || !w) return RK_NPU_ERR_PARAM;
    if (!w->owner.same(ws->owner)) return RK_NPU_ERR_DOMAIN;
    const int K = ws->K, N = swiglu ? w->config.N / 2 : w->config.N;
    if (w->config.K != K || w->config.N > ws->N || (w->config.gate_up != 0) != swiglu || rows < 0 || rows > ws->rows || !half_type(a_type) ||
        !valid_rows(A, a_type, rows, lda, K) || !valid_rows(C, c_type, rows, ldc, N) || values(A, a_type, rows, lda, K).meets(values(C, c_type, rows, ldc, N)))
        return RK_NPU_ERR_PARAM;
    BusyLock lock(ws->busy);
    if (!lock) return RK_NPU_ERR_BUSY;
    if (!rows) return RK_NPU_OK;
    rkh_g4_args g{};
    g.W = w->codes.as<>();
    g.w_scale = w->scales.as<uint32_t>();
    g.gpb = rkh_g4_gpb(w->config.group >= K ? 128 : w->config.group);
    g.scale_type = w->config.scale_type;
    g.x = A;
    g.ldx = lda;
    g.x_type = a_type;
    g.M = rows;
    g.N = N;
    g.K = K;
    g.swiglu = swiglu;
    g.out_type = c_type;
    g.C = C;
    g.ldc = ldc;
    g.staged = ws->staged.as<uint16_t>();
    g.exponents = ws->exponents.as<int>();
    g.scratch = ws->scratch.as<float>();
    g.scratch_bytes = ws->scratch.bytes();
    const OnDevice device(ws->owner.ctx->device);
    if (!device) return RK_NPU_ERR_SUBMIT;
    std::lock_guard<std::mutex> submit(ws->owner.ctx->submit_mutex);
    return map_error(rkh_g4_run(ws->owner.ctx->stream, &g));
}

} // namespace

extern "C" {

rk_npu_g4_weights* rk_npu_g4_weights_create(rk_npu_iommu_domain* domain, const rk_npu_g4_weight_config* config, const uint8_t* codes, const void* scales,
                                            const uint8_t* zeros) {
    return create_weights(domain, config, codes, scales, zeros, true);
}
rk_npu_g4_weights* rk_npu_g4_weights_create_device(rk_npu_iommu_domain* domain, const rk_npu_g4_weight_config* config, const uint8_t* codes,
                                                   const void* scales, const uint8_t* zeros) {
    return create_weights(domain, config, codes, scales, zeros, false);
}
void rk_npu_g4_weights_free(rk_npu_g4_weights* weights) { delete weights; }
int rk_npu_g4_weights_query(const rk_npu_g4_weights* weights, rk_npu_g4_weight_config* config, uint64_t* device_bytes) {
    if (!weights) return RK_NPU_ERR_PARAM;
    if (config) *config = weights->config;
    if (device_bytes) *device_bytes = weights->codes.bytes() + weights->scales.bytes();
    return RK_NPU_OK;
}

rk_npu_g4_workspace* rk_npu_g4_workspace_create(rk_npu_iommu_domain* domain, int max_rows, int K, int N) {
    if (!domain || !domain->ctx || max_rows < 1 || max_rows > INT_MAX - 255 || !valid_length(K) || N < 1 || N > INT_MAX - 127) return nullptr;
    std::unique_ptr<rk_npu_g4_workspace> ws(new (std::nothrow) rk_npu_g4_workspace());
    if (!ws) return nullptr;
    ws->owner.bind(domain);
    ws->rows = max_rows;
    ws->K = K;
    ws->N = N;
    const size_t scratch = rkh_g4_scratch_most(max_rows, K);
    const OnDevice device(domain->ctx->device);
    if (!device) return nullptr;
    std::lock_guard<std::mutex> lock(domain->ctx->submit_mutex);
    if (ws->staged.alloc(ws->owner, rkh_g4_staged_bytes(max_rows, K), false) || ws->exponents.alloc(ws->owner, (size_t)rkh_align_up(max_rows, 256) * 4, false) ||
        (scratch && ws->scratch.alloc(ws->owner, scratch, false)))
        return nullptr;
    return ws.release();
}
void rk_npu_g4_workspace_free(rk_npu_g4_workspace* workspace) { delete workspace; }

int rk_npu_g4_run_device(rk_npu_g4_workspace* ws, const rk_npu_g4_weights* w, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C,
                         int64_t ldc) {
    return run(ws, w, false, rows, a_type, A, lda, c_type, C, ldc);
}
int rk_npu_g4_run_swiglu_device(rk_npu_g4_workspace* ws, const rk_npu_g4_weights* w, int rows, int a_type, const void* A, int64_t lda, int c_type, void* C,
                                int64_t ldc) {
    return run(ws, w, true, rows, a_type, A, lda, c_type, C, ldc);
}

} // extern "C"
