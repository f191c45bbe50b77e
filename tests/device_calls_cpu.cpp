// The host layers of G4 layers and of the heads over devices made of host memory: on which device a launch is made, and that none is made where the context's could
// not be made current.  Ends with 0 or says what is wrong.
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "rk_g4_shim.h"
#include "rk_heads_shim.h"
#include "rk_hip_shim.h"
#include "rk_npu_g4.h"
#include "rk_npu_heads.h"
#include "rk_npu_hip.h"

static int g_current = 1;      // the calling thread's device; the context's is 0
static bool g_lost = false;    // .. which cannot be made current
static int g_launches, g_elsewhere, g_live;

static int launch() {
    ++g_launches;
    g_elsewhere += g_current != 0;
    return RKH_OK;
}

extern "C" {
int rkh_device_count(void) { return 2; }
int rkh_open(int, void** s, char* name, int, int* cus, int* khz) {
    static char stream;
    *s = &stream;
    name[0] = 0;
    *cus = *khz = 1;
    return RKH_OK;
}
void rkh_close(int, void*) {}
int rkh_enter_device(int device, int* before) {
    *before = -1;
    if (g_current == device) return RKH_OK;
    if (g_lost) return RKH_ERR_RUNTIME;
    *before = g_current;
    g_current = device;
    return RKH_OK;
}
void rkh_leave_device(int before) {
    if (before >= 0) g_current = before;
}
int rkh_malloc(int, void** p, size_t n) { return ++g_live, *p = std::malloc(n), RKH_OK; }
void rkh_free(int, void* p) { --g_live, std::free(p); }
int rkh_h2d(void*, void* d, const void* s, size_t n) { return std::memcpy(d, s, n), RKH_OK; }
int rkh_sync(void*) { return RKH_OK; }
int rkh_static_scratch(int, void**, size_t*) { return RKH_ERR_RUNTIME; }
void rkh_set_marker(rkh_marker_fn, void*) {}
int rkh_g4_pack(void*, const uint8_t*, const uint16_t*, const uint8_t*, int, int, int, int, uint8_t*, uint32_t*) { return launch(); }
int rkh_g4_run(void*, const rkh_g4_args*) { return launch(); }
size_t rkh_g4_scratch_most(int, int) { return 0; }
int rkh_heads(void*, const rkh_heads_args*) { return launch(); }
}

#define CHECK(x)                                                         \
    do {                                                                 \
        if (!(x)) {                                                      \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #x);         \
            return 1;                                                    \
        }                                                                \
    } while (0)

int main() {
    rk_npu_ctx* ctx = rk_npu_open(nullptr);
    rk_npu_iommu_domain* domain = rk_npu_iommu_domain_create(ctx, 0);
    CHECK(ctx && domain);
    static uint8_t codes[64 * 16];
    static uint16_t scales[64], x[4 * 32], y[4 * 64];
    const rk_npu_g4_weight_config config{32, 64, 32, 0, RK_NPU_MX4_F16};
    rk_npu_heads_args heads;
    rk_npu_heads_args_init(&heads, 1, 32);
    heads.type = RK_NPU_MX4_F16, heads.rotary_dim = 0, heads.q_heads = 1, heads.q = x, heads.q_out = y;

    rk_npu_g4_weights* w = rk_npu_g4_weights_create(domain, &config, codes, scales, nullptr);
    rk_npu_g4_workspace* ws = rk_npu_g4_workspace_create(domain, 4, 32, 64);
    CHECK(w && ws && g_launches == 1);
    const auto run = [&] { return rk_npu_g4_run_device(ws, w, 4, RK_NPU_MX4_F16, x, 32, RK_NPU_MX4_F16, y, 64); };
    CHECK(run() == RK_NPU_OK && rk_npu_heads_norm_rotate_device(ctx, &heads) == RK_NPU_OK && g_launches == 3);
    CHECK(g_elsewhere == 0 && g_current == 1);

    g_lost = true;
    const int live = g_live;
    CHECK(run() == RK_NPU_ERR_SUBMIT);
    CHECK(rk_npu_heads_norm_rotate_device(ctx, &heads) == RK_NPU_ERR_SUBMIT);
    CHECK(!rk_npu_g4_weights_create(domain, &config, codes, scales, nullptr));
    CHECK(!rk_npu_g4_weights_create_device(domain, &config, codes, scales, nullptr));
    CHECK(!rk_npu_g4_workspace_create(domain, 4, 32, 64));
    CHECK(g_launches == 3 && g_live == live && g_current == 1);

    g_current = 0; // (what is current need not be made so)
    CHECK(run() == RK_NPU_OK && g_current == 0);
    g_lost = false, g_current = 1;
    CHECK(run() == RK_NPU_OK && rk_npu_heads_norm_rotate_device(ctx, &heads) == RK_NPU_OK && g_launches == 6 && g_elsewhere == 0 && g_current == 1);
    rk_npu_g4_workspace_free(ws);
    rk_npu_g4_weights_free(w);
    CHECK(g_live == 0);
    return 0;
}
