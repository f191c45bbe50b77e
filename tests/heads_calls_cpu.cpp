// The heads' host layer over a device that notes what reaches it.  Cases from standard input, a line each: rows, heads, head_dim, row stride, head stride; prints the call's
// code and how many launches it asked for.
#include <cstdio>

#include "rk_heads_shim.h"
#include "rk_host.h"
#include "rk_npu_heads.h"

static int g_launches;

extern "C" {
int rkh_heads(void*, const rkh_heads_args*) { return ++g_launches, RKH_OK; }
int rkh_enter_device(int, int* before) { return *before = -1, RKH_OK; }
void rkh_leave_device(int) {}
}

int main() {
    rk_npu_ctx ctx;
    long long rows, heads, dim, row, head;
    while (std::scanf("%lld %lld %lld %lld %lld", &rows, &heads, &dim, &row, &head) == 5) {
        rk_npu_heads_args a;
        rk_npu_heads_args_init(&a, (int)rows, (int)dim);
        a.type = RK_NPU_MX4_F32;
        a.rotary_dim = 0;
        a.q_heads = (int)heads;
        a.q = a.q_out = reinterpret_cast<void*>(4096);
        a.q_row = a.q_out_row = row;
        a.q_head = a.q_out_head = head;
        g_launches = 0;
        const int rc = rk_npu_heads_norm_rotate_device(&ctx, &a);
        std::printf("%d %d\n", rc, g_launches);
    }
    return 0;
}
