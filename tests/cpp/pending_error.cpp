// A CUDA error that is pending when an operator is called is neither the call's
// nor taken from the caller.  Linked with the library's objects, so that both
// share one CUDA runtime.
#include "seedvr2_b200.h"
#include <cuda_runtime.h>
#include <cstdio>

static int fails = 0;
static void expect(bool ok, const char* what, int got) {
    if (!ok) { std::fprintf(stderr, "%s: %d\n", what, got); fails++; }
}

int main() {
    s2b_ctx* ctx = nullptr;
    if (int rc = s2b_ctx_create(0, S2B_PREC_BF16, &ctx)) { std::fprintf(stderr, "create: %d\n", rc); return 2; }
    char* d = nullptr;
    if (cudaMalloc((void**)&d, 8 << 20) != cudaSuccess || cudaMemset(d, 0, 8 << 20) != cudaSuccess) return 2;
    char *x = d, *q = d + (1 << 20), *s = d + (2 << 20), *w = d + (3 << 20), *ws = d + (4 << 20), *y = d + (5 << 20), *work = d + (6 << 20);
    s2b_rope_config rc = {S2B_ROPE_HALF, 1, {64, 0, 0}, 10000.0, S2B_ROPE_SCALE_NONE, 1.0, 0, 0, 0};
    s2b_rope plan;
    if (s2b_rope_plan(&rc, &plan)) return 2;
    const long st[3] = {0, 128, 128};
    for (int op = 0; op < 4; op++) {
        expect(cudaGetLastError() == cudaSuccess, "clean before", op);
        cudaSetDevice(1 << 20);                          // no such device: pending from here on
        expect(cudaPeekAtLastError() == cudaErrorInvalidDevice, "pending", op);
        int r = -1;
        if (op == 0) r = s2b_fp8_quant_dev(ctx, x, S2B_PREC_FP32, 16, 128, 128, 1, q, 128, (float*)s, nullptr);
        if (op == 1) r = s2b_linear_fp8_dev(ctx, q, 128, (float*)s, 16, 128, w, 128, (float*)ws, 128, nullptr, y, S2B_PREC_FP32, 128, nullptr);
        if (op == 2) r = s2b_rope_dev(ctx, &plan, x, S2B_PREC_FP32, 1, 16, 1, 128, st, nullptr, 0, 0, y, st, 0, nullptr);
        if (op == 3) r = s2b_groupnorm_dev(ctx, x, S2B_PREC_FP32, 1, 16, 128, 128, 8, nullptr, nullptr, 1e-6f, S2B_ACT_NONE, y, S2B_PREC_FP32,
                                           128, work, 1 << 20, nullptr);
        expect(r == S2B_OK, "operator", op * 100 + r);
        expect(cudaGetLastError() == cudaErrorInvalidDevice, "still pending after operator", op);
        expect(cudaDeviceSynchronize() == cudaSuccess, "synchronise", op);
    }
    s2b_ctx_destroy(ctx);
    cudaFree(d);
    if (!fails) std::puts("ok");
    return fails ? 1 : 0;
}
