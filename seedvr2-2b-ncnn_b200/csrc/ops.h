// ops.h -- the operators beside the DiT: argument structs, host-side checks
// and launchers.  The checks touch no device, so a refused call costs nothing
// and needs no GPU.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>
#include "../../include/seedvr2_b200.h"

namespace s2b {

// Codes and scales of x in blocks of 128 columns x block_rows rows.
struct Fp8QuantArgs {
    const void* x; int x_type, rows, cols, ldx, block_rows;
    void* q; int ldq;
    float* scale;
};
// y = (xq . xs) (wq . ws)^T + bias.
struct Fp8LinearArgs {
    const void* xq; int ldx; const float* xs; int M, K;
    const void* wq; int ldw; const float* ws; int N;
    const float* bias;
    void* y; int y_type, ldy;
};
struct RopeArgs {
    const s2b_rope* plan;
    const void* x; int type, batch, tokens, heads, head_dim;
    long xs[3];                 // element strides of batch, token, head
    const int* pos; long pos_bs;
    int pos0;
    void* y; long ys[3];
    int inverse;
};
struct GroupNormArgs {
    const void* x; int x_type, batch, rows, channels, ldx, groups;
    const float *gamma, *beta;
    float eps; int act;
    void* y; int y_type, ldy;
    void* work; size_t work_bytes;
};

// Why the arguments are refused, or null.
const char* op_check(const Fp8QuantArgs& a);
const char* op_check(const Fp8LinearArgs& a);
const char* op_check(const RopeArgs& a);
const char* op_check(const GroupNormArgs& a);
// A call that has nothing to write.
inline bool op_empty(const Fp8QuantArgs& a) { return a.rows == 0 || a.cols == 0; }
inline bool op_empty(const Fp8LinearArgs& a) { return a.M == 0 || a.N == 0; }
inline bool op_empty(const RopeArgs& a) { return a.batch == 0 || a.tokens == 0 || a.heads == 0; }
inline bool op_empty(const GroupNormArgs& a) { return a.batch == 0 || a.rows == 0; }
// The device buffers of a call (nulls allowed), for the check that they live
// on the context's device.
struct OpPtrs { const void* p[8]; int n; };
inline OpPtrs op_ptrs(const Fp8QuantArgs& a) { return {{a.x, a.q, a.scale}, 3}; }
inline OpPtrs op_ptrs(const Fp8LinearArgs& a) { return {{a.xq, a.xs, a.wq, a.ws, a.y, a.bias}, 6}; }
inline OpPtrs op_ptrs(const RopeArgs& a) { return {{a.x, a.y, a.pos}, 3}; }
inline OpPtrs op_ptrs(const GroupNormArgs& a) { return {{a.x, a.y, a.work, a.gamma, a.beta}, 5}; }

// Enqueue on s, on the current device; returns the number of kernels
// launched, -1 when the launch could not be set up, or -1 - the CUDA error of a
// launch that was refused.
int op_launch(const Fp8QuantArgs& a, cudaStream_t s);
int op_launch(const Fp8LinearArgs& a, cudaStream_t s);
int op_launch(const RopeArgs& a, cudaStream_t s);
int op_launch(const GroupNormArgs& a, cudaStream_t s);

// Rotary frequencies of a configuration; null, or why it is refused.
const char* rope_plan(const s2b_rope_config& c, s2b_rope* out);
// Bytes of device workspace of a GroupNorm call; 0 when it needs none.
const char* groupnorm_limits(int batch, int rows, int channels);
size_t groupnorm_workspace(int batch, int rows, int channels, int groups);

// SMs of the current device (148 when it was not initialised).
int op_sms();

}  // namespace s2b
