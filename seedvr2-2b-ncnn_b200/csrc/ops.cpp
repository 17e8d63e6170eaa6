// ops.cpp -- host side of the operators beside the DiT: argument checks and
// the rotary plan.
#include "ops.h"
#include <cmath>
#include <cstring>

namespace s2b {
namespace {

inline bool type_ok(int t) { return t == S2B_PREC_FP32 || t == S2B_PREC_FP16 || t == S2B_PREC_BF16; }
inline int type_bytes(int t) { return t == S2B_PREC_FP32 ? 4 : 2; }
constexpr long MAX_STRIDE = 1L << 40;   // elements
constexpr int MAX_SIZE = 1 << 30;       // tile arithmetic stays in 32 bits

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// [p, p + bytes) and [q, q + more) share an address.
inline bool overlap(const void* p, size_t bytes, const void* q, size_t more) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return a < b + more && b < a + bytes;
}
// bytes from the first to the last element of rows x cols with a row pitch
inline size_t span(size_t rows, size_t cols, size_t ld, size_t e) { return rows ? ((rows - 1) * ld + cols) * e : 0; }
// n steps of a stride reach further than any memory, and than 64-bit offsets
// can be trusted with (both not negative).
inline bool too_far(long n, long stride) { return n > 1 && stride > MAX_STRIDE / (n - 1); }

}  // namespace

const char* op_check(const Fp8QuantArgs& a) {
    if (!type_ok(a.x_type)) return "fp8 quantise: x_type must be S2B_PREC_FP32, _FP16 or _BF16";
    if (a.rows < 0 || a.cols < 0) return "fp8 quantise: negative size";
    if (a.block_rows != 1 && a.block_rows != 128) return "fp8 quantise: block_rows must be 1 or 128";
    if (op_empty(a)) return nullptr;
    if (!a.x || !a.q || !a.scale) return "fp8 quantise: null buffer";
    if (a.ldx < a.cols || a.ldq < a.cols) return "fp8 quantise: row pitch below cols";
    if (a.ldq % 16 || !aligned(a.q, 16)) return "fp8 quantise: q needs 16-byte alignment and a pitch that is a multiple of 16";
    if (!aligned(a.x, type_bytes(a.x_type)) || !aligned(a.scale, 4)) return "fp8 quantise: buffer not aligned to its type";
    const size_t qb = span(a.rows, a.cols, a.ldq, 1), xb = span(a.rows, a.cols, a.ldx, type_bytes(a.x_type));
    const size_t rb = a.block_rows == 1 ? (size_t)a.rows : ((size_t)a.rows + 127) / 128;
    const size_t sb = rb * (((size_t)a.cols + 127) / 128) * 4;
    if (overlap(a.x, xb, a.q, qb) || overlap(a.x, xb, a.scale, sb) || overlap(a.q, qb, a.scale, sb))
        return "fp8 quantise: buffers overlap";
    return nullptr;
}

const char* op_check(const Fp8LinearArgs& a) {
    if (!type_ok(a.y_type)) return "fp8 linear: y_type must be S2B_PREC_FP32, _FP16 or _BF16";
    if (a.M < 0 || a.N < 0 || a.K <= 0) return "fp8 linear: M and N must not be negative, K must be positive";
    if (a.M > MAX_SIZE || a.N > MAX_SIZE || a.K > MAX_SIZE) return "fp8 linear: M, N or K above 2^30";
    if (op_empty(a)) return nullptr;
    if (!a.xq || !a.xs || !a.wq || !a.ws || !a.y) return "fp8 linear: null buffer";
    if (a.ldx < a.K || a.ldw < a.K || a.ldy < a.N) return "fp8 linear: row pitch below the row's length";
    if (a.ldx % 16 || a.ldw % 16 || !aligned(a.xq, 16) || !aligned(a.wq, 16))
        return "fp8 linear: codes need 16-byte alignment and pitches that are multiples of 16";
    if (!aligned(a.xs, 4) || !aligned(a.ws, 4) || !aligned(a.bias, 4) || !aligned(a.y, type_bytes(a.y_type)))
        return "fp8 linear: buffer not aligned to its type";
    const size_t yb = span(a.M, a.N, a.ldy, type_bytes(a.y_type)), kb = ((size_t)a.K + 127) / 128;
    if (overlap(a.y, yb, a.xq, span(a.M, a.K, a.ldx, 1)) || overlap(a.y, yb, a.wq, span(a.N, a.K, a.ldw, 1)) ||
        overlap(a.y, yb, a.xs, kb * a.M * 4) || overlap(a.y, yb, a.ws, kb * (((size_t)a.N + 127) / 128) * 4) ||
        (a.bias && overlap(a.y, yb, a.bias, (size_t)a.N * 4)))
        return "fp8 linear: y overlaps an operand";
    return nullptr;
}

const char* op_check(const RopeArgs& a) {
    if (!type_ok(a.type)) return "rope: type must be S2B_PREC_FP32, _FP16 or _BF16";
    if (a.batch < 0 || a.tokens < 0 || a.heads < 0 || a.head_dim <= 0)
        return "rope: batch, tokens and heads must not be negative, head_dim must be positive";
    if (a.head_dim > MAX_SIZE) return "rope: head_dim above 2^30";
    if (!a.plan) return "rope: null plan";
    const s2b_rope& p = *a.plan;
    if (p.pairs < 0 || p.pairs > S2B_ROPE_MAX_PAIRS || p.axes < 1 || p.axes > 3 || (p.half != 0 && p.half != 1) ||
        !std::isfinite(p.amplitude))
        return "rope: not a plan of s2b_rope_plan";
    for (int i = 0; i < p.pairs; i++)
        if (p.axis[i] >= p.axes) return "rope: not a plan of s2b_rope_plan";
    if (2 * p.pairs > a.head_dim) return "rope: the plan rotates more than head_dim values";
    if (op_empty(a)) return nullptr;
    if (!a.x || !a.y) return "rope: null buffer";
    if (!aligned(a.x, type_bytes(a.type)) || !aligned(a.y, type_bytes(a.type)) || !aligned(a.pos, 4))
        return "rope: buffer not aligned to its type";
    for (int i = 0; i < 3; i++)
        if (a.xs[i] < 0 || a.ys[i] < 0 || a.xs[i] > MAX_STRIDE || a.ys[i] > MAX_STRIDE)
            return "rope: stride negative or above 2^40";
    if (a.pos && (a.pos_bs < 0 || a.pos_bs > MAX_STRIDE)) return "rope: stride negative or above 2^40";
    const long D = a.head_dim, n[3] = {a.batch, a.tokens, a.heads};
    for (int i = 0; i < 3; i++)
        if (too_far(n[i], a.xs[i]) || too_far(n[i], a.ys[i])) return "rope: x or y reaches over more than 2^40 values";
    if (a.pos && too_far(a.batch, a.pos_bs)) return "rope: the positions reach over more than 2^40 values";
    // y is written by many threads at once: no two of its heads may share an
    // element, whichever order the three strides nest in
    int ord[3] = {0, 1, 2};
    for (int i = 0; i < 3; i++)
        for (int j = i + 1; j < 3; j++)
            if (a.ys[ord[j]] < a.ys[ord[i]]) { const int t = ord[i]; ord[i] = ord[j]; ord[j] = t; }
    long reach = D;
    for (int i = 0; i < 3; i++) {
        if (n[ord[i]] > 1) {
            if (a.ys[ord[i]] < reach) return "rope: y's strides make its heads overlap";
            reach += (n[ord[i]] - 1) * a.ys[ord[i]];
        }
    }
    size_t xr = D, e = type_bytes(a.type);
    bool same = a.x == a.y;
    for (int i = 0; i < 3; i++) {
        xr += (size_t)(n[i] - 1) * a.xs[i];
        if (n[i] > 1 && a.xs[i] != a.ys[i]) same = false;
    }
    if (!same && overlap(a.x, xr * e, a.y, (size_t)reach * e))
        return "rope: x and y overlap without being the same values";
    if (a.pos && overlap(a.y, (size_t)reach * e, a.pos,
                         4 * ((size_t)(a.batch - 1) * a.pos_bs + (size_t)a.tokens * p.axes)))
        return "rope: y overlaps the positions";
    return nullptr;
}

const char* groupnorm_limits(int batch, int rows, int channels) {
    return batch > 65535 || rows > MAX_SIZE || channels > 1 << 23
               ? "groupnorm: more than 65535 samples, 2^30 rows or 2^23 channels" : nullptr;
}

const char* op_check(const GroupNormArgs& a) {
    if (!type_ok(a.x_type) || !type_ok(a.y_type)) return "groupnorm: types must be S2B_PREC_FP32, _FP16 or _BF16";
    if (a.batch < 0 || a.rows < 0 || a.channels <= 0 || a.groups <= 0)
        return "groupnorm: batch and rows must not be negative, channels and groups must be positive";
    if (a.channels % a.groups) return "groupnorm: channels must be a multiple of groups";
    if (a.act != 0 && a.act != 1) return "groupnorm: act must be S2B_ACT_NONE or S2B_ACT_SILU";
    if (!(a.eps >= 0.f) || !std::isfinite(a.eps)) return "groupnorm: eps must be finite and not negative";
    if (const char* why = groupnorm_limits(a.batch, a.rows, a.channels)) return why;
    if (op_empty(a)) return nullptr;
    if (!a.x || !a.y) return "groupnorm: null buffer";
    if (a.ldx < a.channels || a.ldy < a.channels) return "groupnorm: row pitch below channels";
    const size_t xe = type_bytes(a.x_type), ye = type_bytes(a.y_type), R = (size_t)a.batch * a.rows;
    if (!aligned(a.x, xe) || !aligned(a.y, ye) || !aligned(a.gamma, 4) || !aligned(a.beta, 4))
        return "groupnorm: buffer not aligned to its type";
    const size_t need = groupnorm_workspace(a.batch, a.rows, a.channels, a.groups);
    if (a.work_bytes < need || (need && !a.work)) return "groupnorm: workspace smaller than s2b_groupnorm_workspace says";
    if (need && !aligned(a.work, 16)) return "groupnorm: workspace not 16-byte aligned";
    const size_t xb = span(R, a.channels, a.ldx, xe), yb = span(R, a.channels, a.ldy, ye);
    const bool same = a.x == a.y && a.ldx == a.ldy && a.x_type == a.y_type;
    if (!same && overlap(a.x, xb, a.y, yb)) return "groupnorm: x and y overlap without being the same rows";
    const size_t cb = (size_t)a.channels * 4;
    if ((a.gamma && overlap(a.y, yb, a.gamma, cb)) || (a.beta && overlap(a.y, yb, a.beta, cb)))
        return "groupnorm: y overlaps gamma or beta";
    if (need && (overlap(a.work, need, a.y, yb) || overlap(a.work, need, a.x, xb) ||
                 (a.gamma && overlap(a.work, need, a.gamma, cb)) || (a.beta && overlap(a.work, need, a.beta, cb))))
        return "groupnorm: the workspace overlaps another buffer";
    return nullptr;
}

// Pair j of an axis with d rotated dims turns by f_j = theta^(-2j/d) radians a
// position.  Scalings for streams longer than the model was trained on:
//   linear  f_j / factor
//   ntk     theta' = theta * factor^(d / (d - 2)): the slowest pair is slowed
//           by factor, the fastest not at all
//   yarn    (Peng et al. 2023) pairs that turn more than beta_fast times over
//           original_length positions keep f_j, those below beta_slow take
//           f_j / factor, a linear ramp over j between; rotated values are
//           multiplied by 0.1 ln(factor) + 1
// f_j is stored as a 64-bit fraction of a turn, f_j / 2 pi * 2^64, so that
// position * fraction modulo 2^64 is the angle's fraction of a turn: the wrap
// of the integer product is the exact range reduction at every position.
const char* rope_plan(const s2b_rope_config& c, s2b_rope* out) {
    if (c.layout != S2B_ROPE_INTERLEAVED && c.layout != S2B_ROPE_HALF) return "rope plan: unknown layout";
    if (c.axes < 1 || c.axes > 3) return "rope plan: axes must be 1, 2 or 3";
    if (!(c.theta > 0) || !std::isfinite(c.theta)) return "rope plan: theta must be positive and finite";
    if (c.scaling < S2B_ROPE_SCALE_NONE || c.scaling > S2B_ROPE_SCALE_YARN) return "rope plan: unknown scaling";
    if (c.scaling != S2B_ROPE_SCALE_NONE && (!(c.factor >= 1) || !std::isfinite(c.factor)))
        return "rope plan: factor must be at least 1";
    const bool yarn = c.scaling == S2B_ROPE_SCALE_YARN;
    if (yarn && (!(c.original_length > 0) || !std::isfinite(c.original_length) || !(c.beta_slow > 0) ||
                 !(c.beta_fast >= c.beta_slow) || !std::isfinite(c.beta_fast) || !(c.theta > 1)))
        return "rope plan: yarn needs theta > 1, original_length > 0 and beta_fast >= beta_slow > 0";
    int pairs = 0;
    for (int a = 0; a < c.axes; a++) {
        if (c.axis_dim[a] < 0 || c.axis_dim[a] % 2) return "rope plan: axis_dim must be even and not negative";
        if (c.axis_dim[a] > 2 * S2B_ROPE_MAX_PAIRS - 2 * pairs) return "rope plan: more than 256 rotated dims";
        pairs += c.axis_dim[a] / 2;
    }
    s2b_rope p;
    std::memset(&p, 0, sizeof p);
    p.pairs = pairs;
    p.half = c.layout == S2B_ROPE_HALF;
    p.axes = c.axes;
    p.amplitude = yarn ? (float)(0.1 * std::log(c.factor) + 1) : 1.f;
    const long double two_pi = 2 * acosl(-1.0L);
    int i = 0;
    for (int a = 0; a < c.axes; a++) {
        const int d = c.axis_dim[a];
        long double theta = c.theta;
        if (c.scaling == S2B_ROPE_SCALE_NTK && d > 2)
            theta *= powl((long double)c.factor, (long double)d / (d - 2));
        double lo = 0, hi = 0;
        if (yarn) {
            const double per = d / (2 * std::log(c.theta));
            lo = std::fmax(std::floor(per * std::log(c.original_length / (c.beta_fast * 2 * M_PI))), 0);
            hi = std::fmin(std::ceil(per * std::log(c.original_length / (c.beta_slow * 2 * M_PI))), d - 1);
        }
        for (int j = 0; j < d / 2; j++, i++) {
            long double f = powl(theta, -2.0L * j / d);
            if (c.scaling == S2B_ROPE_SCALE_LINEAR) f /= c.factor;
            if (yarn) {
                const double ramp = std::fmin(std::fmax((j - lo) / std::fmax(hi - lo, 0.001), 0), 1);
                f = f * (1 - ramp) + f / c.factor * ramp;
            }
            // theta < 1 makes f exceed a turn: only its fraction matters
            long double turns = f / two_pi;
            if (!std::isfinite((double)turns)) return "rope plan: a frequency is not finite";
            turns -= floorl(turns);
            const long double scaled = roundl(turns * 18446744073709551616.0L);
            p.turns[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
            p.axis[i] = (uint8_t)a;
        }
    }
    *out = p;
    return nullptr;
}

}  // namespace s2b
