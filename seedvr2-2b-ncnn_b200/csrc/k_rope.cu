// k_rope.cu -- rotary positions on strided heads.
//
// Pair i of a head, (a, b) = (x[2i], x[2i + 1]) or (x[i], x[i + P]), becomes
// (a cos - b sin, a sin + b cos) * amplitude with the angle pos[axis(i)] * f_i;
// the other dims are copied.  The angle is the integer product pos * turns[i]
// modulo 2^64, a fraction of a turn: exact range reduction at any position,
// where pos * f_i in fp32 is off by 0.06 rad at a million.
//
// Bound by HBM: every element is read and written once.  A thread owns one
// 16-byte piece of a head (or of its two halves) in up to four heads of a
// token, all loaded before anything else: the sines, one evaluation per (token,
// pair, four heads), are computed while the loads are in flight.  Chunks of
// heads are neighbouring CTAs, so the CTAs together walk through memory in
// order.  B200: 40 heads of 128 at 5440 tokens (111 MB) 25.7 us, 8 heads of 128
// at 131042 tokens in fp32 (1.07 GB) 191 us, 5.6 TB/s.
#include "kcommon.cuh"
#include "launch.cuh"
#include "ops.h"

namespace s2b {
namespace {

// CTAs an SM: 64 registers a thread hold four heads' pieces; eight heads a
// thread (half the sines) need 101 and run two CTAs an SM, 27 us against 25.7
// for 40 heads of 5440 tokens.
constexpr int ROPE_CTAS = 4;
struct RopeParams {
    s2b_rope p;
    const void* x; void* y;
    long xb, xt, xh, yb, yt, yh;        // element strides
    const int* pos; long pos_bs;
    int pos0, tokens, heads, D;
    int items, tpc, jt, chunks;         // pieces a token, tokens a CTA, CTAs a token, CTAs of heads
    long rows;                          // batch * tokens
    float sign;                         // -1 turns back
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

// The plan in shared memory: lanes read different pairs, which the constant
// bank of the kernel's arguments would serve one after another.
struct SharedPlan {
    uint64_t turns[S2B_ROPE_MAX_PAIRS];
    uint8_t axis[S2B_ROPE_MAX_PAIRS];
};

// (a, d) -> (a c - d s, a s + d c): two packed multiply-adds.
__device__ __forceinline__ float2 rotate(float a, float d, float c, float s) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, cc, ss, t;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%3, %2};\n\t"
        "mov.b64 cc, {%4, %4};\n\tmov.b64 ss, {%6, %5};\n\t"
        "mul.rn.f32x2 t, y, ss;\n\tfma.rn.f32x2 t, x, cc, t;\n\t"
        "mov.b64 {%0, %1}, t;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a), "f"(d), "f"(c), "f"(s), "f"(-s));
    return r;
}

__device__ __forceinline__ void turn(const RopeParams& P, const SharedPlan& S, int i, const int* pos, int t, float& c, float& s) {
    const int64_t p = pos ? (int64_t)pos[S.axis[i]] : (int64_t)P.pos0 + t;
    const uint64_t f = (uint64_t)p * S.turns[i];         // wraps whole turns away
    // top 32 bits as a signed fraction of half a turn in [-1, 1)
    const float half = (float)(int32_t)(f >> 32) * 4.656612873077393e-10f;
    sincospif(half, &s, &c);
    c *= P.p.amplitude;
    s *= P.p.amplitude * P.sign;
}

// Item j of a token's head: interleaved, elements [j VEC, (j + 1) VEC); half,
// the first pairs / VEC items hold elements [j VEC, ..) of both halves and the
// rest the copied tail.  VEC = 1 interleaved items hold one element pair.  In
// HU heads from x (to y), all loaded together and ahead of the stores: x and y
// may be the same buffer, so the compiler cannot reorder them.
template <typename T, int VEC, bool HALF, int HU>
__device__ __forceinline__ void rope_item(const RopeParams& P, const SharedPlan& S, int j, const T* x, T* y, const int* pos, int t) {
    const int np = P.p.pairs;
    if constexpr (HALF) {
        typedef Pack<T, VEC> V;
        const int nrot = np / VEC;
        if (j < nrot) {
            V u[HU], w[HU];
            #pragma unroll
            for (int k = 0; k < HU; k++)
            {
                u[k] = *reinterpret_cast<const V*>(x + k * P.xh + j * VEC);
                w[k] = *reinterpret_cast<const V*>(x + k * P.xh + j * VEC + np);
            }
            #pragma unroll
            for (int i = 0; i < VEC; i++) {
                float c, s;
                turn(P, S, j * VEC + i, pos, t, c, s);
                #pragma unroll
                for (int k = 0; k < HU; k++) {
                    const float a = Cvt<T>::to_f(u[k].v[i]), d = Cvt<T>::to_f(w[k].v[i]);
                    const float2 r = rotate(a, d, c, s);
                    u[k].v[i] = Cvt<T>::from_f(r.x);
                    w[k].v[i] = Cvt<T>::from_f(r.y);
                }
            }
            #pragma unroll
            for (int k = 0; k < HU; k++)
            {
                *reinterpret_cast<V*>(y + k * P.yh + j * VEC) = u[k];
                *reinterpret_cast<V*>(y + k * P.yh + j * VEC + np) = w[k];
            }
        } else {
            if (P.x == P.y) return;
            const int o = 2 * np + (j - nrot) * VEC;
            V u[HU];
            #pragma unroll
            for (int k = 0; k < HU; k++)
                u[k] = *reinterpret_cast<const V*>(x + k * P.xh + o);
            #pragma unroll
            for (int k = 0; k < HU; k++)
                *reinterpret_cast<V*>(y + k * P.yh + o) = u[k];
        }
    } else if constexpr (VEC > 1) {
        typedef Pack<T, VEC> V;
        constexpr int N = VEC / 2;                      // pairs of an item
        if (j * N >= np && P.x == P.y) return;
        V u[HU];
        #pragma unroll
        for (int k = 0; k < HU; k++)
            u[k] = *reinterpret_cast<const V*>(x + k * P.xh + j * VEC);
        #pragma unroll
        for (int i = 0; i < N; i++) {
            if (j * N + i >= np) break;                 // copied bits stay the bits they were
            float c, s;
            turn(P, S, j * N + i, pos, t, c, s);
            #pragma unroll
            for (int k = 0; k < HU; k++) {
                const float a = Cvt<T>::to_f(u[k].v[2 * i]), d = Cvt<T>::to_f(u[k].v[2 * i + 1]);
                const float2 r = rotate(a, d, c, s);
                u[k].v[2 * i] = Cvt<T>::from_f(r.x);
                u[k].v[2 * i + 1] = Cvt<T>::from_f(r.y);
            }
        }
        #pragma unroll
        for (int k = 0; k < HU; k++)
            *reinterpret_cast<V*>(y + k * P.yh + j * VEC) = u[k];
    } else {
        const int o = 2 * j;
        const bool rot = j < np, two = o + 1 < P.D;     // an odd head's last element stands alone
        if (!rot && P.x == P.y) return;
        float c = 1.f, s = 0.f;
        if (rot) turn(P, S, j, pos, t, c, s);
        for (int k = 0; k < HU; k++, x += P.xh, y += P.yh) {
            const T u = x[o], w = two ? x[o + 1] : u;
            if (rot) {
                const float a = Cvt<T>::to_f(u), d = Cvt<T>::to_f(w);
                y[o] = Cvt<T>::from_f(a * c - d * s);
                y[o + 1] = Cvt<T>::from_f(a * s + d * c);
            } else {
                y[o] = u;
                if (two) y[o + 1] = w;
            }
        }
    }
}

template <typename T, int VEC, bool HALF, int HU>
__global__ void __launch_bounds__(256, ROPE_CTAS) k_rope(const __grid_constant__ RopeParams P) {
    __shared__ SharedPlan S;
    if (threadIdx.x < P.p.pairs) {
        S.turns[threadIdx.x] = P.p.turns[threadIdx.x];
        S.axis[threadIdx.x] = P.p.axis[threadIdx.x];
    }
    __syncthreads();
    chain_begin();
    unsigned at = blockIdx.x;
    const int chunk = at % P.chunks;
    at /= P.chunks;
    const int jt = at % P.jt;
    const int tok = threadIdx.x / P.items, j = threadIdx.x - tok * P.items + jt * 256;
    const long row = (long)(at / P.jt) * P.tpc + tok;
    if (tok >= P.tpc || row >= P.rows || j >= P.items) return;
    // 64-bit division costs more than the rest of a thread's work
    const long b = P.rows < (1L << 32) ? (long)((unsigned)row / (unsigned)P.tokens) : row / P.tokens;
    const int t = (int)(row - b * P.tokens);
    rope_item<T, VEC, HALF, HU>(P, S, j, (const T*)P.x + b * P.xb + t * P.xt + chunk * HU * P.xh,
                                (T*)P.y + b * P.yb + t * P.yt + chunk * HU * P.yh,
                                P.pos ? P.pos + b * P.pos_bs + (long)t * P.p.axes : nullptr, t);
}

template <typename T, int VEC, int HU>
int launch_hu(RopeParams& P, long ctas, cudaStream_t s) {
    P.chunks = P.heads / HU;
    const long g = ctas * P.chunks;
    if (g > 2147483647L) return -1;
    return launch_chained(P.p.half ? k_rope<T, VEC, true, HU> : k_rope<T, VEC, false, HU>, dim3((unsigned)g), 256, 0, 0, s, P) ? 1 : -1;
}

template <typename T, int VEC>
int launch(const RopeArgs& a, cudaStream_t s) {
    RopeParams P;
    P.p = *a.plan;
    P.x = a.x; P.y = a.y;
    P.xb = a.xs[0]; P.xt = a.xs[1]; P.xh = a.xs[2];
    P.yb = a.ys[0]; P.yt = a.ys[1]; P.yh = a.ys[2];
    P.pos = a.pos; P.pos_bs = a.pos_bs; P.pos0 = a.pos0;
    P.tokens = a.tokens; P.heads = a.heads; P.D = a.head_dim;
    P.rows = (long)a.batch * a.tokens;
    P.sign = a.inverse ? -1.f : 1.f;
    const int D = a.head_dim, np = P.p.pairs;
    if (P.p.half) P.items = np / VEC + (D - 2 * np) / VEC;
    else P.items = VEC > 1 ? D / VEC : (D + 1) / 2;
    P.tpc = P.items < 256 ? 256 / (P.items ? P.items : 1) : 1;
    P.jt = (P.items + 255) / 256;
    const long ctas = (P.rows + P.tpc - 1) / P.tpc * P.jt;
    if (P.items == 0 || ctas == 0) return 0;
    // Heads that share a thread's sines: the most, up to four, that divide the
    // heads (no thread has a partial batch, whose guarded loads would go out one
    // by one) and, when tokens are few, leave every SM a CTA or two.
    for (int hu = 4; hu > 1; hu--) {
        if (a.heads % hu || ctas * (a.heads / hu) < 2L * op_sms()) continue;
        switch (hu) {
            case 4: return launch_hu<T, VEC, 4>(P, ctas, s);
            case 3: return launch_hu<T, VEC, 3>(P, ctas, s);
            case 2: return launch_hu<T, VEC, 2>(P, ctas, s);
        }
    }
    return launch_hu<T, VEC, 1>(P, ctas, s);
}

template <typename T>
int launch_t(const RopeArgs& a, cudaStream_t s) {
    // 16-byte pieces where every head starts on one and neither layout cuts
    // a piece in two, pieces of two elements likewise, single elements otherwise
    auto fits = [&](int v) {
        bool ok = (uintptr_t)a.x % (v * sizeof(T)) == 0 && (uintptr_t)a.y % (v * sizeof(T)) == 0 && a.head_dim % v == 0 &&
                  (!a.plan->half || a.plan->pairs % v == 0);
        const long n[3] = {a.batch, a.tokens, a.heads};
        for (int i = 0; i < 3; i++) ok = ok && (n[i] <= 1 || (a.xs[i] % v == 0 && a.ys[i] % v == 0));
        return ok;
    };
    constexpr int V = 16 / (int)sizeof(T);
    return fits(V) ? launch<T, V>(a, s) : fits(2) ? launch<T, 2>(a, s) : launch<T, 1>(a, s);
}

}  // namespace

int op_launch(const RopeArgs& a, cudaStream_t s) {
    switch (a.type) {
        case S2B_PREC_FP32: return launch_t<float>(a, s);
        case S2B_PREC_FP16: return launch_t<f16>(a, s);
        default: return launch_t<bf16>(a, s);
    }
}

}  // namespace s2b
