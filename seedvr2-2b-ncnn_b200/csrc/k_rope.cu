// k_rope.cu -- rotary positions on strided heads.
//
// Pair i of a head, (a, b) = (x[2i], x[2i + 1]) or (x[i], x[i + P]), becomes
// (a cos - b sin, a sin + b cos) * amplitude with the angle pos[axis(i)] * f_i;
// the other dims are copied.  The angle is the integer product pos * turns[i]
// modulo 2^64, a fraction of a turn: exact range reduction at any position,
// where pos * f_i in fp32 is off by 0.06 rad at a million.
//
// Bound by HBM: every element is read and written once.  A thread owns one
// 16-byte piece of a head (or of its two halves), computes its few sines once
// and walks over the heads of its token, so the sines cost one evaluation per
// (token, pair, chunk of heads) and the loads of several heads are in flight.
#include "kcommon.cuh"
#include "ops.h"

namespace s2b {
namespace {

// Heads whose loads are in flight together.  Loaded ahead of the stores by
// hand: x and y may be the same buffer, so the compiler cannot reorder them.
constexpr int HU = 4;

struct RopeParams {
    s2b_rope p;
    const void* x; void* y;
    long xb, xt, xh, yb, yt, yh;        // element strides
    const int* pos; long pos_bs;
    int pos0, tokens, heads, D, hchunk, items;
    long rows;                          // batch * tokens
    float sign;                         // -1 turns back
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

__device__ __forceinline__ void turn(const RopeParams& P, int i, const int* pos, int t, float& c, float& s) {
    const int64_t p = pos ? (int64_t)pos[P.p.axis[i]] : (int64_t)P.pos0 + t;
    const uint64_t f = (uint64_t)p * P.p.turns[i];       // wraps whole turns away
    // top 32 bits as a signed fraction of half a turn in [-1, 1)
    const float half = (float)(int32_t)(f >> 32) * 4.656612873077393e-10f;
    sincospif(half, &s, &c);
    c *= P.p.amplitude;
    s *= P.p.amplitude * P.sign;
}

// Item j of a token's head: interleaved, elements [j VEC, (j + 1) VEC); half,
// the first pairs / VEC items hold elements [j VEC, ..) of both halves and the
// rest the copied tail.  VEC = 1 interleaved items hold one element pair.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(256) k_rope(const __grid_constant__ RopeParams P) {
    const long idx = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = idx / P.items;
    const int j = (int)(idx - row * P.items);
    if (row >= P.rows) return;
    const long b = row / P.tokens;
    const int t = (int)(row - b * P.tokens);
    const int h0 = blockIdx.y * P.hchunk, h1 = min(P.heads, h0 + P.hchunk);
    const T* x = (const T*)P.x + b * P.xb + t * P.xt + h0 * P.xh;
    T* y = (T*)P.y + b * P.yb + t * P.yt + h0 * P.yh;
    const int* pos = P.pos ? P.pos + b * P.pos_bs + (long)t * P.p.axes : nullptr;
    const int np = P.p.pairs;
    if constexpr (HALF) {
        typedef Pack<T, VEC> V;
        const int nrot = np / VEC;
        if (j < nrot) {
            float c[VEC], s[VEC];
            #pragma unroll
            for (int i = 0; i < VEC; i++) turn(P, j * VEC + i, pos, t, c[i], s[i]);
            const int o0 = j * VEC, o1 = o0 + np;
            for (int h = h0; h < h1; h += HU, x += HU * P.xh, y += HU * P.yh) {
                V u[HU], w[HU];
                #pragma unroll
                for (int k = 0; k < HU; k++)
                    if (h + k < h1) {
                        u[k] = *reinterpret_cast<const V*>(x + k * P.xh + o0);
                        w[k] = *reinterpret_cast<const V*>(x + k * P.xh + o1);
                    }
                #pragma unroll
                for (int k = 0; k < HU; k++) {
                    if (h + k >= h1) break;
                    V p, q;
                    #pragma unroll
                    for (int i = 0; i < VEC; i++) {
                        const float a = Cvt<T>::to_f(u[k].v[i]), d = Cvt<T>::to_f(w[k].v[i]);
                        p.v[i] = Cvt<T>::from_f(a * c[i] - d * s[i]);
                        q.v[i] = Cvt<T>::from_f(a * s[i] + d * c[i]);
                    }
                    *reinterpret_cast<V*>(y + k * P.yh + o0) = p;
                    *reinterpret_cast<V*>(y + k * P.yh + o1) = q;
                }
            }
        } else {
            if (P.x == P.y) return;
            const int o = 2 * np + (j - nrot) * VEC;
            for (int h = h0; h < h1; h += HU, x += HU * P.xh, y += HU * P.yh) {
                V u[HU];
                #pragma unroll
                for (int k = 0; k < HU; k++)
                    if (h + k < h1) u[k] = *reinterpret_cast<const V*>(x + k * P.xh + o);
                #pragma unroll
                for (int k = 0; k < HU; k++)
                    if (h + k < h1) *reinterpret_cast<V*>(y + k * P.yh + o) = u[k];
            }
        }
    } else {
        constexpr int N = VEC > 1 ? VEC / 2 : 1;       // pairs of an item
        float c[N], s[N];
        #pragma unroll
        for (int i = 0; i < N; i++) {
            c[i] = 1.f; s[i] = 0.f;
            if (j * N + i < np) turn(P, j * N + i, pos, t, c[i], s[i]);
        }
        const int o = j * 2 * N;
        const bool rot0 = j * N < np;
        if (!rot0 && P.x == P.y) return;
        if constexpr (VEC > 1) {
            typedef Pack<T, VEC> V;
            for (int h = h0; h < h1; h += HU, x += HU * P.xh, y += HU * P.yh) {
                V u[HU];
                #pragma unroll
                for (int k = 0; k < HU; k++)
                    if (h + k < h1) u[k] = *reinterpret_cast<const V*>(x + k * P.xh + o);
                #pragma unroll
                for (int k = 0; k < HU; k++) {
                    if (h + k >= h1) break;
                    #pragma unroll
                    for (int i = 0; i < N; i++) {
                        if (j * N + i >= np) continue;      // copied bits stay the bits they were
                        const float a = Cvt<T>::to_f(u[k].v[2 * i]), d = Cvt<T>::to_f(u[k].v[2 * i + 1]);
                        u[k].v[2 * i] = Cvt<T>::from_f(a * c[i] - d * s[i]);
                        u[k].v[2 * i + 1] = Cvt<T>::from_f(a * s[i] + d * c[i]);
                    }
                    *reinterpret_cast<V*>(y + k * P.yh + o) = u[k];
                }
            }
        } else {
            const bool two = o + 1 < P.D;               // an odd head's last element stands alone
            for (int h = h0; h < h1; h++, x += P.xh, y += P.yh) {
                const T u = x[o], w = two ? x[o + 1] : u;
                if (rot0) {
                    const float a = Cvt<T>::to_f(u), d = Cvt<T>::to_f(w);
                    y[o] = Cvt<T>::from_f(a * c[0] - d * s[0]);
                    y[o + 1] = Cvt<T>::from_f(a * s[0] + d * c[0]);
                } else {
                    y[o] = u;
                    if (two) y[o + 1] = w;
                }
            }
        }
    }
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
    // Heads a thread walks over: as many as leave 8 warps on every scheduler
    // (the sines are then shared by the most heads), at least one.
    const long threads = P.rows * P.items, want = (long)op_sms() * 1024;
    long chunks = (want + threads - 1) / threads;
    if (chunks > a.heads) chunks = a.heads;
    P.hchunk = (int)((a.heads + chunks - 1) / chunks);
    const dim3 g((unsigned)((threads + 255) / 256), (a.heads + P.hchunk - 1) / P.hchunk);
    if (threads > 256L * 2147483647L || g.y > 65535) return -1;
    if (P.p.half) k_rope<T, VEC, true><<<g, 256, 0, s>>>(P);
    else k_rope<T, VEC, false><<<g, 256, 0, s>>>(P);
    return 1;
}

template <typename T>
int launch_t(const RopeArgs& a, cudaStream_t s) {
    // 16-byte pieces where every head starts on one and neither layout cuts
    // a piece in two; single elements otherwise
    constexpr int V = 16 / (int)sizeof(T);
    bool ok = ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.y & 15) == 0 && a.head_dim % V == 0 &&
              (!a.plan->half || a.plan->pairs % V == 0);
    const long n[3] = {a.batch, a.tokens, a.heads};
    for (int i = 0; i < 3; i++)
        if (n[i] > 1 && (a.xs[i] % V || a.ys[i] % V)) ok = false;
    return ok ? launch<T, V>(a, s) : launch<T, 1>(a, s);
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
