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
// token at a time.  The first heads are loaded before anything else; while they
// are on their way a token's threads share the evaluation of its sines, and all
// heads of the CTA read them from shared memory.  (Each thread its own sines:
// where only 16 of 64 pairs turn, every warp waits for the few threads that
// turn, 147 us against 99 for 8 heads of 131042 tokens in bf16; 25 against 20
// for the grid below.)  Chunks of heads are neighbouring CTAs, so the CTAs
// together walk through memory in order.  B200, in a burst: 40 heads of 128 at
// 5440 tokens in bf16 (111 MB) 19.8 us; 8 heads of 128 at 131042 tokens in fp32
// (1.07 GB) 170 us, 6.3 TB/s (176 to 182 in a long run).
#include "kcommon.cuh"
#include "launch.cuh"
#include "ops.h"

namespace s2b {
namespace {

// CTAs an SM: 64 registers a thread hold four heads' pieces; three CTAs of 85
// take 25.1 us against 22.5 for 40 heads of 5440 tokens in halves.
constexpr int ROPE_CTAS = 4;
// CTAs an SM that a launch keeps when its CTAs take several batches of heads:
// at 16 the grid of 5440 tokens takes one batch a CTA, 23.8 us against 19.8.
constexpr int ROPE_WAVES = 8, ROPE_PASSES = 3;
struct RopeParams {
    s2b_rope p;
    const void* x; void* y;
    long xb, xt, xh, yb, yt, yh;        // element strides
    const int* pos; long pos_bs;
    int pos0, tokens, heads, D;
    int items, tpc, per, jt;            // pieces a token, tokens a CTA, threads a token, CTAs a token
    int chunks, passes;                 // CTAs of heads, batches of heads a CTA
    long rows;                          // batch * tokens
    float sign;                         // -1 turns back
};

// A piece of VEC >= 2 values as 32-bit words: moved whole (value by value the
// compiler splits the stores of 16-bit types, 25 us against 22 for 40 heads of
// 5440 tokens), converted two at a time.
template <int WORDS> struct alignas(WORDS * 4) Words { uint32_t w[WORDS]; };
template <typename T> struct Two;        // the pairs of values that words hold
template <> struct Two<float> {
    static constexpr int W = 2;          // words of two values
    static __device__ __forceinline__ float2 get(const uint32_t* w) { return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1])); }
    static __device__ __forceinline__ void put(uint32_t* w, float a, float b) { w[0] = __float_as_uint(a); w[1] = __float_as_uint(b); }
};
template <> struct Two<bf16> {
    static constexpr int W = 1;
    static __device__ __forceinline__ float2 get(const uint32_t* w) { return make_float2(__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u)); }
    static __device__ __forceinline__ void put(uint32_t* w, float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        w[0] = *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct Two<f16> {
    static constexpr int W = 1;
    static __device__ __forceinline__ float2 get(const uint32_t* w) { return __half22float2(*reinterpret_cast<const __half2*>(w)); }
    static __device__ __forceinline__ void put(uint32_t* w, float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        w[0] = *reinterpret_cast<const uint32_t*>(&h);
    }
};

// The plan in shared memory: lanes read different pairs, which the constant
// bank of the kernel's arguments would serve one after another.
struct SharedPlan {
    uint64_t turns[S2B_ROPE_MAX_PAIRS];
    uint8_t axis[S2B_ROPE_MAX_PAIRS];
};

// (a, d) -> (a c - d s, a s + d c): two packed multiply-adds.
__device__ __forceinline__ float2 rotate(float a, float d, float2 cs) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, cc, ss, t;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%3, %2};\n\t"
        "mov.b64 cc, {%4, %4};\n\tmov.b64 ss, {%6, %5};\n\t"
        "mul.rn.f32x2 t, y, ss;\n\tfma.rn.f32x2 t, x, cc, t;\n\t"
        "mov.b64 {%0, %1}, t;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a), "f"(d), "f"(cs.x), "f"(cs.y), "f"(-cs.y));
    return r;
}

// Cosine and sine, times the amplitude, of pair i at a token.
__device__ __forceinline__ float2 turn(const RopeParams& P, const SharedPlan& S, int i, const int* pos, int t) {
    const int64_t p = pos ? (int64_t)pos[S.axis[i]] : (int64_t)P.pos0 + t;
    const uint64_t f = (uint64_t)p * S.turns[i];         // wraps whole turns away
    // top 32 bits as a signed fraction of half a turn in [-1, 1), rounded to fp32:
    // by up to 2^-26 of a turn next to half a turn
    const float half = (float)(int32_t)(f >> 32) * 4.656612873077393e-10f;
    float2 r;
    sincospif(half, &r.y, &r.x);
    r.x *= P.p.amplitude;
    r.y *= P.p.amplitude * P.sign;
    return r;
}

// Item j of a token's head: interleaved, elements [j VEC, (j + 1) VEC); half,
// the first pairs / VEC items hold elements [j VEC, ..) of both halves and the
// rest the copied tail.  VEC = 1 interleaved items hold one element pair.  In HU
// heads from x (to y): load() has all of them on their way, store() turns them
// by the token's cosines and sines cs and writes them.  Loads go ahead of every
// store of their heads: x and y may be the same buffer.
template <typename T, int VEC, bool HALF, int HU> struct Item {
    static constexpr int NW = VEC * (int)sizeof(T) / 4;
    typedef Words<NW> V;
    V u[HU], w[HALF ? HU : 1];
    __device__ __forceinline__ void load(const RopeParams& P, int j, const T* x) {
        const int np = P.p.pairs, nrot = np / VEC;
        const bool turned = HALF ? j < nrot : j * VEC < 2 * np;
        if (!turned && P.x == P.y) return;
        const int o = !HALF || turned ? j * VEC : 2 * np + (j - nrot) * VEC;
        #pragma unroll
        for (int k = 0; k < HU; k++) {
            u[k] = *reinterpret_cast<const V*>(x + k * P.xh + o);
            if constexpr (HALF)
                if (turned) w[k] = *reinterpret_cast<const V*>(x + k * P.xh + o + np);
        }
    }
    __device__ __forceinline__ void store(const RopeParams& P, int j, T* y, const float2* cs) {
        constexpr int W2 = Two<T>::W;
        const int np = P.p.pairs, nrot = np / VEC;
        const bool turned = HALF ? j < nrot : j * VEC < 2 * np;
        if (!turned && P.x == P.y) return;
        const int o = !HALF || turned ? j * VEC : 2 * np + (j - nrot) * VEC;
        if (turned) {
            if constexpr (HALF) {
                #pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    const float4 c = *reinterpret_cast<const float4*>(cs + j * VEC + 2 * i);
                    #pragma unroll
                    for (int k = 0; k < HU; k++) {
                        const float2 a = Two<T>::get(u[k].w + i * W2), d = Two<T>::get(w[k].w + i * W2);
                        const float2 r = rotate(a.x, d.x, make_float2(c.x, c.y)), q = rotate(a.y, d.y, make_float2(c.z, c.w));
                        Two<T>::put(u[k].w + i * W2, r.x, q.x);
                        Two<T>::put(w[k].w + i * W2, r.y, q.y);
                    }
                }
            } else {
                #pragma unroll
                for (int i = 0; i < VEC / 2; i++) {
                    if (j * (VEC / 2) + i >= np) break;          // copied bits stay the bits they were
                    const float2 c = cs[j * (VEC / 2) + i];
                    #pragma unroll
                    for (int k = 0; k < HU; k++) {
                        const float2 a = Two<T>::get(u[k].w + i * W2), r = rotate(a.x, a.y, c);
                        Two<T>::put(u[k].w + i * W2, r.x, r.y);
                    }
                }
            }
        }
        #pragma unroll
        for (int k = 0; k < HU; k++) {
            *reinterpret_cast<V*>(y + k * P.yh + o) = u[k];
            if constexpr (HALF)
                if (turned) *reinterpret_cast<V*>(y + k * P.yh + o + np) = w[k];
        }
    }
};
// Single values.
template <typename T, bool HALF, int HU> struct Item<T, 1, HALF, HU> {
    T u[HU], w[HU];
    static __device__ __forceinline__ bool place(const RopeParams& P, int j, int& a, int& b) {
        const int np = P.p.pairs;
        if (j < np) { a = HALF ? j : 2 * j; b = HALF ? j + np : 2 * j + 1; return true; }
        a = HALF ? np + j : 2 * j;
        b = HALF || a + 1 >= P.D ? -1 : a + 1;                   // an odd head's last element stands alone
        return P.x != P.y;
    }
    __device__ __forceinline__ void load(const RopeParams& P, int j, const T* x) {
        int a, b;
        if (!place(P, j, a, b)) return;
        #pragma unroll
        for (int k = 0; k < HU; k++) {
            u[k] = x[k * P.xh + a];
            if (b >= 0) w[k] = x[k * P.xh + b];
        }
    }
    __device__ __forceinline__ void store(const RopeParams& P, int j, T* y, const float2* cs) {
        int a, b;
        if (!place(P, j, a, b)) return;
        const bool turned = j < P.p.pairs;
        const float2 c = turned ? cs[j] : make_float2(1.f, 0.f);
        #pragma unroll
        for (int k = 0; k < HU; k++) {
            T lo = u[k], hi = w[k];
            if (turned) {
                const float2 r = rotate(Cvt<T>::to_f(lo), Cvt<T>::to_f(hi), c);
                lo = Cvt<T>::from_f(r.x);
                hi = Cvt<T>::from_f(r.y);
            }
            y[k * P.yh + a] = lo;
            if (b >= 0) y[k * P.yh + b] = hi;
        }
    }
};

template <typename T, int VEC, bool HALF, int HU>
__global__ void __launch_bounds__(256, ROPE_CTAS) k_rope(const __grid_constant__ RopeParams P) {
    __shared__ SharedPlan S;
    // a CTA's tokens x pairs: 256 items of VEC pairs (half) or VEC / 2, rows
    // rounded up to an even number
    __shared__ alignas(16) float2 cs[256 * (HALF || VEC == 1 ? VEC : VEC / 2) + 256];
    const int np = P.p.pairs, pitch = (np + 1) & ~1;
    if (threadIdx.x < np) {
        S.turns[threadIdx.x] = P.p.turns[threadIdx.x];
        S.axis[threadIdx.x] = P.p.axis[threadIdx.x];
    }
    __syncthreads();
    chain_begin();
    unsigned at = blockIdx.x;
    const int chunk = at % P.chunks;
    at /= P.chunks;
    const int jt = at % P.jt;
    const int tok = threadIdx.x / P.per, slot = threadIdx.x - tok * P.per, j = slot + jt * 256;
    const long row = (long)(at / P.jt) * P.tpc + tok;
    const bool mine = tok < P.tpc && row < P.rows, on = mine && slot < P.items && j < P.items;
    // 64-bit division costs more than the rest of a thread's work
    const long b = !mine ? 0 : P.rows < (1L << 32) ? (long)((unsigned)row / (unsigned)P.tokens) : row / P.tokens;
    const int t = mine ? (int)(row - b * P.tokens) : 0;
    const T* x = (const T*)P.x + b * P.xb + t * P.xt + (long)chunk * P.passes * HU * P.xh;
    T* y = (T*)P.y + b * P.yb + t * P.yt + (long)chunk * P.passes * HU * P.yh;
    Item<T, VEC, HALF, HU> item;
    if (on) item.load(P, j, x);
    // the sines while the first heads are on their way: a token's threads share
    // its pairs, and the CTA's heads their values
    float2* tcs = cs + tok * pitch;
    if (mine) {
        const int* pos = P.pos ? P.pos + b * P.pos_bs + (long)t * P.p.axes : nullptr;
        #pragma unroll 2
        for (int i = slot; i < np; i += P.per) tcs[i] = turn(P, S, i, pos, t);
    }
    __syncthreads();
    if (!on) return;
    item.store(P, j, y, tcs);
    for (int n = 1; n < P.passes; n++) {
        x += HU * P.xh;
        y += HU * P.yh;
        item.load(P, j, x);
        item.store(P, j, y, tcs);
    }
}

template <typename T, int VEC, int HU>
int launch_hu(RopeParams& P, long ctas, cudaStream_t s) {
    // batches of heads that share a CTA's sines; they are loaded one after the
    // other, so more than ROPE_PASSES cost more than they save (five: 36.6 us
    // against 34.7 for the grid in fp32)
    const int batches = P.heads / HU;
    P.passes = 1;
    for (int p = 2; p <= ROPE_PASSES && ctas * (batches / p) >= ROPE_WAVES * (long)op_sms(); p++)
        if (batches % p == 0) P.passes = p;
    P.chunks = batches / P.passes;
    const long g = ctas * P.chunks;
    if (g > 2147483647L) return -1;
    return launch_chained(P.p.half ? k_rope<T, VEC, true, HU> : k_rope<T, VEC, false, HU>, dim3((unsigned)g), 256, 0, 0, s, P);
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
    if (P.rows < P.tpc) P.tpc = P.rows ? (int)P.rows : 1;
    P.per = 256 / P.tpc;
    P.jt = (P.items + 255) / 256;
    const long ctas = (P.rows + P.tpc - 1) / P.tpc * P.jt;
    if (P.items == 0 || ctas == 0) return 0;
    // Heads that a thread loads together: the most, up to four, that divide the
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
