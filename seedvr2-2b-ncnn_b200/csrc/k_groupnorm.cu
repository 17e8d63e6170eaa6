// k_groupnorm.cu -- GroupNorm (+ SiLU) over channel-last rows.
//
//   y = act((x - mean_g) * rstd_g * gamma_c + beta_c), rstd = 1 / sqrt(var + eps),
//   mean and (biased) variance over the rows and channels of group g of one
//   sample.
//
// Statistics are fp32: every thread sums d = x - x0 and d^2 about the first
// value x0 that it meets in a channel, so a mean far from zero cancels
// nothing, and (n, mean, M2) triples are joined pairwise by
//   mean = m1 + (m2 - m1) n2 / n,  M2 = M2_1 + M2_2 + (m2 - m1)^2 n1 n2 / n
// (Chan, Golub, LeVeque 1979) in an order that depends on the sizes alone.
// Means are kept as offsets from the group's first value `ref`, and the
// normalisation computes (x - ref) - offset: a mean far from zero is never
// rounded to fp32's step at its own size.
//
// Bound by HBM.  Three launches: partial statistics of row chunks, their join
// per group, and the normalisation, which reads x again.
#include "kcommon.cuh"
#include "ops.h"

namespace s2b {
namespace {

constexpr int THREADS = 256;

struct GnParams {
    const void* x; void* y;
    const float *gamma, *beta;
    float4* stat;       // [batch][groups] (ref, mean - ref, rstd, -)
    float2* part;       // [batch][chunks][channels] (mean - ref, M2) of a chunk's rows
    int rows, C, ldx, ldy, G, cpg, chunk, chunks;
    float eps;
    int silu;
};

struct Moments { float n, mean, m2; };
__device__ __forceinline__ Moments join(Moments a, Moments b) {
    if (b.n == 0.f) return a;
    if (a.n == 0.f) return b;
    const float n = a.n + b.n, d = b.mean - a.mean, w = __fdividef(b.n, n);
    return {n, fmaf(d, w, a.mean), a.m2 + b.m2 + d * d * a.n * w};
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

// Vector columns a CTA covers and the rows it takes side by side.
__host__ __device__ inline int tile_cols(int vecs) { return vecs < THREADS ? vecs : THREADS; }

constexpr int UNROLL = 4;

template <typename T, int VEC>
__global__ void __launch_bounds__(THREADS) k_gn_stats(const GnParams P) {
    typedef Vec<T, VEC> V;
    __shared__ float2 sm[THREADS * VEC];
    const int vecs = P.C / VEC, tw = tile_cols(vecs), rp = THREADS / tw;
    const int tc = threadIdx.x % tw, tr = threadIdx.x / tw;
    const int vc = blockIdx.y * tw + tc;
    const int r0 = blockIdx.x * P.chunk, r1 = min(P.rows, r0 + P.chunk);
    const bool on = tr < rp && vc < vecs;
    const T* x = (const T*)P.x + ((size_t)blockIdx.z * P.rows) * P.ldx + (size_t)vc * VEC;
    float x0[VEC], s[VEC], q[VEC];
    int n = 0;
    #pragma unroll
    for (int i = 0; i < VEC; i++) { x0[i] = 0.f; s[i] = 0.f; q[i] = 0.f; }
    if (on && r0 + tr < r1) {
        const V f = *reinterpret_cast<const V*>(x + (size_t)(r0 + tr) * P.ldx);
        #pragma unroll
        for (int i = 0; i < VEC; i++) x0[i] = Cvt<T>::to_f(f.v[i]);
        int r = r0 + tr;
        for (; r + (UNROLL - 1) * rp < r1; r += UNROLL * rp) {
            V u[UNROLL];
            #pragma unroll
            for (int k = 0; k < UNROLL; k++) u[k] = *reinterpret_cast<const V*>(x + (size_t)(r + k * rp) * P.ldx);
            #pragma unroll
            for (int k = 0; k < UNROLL; k++)
                #pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = Cvt<T>::to_f(u[k].v[i]) - x0[i];
                    s[i] += d;
                    q[i] = fmaf(d, d, q[i]);
                }
            n += UNROLL;
        }
        for (; r < r1; r += rp, n++) {
            const V u = *reinterpret_cast<const V*>(x + (size_t)r * P.ldx);
            #pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = Cvt<T>::to_f(u.v[i]) - x0[i];
                s[i] += d;
                q[i] = fmaf(d, d, q[i]);
            }
        }
    }
    // (mean, M2) of every thread's rows, then the rp row lanes of a channel in order
    const float inv = n ? 1.f / (float)n : 0.f;
    #pragma unroll
    for (int i = 0; i < VEC; i++) {
        const float m = s[i] * inv, m2 = q[i] - s[i] * m;
        const int c = vc * VEC + i;
        const float ref = n ? Cvt<T>::to_f(((const T*)P.x)[(size_t)blockIdx.z * P.rows * P.ldx + c - c % P.cpg]) : 0.f;
        sm[threadIdx.x * VEC + i] = make_float2((x0[i] - ref) + m, m2 < 0.f ? 0.f : m2);     // NaN stays
    }
    __syncthreads();
    const int len = r1 - r0;
    for (int c = threadIdx.x; c < tw * VEC; c += THREADS) {
        if (blockIdx.y * tw * VEC + c >= P.C) break;
        Moments a = {0.f, 0.f, 0.f};
        for (int k = 0; k < rp; k++) {
            const float2 v = sm[k * tw * VEC + c];
            const int nk = k < len ? (len - k + rp - 1) / rp : 0;
            a = join(a, {(float)nk, v.x, v.y});
        }
        P.part[((size_t)blockIdx.z * P.chunks + blockIdx.x) * P.C + blockIdx.y * tw * VEC + c] = make_float2(a.mean, a.m2);
    }
}

// One CTA joins the chunks and channels of one group of one sample.
template <typename T>
__global__ void __launch_bounds__(THREADS) k_gn_join(const GnParams P) {
    __shared__ float sn[8], smean[8], sm2[8];
    const int g = blockIdx.x, b = blockIdx.y;
    const float2* part = P.part + (size_t)b * P.chunks * P.C + (size_t)g * P.cpg;
    const long entries = (long)P.chunks * P.cpg;
    Moments a = {0.f, 0.f, 0.f};
    for (long e = threadIdx.x; e < entries; e += THREADS) {
        const int k = (int)(e / P.cpg), c = (int)(e % P.cpg);
        const float2 v = part[(size_t)k * P.C + c];
        a = join(a, {(float)min(P.chunk, P.rows - k * P.chunk), v.x, v.y});
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Moments u = {__shfl_down_sync(0xffffffffu, a.n, o), __shfl_down_sync(0xffffffffu, a.mean, o),
                           __shfl_down_sync(0xffffffffu, a.m2, o)};
        a = join(a, u);
    }
    if ((threadIdx.x & 31) == 0) {
        sn[threadIdx.x >> 5] = a.n; smean[threadIdx.x >> 5] = a.mean; sm2[threadIdx.x >> 5] = a.m2;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; i++) a = join(a, {sn[i], smean[i], sm2[i]});
        const float ref = Cvt<T>::to_f(((const T*)P.x)[(size_t)b * P.rows * P.ldx + (size_t)g * P.cpg]);
        P.stat[(size_t)b * P.G + g] = make_float4(ref, a.mean, 1.f / sqrtf(a.m2 / a.n + P.eps), 0.f);
    }
}

__device__ __forceinline__ float gn_silu(float v) { return v * __fdividef(1.f, 1.f + __expf(-v)); }

template <typename TX, typename TY, int VEC>
__global__ void __launch_bounds__(THREADS) k_gn_apply(const GnParams P) {
    typedef Vec<TX, VEC> VX;
    typedef Vec<TY, VEC> VY;
    const int vecs = P.C / VEC, tw = tile_cols(vecs), rp = THREADS / tw;
    const int tc = threadIdx.x % tw, tr = threadIdx.x / tw;
    const int vc = blockIdx.y * tw + tc;
    if (tr >= rp || vc >= vecs) return;
    const int r0 = blockIdx.x * P.chunk, r1 = min(P.rows, r0 + P.chunk);
    float ref[VEC], mean[VEC], a[VEC], beta[VEC];
    #pragma unroll
    for (int i = 0; i < VEC; i++) {
        const int c = vc * VEC + i;
        const float4 st = P.stat[(size_t)blockIdx.z * P.G + c / P.cpg];
        ref[i] = st.x;
        mean[i] = st.y;
        a[i] = P.gamma ? st.z * P.gamma[c] : st.z;
        beta[i] = P.beta ? P.beta[c] : 0.f;
    }
    const TX* x = (const TX*)P.x + ((size_t)blockIdx.z * P.rows) * P.ldx + (size_t)vc * VEC;
    TY* y = (TY*)P.y + ((size_t)blockIdx.z * P.rows) * P.ldy + (size_t)vc * VEC;
    auto put = [&](int r, const VX& u) {
        VY o;
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            float v = fmaf((Cvt<TX>::to_f(u.v[i]) - ref[i]) - mean[i], a[i], beta[i]);
            if (P.silu) v = gn_silu(v);
            o.v[i] = Cvt<TY>::from_f(v);
        }
        *reinterpret_cast<VY*>(y + (size_t)r * P.ldy) = o;
    };
    int r = r0 + tr;
    for (; r + (UNROLL - 1) * rp < r1; r += UNROLL * rp) {
        VX u[UNROLL];
        #pragma unroll
        for (int k = 0; k < UNROLL; k++) u[k] = *reinterpret_cast<const VX*>(x + (size_t)(r + k * rp) * P.ldx);
        #pragma unroll
        for (int k = 0; k < UNROLL; k++) put(r + k * rp, u[k]);
    }
    for (; r < r1; r += rp) {
        const VX u = *reinterpret_cast<const VX*>(x + (size_t)r * P.ldx);
        put(r, u);
    }
}

// Row chunks of a sample: enough that batch * chunks fill the GPU several
// times over, at least 16 rows each (the partials are 8 bytes a channel and
// chunk, against 16 rows * 2 bytes of data).
int chunk_rows(int batch, int rows) {
    const long want = (4L * 148 + batch - 1) / batch;
    long c = (rows + want - 1) / want;
    return (int)(c < 16 ? 16 : c);
}

template <typename TX, typename TY>
int launch(const GroupNormArgs& a, cudaStream_t s) {
    GnParams P;
    P.x = a.x; P.y = a.y; P.gamma = a.gamma; P.beta = a.beta;
    P.rows = a.rows; P.C = a.channels; P.ldx = a.ldx; P.ldy = a.ldy;
    P.G = a.groups; P.cpg = a.channels / a.groups;
    P.eps = a.eps; P.silu = a.act;
    P.chunk = chunk_rows(a.batch, a.rows);
    P.chunks = (a.rows + P.chunk - 1) / P.chunk;
    P.stat = (float4*)a.work;
    P.part = (float2*)(P.stat + (size_t)a.batch * P.G);
    constexpr int V = 16 / (int)(sizeof(TX) > sizeof(TY) ? sizeof(TX) : sizeof(TY));
    const bool vec = a.channels % V == 0 && a.ldx % V == 0 && a.ldy % V == 0 &&
                     ((uintptr_t)a.x % (V * sizeof(TX))) == 0 && ((uintptr_t)a.y % (V * sizeof(TY))) == 0;
    const int vecs = a.channels / (vec ? V : 1), tiles = (vecs + tile_cols(vecs) - 1) / tile_cols(vecs);
    if (tiles > 65535) return -1;
    const dim3 g(P.chunks, tiles, a.batch);
    if (vec) k_gn_stats<TX, V><<<g, THREADS, 0, s>>>(P);
    else k_gn_stats<TX, 1><<<g, THREADS, 0, s>>>(P);
    k_gn_join<TX><<<dim3(P.G, a.batch), THREADS, 0, s>>>(P);
    if (vec) k_gn_apply<TX, TY, V><<<g, THREADS, 0, s>>>(P);
    else k_gn_apply<TX, TY, 1><<<g, THREADS, 0, s>>>(P);
    return 3;
}

template <typename TX>
int launch_y(const GroupNormArgs& a, cudaStream_t s) {
    switch (a.y_type) {
        case S2B_PREC_FP32: return launch<TX, float>(a, s);
        case S2B_PREC_FP16: return launch<TX, f16>(a, s);
        default: return launch<TX, bf16>(a, s);
    }
}

}  // namespace

size_t groupnorm_workspace(int batch, int rows, int channels, int groups) {
    if (batch <= 0 || rows <= 0 || channels <= 0 || groups <= 0) return 0;
    const int chunk = chunk_rows(batch, rows);
    const size_t chunks = ((size_t)rows + chunk - 1) / chunk;
    return (size_t)batch * chunks * channels * sizeof(float2) + (size_t)batch * groups * sizeof(float4);
}

int op_launch(const GroupNormArgs& a, cudaStream_t s) {
    switch (a.x_type) {
        case S2B_PREC_FP32: return launch_y<float>(a, s);
        case S2B_PREC_FP16: return launch_y<f16>(a, s);
        default: return launch_y<bf16>(a, s);
    }
}

}  // namespace s2b
