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
// Bound by HBM, or by launches and latency when small.  Two forms:
//   on chip   a cluster of CTAs takes one sample's slab of whole groups,
//             holds it in registers between the statistics and the
//             normalisation: x is read once, one launch;
//   streamed  samples whose slabs exceed a cluster's registers: partial
//             statistics of row chunks, their join per group, and the
//             normalisation, which reads x again, last chunk first: what the
//             statistics read last is still in L2.
//
// B200: on chip 1360 x 512 bf16 6.6 us; streamed 3 x 21760 x 512 (134 MB read and
// written once) 41 us, 1392640 x 128 with SiLU (713 MB, x read twice) 200 us,
// 184 without: 5.4 TB/s of what DRAM has to move.
#include "kcommon.cuh"
#include "launch.cuh"
#include "ops.h"
#include "sm100.cuh"

namespace s2b {
namespace {

constexpr int THREADS = 256;
constexpr int STATS_CTAS = 3, APPLY_CTAS = 4;      // resident on an SM
constexpr int CHIP_GROUPS = 64;          // groups of an on-chip slab

struct GnParams {
    const void* x; void* y;
    const float *gamma, *beta;
    float4* stat;       // [batch][groups] (ref, mean - ref, rstd, -)
    float4* part;       // [batch][chunks * tiles][groups] (n, mean - ref, M2, -); n 0: none of the group's channels
    int rows, C, ldx, ldy, G, cpg;
    int chunk, chunks, tiles;           // streamed
    int slab, slabs, split, share;      // on chip: channels a slab, slabs, CTAs a cluster, rows a CTA
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

__device__ __forceinline__ Moments shfl_join(Moments a) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = join(a, {__shfl_down_sync(0xffffffffu, a.n, o), __shfl_down_sync(0xffffffffu, a.mean, o),
                     __shfl_down_sync(0xffffffffu, a.m2, o)});
    return a;
}

// Joins what the threads of a CTA hold of each group: sm[k * width + c] is
// (mean - ref, M2) of row lane k and the CTA's run c of SUB channels (the
// first is the operator's run c0), from count(k) rows of them.  One warp a
// group, lanes over its runs and row lanes; done(g, moments) runs on lane 0.
template <int SUB, typename Count, typename Done>
__device__ __forceinline__ void join_groups(const float2* sm, int width, int lanes, int c0, int cpg, Count count, Done done) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = cpg / SUB;     // runs a group
    const int g0 = c0 / per, g1 = (c0 + width - 1) / per;
    for (int g = g0 + warp; g <= g1; g += THREADS / 32) {
        const int a = max(g * per - c0, 0), b = min((g + 1) * per - c0, width), w = b - a;
        Moments m = {0.f, 0.f, 0.f};
        int k = lane / w, c = lane - k * w;
        const int dk = 32 / w, dc = 32 - dk * w;
        for (; k < lanes;) {
            const float2 v = sm[k * width + a + c];
            m = join(m, {(float)(count(k) * SUB), v.x, v.y});
            k += dk; c += dc;
            if (c >= w) { c -= w; k++; }
        }
        m = shfl_join(m);
        if (lane == 0) done(g, m);
    }
}

// Vector columns a CTA covers and the rows it takes side by side.
__host__ __device__ inline int tile_cols(int vecs) { return vecs < THREADS ? vecs : THREADS; }

// SUB: channels of a vector that share a group, taken together (VEC, VEC / 2,
// or 1 for groups that cut vectors otherwise).
template <typename T, int VEC, int SUB>
__global__ void __launch_bounds__(THREADS, STATS_CTAS) k_gn_stats(const GnParams P) {
    typedef Vec<T, VEC> V;
    constexpr int N = VEC / SUB, UNROLL = 8;
    __shared__ float2 sm[THREADS * N];
    chain_begin();
    const int vecs = P.C / VEC, tw = tile_cols(vecs), rp = THREADS / tw;
    const int tc = threadIdx.x % tw, tr = threadIdx.x / tw;
    const int vc = blockIdx.y * tw + tc;
    const int r0 = blockIdx.x * P.chunk, r1 = min(P.rows, r0 + P.chunk);
    const bool on = tr < rp && vc < vecs;
    const T* base = (const T*)P.x + ((size_t)blockIdx.z * P.rows) * P.ldx;
    const T* x = base + (size_t)vc * VEC;
    float x0[N], s[N], q[N];
    #pragma unroll
    for (int i = 0; i < N; i++) { x0[i] = 0.f; s[i] = 0.f; q[i] = 0.f; }
    auto add = [&](const V& u) {
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float d = Cvt<T>::to_f(u.v[i]) - x0[i / SUB];
            s[i / SUB] += d;
            q[i / SUB] = fmaf(d, d, q[i / SUB]);
        }
    };
    const int width = (min(tw * VEC, P.C - (int)blockIdx.y * tw * VEC)) / SUB, len = r1 - r0;
    if (on) {
        int n = 0;
        if (r0 + tr < r1) {
            const V f = *reinterpret_cast<const V*>(x + (size_t)(r0 + tr) * P.ldx);
            #pragma unroll
            for (int i = 0; i < N; i++) x0[i] = Cvt<T>::to_f(f.v[i * SUB]);
            n = (len - tr + rp - 1) / rp;
            const T* p = x + (size_t)(r0 + tr) * P.ldx;
            const size_t step = (size_t)rp * P.ldx;
            int k = 0;
            for (; k + UNROLL <= n; k += UNROLL, p += UNROLL * step) {
                V u[UNROLL];
                #pragma unroll
                for (int j = 0; j < UNROLL; j++) u[j] = *reinterpret_cast<const V*>(p + j * step);
                #pragma unroll
                for (int j = 0; j < UNROLL; j++) add(u[j]);
            }
            for (; k < n; k++, p += step) add(*reinterpret_cast<const V*>(p));
        }
        const float inv = n ? 1.f / (float)(n * SUB) : 0.f;
        #pragma unroll
        for (int i = 0; i < N; i++) {
            const float m = s[i] * inv, m2 = q[i] - s[i] * m;
            const float ref = Cvt<T>::to_f(base[(vc * VEC + i * SUB) / P.cpg * P.cpg]);
            sm[tr * width + tc * N + i] = make_float2((x0[i] - ref) + m, m2 < 0.f ? 0.f : m2);     // NaN stays
        }
    }
    // groups that have no channel in this tile
    float4* part = P.part + (((size_t)blockIdx.z * P.chunks + blockIdx.x) * P.tiles + blockIdx.y) * P.G;
    const int run0 = blockIdx.y * tw * N;
    if (P.tiles > 1) {
        const int per = P.cpg / SUB, g0 = run0 / per, g1 = (run0 + width - 1) / per;
        for (int g = threadIdx.x; g < P.G; g += THREADS)
            if (g < g0 || g > g1) part[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
    join_groups<SUB>(sm, width, rp, run0, P.cpg, [&](int k) { return k < len ? (len - k + rp - 1) / rp : 0; },
                     [&](int g, Moments m) { part[g] = make_float4(m.n, m.mean, m.m2, 0.f); });
}

__device__ __forceinline__ float4 finish(float ref, Moments m, float eps) {
    return make_float4(ref, m.mean, 1.f / sqrtf(m.m2 / m.n + eps), 0.f);
}

// One CTA joins the chunks of one group of one sample: at most four of them a
// thread at the usual sizes, all loaded together.
template <typename T>
__global__ void __launch_bounds__(128) k_gn_join(const GnParams P) {
    __shared__ float4 sm[4];
    chain_begin();
    const int g = blockIdx.x, b = blockIdx.y;
    const float ref = Cvt<T>::to_f(((const T*)P.x)[(size_t)b * P.rows * P.ldx + (size_t)g * P.cpg]);
    const int entries = P.chunks * P.tiles;
    const float4* part = P.part + (size_t)b * entries * P.G + g;
    Moments a = {0.f, 0.f, 0.f};
    for (int e = threadIdx.x; e < entries; e += 4 * 128) {
        float4 v[4];
        #pragma unroll
        for (int k = 0; k < 4; k++) v[k] = e + 128 * k < entries ? part[(size_t)(e + 128 * k) * P.G] : make_float4(0.f, 0.f, 0.f, 0.f);
        #pragma unroll
        for (int k = 0; k < 4; k++) a = join(a, {v[k].x, v[k].y, v[k].z});
    }
    a = shfl_join(a);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_float4(a.n, a.mean, a.m2, 0.f);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 4; i++) a = join(a, {sm[i].x, sm[i].y, sm[i].z});
        P.stat[(size_t)b * P.G + g] = finish(ref, a, P.eps);
    }
}

// v / (1 + e^-v); the fast exponential and division are off by 2^-21 together,
// far below a 16-bit output's half step and within a few steps of fp32's.
__device__ __forceinline__ float gn_silu(float v) { return v * __fdividef(1.f, 1.f + __expf(-v)); }

// act((x - ref - mean) * a + beta) of VEC channels.
template <typename TX, typename TY, int VEC, int SUB>
struct Affine {
    float ref[VEC / SUB], mean[VEC / SUB], a[VEC], beta[VEC];
    __device__ __forceinline__ void weights(const GnParams& P, int c0) {
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            a[i] = P.gamma ? P.gamma[c0 + i] : 1.f;
            beta[i] = P.beta ? P.beta[c0 + i] : 0.f;
        }
    }
    __device__ __forceinline__ void stats(int i, float4 st) {       // run i
        ref[i] = st.x;
        mean[i] = st.y;
        #pragma unroll
        for (int j = i * SUB; j < (i + 1) * SUB; j++) a[j] *= st.z;
    }
    template <bool SILU>
    __device__ __forceinline__ Vec<TY, VEC> run(const Vec<TX, VEC>& u) const {
        Vec<TY, VEC> o;
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            float v = fmaf((Cvt<TX>::to_f(u.v[i]) - ref[i / SUB]) - mean[i / SUB], a[i], beta[i]);
            if (SILU) v = gn_silu(v);
            o.v[i] = Cvt<TY>::from_f(v);
        }
        return o;
    }
    __device__ __forceinline__ Vec<TY, VEC> operator()(const Vec<TX, VEC>& u, bool silu) const {
        return silu ? run<true>(u) : run<false>(u);
    }
};

template <typename TX, typename TY, int VEC, int SUB>
__global__ void __launch_bounds__(THREADS, APPLY_CTAS) k_gn_apply(const GnParams P) {
    typedef Vec<TX, VEC> VX;
    typedef Vec<TY, VEC> VY;
    constexpr int U = 4;
    const int vecs = P.C / VEC, tw = tile_cols(vecs), rp = THREADS / tw;
    const int tc = threadIdx.x % tw, tr = threadIdx.x / tw;
    const int vc = blockIdx.y * tw + tc;
    const int b = gridDim.z - 1 - blockIdx.z;
    chain_begin();
    if (tr >= rp || vc >= vecs) return;
    Affine<TX, TY, VEC, SUB> f;
    f.weights(P, vc * VEC);
    #pragma unroll
    for (int i = 0; i < VEC / SUB; i++) f.stats(i, P.stat[(size_t)b * P.G + (vc * VEC + i * SUB) / P.cpg]);
    // tiles of U * rp rows, the CTAs side by side through the sample from its
    // end: the rows that the statistics read last come first, and all CTAs
    // together touch one window of memory
    const int tile = U * rp, tiles = (P.rows + tile - 1) / tile;
    const size_t sx = (size_t)rp * P.ldx, sy = (size_t)rp * P.ldy;
    for (int t = tiles - 1 - (int)blockIdx.x; t >= 0; t -= (int)gridDim.x) {
        const int r = t * tile + tr;
        const TX* x = (const TX*)P.x + ((size_t)b * P.rows + r) * P.ldx + (size_t)vc * VEC;
        TY* y = (TY*)P.y + ((size_t)b * P.rows + r) * P.ldy + (size_t)vc * VEC;
        if (r + (U - 1) * rp < P.rows) {
            VX u[U];
            #pragma unroll
            for (int j = 0; j < U; j++) u[j] = *reinterpret_cast<const VX*>(x + j * sx);
            #pragma unroll
            for (int j = 0; j < U; j++) *reinterpret_cast<VY*>(y + j * sy) = f(u[j], P.silu);
        } else {
            for (int j = 0; j < U && r + j * rp < P.rows; j++)
                *reinterpret_cast<VY*>(y + j * sy) = f(*reinterpret_cast<const VX*>(x + j * sx), P.silu);
        }
    }
}

// ---------------------------------------------------------------- on chip
// Cluster rank k takes rows [k share, (k + 1) share) of a slab; a thread keeps
// up to RV vectors of one vector column.  The CTAs swap their groups' moments
// through distributed shared memory and join them in rank order.
template <typename TX, typename TY, int VEC, int SUB, int RV>
__global__ void __launch_bounds__(THREADS, RV <= 4 ? 3 : 2) k_gn_chip(const GnParams P) {
    typedef Vec<TX, VEC> VX;
    typedef Vec<TY, VEC> VY;
    constexpr int N = VEC / SUB;
    __shared__ float2 sm[THREADS * N];
    __shared__ float4 mine[CHIP_GROUPS];         // this CTA's (n, mean - ref, M2) of the slab's groups
    __shared__ float4 stat[CHIP_GROUPS];
    __shared__ float sref[CHIP_GROUPS];
    chain_begin();
    const int rank = P.split > 1 ? (int)sm100::cluster_ctarank() : 0;
    const int item = blockIdx.x / P.split, b = item / P.slabs, c0 = item % P.slabs * P.slab;
    const int vw = P.slab / VEC, rp = THREADS / vw, width = P.slab / SUB;
    const int tc = threadIdx.x % vw, tr = threadIdx.x / vw;
    const int r0 = rank * P.share, len = max(min(P.rows, r0 + P.share) - r0, 0);
    const bool on = tr < rp;
    const int n = on && tr < len ? (len - tr + rp - 1) / rp : 0;
    const TX* base = (const TX*)P.x + ((size_t)b * P.rows) * P.ldx + c0;
    const int groups = P.slab / P.cpg;
    VX u[RV];
    Affine<TX, TY, VEC, SUB> f;
    if (threadIdx.x < groups) sref[threadIdx.x] = Cvt<TX>::to_f(base[threadIdx.x * P.cpg]);
    if (on) {
        f.weights(P, c0 + tc * VEC);
        const TX* p = base + (size_t)(r0 + tr) * P.ldx + tc * VEC;
        const size_t step = (size_t)rp * P.ldx;
        #pragma unroll
        for (int k = 0; k < RV; k++)
            if (k < n) u[k] = *reinterpret_cast<const VX*>(p + k * step);
        float ref[N];
        #pragma unroll
        for (int i = 0; i < N; i++) ref[i] = Cvt<TX>::to_f(base[(tc * VEC + i * SUB) / P.cpg * P.cpg]);
        float s[N], q[N];
        #pragma unroll
        for (int i = 0; i < N; i++) s[i] = q[i] = 0.f;
        #pragma unroll
        for (int k = 0; k < RV; k++)
            if (k < n) {
                #pragma unroll
                for (int i = 0; i < VEC; i++) s[i / SUB] += Cvt<TX>::to_f(u[k].v[i]) - ref[i / SUB];
            }
        const float inv = n ? 1.f / (float)(n * SUB) : 0.f;
        #pragma unroll
        for (int i = 0; i < N; i++) s[i] *= inv;
        #pragma unroll
        for (int k = 0; k < RV; k++)
            if (k < n) {
                #pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = (Cvt<TX>::to_f(u[k].v[i]) - ref[i / SUB]) - s[i / SUB];
                    q[i / SUB] = fmaf(d, d, q[i / SUB]);
                }
            }
        #pragma unroll
        for (int i = 0; i < N; i++) sm[tr * width + tc * N + i] = make_float2(s[i], q[i]);
    }
    __syncthreads();
    join_groups<SUB>(sm, width, rp, 0, P.cpg, [&](int k) { return k < len ? (len - k + rp - 1) / rp : 0; },
                     [&](int g, Moments m) { mine[g] = make_float4(m.n, m.mean, m.m2, 0.f); });
    if (P.split > 1) sm100::cluster_sync();
    else __syncthreads();
    // a warp a group, a lane a rank: the ranks' moments arrive together
    for (int g = threadIdx.x >> 5; g < groups; g += THREADS / 32) {
        const int r = threadIdx.x & 31;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < P.split) v = P.split > 1 ? sm100::ld_cluster_f32x4(sm100::map_to_rank(&mine[g], r)) : mine[g];
        const Moments a = shfl_join({v.x, v.y, v.z});
        if (r == 0) stat[g] = finish(sref[g], a, P.eps);
    }
    // every rank has read the others' moments and row 0's references: shared
    // memory may go away and y (which may be x) may be written
    if (P.split > 1) sm100::cluster_sync();
    else __syncthreads();
    if (!on) return;
    #pragma unroll
    for (int i = 0; i < N; i++) f.stats(i, stat[(tc * VEC + i * SUB) / P.cpg]);
    TY* y = (TY*)P.y + ((size_t)b * P.rows + r0 + tr) * P.ldy + c0 + tc * VEC;
    const size_t step = (size_t)rp * P.ldy;
    #pragma unroll
    for (int k = 0; k < RV; k++)
        if (k < n) *reinterpret_cast<VY*>(y + k * step) = f(u[k], P.silu);
}

// ---------------------------------------------------------------- host
// Rows of a CTA when `per_sm` CTAs an SM share the batch's rows in one wave,
// rounded up to whole rounds of the row loop (a round is `round` rows; the rest
// of a chunk is loaded one row at a time).
int chunk_rows(long batch, int rows, int per_sm, int round) {
    const long want = (per_sm * 148L + batch - 1) / batch;       // B200's SMs, so that the workspace is a function of sizes
    const long c = (rows + want - 1) / want;
    return (int)((c + round - 1) / round * round);
}
// The on-chip form's slab, cluster and vectors a thread; false when it does
// not fit.  Slabs are the fewest whole groups that make rows of 64 bytes or
// more (two sectors), clusters the smallest that hold a sample's slab and
// then larger while the GPU has idle SMs and a CTA more than 32 rows.
bool plan_chip(const GroupNormArgs& a, int vec, int xe, GnParams& P, int& rv) {
    P.slab = 0;
    for (int k = 1; k <= P.G && k <= CHIP_GROUPS; k++) {
        const long w = (long)k * P.cpg;
        if (P.G % k || w % vec || (w * xe < 64 && w < P.C)) continue;
        if (w / vec > THREADS) break;
        P.slab = (int)w;
        break;
    }
    if (!P.slab) return false;
    P.slabs = P.C / P.slab;
    const int rp = THREADS / (P.slab / vec);
    const long items = (long)a.batch * P.slabs;
    int split = 1;
    while (split < 8 && (a.rows + split - 1) / split > 16 * rp) split *= 2;
    while (split < 8 && items * split < op_sms() && a.rows / split > 32) split *= 2;
    P.share = (a.rows + split - 1) / split;
    const int need = (P.share + rp - 1) / rp;
    if (need > 16 || items * split > 2147483647L) return false;
    P.split = split;
    rv = need <= 4 ? 4 : 16;
    return true;
}

template <typename TX, typename TY, int VEC, int SUB>
bool launch_chip(const GnParams& P, int batch, int rv, cudaStream_t s) {
    return launch_chained(rv == 4 ? k_gn_chip<TX, TY, VEC, SUB, 4> : k_gn_chip<TX, TY, VEC, SUB, 16>,
                          dim3((unsigned)((long)batch * P.slabs * P.split)), THREADS, 0, P.split, s, P);
}

template <typename TX, typename TY, int VEC, int SUB>
int launch_v(const GroupNormArgs& a, GnParams& P, cudaStream_t s) {
    int rv;
    if (plan_chip(a, VEC, sizeof(TX), P, rv)) return launch_chip<TX, TY, VEC, SUB>(P, a.batch, rv, s) ? 1 : -1;
    const int vecs = P.C / VEC;
    P.tiles = (vecs + tile_cols(vecs) - 1) / tile_cols(vecs);
    if (P.tiles > 65535) return -1;
    const int rp = THREADS / tile_cols(vecs);
    P.chunk = chunk_rows((long)a.batch * P.tiles, a.rows, STATS_CTAS, 8 * rp);
    P.chunks = (a.rows + P.chunk - 1) / P.chunk;
    const int achunk = chunk_rows((long)a.batch * P.tiles, a.rows, APPLY_CTAS, 4 * rp);
    P.stat = (float4*)a.work;
    P.part = P.stat + (size_t)a.batch * P.G;
    const dim3 g(P.chunks, P.tiles, a.batch), ga((a.rows + achunk - 1) / achunk, P.tiles, a.batch);
    if (!launch_chained(k_gn_stats<TX, VEC, SUB>, g, THREADS, 0, 0, s, P)) return -1;
    if (!launch_chained(k_gn_join<TX>, dim3(P.G, a.batch), 128, 0, 0, s, P)) return -1;
    if (!launch_chained(k_gn_apply<TX, TY, VEC, SUB>, ga, THREADS, 0, 0, s, P)) return -1;
    return 3;
}

template <typename TX, typename TY>
int launch(const GroupNormArgs& a, cudaStream_t s) {
    GnParams P = {};
    P.x = a.x; P.y = a.y; P.gamma = a.gamma; P.beta = a.beta;
    P.rows = a.rows; P.C = a.channels; P.ldx = a.ldx; P.ldy = a.ldy;
    P.G = a.groups; P.cpg = a.channels / a.groups;
    P.eps = a.eps; P.silu = a.act;
    constexpr int V = 16 / (int)(sizeof(TX) > sizeof(TY) ? sizeof(TX) : sizeof(TY));
    const bool vec = a.channels % V == 0 && a.ldx % V == 0 && a.ldy % V == 0 &&
                     ((uintptr_t)a.x % (V * sizeof(TX))) == 0 && ((uintptr_t)a.y % (V * sizeof(TY))) == 0;
    if (!vec) return launch_v<TX, TY, 1, 1>(a, P, s);
    if (P.cpg % V == 0) return launch_v<TX, TY, V, V>(a, P, s);
    if (P.cpg % (V / 2) == 0) return launch_v<TX, TY, V, V / 2>(a, P, s);
    return launch_v<TX, TY, V, 1>(a, P, s);
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
    // the most chunks x column tiles a call of these sizes can have: whatever
    // the vector width, a wave of CTAs over batch x tiles, or one a tile
    size_t most = 0;
    for (int vec = 1; vec <= 8; vec *= 2) {
        const int vecs = channels / vec < 1 ? 1 : channels / vec, tw = tile_cols(vecs);
        const size_t tiles = (vecs + tw - 1) / tw;
        const int chunk = chunk_rows((long)(batch * tiles), rows, STATS_CTAS, 8 * (THREADS / tw));
        const size_t n = ((size_t)rows + chunk - 1) / chunk * tiles;
        if (n > most) most = n;
    }
    return (size_t)batch * groups * (most + 1) * sizeof(float4);
}

int op_launch(const GroupNormArgs& a, cudaStream_t s) {
    switch (a.x_type) {
        case S2B_PREC_FP32: return launch_y<float>(a, s);
        case S2B_PREC_FP16: return launch_y<f16>(a, s);
        default: return launch_y<bf16>(a, s);
    }
}

}  // namespace s2b
