// k_groupnorm.cu -- GroupNorm (+ SiLU) over channel-last rows.
//
//   y = act((x - mean_g) * rstd_g * gamma_c + beta_c), rstd = 1 / sqrt(var + eps),
//   mean and (biased) variance over the rows and channels of group g of one
//   sample.
//
// Statistics are fp32: a thread takes the values that it holds in registers twice,
// for their mean and for the deviations from it (on chip), or about the mean so
// far (streamed, after the first row), and (n, mean, M2) triples are joined
// pairwise by
//   mean = m1 + (m2 - m1) n2 / n,  M2 = M2_1 + M2_2 + (m2 - m1)^2 n1 n2 / n
// (Chan, Golub, LeVeque 1979) in an order that depends on the sizes alone.
// A mean is a head and the remainder of its rounding (two-sum, Knuth), and the
// normalisation computes (x - head) - remainder: a mean far from zero is never
// rounded to fp32's step at its own size, and nothing hangs on single values:
// sums about the group's first one lost three digits where that was an outlier.
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
// B200, in a burst: on chip 1360 x 512 bf16 6.3 us; streamed 3 x 21760 x 512 (134 MB
// read and written once) 38.4 us, 1392640 x 128 with SiLU (713 MB, x read twice)
// 197 us (204 to 209 in a long run): 5.4 TB/s of what DRAM has to move.  A sample
// of 22 MB is still half in L2 when it is read again (30 MB of 67 come from DRAM).
// The vectors of the 16-row bf16 form on chip are converted once a pass and kept:
// 570 bytes of spill loads a thread.
#include "kcommon.cuh"
#include "launch.cuh"
#include "ops.h"
#include "sm100.cuh"
#include <type_traits>

namespace s2b {
namespace {

constexpr int THREADS = 256;
constexpr int STATS_CTAS = 3, APPLY_CTAS = 4;      // resident on an SM
constexpr int CHIP_GROUPS = 64;          // groups of an on-chip slab

struct GnParams {
    const void* x; void* y;
    const float *gamma, *beta;
    float4* stat;       // [batch][groups] (mean's head, remainder, rstd, -)
    float4* part;       // [batch][chunks * tiles][groups] (n, mean's head, remainder, M2); n 0: none of the group's channels
    int rows, C, ldx, ldy, G, cpg;
    int chunk, chunks, tiles;           // streamed
    int slab, slabs, split, share;      // on chip: channels a slab, slabs, CTAs a cluster, rows a CTA
    float eps;
    int silu;
};

// a + b as the rounded sum and what the rounding lost.
__device__ __forceinline__ void two_sum(float a, float b, float& head, float& rest) {
    head = a + b;
    const float t = head - a;
    rest = (a - (head - t)) + (b - t);
}

// n values about the mean hi + lo; M2 is their squared deviations' sum.
struct Moments { float n, hi, lo, m2; };
// Without branches: the mean moves from the larger side, by at most half the
// difference, and an empty side adds nothing.
__device__ __forceinline__ Moments join(Moments a, Moments b) {
    const bool swap = b.n > a.n;
    const float n = a.n + b.n, few = fminf(a.n, b.n), many = fmaxf(a.n, b.n);
    const float w = few == 0.f ? 0.f : __fdividef(few, n);
    float d = (b.hi - a.hi) + (b.lo - a.lo);
    d = few == 0.f ? 0.f : swap ? -d : d;
    Moments r = {n, 0.f, 0.f, a.m2 + b.m2 + d * d * many * w};
    two_sum(swap ? b.hi : a.hi, fmaf(d, w, swap ? b.lo : a.lo), r.hi, r.lo);
    return r;
}

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

// Moments of the `count` values that `each` hands to its argument: about `base`
// (one of them, so that equal values leave exact zeros) for the mean p, then
// about p.  base may be any distance off: it only moves p, whose own distance
// from the mean the second pass makes good.
template <typename Each>
__device__ __forceinline__ Moments batch_moments(float count, float inv, float base, Each each) {
    float s = 0.f, q = 0.f;
    each([&](float x) { s += x - base; });
    const float p = fmaf(s, inv, base);
    s = 0.f;
    each([&](float x) {
        const float d = x - p;
        s += d;
        q = fmaf(d, d, q);
    });
    const float m = s * inv, m2 = fmaf(-s, m, q);
    Moments r = {count, 0.f, 0.f, m2 < 0.f ? 0.f : m2};          // NaN stays
    two_sum(p, m, r.hi, r.lo);
    return r;
}

// Joined over each `lanes` (a power of two) neighbouring lanes, into their first.
__device__ __forceinline__ Moments shfl_join(Moments a, int lanes) {
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < lanes)
            a = join(a, {__shfl_down_sync(0xffffffffu, a.n, o), __shfl_down_sync(0xffffffffu, a.hi, o),
                         __shfl_down_sync(0xffffffffu, a.lo, o), __shfl_down_sync(0xffffffffu, a.m2, o)});
    return a;
}

// Joins what the threads of a CTA hold of each group: sm[k * width + c] is the
// mean and M2 of row lane k and the CTA's run c of SUB channels (the first is
// the operator's run c0), from count(k) rows of them.  As many threads a group,
// up to a warp, as make one round of it, over its runs and row lanes (a warp a
// group, four rounds of six joins for 32 groups: 43.4 us against 38.4 for three
// samples of 21760 x 512); done(g, moments) runs on the first.
template <int SUB, typename Count, typename Done>
__device__ __forceinline__ void join_groups(const float3* sm, int width, int lanes, int c0, int cpg, Count count, Done done) {
    const int per = cpg / SUB;                   // runs a group
    const int g0 = c0 / per, groups = (c0 + width - 1) / per - g0 + 1;
    int lg = 5;
    while (lg > 0 && groups << lg > THREADS) lg--;
    const int L = 1 << lg, l = threadIdx.x & (L - 1);
    for (int first = 0; first < groups; first += THREADS >> lg) {
        const int g = g0 + first + (threadIdx.x >> lg);
        if (!__any_sync(0xffffffffu, g < g0 + groups)) break;
        const bool on = g < g0 + groups;
        const int a = max(g * per - c0, 0), w = on ? min((g + 1) * per - c0, width) - a : 1;
        Moments m = {0.f, 0.f, 0.f, 0.f};
        int k = on ? l / w : lanes, c = l - l / w * w;
        const int dk = L / w, dc = L - dk * w;
        for (; k < lanes;) {
            const float3 v = sm[k * width + a + c];
            m = join(m, {(float)(count(k) * SUB), v.x, v.y, v.z});
            k += dk; c += dc;
            if (c >= w) { c -= w; k++; }
        }
        __syncwarp();
        m = shfl_join(m, L);
        if (on && l == 0) done(g, m);
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
    __shared__ float3 sm[THREADS * N];
    chain_begin();
    const int vecs = P.C / VEC, tw = tile_cols(vecs), rp = THREADS / tw;
    const int tc = threadIdx.x % tw, tr = threadIdx.x / tw;
    const int vc = blockIdx.y * tw + tc;
    const int r0 = blockIdx.x * P.chunk, r1 = min(P.rows, r0 + P.chunk);
    const bool on = tr < rp && vc < vecs;
    const T* x = (const T*)P.x + ((size_t)blockIdx.z * P.rows) * P.ldx + (size_t)vc * VEC;
    // n values so far about the mean hi + lo, and their M2, run by run
    float n = 0.f, hi[N], lo[N], m2[N];
    #pragma unroll
    for (int i = 0; i < N; i++) { hi[i] = 0.f; lo[i] = 0.f; m2[i] = 0.f; }
    auto first = [&](const V& u) {
        n = SUB;
        #pragma unroll
        for (int i = 0; i < N; i++) {
            const Moments m = batch_moments(SUB, 1.f / SUB, Cvt<T>::to_f(u.v[i * SUB]), [&](auto take) {
                #pragma unroll
                for (int c = 0; c < SUB; c++) take(Cvt<T>::to_f(u.v[i * SUB + c]));
            });
            hi[i] = m.hi; lo[i] = m.lo; m2[i] = m.m2;
        }
    };
    // Rows J .. of u: B values of a run.  With s, q the sums of e = x - mean and of
    // e^2, M2 grows by q - s^2 / (n + B) >= q n / (n + B): an eighth of q behind the
    // first row, half or more from then on, so little cancels wherever the values
    // lie.  (Two passes over every batch took 10 to 15 % longer where groups cut
    // vectors.)
    auto more = [&](const auto& u, auto from) {
        constexpr int J = decltype(from)::value, R = sizeof(u) / sizeof(V), B = (R - J) * SUB;
        n += B;
        const float inv = __fdividef(1.f, n);
        #pragma unroll
        for (int i = 0; i < N; i++) {
            float s = 0.f, q = 0.f;
            #pragma unroll
            for (int j = J; j < R; j++)
                #pragma unroll
                for (int c = 0; c < SUB; c++) {
                    const float d = Cvt<T>::to_f(u[j].v[i * SUB + c]) - hi[i];
                    s += d;
                    q = fmaf(d, d, q);
                }
            const float t = fmaf(-(float)B, lo[i], s);           // about the remainder too
            q = fmaf(-lo[i], s + t, q);
            m2[i] += fmaf(-t * inv, t, q);
            // fast two-sum (Dekker): where the mean moves by more than its own
            // size it errs by a rounding of the step, which M2 holds
            const float g = fmaf(t, inv, lo[i]), h = hi[i] + g;
            lo[i] = g - (h - hi[i]);
            hi[i] = h;
        }
    };
    const std::integral_constant<int, 0> whole;
    const std::integral_constant<int, 1> rest;
    const int width = (min(tw * VEC, P.C - (int)blockIdx.y * tw * VEC)) / SUB, len = r1 - r0;
    if (on) {
        if (r0 + tr < r1) {
            const int rows = (len - tr + rp - 1) / rp;
            const T* p = x + (size_t)(r0 + tr) * P.ldx;
            const size_t step = (size_t)rp * P.ldx;
            auto load = [&](auto& u) {
                constexpr int R = sizeof(u) / sizeof(V);
                #pragma unroll
                for (int j = 0; j < R; j++) u[j] = *reinterpret_cast<const V*>(p + j * step);
                p += R * step;
            };
            V u[UNROLL], one[1];
            int k = 0;
            if (rows >= UNROLL) {
                load(u);
                first(u[0]);
                more(u, rest);
                for (k = UNROLL; k + UNROLL <= rows; k += UNROLL) { load(u); more(u, whole); }
            } else {
                load(one);
                first(one[0]);
                k = 1;
            }
            for (; k < rows; k++) { load(one); more(one, whole); }
        }
        #pragma unroll
        for (int i = 0; i < N; i++) sm[tr * width + tc * N + i] = make_float3(hi[i], lo[i], m2[i] < 0.f ? 0.f : m2[i]);     // NaN stays
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
                     [&](int g, Moments m) { part[g] = make_float4(m.n, m.hi, m.lo, m.m2); });
}

__device__ __forceinline__ float4 finish(Moments m, float eps) {
    return make_float4(m.hi, m.lo, 1.f / sqrtf(m.m2 / m.n + eps), 0.f);
}

// One CTA joins the chunks of one group of one sample: at most four of them a
// thread at the usual sizes, all loaded together.
__global__ void __launch_bounds__(128) k_gn_join(const GnParams P) {
    __shared__ float4 sm[4];
    chain_begin();
    const int g = blockIdx.x, b = blockIdx.y;
    const int entries = P.chunks * P.tiles;
    const float4* part = P.part + (size_t)b * entries * P.G + g;
    Moments a = {0.f, 0.f, 0.f, 0.f};
    for (int e = threadIdx.x; e < entries; e += 4 * 128) {
        float4 v[4];
        #pragma unroll
        for (int k = 0; k < 4; k++) v[k] = e + 128 * k < entries ? part[(size_t)(e + 128 * k) * P.G] : make_float4(0.f, 0.f, 0.f, 0.f);
        const auto of = [](float4 f) { return Moments{f.x, f.y, f.z, f.w}; };
        const Moments four = join(join(of(v[0]), of(v[1])), join(of(v[2]), of(v[3])));
        a = e == (int)threadIdx.x ? four : join(a, four);
    }
    a = shfl_join(a, 32);
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = make_float4(a.n, a.hi, a.lo, a.m2);
    __syncthreads();
    if (threadIdx.x == 0) {
        const auto at = [&](int i) { return Moments{sm[i].x, sm[i].y, sm[i].z, sm[i].w}; };
        P.stat[(size_t)b * P.G + g] = finish(join(join(a, at(1)), join(at(2), at(3))), P.eps);
    }
}

// v sigmoid(v) = v / (1 + e^-v), from e^-|v| so that nothing overflows and the
// denominator lies in [1, 2].  fp32 outputs take expf, within 2 ulp.  For 16-bit
// ones e^-|v| is the square of 2^(-|v| log2(e) / 2): the instruction's flush of
// subnormal results is out of reach, the square may be subnormal, and the error,
// |v| + 5 ulp of fp32, is far below their half step.
template <typename TY>
__device__ __forceinline__ float gn_silu(float v) {
    float e, r;
    if (sizeof(TY) == 4) {
        e = expf(-fabsf(v));
        return __fdividef(v < 0.f ? v * e : v, 1.f + e);
    }
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(v) * -0.72134752f));
    e *= e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return (v < 0.f ? v * e : v) * r;
}

// act(((x - hi) - lo) * a + beta) of VEC channels.
template <typename TX, typename TY, int VEC, int SUB>
struct Affine {
    float hi[VEC / SUB], lo[VEC / SUB], a[VEC], beta[VEC];
    __device__ __forceinline__ void weights(const GnParams& P, int c0) {
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            a[i] = P.gamma ? P.gamma[c0 + i] : 1.f;
            beta[i] = P.beta ? P.beta[c0 + i] : 0.f;
        }
    }
    __device__ __forceinline__ void stats(int i, float4 st) {       // run i
        hi[i] = st.x;
        lo[i] = st.y;
        #pragma unroll
        for (int j = i * SUB; j < (i + 1) * SUB; j++) a[j] *= st.z;
    }
    template <bool SILU>
    __device__ __forceinline__ Vec<TY, VEC> run(const Vec<TX, VEC>& u) const {
        Vec<TY, VEC> o;
        #pragma unroll
        for (int i = 0; i < VEC; i++) {
            float v = fmaf((Cvt<TX>::to_f(u.v[i]) - hi[i / SUB]) - lo[i / SUB], a[i], beta[i]);
            if (SILU) v = gn_silu<TY>(v);
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
    __shared__ float3 sm[THREADS * N];
    __shared__ float4 mine[CHIP_GROUPS];         // this CTA's moments of the slab's groups
    __shared__ float4 stat[CHIP_GROUPS];
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
    if (on) {
        f.weights(P, c0 + tc * VEC);
        const TX* p = base + (size_t)(r0 + tr) * P.ldx + tc * VEC;
        const size_t step = (size_t)rp * P.ldx;
        #pragma unroll
        for (int k = 0; k < RV; k++)
            if (k < n) u[k] = *reinterpret_cast<const VX*>(p + k * step);
        const float count = (float)(n * SUB), inv = n ? 1.f / count : 0.f;
        #pragma unroll
        for (int i = 0; i < N; i++) {
            Moments m = {0.f, 0.f, 0.f, 0.f};
            if (n)
                m = batch_moments(count, inv, Cvt<TX>::to_f(u[0].v[i * SUB]), [&](auto take) {
                    #pragma unroll
                    for (int k = 0; k < RV; k++)
                        if (k < n) {
                            #pragma unroll
                            for (int c = 0; c < SUB; c++) take(Cvt<TX>::to_f(u[k].v[i * SUB + c]));
                        }
                });
            sm[tr * width + tc * N + i] = make_float3(m.hi, m.lo, m.m2);
        }
    }
    __syncthreads();
    join_groups<SUB>(sm, width, rp, 0, P.cpg, [&](int k) { return k < len ? (len - k + rp - 1) / rp : 0; },
                     [&](int g, Moments m) { mine[g] = make_float4(m.n, m.hi, m.lo, m.m2); });
    if (P.split > 1) sm100::cluster_sync();
    else __syncthreads();
    // a warp a group, a lane a rank: the ranks' moments arrive together
    for (int g = threadIdx.x >> 5; g < groups; g += THREADS / 32) {
        const int r = threadIdx.x & 31;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < P.split) v = P.split > 1 ? sm100::ld_cluster_f32x4(sm100::map_to_rank(&mine[g], r)) : mine[g];
        const Moments a = shfl_join({v.x, v.y, v.z, v.w}, 8);      // up to eight ranks
        if (r == 0) stat[g] = finish(a, P.eps);
    }
    // every rank has read the others' moments: shared memory may go away
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
int launch_chip(const GnParams& P, int batch, int rv, cudaStream_t s) {
    return launch_chained(rv == 4 ? k_gn_chip<TX, TY, VEC, SUB, 4> : k_gn_chip<TX, TY, VEC, SUB, 16>,
                          dim3((unsigned)((long)batch * P.slabs * P.split)), THREADS, 0, P.split, s, P);
}

template <typename TX, typename TY, int VEC, int SUB>
int launch_v(const GroupNormArgs& a, GnParams& P, cudaStream_t s) {
    int rv;
    if (plan_chip(a, VEC, sizeof(TX), P, rv)) return launch_chip<TX, TY, VEC, SUB>(P, a.batch, rv, s);
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
    int n = launch_chained(k_gn_stats<TX, VEC, SUB>, g, THREADS, 0, 0, s, P);
    if (n > 0) n = launch_chained(k_gn_join, dim3(P.G, a.batch), 128, 0, 0, s, P);
    if (n > 0) n = launch_chained(k_gn_apply<TX, TY, VEC, SUB>, ga, THREADS, 0, 0, s, P);
    return n > 0 ? 3 : n;
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
