// k_fp8_quant.cu -- 8-bit codes (e4m3) with one scale for each block of 128
// columns x 1 row (activations) or x 128 rows (weights).
//
//   s = 2^k, k the smallest >= -126 with amax <= 448 * 2^k (amax the block's
//   largest finite |x|); code = e4m3(x / s), round to nearest even.
//
// A power of two loses no relative precision in a floating-point code (the
// block's largest value lands in (224, 448]) and makes x / s exact, so the
// only rounding is the one to e4m3: the codes equal the definition's bit for
// bit.  NaN and infinities become the code's NaN; they take no part in amax.
//
// Bound by HBM: e + 1 bytes per element.  A lane holds 32 bytes of a row, one
// 256-bit load (16 elements of a 16-bit type, 8 of fp32), so 8 or 16 lanes hold
// a block's row; the maximum of |x| is taken on the bit patterns (ordered like
// the values), two 16-bit elements at a time.
#include "kcommon.cuh"
#include "launch.cuh"
#include "ops.h"

namespace s2b {
namespace {

constexpr int WORDS = 8;               // 32-bit words a lane holds of a row

template <typename T> struct Bits;      // bit patterns of a lane's elements, packed
template <> struct Bits<float> {
    static constexpr int E = 8;         // elements a lane
    static constexpr uint32_t INF = 0x7F800000u;
    static __device__ __forceinline__ uint32_t mag(uint32_t w) { return w & 0x7FFFFFFFu; }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t fold(uint32_t w) { return w; }
    static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
    static __device__ __forceinline__ uint32_t finite(uint32_t m) { return m < INF ? m : 0u; }
    // the two elements 2 i and 2 i + 1
    static __device__ __forceinline__ float2 pair(const uint32_t w[WORDS], int i) {
        return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    }
};
template <typename H, uint32_t INF16> struct Bits16 {
    static constexpr int E = 16;
    static constexpr uint32_t INF = INF16;
    static __device__ __forceinline__ uint32_t mag(uint32_t w) { return w & 0x7FFF7FFFu; }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t fold(uint32_t w) { return max(w & 0xFFFFu, w >> 16); }
    static __device__ __forceinline__ uint32_t finite(uint32_t m) {
        return ((m & 0xFFFFu) < INF ? m & 0xFFFFu : 0u) | ((m >> 16) < INF ? m & 0xFFFF0000u : 0u);
    }
};
template <> struct Bits<bf16> : Bits16<bf16, 0x7F80u> {
    static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m << 16); }
    static __device__ __forceinline__ float2 pair(const uint32_t w[WORDS], int i) {
        return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
    }
};
template <> struct Bits<f16> : Bits16<f16, 0x7C00u> {
    static __device__ __forceinline__ float value(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)m)); }
    static __device__ __forceinline__ float2 pair(const uint32_t w[WORDS], int i) {
        return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
};

// Biased exponent of the scale 2^k of a block whose largest finite |x| is
// amax = 1.m * 2^E: k = E - 8 when 1.m <= 1.75 (448 = 1.75 * 2^8), else E - 7.
__device__ __forceinline__ uint32_t scale_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 8 + ((u & 0x7FFFFFu) > 0x600000u);
    return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float pow2_biased(uint32_t e) { return __uint_as_float(e << 23); }

// e4m3 codes of (lo, hi), lo in the low byte; both at most 448 or NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// A lane's elements from column c of a row (n of the row are left; what lies
// past them reads 0).
template <typename T, bool VEC>
__device__ __forceinline__ void load_lane(const T* row, long c, long n, uint32_t w[WORDS]) {
    constexpr int E = Bits<T>::E;
    if (VEC && n >= E) {
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(row + c));
        return;
    }
    #pragma unroll
    for (int i = 0; i < WORDS; i++) w[i] = 0;
    #pragma unroll
    for (int i = 0; i < E; i++) {
        if (i >= n) break;
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(((const float*)row)[c + i]);
        else w[i / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(row)[c + i] << (16 * (i & 1));
    }
}

template <typename T>
__device__ __forceinline__ uint32_t mag_max(const uint32_t w[WORDS]) {
    uint32_t m = Bits<T>::mag(w[0]);
    #pragma unroll
    for (int i = 1; i < WORDS; i++) m = Bits<T>::max2(m, Bits<T>::mag(w[i]));
    return Bits<T>::fold(m);
}
// The same over the finite elements (rare: out of line).
template <typename T>
__device__ __noinline__ uint32_t mag_max_finite(uint4 a, uint4 b) {
    const uint32_t w[WORDS] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    uint32_t m = 0;
    for (int i = 0; i < WORDS; i++) m = Bits<T>::max2(m, Bits<T>::finite(Bits<T>::mag(w[i])));
    return Bits<T>::fold(m);
}

// Codes of a lane's elements times inv (a power of two).  `odd`: the block
// holds NaN or infinities, which become the code's NaN.
template <typename T>
__device__ __forceinline__ void store_lane(uint8_t* dst, const uint32_t w[WORDS], float inv, long n, bool odd) {
    constexpr int E = Bits<T>::E;
    uint32_t o[E / 4];
    #pragma unroll
    for (int i = 0; i < E / 4; i++) {
        float2 a = Bits<T>::pair(w, 2 * i), b = Bits<T>::pair(w, 2 * i + 1);
        const float nan = __uint_as_float(0x7FFFFFFFu);
        if (odd) {
            if (!(fabsf(a.x) < INFINITY)) a.x = nan;
            if (!(fabsf(a.y) < INFINITY)) a.y = nan;
            if (!(fabsf(b.x) < INFINITY)) b.x = nan;
            if (!(fabsf(b.y) < INFINITY)) b.y = nan;
        }
        o[i] = e4m3x2(__fmul_rn(a.x, inv), __fmul_rn(a.y, inv)) | e4m3x2(__fmul_rn(b.x, inv), __fmul_rn(b.y, inv)) << 16;
    }
    if (n >= E) {
        if constexpr (E == 16) *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    } else {
        #pragma unroll
        for (int i = 0; i < E; i++)
            if (i < n) dst[i] = (uint8_t)(o[i / 4] >> (8 * (i & 3)));
    }
}

// Largest of the LANES lanes that share a block's row.
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t m) {
    #pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Rows: a CTA takes 32 rows x 512 columns, a lane group (8 lanes of a 16-bit
// type, 16 of fp32) four blocks of one or two rows: four 256-bit loads in flight
// a lane.  Scales go out as 32 consecutive rows of one column block.  B200, bf16
// 5498 x 6912 (115 MB): 21.7 us, 5.3 TB/s.
constexpr int QR_ROWS = 32, QR_BLKS = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 3) k_fp8_quant_rows(const T* x, int rows, int cols, int ldx,
                                                           uint8_t* q, int ldq, float* scale) {
    constexpr int LANES = 128 / Bits<T>::E, GROUPS = 256 / LANES;
    __shared__ float ss[QR_BLKS][QR_ROWS];
    constexpr bool STAGED = !VEC && sizeof(T) == 2;
    __shared__ uint4 sx[STAGED ? 8 : 1][STAGED ? 64 : 1];        // a warp's 32 x 32 bytes
    chain_begin();
    const int grp = threadIdx.x / LANES, l = threadIdx.x % LANES;
    const int kb = cols / 128 + (cols % 128 != 0), across = (kb + QR_BLKS - 1) / QR_BLKS;
    const long r0 = (long)(blockIdx.x / across) * QR_ROWS;
    const int b0 = blockIdx.x % across * QR_BLKS;
    for (int i = grp; i < QR_ROWS; i += GROUPS) {
        const long r = r0 + i;
        if (r0 + i - grp >= rows) break;             // uniform: nothing left for any group
        const long left = r < rows ? cols : 0;
        uint32_t w[QR_BLKS][WORDS];
        if constexpr (!STAGED) {
            #pragma unroll
            for (int j = 0; j < QR_BLKS; j++) {
                const long c = (b0 + j) * 128L + l * Bits<T>::E;
                load_lane<T, VEC>(x + (size_t)r * ldx, c, left - c, w[j]);
            }
        } else {
            // 16-bit rows that start anywhere: neighbouring lanes load neighbouring
            // elements of the warp's rows, a block ahead, and take their 32 bytes
            // from shared memory (5498 x 6910: 66 us lane by lane, 33 so; fp32
            // rows, half as many loads, take 25 us lane by lane and 62 so)
            constexpr int PER = 32 / LANES * 4;      // a lane's elements of the warp's rows of a block
            uint4* mine = sx[threadIdx.x >> 5];
            T* buf = reinterpret_cast<T*>(mine);
            const int lane = threadIdx.x & 31;
            const long rw = r0 + i - grp + (threadIdx.x >> 5) * (32 / LANES);
            T v[PER];
            auto fetch = [&](int j) {
                #pragma unroll
                for (int e = 0; e < PER; e++) {
                    const long row = rw + e / 4, c = (b0 + j) * 128L + e % 4 * 32 + lane;
                    v[e] = row < rows && c < cols ? x[(size_t)row * ldx + c] : T(0.f);
                }
            };
            fetch(0);
            #pragma unroll
            for (int j = 0; j < QR_BLKS; j++) {
                __syncwarp();
                #pragma unroll
                for (int e = 0; e < PER; e++) buf[e * 32 + lane] = v[e];
                if (j + 1 < QR_BLKS) fetch(j + 1);
                __syncwarp();
                const uint4 a = mine[2 * lane], b = mine[2 * lane + 1];
                w[j][0] = a.x; w[j][1] = a.y; w[j][2] = a.z; w[j][3] = a.w;
                w[j][4] = b.x; w[j][5] = b.y; w[j][6] = b.z; w[j][7] = b.w;
            }
        }
        #pragma unroll
        for (int j = 0; j < QR_BLKS; j++) {
            const long c = (b0 + j) * 128L + l * Bits<T>::E;
            uint32_t m = lanes_max<LANES>(mag_max<T>(w[j]));
            const bool odd = __any_sync(0xffffffffu, m >= Bits<T>::INF);
            if (odd)                                 // rare: NaN or infinity in one of the warp's blocks
                m = lanes_max<LANES>(mag_max_finite<T>(make_uint4(w[j][0], w[j][1], w[j][2], w[j][3]),
                                                       make_uint4(w[j][4], w[j][5], w[j][6], w[j][7])));
            const uint32_t e = scale_exp(Bits<T>::value(m));
            if (c < left) store_lane<T>(q + (size_t)r * ldq + c, w[j], pow2_biased(254 - e), left - c, odd);
            if (l == 0) ss[j][i] = pow2_biased(e);
        }
    }
    __syncthreads();
    if (threadIdx.x < QR_BLKS * QR_ROWS) {
        const int j = threadIdx.x / QR_ROWS, r = threadIdx.x % QR_ROWS;
        if (b0 + j < kb && r0 + r < rows) scale[(size_t)(b0 + j) * rows + r0 + r] = ss[j][r];
    }
}

// Weights: a CTA takes one 128 x 128 block, held in registers between the
// maximum and the codes.  B200, fp32 7680 x 2560 (98 MB): 20.3 us, 4.8 TB/s.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256, 2) k_fp8_quant_blocks(const T* x, int rows, int cols, int ldx,
                                                             uint8_t* q, int ldq, float* scale) {
    constexpr int LANES = 128 / Bits<T>::E, GROUPS = 256 / LANES, PER = 128 / GROUPS;     // rows a lane
    __shared__ uint32_t sm[8], sf[8];
    chain_begin();
    const int grp = threadIdx.x / LANES, l = threadIdx.x % LANES, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kb = cols / 128 + (cols % 128 != 0);
    const long c = blockIdx.x % kb * 128L + l * Bits<T>::E, rb = blockIdx.x / kb;
    uint32_t w[PER][WORDS];
    uint32_t m = 0, f = 0;
    #pragma unroll
    for (int i = 0; i < PER; i++) {
        const long r = rb * 128 + grp + GROUPS * i;
        load_lane<T, VEC>(x + (size_t)r * ldx, c, r < rows ? cols - c : 0, w[i]);
    }
    #pragma unroll
    for (int i = 0; i < PER; i++) m = max(m, mag_max<T>(w[i]));
    m = lanes_max<32>(m);
    const bool warp_odd = m >= Bits<T>::INF;
    f = m;
    if (warp_odd) {                                  // rare, and the same for the whole warp
        f = 0;
        #pragma unroll
        for (int i = 0; i < PER; i++)
            f = max(f, mag_max_finite<T>(make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]), make_uint4(w[i][4], w[i][5], w[i][6], w[i][7])));
        f = lanes_max<32>(f);
    }
    if (lane == 0) { sm[warp] = warp_odd; sf[warp] = f; }
    __syncthreads();
    uint32_t top = 0, any = 0;
    #pragma unroll
    for (int i = 0; i < 8; i++) { top = max(top, sf[i]); any |= sm[i]; }
    const uint32_t e = scale_exp(Bits<T>::value(top));
    if (threadIdx.x == 0) scale[blockIdx.x] = pow2_biased(e);
    #pragma unroll
    for (int i = 0; i < PER; i++) {
        const long r = rb * 128 + grp + GROUPS * i;
        if (r < rows && c < cols) store_lane<T>(q + (size_t)r * ldq + c, w[i], pow2_biased(254 - e), cols - c, any != 0);
    }
}

template <typename T>
int launch(const Fp8QuantArgs& a, cudaStream_t s) {
    const T* x = (const T*)a.x;
    uint8_t* q = (uint8_t*)a.q;
    // 256-bit loads where every row starts on 32 bytes, single elements elsewhere
    const bool vec = ((uintptr_t)a.x & 31) == 0 && ((size_t)a.ldx * sizeof(T)) % 32 == 0;
    const long kb = (a.cols + 127L) / 128;
    if (a.block_rows == 1) {
        const long g = ((kb + QR_BLKS - 1) / QR_BLKS) * ((a.rows + QR_ROWS - 1L) / QR_ROWS);
        if (g > 2147483647L) return -1;
        return launch_chained(vec ? k_fp8_quant_rows<T, true> : k_fp8_quant_rows<T, false>, dim3((unsigned)g), 256, 0, 0, s, x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
    }
    const long g = kb * ((a.rows + 127L) / 128);
    if (g > 2147483647L) return -1;
    return launch_chained(vec ? k_fp8_quant_blocks<T, true> : k_fp8_quant_blocks<T, false>, dim3((unsigned)g), 256, 0, 0, s, x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
}

}  // namespace

int op_launch(const Fp8QuantArgs& a, cudaStream_t s) {
    switch (a.x_type) {
        case S2B_PREC_FP32: return launch<float>(a, s);
        case S2B_PREC_FP16: return launch<f16>(a, s);
        default: return launch<bf16>(a, s);
    }
}

}  // namespace s2b
