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
// Bound by HBM: e + 1 bytes per element.  Half a warp holds one 128-column
// row segment, 8 elements a lane in one or two 16-byte loads; the maximum of
// |x| is taken on the bit patterns (ordered like the values), two 16-bit
// elements at a time.
#include "kcommon.cuh"
#include "ops.h"

namespace s2b {
namespace {

template <typename T> struct Bits;      // patterns of 8 elements, as packed 32-bit words
template <> struct Bits<float> {
    static constexpr int WORDS = 8;
    static constexpr uint32_t INF = 0x7F800000u;
    static __device__ __forceinline__ uint32_t mag(uint32_t w) { return w & 0x7FFFFFFFu; }
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) { return max(a, b); }
    static __device__ __forceinline__ uint32_t fold(uint32_t w) { return w; }
    static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
    static __device__ __forceinline__ uint32_t finite(uint32_t m) { return m < INF ? m : 0u; }
    static __device__ __forceinline__ void floats(const uint32_t w[8], float v[8]) {
        #pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i]);
    }
};
template <typename H, uint32_t INF16> struct Bits16 {
    static constexpr int WORDS = 4;
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
    static __device__ __forceinline__ void floats(const uint32_t w[4], float v[8]) {
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <> struct Bits<f16> : Bits16<f16, 0x7C00u> {
    static __device__ __forceinline__ float value(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)m)); }
    static __device__ __forceinline__ void floats(const uint32_t w[4], float v[8]) {
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x; v[2 * i + 1] = f.y;
        }
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

// 8 elements from column c of a row (n of them inside it; the rest read 0).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, long c, long n, uint32_t w[Bits<T>::WORDS]) {
    #pragma unroll
    for (int i = 0; i < Bits<T>::WORDS; i++) w[i] = 0;
    if (n <= 0) return;
    if (VEC && n >= 8) {
        #pragma unroll
        for (int i = 0; i < Bits<T>::WORDS / 4; i++) {
            const uint4 t = __ldcs(reinterpret_cast<const uint4*>(row + c) + i);
            w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
        }
        return;
    }
    #pragma unroll
    for (int i = 0; i < 8; i++) {
        if (i >= n) break;
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(((const float*)row)[c + i]);
        else w[i / 2] |= (uint32_t)reinterpret_cast<const unsigned short*>(row)[c + i] << (16 * (i & 1));
    }
}

template <typename T>
__device__ __forceinline__ uint32_t mag_max(const uint32_t w[Bits<T>::WORDS], bool finite_only) {
    uint32_t m = 0;
    #pragma unroll
    for (int i = 0; i < Bits<T>::WORDS; i++) {
        uint32_t a = Bits<T>::mag(w[i]);
        if (finite_only) a = Bits<T>::finite(a);
        m = Bits<T>::max2(m, a);
    }
    return Bits<T>::fold(m);
}

// Codes of 8 elements times inv (a power of two), n of them inside the row.
// `odd`: the block holds NaN or infinities, which become the code's NaN.
template <typename T>
__device__ __forceinline__ void store8(uint8_t* dst, const uint32_t w[Bits<T>::WORDS], float inv, long n, bool odd) {
    float v[8];
    Bits<T>::floats(w, v);
    #pragma unroll
    for (int i = 0; i < 8; i++) {
        if (odd && !(fabsf(v[i]) < INFINITY)) v[i] = __uint_as_float(0x7FFFFFFFu);
        else v[i] = __fmul_rn(v[i], inv);
    }
    const uint32_t lo = e4m3x2(v[0], v[1]) | e4m3x2(v[2], v[3]) << 16;
    const uint32_t hi = e4m3x2(v[4], v[5]) | e4m3x2(v[6], v[7]) << 16;
    if (n >= 8) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    } else {
        #pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) dst[i] = (uint8_t)((i < 4 ? lo >> (8 * i) : hi >> (8 * (i - 4))) & 0xFFu);
    }
}

// Rows: a CTA takes 32 rows x 512 columns; half-warp h rows h and h + 16,
// four blocks each (eight 16-byte loads in flight a lane for 16-bit x).
// Scales go out as 32 consecutive rows of one column block.
constexpr int QR_ROWS = 32, QR_BLKS = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_fp8_quant_rows(const T* __restrict__ x, int rows, int cols, int ldx,
                                                        uint8_t* __restrict__ q, int ldq, float* __restrict__ scale) {
    __shared__ float ss[QR_BLKS][QR_ROWS];
    const int hw = threadIdx.x >> 4, l = threadIdx.x & 15;
    const int kb = cols / 128 + (cols % 128 != 0), across = (kb + QR_BLKS - 1) / QR_BLKS;
    const long r0 = (long)(blockIdx.x / across) * QR_ROWS;
    const int b0 = blockIdx.x % across * QR_BLKS;
    uint32_t w[2][QR_BLKS][Bits<T>::WORDS];
    #pragma unroll
    for (int i = 0; i < 2; i++) {
        const long r = r0 + hw + 16 * i;
        #pragma unroll
        for (int j = 0; j < QR_BLKS; j++) {
            const long c = (b0 + j) * 128L + l * 8;
            load8<T, VEC>(x + (size_t)r * ldx, c, r < rows ? cols - c : 0, w[i][j]);
        }
    }
    #pragma unroll
    for (int i = 0; i < 2; i++) {
        const long r = r0 + hw + 16 * i;
        #pragma unroll
        for (int j = 0; j < QR_BLKS; j++) {
            const long c = (b0 + j) * 128L + l * 8;
            uint32_t m = mag_max<T>(w[i][j], false);
            #pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const bool odd = __any_sync(0xffffffffu, m >= Bits<T>::INF);
            if (odd) {                               // rare: NaN or infinity in either half-warp's block
                m = mag_max<T>(w[i][j], true);
                #pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            }
            const uint32_t e = scale_exp(Bits<T>::value(m));
            if (r < rows && c < cols) store8<T>(q + (size_t)r * ldq + c, w[i][j], pow2_biased(254 - e), cols - c, odd);
            if (l == 0) ss[j][hw + 16 * i] = pow2_biased(e);
        }
    }
    __syncthreads();
    if (threadIdx.x < QR_BLKS * QR_ROWS) {
        const int j = threadIdx.x / QR_ROWS, r = threadIdx.x % QR_ROWS;
        if (b0 + j < kb && r0 + r < rows) scale[(size_t)(b0 + j) * rows + r0 + r] = ss[j][r];
    }
}

// Weights: a CTA takes one 128 x 128 block, eight rows a half-warp, held in
// registers between the maximum and the codes.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) k_fp8_quant_blocks(const T* __restrict__ x, int rows, int cols, int ldx,
                                                          uint8_t* __restrict__ q, int ldq, float* __restrict__ scale) {
    __shared__ uint32_t sm[8], sf[8];
    const int hw = threadIdx.x >> 4, l = threadIdx.x & 15, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kb = cols / 128 + (cols % 128 != 0);
    const long c = blockIdx.x % kb * 128L + l * 8, rb = blockIdx.x / kb;
    uint32_t w[8][Bits<T>::WORDS];
    uint32_t m = 0, f = 0;
    #pragma unroll
    for (int i = 0; i < 8; i++) {
        const long r = rb * 128 + hw + 16 * i;
        load8<T, VEC>(x + (size_t)r * ldx, c, r < rows ? cols - c : 0, w[i]);
    }
    #pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, mag_max<T>(w[i], false));
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool warp_odd = m >= Bits<T>::INF;
    f = m;
    if (warp_odd) {                                  // rare, and the same for the whole warp
        f = 0;
        #pragma unroll
        for (int i = 0; i < 8; i++) f = max(f, mag_max<T>(w[i], true));
        #pragma unroll
        for (int o = 16; o > 0; o >>= 1) f = max(f, __shfl_xor_sync(0xffffffffu, f, o));
    }
    if (lane == 0) { sm[warp] = warp_odd; sf[warp] = f; }
    __syncthreads();
    uint32_t top = 0, any = 0;
    #pragma unroll
    for (int i = 0; i < 8; i++) { top = max(top, sf[i]); any |= sm[i]; }
    const uint32_t e = scale_exp(Bits<T>::value(top));
    if (threadIdx.x == 0) scale[blockIdx.x] = pow2_biased(e);
    #pragma unroll
    for (int i = 0; i < 8; i++) {
        const long r = rb * 128 + hw + 16 * i;
        if (r < rows && c < cols) store8<T>(q + (size_t)r * ldq + c, w[i], pow2_biased(254 - e), cols - c, any != 0);
    }
}

template <typename T>
int launch(const Fp8QuantArgs& a, cudaStream_t s) {
    const T* x = (const T*)a.x;
    uint8_t* q = (uint8_t*)a.q;
    const bool vec = ((uintptr_t)a.x & 15) == 0 && ((size_t)a.ldx * sizeof(T)) % 16 == 0;
    const long kb = (a.cols + 127L) / 128;
    if (a.block_rows == 1) {
        const long g = ((kb + QR_BLKS - 1) / QR_BLKS) * ((a.rows + QR_ROWS - 1L) / QR_ROWS);
        if (g > 2147483647L) return -1;
        if (vec) k_fp8_quant_rows<T, true><<<(unsigned)g, 256, 0, s>>>(x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
        else k_fp8_quant_rows<T, false><<<(unsigned)g, 256, 0, s>>>(x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
        return 1;
    }
    const long g = kb * ((a.rows + 127L) / 128);
    if (g > 2147483647L) return -1;
    if (vec) k_fp8_quant_blocks<T, true><<<(unsigned)g, 256, 0, s>>>(x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
    else k_fp8_quant_blocks<T, false><<<(unsigned)g, 256, 0, s>>>(x, a.rows, a.cols, a.ldx, q, a.ldq, a.scale);
    return 1;
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
