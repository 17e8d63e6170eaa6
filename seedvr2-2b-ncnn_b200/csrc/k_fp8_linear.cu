// k_fp8_linear.cu -- y = sum_b xs[b, m] ws[n / 128, b] (xq . wq over block b) + bias
// on the tcgen05 tensor cores (kind::f8f6f4, e4m3 codes), blocks of 128 along K.
//
// The scales change with every block of K, so a block's products cannot stay
// in the accumulator: each block's fp32 sum (4 MMAs of 32 codes) goes to one
// of two TMEM slots, and the epilogue warps read it and add scale * sum to
// fp32 registers while the tensor core works on the next block.  Scales are
// any fp32 values; sums and scale products are fp32, rounded once to y's type.
#include "kcommon.cuh"
#include "ops.h"
#include "sm100.cuh"
#include <atomic>
#include <cuda.h>

namespace s2b {

// encoder of tensor maps over bytes (k_gemm_tc.cu)
bool make_tmap_u8(CUtensorMap* m, const void* base, int rows, int cols, int ld, int box_rows);
bool make_tmap_out(CUtensorMap* m, void* base, int type, int rows, int cols, int ld);
int gemm_tc_flag_ptr(int** p);

namespace {

constexpr int KB = 128;                  // K elements of a block (and bytes of a swizzled row)

struct LinParams {
    const float *xs, *ws, *bias;
    void* y;
    int M, N, nkb, ldy, y_type;
    int* flag;                           // the GEMM class's device error flag
};

// Bounded wait; on expiry raises the CTA's abort flag and the device flag.
__device__ __forceinline__ bool wait_flag(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* flag) {
    for (uint32_t i = 0; i < sm100::WAIT_LIMIT; i++) {
        if (sm100::mbar_try_wait(bar, parity)) return true;
        if ((i & 1023) == 1023 && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(flag, 1);
    return false;
}

__device__ __forceinline__ void store_y(void* y, int t, size_t i, float v) {
    if (t == S2B_PREC_FP32) ((float*)y)[i] = v;
    else if (t == S2B_PREC_FP16) ((f16*)y)[i] = __float2half_rn(v);
    else ((bf16*)y)[i] = __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------- few rows
// Weights as the MMA's 128-row operand and BT tokens as its N: one token
// fills 1/16 of an MMA instead of 1/128.  A cluster of `split` CTAs divides K
// and joins its sums through shared memory in rank order (no atomics, no
// workspace), so that few tiles still stream the weights from every SM.
template <int BT> struct NarrowCfg {
    static constexpr int W_BYTES = 128 * KB, X_BYTES = BT * KB, STAGE = W_BYTES + X_BYTES;
    static constexpr int STAGES = BT == 64 ? 4 : 5;
    static constexpr int COLS = BT == 16 ? 32 : 2 * BT;          // TMEM: two slots of BT columns
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256 + 4 * 2 * BT * 4;
    static_assert(128 * BT * 4 <= STAGES * STAGE, "the joined sums reuse the stages");
};
template <int STAGES> struct NarrowCtl {
    uint64_t full[STAGES], done[STAGES], tempty[2];
    uint32_t tmem_slot;
    int abort;
};

template <int BT>
__global__ void __launch_bounds__(192) k_fp8_linear_narrow(const __grid_constant__ CUtensorMap mw,
                                                           const __grid_constant__ CUtensorMap mx,
                                                           const __grid_constant__ LinParams P, int split) {
    using C = NarrowCfg<BT>;
    constexpr int ST = C::STAGES;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    NarrowCtl<ST>* ctl = reinterpret_cast<NarrowCtl<ST>*>(smem + ST * C::STAGE);
    float* sc = reinterpret_cast<float*>(smem + ST * C::STAGE + 256);    // [4 warps][2][BT]
    static_assert(sizeof(NarrowCtl<ST>) <= 256, "control block");
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)sm100::cluster_ctarank() : 0;
    const int tile = blockIdx.x / split;
    const int ntn = (P.N + 127) / 128;
    const int nb = tile % ntn, n0 = nb * 128, m0 = tile / ntn * BT;
    const int kb0 = (int)((long)P.nkb * rank / split), kb1 = (int)((long)P.nkb * (rank + 1) / split);

    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) { sm100::mbar_init(&ctl->full[s], 1); sm100::mbar_init(&ctl->done[s], 1); }
        sm100::mbar_init(&ctl->tempty[0], 4);
        sm100::mbar_init(&ctl->tempty[1], 4);
        ctl->abort = 0;
        sm100::fence_barrier_init();
        sm100::tma_prefetch_desc(&mw);
        sm100::tma_prefetch_desc(&mx);
    }
    if (warp == 1) {
        sm100::tmem_alloc(&ctl->tmem_slot, C::COLS);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = ctl->tmem_slot;
    float acc[BT];
    #pragma unroll
    for (int c = 0; c < BT; c++) acc[c] = 0.f;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            long issued = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!wait_flag(&ctl->done[s], ph ^ 1, abort_flag, P.flag)) break;
                uint8_t* st = smem + s * C::STAGE;
                sm100::mbar_arrive_expect_tx(&ctl->full[s], C::STAGE);
                sm100::tma_load_2d(st, &mw, &ctl->full[s], kb * KB, n0);
                sm100::tma_load_2d(st + C::W_BYTES, &mx, &ctl->full[s], kb * KB, m0);
                issued++;
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            // every load has landed before shared memory is used otherwise
            for (long i = 1; i <= ST && i <= issued; i++) {
                const long k = issued - i;
                for (uint32_t w = 0; w < sm100::WAIT_LIMIT && !sm100::mbar_try_wait(&ctl->full[k % ST], (k / ST) & 1); w++) {}
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = sm100::idesc_e4m3_f32(128, BT);
            int s = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                const int i = kb - kb0, slot = i & 1;
                if (!wait_flag(&ctl->tempty[slot], ((i >> 1) & 1) ^ 1, abort_flag, P.flag)) break;
                if (!wait_flag(&ctl->full[s], ph, abort_flag, P.flag)) break;
                sm100::tc_fence_after();
                const uint8_t* st = smem + s * C::STAGE;
                #pragma unroll
                for (int k = 0; k < 4; k++)
                    sm100::mma_f8(tmem + slot * BT, sm100::desc_kmajor_sw128(st, k * 32),
                                  sm100::desc_kmajor_sw128(st + C::W_BYTES, k * 32), idesc, k != 0);
                sm100::mma_commit(&ctl->done[s]);
                if (++s == ST) { s = 0; ph ^= 1; }
            }
        }
    } else {
        const int q = warp & 3;
        float* my = sc + (warp - 2) * 2 * BT;
        const float* wrow = P.ws + (size_t)nb * P.nkb;
        // scale products of a block: lane l holds tokens l and l + 32
        auto fetch = [&](int kb, float v[2]) {
            v[0] = v[1] = 0.f;
            if (kb >= kb1) return;
            const float w = __ldg(wrow + kb);
            #pragma unroll
            for (int j = 0; j < (BT + 31) / 32; j++) {
                const int c = lane + 32 * j;
                if (c < BT && m0 + c < P.M) v[j] = w * __ldg(P.xs + (size_t)kb * P.M + m0 + c);
            }
        };
        float v[2], vn[2];
        fetch(kb0, v);
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            const int slot = (kb - kb0) & 1;
            float* sb = my + slot * BT;
            #pragma unroll
            for (int j = 0; j < (BT + 31) / 32; j++)
                if (lane + 32 * j < BT) sb[lane + 32 * j] = v[j];
            fetch(kb + 1, vn);
            __syncwarp();
            if (!__all_sync(0xffffffffu, wait_flag(&ctl->done[s], ph, abort_flag, P.flag))) break;
            sm100::tc_fence_after();
            #pragma unroll
            for (int c0 = 0; c0 < BT; c0 += 16) {
                float d[16];
                sm100::tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + slot * BT + c0, d);
                #pragma unroll
                for (int c = 0; c < 16; c += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(sb + c0 + c);
                    acc[c0 + c] = fmaf(d[c], f.x, acc[c0 + c]);
                    acc[c0 + c + 1] = fmaf(d[c + 1], f.y, acc[c0 + c + 1]);
                    acc[c0 + c + 2] = fmaf(d[c + 2], f.z, acc[c0 + c + 2]);
                    acc[c0 + c + 3] = fmaf(d[c + 3], f.w, acc[c0 + c + 3]);
                }
            }
            sm100::tc_fence_before();
            __syncwarp();
            if (lane == 0) sm100::mbar_arrive(&ctl->tempty[slot]);
            v[0] = vn[0]; v[1] = vn[1];
            if (++s == ST) { s = 0; ph ^= 1; }
        }
    }
    __syncwarp();
    __syncthreads();                     // every MMA and load of this CTA is done: the stages are free
    const bool epi = warp >= 2;
    const int nl = (warp & 3) * 32 + lane, n = n0 + nl;
    if (split == 1) {
        if (epi && n < P.N) {
            const float b = P.bias ? __ldg(P.bias + n) : 0.f;
            #pragma unroll
            for (int c = 0; c < BT; c++)
                if (m0 + c < P.M) store_y(P.y, P.y_type, (size_t)(m0 + c) * P.ldy + n, acc[c] + b);
        }
    } else {
        float* red = reinterpret_cast<float*>(smem);             // [BT][128]
        if (epi) {
            #pragma unroll
            for (int c = 0; c < BT; c++) red[c * 128 + nl] = acc[c];
        }
        sm100::cluster_sync();
        if (epi && n < P.N) {
            const float b = P.bias ? __ldg(P.bias + n) : 0.f;
            for (int c = rank; c < BT; c += split) {
                if (m0 + c >= P.M) break;
                float t = 0.f;
                for (int r = 0; r < split; r++) t += sm100::ld_cluster_f32(sm100::map_to_rank(red + c * 128 + nl, r));
                store_y(P.y, P.y_type, (size_t)(m0 + c) * P.ldy + n, t + b);
            }
        }
        sm100::cluster_sync();           // no CTA leaves while another reads its sums
    }
    if (warp == 1) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem, C::COLS);
    }
}

// Device address of the GEMM class's error flag, looked up once a device.
int* device_flag() {
    static std::atomic<int*> at[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return nullptr;
    int* p = at[dev].load(std::memory_order_relaxed);
    if (!p) {
        if (gemm_tc_flag_ptr(&p)) return nullptr;
        at[dev].store(p, std::memory_order_relaxed);
    }
    return p;
}

template <int BT>
int launch_narrow(const Fp8LinearArgs& a, const LinParams& P, cudaStream_t s) {
    using C = NarrowCfg<BT>;
    CUtensorMap mw, mx;
    if (!make_tmap_u8(&mw, a.wq, a.N, a.K, a.ldw, 128) || !make_tmap_u8(&mx, a.xq, a.M, a.K, a.ldx, BT)) return -1;
    const long tiles = ((a.N + 127L) / 128) * ((a.M + BT - 1L) / BT);
    // ranks along K: as many as two CTAs an SM hold, each with two blocks or more
    int split = 1;
    while (split < 8 && tiles * split * 2 <= 2L * op_sms() && P.nkb >= 4 * split) split *= 2;
    if (tiles * split > 2147483647L) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * split));
    cfg.blockDim = dim3(192);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = split; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, k_fp8_linear_narrow<BT>, mw, mx, P, split) != cudaSuccess) return -1;
    return 1;
}

// ---------------------------------------------------------------- many rows
// Persistent CTA pairs (cta_group::2), 256 x 256 tiles: a CTA holds 128 rows
// of A and 128 of B of every block of K, its 128 x 256 fp32 sums fill one of
// the two TMEM slots.  Warp 0 loads, warp 1 of the even CTA issues the MMAs,
// eight epilogue warps each own 32 rows x 128 columns -- one weight block, so
// a thread's scale is one number a block -- and keep 128 sums in registers.
// The MMAs of a block take 512 cycles of the tensor core; reading the sums
// (256 columns a lane quadrant) and 64 packed FMAs a thread take fewer.
constexpr int PBM = 256, PBN = 256, PSTAGES = 5, PTHREADS = 384;
constexpr int P_TILE = 128 * KB, P_STAGE = 2 * P_TILE, P_BOX = 32 * 128;
constexpr int P_SMEM = PSTAGES * P_STAGE + 8 * 2 * P_BOX + 1024 + 512;
// Register shares: 168 a thread at launch; the epilogue's eight warps take 224
// of the four others' 168 - 56.
constexpr int P_REGS = 168, P_REGS_LOW = 56, P_REGS_HIGH = 224;
static_assert(128 * P_REGS_LOW + 256 * P_REGS_HIGH <= PTHREADS * P_REGS, "register shares exceed the launch's");

struct PairCtl {
    uint64_t full[PSTAGES], done[PSTAGES], tempty[2];
    uint32_t tmem_slot;
    int abort;
};

struct PairTiles {
    int num_m, num_n, total;
    int tma_y;                           // y through TMA boxes (16-byte rows)
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ float lo_f(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_f(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// Two values in y's 16-bit type.
__device__ __forceinline__ uint32_t half2_bits(float a, float b, int t) {
    if (t == S2B_PREC_FP16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Writes 32 rows x 128 columns from (row0, col0): lane = row, acc its columns,
// through this warp's two staging boxes of 32 rows x 128 bytes (128-byte
// swizzle: conflict-free 16-byte stores).  Leaves its TMA stores in flight.
__device__ __forceinline__ void pair_store(const LinParams& P, const PairTiles& T, const CUtensorMap* my, uint8_t* box, int row0,
                                           int col0, uint64_t acc[64]) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) sm100::bulk_wait_read_all();          // the boxes' previous stores
    __syncwarp();
    if (P.bias) {
        float* b = reinterpret_cast<float*>(box);
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = col0 + lane + 32 * j;
            b[lane + 32 * j] = c < P.N ? __ldg(P.bias + c) : 0.f;
        }
        __syncwarp();
        #pragma unroll
        for (int j = 0; j < 32; j++) {
            const float4 f = reinterpret_cast<const float4*>(b)[j];
            acc[2 * j] = pack2(__float_as_uint(lo_f(acc[2 * j]) + f.x), __float_as_uint(hi_f(acc[2 * j]) + f.y));
            acc[2 * j + 1] = pack2(__float_as_uint(lo_f(acc[2 * j + 1]) + f.z), __float_as_uint(hi_f(acc[2 * j + 1]) + f.w));
        }
        __syncwarp();
    }
    const bool wide = P.y_type == S2B_PREC_FP32;
    const int per = wide ? 32 : 64;                      // columns of a box
    #pragma unroll
    for (int pass = 0; pass < 2; pass++) {
        if (pass && !wide) break;
        if (pass) {
            if (lane == 0) sm100::bulk_wait_read_all();
            __syncwarp();
        }
        #pragma unroll
        for (int b = 0; b < 2; b++) {
            #pragma unroll
            for (int j = 0; j < 8; j++) {
                uint4 v;
                if (wide) {
                    const uint64_t *a = acc + pass * 32 + b * 16 + j * 2;
                    v = make_uint4((uint32_t)a[0], (uint32_t)(a[0] >> 32), (uint32_t)a[1], (uint32_t)(a[1] >> 32));
                } else {
                    const uint64_t *a = acc + b * 32 + j * 4;
                    v.x = half2_bits(lo_f(a[0]), hi_f(a[0]), P.y_type);
                    v.y = half2_bits(lo_f(a[1]), hi_f(a[1]), P.y_type);
                    v.z = half2_bits(lo_f(a[2]), hi_f(a[2]), P.y_type);
                    v.w = half2_bits(lo_f(a[3]), hi_f(a[3]), P.y_type);
                }
                *reinterpret_cast<uint4*>(box + b * P_BOX + lane * 128 + ((j ^ (lane & 7)) << 4)) = v;
            }
        }
        const int c0 = col0 + pass * 64;
        if (T.tma_y) {
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                for (int b = 0; b < 2; b++)
                    if (row0 < P.M && c0 + b * per < P.N) sm100::tma_store_2d(my, box + b * P_BOX, c0 + b * per, row0);
                sm100::bulk_commit_group();
            }
        } else {
            __syncwarp();
            const int rows = min(32, P.M - row0), e = wide ? 4 : 2;
            for (int r = 0; r < rows; r++)
                for (int c = lane; c < 2 * per; c += 32) {
                    if (c0 + c >= P.N) break;
                    const int k = c % per * e;           // byte of the box's row
                    const uint8_t* src = box + c / per * P_BOX + r * 128 + (((k >> 4) ^ (r & 7)) << 4) + (k & 15);
                    const size_t at = (size_t)(row0 + r) * P.ldy + c0 + c;
                    if (wide) ((uint32_t*)P.y)[at] = *reinterpret_cast<const uint32_t*>(src);
                    else ((uint16_t*)P.y)[at] = *reinterpret_cast<const uint16_t*>(src);
                }
            __syncwarp();
        }
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PTHREADS, 1)
k_fp8_linear_pair(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw,
                  const __grid_constant__ CUtensorMap my, const __grid_constant__ LinParams P,
                  const __grid_constant__ PairTiles T) {
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* boxes = smem + PSTAGES * P_STAGE;
    PairCtl* ctl = reinterpret_cast<PairCtl*>(boxes + 8 * 2 * P_BOX);
    static_assert(sizeof(PairCtl) <= 512, "control block");
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = sm100::cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < PSTAGES; s++) { sm100::mbar_init(&ctl->full[s], 1); sm100::mbar_init(&ctl->done[s], 1); }
        sm100::mbar_init(&ctl->tempty[0], 16);
        sm100::mbar_init(&ctl->tempty[1], 16);
        ctl->abort = 0;
        sm100::fence_barrier_init();
        sm100::tma_prefetch_desc(&mx);
        sm100::tma_prefetch_desc(&mw);
    }
    if (warp == 1) {
        sm100::tmem_alloc_pair(&ctl->tmem_slot, 512);
        sm100::tmem_relinquish_pair();
    }
    sm100::tc_fence_before();
    sm100::cluster_sync();
    sm100::tc_fence_after();
    const uint32_t tmem = ctl->tmem_slot;

    if (warp < 4) {
        sm100::regs_shrink<P_REGS_LOW>();
        if (warp == 0 && lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            long issued = 0;
            bool ok = true;
            for (int tile = pair; tile < T.total && ok; tile += npairs) {
                const int xr = tile % T.num_m * PBM + (int)rank * 128, wr = tile / T.num_m * PBN + (int)rank * 128;
                for (int kb = 0; kb < P.nkb; kb++) {
                    // both CTAs' MMAs on this stage are done
                    if (!wait_flag(&ctl->done[s], ph ^ 1, abort_flag, P.flag)) { ok = false; break; }
                    if (rank == 0) sm100::mbar_arrive_expect_tx(&ctl->full[s], 2 * P_STAGE);
                    const uint32_t fb = sm100::map_to_rank(&ctl->full[s], 0);
                    sm100::tma_load_2d_pair(smem + s * P_STAGE, &mx, fb, kb * KB, xr);
                    sm100::tma_load_2d_pair(smem + s * P_STAGE + P_TILE, &mw, fb, kb * KB, wr);
                    issued++;
                    if (++s == PSTAGES) { s = 0; ph ^= 1; }
                }
            }
            if (rank == 0)               // every load of the pair has landed (bounded) before anyone leaves
                for (long i = 1; i <= PSTAGES && i <= issued; i++) {
                    const long k = issued - i;
                    for (uint32_t w = 0; w < sm100::WAIT_LIMIT && !sm100::mbar_try_wait(&ctl->full[k % PSTAGES], (k / PSTAGES) & 1); w++) {}
                }
        } else if (warp == 1 && rank == 0) {
            constexpr uint32_t idesc = sm100::idesc_e4m3_f32(PBM, PBN);
            const uint64_t da = sm100::desc_kmajor_sw128(smem, 0), db = sm100::desc_kmajor_sw128(smem + P_TILE, 0);
            const long blocks = (long)((T.total - pair + npairs - 1) / npairs) * P.nkb;
            int s = 0;
            uint32_t ph = 0, use = 0;
            const bool lead = sm100::elect_one();
            for (long blk = 0; blk < blocks; blk++) {
                const uint32_t slot = (uint32_t)(blk & 1);
                bool ok = __all_sync(0xffffffffu, wait_flag(&ctl->full[s], ph, abort_flag, P.flag)) &&
                          __all_sync(0xffffffffu, wait_flag(&ctl->tempty[slot], use ^ 1, abort_flag, P.flag));
                if (!ok) break;
                const uint64_t oa = da + (uint64_t)(s * P_STAGE >> 4), ob = db + (uint64_t)(s * P_STAGE >> 4);
                sm100::tc_fence_after();
                if (lead) {
                    #pragma unroll
                    for (int k = 0; k < 4; k++)
                        sm100::mma_f8_pair(tmem + slot * PBN, oa + 2 * k, ob + 2 * k, idesc, k != 0);
                    sm100::mma_commit_pair_mc(&ctl->done[s], 0x3);
                }
                __syncwarp();
                if (++s == PSTAGES) { s = 0; ph ^= 1; }
                use ^= (uint32_t)blk & 1;
            }
        }
    } else {
        sm100::regs_grow<P_REGS_HIGH>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        uint8_t* box = boxes + (warp - 4) * 2 * P_BOX;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + half * 128;
        const int nwb = (P.N + KB - 1) / KB;
        // scales run two blocks ahead of their use, across tiles
        int ft = pair, fk = 0;
        const float *fx = nullptr, *fw = nullptr;
        auto next_scale = [&](float& x, float& w) {
            if (ft >= T.total) { x = w = 0.f; return; }
            if (fk == 0) {
                const int row = ft % T.num_m * PBM + (int)rank * 128 + q * 32 + lane, wb = ft / T.num_m * 2 + half;
                fx = row < P.M ? P.xs + row : nullptr;
                fw = wb < nwb ? P.ws + (size_t)wb * P.nkb : nullptr;
            }
            x = fx ? __ldg(fx + (size_t)fk * P.M) : 0.f;
            w = fw ? __ldg(fw + fk) : 0.f;
            if (++fk == P.nkb) { fk = 0; ft += npairs; }
        };
        float x0, w0, x1, w1;
        next_scale(x0, w0);
        next_scale(x1, w1);
        int s = 0;
        uint32_t ph = 0, it = 0;
        bool ok = true;
        for (int tile = pair; tile < T.total; tile += npairs) {
            uint64_t acc[64];
            #pragma unroll
            for (int i = 0; i < 64; i++) acc[i] = 0;
            for (int kb = 0; kb < P.nkb; kb++, it++) {
                const uint32_t sb = __float_as_uint(x0 * w0);
                const uint64_t ss = pack2(sb, sb);
                x0 = x1; w0 = w1;
                next_scale(x1, w1);
                const uint32_t slot = it & 1;
                if (!__all_sync(0xffffffffu, wait_flag(&ctl->done[s], ph, abort_flag, P.flag))) { ok = false; break; }
                sm100::tc_fence_after();
                const uint32_t ta = taddr + slot * PBN;
                uint32_t d[2][32];
                sm100::tmem_ld32_async(ta, d[0]);
                #pragma unroll
                for (int j = 0; j < 4; j++) {
                    sm100::tmem_wait32(d[j & 1]);
                    if (j < 3) {
                        sm100::tmem_ld32_async(ta + 32 * (j + 1), d[(j + 1) & 1]);
                    } else {             // the slot is read: both CTAs' warps give it back to the MMA thread
                        sm100::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) sm100::mbar_arrive_cluster_cta(sm100::map_to_rank(&ctl->tempty[slot], 0));
                    }
                    #pragma unroll
                    for (int i = 0; i < 16; i++)
                        acc[16 * j + i] = fma2(pack2(d[j & 1][2 * i], d[j & 1][2 * i + 1]), ss, acc[16 * j + i]);
                }
                if (++s == PSTAGES) { s = 0; ph ^= 1; }
            }
            if (!ok) break;
            pair_store(P, T, &my, box, tile % T.num_m * PBM + (int)rank * 128 + q * 32, tile / T.num_m * PBN + half * 128, acc);
        }
        if (lane == 0) sm100::bulk_wait_all();
    }
    sm100::tc_fence_before();
    sm100::cluster_sync();               // no CTA leaves while its pair still signals it
    if (warp == 1) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc_pair(tmem, 512);
    }
}

int launch_pair(const Fp8LinearArgs& a, const LinParams& P, cudaStream_t s) {
    CUtensorMap mx, mw, my;
    if (!make_tmap_u8(&mx, a.xq, a.M, a.K, a.ldx, 128) || !make_tmap_u8(&mw, a.wq, a.N, a.K, a.ldw, 128)) return -1;
    PairTiles T;
    T.num_m = (a.M + PBM - 1) / PBM;
    T.num_n = (a.N + PBN - 1) / PBN;
    const long tiles = (long)T.num_m * T.num_n;
    if (tiles > 2147483647L - 1024) return -1;
    T.total = (int)tiles;
    const size_t e = a.y_type == S2B_PREC_FP32 ? 4 : 2;
    T.tma_y = ((uintptr_t)a.y & 15) == 0 && (size_t)a.ldy * e % 16 == 0;
    if (T.tma_y) {
        if (!make_tmap_out(&my, a.y, a.y_type, a.M, a.N, a.ldy)) return -1;
    } else {
        my = mx;                         // not used
    }
    int pairs = op_sms() / 2;
    if (T.total < pairs) pairs = T.total;
    k_fp8_linear_pair<<<2 * pairs, PTHREADS, P_SMEM, s>>>(mx, mw, my, P, T);
    return 1;
}

}  // namespace

int op_launch(const Fp8LinearArgs& a, cudaStream_t s) {
    LinParams P;
    P.xs = a.xs; P.ws = a.ws; P.bias = a.bias; P.y = a.y;
    P.M = a.M; P.N = a.N; P.nkb = (int)((a.K + KB - 1L) / KB); P.ldy = a.ldy; P.y_type = a.y_type;
    P.flag = device_flag();
    if (!P.flag) return -1;
    static const int force = getenv("S2B_X") ? atoi(getenv("S2B_X")) : 0;
    if (force == 1 || (!force && a.M > 256)) return launch_pair(a, P, s);
    if (a.M <= 16) return launch_narrow<16>(a, P, s);
    if (a.M <= 32) return launch_narrow<32>(a, P, s);
    return launch_narrow<64>(a, P, s);
}

int fp8_linear_init_device() {
    const void* f[3] = {(const void*)k_fp8_linear_narrow<16>, (const void*)k_fp8_linear_narrow<32>,
                        (const void*)k_fp8_linear_narrow<64>};
    const int b[3] = {NarrowCfg<16>::SMEM, NarrowCfg<32>::SMEM, NarrowCfg<64>::SMEM};
    for (int i = 0; i < 3; i++)
        if (cudaError_t e = cudaFuncSetAttribute(f[i], cudaFuncAttributeMaxDynamicSharedMemorySize, b[i])) return (int)e;
    // the pair kernel's warpgroups exchange registers: they wait for ever if
    // the kernel was compiled to fewer than their shares add up to
    cudaFuncAttributes at;
    if (cudaError_t e = cudaFuncGetAttributes(&at, (const void*)k_fp8_linear_pair)) return (int)e;
    if (at.numRegs != P_REGS) return (int)cudaErrorInvalidKernelImage;
    return (int)cudaFuncSetAttribute((const void*)k_fp8_linear_pair, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM);
}

}  // namespace s2b
