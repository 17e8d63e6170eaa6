// k_fp8_linear.cu -- y = sum_b xs[b, m] ws[n / 128, b] (xq . wq over block b) + bias
// on the tcgen05 tensor cores (kind::f8f6f4, e4m3 codes), blocks of 128 along K.
//
// Two kernels: few rows (a cluster divides K) and many (persistent CTA pairs).
// The scales change with every block of K, so a block's products cannot simply
// stay in the accumulator.  Either the tensor core applies the scales, where
// they are powers of two, or each block's fp32 sum (4 MMAs of 32 codes) goes to a
// TMEM slot of its own and the epilogue warps add scale * sum to fp32 registers
// while the next block runs.  Scales are any fp32 values; sums and scale products
// are fp32, rounded once to y's type.  The tensor core's own sums cut their low
// bits: 7e-7 of y's norm at K 6912 with power-of-two scales, 1.2e-7 otherwise.
#include "kcommon.cuh"
#include "launch.cuh"
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
// CLUSTER: on a barrier that the other CTA of a pair arrives at.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_flag(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* flag) {
    for (uint32_t i = 0; i < sm100::WAIT_LIMIT; i++) {
        if (CLUSTER ? sm100::mbar_try_wait_cluster(bar, parity) : sm100::mbar_try_wait(bar, parity)) return true;
        if ((i & 1023) == 1023 && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(flag, 1);
    return false;
}

// The same for waits of thousands of cycles: the warp sleeps between polls and
// leaves the issue slots of its scheduler to the warps that feed the tensor core.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_flag_idle(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* flag) {
    for (uint32_t i = 0; i < (1u << 22); i++) {
        if (CLUSTER ? sm100::mbar_try_wait_cluster(bar, parity) : sm100::mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *abort_flag) return false;
        __nanosleep(100);
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
// Bound by latency: of the 6.5 us that a CTA takes for 58 rows x 5120 x 2560
// (13.7 MB), 1.4 pass before the first block has arrived, 2 in five blocks, 3 in
// joining eight ranks.  B200, in a burst: that call 9.5 us, 1 x 2560 x 7680 6.6 us,
// the smallest call 5.2 us.
template <int BT> struct NarrowCfg {
    static constexpr int W_BYTES = 128 * KB, X_BYTES = BT * KB, STAGE = W_BYTES + X_BYTES;
    static constexpr int STAGES = BT == 64 ? 4 : 5;
    // TMEM slots of BT columns: as many as 256 columns hold (two CTAs an SM).  A
    // rank of a split K has fewer blocks than that, so its MMAs never wait for
    // the epilogue.
    static constexpr int COLS = 256, SLOTS = COLS / BT;
    static constexpr int G = SLOTS / 2 < 4 ? SLOTS / 2 : 4;      // blocks the epilogue takes at a time
    static constexpr int SMEM = STAGES * STAGE + 1024 + 512 + 4 * G * BT * 4;
    static_assert(128 * BT * 4 <= STAGES * STAGE, "the joined sums reuse the stages");
};
template <int STAGES, int SLOTS> struct NarrowCtl {
    uint64_t full[STAGES], done[STAGES], tfull[SLOTS], tempty[SLOTS];
    uint32_t tmem_slot;
    int abort;
};

// Sums the ranks' sums of weight row n in rank order and writes this rank's
// tokens, four at a time: red is [BT / 4][128 weight rows][4 tokens].  Every load
// from the other ranks is in flight before the first sum.
template <int BT, int SPLIT>
__device__ __forceinline__ void join_ranks(const LinParams& P, float4* red, int rank, int m0, int n) {
    constexpr int G = (BT / 4 + SPLIT - 1) / SPLIT;      // groups of four tokens a rank
    const float b = P.bias ? P.bias[n] : 0.f;
    float4 v[G][SPLIT];
    #pragma unroll
    for (int g = 0; g < G; g++) {
        const int c4 = g * SPLIT + rank;
        if (c4 * 4 >= BT || m0 + c4 * 4 >= P.M) break;
        #pragma unroll
        for (int r = 0; r < SPLIT; r++) v[g][r] = sm100::ld_cluster_f32x4(sm100::map_to_rank(red + c4 * 128, r));
    }
    #pragma unroll
    for (int g = 0; g < G; g++) {
        const int m = m0 + (g * SPLIT + rank) * 4;
        if ((g * SPLIT + rank) * 4 >= BT || m >= P.M) break;
        float4 t = v[g][0];
        #pragma unroll
        for (int r = 1; r < SPLIT; r++) { t.x += v[g][r].x; t.y += v[g][r].y; t.z += v[g][r].z; t.w += v[g][r].w; }
        const float o[4] = {t.x, t.y, t.z, t.w};
        #pragma unroll
        for (int i = 0; i < 4; i++)
            if (m + i < P.M) store_y(P.y, P.y_type, (size_t)(m + i) * P.ldy + n, o[i] + b);
    }
}

template <int BT>
__global__ void __launch_bounds__(192) k_fp8_linear_narrow(const __grid_constant__ CUtensorMap mw,
                                                           const __grid_constant__ CUtensorMap mx,
                                                           const __grid_constant__ LinParams P, int split) {
    using C = NarrowCfg<BT>;
    constexpr int ST = C::STAGES;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    typedef NarrowCtl<ST, C::SLOTS> Ctl;
    Ctl* ctl = reinterpret_cast<Ctl*>(smem + ST * C::STAGE);
    float* sc = reinterpret_cast<float*>(smem + ST * C::STAGE + 512);    // [4 warps][G][BT]
    static_assert(sizeof(Ctl) <= 512, "control block");
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = split > 1 ? (int)sm100::cluster_ctarank() : 0;
    const int tile = blockIdx.x / split;
    const int ntn = (P.N + 127) / 128;
    const int nb = tile % ntn, n0 = nb * 128, m0 = tile / ntn * BT;
    const int kb0 = (int)((long)P.nkb * rank / split), kb1 = (int)((long)P.nkb * (rank + 1) / split);

    auto load_block = [&](int kb, int s) {
        uint8_t* st = smem + s * C::STAGE;
        sm100::mbar_arrive_expect_tx(&ctl->full[s], C::STAGE);
        sm100::tma_load_2d(st, &mw, &ctl->full[s], kb * KB, n0);
        sm100::tma_load_2d(st + C::W_BYTES, &mx, &ctl->full[s], kb * KB, m0);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < ST; s++) { sm100::mbar_init(&ctl->full[s], 1); sm100::mbar_init(&ctl->done[s], 1); }
        for (int i = 0; i < C::SLOTS; i++) { sm100::mbar_init(&ctl->tfull[i], 1); sm100::mbar_init(&ctl->tempty[i], 4); }
        ctl->abort = 0;
        sm100::fence_barrier_init();
        chain_wait();
        // the first loads are on their way while TMEM is allocated
        for (int s = 0; s < ST && kb0 + s < kb1; s++) load_block(kb0 + s, s);
    }
    if (warp == 1) {
        sm100::tmem_alloc(&ctl->tmem_slot, C::COLS);
        sm100::tmem_relinquish();
    }
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = ctl->tmem_slot;
    chain_release();                     // not before this CTA has its TMEM: the next kernel's could take it first
    chain_wait();
    float acc[BT];
    #pragma unroll
    for (int c = 0; c < BT; c++) acc[c] = 0.f;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            long issued = min(ST, kb1 - kb0);
            for (int kb = kb0 + ST; kb < kb1; kb++) {
                if (!wait_flag(&ctl->done[s], ph, abort_flag, P.flag)) break;
                load_block(kb, s);
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
        // the whole warp walks the loop and one elected lane issues: descriptors
        // stay in uniform registers (a lane on its own took three times as long)
        constexpr uint32_t idesc = sm100::idesc_e4m3_f32(128, BT);
        const uint64_t dw = sm100::desc_kmajor_sw128(smem, 0), dx = sm100::desc_kmajor_sw128(smem + C::W_BYTES, 0);
        const bool lead = sm100::elect_one();
        auto wait = [&](uint64_t* bar, uint32_t par) { return __all_sync(0xffffffffu, wait_flag(bar, par, abort_flag, P.flag)) != 0; };
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            const int i = kb - kb0, slot = i % C::SLOTS;
            if (i >= C::SLOTS && !wait(&ctl->tempty[slot], ((i / C::SLOTS) & 1) ^ 1)) break;
            if (!wait(&ctl->full[s], ph)) break;
            sm100::tc_fence_after();
            if (lead) {
                const uint64_t off = (uint64_t)(s * C::STAGE >> 4);      // descriptors count 16-byte units
                #pragma unroll
                for (int k = 0; k < 4; k++) sm100::mma_f8(tmem + slot * BT, dw + off + 2 * k, dx + off + 2 * k, idesc, k != 0);
                sm100::mma_commit(&ctl->tfull[slot]);
                if (kb + ST < kb1) sm100::mma_commit(&ctl->done[s]);     // loaded again
            }
            __syncwarp();
            if (++s == ST) { s = 0; ph ^= 1; }
        }
    } else {
        const int q = warp & 3;
        constexpr int G = C::G, PER = (BT + 31) / 32;
        float* my = sc + (warp - 2) * G * BT;
        const float* wrow = P.ws + (size_t)nb * P.nkb;
        // Scales of the next G blocks as loaded: lane l holds tokens l and l + 32.
        float w[G], x[G][PER];
        auto fetch = [&](int kb, float& wv, float (&xv)[PER]) {
            const bool in = kb < kb1;
            wv = in ? wrow[kb] : 0.f;
            #pragma unroll
            for (int j = 0; j < PER; j++) {
                const int c = lane + 32 * j;
                xv[j] = in && c < BT && m0 + c < P.M ? P.xs[(size_t)kb * P.M + m0 + c] : 0.f;
            }
        };
        #pragma unroll
        for (int a = 0; a < G; a++) fetch(kb0 + a, w[a], x[a]);
        // G blocks at a time, after the last one's MMAs (which end in order): one
        // wait and one release instead of G, each a few hundred cycles
        for (int kb = kb0; kb < kb1; kb += G) {
            const int n = min(G, kb1 - kb), i0 = kb - kb0;
            #pragma unroll
            for (int a = 0; a < G; a++) {
                #pragma unroll
                for (int j = 0; j < PER; j++)
                    if (lane + 32 * j < BT) my[a * BT + lane + 32 * j] = w[a] * x[a][j];
                fetch(kb + G + a, w[a], x[a]);
            }
            __syncwarp();
            const int last = i0 + n - 1;
            if (!__all_sync(0xffffffffu, wait_flag(&ctl->tfull[last % C::SLOTS], (last / C::SLOTS) & 1, abort_flag, P.flag))) break;
            sm100::tc_fence_after();
            #pragma unroll
            for (int a = 0; a < G; a++) {
                if (a >= n) break;
                const uint32_t ta = tmem + ((uint32_t)(q * 32) << 16) + (i0 + a) % C::SLOTS * BT;
                #pragma unroll
                for (int c0 = 0; c0 < BT; c0 += 16) {
                    float d[16];
                    sm100::tmem_ld16(ta + c0, d);
                    #pragma unroll
                    for (int c = 0; c < 16; c += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(my + a * BT + c0 + c);
                        acc[c0 + c] = fmaf(d[c], f.x, acc[c0 + c]);
                        acc[c0 + c + 1] = fmaf(d[c + 1], f.y, acc[c0 + c + 1]);
                        acc[c0 + c + 2] = fmaf(d[c + 2], f.z, acc[c0 + c + 2]);
                        acc[c0 + c + 3] = fmaf(d[c + 3], f.w, acc[c0 + c + 3]);
                    }
                }
            }
            sm100::tc_fence_before();
            __syncwarp();
            if (lane < n) sm100::mbar_arrive(&ctl->tempty[(i0 + lane) % C::SLOTS]);
        }
    }
    __syncwarp();
    __syncthreads();                     // every MMA and load of this CTA is done: the stages are free
    const bool epi = warp >= 2;
    const int nl = (warp & 3) * 32 + lane, n = n0 + nl;
    if (split == 1) {
        if (epi && n < P.N) {
            const float b = P.bias ? P.bias[n] : 0.f;
            #pragma unroll
            for (int c = 0; c < BT; c++)
                if (m0 + c < P.M) store_y(P.y, P.y_type, (size_t)(m0 + c) * P.ldy + n, acc[c] + b);
        }
    } else {
        float4* red = reinterpret_cast<float4*>(smem) + nl;      // [BT / 4][128] of four tokens
        if (epi) {
            #pragma unroll
            for (int c = 0; c < BT; c += 4) red[c / 4 * 128] = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
        }
        sm100::cluster_sync();
        if (epi && n < P.N) {
            if (split == 2) join_ranks<BT, 2>(P, red, rank, m0, n);
            else if (split == 4) join_ranks<BT, 4>(P, red, rank, m0, n);
            else join_ranks<BT, 8>(P, red, rank, m0, n);
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
    return launch_chained(k_fp8_linear_narrow<BT>, dim3((unsigned)(tiles * split)), 192, C::SMEM, split, s, mw, mx, P, split);
}

// ---------------------------------------------------------------- many rows
// Persistent CTA pairs (cta_group::2), tiles of 256 rows x BN columns: a CTA
// holds 128 rows of A and BN / 2 of B of every block of K and gets 128 x BN
// fp32 sums in one of two TMEM slots.  Each tile runs one of two ways:
//
//   scaled   every scale of the tile is a power of two (what the quantiser
//            writes): the tensor core applies them (kind::mxf8f6f4, one E8M0
//            byte a row and 32 codes; the four MMAs of a block use one byte)
//            and sums the whole of K in a slot.  The epilogue of a tile runs
//            beside the next tile's MMAs.
//   general  any fp32 scales: a block's sum goes to a slot, the epilogue warps
//            add scale * sum to registers while the next block runs.
//
// The general way is bound by the round trip MMA -> commit -> TMEM read ->
// release -> MMA, about 2700 cycles for two blocks of 470 (5498 x 2560 x 13824:
// 360 us in a burst, where a form of this kernel without the scaled way, its
// accumulators read 32 columns at a time, took 226). The scaled one takes about 610 cycles a block where the MMAs alone
// need 470 (shared memory feeds the tensor core and takes the loads at the same
// time) and loses 10 % between tiles: 173 us, 2.2 PFLOP/s; in a long run the
// 1000 W cap lowers the clock and it takes a fifth longer.
//
// Warpgroup 0: warps 0 and 2 load by TMA, warp 1 (even CTA) issues the MMAs.
// Warpgroup 1 looks at its CTA's part of each tile's scales, a tile ahead, tells
// both CTAs, and writes the scale bytes of four blocks at a time to TMEM; warp 3
// passes on that a verdict's readers are done.  Warpgroups 2 and 3 are the epilogue: a warp owns 32 rows and
// CH0 (the rest) chunks of 32 columns -- a chunk lies in one weight block.
// Two consecutive blocks share one full barrier (a wait costs the MMA warp about
// 200 cycles), each stage has its own done barrier (loads follow one by one).
constexpr int PBM = 256, PSTAGES = 6, PBARS = PSTAGES / 2, PTHREADS = 512, RING = 4;
// Register shares: 128 a thread at launch.
constexpr int P_REGS = 128, P_REGS_0 = 48, P_REGS_1 = 80, P_REGS_EPI = 192;
static_assert(P_REGS_0 + P_REGS_1 + 2 * P_REGS_EPI <= 4 * P_REGS, "register shares exceed the launch's");

template <int BN> struct PairCfg8 {
    static constexpr int CH = BN / 32, CH0 = (CH + 1) / 2;       // chunks of a tile, of warpgroup 2
    static constexpr int A_TILE = 128 * KB, B_TILE = BN / 2 * KB, STAGE = A_TILE + B_TILE;
    static constexpr int BOX = 4096;                             // a warp's staging: two boxes of 16-bit y, one of fp32
    static constexpr int SMEM = PSTAGES * STAGE + 8 * BOX + 1024 + 1024;
    static constexpr int SF = 2 * BN;                            // TMEM column of the scale bytes: RING x 16
    static_assert(SF + RING * 16 <= 512 && BN % 32 == 0 && CH <= 8 && STAGE % 1024 == 0, "TMEM and tile layout");
};

struct alignas(16) PairCtl {
    uint64_t full[PBARS], done[PSTAGES], tfull[2], tempty[2];
    uint64_t sfull[RING], sempty[RING];          // scale bytes of four blocks
    uint64_t mfull[RING], mempty[RING];          // the way a tile runs; this CTA's readers of it are done
    uint64_t mgone[RING];                        // both CTAs' are
    uint4 odd[RING][2];                          // word q of CTA r: a scale that its warp q looked at is no power of two
    uint32_t tmem_slot;
    int abort;
};

struct PairTiles {
    int num_m, num_n, total;
    int tma_y, tma_edge;                 // y through TMA boxes (16-byte rows); the last columns too
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)hi << 32 | lo; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// Two values in y's 16-bit type.
__device__ __forceinline__ uint32_t half2_bits(float a, float b, int t) {
    if (t == S2B_PREC_FP16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Lane = row: 32 columns of it into a staging box of 32 rows x 128 bytes (fp32)
// or x 64 bytes (16-bit), swizzled so that the 16-byte stores hit all banks.
// `bias` is lane l's: column l's.
template <bool BIAS>
__device__ __forceinline__ void stage_chunk(uint8_t* box, const uint32_t v[32], float bias, int type) {
    const int lane = threadIdx.x & 31;
    auto at = [&](int i) { return BIAS ? __uint_as_float(v[i]) + __shfl_sync(0xffffffffu, bias, i) : __uint_as_float(v[i]); };
    if (type == S2B_PREC_FP32) {
        #pragma unroll
        for (int j = 0; j < 8; j++) {
            const float4 f = make_float4(at(4 * j), at(4 * j + 1), at(4 * j + 2), at(4 * j + 3));
            *reinterpret_cast<float4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = f;
        }
    } else {
        #pragma unroll
        for (int j = 0; j < 4; j++) {
            uint4 u;
            u.x = half2_bits(at(8 * j), at(8 * j + 1), type);
            u.y = half2_bits(at(8 * j + 2), at(8 * j + 3), type);
            u.z = half2_bits(at(8 * j + 4), at(8 * j + 5), type);
            u.w = half2_bits(at(8 * j + 6), at(8 * j + 7), type);
            *reinterpret_cast<uint4*>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = u;
        }
    }
}

// The warp's staged box of 32 columns from column c to y: one TMA store, or
// element by element where y's rows start on no 16 bytes, and in the last
// columns where y's width is no multiple of 16 bytes (the store writes whole
// 16-byte pieces, past the tensor map's width).
__device__ __forceinline__ void flush_chunk(const LinParams& P, const PairTiles& T, const CUtensorMap* my, const uint8_t* box, int row0,
                                            int c) {
    const int lane = threadIdx.x & 31;
    if (row0 >= P.M || c >= P.N) return;
    if (T.tma_y && (T.tma_edge || c + 32 <= P.N)) {
        if (lane == 0) sm100::tma_store_2d(my, box, c, row0);
        return;
    }
    const int rows = min(32, P.M - row0);
    if (c + lane >= P.N) return;
    for (int r = 0; r < rows; r++) {
        const size_t at = (size_t)(row0 + r) * P.ldy + c + lane;
        if (P.y_type == S2B_PREC_FP32)
            ((uint32_t*)P.y)[at] = *reinterpret_cast<const uint32_t*>(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
        else
            ((uint16_t*)P.y)[at] = *reinterpret_cast<const uint16_t*>(box + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
    }
}

// Positive normal powers of two are what an E8M0 byte (the exponent) can say.
__device__ __forceinline__ bool no_power(float s) {
    const uint32_t u = __float_as_uint(s);
    return (u & 0x807FFFFFu) != 0 || u == 0 || u == 0x7F800000u;
}

template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PTHREADS, 1)
k_fp8_linear_pair(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw,
                  const __grid_constant__ CUtensorMap my, const __grid_constant__ LinParams P,
                  const __grid_constant__ PairTiles T) {
    using C = PairCfg8<BN>;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    uint8_t* boxes = smem + PSTAGES * C::STAGE;
    PairCtl* ctl = reinterpret_cast<PairCtl*>(boxes + 8 * C::BOX);
    static_assert(sizeof(PairCtl) <= 1024, "control block");
    volatile int* abort_flag = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2, q = warp & 3;
    const uint32_t rank = sm100::cluster_ctarank();
    const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < PBARS; s++) sm100::mbar_init(&ctl->full[s], 1);
        for (int s = 0; s < PSTAGES; s++) sm100::mbar_init(&ctl->done[s], 1);
        for (int i = 0; i < 2; i++) { sm100::mbar_init(&ctl->tfull[i], 1); sm100::mbar_init(&ctl->tempty[i], 16); }
        for (int i = 0; i < RING; i++) {
            sm100::mbar_init(&ctl->sfull[i], 8);         // warpgroup 1 of both CTAs
            sm100::mbar_init(&ctl->sempty[i], 1);
            sm100::mbar_init(&ctl->mfull[i], 5);         // this CTA's, and the expectation of the other's four words
            sm100::mbar_init(&ctl->mempty[i], rank == 0 ? 13 : 12);      // warpgroups 1 to 3, the MMA warp
            sm100::mbar_init(&ctl->mgone[i], 2);         // warp 3 of both CTAs
        }
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
    chain_release();                     // not before this CTA has its TMEM
    chain_wait();

    // The way tile number ti of this pair runs, read by a whole warp: 1
    // scaled, 0 general, -1 when the wait expired.
    auto tile_way = [&](uint32_t ti) -> int {
        const uint32_t e = ti % RING, par = (ti / RING) & 1;
        bool ok = false;
        for (uint32_t i = 0; i < (1u << 22) && !ok; i++) {
            ok = sm100::mbar_try_wait_cluster(&ctl->mfull[e], par);
            if (!ok && (i & 1023) == 1023 && *abort_flag) break;
            if (!ok && wg != 0) __nanosleep(100);
        }
        if (!__all_sync(0xffffffffu, ok)) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(P.flag, 1);
            return -1;
        }
        const uint4 a = ctl->odd[e][0], b = ctl->odd[e][1];
        const int way = !(a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w);
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&ctl->mempty[e]);
        return way;
    };

    if (wg == 0) {
        sm100::regs_shrink<P_REGS_0>();
        if (warp != 1 && warp != 3 && lane == 0) {
            // warp 0 loads A's tiles, warp 2 B's
            const bool isb = warp == 2;
            const CUtensorMap* map = isb ? &mw : &mx;
            int s = 0;                                   // stage
            uint32_t ph = 0;
            long issued = 0;                             // full barriers begun
            bool ok = true;
            for (int tile = pair; tile < T.total && ok; tile += npairs) {
                const int r = isb ? tile / T.num_m * BN + (int)rank * (BN / 2) : tile % T.num_m * PBM + (int)rank * 128;
                for (int kb = 0; kb < P.nkb; kb++) {
                    // both CTAs' MMAs on this stage are done
                    if (!wait_flag(&ctl->done[s], ph ^ 1, abort_flag, P.flag)) { ok = false; break; }
                    const bool first = (kb & 1) == 0;
                    if (first && !isb) {
                        if (rank == 0) sm100::mbar_arrive_expect_tx(&ctl->full[s >> 1], min(2, P.nkb - kb) * 2 * C::STAGE);
                        issued++;
                    }
                    const uint32_t fb = sm100::map_to_rank(&ctl->full[s >> 1], 0);
                    sm100::tma_load_2d_pair(smem + s * C::STAGE + (isb ? C::A_TILE : 0), map, fb, kb * KB, r);
                    s++;
                    if (kb == P.nkb - 1 && first) s++;   // an odd block's partner stage stays empty
                    if (s >= PSTAGES) { s = 0; ph ^= 1; }
                }
            }
            if (rank == 0 && !isb)       // every load of the pair has landed (bounded) before anyone leaves
                for (long i = 1; i <= PBARS && i <= issued; i++) {
                    const long k = issued - i;
                    for (uint32_t w = 0; w < sm100::WAIT_LIMIT && !sm100::mbar_try_wait(&ctl->full[k % PBARS], (k / PBARS) & 1); w++) {}
                }
        } else if (warp == 3 && lane == 0) {
            // the release to the cluster that no reader of a verdict waits for
            uint32_t ti = 0;
            for (int tile = pair; tile < T.total; tile += npairs, ti++) {
                const uint32_t e = ti % RING;
                if (!wait_flag_idle(&ctl->mempty[e], (ti / RING) & 1, abort_flag, P.flag)) break;
                for (uint32_t r = 0; r < 2; r++) sm100::mbar_arrive_cluster(sm100::map_to_rank(&ctl->mgone[e], r));
            }
        } else if (warp == 1 && rank == 0) {
            constexpr uint32_t idesc = sm100::idesc_e4m3_f32(PBM, BN);
            const uint64_t da = sm100::desc_kmajor_sw128(smem, 0), db = sm100::desc_kmajor_sw128(smem + C::A_TILE, 0);
            const bool lead = sm100::elect_one();
            int s = 0;
            uint32_t ph = 0, use = 0, grp = 0, ti = 0;     // stage, slot uses, groups of scale bytes, tiles
            bool ok = true;
            auto wait = [&](uint64_t* bar, uint32_t par) { return __all_sync(0xffffffffu, wait_flag(bar, par, abort_flag, P.flag)) != 0; };
            auto wait_cluster = [&](uint64_t* bar, uint32_t par) { return __all_sync(0xffffffffu, wait_flag<true>(bar, par, abort_flag, P.flag)) != 0; };
            for (int tile = pair; tile < T.total && ok; tile += npairs, ti++) {
                const int way = tile_way(ti);
                if (way < 0) break;
                if (way) {
                    const uint32_t slot = use & 1, d = tmem + slot * BN;
                    if (!(ok = wait_cluster(&ctl->tempty[slot], ((use >> 1) & 1) ^ 1))) break;
                    for (int kb0 = 0; kb0 < P.nkb && ok; kb0 += 4, grp++) {
                        if (!(ok = wait_cluster(&ctl->sfull[grp % RING], (grp / RING) & 1))) break;
                        const uint32_t sf = tmem + C::SF + grp % RING * 16;
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int left = P.nkb - kb0 - 2 * h;        // blocks from here
                            if (left <= 0) break;
                            if (!(ok = wait(&ctl->full[s], ph))) break;
                            sm100::tc_fence_after();
                            if (lead) {
                                #pragma unroll
                                for (int b = 0; b < 2; b++) {
                                    if (b >= left) break;
                                    const uint64_t off = (uint64_t)((2 * s + b) * C::STAGE >> 4);    // descriptors count 16-byte units
                                    #pragma unroll
                                    for (int k = 0; k < 4; k++)
                                        sm100::mma_mxf8_pair(d, da + off + 2 * k, db + off + 2 * k, sm100::idesc_mxe4m3(PBM, BN, 2 * h + b), sf,
                                                             sf + 4, (kb0 | h | b | k) != 0);
                                    sm100::mma_commit_pair_mc(&ctl->done[2 * s + b], 0x3);
                                }
                                if (left == 1) sm100::mma_commit_pair_mc(&ctl->done[2 * s + 1], 0x3);    // the empty partner
                            }
                            __syncwarp();
                            if (++s == PBARS) { s = 0; ph ^= 1; }
                        }
                        if (ok && lead) sm100::mma_commit_pair_mc(&ctl->sempty[grp % RING], 0x3);
                        __syncwarp();
                    }
                    if (ok && lead) sm100::mma_commit_pair_mc(&ctl->tfull[slot], 0x3);
                    __syncwarp();
                    use++;
                } else {
                    for (int kb = 0; kb < P.nkb; kb++, use++) {
                        const uint32_t slot = use & 1, d = tmem + slot * BN;
                        if (!(kb & 1) && !(ok = wait(&ctl->full[s], ph))) break;
                        if (!(ok = wait_cluster(&ctl->tempty[slot], ((use >> 1) & 1) ^ 1))) break;
                        sm100::tc_fence_after();
                        const bool last = (kb & 1) || kb == P.nkb - 1;
                        if (lead) {
                            const uint64_t off = (uint64_t)((2 * s + (kb & 1)) * C::STAGE >> 4);
                            #pragma unroll
                            for (int k = 0; k < 4; k++) sm100::mma_f8_pair(d, da + off + 2 * k, db + off + 2 * k, idesc, k != 0);
                            sm100::mma_commit_pair_mc(&ctl->done[2 * s + (kb & 1)], 0x3);
                            if (last && !(kb & 1)) sm100::mma_commit_pair_mc(&ctl->done[2 * s + 1], 0x3);    // the empty partner
                            sm100::mma_commit_pair_mc(&ctl->tfull[slot], 0x3);
                        }
                        __syncwarp();
                        if (last && ++s == PBARS) { s = 0; ph ^= 1; }
                    }
                }
            }
        }
    } else if (wg == 1) {
        sm100::regs_shrink<P_REGS_1>();
        // A look at every scale of this CTA's part of tile number ti, a quarter a
        // warp, posted to both CTAs: into this one's shared memory, and to the other
        // as a word that carries its own signal (cluster-scope releases for it took
        // 4 % of the whole call: 181 against 173 us).
        auto look = [&](int tile, uint32_t ti) {
            const int row = tile % T.num_m * PBM + (int)rank * 128 + (threadIdx.x & 127), n0 = tile / T.num_m * BN;
            const int wb0 = n0 / KB, words = ((min(n0 + BN, P.N) - 1) / KB - wb0 + 1) * P.nkb;
            bool odd = false;
            if (row < P.M) {
                const float* p = P.xs + row;
                #pragma unroll 20
                for (int kb = 0; kb < P.nkb; kb++) odd |= no_power(p[(size_t)kb * P.M]);
            }
            for (int i = threadIdx.x & 127; i < words; i += 128) odd |= no_power(P.ws[(size_t)wb0 * P.nkb + i]);
            const uint32_t any = __any_sync(0xffffffffu, odd), e = ti % RING;
            if (lane == 0) {
                // the entry's readers of RING tiles ago are done, in both CTAs
                wait_flag_idle<true>(&ctl->mgone[e], ((ti / RING) & 1) ^ 1, abort_flag, P.flag);
                uint32_t* word = reinterpret_cast<uint32_t*>(&ctl->odd[e][rank]) + q;
                *word = any;
                if (q == 0) sm100::mbar_arrive_expect_tx(&ctl->mfull[e], 16);
                sm100::mbar_arrive(&ctl->mfull[e]);
                sm100::st_async_u32(sm100::map_to_rank(word, rank ^ 1), any, sm100::map_to_rank(&ctl->mfull[e], rank ^ 1));
            }
            __syncwarp();
        };
        uint32_t grp = 0, ti = 0;
        look(pair, 0);
        for (int tile = pair; tile < T.total; tile += npairs, ti++) {
            // the next tile's verdict is there before its MMAs ask for it
            if (tile + npairs < T.total) look(tile + npairs, ti + 1);
            const int m0 = tile % T.num_m * PBM + (int)rank * 128, n0 = tile / T.num_m * BN;
            const int wb0 = n0 / KB, wbs = (min(n0 + BN, P.N) - 1) / KB - wb0 + 1;
            const int way = tile_way(ti);
            if (way < 0) break;
            if (!way) continue;
            // The next group's scales are on their way while this one is
            // written: held as loaded, packed only when their turn comes.
            struct Raw { float a[4][4], w[3][4]; };
            auto load = [&](int kb0) {
                Raw v;
                #pragma unroll
                for (int b = 0; b < 4; b++) {
                    const bool in = kb0 + b < P.nkb;
                    #pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int row = m0 + 32 * j + lane;
                        v.a[j][b] = in && row < P.M ? P.xs[(size_t)(kb0 + b) * P.M + row] : 1.f;
                    }
                    #pragma unroll
                    for (int j = 0; j < 3; j++) v.w[j][b] = in && j < wbs ? P.ws[(size_t)(wb0 + j) * P.nkb + kb0 + b] : 1.f;
                }
                return v;
            };
            // byte b of a word: the exponent of block kb0 + b
            auto pack = [](const float f[4]) {
                return __float_as_uint(f[0]) >> 23 | __float_as_uint(f[1]) >> 23 << 8 | __float_as_uint(f[2]) >> 23 << 16 |
                       __float_as_uint(f[3]) >> 23 << 24;
            };
            bool ok = true;
            Raw next = load(0);
            for (int kb0 = 0; kb0 < P.nkb; kb0 += 4, grp++) {
                uint32_t sa[4], w3[3], sb[8];
                #pragma unroll
                for (int j = 0; j < 4; j++) sa[j] = pack(next.a[j]);
                #pragma unroll
                for (int j = 0; j < 3; j++) w3[j] = pack(next.w[j]);
                #pragma unroll
                for (int c = 0; c < 8; c++) {
                    const int j = (n0 + 32 * c) / KB - wb0;
                    sb[c] = j == 0 ? w3[0] : j == 1 ? w3[1] : w3[2];
                }
                if (kb0 + 4 < P.nkb) next = load(kb0 + 4);
                ok = __all_sync(0xffffffffu, wait_flag_idle(&ctl->sempty[grp % RING], ((grp / RING) & 1) ^ 1, abort_flag, P.flag));
                if (!ok) break;
                sm100::tc_fence_after();
                const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + C::SF + grp % RING * 16;
                sm100::tmem_st4(at, sa);
                sm100::tmem_st8(at + 4, sb);
                sm100::tmem_wait_st();
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0) sm100::mbar_arrive_cluster_relaxed(sm100::map_to_rank(&ctl->sfull[grp % RING], 0));
            }
            if (!ok) break;
        }
    } else {
        sm100::regs_grow<P_REGS_EPI>();
        const int side = wg - 2, c0 = side * C::CH0, nc = side ? C::CH - C::CH0 : C::CH0;      // this warp's chunks
        uint8_t* box = boxes + (warp - 8) * C::BOX;
        const int per_box = P.y_type == S2B_PREC_FP32 ? 4096 : 2048, boxes_n = C::BOX / per_box;
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + c0 * 32;
        uint32_t tempty[2];
        tempty[0] = sm100::map_to_rank(&ctl->tempty[0], 0);
        tempty[1] = sm100::map_to_rank(&ctl->tempty[1], 0);
        uint32_t use = 0, ti = 0;
        int put = 0;                     // the staging box that comes next
        bool ok = true;
        for (int tile = pair; tile < T.total && ok; tile += npairs, ti++) {
            const int row0 = tile % T.num_m * PBM + (int)rank * 128 + q * 32, n0 = tile / T.num_m * BN + c0 * 32;
            const int way = tile_way(ti);
            if (way < 0) break;
            uint64_t acc[C::CH0][16];
            if (!way) {
                #pragma unroll
                for (int c = 0; c < C::CH0; c++)
                    #pragma unroll
                    for (int i = 0; i < 16; i++) acc[c][i] = 0;
                const float* px = row0 + lane < P.M ? P.xs + row0 + lane : nullptr;
                const float* pw = P.ws + (size_t)(n0 / KB) * P.nkb;
                const int nwb = (P.N + KB - 1) / KB;
                // chunk c is in weight block n0 / KB + step(c)
                auto step = [&](int c) { return (n0 % KB + 32 * c) / KB; };
                // scales two blocks ahead of their use
                struct Scale { float x, w[2]; };
                auto scale = [&](int kb) {
                    Scale v = {0.f, {0.f, 0.f}};
                    if (kb >= P.nkb) return v;
                    if (px) v.x = px[(size_t)kb * P.M];
                    v.w[0] = n0 / KB < nwb ? pw[kb] : 0.f;
                    v.w[1] = n0 / KB + 1 < nwb ? pw[P.nkb + kb] : 0.f;
                    return v;
                };
                Scale v0 = scale(0), v1 = scale(1);
                for (int kb = 0; kb < P.nkb; kb++, use++) {
                    const float s0 = v0.x * v0.w[0], s1 = v0.x * v0.w[1];
                    v0 = v1;
                    v1 = scale(kb + 2);
                    const uint32_t slot = use & 1, ta = taddr + slot * BN;
                    if (!__all_sync(0xffffffffu, wait_flag(&ctl->tfull[slot], (use >> 1) & 1, abort_flag, P.flag))) { ok = false; break; }
                    sm100::tc_fence_after();
                    // 16 columns on their way while 16 are added
                    uint32_t d[2][16];
                    sm100::tmem_ld16_async(ta, d[0]);
                    #pragma unroll
                    for (int c = 0; c < 2 * C::CH0; c++) {
                        if (c >= 2 * nc) break;
                        sm100::tmem_wait16(d[c & 1]);
                        if (c + 1 < 2 * nc) {
                            sm100::tmem_ld16_async(ta + 16 * (c + 1), d[(c + 1) & 1]);
                        } else {                 // the slot is read: back to the MMA warp
                            sm100::tc_fence_before();
                            __syncwarp();
                            if (lane == 0) sm100::mbar_arrive_cluster_relaxed(slot ? tempty[1] : tempty[0]);
                        }
                        const uint32_t sb = __float_as_uint(step(c / 2) ? s1 : s0);
                        const uint64_t ss = pack2(sb, sb);
                        #pragma unroll
                        for (int i = 0; i < 8; i++)
                            acc[c / 2][c % 2 * 8 + i] = fma2(pack2(d[c & 1][2 * i], d[c & 1][2 * i + 1]), ss, acc[c / 2][c % 2 * 8 + i]);
                    }
                }
                if (!ok) break;
            } else if (!__all_sync(0xffffffffu, wait_flag_idle(&ctl->tfull[use & 1], (use >> 1) & 1, abort_flag, P.flag))) {
                ok = false;
                break;
            }
            sm100::tc_fence_after();
            #pragma unroll
            for (int c = 0; c < C::CH0; c++) {
                if (c >= nc) break;
                const int col = n0 + 32 * c;
                const float bias = P.bias && col + lane < P.N ? P.bias[col + lane] : 0.f;
                uint32_t d[32];
                if (way) {
                    sm100::tmem_ld32_async(taddr + (use & 1) * BN + 32 * c, d);
                    sm100::tmem_wait32(d);
                    if (c == nc - 1) {
                        sm100::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) sm100::mbar_arrive_cluster_relaxed((use & 1) ? tempty[1] : tempty[0]);
                    }
                } else {
                    #pragma unroll
                    for (int i = 0; i < 16; i++) { d[2 * i] = (uint32_t)acc[c][i]; d[2 * i + 1] = (uint32_t)(acc[c][i] >> 32); }
                }
                // the box's previous store has been read
                uint8_t* st = box + put * per_box;
                put = (put + 1) % boxes_n;
                if (lane == 0) {
                    if (boxes_n == 2) sm100::bulk_wait_read<1>();
                    else sm100::bulk_wait_read<0>();
                }
                __syncwarp();
                if (P.bias) stage_chunk<true>(st, d, bias, P.y_type);
                else stage_chunk<false>(st, d, 0.f, P.y_type);
                if (T.tma_y) sm100::fence_proxy_async_smem();
                __syncwarp();
                flush_chunk(P, T, &my, st, row0, col);
                if (lane == 0) sm100::bulk_commit_group();
            }
            if (way) use++;
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

template <int BN>
int launch_pair(const Fp8LinearArgs& a, const LinParams& P, cudaStream_t s) {
    CUtensorMap mx, mw, my;
    if (!make_tmap_u8(&mx, a.xq, a.M, a.K, a.ldx, 128) || !make_tmap_u8(&mw, a.wq, a.N, a.K, a.ldw, BN / 2)) return -1;
    PairTiles T;
    T.num_m = (a.M + PBM - 1) / PBM;
    T.num_n = (a.N + BN - 1) / BN;
    const long tiles = (long)T.num_m * T.num_n;
    if (tiles > 2147483647L - 1024) return -1;
    T.total = (int)tiles;
    const size_t e = a.y_type == S2B_PREC_FP32 ? 4 : 2;
    T.tma_y = ((uintptr_t)a.y & 15) == 0 && (size_t)a.ldy * e % 16 == 0;
    T.tma_edge = (size_t)a.N * e % 16 == 0;
    if (T.tma_y) {
        if (!make_tmap_out(&my, a.y, a.y_type, a.M, a.N, a.ldy)) return -1;
    } else {
        my = mx;                         // not used
    }
    int pairs = op_sms() / 2;
    if (T.total < pairs) pairs = T.total;
    return launch_chained(k_fp8_linear_pair<BN>, dim3(2 * pairs), PTHREADS, PairCfg8<BN>::SMEM, 0, s, mx, mw, my, P, T);
}

}  // namespace

int op_launch(const Fp8LinearArgs& a, cudaStream_t s) {
    LinParams P;
    P.xs = a.xs; P.ws = a.ws; P.bias = a.bias; P.y = a.y;
    P.M = a.M; P.N = a.N; P.nkb = (int)((a.K + KB - 1L) / KB); P.ldy = a.ldy; P.y_type = a.y_type;
    P.flag = device_flag();
    if (!P.flag) return -1;
    // The narrow kernel while its tiles are few enough for four ranks or more
    // along K at two CTAs an SM; past that the pair kernel even where it leaves
    // SMs idle (K 2560, N 2560, in a burst: 192 rows 9.6 against 11.6 us, 256 rows
    // 11.9 against 11.8).
    const long narrow = ((a.N + 127L) / 128) * ((a.M + 63L) / 64);
    if (a.M > 64 && 4 * narrow > 2L * op_sms()) {
        // The tile width with the cheaper waves: a 192-column tile takes 0.94 of
        // a 224-column one's time.
        const int pairs = op_sms() / 2;
        const long tm = (a.M + PBM - 1L) / PBM;
        const double w224 = (double)((tm * ((a.N + 223L) / 224) + pairs - 1) / pairs);
        const double w192 = 0.94 * (double)((tm * ((a.N + 191L) / 192) + pairs - 1) / pairs);
        return w192 < w224 ? launch_pair<192>(a, P, s) : launch_pair<224>(a, P, s);
    }
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
    // the pair kernels' warpgroups exchange registers: they wait for ever if
    // the kernel was compiled to fewer than their shares add up to
    const void* p[2] = {(const void*)k_fp8_linear_pair<224>, (const void*)k_fp8_linear_pair<192>};
    const int pb[2] = {PairCfg8<224>::SMEM, PairCfg8<192>::SMEM};
    for (int i = 0; i < 2; i++) {
        cudaFuncAttributes at;
        if (cudaError_t e = cudaFuncGetAttributes(&at, p[i])) return (int)e;
        if (at.numRegs != P_REGS) return (int)cudaErrorInvalidKernelImage;
        if (cudaError_t e = cudaFuncSetAttribute(p[i], cudaFuncAttributeMaxDynamicSharedMemorySize, pb[i])) return (int)e;
    }
    return 0;
}

}  // namespace s2b
