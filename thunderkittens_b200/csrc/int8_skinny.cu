// 8-bit integer GEMM with few tokens ("decode"): D[M, N] = A_sc[m] * B_sc[n] * sum_k A[m, k] * B[n, k] with M <= 128.
//
// Bound by streaming the N * K bytes of weights from HBM once.  Two kernels, neither of which shares anything between CTAs or leaves
// anything but D in global memory, so that calls on any number of streams and captured graphs do not meet:
//
// Long streams: operands are swapped as in the NVFP4 decode kernel (decode.cu): weight rows are the M side of a tcgen05.mma (128
// lanes), the tokens its N side.  What matters is that every SM streams the same number of bytes
// without a gap:
//   * tokens are padded to the next multiple of 16 only;
//   * slabs have R <= 128 weight rows, R chosen so that they divide evenly over the SMs (a TMA box may have any number of rows;
//     the lanes past R multiply whatever is in shared memory and are not read).  N = 28672: two slabs of 97 rows for each SM;
//   * a CTA walks over its slabs; two accumulators in tensor memory, so that the epilogue of a slab overlaps the next one's loads;
//   * warp 0 = TMA producer, warp 1 = MMA issuer + tensor-memory owner, warps 2..9 = epilogue.
//
// Short streams: an SM's share of the weights is a few dozen KB, and a single pass through TMA, barriers and tensor memory costs
// more than the bytes.  A CTA takes 16 rows; its warps take 128-byte pieces of K in turn, straight from global memory into the
// registers of warp-level MMAs (m16n8k32), all loads of a thread in flight together, and add up in shared memory.
#include <atomic>
#include "ptx.cuh"
#include "internal.h"
#include "../../include/tkb200.h"

namespace tkb {

constexpr int kSkinnyStages = 16;
constexpr int kSkinnySmem = 208 * 1024;
constexpr int kSkinnyThreads = 10 * 32;

struct SkinnyParams {
    const float* a_sc; const float* b_sc;
    void* D; int64_t ldd;
    const uint8_t* B; int64_t ldb;
    int M, N, K, out_dtype;
    int rows, slabs;                        // weight rows of a slab, slabs
    int nb, acc_cols;                       // tokens padded to the MMA's N; tensor-memory columns of an accumulator
    int group, stages, w_bytes;             // operand ring: 128-byte blocks of K of a stage, stages, bytes from one block's weights to the next's
    int prefetch;                           // 128-byte pieces of its weights that a CTA asks L2 for early
    int* status;
    long long wait_limit;
};

// The same wait as mbar_wait, whose slow path stays out of the loops of one thread: they would run over it (see below)
__device__ __noinline__ bool skinny_wait_slow(int* abort_flag, int* status, long long limit, uint32_t bar, uint32_t parity) {
    return mbar_wait(WaitCtx{abort_flag, status, limit}, bar, parity);
}

__device__ __forceinline__ float scaled(int sum, float a_sc, float b_sc) { return __int2float_rn(sum) * a_sc * b_sc; }
__device__ __forceinline__ void put(float* d, float v) { *d = v; }
__device__ __forceinline__ void put(__half* d, float v) { *d = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* d, float v) { *d = __float2bfloat16_rn(v); }
// Calls f with D as a pointer to its type
template <typename F>
__device__ __forceinline__ void typed_out(const SkinnyParams& p, F f) {
    if (p.out_dtype == TKB_DTYPE_FP32) f(static_cast<float*>(p.D));
    else if (p.out_dtype == TKB_DTYPE_FP16) f(static_cast<__half*>(p.D));
    else f(static_cast<__nv_bfloat16*>(p.D));
}

// GROUP blocks of K share a stage and its barriers, since what the producer's and the MMA issuer's threads spend on a turn of their loops
// bounds slabs of few rows: M=1 N=1000 K=8192 (64 blocks) 16.1 us with 1 block, 12.6 with 2, 10.6 with 4, 10.1 with waits out of line.
template <int GROUP>
__global__ void __launch_bounds__(kSkinnyThreads)
int8_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const SkinnyParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[kSkinnyStages];
    __shared__ __align__(8) uint64_t bar_empty[kSkinnyStages];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;
    __shared__ float s_a_sc[128];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nst = p.stages;
    const uint32_t x_bytes = uint32_t(p.nb) * 128u, w_bytes = uint32_t(p.w_bytes);
    const uint32_t sX = (smem_u32(smem_raw) + 1023u) & ~1023u;      // tokens first: an MMA reads 128 rows from a block's weights on
    const uint32_t sW = sX + nst * GROUP * x_bytes;
    const int unit = int(blockIdx.x), units = int(gridDim.x);
    const int kblk = (p.K + 127) / 128;
    const uint32_t tmem_cols = p.acc_cols <= 32 ? 64u : (p.acc_cols <= 64 ? 128u : 256u);       // two accumulators

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < nst; s++) { mbar_init(smem_u32(&bar_full[s]), 1); mbar_init(smem_u32(&bar_empty[s]), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(smem_u32(&bar_acc_full[b]), 1); mbar_init(smem_u32(&bar_acc_empty[b]), 8); }
        fence_mbar_init();
        prefetch_tensormap(&tmW); prefetch_tensormap(&tmX);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&s_tmem_base), tmem_cols);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem_base;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        return mbar_try_wait(smem_u32(bar), parity) || skinny_wait_slow(&s_abort, p.status, p.wait_limit, smem_u32(bar), parity);
    };

    if (warp == 0) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, issued = 0;
            bool ok = true;
            asm volatile("griddepcontrol.wait;" ::: "memory");      // the tokens come from the kernel before this one
            const uint32_t tx = uint32_t(p.rows) * 128u + x_bytes;
            for (int slab = unit; slab < p.slabs && ok; slab += units)
                for (int kb = 0; kb < kblk; kb += GROUP) {
                    if (!wait(&bar_empty[stage], phase ^ 1)) { ok = false; break; }
                    const uint32_t full = smem_u32(&bar_full[stage]);
                    mbar_arrive_expect_tx(full, tx * uint32_t(min(GROUP, kblk - kb)));
#pragma unroll
                    for (int g = 0; g < GROUP; g++)
                        if (kb + g < kblk) {
                            tma_load_2d(sW + (stage * GROUP + g) * w_bytes, &tmW, full, (kb + g) * 128, slab * p.rows);
                            tma_load_2d(sX + (stage * GROUP + g) * x_bytes, &tmX, full, (kb + g) * 128, 0);
                        }
                    issued++;
                    if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
                }
            // this SM's loads are all on their way: the next kernel may set itself up
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (int s = 0; s < nst && ok; s++) {                   // stage releases of the MMA thread may still be in flight
                ok = wait(&bar_empty[stage], phase ^ 1);
                if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
            }
            if (!ok) drain_ring(bar_full, nst, issued, p.wait_limit);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, seg = 0;
            bool ok = true;
            const uint32_t idesc = idesc_int8(128, p.nb);
            for (int slab = unit; slab < p.slabs && ok; slab += units, seg++) {
                const uint32_t buf = seg & 1u, acc = tmem_base + buf * p.acc_cols;
                if (!wait(&bar_acc_empty[buf], ((seg >> 1) & 1u) ^ 1u)) { ok = false; break; }
                tc_fence_after();
                for (int kb = 0; kb < kblk; kb += GROUP) {
                    if (!wait(&bar_full[stage], phase)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (int g = 0; g < GROUP; g++)
                        if (kb + g < kblk) {
                            const uint64_t a_desc = smem_desc_sw128(sW + (stage * GROUP + g) * w_bytes);
                            const uint64_t b_desc = smem_desc_sw128(sX + (stage * GROUP + g) * x_bytes);
#pragma unroll
                            for (int j = 0; j < 4; j++) mma_i8<1>(acc, a_desc + 2 * j, b_desc + 2 * j, idesc, (kb + g > 0 || j > 0) ? 1u : 0u);
                        }
                    tc_commit<1>(smem_u32(&bar_empty[stage]));
                    if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
                }
                if (ok) tc_commit<1>(smem_u32(&bar_acc_full[buf]));
            }
        }
        __syncwarp();
    } else {
        // rows of the accumulator, and every other 32 of its columns (one warp for all of them: M=48 N=50257 K=2048 20.7 us against 19.8 us,
        // M=128 26.2 against 23.3; a warp for every 32 columns, 16 in all, 25.0 and 25.4)
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const int n_local = quarter * 32 + lane;
        // The first weights may be asked for before the previous kernel is done, whoever writes them: this only moves lines into L2,
        // where a later write finds them.
        for (int i = int(threadIdx.x) - 64; i < p.prefetch; i += 256) {
            const int kb = i / p.rows, row = unit * p.rows + i % p.rows;
            if (kb < kblk && row < p.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(p.B + int64_t(row) * p.ldb + kb * 128));
        }
        asm volatile("griddepcontrol.wait;" ::: "memory");          // D may still be read, and the scales written, by the kernel before this one
        if (int(threadIdx.x) - 64 < p.M) s_a_sc[threadIdx.x - 64] = p.a_sc[threadIdx.x - 64];
        asm volatile("bar.sync 1, 256;" ::: "memory");
        uint32_t seg = 0;
        for (int slab = unit; slab < p.slabs; slab += units, seg++) {
            const uint32_t buf = seg & 1u;
            const int n = slab * p.rows + n_local;
            const bool mine = n_local < p.rows && n < p.N;
            const float b_sc = mine ? p.b_sc[n] : 0.f;
            const bool full = wait(&bar_acc_full[buf], (seg >> 1) & 1u);
            if (!__all_sync(0xffffffffu, full)) break;              // (lanes together: the loads below are the warp's)
            tc_fence_after();
            for (int c0 = 32 * half; c0 < p.M; c0 += 64) {                  // (an accumulator has a multiple of 32 columns)
                uint32_t r[32];
                __syncwarp();
                tmem_ld_32x32_wait(tmem_base + (uint32_t(quarter * 32) << 16) + buf * p.acc_cols + c0, r);
                if (mine)
                    typed_out(p, [&](auto* D) {
                        auto* d = D + int64_t(c0) * p.ldd + n;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (c0 + i < p.M) put(d + i * p.ldd, scaled(int(r[i]), s_a_sc[c0 + i], b_sc));
                    });
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[buf]));
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, tmem_cols);
    }
}

// ---- short streams --------------------------------------------------------------------------

// (Plain loads here and below: what the kernel before this one wrote may not be read through the read-only path, which is free to
// fetch before griddepcontrol.wait.)
// 16 bytes at p, of which the first `left` belong to the row; the others count as zeros.  TAIL: rows may end inside 16 bytes.
template <bool TAIL>
__device__ __forceinline__ uint4 load16(const uint8_t* p, int left) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (left >= (TAIL ? 16 : 1)) v = *reinterpret_cast<const uint4*>(p);
    if constexpr (TAIL) {
        if (left > 0 && left < 16) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 15; i++)
                if (i < left) w[i >> 2] |= uint32_t(p[i]) << (8 * (i & 3));
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kShortWarps = 16;
constexpr int kShortRows = 16;

struct ShortParams {
    SkinnyParams s;
    const uint8_t* A; int64_t lda;
};

// One CTA: weight rows 16 blockIdx.x .. + 15 (the MMA's 16 rows) times up to 8 TT tokens (its columns).  In a piece of 128 bytes of K,
// lane 4 g + t holds bytes 16 t .. 16 t + 15 of each half, of rows g and g + 8 and of token g: the words of a 16-byte load are the
// operands of two MMAs.  That assigns the bytes of K to the MMA's K indices in another order than memory's, but to both operands
// alike, which a sum does not notice.
template <int TT, bool TAIL>
__global__ void __launch_bounds__(kShortWarps * 32) int8_short_kernel(const ShortParams q) {
    const SkinnyParams& p = q.s;
    extern __shared__ int red[];                                    // [warp][16 rows][8 TT tokens]
    constexpr int TOKENS = 8 * TT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = int(blockIdx.x) * kShortRows;
    const uint8_t* w0 = n0 + g < p.N ? p.B + int64_t(n0 + g) * p.ldb : nullptr;
    const uint8_t* w1 = n0 + g + 8 < p.N ? p.B + int64_t(n0 + g + 8) * p.ldb : nullptr;
    int acc[TT][4] = {};
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int UNROLL = TT <= 2 ? 4 : 2;
    for (int k0 = warp * 128; k0 < p.K; k0 += kShortWarps * 128 * UNROLL) {
        uint4 a[UNROLL][2][2];
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = k0 + u * kShortWarps * 128 + h * 64 + t * 16;
                a[u][h][0] = load16<TAIL>(w0 + k, w0 ? p.K - k : 0);
                a[u][h][1] = load16<TAIL>(w1 + k, w1 ? p.K - k : 0);
            }
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int k = k0 + u * kShortWarps * 128 + h * 64 + t * 16;
                uint4 b[TT];
#pragma unroll
                for (int c = 0; c < TT; c++) b[c] = load16<TAIL>(q.A + int64_t(8 * c + g) * q.lda + k, 8 * c + g < p.M ? p.K - k : 0);
#pragma unroll
                for (int c = 0; c < TT; c++) {
                    mma_s8(acc[c], a[u][h][0].x, a[u][h][1].x, a[u][h][0].y, a[u][h][1].y, b[c].x, b[c].y);
                    mma_s8(acc[c], a[u][h][0].z, a[u][h][1].z, a[u][h][0].w, a[u][h][1].w, b[c].z, b[c].w);
                }
            }
    }
    // result i of tile c: row g + 8 (i / 2), token 8 c + 2 t + i % 2
#pragma unroll
    for (int c = 0; c < TT; c++)
#pragma unroll
        for (int i = 0; i < 4; i++) red[(warp * TOKENS + 8 * c + 2 * t + (i & 1)) * kShortRows + g + 8 * (i >> 1)] = acc[c][i];
    __syncthreads();
    for (int e = threadIdx.x; e < TOKENS * kShortRows; e += kShortWarps * 32) {
        const int m = e / kShortRows, n = n0 + e % kShortRows;
        if (m >= p.M || n >= p.N) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kShortWarps; w++) sum += red[w * TOKENS * kShortRows + e];
        const float v = scaled(sum, p.a_sc[m], p.b_sc[n]);
        typed_out(p, [&](auto* D) { put(D + int64_t(m) * p.ldd + n, v); });
    }
}

// ---- launches -------------------------------------------------------------------------------

static cudaError_t launch_dependent(const void* kern, dim3 grid, int threads, int smem, cudaStream_t stream, void** args, int smem_attr, std::atomic<bool>* attr_set) {
    // the attribute belongs to the (kernel, device) pair: remember it per device, not per process
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_attr); e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelExC(&cfg, kern, args);
}

int int8_skinny_padded_rows(int M) { return (M + 15) / 16 * 16; }

// Slabs: every SM's share of N, in as few pieces of at most 128 rows as it takes.
static void skinny_plan(int M, int N, int sm_count, SkinnyParams& p) {
    const int per_sm = ((N + 127) / 128 + sm_count - 1) / sm_count;
    p.nb = int8_skinny_padded_rows(M);
    p.acc_cols = (p.nb + 31) / 32 * 32;
    p.rows = (N + sm_count * per_sm - 1) / (sm_count * per_sm);
    p.slabs = (N + p.rows - 1) / p.rows;
    p.w_bytes = (p.rows * 128 + 1023) / 1024 * 1024;
    // at least four stages of four blocks, or five of two: M=48 N=K=4096 (16 blocks fit) 11.7 us with 1 a stage, 10.7 with 2, 10.0 with 4;
    // M=48 N=28672 K=8192 (9 fit) 40.1, 40.6, 42.6
    const int blocks = (kSkinnySmem - 1024 - (128 * 128 - p.w_bytes)) / (p.w_bytes + p.nb * 128);       // the last block's MMAs read 128 rows
    p.group = blocks >= 16 ? 4 : (blocks >= 10 ? 2 : 1);
    p.stages = blocks / p.group < kSkinnyStages ? blocks / p.group : kSkinnyStages;
    // 256 KB, where a CTA has over 1 MB: M=16 N=28672 K=8192 38.7 us against 40.4 us; M=1 N=K=8192 16.9 us against 15.3 us
    p.prefetch = int64_t(p.rows) * per_sm * p.K > (1 << 20) ? 256 * 1024 / 128 : 0;
}

template <int GROUP>
static cudaError_t launch_skinny_t(const SkinnyArgs& a, SkinnyParams p) {
    static std::atomic<bool> attr_set[64] = {};
    CUtensorMap tmW = a.tmW, tmX = a.tmX;
    void* args[3] = {&tmW, &tmX, &p};
    return launch_dependent(reinterpret_cast<const void*>(int8_skinny_kernel<GROUP>), dim3(unsigned(p.slabs < a.sm_count ? p.slabs : a.sm_count)), kSkinnyThreads, kSkinnySmem,
                            a.stream, args, kSkinnySmem, attr_set);
}

template <int TT, bool TAIL>
static cudaError_t launch_short_t(const SkinnyArgs& a, const SkinnyParams& p) {
    static std::atomic<bool> attr_set[64] = {};
    ShortParams q{p, static_cast<const uint8_t*>(a.A), a.lda};
    void* args[1] = {&q};
    constexpr int smem = kShortWarps * kShortRows * 8 * TT * 4;
    return launch_dependent(reinterpret_cast<const void*>(int8_short_kernel<TT, TAIL>), dim3(unsigned((p.N + kShortRows - 1) / kShortRows)), kShortWarps * 32, smem,
                            a.stream, args, smem, attr_set);
}
template <bool TAIL>
static cudaError_t launch_short(const SkinnyArgs& a, const SkinnyParams& p) {
    if (a.M <= 8) return launch_short_t<1, TAIL>(a, p);
    if (a.M <= 16) return launch_short_t<2, TAIL>(a, p);
    return launch_short_t<4, TAIL>(a, p);
}

int int8_skinny_slab_rows(int M, int N, int sm_count) {
    SkinnyParams p;
    skinny_plan(M, N, sm_count, p);
    return p.rows;
}
// Long streams pay about 0.1 us for each 128-byte block of K, however few weight rows an SM has; short ones read the tokens again for
// every 16 rows.  Measured, long / short in us: M=1 N=2048 K=7168 9.4 / 5.7, M=32 10.1 / 9.3; M=8 N=K=4096 7.3 / 5.8, M=16 7.4 / 7.5;
// M=4 N=7168 K=2048 6.1 / 7.6; M=16 N=K=8192 14.0 / 19.6.
bool int8_skinny_short(int M, int N, int sm_count) { return M <= 32 && N <= (M <= 8 ? 32 : 16) * sm_count; }

cudaError_t launch_int8_skinny(const SkinnyArgs& a) {
    SkinnyParams p = {};
    p.a_sc = a.a_sc; p.b_sc = a.b_sc; p.D = a.D; p.ldd = a.ldd; p.B = static_cast<const uint8_t*>(a.B); p.ldb = a.ldb; p.M = a.M; p.N = a.N; p.K = a.K; p.out_dtype = a.out_dtype;
    p.status = a.status; p.wait_limit = api_wait_limit();
    if (int8_skinny_short(a.M, a.N, a.sm_count)) {
        return a.K % 16 ? launch_short<true>(a, p) : launch_short<false>(a, p);
    }
    skinny_plan(a.M, a.N, a.sm_count, p);
    switch (p.group) {
        case 4: return launch_skinny_t<4>(a, p);
        case 2: return launch_skinny_t<2>(a, p);
        default: return launch_skinny_t<1>(a, p);
    }
}

} // namespace tkb
