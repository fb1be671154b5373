// Skinny-M ("decode") 8-bit integer GEMM: D[M, N] = A_sc[m] * B_sc[n] * sum_k A[m, k] * B[n, k] with M <= 128.
//
// Bound by streaming the N * K bytes of weights from HBM once.  Operands are swapped as in the NVFP4 decode kernel (decode.cu):
// weight rows are the MMA's M side (128 lanes), the tokens, padded to 16 / 32 / 64 / 128, its N side.  What matters is that every
// SM streams the same number of bytes without a gap:
//   * slabs have R <= 128 weight rows, R chosen so that they divide evenly over the SMs (a TMA box may have any number of rows;
//     the lanes past R multiply whatever is in shared memory and are not read).  N = 28672: two slabs of 97 rows for each SM;
//   * a CTA walks over its slabs; two accumulators in tensor memory, so that the epilogue of a slab overlaps the next one's loads;
//   * where N is too small for that, K is split over the CTAs of a cluster.  Each keeps its int32 partial tile in tensor memory
//     and, once all of its K is in, sends the rows of every 4 tokens to the CTA that owns them (group g: CTA g % split) through
//     distributed shared memory.  Integer sums do not depend on the order, so results do not depend on the split, and nothing
//     but D is written to global memory: calls on any number of streams and captured graphs share no scratch.
//   warp 0 = TMA producer, warp 1 = MMA issuer + tensor-memory owner, warps 2..5 = exchange and epilogue.
#include <atomic>
#include "ptx.cuh"
#include "internal.h"
#include "../../include/tkb200.h"

namespace tkb {

constexpr int kSkinnyStages = 16;
// Shared memory of a CTA.  Short streams of weights leave half an SM's, so that the next kernel's CTAs set themselves up, and ask L2
// for their weights, while this kernel ends: M=32 N=2048 K=7168 6.6 us against 10.7 us with the large one, whose CTAs (clusters,
// above all) only start once the SM is empty.  Long streams gain more from a deeper ring: M=16 N=28672 K=8192 38.9 us against 41.2.
constexpr int kSkinnySmemShort = 112 * 1024, kSkinnySmemLong = 208 * 1024;
constexpr int kSkinnyLongStream = 384 * 1024;       // bytes of weights of one CTA

template <int NB>
struct SkinnyCfg {
    static constexpr int X_BYTES = NB * 128;
    static constexpr int ACC_COLS = NB < 32 ? 32 : NB;   // of one accumulator
    static constexpr int TMEM_COLS = 2 * ACC_COLS;
    static constexpr int THREADS = 6 * 32;
    static constexpr int CHUNK = NB < 32 ? 16 : 32;      // accumulator columns read per tcgen05.ld
};

struct SkinnyParams {
    const float* a_sc; const float* b_sc;
    void* D; int64_t ldd;
    int M, N, kblk, out_dtype;
    int rows, slabs, split_log2;            // weight rows of a slab, slabs, log2 of the CTAs that share a slab's K
    int stages, w_bytes;                    // operand ring: stages, bytes from one stage's weights to the next's
    int prefetch;                           // K blocks of its weights that a CTA asks L2 for before the previous kernel is done
    int smem;                               // bytes of dynamic shared memory
    int* status;
    long long wait_limit;
};

__device__ __forceinline__ void tmem_ld_32x16_i(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// Cluster barrier of warps whose lanes may come out of a wait one after the other: the forms without .aligned, and the lanes
// together first.
__device__ __forceinline__ void split_arrive() { __syncwarp(); asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void split_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); __syncwarp(); }

__device__ __forceinline__ void store_out(const SkinnyParams& p, int m, int n, int sum, float a_sc, float b_sc) {
    const float v = __int2float_rn(sum) * a_sc * b_sc;
    const int64_t at = int64_t(m) * p.ldd + n;
    if (p.out_dtype == TKB_DTYPE_FP32) static_cast<float*>(p.D)[at] = v;
    else if (p.out_dtype == TKB_DTYPE_FP16) static_cast<__half*>(p.D)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p.D)[at] = __float2bfloat16_rn(v);
}

template <int NB>
__global__ void __launch_bounds__(SkinnyCfg<NB>::THREADS)
int8_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const SkinnyParams p) {
    using C = SkinnyCfg<NB>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[kSkinnyStages];
    __shared__ __align__(8) uint64_t bar_empty[kSkinnyStages];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nst = p.stages;
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sX = smem0;                                      // tokens first: an MMA reads 128 rows from a stage's weights on
    const uint32_t sW = smem0 + nst * C::X_BYTES;
    const uint32_t sRecv = smem0;                                   // split K: partial sums, once every ring of the cluster is idle
    const int split = 1 << p.split_log2;
    const int rank = split > 1 ? int(cluster_ctarank()) : 0;
    const int unit = int(blockIdx.x) >> p.split_log2, units = int(gridDim.x) >> p.split_log2;
    const int kb0 = (p.kblk * rank) >> p.split_log2, kb1 = (p.kblk * (rank + 1)) >> p.split_log2;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < nst; s++) { mbar_init(smem_u32(&bar_full[s]), 1); mbar_init(smem_u32(&bar_empty[s]), 1); }
        for (int b = 0; b < 2; b++) { mbar_init(smem_u32(&bar_acc_full[b]), 1); mbar_init(smem_u32(&bar_acc_empty[b]), 4); }
        fence_mbar_init();
        prefetch_tensormap(&tmW); prefetch_tensormap(&tmX);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&s_tmem_base), C::TMEM_COLS);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem_base;
    WaitCtx wc{&s_abort, p.status, p.wait_limit};

    if (warp == 0) {
        const bool leader = elect_one();
        uint32_t stage = 0, phase = 0, issued = 0;
        bool ok = true;
        if (leader) {
            // Weights may be asked for before the previous kernel is done, whoever writes them: this only moves lines into L2,
            // where a later write finds them.
            int left = p.prefetch;
            for (int slab = unit; slab < p.slabs && left > 0; slab += units)
                for (int kb = kb0; kb < kb1 && left > 0; kb++, left--) tma_prefetch_2d(&tmW, kb * 128, slab * p.rows);
            asm volatile("griddepcontrol.wait;" ::: "memory");      // the tokens come from the kernel before this one
            const uint32_t tx = uint32_t(p.rows) * 128u + C::X_BYTES;
            for (int slab = unit; slab < p.slabs && ok; slab += units)
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!mbar_wait(wc, smem_u32(&bar_empty[stage]), phase ^ 1)) { ok = false; break; }
                    const uint32_t full = smem_u32(&bar_full[stage]);
                    mbar_arrive_expect_tx(full, tx);
                    tma_load_2d(sW + stage * p.w_bytes, &tmW, full, kb * 128, slab * p.rows);
                    tma_load_2d(sX + stage * C::X_BYTES, &tmX, full, kb * 128, 0);
                    issued++;
                    if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
                }
            // the memory system is about to run dry: let the next kernel set itself up and ask for its weights
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        }
        __syncwarp();
        if (split > 1) split_arrive();      // (1): the epilogue warps arrive when this CTA's MMAs are done
        if (leader) {
            for (int s = 0; s < nst && ok; s++) {                   // stage releases of the MMA thread may still be in flight
                ok = mbar_wait(wc, smem_u32(&bar_empty[stage]), phase ^ 1);
                if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
            }
            if (!ok) drain_ring(bar_full, nst, issued, p.wait_limit);
        }
        __syncwarp();
        if (split > 1) { split_wait(); split_arrive(); split_wait(); }
    } else if (warp == 1) {
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, seg = 0;
            bool ok = true;
            for (int slab = unit; slab < p.slabs && ok; slab += units, seg++) {
                const uint32_t buf = seg & 1u;
                if (!mbar_wait(wc, smem_u32(&bar_acc_empty[buf]), ((seg >> 1) & 1u) ^ 1u)) { ok = false; break; }
                tc_fence_after();
                for (int kb = kb0; kb < kb1; kb++) {
                    if (!mbar_wait(wc, smem_u32(&bar_full[stage]), phase)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t a_desc = smem_desc_sw128(sW + stage * p.w_bytes);
                    const uint64_t b_desc = smem_desc_sw128(sX + stage * C::X_BYTES);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        mma_i8<1>(tmem_base + buf * C::ACC_COLS, a_desc + 2 * j, b_desc + 2 * j, idesc_int8(128, NB), (kb > kb0 || j > 0) ? 1u : 0u);
                    tc_commit<1>(smem_u32(&bar_empty[stage]));
                    if (++stage == uint32_t(nst)) { stage = 0; phase ^= 1; }
                }
                if (ok) tc_commit<1>(smem_u32(&bar_acc_full[buf]));
            }
        }
        __syncwarp();
        if (split > 1) { split_arrive(); split_wait(); split_arrive(); split_wait(); }
    } else {
        const int quarter = warp & 3;
        const int n_local = quarter * 32 + lane;
        asm volatile("griddepcontrol.wait;" ::: "memory");          // D may still be read, and the scales written, by the kernel before this one
        if (split == 1) {
            uint32_t seg = 0;
            for (int slab = unit; slab < p.slabs; slab += units, seg++) {
                const uint32_t buf = seg & 1u;
                const int n = slab * p.rows + n_local;
                const bool mine = n_local < p.rows && n < p.N;
                const float b_sc = mine ? __ldg(p.b_sc + n) : 0.f;
                const bool full = mbar_wait(wc, smem_u32(&bar_acc_full[buf]), (seg >> 1) & 1u);
                if (!__all_sync(0xffffffffu, full)) break;          // (lanes together: the loads below are the warp's)
                tc_fence_after();
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += C::CHUNK) {
                    if (c0 < p.M) {
                        uint32_t r[C::CHUNK];
                        const uint32_t at = tmem_base + (uint32_t(quarter * 32) << 16) + buf * C::ACC_COLS + c0;
                        if constexpr (C::CHUNK == 32) tmem_ld_32x32(at, r); else tmem_ld_32x16_i(at, r);
                        tmem_ld_wait();
                        if (mine) {
#pragma unroll
                            for (int i = 0; i < C::CHUNK; i++)
                                if (c0 + i < p.M) store_out(p, c0 + i, n, int(r[i]), __ldg(p.a_sc + c0 + i), b_sc);
                        }
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[buf]));
            }
        } else {
            // one slab for each cluster (units >= slabs)
            const int n = unit * p.rows + n_local;
            const bool mine = n_local < p.rows && n < p.N;
            const float b_sc = mine ? __ldg(p.b_sc + n) : 0.f;
            const bool ok = __all_sync(0xffffffffu, mbar_wait(wc, smem_u32(&bar_acc_full[0]), 0));
            tc_fence_after();
            split_arrive();                                         // (1)
            split_wait();                                           // every CTA's MMAs are done: the rings may be written over
            if (ok) {
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += C::CHUNK) {
                    if (c0 < p.M) {
                        uint32_t r[C::CHUNK];
                        const uint32_t at = tmem_base + (uint32_t(quarter * 32) << 16) + c0;
                        if constexpr (C::CHUNK == 32) tmem_ld_32x32(at, r); else tmem_ld_32x16_i(at, r);
                        tmem_ld_wait();
                        // tokens 4 g .. 4 g + 3 go to CTA g % split: [g / split][source CTA][weight row][4]
#pragma unroll
                        for (int i = 0; i < C::CHUNK; i += 4) {
                            const int g = (c0 + i) >> 2, owner = g & (split - 1);
                            if (c0 + i < p.M) {
                                const uint32_t dst = mapa(sRecv + uint32_t((g - owner + rank) * 128 + n_local) * 16, uint32_t(owner));
                                asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]) : "memory");
                            }
                        }
                    }
                }
            }
            tc_fence_before();
            split_arrive();                                         // (2)
            split_wait();                                           // the partial sums sent above are where they belong
            if (ok && mine) {
                for (int g = rank; 4 * g < p.M; g += split) {
                    const uint32_t src = sRecv + uint32_t((g - rank) * 128 + n_local) * 16;
                    int sum[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < 8; s++) {
                        if (s < split) {
                            int v[4];
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src + s * 2048));
#pragma unroll
                            for (int i = 0; i < 4; i++) sum[i] += v[i];
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (4 * g + i < p.M) store_out(p, 4 * g + i, n, sum[i], __ldg(p.a_sc + 4 * g + i), b_sc);
                }
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, C::TMEM_COLS);
    }
}

// How N and K are cut.  Slabs of a CTA's share of N, in as few pieces of at most 128 rows as it takes, if that share is a fair
// tile; else K is split, which keeps the tokens from being read by more CTAs than needed.  Cost of a 128-byte K block on a CTA in
// cycles: its bytes at an SM's share of the HBM rate (23 bytes a cycle; tokens, from L2, at twice that), but not below the 420
// that its barriers, copies and MMAs take to issue; an exchange of partial sums on top.  Measured, M=1 N=2048 K=7168: split 1 (14
// rows, 56 blocks) 12.5 us, 2 9.2 us, 4 6.6 us, 8 5.7 us.
static void skinny_plan(int M, int N, int K, int sm_count, int nb, SkinnyParams& p) {
    const int kblk = (K + 127) / 128;
    double best = 1e30;
    for (int lg = 0; lg <= 3; lg++) {
        const int split = 1 << lg;
        if (split > kblk) break;
        const int units = lg == 3 ? sm_count / 8 - 2 : (lg == 2 ? sm_count / 4 - 1 : sm_count / split);         // clusters that the GPCs hold at once
        const int per_unit = ((N + 127) / 128 + units - 1) / units;                                             // slabs
        if (lg > 0 && per_unit > 1) break;
        const int rows = (N + units * per_unit - 1) / (units * per_unit);
        const double block = (rows + 0.5 * M) * 128 / 23.0;
        const double cost = double(per_unit) * ((kblk + split - 1) / split) * (block < 420 ? 420 : block) + (lg ? 1400 + 10 * M : 0);
        if (cost < best) {
            best = cost;
            p.split_log2 = lg; p.rows = rows; p.slabs = (N + rows - 1) / rows;
            p.smem = double(per_unit) * rows * K / split >= kSkinnyLongStream ? kSkinnySmemLong : kSkinnySmemShort;
        }
    }
    p.kblk = kblk;
    p.w_bytes = (p.rows * 128 + 1023) / 1024 * 1024;
    p.stages = (p.smem - 1024 - (128 * 128 - p.w_bytes)) / (p.w_bytes + nb * 128);       // the last stage's MMAs read 128 rows
    if (p.stages > kSkinnyStages) p.stages = kSkinnyStages;
    p.prefetch = (p.smem == kSkinnySmemLong ? 256 : 64) * 1024 / (p.rows * 128);
}

template <int NB>
static cudaError_t launch_skinny_t(const SkinnyArgs& a, const SkinnyParams& p) {
    using C = SkinnyCfg<NB>;
    auto kern = int8_skinny_kernel<NB>;
    // the attribute belongs to the (kernel, device) pair: remember it per device, not per process
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSkinnySmemLong); e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev].store(true, std::memory_order_release);
    }
    const int split = 1 << p.split_log2;
    const int units = split > 1 || p.slabs < a.sm_count ? p.slabs : a.sm_count;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(units) * split); cfg.blockDim = dim3(C::THREADS); cfg.dynamicSmemBytes = p.smem; cfg.stream = a.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a.tmW, a.tmX, p);
}

int int8_skinny_padded_rows(int M) { return M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128)); }
int int8_skinny_slab_rows(int M, int N, int K, int sm_count) {
    SkinnyParams p;
    skinny_plan(M, N, K, sm_count, int8_skinny_padded_rows(M), p);
    return p.rows;
}

cudaError_t launch_int8_skinny(const SkinnyArgs& a) {
    SkinnyParams p = {};
    p.a_sc = a.a_sc; p.b_sc = a.b_sc; p.D = a.D; p.ldd = a.ldd; p.M = a.M; p.N = a.N; p.out_dtype = a.out_dtype;
    p.status = a.status; p.wait_limit = api_wait_limit();
    const int nb = int8_skinny_padded_rows(a.M);
    skinny_plan(a.M, a.N, a.K, a.sm_count, nb, p);
    switch (nb) {
        case 16: return launch_skinny_t<16>(a, p);
        case 32: return launch_skinny_t<32>(a, p);
        case 64: return launch_skinny_t<64>(a, p);
        default: return launch_skinny_t<128>(a, p);
    }
}

} // namespace tkb
