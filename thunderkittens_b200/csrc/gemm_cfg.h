// What the instances of the GEMM template (gemm.cu) are made of: tile, stage, shared-memory and tensor-memory sizes.
#pragma once
#include <cstdint>
#include "internal.h"

namespace tkb {

template <int KIND, int CTAS, int BN, int MH = 1>
struct GemmCfg {
    static_assert(CTAS == 1 || CTAS == 2, "");
    // (of a stage with two blocks of K only the single-CTA producer loads both, and B's second block is addressed as that of one CTA)
    static_assert(BN == 128 || BN == 256 || (BN == 64 && KIND == KIND_INT8 && CTAS == 1 && MH == 1), "N tile 64 is for int8 and single CTAs");
    // MH = 2 (dense kinds, CTA pairs, N tile 256): every CTA carries TWO 128-row halves of A per stage against the same B rows,
    // i.e. a 512 x 256 cluster tile with one accumulator per half: a third more FLOPs per byte that crosses from L2 into
    // shared memory than the 256 x 256 tile, which is what bounds the dense kernels
    static_assert(MH == 1 || (MH == 2 && CTAS == 2 && BN == 256 && (KIND == KIND_BF16 || KIND == KIND_FP8)), "");
    static constexpr int BM = 128 * CTAS * MH;            // rows of D per cluster tile
    static constexpr int MMA_M = 128 * CTAS;              // rows of one MMA instruction (per CTA pair)
    static constexpr int BN_CTA = BN / CTAS;              // rows of B each CTA loads
    // blocks of 128 bytes of K in a stage: two for N tile 64, where the loops of the two threads that feed it take longer than one (M=129
    // N=200 K=8192 13.5 us with one, 10.8 with two); past the end of K the second loads zeros
    static constexpr int GROUP = BN == 64 ? 2 : 1;
    static constexpr int KB = GROUP * (KIND == KIND_BF16 ? 64 : (KIND == KIND_NVFP4 ? 256 : 128));   // K elements per stage
    static constexpr int A_BYTES = GROUP * MH * 128 * 128;
    static constexpr int B_BYTES = GROUP * BN_CTA * 128;
    static constexpr int SF_CHUNKS = KIND == KIND_NVFP4 ? 4 : (KIND == KIND_MXFP8 ? 1 : 0);  // 512-byte chunks per 128 rows per stage
    static constexpr int SFA_BYTES = SF_CHUNKS * 512;
    static constexpr int SFB_BYTES = SF_CHUNKS * 512 * (BN / 128);
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
    static constexpr int EPI_WARPS = BN == 256 || (KIND == KIND_INT8 && BN == 128) ? 8 : 4;
    static constexpr int EPI_WARP_BYTES = 32 * 128;                  // one 32-row x 64-column bf16 store box per warp
    static constexpr int EPI_BYTES = EPI_WARPS * EPI_WARP_BYTES;
    static constexpr int SMEM_BUDGET = 227 * 1024 - 2048 - EPI_BYTES;
    static constexpr int STAGES_RAW = SMEM_BUDGET / STAGE_BYTES;
    static constexpr int STAGES = STAGES_RAW > 8 ? 8 : STAGES_RAW;
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + 2048;   // + alignment slack (base and staging area)
    static constexpr int THREADS = (2 + EPI_WARPS) * 32;
    static constexpr int COLS_PER_EPI_WARP = BN / (EPI_WARPS / 4);   // 128
    // tensor memory: accumulator at column 0, then rotating scale slots
    static constexpr int SFA_COLS = SF_CHUNKS * 4;                   // per stage
    static constexpr int SFB_COLS = SF_CHUNKS * 4 * (BN / 128);
    static constexpr int SF_SLOTS = 4;
    static constexpr int TMEM_COLS = 512;
    // two accumulators where they fit next to the scale slots (dense kinds, or N tile 128): the epilogue of tile i then overlaps
    // the MMAs of tile i + 1; otherwise one
    static constexpr int ACC_COLS = MH * BN;              // columns of one accumulator set (half h at column h * BN)
    static constexpr int ACC_BUFS = (2 * ACC_COLS + SF_SLOTS * (SFA_COLS + SFB_COLS) <= TMEM_COLS) ? 2 : 1;
    static constexpr int SF_BASE = ACC_BUFS * ACC_COLS;
    static_assert(ACC_BUFS * ACC_COLS + SF_SLOTS * (SFA_COLS + SFB_COLS) <= TMEM_COLS, "tensor memory overflow");
    static_assert(STAGES >= 3, "not enough pipeline stages");
    static constexpr uint32_t TX_BYTES = CTAS * STAGE_BYTES;
};

} // namespace tkb
