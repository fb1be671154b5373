// Row kernels in front of the 8-bit integer GEMM: per-token int8 quantization and the norms around a block.
//
// A CTA holds a row of K elements in registers, so every operator here is ONE pass over its data:
//   ROWS_QUANT  codes = rint(x * fl32(127 / amax)), sc = fl32(amax / 127), amax = max(max |x|, 2^-100)
//   ROWS_NORM   y = x * w_pre * rsqrt(mean(x^2) + eps)
//   ROWS_BLOCK  p = h * rsqrt(mean(h^2) + eps) * w_post (or h); r = residual_scale * x + gate * p; y from r as above
// y leaves as 16-bit values, or quantized like ROWS_QUANT, or both.  All of it is arithmetic in fp32: r and y are rounded
// to 16 bits only where they are stored, and y comes from the unrounded r, the codes from the unrounded y.
//
// Bound by HBM.  CTAs are persistent; while one works on a row in its registers, its next row is on the way to shared memory, so
// that loads are in flight all the time and cost no registers.  The largest |y| is rsqrt(..) times the largest |x * w_pre| (rounding
// is monotonic), so the sum of squares and the maximum share one reduction over the CTA.
//
// No counterpart in the reference, whose quantizers are block-scaled; the operators stand next to those (quantize.cu).
#include <atomic>
#include "ptx.cuh"
#include "internal.h"
#include "../../include/tkb200.h"

namespace tkb {

int api_fail(int code, const char* fmt, ...);          // api.cu
int api_device(int* sm_count, int** status);

enum RowsMode : int { ROWS_QUANT = 0, ROWS_NORM = 1, ROWS_BLOCK = 2 };
constexpr int kNormMaxK = 16384, kQuantMaxK = 65536;

struct RowsParams {
    const void *x, *h, *w_post, *gate, *w_pre;
    void *r, *y;
    int8_t* codes;
    float* sc;
    int64_t ldx, ldh, ldg, ldr, ldy, ldc;      // elements
    int M, K, rows_per_gate;
    float residual_scale, eps;
};

// Two 16-bit values of a register word
template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t down(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <> struct Pair<__half> {
    static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w))); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half(uint16_t(w >> 16))); }
    static __device__ __forceinline__ uint32_t down(float lo, float hi) { return pack_f16x2(lo, hi); }
};
// Two fp32 values in a register pair, which sm_100 adds and multiplies with one instruction
struct F2 { uint64_t v; };
__device__ __forceinline__ F2 f2(float lo, float hi) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
template <typename T> __device__ __forceinline__ F2 up2(uint32_t w) { return f2(Pair<T>::lo(w), Pair<T>::hi(w)); }
template <typename T> __device__ __forceinline__ uint32_t down2(F2 a) { float lo, hi; split(a, lo, hi); return Pair<T>::down(lo, hi); }
// max(|m|, |a|, |b|); a NaN stays one
__device__ __forceinline__ float max_abs3(float m, float a, float b) { float d; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b)); return d; }

// The elements of a row that a thread holds, and how it reaches them in memory, W at a time:
//   W = 8  groups of 8 in 16-byte accesses: K, the pitches and the bases allow it
//   W = 2  pairs in 4-byte accesses, for odd K or pitches: in a row that begins in the middle of a word the pairs begin one
//          element earlier (`shift` = 1) in all of the call's row tensors alike
//   W = 1  single elements, where the tensors begin differently
template <int V, int W>
struct Slots {
    static constexpr int E = 8 * V;
    static __device__ __forceinline__ int at(int j, int shift) { return (int(threadIdx.x) + (j / W) * int(blockDim.x)) * W + j % W - (W == 2 ? shift : 0); }
    // a row tensor's elements into the thread's own words of shared memory, asynchronously where the access is 4 bytes or more
    static __device__ __forceinline__ void fetch(const uint16_t* row, int K, int shift, uint32_t slot) {
        if constexpr (W == 8) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (at(8 * i, 0) < K)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + (i * blockDim.x + threadIdx.x) * 16), "l"(row + at(8 * i, 0)) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const int e0 = at(2 * i, shift), e1 = at(2 * i + 1, shift);
                const uint32_t dst = slot + (i * blockDim.x + threadIdx.x) * 4;
                if constexpr (W == 2) {
                    if (e0 >= 0 && e1 < K) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(row + e0) : "memory");
                    if (e1 == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(uint32_t(row[0]) << 16) : "memory");
                    if (e0 == K - 1) asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(uint32_t(row[e0])) : "memory");
                } else if (e0 < K) {
                    asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(row[e0] | (e1 < K ? uint32_t(row[e1]) << 16 : 0u)) : "memory");
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    static __device__ __forceinline__ void take(uint32_t slot, int K, int shift, uint32_t (&w)[E / 2]) {
        if constexpr (W == 8) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                w[4 * i] = w[4 * i + 1] = w[4 * i + 2] = w[4 * i + 3] = 0;
                if (at(8 * i, 0) < K)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                                 : "r"(slot + (i * blockDim.x + threadIdx.x) * 16)
                                 : "memory");
            }
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                w[i] = 0;
                if (at(2 * i, shift) < K) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(slot + (i * blockDim.x + threadIdx.x) * 4) : "memory");
            }
        }
    }
    // group g (8 elements: 4 words) of a tensor that every row reads (weights, gates): from L1, and again where it is needed
    // again, rather than kept in registers
    static __device__ __forceinline__ void peek(const uint16_t* row, int K, int shift, int g, uint32_t (&w)[4]) {
        if constexpr (W == 8) {
            w[0] = w[1] = w[2] = w[3] = 0;
            if (at(8 * g, 0) < K)
                asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(row + at(8 * g, 0)));
        } else {
            // outside the row any element will do: it meets a zero
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e0 = min(max(at(8 * g + 2 * i, shift), 0), K - 1), e1 = min(at(8 * g + 2 * i + 1, shift), K - 1);
                w[i] = __ldg(row + e0) | uint32_t(__ldg(row + e1)) << 16;
            }
        }
    }
    static __device__ __forceinline__ void store(uint16_t* row, int K, int shift, const uint32_t (&w)[E / 2]) {
        if constexpr (W == 8) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (at(8 * i, 0) < K) *reinterpret_cast<uint4*>(row + at(8 * i, 0)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                const int e0 = at(2 * i, shift), e1 = at(2 * i + 1, shift);
                if constexpr (W == 2) {
                    if (e0 >= 0 && e1 < K) *reinterpret_cast<uint32_t*>(row + e0) = w[i];
                    if (e1 == 0) row[0] = uint16_t(w[i] >> 16);
                    if (e0 == K - 1) row[e0] = uint16_t(w[i]);
                } else {
                    if (e0 < K) row[e0] = uint16_t(w[i]);
                    if (e1 < K) row[e1] = uint16_t(w[i] >> 16);
                }
            }
        }
    }
};

__device__ __forceinline__ float warp_sum(float s) {
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
__device__ __forceinline__ float warp_max_abs(float m) {
    float d;
    asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(m));
    return d;
}
// Sum of s and maximum of m >= 0 (or NaN) over the CTA, the same values in every thread.  `part` is shared memory that no thread
// can still be reading: the CTA has passed a barrier since it last used it.
template <bool SUM, bool MAX>
__device__ __forceinline__ void cta_reduce(float& s, float& m, float2* part) {
    const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (SUM) s = warp_sum(s);
    if (MAX) m = warp_max_abs(m);
    if (nw == 1) return;
    if (lane == 0) part[threadIdx.x >> 5] = make_float2(s, m);
    __syncthreads();
    const float2 q = lane < nw ? part[lane] : make_float2(0.f, 0.f);
    if (SUM) s = warp_sum(q.x);
    if (MAX) m = warp_max_abs(q.y);
}

// Steps and int8 codes of a row of fp32 values whose largest magnitude is m (NaN if there is one); value(i) gives pair i.  A code is
// the halves-to-even rounding of the exact product value * inv: the fused multiply-add rounds once, to the integer grid that adding
// 1.5 * 2^23 leaves, and the low byte is the two's complement of the code.  |value| <= m, hence |code| <= 127.  A row that holds an
// infinity or a NaN has step NaN and codes 0: its products are NaN, and no garbage is taken for a number.
template <int V, int W, typename F>
__device__ __forceinline__ void quantize_row(const RowsParams& p, int row, int shift, float m, F value) {
    using S = Slots<V, W>;
    const bool fine = m < __uint_as_float(0x7f800000u);
    const float amax = fmaxf(m, 0x1p-100f);
    const float inv = __fdiv_rn(127.0f, amax);
    if (threadIdx.x == 0) p.sc[row] = fine ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
    int8_t* out = p.codes + int64_t(row) * p.ldc;
    const F2 inv2 = f2(inv, inv), grid = f2(12582912.0f, 12582912.0f);
    // the codes of pair i in bits 0-7 and 8-15
    auto codes = [&](int i) {
        float lo, hi;
        split(fma2(value(i), inv2, grid), lo, hi);
        return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x0040);
    };
    if constexpr (W == 8) {
#pragma unroll
        for (int g = 0; g < V; g++) {
            uint32_t w0 = __byte_perm(codes(4 * g), codes(4 * g + 1), 0x5410), w1 = __byte_perm(codes(4 * g + 2), codes(4 * g + 3), 0x5410);
            if (!fine) w0 = w1 = 0;
            if (S::at(8 * g, 0) < p.K) *reinterpret_cast<uint2*>(out + S::at(8 * g, 0)) = make_uint2(w0, w1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * V; i++) {
            const uint32_t c = fine ? codes(i) : 0u;
            const int e0 = S::at(2 * i, shift), e1 = S::at(2 * i + 1, shift);
            if (e0 >= 0 && e0 < p.K) out[e0] = int8_t(c);
            if (e1 < p.K) out[e1] = int8_t(c >> 8);
        }
    }
}

template <typename T, int MODE, int V, int W, int THREADS>
__global__ void __launch_bounds__(THREADS) rows_kernel(const RowsParams p) {
    using S = Slots<V, W>;
    constexpr int P = 4 * V;                                      // pairs of elements of a thread
    extern __shared__ __align__(16) uint8_t slots[];
    __shared__ float2 part[2][2][32];
    const int K = p.K;
    const uint32_t slot_x = smem_u32(slots), slot_h = slot_x + blockDim.x * V * 16;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto row_of = [](const void* base, int64_t pitch, int row) { return static_cast<const uint16_t*>(base) + int64_t(row) * pitch; };
    auto shift_of = [&](int row) { return W == 2 ? int(reinterpret_cast<uintptr_t>(row_of(p.x, p.ldx, row)) >> 1) & 1 : 0; };
    // (r may be x: a row is written by the CTA that has read it)
    auto fetch = [&](int row, int shift) {
        if (MODE == ROWS_BLOCK) S::fetch(row_of(p.h, p.ldh, row), K, shift, slot_h);
        S::fetch(row_of(p.x, p.ldx, row), K, shift, slot_x);
    };
    int row = blockIdx.x, shift = shift_of(row), turn = 0;
    fetch(row, shift);
    while (true) {
        const int next = row + int(gridDim.x), next_shift = shift_of(next < p.M ? next : row);
        uint32_t x[P];
        float s = 0.f, m = 0.f;
        asm volatile("cp.async.wait_all;" ::: "memory");         // this thread reads only what it has fetched itself: no barrier
        S::take(slot_x, K, shift, x);
        if constexpr (MODE == ROWS_QUANT) {
            if (next < p.M) fetch(next, next_shift);
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < P; i++) bits = __vmaxu2(bits, x[i] & 0x7fff7fffu);      // magnitudes order like their bits, NaN above all
            m = Pair<T>::lo(max(bits & 0xffffu, bits >> 16));
            cta_reduce<false, true>(s, m, part[turn][0]);
            quantize_row<V, W>(p, row, shift, m, [&](int i) { return up2<T>(x[i]); });
        } else {
            F2 v[P];                                              // r * w_pre, then y
            F2 sum = f2(0.f, 0.f);
            float rstd = 1.0f;
            if constexpr (MODE == ROWS_BLOCK) {
                uint32_t h[P];
                S::take(slot_h, K, shift, h);
                if (next < p.M) fetch(next, next_shift);
#pragma unroll
                for (int i = 0; i < P; i++) v[i] = up2<T>(h[i]);
                if (p.w_post) {
#pragma unroll
                    for (int i = 0; i < P; i++) sum = fma2(v[i], v[i], sum);
                    float s1;
                    split(sum, s, s1);
                    s += s1;
                    cta_reduce<true, false>(s, m, part[turn][0]);
                    rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
                    sum = f2(0.f, 0.f);
                }
                const uint16_t* gate = p.gate ? row_of(p.gate, p.ldg, row / p.rows_per_gate) : nullptr;
#pragma unroll
                for (int g = 0; g < V; g++) {
                    uint32_t w[4];
                    if (p.w_post) {
                        S::peek(static_cast<const uint16_t*>(p.w_post), K, shift, g, w);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[4 * g + i] = mul2(mul2(v[4 * g + i], f2(rstd, rstd)), up2<T>(w[i]));
                    }
                    if (gate) {
                        S::peek(gate, K, shift, g, w);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[4 * g + i] = mul2(v[4 * g + i], up2<T>(w[i]));
                    }
#pragma unroll
                    for (int i = 4 * g; i < 4 * g + 4; i++) {
                        v[i] = fma2(f2(p.residual_scale, p.residual_scale), up2<T>(x[i]), v[i]);
                        x[i] = down2<T>(v[i]);
                    }
                }
                S::store(const_cast<uint16_t*>(row_of(p.r, p.ldr, row)), K, shift, x);
            } else {
                if (next < p.M) fetch(next, next_shift);
#pragma unroll
                for (int i = 0; i < P; i++) v[i] = up2<T>(x[i]);
            }
            if (MODE == ROWS_NORM || p.w_pre) {
#pragma unroll
                for (int g = 0; g < V; g++) {
                    uint32_t w[4];
                    S::peek(static_cast<const uint16_t*>(p.w_pre), K, shift, g, w);
#pragma unroll
                    for (int i = 4 * g; i < 4 * g + 4; i++) {
                        if (MODE == ROWS_BLOCK && W != 8) {
                            // outside the row h and x are zeros, but the gates and weights that they met may be no numbers
                            const int e0 = S::at(2 * i, shift), e1 = S::at(2 * i + 1, shift);
                            float lo, hi;
                            split(v[i], lo, hi);
                            v[i] = f2(e0 >= 0 && e0 < K ? lo : 0.f, e1 < K ? hi : 0.f);
                        }
                        sum = fma2(v[i], v[i], sum);
                        v[i] = mul2(v[i], up2<T>(w[i - 4 * g]));
                        float lo, hi;
                        split(v[i], lo, hi);
                        m = max_abs3(m, lo, hi);
                    }
                }
                float s1;
                split(sum, s, s1);
                s += s1;
                cta_reduce<true, true>(s, m, part[turn][1]);
                rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
                if (p.y) {
#pragma unroll
                    for (int i = 0; i < P; i++) x[i] = down2<T>(mul2(v[i], f2(rstd, rstd)));
                    S::store(const_cast<uint16_t*>(row_of(p.y, p.ldy, row)), K, shift, x);
                }
                if (p.codes) quantize_row<V, W>(p, row, shift, m * rstd, [&](int i) { return mul2(v[i], f2(rstd, rstd)); });
            }
        }
        if (next >= p.M) break;
        row = next; shift = next_shift; turn ^= 1;
    }
}

template <typename T, int MODE, int V, int W, int THREADS>
static cudaError_t launch_rows_w(const RowsParams& p, int threads, int sm_count, cudaStream_t s) {
    auto kern = rows_kernel<T, MODE, V, W, THREADS>;
    const int smem = threads * V * 16 * (MODE == ROWS_BLOCK ? 2 : 1);
    // CTAs of this size that an SM holds, asked for once for each device together with the shared memory
    static std::atomic<int> held[64][THREADS / 32 + 1] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int per_sm = held[dev][threads / 32].load(std::memory_order_acquire);
    if (per_sm == 0) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, THREADS * V * 16 * (MODE == ROWS_BLOCK ? 2 : 1));
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, smem);
        if (e != cudaSuccess) return e;
        held[dev][threads / 32].store(per_sm, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    const int64_t fit = int64_t(sm_count) * per_sm;
    cfg.gridDim = dim3(unsigned(p.M < fit ? p.M : fit)); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename T, int MODE, int V, int THREADS>
static cudaError_t launch_rows_v(const RowsParams& p, int width, int threads, int sm_count, cudaStream_t s) {
    switch (width) {
        case 8: return launch_rows_w<T, MODE, V, 8, THREADS>(p, threads, sm_count, s);
        case 2: return launch_rows_w<T, MODE, V, 2, THREADS>(p, threads, sm_count, s);
        default: return launch_rows_w<T, MODE, V, 1, THREADS>(p, threads, sm_count, s);
    }
}

// Threads of a CTA and groups of 8 elements for each: few rows get many threads, since one row after the other counts; many rows
// get up to 256, so that several CTAs share an SM and their reductions overlap.
template <typename T, int MODE>
static cudaError_t launch_rows_t(const RowsParams& p, int width, int sm_count, cudaStream_t s) {
    const int groups = (p.K + (width == 2 ? 1 : 0) + 7) / 8;
    auto threads = [&](int v) { return ((groups + v - 1) / v + 31) / 32 * 32; };
    if (p.M <= 2 * sm_count && groups <= 1024) return launch_rows_v<T, MODE, 1, 1024>(p, width, threads(1), sm_count, s);
    if (groups <= 256) return launch_rows_v<T, MODE, 1, 256>(p, width, threads(1), sm_count, s);
    if (groups <= 512) return launch_rows_v<T, MODE, 2, 256>(p, width, threads(2), sm_count, s);
    if (groups <= 1024) return launch_rows_v<T, MODE, 4, 256>(p, width, threads(4), sm_count, s);
    if (groups <= 2049) return launch_rows_v<T, MODE, 4, 544>(p, width, threads(4), sm_count, s);       // (2049: 16384 elements from the middle of a word)
    if constexpr (MODE == ROWS_QUANT) return launch_rows_v<T, MODE, 8, 1024>(p, width, threads(8), sm_count, s);
    return cudaErrorInvalidValue;
}

// ---- argument checks ------------------------------------------------------------------------
struct Span { const char* name; const void* ptr; int64_t pitch, width; };     // bytes; M rows

// Whether two row-strided buffers share a byte.  Column slices of one buffer (equal pitches) interleave without touching.
static bool overlap(const Span& a, const Span& b, int M) {
    if (!a.ptr || !b.ptr) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
    if (pa + uintptr_t((M - 1) * a.pitch + a.width) <= pb || pb + uintptr_t((M - 1) * b.pitch + b.width) <= pa) return false;
    if (a.pitch != b.pitch || M == 1) return true;
    const int64_t d = pb >= pa ? int64_t((pb - pa) % uintptr_t(a.pitch)) : a.pitch - 1 - int64_t((pa - pb - 1) % uintptr_t(a.pitch));      // (pb - pa) mod pitch
    return d < a.width || d + b.width > a.pitch;
}

static int rows_call(const char* what, RowsParams p, int mode, int dtype, void* stream) {
    if (dtype != TKB_DTYPE_BF16 && dtype != TKB_DTYPE_FP16) return api_fail(TKB_ERR_INVALID_ARG, "%s: dtype %d is neither TKB_DTYPE_BF16 nor TKB_DTYPE_FP16", what, dtype);
    if (p.M < 0 || p.K < 1) return api_fail(TKB_ERR_INVALID_ARG, "%s: need M >= 0 and K >= 1 (got M=%d K=%d)", what, p.M, p.K);
    const int max_k = mode == ROWS_QUANT ? kQuantMaxK : kNormMaxK;
    if (p.K > max_k) return api_fail(TKB_ERR_INVALID_ARG, "%s: K=%d is above %d, the longest row that one CTA holds", what, p.K, max_k);
    if ((p.codes == nullptr) != (p.sc == nullptr) && p.M > 0) return api_fail(TKB_ERR_INVALID_ARG, "%s: int8 codes and their scales come together", what);
    if (mode == ROWS_BLOCK && !(p.residual_scale >= -1e30f && p.residual_scale <= 1e30f)) return api_fail(TKB_ERR_INVALID_ARG, "%s: residual_scale must be a number", what);
    if (mode != ROWS_QUANT && !(p.eps >= 0.0f && p.eps < 1e30f)) return api_fail(TKB_ERR_INVALID_ARG, "%s: eps must be a number >= 0", what);
    if (p.M > 0) {
        if (!p.x) return api_fail(TKB_ERR_INVALID_ARG, "%s: null input", what);
        if (mode == ROWS_QUANT && !p.codes) return api_fail(TKB_ERR_INVALID_ARG, "%s: null output", what);
        if (mode == ROWS_NORM && (!p.w_pre || (!p.y && !p.codes))) return api_fail(TKB_ERR_INVALID_ARG, "%s: null weight or no output", what);
        if (mode == ROWS_BLOCK) {
            if (!p.h || !p.r) return api_fail(TKB_ERR_INVALID_ARG, "%s: null block output or residual output", what);
            if ((p.w_pre != nullptr) != (p.y != nullptr || p.codes != nullptr))
                return api_fail(TKB_ERR_INVALID_ARG, "%s: the second norm needs a weight and an output, or neither", what);
            if (p.gate && p.rows_per_gate < 1) return api_fail(TKB_ERR_INVALID_ARG, "%s: rows_per_gate must be positive", what);
        }
    }
    int64_t* const pitches[6] = {&p.ldx, &p.ldh, &p.ldg, &p.ldr, &p.ldy, &p.ldc};
    for (int64_t* ld : pitches) {
        if (*ld == 0) *ld = p.K;
        if (*ld < p.K) return api_fail(TKB_ERR_BAD_ALIGNMENT, "%s: a row pitch of %lld elements is below K=%d", what, (long long)*ld, p.K);
    }
    const void* const halves[7] = {p.x, p.h, p.w_post, p.gate, p.w_pre, p.r, p.y};
    uintptr_t bits = 0;
    for (const void* q : halves) bits |= reinterpret_cast<uintptr_t>(q);
    if (bits & 1u) return api_fail(TKB_ERR_BAD_ALIGNMENT, "%s: 16-bit tensors must be 2-byte aligned", what);
    if (reinterpret_cast<uintptr_t>(p.sc) & 3u) return api_fail(TKB_ERR_BAD_ALIGNMENT, "%s: scales must be 4-byte aligned", what);
    if (p.M == 0) return TKB_OK;
    // outputs may not touch anything else, but for r, which may be x itself
    const int64_t row = int64_t(p.K) * 2;
    const Span in[2] = {{"x", p.x, p.ldx * 2, row}, {"h", p.h, p.ldh * 2, row}};
    const Span out[3] = {{"r", p.r, p.ldr * 2, row}, {"y", p.y, p.ldy * 2, row}, {"codes", p.codes, p.ldc, p.K}};
    for (int i = 0; i < 3; i++) {
        for (const Span& s : in)
            if (overlap(out[i], s, p.M) && !(i == 0 && s.ptr == p.x && out[i].ptr == p.x && out[i].pitch == s.pitch))
                return api_fail(TKB_ERR_INVALID_ARG, "%s: output %s overlaps input %s", what, out[i].name, s.name);
        for (int k = 0; k < i; k++)
            if (overlap(out[i], out[k], p.M)) return api_fail(TKB_ERR_INVALID_ARG, "%s: outputs %s and %s overlap", what, out[i].name, out[k].name);
    }
    // 16-byte accesses where every row of every 16-bit tensor begins on 16 bytes (codes: on 8) and holds whole groups of 8; 4-byte
    // ones where the rows of all of them begin alike within a word
    const bool one = p.M == 1;
    auto whole = [&](const void* q, int64_t ld) { return !q || one || ld % 8 == 0; };
    auto alike = [&](const void* q, int64_t ld) { return !q || (((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.x)) & 2u) == 0 && (one || ((ld ^ p.ldx) & 1) == 0)); };
    int width = 1;
    if ((bits & 15u) == 0 && p.K % 8 == 0 && whole(p.x, p.ldx) && whole(p.h, p.ldh) && whole(p.r, p.ldr) && whole(p.y, p.ldy) && whole(p.codes, p.ldc) &&
        (reinterpret_cast<uintptr_t>(p.codes) & 7u) == 0 && (!p.gate || p.M <= p.rows_per_gate || p.ldg % 8 == 0))
        width = 8;
    else if (p.K < kQuantMaxK && alike(p.h, p.ldh) && alike(p.r, p.ldr) && alike(p.y, p.ldy))
        width = 2;
    int sm_count; int* status;
    if (int e = api_device(&sm_count, &status)) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
#define TKB_ROWS(MODE) (dtype == TKB_DTYPE_BF16 ? launch_rows_t<__nv_bfloat16, MODE>(p, width, sm_count, s) : launch_rows_t<__half, MODE>(p, width, sm_count, s))
    e = mode == ROWS_QUANT ? TKB_ROWS(ROWS_QUANT) : (mode == ROWS_NORM ? TKB_ROWS(ROWS_NORM) : TKB_ROWS(ROWS_BLOCK));
#undef TKB_ROWS
    if (e != cudaSuccess) return api_fail(TKB_ERR_CUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
    return TKB_OK;
}

} // namespace tkb

using namespace tkb;

extern "C" {

int tkb_int8_quantize(const void* A, int64_t lda, int dtype, void* codes, int64_t ldc, float* sc, int M, int K, void* stream) {
    RowsParams p = {};
    p.x = A; p.ldx = lda; p.codes = static_cast<int8_t*>(codes); p.ldc = ldc; p.sc = sc; p.M = M; p.K = K;
    return rows_call("int8_quantize", p, ROWS_QUANT, dtype, stream);
}

int tkb_rms_norm(const void* X, int64_t ldx, const void* W, void* Y, int64_t ldy, void* codes, int64_t ldc, float* sc, int dtype, int M, int K,
                 float eps, void* stream) {
    RowsParams p = {};
    p.x = X; p.ldx = ldx; p.w_pre = W; p.y = Y; p.ldy = ldy; p.codes = static_cast<int8_t*>(codes); p.ldc = ldc; p.sc = sc;
    p.M = M; p.K = K; p.eps = eps;
    return rows_call("rms_norm", p, ROWS_NORM, dtype, stream);
}

int tkb_block_norm(const void* H, int64_t ldh, const void* X, int64_t ldx, void* R, int64_t ldr, const void* W_post, const void* gate, int64_t ldg,
                   int rows_per_gate, float residual_scale, const void* W_pre, void* Y, int64_t ldy, void* codes, int64_t ldc, float* sc,
                   int dtype, int M, int K, float eps, void* stream) {
    RowsParams p = {};
    p.h = H; p.ldh = ldh; p.x = X; p.ldx = ldx; p.r = R; p.ldr = ldr; p.w_post = W_post; p.gate = gate; p.ldg = ldg;
    p.rows_per_gate = rows_per_gate; p.residual_scale = residual_scale; p.w_pre = W_pre; p.y = Y; p.ldy = ldy;
    p.codes = static_cast<int8_t*>(codes); p.ldc = ldc; p.sc = sc; p.M = M; p.K = K; p.eps = eps;
    return rows_call("block_norm", p, ROWS_BLOCK, dtype, stream);
}

} // extern "C"
