// Row kernels in front of the 8-bit integer GEMM: per-token int8 quantization and the norms around a block.
//
// A group of threads holds a row of K elements in registers, so every operator here is ONE pass over its data:
//   ROWS_QUANT  codes = rint(x * fl32(127 / amax)), sc = fl32(amax / 127), amax = max(max |x|, 2^-100)
//   ROWS_NORM   y = x * w_pre * rsqrt(mean(x^2) + eps)
//   ROWS_BLOCK  p = h * rsqrt(mean(h^2) + eps) * w_post (or h); r = residual_scale * x + gate * p; y from r as above
// y leaves as 16-bit values, or quantized like ROWS_QUANT, or both.  All of it is arithmetic in fp32: r and y are rounded
// to 16 bits only where they are stored, and y comes from the unrounded r, the codes from the unrounded y.
//
// Bound by HBM.  CTAs are persistent; while a group works on a row in its registers, its next row is on the way to shared memory, so
// that loads are in flight all the time and cost no registers.  The largest |y| is rsqrt(..) times the largest |x * w_pre| (rounding
// is monotonic), so the sum of squares and the maximum share one reduction.  Next after HBM comes the issue of instructions: fp32
// arithmetic on register pairs, and, where a CTA has many rows, weights in shared memory as fp32, for all groups of the CTA.
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
// How a thread's elements lie in memory:
//   ROWS_WHOLE    groups of 8 in 16-byte accesses: K, the pitches and the bases allow it
//   ROWS_SHIFTED  the same for rows that begin anywhere, but all of the call's row tensors alike within 16 bytes: groups begin `shift`
//                 elements before the row, its first and last group are partial
//   ROWS_SINGLE   single elements, where the tensors begin differently
enum RowsKind : int { ROWS_WHOLE = 0, ROWS_SHIFTED = 1, ROWS_SINGLE = 2 };
// How rows share a CTA: one row each (everything that depends on the row is uniform over the CTA); a row for each warp (no barriers);
// several groups of warps with a row each, which also share weights in shared memory; the same with rows dealt out in one piece for each
// CTA, which meets up to two gates, each in shared memory with the weights
enum RowsLayout : int { ROWS_ONE = 0, ROWS_WARPS = 1, ROWS_STAGED = 2, ROWS_GATES = 3 };
constexpr int kRowsSmem = 220 * 1024;          // dynamic shared memory that a CTA may have
constexpr int kNormMaxK = 16384, kQuantMaxK = 65536, kMaxRows = 1 << 30;

struct RowsParams {
    const void *x, *h, *w_post, *gate, *w_pre;
    void *r, *y;
    int8_t* codes;
    float* sc;
    int64_t ldx, ldh, ldg, ldr, ldy, ldc;      // elements
    int M, K, rows_per_gate;
    int chunk;                                 // ROWS_GATES: rows of a CTA
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
typedef float2 F2;
__device__ __forceinline__ F2 f2(float lo, float hi) { return make_float2(lo, hi); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { return __fmul2_rn(a, b); }
template <typename T> __device__ __forceinline__ F2 up2(uint32_t w) { return f2(Pair<T>::lo(w), Pair<T>::hi(w)); }
template <typename T> __device__ __forceinline__ uint32_t down2(F2 a) { return Pair<T>::down(a.x, a.y); }
// max(|m|, |a|, |b|); a NaN stays one
__device__ __forceinline__ float max_abs3(float m, float a, float b) { float d; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(a), "f"(b)); return d; }

// The 8 V elements of a row that a thread holds, in 4 V pairs
template <int V, int KIND>
struct Slots {
    static constexpr int P = 4 * V;
    static __device__ __forceinline__ int at(int j, int shift) {
        if (KIND == ROWS_SINGLE) return int(threadIdx.x) + j * int(blockDim.x);
        return (int(threadIdx.x) + (j >> 3) * int(blockDim.x)) * 8 + (j & 7) - (KIND == ROWS_SHIFTED ? shift : 0);
    }
    // address of words 4 g .. 4 g + 3 of the thread in a slot
    static __device__ __forceinline__ uint32_t word(uint32_t slot, int g) { return slot + (g * blockDim.x + threadIdx.x) * 16; }

    // A row into the thread's own words of shared memory, asynchronously where a group is whole.  Groups outside the row hold zeros:
    // they are cleared once, and one that lies in some rows and not in others is written anew for every row.
    static __device__ __forceinline__ void clear(int K, uint32_t slot) {
#pragma unroll
        for (int g = 0; g < V; g++)
            if (at(8 * g, 0) >= K) st_shared_v4(word(slot, g), 0u, 0u, 0u, 0u);
    }
    static __device__ __forceinline__ void fetch(const uint16_t* row, int K, int shift, uint32_t slot) {
#pragma unroll
        for (int g = 0; g < V; g++) {
            const int e = at(8 * g, shift);
            if (KIND == ROWS_WHOLE ? e < K : (KIND == ROWS_SHIFTED && e >= 0 && e + 8 <= K)) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(word(slot, g)), "l"(row + e) : "memory");
            } else if (KIND != ROWS_WHOLE && e < K + 8) {
                uint32_t w[4];
                gather(row, K, shift, g, w);
                st_shared_v4(word(slot, g), w[0], w[1], w[2], w[3]);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // the elements of group g that lie in the row, one by one; zeros for the others
    static __device__ __forceinline__ void gather(const uint16_t* row, int K, int shift, int g, uint32_t (&w)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e0 = at(8 * g + 2 * i, shift), e1 = at(8 * g + 2 * i + 1, shift);
            w[i] = e0 >= 0 && e0 < K ? row[e0] : 0u;
            if (e1 >= 0 && e1 < K) w[i] |= uint32_t(row[e1]) << 16;
        }
    }
    static __device__ __forceinline__ void take(uint32_t slot, uint32_t (&w)[P]) {
#pragma unroll
        for (int g = 0; g < V; g++)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[4 * g]), "=r"(w[4 * g + 1]), "=r"(w[4 * g + 2]), "=r"(w[4 * g + 3])
                         : "r"(word(slot, g))
                         : "memory");
    }
    static __device__ __forceinline__ void store(uint16_t* row, int K, int shift, const uint32_t (&w)[P]) {
#pragma unroll
        for (int g = 0; g < V; g++) {
            const int e = at(8 * g, shift);
            if (KIND == ROWS_WHOLE ? e < K : (KIND == ROWS_SHIFTED && e >= 0 && e + 8 <= K)) {
                *reinterpret_cast<uint4*>(row + e) = make_uint4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
            } else if (KIND != ROWS_WHOLE && e < K) {
#pragma unroll
                for (int i = 4 * g; i < 4 * g + 4; i++) {
                    const int e0 = at(2 * i, shift), e1 = at(2 * i + 1, shift);
                    if (e0 >= 0 && e0 < K) row[e0] = uint16_t(w[i]);
                    if (e1 >= 0 && e1 < K) row[e1] = uint16_t(w[i] >> 16);
                }
            }
        }
    }
    // group g of a vector that rows meet (weights, gates), from L1, and again where it is needed again; zeros outside the row
    template <typename T>
    static __device__ __forceinline__ void peek(const void* vec, int K, int shift, int g, F2 (&w)[4]) {
        uint32_t b[4] = {0u, 0u, 0u, 0u};
        const uint16_t* v = static_cast<const uint16_t*>(vec);
        const int e = at(8 * g, shift);
        if constexpr (KIND == ROWS_WHOLE) {
            if (e < K) asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "l"(v + e));
        } else if (KIND == ROWS_SHIFTED && e >= 0 && e + 8 <= K) {
#pragma unroll
            for (int i = 0; i < 4; i++) b[i] = v[e + 2 * i] | uint32_t(v[e + 2 * i + 1]) << 16;
        } else {
            gather(v, K, shift, g, b);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = up2<T>(b[i]);
    }
    // The same from shared memory as fp32, for the elements of all threads (zeros outside the row).  Layouts without bank conflicts:
    // WHOLE two halves, of the first and last 4 of every group (16-byte accesses); SHIFTED one word of padding for every 8.
    static __host__ __device__ __forceinline__ int staged_words(int threads) { return KIND == ROWS_SHIFTED ? (threads * V + 1) * 9 : threads * V * 8; }
    static __device__ __forceinline__ int staged_at(int e) {
        const int half = int(blockDim.x) * V * 4;
        return KIND == ROWS_WHOLE ? ((e >> 2) & 1) * half + (e >> 3) * 4 + (e & 3) : (KIND == ROWS_SHIFTED ? e + 8 + ((e + 8) >> 3) : e);
    }
    static __device__ __forceinline__ void staged(const float* vec, int shift, int g, F2 (&w)[4]) {
        const int c = int(threadIdx.x) + g * int(blockDim.x);
        if constexpr (KIND == ROWS_WHOLE) {
            const float4 a = *reinterpret_cast<const float4*>(vec + c * 4), b = *reinterpret_cast<const float4*>(vec + int(blockDim.x) * V * 4 + c * 4);
            w[0] = f2(a.x, a.y); w[1] = f2(a.z, a.w); w[2] = f2(b.x, b.y); w[3] = f2(b.z, b.w);
        } else if constexpr (KIND == ROWS_SHIFTED) {
            // staged_at(8 c - shift + j) = 9 (c + 1) - shift + j - (j < shift): one address for all but `shift`
            const float* q = vec + 9 * (c + 1) - shift;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = f2(q[2 * i - (2 * i < shift)], q[2 * i + 1 - (2 * i + 1 < shift)]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = f2(vec[at(8 * g + 2 * i, 0)], vec[at(8 * g + 2 * i + 1, 0)]);
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
// Sum of s and maximum of m >= 0 (or NaN) over the threads of a row (threadIdx.y), the same values in each.  `part` is shared memory
// that none of them can still be reading: they have passed a barrier since they last used it.
template <bool SUM, bool MAX, int LAYOUT>
__device__ __forceinline__ void row_reduce(float& s, float& m, float2* part) {
    const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    if (SUM) s = warp_sum(s);
    if (MAX) m = warp_max_abs(m);
    if (LAYOUT == ROWS_WARPS || nw == 1) return;
    if (lane == 0) part[threadIdx.x >> 5] = make_float2(s, m);
    // (a barrier chosen at run time takes all 16 of the CTA, so that no more than 4 CTAs fit an SM: only where rows share a CTA)
    if (LAYOUT >= ROWS_STAGED) asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.y), "r"(blockDim.x) : "memory");
    else __syncthreads();
    const float2 q = lane < nw ? part[lane] : make_float2(0.f, 0.f);
    if (SUM) s = warp_sum(q.x);
    if (MAX) m = warp_max_abs(q.y);
}

// Steps and int8 codes of a row of fp32 values whose largest magnitude is m (NaN if there is one); value(i) gives pair i.  A code is
// the halves-to-even rounding of the exact product value * inv: the fused multiply-add rounds once, to the integer grid that adding
// 1.5 * 2^23 leaves, and the low byte is the two's complement of the code.  |value| <= m, hence |code| <= 127.  A row that holds an
// infinity or a NaN has step NaN and codes 0: its products are NaN, and no garbage is taken for a number.
template <int V, int KIND, typename F>
__device__ __forceinline__ void quantize_row(const RowsParams& p, int row, int shift, float m, F value) {
    using S = Slots<V, KIND>;
    const bool fine = m < __uint_as_float(0x7f800000u);
    const float amax = fmaxf(m, 0x1p-100f);
    const float inv = __fdiv_rn(127.0f, amax);
    if (threadIdx.x == 0) p.sc[row] = fine ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
    int8_t* out = p.codes + int64_t(row) * p.ldc;
    const F2 inv2 = f2(inv, inv), grid = f2(12582912.0f, 12582912.0f);
    // the codes of pair i in bits 0-7 and 8-15
    auto codes = [&](int i) {
        const F2 c = fma2(value(i), inv2, grid);
        return __byte_perm(__float_as_uint(c.x), __float_as_uint(c.y), 0x0040);
    };
    if constexpr (KIND == ROWS_WHOLE) {
#pragma unroll
        for (int g = 0; g < V; g++) {
            uint32_t w0 = __byte_perm(codes(4 * g), codes(4 * g + 1), 0x5410), w1 = __byte_perm(codes(4 * g + 2), codes(4 * g + 3), 0x5410);
            if (!fine) w0 = w1 = 0;
            if (S::at(8 * g, 0) < p.K) *reinterpret_cast<uint2*>(out + S::at(8 * g, 0)) = make_uint2(w0, w1);
        }
    } else if constexpr (KIND == ROWS_SHIFTED) {
        // Whole words of codes: a thread's 8 begin d bytes before a word of the output, so its second word ends with the first d codes
        // of the next lane.  What no word covers (between two warps, at the row's ends) goes byte by byte.
        const int lane = threadIdx.x & 31;
        auto bytes = [&](uint32_t w, int e, int n) {
            for (int k = 0; k < n; k++, w >>= 8)
                if (e + k >= 0 && e + k < p.K) out[e + k] = int8_t(w);
        };
#pragma unroll
        for (int g = 0; g < V; g++) {
            const int e = S::at(8 * g, shift), d = -int(reinterpret_cast<uintptr_t>(out + e)) & 3;
            uint32_t w0 = __byte_perm(codes(4 * g), codes(4 * g + 1), 0x5410), w1 = __byte_perm(codes(4 * g + 2), codes(4 * g + 3), 0x5410);
            if (!fine) w0 = w1 = 0;
            const uint32_t w2 = __shfl_down_sync(0xffffffffu, w0, 1);
            const uint32_t a = __funnelshift_r(w0, w1, 8 * d), b = __funnelshift_r(w1, w2, 8 * d);
            if (!(lane > 0 && e + d - 4 >= 0 && e + d <= p.K)) bytes(w0, e, d);
            if (e + d >= 0 && e + d + 4 <= p.K) *reinterpret_cast<uint32_t*>(out + e + d) = a;
            else bytes(a, e + d, 4);
            if (lane < 31 && e + d + 4 >= 0 && e + d + 8 <= p.K) *reinterpret_cast<uint32_t*>(out + e + d + 4) = b;
            else bytes(b, e + d + 4, 4 - d);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4 * V; i++) {
            const uint32_t c = fine ? codes(i) : 0u;
            const int e0 = S::at(2 * i, shift), e1 = S::at(2 * i + 1, shift);
            if (e0 < p.K) out[e0] = int8_t(c);
            if (e1 < p.K) out[e1] = int8_t(c >> 8);
        }
    }
}

constexpr int rows_arrays(int mode) { return mode == ROWS_BLOCK ? 2 : 1; }         // row tensors read

template <typename T, int MODE, int V, int KIND, int THREADS, int LAYOUT>
__global__ void __launch_bounds__(THREADS) rows_kernel(const RowsParams p) {
    using S = Slots<V, KIND>;
    constexpr bool STAGED = LAYOUT >= ROWS_STAGED, GATES = LAYOUT == ROWS_GATES;
    // the row's place in its CTA, uniform over a warp
    const int ty = LAYOUT == ROWS_ONE ? 0 : __shfl_sync(0xffffffffu, int(threadIdx.y), 0), ny = LAYOUT == ROWS_ONE ? 1 : int(blockDim.y);
    constexpr int P = S::P;                                       // pairs of elements of a thread
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float2 part[2][2][THREADS / 32];
    const int K = p.K;
    const uint32_t slot_bytes = blockDim.x * V * 16;
    const uint32_t slot_x = smem_u32(smem) + ty * (rows_arrays(MODE) * slot_bytes), slot_h = slot_x + slot_bytes;
    const int staged_words = S::staged_words(blockDim.x);
    float* const staged_pre = reinterpret_cast<float*>(smem + ny * (rows_arrays(MODE) * slot_bytes));
    float* const staged_post = staged_pre + staged_words;       // with the gate, or two of them with one gate each
    float2* const my_part = &part[0][0][0] + ty * (blockDim.x / 32);      // of [2][2]: this row's warps
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // One pass over the grid: the next kernel may set itself up meanwhile.  Not beside a persistent grid: CTAs that come early take
    // the first places that fall free, unevenly over the SMs, and their rows are dealt out already (rms_norm after rms_norm, 16384 x
    // 7168: 84 us against 77 us).
    if (int(gridDim.x) * ny >= p.M) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto row_of = [](const void* base, int64_t pitch, int row) { return static_cast<const uint16_t*>(base) + int64_t(row) * pitch; };
    auto shift_of = [&](int row) { return KIND == ROWS_SHIFTED ? int(reinterpret_cast<uintptr_t>(row_of(p.x, p.ldx, row)) >> 1) & 7 : 0; };
    // (r may be x: a row is written by the threads that have read it)
    auto fetch = [&](int row, int shift) {
        if (MODE == ROWS_BLOCK) S::fetch(row_of(p.h, p.ldh, row), K, shift, slot_h);
        S::fetch(row_of(p.x, p.ldx, row), K, shift, slot_x);
    };
    const bool staged_gate = STAGED && p.gate && (GATES || p.rows_per_gate >= p.M);
    const int begin = int(blockIdx.x) * (GATES ? p.chunk : ny);
    const int end = GATES && begin + p.chunk < p.M ? begin + p.chunk : p.M, step = GATES ? ny : int(gridDim.x) * ny;
    const int first_gate = GATES ? begin / p.rows_per_gate : 0;
    int row = begin + ty, turn = 0;
    int shift = shift_of(row < end ? row : 0);
    S::clear(K, slot_x);
    if (MODE == ROWS_BLOCK) S::clear(K, slot_h);
    if (row < end) fetch(row, shift);
    if constexpr (STAGED) {
        const uint16_t* w_pre = static_cast<const uint16_t*>(p.w_pre);
        const uint16_t* w_post = static_cast<const uint16_t*>(p.w_post);
        const uint16_t* gate = static_cast<const uint16_t*>(p.gate) + int64_t(first_gate) * p.ldg;
        const bool two = GATES && int64_t(first_gate + 1) * p.rows_per_gate < end;
        const int first = KIND == ROWS_SHIFTED ? -8 : 0, last = int(blockDim.x) * V * 8;
        for (int e = int(ty * blockDim.x + threadIdx.x) + first; e < last; e += int(blockDim.x) * ny) {
            const bool in = e >= 0 && e < K;
            const int at = S::staged_at(e);
            if (p.w_pre) staged_pre[at] = in ? Pair<T>::lo(w_pre[e]) : 0.f;
            if (MODE == ROWS_BLOCK) {
                float c = in ? 1.f : 0.f;
                if (in && p.w_post) c = Pair<T>::lo(w_post[e]);
                if (two) staged_post[staged_words + at] = in ? c * Pair<T>::lo(gate[p.ldg + e]) : 0.f;
                if (in && staged_gate) c *= Pair<T>::lo(gate[e]);
                staged_post[at] = c;
            }
        }
        __syncthreads();
    }
    while (row < end) {
        const int next = row + step, next_shift = shift_of(next < end ? next : row);
        float2* const red = my_part + turn * 2 * (THREADS / 32);
        uint32_t x[P];
        float s = 0.f, m = 0.f;
        asm volatile("cp.async.wait_all;" ::: "memory");         // a thread reads only what it has fetched itself: no barrier
        S::take(slot_x, x);
        if constexpr (MODE == ROWS_QUANT) {
            if (next < end) fetch(next, next_shift);
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < P; i++) bits = __vmaxu2(bits, x[i] & 0x7fff7fffu);      // magnitudes order like their bits, NaN above all
            m = Pair<T>::lo(max(bits & 0xffffu, bits >> 16));
            row_reduce<false, true, LAYOUT>(s, m, red);
            quantize_row<V, KIND>(p, row, shift, m, [&](int i) { return up2<T>(x[i]); });
        } else {
            F2 v[P];                                              // r, r * w_pre, then y
            F2 sum = f2(0.f, 0.f);
            float rstd = 1.0f;
            auto total = [&]() {
                const float t = sum.x + sum.y;
                sum = f2(0.f, 0.f);
                return t;
            };
            if constexpr (MODE == ROWS_BLOCK) {
                uint32_t h[P];
                S::take(slot_h, h);
                if (next < end) fetch(next, next_shift);
#pragma unroll
                for (int i = 0; i < P; i++) v[i] = up2<T>(h[i]);
                if (p.w_post) {
#pragma unroll
                    for (int i = 0; i < P; i++) sum = fma2(v[i], v[i], sum);
                    s = total();
                    row_reduce<true, false, LAYOUT>(s, m, red);
                    rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
                }
                const F2 rstd2 = f2(rstd, rstd), scale2 = f2(p.residual_scale, p.residual_scale);
                const float* const post = GATES && row >= (first_gate + 1) * p.rows_per_gate ? staged_post + staged_words : staged_post;
                const uint16_t* gate = p.gate && !staged_gate ? row_of(p.gate, p.ldg, row / p.rows_per_gate) : nullptr;
#pragma unroll
                for (int g = 0; g < V; g++) {
                    F2 w[4];
                    if (STAGED || p.w_post) {
                        if (STAGED) S::staged(post, shift, g, w);
                        else S::template peek<T>(p.w_post, K, shift, g, w);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[4 * g + i] = mul2(mul2(v[4 * g + i], rstd2), w[i]);
                    }
                    if (gate) {
                        S::template peek<T>(gate, K, shift, g, w);
#pragma unroll
                        for (int i = 0; i < 4; i++) v[4 * g + i] = mul2(v[4 * g + i], w[i]);
                    }
#pragma unroll
                    for (int i = 4 * g; i < 4 * g + 4; i++) {
                        v[i] = fma2(scale2, up2<T>(x[i]), v[i]);
                        x[i] = down2<T>(v[i]);
                    }
                }
                S::store(const_cast<uint16_t*>(row_of(p.r, p.ldr, row)), K, shift, x);
            } else {
                if (next < end) fetch(next, next_shift);
#pragma unroll
                for (int i = 0; i < P; i++) v[i] = up2<T>(x[i]);
            }
            // (outside the row everything that v met is zero)
            if (MODE == ROWS_NORM || p.w_pre) {
#pragma unroll
                for (int g = 0; g < V; g++) {
                    F2 w[4];
                    if (STAGED) S::staged(staged_pre, shift, g, w);
                    else S::template peek<T>(p.w_pre, K, shift, g, w);
#pragma unroll
                    for (int i = 4 * g; i < 4 * g + 4; i++) {
                        sum = fma2(v[i], v[i], sum);
                        v[i] = mul2(v[i], w[i - 4 * g]);
                        m = max_abs3(m, v[i].x, v[i].y);
                    }
                }
                s = total();
                row_reduce<true, true, LAYOUT>(s, m, red + THREADS / 32);
                rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
                const F2 rstd2 = f2(rstd, rstd);
                if (p.y) {
#pragma unroll
                    for (int i = 0; i < P; i++) x[i] = down2<T>(mul2(v[i], rstd2));
                    S::store(const_cast<uint16_t*>(row_of(p.y, p.ldy, row)), K, shift, x);
                }
                if (p.codes) quantize_row<V, KIND>(p, row, shift, m * rstd, [&](int i) { return mul2(v[i], rstd2); });
            }
        }
        row = next; shift = next_shift; turn ^= 1;
    }
}

// Whether a call writes as many bytes as it reads and more than L2 takes up.  More loads in flight then only make HBM turn more
// often: 16384 x 7168 rms_norm with 3 rows on an SM 72 us, with 4 rows 84 us; block_norm with 2 rows 158 us, with 3 rows 175 us (and
// with int8 results, which write half, 65 against 60 us and 158 against 131 us).  So such calls keep about 48 KB (two row tensors: 64 KB)
// in flight on an SM.
static bool rows_turn(const RowsParams& p) { return p.y && !p.codes && int64_t(p.M) * p.K * (p.h ? 8 : 4) > (int64_t(256) << 20); }

template <int MODE, int V, int KIND, int LAYOUT>
static int rows_smem(int threads, int groups) {
    const int arrays = LAYOUT == ROWS_GATES ? 3 : (LAYOUT == ROWS_STAGED ? rows_arrays(MODE) : 0);       // of staged vectors
    return groups * threads * V * 16 * rows_arrays(MODE) + Slots<V, KIND>::staged_words(threads) * 4 * arrays;
}

template <typename T, int MODE, int V, int KIND, int THREADS, int LAYOUT>
static cudaError_t launch_rows_k(RowsParams p, int threads, int groups, int sm_count, cudaStream_t s) {
    auto kern = rows_kernel<T, MODE, V, KIND, THREADS, LAYOUT>;
    const int smem = rows_smem<MODE, V, KIND, LAYOUT>(threads, groups);
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev); e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    static std::atomic<bool> attr_set[64] = {};
    if (!attr_set[dev].load(std::memory_order_acquire)) {
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowsSmem); e != cudaSuccess) return e;
        attr_set[dev].store(true, std::memory_order_release);
    }
    // CTAs that an SM holds, remembered for each device and warps of a row (of which the rows of a CTA, nearly always, and the shared
    // memory follow), so that calls of several row lengths in turn do not ask again and again (int8_quantize of
    // 4 rows of 2048 and 7168 in turn, the host: 3.03 -> 2.90 us a call)
    static std::atomic<uint16_t> known[64][33] = {};                 // rows of a CTA, CTAs
    std::atomic<uint16_t>& memo = known[dev][threads / 32];
    int held = memo.load(std::memory_order_relaxed);
    if (held >> 8 != groups) {
        int per_sm = 0;
        if (cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads * groups, smem); e != cudaSuccess) return e;
        held = groups << 8 | per_sm;
        memo.store(uint16_t(held), std::memory_order_relaxed);
    }
    held &= 255;
    if (MODE == ROWS_NORM && LAYOUT == ROWS_ONE && rows_turn(p)) {
        const int rows = 48 * 1024 / smem < 2 ? 2 : 48 * 1024 / smem;
        if (held > rows) held = rows;
    }
    const int64_t fit = int64_t(sm_count) * held;
    if (LAYOUT == ROWS_GATES) p.chunk = int((p.M + fit - 1) / fit);
    const int64_t want = LAYOUT == ROWS_GATES ? (int64_t(p.M) + p.chunk - 1) / p.chunk : (int64_t(p.M) + groups - 1) / groups;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(want < fit ? want : fit)); cfg.blockDim = dim3(threads, groups); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

// Several gates are staged where sequences are no shorter than a CTA's rows (at most M / SMs), which then meet no more than two, and
// there is room beside as many rows as a CTA may have: gate rows read again and again against staged ones, in us: 4098 x 5001 with 6
// gates 59.0 / 51.5, 16384 x 7168 with 8 188 / 167, 8192 x 2048 with 16 38.4 / 26.6.  Where only fewer rows leave the room, rows count for
// more: 4096 x 12288 with 2, int8 result, 80 / 99.  The two round apart (one multiplies by the product w_post * gate, the other by one after
// the other), so the choice may not depend on which results are asked for, as the rows of a CTA do (rows_turn).
template <typename T, int MODE, int V, int KIND, int THREADS>
static cudaError_t launch_rows_staged(const RowsParams& p, int threads, int most, int sm_count, cudaStream_t s) {
    const int fit = most / threads < 15 ? most / threads : 15;                  // rows of a CTA (15: as many as it has barriers)
    const int turn = 64 * 1024 / (threads * V * 16 * rows_arrays(MODE));
    const int groups = rows_turn(p) && turn < fit ? (turn < 1 ? 1 : turn) : fit;
    if constexpr (MODE == ROWS_BLOCK)
        if (p.gate && p.rows_per_gate < p.M && p.rows_per_gate >= (p.M + sm_count - 1) / sm_count && rows_smem<MODE, V, KIND, ROWS_GATES>(threads, fit) <= kRowsSmem)
            return launch_rows_k<T, MODE, V, KIND, THREADS, ROWS_GATES>(p, threads, groups, sm_count, s);
    return launch_rows_k<T, MODE, V, KIND, THREADS, ROWS_STAGED>(p, threads, groups, sm_count, s);
}

// Few rows: as many threads for a row as it has groups of 8 elements (up to 1024), since the time from the first load to the last
// store counts.  Many rows: up to 4 groups for each thread, so that enough bytes are in flight and several rows share an SM.  Staging
// the weights pays where a row meets two of them or reaches them unaligned: 16384 x 7168 block_norm 161 -> 156 us, 4098 x 5001 90 ->
// 52 us, rms_norm 28.7 -> 24.9 us; an aligned rms_norm does better with its weights from L1 and more rows on an SM: 2048 x 8192 12.6
// against 15.8 us.
// One row for each CTA (the last branch): groups for each thread so that a CTA has up to 8 warps, 16 for the longest.  In us for rms_norm / with
// int8 result / int8_quantize, by this rule against others: 16384 x 512 a warp for each row 7.0 / 6.7 / 5.9, a CTA 8.4 / 9.5 / 6.4; 16384 x 2048 1
// group 27.6 / 31.5 / 17.7, 2 22.6 / 21.2 / 16.9; 16384 x 4096 2 groups 46.0 / 39.9 / 31.4, 1 56.0 / 63.3 / 33.5, 4 46.9 / 34.3 / 31.6; 16384 x
// 8192 4 groups 90.3 / 66.5 / 61.5, 2 92.4 / 76.4 / 62.5, 8 83.4 / 62.1 / 63.6; 8192 x 16384 4 groups 91.8 / 78.9 / 61.1, 2 92.5 / 84.3 / 69.4,
// 8 94.3 / 63.7 / 63.9; of few rows (400 x 8192) 4 groups 4.0 / 3.4 / 3.1, 8 4.8 / 3.9 / 3.3.
template <typename T, int MODE, int KIND>
static cudaError_t launch_rows_m(const RowsParams& p, int sm_count, cudaStream_t s) {
    const int n8 = (p.K + (KIND == ROWS_SHIFTED ? 7 : 0) + 7) / 8;
    auto threads = [&](int v) { return ((n8 + v - 1) / v + 31) / 32 * 32; };
    if constexpr (MODE == ROWS_QUANT && KIND == ROWS_SINGLE)         // (only rows that are too long to be shifted)
        return launch_rows_k<T, MODE, 8, KIND, 1024, ROWS_ONE>(p, threads(8), 1, sm_count, s);
    else if (p.M <= 2 * sm_count && n8 <= 1024)
        return launch_rows_k<T, MODE, 1, KIND, 1024, ROWS_ONE>(p, threads(1), 1, sm_count, s);
    else if constexpr (MODE == ROWS_BLOCK || (MODE == ROWS_NORM && KIND != ROWS_WHOLE)) {
        if (p.M <= 2 * sm_count) return launch_rows_k<T, MODE, 2, KIND, 1024, ROWS_ONE>(p, threads(2), 1, sm_count, s);
        if (n8 <= 64) return launch_rows_staged<T, MODE, 1, KIND, 768>(p, threads(1), 768, sm_count, s);
        // Two groups for each thread rather than four shorten the way from load to store, where as many bytes stay in flight: rows of
        // which a CTA holds one either way (4096 x 16384 102.8 -> 96.5 us; 16384 x 8192 with int8 result, 2 rows rather than 3, 148 -> 164
        // us); short shifted rows, of which four groups would make one or two warps (8190 x 1001 28.2 -> 24.2 us, 8190 x 1501 36.3 -> 32.5,
        // 4090 x 3001 30.7 -> 33.6); single elements, whose addresses do not fit the registers of four groups (4098 x 5001 136 -> 104 us)
        if (KIND == ROWS_SINGLE || n8 > 1536 || (KIND == ROWS_SHIFTED && n8 <= 192))
            return launch_rows_staged<T, MODE, 2, KIND, 1024>(p, threads(2), 1024, sm_count, s);
        if constexpr (KIND != ROWS_SINGLE) return launch_rows_staged<T, MODE, 4, KIND, 768>(p, threads(4), 768, sm_count, s);
        return cudaErrorInvalidValue;
    } else {
        if (n8 <= 64) return launch_rows_k<T, MODE, 2, KIND, 256, ROWS_WARPS>(p, 32, 8, sm_count, s);        // a warp for each row
        if (n8 <= 256) return launch_rows_k<T, MODE, 1, KIND, 256, ROWS_ONE>(p, threads(1), 1, sm_count, s);
        if (n8 <= 512) return launch_rows_k<T, MODE, 2, KIND, 256, ROWS_ONE>(p, threads(2), 1, sm_count, s);
        if (n8 <= 1024) return launch_rows_k<T, MODE, 4, KIND, 256, ROWS_ONE>(p, threads(4), 1, sm_count, s);
        if (n8 <= 2048) return launch_rows_k<T, MODE, 4, KIND, 512, ROWS_ONE>(p, threads(4), 1, sm_count, s);
        if constexpr (MODE == ROWS_QUANT) return launch_rows_k<T, MODE, 8, KIND, 1024, ROWS_ONE>(p, threads(8), 1, sm_count, s);
        return cudaErrorInvalidValue;
    }
}

template <typename T, int MODE>
static cudaError_t launch_rows_t(const RowsParams& p, int kind, int sm_count, cudaStream_t s) {
    switch (kind) {
        case ROWS_WHOLE: return launch_rows_m<T, MODE, ROWS_WHOLE>(p, sm_count, s);
        case ROWS_SHIFTED: return launch_rows_m<T, MODE, ROWS_SHIFTED>(p, sm_count, s);
        default: return launch_rows_m<T, MODE, ROWS_SINGLE>(p, sm_count, s);
    }
}

// ---- argument checks ------------------------------------------------------------------------
// Whether two row-strided buffers share a byte.  Column slices of one buffer (equal pitches) interleave without touching.
bool overlap(const Span& a, const Span& b) {
    if (!a.ptr || !b.ptr) return false;
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.ptr), pb = reinterpret_cast<uintptr_t>(b.ptr);
    if (pa + uintptr_t((a.rows - 1) * a.pitch + a.width) <= pb || pb + uintptr_t((b.rows - 1) * b.pitch + b.width) <= pa) return false;
    if (a.pitch != b.pitch || a.rows == 1 || b.rows == 1) return true;
    const int64_t d = pb >= pa ? int64_t((pb - pa) % uintptr_t(a.pitch)) : a.pitch - 1 - int64_t((pa - pb - 1) % uintptr_t(a.pitch));      // (pb - pa) mod pitch
    return d < a.width || d + b.width > a.pitch;
}

static int rows_call(const char* what, RowsParams p, int mode, int dtype, void* stream) {
    if (dtype != TKB_DTYPE_BF16 && dtype != TKB_DTYPE_FP16) return api_fail(TKB_ERR_INVALID_ARG, "%s: dtype %d is neither TKB_DTYPE_BF16 nor TKB_DTYPE_FP16", what, dtype);
    if (p.M < 0 || p.M > kMaxRows || p.K < 1) return api_fail(TKB_ERR_INVALID_ARG, "%s: need 0 <= M <= 2^30 and K >= 1 (got M=%d K=%d)", what, p.M, p.K);
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
    const int64_t row = int64_t(p.K) * 2, gates = p.gate ? (int64_t(p.M) + p.rows_per_gate - 1) / p.rows_per_gate : 1;
    const Span in[5] = {{"x", p.x, p.M, p.ldx * 2, row}, {"h", p.h, p.M, p.ldh * 2, row}, {"gate", p.gate, gates, p.ldg * 2, row},
                        {"the weight after the block", p.w_post, 1, row, row}, {"the weight", p.w_pre, 1, row, row}};
    const Span out[4] = {{"r", p.r, p.M, p.ldr * 2, row}, {"y", p.y, p.M, p.ldy * 2, row}, {"codes", p.codes, p.M, p.ldc, p.K},
                         {"scales", p.sc, 1, int64_t(p.M) * 4, int64_t(p.M) * 4}};
    for (int i = 0; i < 4; i++) {
        for (const Span& s : in)
            if (overlap(out[i], s) && !(i == 0 && s.ptr == p.x && out[i].ptr == p.x && out[i].pitch == s.pitch))
                return api_fail(TKB_ERR_INVALID_ARG, "%s: output %s overlaps input %s", what, out[i].name, s.name);
        for (int k = 0; k < i; k++)
            if (overlap(out[i], out[k])) return api_fail(TKB_ERR_INVALID_ARG, "%s: outputs %s and %s overlap", what, out[i].name, out[k].name);
    }
    // 16-byte accesses where every row of every 16-bit tensor begins on 16 bytes (codes: on 8) and holds whole groups of 8, or where the
    // rows of all of them begin alike within 16 bytes
    // (a longest row that begins inside a group would need one group more than there are)
    const bool one = p.M == 1;
    auto whole = [&](const void* q, int64_t ld) { return !q || one || ld % 8 == 0; };
    auto alike = [&](const void* q, int64_t ld) { return !q || (((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.x)) & 15u) == 0 && (one || ((ld ^ p.ldx) & 7) == 0)); };
    int kind = ROWS_SINGLE;
    if ((bits & 15u) == 0 && p.K % 8 == 0 && whole(p.x, p.ldx) && whole(p.h, p.ldh) && whole(p.r, p.ldr) && whole(p.y, p.ldy) && whole(p.codes, p.ldc) &&
        (reinterpret_cast<uintptr_t>(p.codes) & 7u) == 0 && (!p.gate || p.M <= p.rows_per_gate || p.ldg % 8 == 0))
        kind = ROWS_WHOLE;
    else if (p.K + 7 <= max_k && alike(p.h, p.ldh) && alike(p.r, p.ldr) && alike(p.y, p.ldy))
        kind = ROWS_SHIFTED;
    int sm_count; int* status;
    if (int e = api_device(&sm_count, &status)) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
#define TKB_ROWS(MODE) (dtype == TKB_DTYPE_BF16 ? launch_rows_t<__nv_bfloat16, MODE>(p, kind, sm_count, s) : launch_rows_t<__half, MODE>(p, kind, sm_count, s))
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
