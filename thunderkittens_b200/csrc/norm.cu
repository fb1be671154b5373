// Row kernels in front of the 8-bit integer GEMM: per-token int8 quantization and the norms around a block.
//
// One CTA holds one row of K elements in registers, so every operator here is ONE pass over its data:
//   ROWS_QUANT  codes = rint(x * fl32(127 / amax)), sc = fl32(amax / 127), amax = max(max |x|, 2^-100)
//   ROWS_NORM   y = x * rsqrt(mean(x^2) + eps) * w_pre
//   ROWS_BLOCK  p = h * rsqrt(mean(h^2) + eps) * w_post (or h); r = residual_scale * x + gate * p; then y from r as above
// y leaves as 16-bit values, or quantized like ROWS_QUANT, or both.  All of it is arithmetic in fp32: r and y are rounded
// to 16 bits only where they are stored, and y comes from the unrounded r, the codes from the unrounded y.
//
// No counterpart in the reference, whose quantizers are block-scaled; the operators stand next to those (quantize.cu).
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
template <typename T, int E>
__device__ __forceinline__ float up(const uint32_t (&w)[E], int j) { return j & 1 ? Pair<T>::hi(w[j >> 1]) : Pair<T>::lo(w[j >> 1]); }

// The elements of a row that a thread holds.  VEC: V groups of 8 consecutive ones (16-byte accesses; K, the pitches and the
// bases allow them).  Otherwise 8 V single elements, one block of threads apart, so that a warp's accesses stay contiguous.
template <int V, bool VEC>
struct Slots {
    static constexpr int E = 8 * V;
    static __device__ __forceinline__ int at(int j) { return VEC ? (int(threadIdx.x) + (j >> 3) * int(blockDim.x)) * 8 + (j & 7) : int(threadIdx.x) + j * int(blockDim.x); }
    static __device__ __forceinline__ void load(const uint16_t* row, int K, uint32_t (&w)[E / 2]) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < V; i++) {
                uint4 q = make_uint4(0, 0, 0, 0);
                if (at(8 * i) < K) q = *reinterpret_cast<const uint4*>(row + at(8 * i));
                w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                w[i] = at(2 * i) < K ? row[at(2 * i)] : 0u;
                if (at(2 * i + 1) < K) w[i] |= uint32_t(row[at(2 * i + 1)]) << 16;
            }
        }
    }
    static __device__ __forceinline__ void store(uint16_t* row, int K, const uint32_t (&w)[E / 2]) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (at(8 * i) < K) *reinterpret_cast<uint4*>(row + at(8 * i)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < E / 2; i++) {
                if (at(2 * i) < K) row[at(2 * i)] = uint16_t(w[i]);
                if (at(2 * i + 1) < K) row[at(2 * i + 1)] = uint16_t(w[i] >> 16);
            }
        }
    }
};

// Sum / maximum over the CTA, the same value in every thread.  `part` is a shared array of 32 words that no reduction of this
// CTA has used since its last barrier but one, so that one barrier is enough.
template <bool MAX>
__device__ __forceinline__ uint32_t cta_reduce(uint32_t v, uint32_t* part) {
    auto warp = [](uint32_t u) {
        if constexpr (MAX) return __reduce_max_sync(0xffffffffu, u);
#pragma unroll
        for (int o = 16; o; o >>= 1) u = __float_as_uint(__uint_as_float(u) + __uint_as_float(__shfl_xor_sync(0xffffffffu, u, o)));
        return u;
    };
    const int lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    v = warp(v);
    if (nw == 1) return v;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp(lane < nw ? part[lane] : 0u);
}

// int8 codes of the fp32 values v and the step of their row.  The code is the halves-to-even rounding of the exact product
// v * inv: the fused multiply-add rounds once, to the integer grid that adding 1.5 * 2^23 leaves, and its low byte is the
// two's complement of the code.  |v| <= amax, hence |code| <= 127.  A row that holds an infinity or a NaN has step NaN and
// codes 0: its products are NaN, and no garbage is taken for a number.
template <int E, typename S, int V, bool VEC>
__device__ __forceinline__ void quantize_row(const float (&v)[E], const RowsParams& p, int row, uint32_t* part) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < E; j++) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);        // NaN > infinity > numbers
    m = cta_reduce<true>(m, part);
    const bool fine = m < 0x7f800000u;
    const float amax = fmaxf(__uint_as_float(m), 0x1p-100f);
    const float inv = __fdiv_rn(127.0f, amax);
    if (threadIdx.x == 0) p.sc[row] = fine ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7fc00000u);
    int8_t* out = p.codes + int64_t(row) * p.ldc;
    uint32_t c[E];
#pragma unroll
    for (int j = 0; j < E; j++) c[j] = fine ? __float_as_uint(__fmaf_rn(v[j], inv, 12582912.0f)) : 0u;
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = S::at(8 * i);
            uint32_t w[2];
#pragma unroll
            for (int k = 0; k < 2; k++)
                w[k] = __byte_perm(__byte_perm(c[8 * i + 4 * k], c[8 * i + 4 * k + 1], 0x0040), __byte_perm(c[8 * i + 4 * k + 2], c[8 * i + 4 * k + 3], 0x0040), 0x5410);
            if (e < p.K) *reinterpret_cast<uint2*>(out + e) = make_uint2(w[0], w[1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < E; j++)
            if (S::at(j) < p.K) out[S::at(j)] = int8_t(c[j]);
    }
}

template <typename T, int MODE, int V, bool VEC>
__global__ void __launch_bounds__(MODE == ROWS_QUANT && V == 8 ? 1024 : 256) rows_kernel(const RowsParams p) {
    using S = Slots<V, VEC>;
    constexpr int E = 8 * V;
    __shared__ uint32_t part[3][32];
    const int row = blockIdx.x, K = p.K;
    uint32_t x[E / 2];
    float v[E];
    S::load(static_cast<const uint16_t*>(p.x) + int64_t(row) * p.ldx, K, x);
    if constexpr (MODE == ROWS_BLOCK) {
        uint32_t h[E / 2], w[E / 2];
        S::load(static_cast<const uint16_t*>(p.h) + int64_t(row) * p.ldh, K, h);
#pragma unroll
        for (int j = 0; j < E; j++) v[j] = up<T>(h, j);
        if (p.w_post) {
            float s = 0.f;
#pragma unroll
            for (int j = 0; j < E; j++) s = fmaf(v[j], v[j], s);
            s = __uint_as_float(cta_reduce<false>(__float_as_uint(s), part[0]));
            const float rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
            S::load(static_cast<const uint16_t*>(p.w_post), K, w);
#pragma unroll
            for (int j = 0; j < E; j++) v[j] = v[j] * rstd * up<T>(w, j);
        }
        if (p.gate) {
            S::load(static_cast<const uint16_t*>(p.gate) + int64_t(row / p.rows_per_gate) * p.ldg, K, w);
#pragma unroll
            for (int j = 0; j < E; j++) v[j] *= up<T>(w, j);
        }
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            // elements past the row's end are made zeros, whatever rstd and the residual scale are
            v[j] = S::at(j) < K ? fmaf(p.residual_scale, up<T>(x, j), v[j]) : 0.f;
            v[j + 1] = S::at(j + 1) < K ? fmaf(p.residual_scale, up<T>(x, j + 1), v[j + 1]) : 0.f;
            h[j >> 1] = Pair<T>::down(v[j], v[j + 1]);
        }
        S::store(static_cast<uint16_t*>(p.r) + int64_t(row) * p.ldr, K, h);
        if (!p.w_pre) return;
    } else {
#pragma unroll
        for (int j = 0; j < E; j++) v[j] = up<T>(x, j);
    }
    if constexpr (MODE != ROWS_QUANT) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < E; j++) s = fmaf(v[j], v[j], s);
        s = __uint_as_float(cta_reduce<false>(__float_as_uint(s), part[1]));
        const float rstd = __frsqrt_rn(__fdiv_rn(s, float(K)) + p.eps);
        uint32_t w[E / 2];
        S::load(static_cast<const uint16_t*>(p.w_pre), K, w);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            v[j] = S::at(j) < K ? v[j] * rstd * up<T>(w, j) : 0.f;
            v[j + 1] = S::at(j + 1) < K ? v[j + 1] * rstd * up<T>(w, j + 1) : 0.f;
            x[j >> 1] = Pair<T>::down(v[j], v[j + 1]);
        }
        if (p.y) S::store(static_cast<uint16_t*>(p.y) + int64_t(row) * p.ldy, K, x);
        if (!p.codes) return;
    }
    quantize_row<E, S, V, VEC>(v, p, row, part[2]);
}

template <typename T, int MODE, int V>
static cudaError_t launch_rows_v(const RowsParams& p, bool vec, int threads, cudaStream_t s) {
    if (vec) rows_kernel<T, MODE, V, true><<<p.M, threads, 0, s>>>(p);
    else rows_kernel<T, MODE, V, false><<<p.M, threads, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int MODE>
static cudaError_t launch_rows_t(const RowsParams& p, bool vec, cudaStream_t s) {
    const int groups = (p.K + 7) / 8;
    int v = 1;
    while (v < 8 && groups > 256 * v) v *= 2;
    const int threads = ((groups + v - 1) / v + 31) / 32 * 32;
    switch (v) {
        case 1: return launch_rows_v<T, MODE, 1>(p, vec, threads, s);
        case 2: return launch_rows_v<T, MODE, 2>(p, vec, threads, s);
        case 4: return launch_rows_v<T, MODE, 4>(p, vec, threads, s);
        default: return launch_rows_v<T, MODE, 8>(p, vec, threads, s);
    }
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
    // 16-byte accesses where every row of every 16-bit tensor begins on 16 bytes (codes: on 8) and holds whole groups of 8
    const bool vec = (bits & 15u) == 0 && p.K % 8 == 0 && p.ldx % 8 == 0 && (!p.h || p.ldh % 8 == 0) && (!p.gate || p.ldg % 8 == 0) &&
                     (!p.r || p.ldr % 8 == 0) && (!p.y || p.ldy % 8 == 0) && (!p.codes || (p.ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(p.codes) & 7u) == 0));
    int sm_count; int* status;
    if (int e = api_device(&sm_count, &status)) return e;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
#define TKB_ROWS(MODE) (dtype == TKB_DTYPE_BF16 ? launch_rows_t<__nv_bfloat16, MODE>(p, vec, s) : launch_rows_t<__half, MODE>(p, vec, s))
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
