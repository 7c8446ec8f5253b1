// k_i8.cu -- rows of int8 with one scale each: from GGUF blocks (weights), from
// an RMS norm with the residual's addition, and from a gated activation. They
// feed the int8 matrix product in k_gemm_i8.cu.
//
// Each operator passes over a row's values twice: for the largest magnitude (and in
// the norm the sum of squares), then for the rounding to int8 (i8.cuh). A row that
// fits a CTA's registers is read once and kept there in between. Sums, scales and
// every value before the rounding are f32.
#include "i8.cuh"
#include "pdl.cuh"

#include <atomic>

namespace lm {
namespace {

constexpr uint32_t kWarpRows = 8;          // rows at a time of a CTA whose warps have one each
// The most threads of a CTA that keeps up to V pieces of E elements a thread in
// registers (1024 up to N elements, 16 without a norm's weights beside them), and
// whether the next row's pieces fit there too.
template <bool WARP, uint32_t E, uint32_t V, uint32_t N> constexpr uint32_t rows_threads() {
    return WARP ? 32 * kWarpRows : V * E <= N || E == 1 ? 1024 : 512;
}
template <uint32_t E, uint32_t V> constexpr bool rows_ahead() { return V * E <= (E == 1 ? 8 : 32); }

// ---------------------------------------------------------------- norm

struct NormArgs {
    const void* x;
    const void* resid;         // may be null
    void* sum;                 // may be null; may be x or resid with its pitch
    const float* w;
    int8_t* q;
    float* scale;
    uint64_t ld_x, ld_resid, ld_sum, ld_q;
    uint32_t rows, cols;
    float eps;
};

// 1 / sqrt(mean + eps) of a row's sum of squares. Squares leave f32's range long before
// the values do (|h| of 1.8e19; with an eps of next to nothing 1e-18 below): a sum that
// is infinite, or so small that its squares were rounded to multiples of 2^-149 that
// count, gives NaN, and the row's scale with it, instead of zeros or a wrong size. (Such
// rows summed again with scaled values cost the others 5 to 30 %: 1 x 2048 f32 1.7 -> 2.3
// us, 4096 x 4096 bf16 20.8 -> 22.1.)
constexpr float kLeastMean = 0x1p-120f;
__device__ __forceinline__ float rms_recip(float ss, uint32_t cols, float eps) {
    const float v = ss / (float)cols + eps;
    return v >= kLeastMean && v < INFINITY ? 1.0f / sqrtf(v) : NAN;
}

// h = x + resid in f32 (its rounding to the type is only for the stored sum),
// y = h / sqrt(mean(h^2) + eps) * w. One CTA a row. Each thread reads an
// element before the same thread overwrites it, in the second pass, so the sum
// may be stored over x or the residual.
template <typename T>
__global__ void __launch_bounds__(512) norm_i8_kernel(const NormArgs a) {
    __shared__ uint32_t red[64];
    const uint64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* r = a.resid ? static_cast<const T*>(a.resid) + row * a.ld_resid : nullptr;
    T* o = a.sum ? static_cast<T*>(a.sum) + row * a.ld_sum : nullptr;
    uint32_t m = 0;
    float ss = 0.f;
    for (uint32_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
        const float h = to_f32(x[i]) + (r ? to_f32(r[i]) : 0.f);
        ss = fmaf(h, h, ss);
        m = max(m, abs_bits(h * a.w[i]));
    }
    block_max_sum(m, ss, red);
    const float rstd = rms_recip(ss, a.cols, a.eps);
    const RowScale s = row_scale(__uint_as_float(m) * rstd);
    for (uint32_t i = threadIdx.x; i < a.cols; i += blockDim.x) {
        const float h = to_f32(x[i]) + (r ? to_f32(r[i]) : 0.f);
        if (o) o[i] = from_f32<T>(h);
        a.q[row * a.ld_q + i] = (int8_t)quant1(h * a.w[i] * rstd, s);
    }
    if (threadIdx.x == 0) a.scale[row] = s.scale();
}

// The same with a row in the registers of G threads (V vectors each), read once:
// h w of every element is kept from the first pass to the second. CTAs walk the
// rows with w in registers and the next row's loads in flight. Bound by memory: bf16
// 4096 x 4096 with residual and sum 20.9 us, 5.63 TB/s (two passes from L2 took 129
// us with the conversion that follows, this 82), f32 2048 x 8192 34.3 us, 6.37 TB/s;
// one row of 2048 1.8 us.
template <typename T, bool RESID, bool WARP, uint32_t E, uint32_t V>
__global__ void __launch_bounds__(rows_threads<WARP, E, V, 8>()) norm_i8_rows_kernel(const NormArgs a) {
    constexpr uint32_t R = WARP ? kWarpRows : 1;     // rows of a CTA at a time
    constexpr bool AHEAD = rows_ahead<E, V>();
    __shared__ uint32_t red[WARP ? 1 : 128];
    const uint32_t G = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31u : threadIdx.x;
    uint64_t row = (uint64_t)blockIdx.x * R + (WARP ? threadIdx.x >> 5 : 0);
    const uint64_t step = (uint64_t)gridDim.x * R;
    pdl_trigger();
    pdl_wait();
    float w[V][E];
#pragma unroll
    for (uint32_t j = 0; j < V; j++)
#pragma unroll
        for (uint32_t i = 0; i < E; i++) {
            const uint32_t at = (t + j * G) * E + i;
            w[j][i] = at < a.cols ? a.w[at] : 0.f;
        }
    Piece<T, E> x[V], r[V];
    auto load = [&](uint64_t at) {
        const T* px = static_cast<const T*>(a.x) + at * a.ld_x;
        const T* pr = static_cast<const T*>(a.resid) + at * a.ld_resid;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
            load_piece<T, E>(x[j], px, (t + j * G) * E, a.cols);
            if (RESID) load_piece<T, E>(r[j], pr, (t + j * G) * E, a.cols);
        }
    };
    if (AHEAD && row < a.rows) load(row);
    for (uint32_t turn = 0; row < a.rows; row += step, turn++) {
        if (!AHEAD) load(row);
        float hw[V][E];
        float top = 0.f, ss = 0.f;
        T* o = a.sum ? static_cast<T*>(a.sum) + row * a.ld_sum : nullptr;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
            piece_to_f32<T, E>(x[j], hw[j]);
            if (RESID) {
                float f[E];
                piece_to_f32<T, E>(r[j], f);
#pragma unroll
                for (uint32_t i = 0; i < E; i++) hw[j][i] += f[i];
            }
            if (o) store_piece<T, E>(o, (t + j * G) * E, a.cols, hw[j]);
#pragma unroll
            for (uint32_t i = 0; i < E; i++) {
                ss = fmaf(hw[j][i], hw[j][i], ss);
                hw[j][i] *= w[j][i];
                top = max_abs(top, hw[j][i]);
            }
        }
        if (AHEAD && row + step < a.rows) load(row + step);
        uint32_t m = abs_bits(top);
        row_max_sum<WARP>(m, ss, red, turn);
        const float rstd = rms_recip(ss, a.cols, a.eps);
        const RowScale s = row_scale(__uint_as_float(m) * rstd);
        float f = rstd * s.inv;
        if (!(s.plain && f < INFINITY)) {            // in two steps
#pragma unroll
            for (uint32_t j = 0; j < V; j++)
#pragma unroll
                for (uint32_t i = 0; i < E; i++) hw[j][i] = s.odd(hw[j][i] * rstd);
            f = s.inv;
        }
#pragma unroll
        for (uint32_t j = 0; j < V; j++) store_quant<E>(a.q + row * a.ld_q, (t + j * G) * E, a.cols, hw[j], f);
        if (t == 0) a.scale[row] = s.scale();
    }
}

// ---------------------------------------------------------------- gated activation

struct GluArgs {
    const void* gate;
    const void* up;            // may be null: act(gate) alone
    int8_t* q;
    float* scale;
    uint64_t ld_gate, ld_up, ld_q;
    uint32_t rows, cols, act;
};

// The activations of model.c:14-25 (and gpt2.c's gelu) times up, in f32, as
// x up / (1 + exp(-z)): SiLU's z is x; GELU's (1 + tanh u) / 2 is 1 / (1 + exp(-2 u)),
// which does not cancel for negative u. With h = exp(-z / 2) = 2^(-z log2 e / 2), the
// factor folded into z's constants, 1 / (1 + h h) is the square of a reciprocal root s,
// and x and up take one s each: where h h nears f32's limit (z = -88.7, beyond which
// 1 + exp(-z) is infinite and the result 0, as in model.c) the reciprocal itself would
// already be below f32's normal numbers, its root is far from there. Two approximate
// instructions, each of relative error 2^-22 that the squares double, and where h h
// counts (z < 0) |z| 2^-23 for SiLU from the argument's rounding (the product and the
// constant) and |z| 2^-22 for GELU (x x, the fused sum, the product and two constants), next
// to a result that is rounded to 8 bits. 26 instructions an element became 15 (4096 x
// 11008 bf16: 58 us with expf and an exact division).
__device__ __forceinline__ float root_sigmoid(float minus_half_z_log2e) {
    float h, s;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(h) : "f"(minus_half_z_log2e));
    asm("rsqrt.approx.ftz.f32 %0, %1;\n" : "=f"(s) : "f"(fmaf(h, h, 1.0f)));
    return s;
}
__device__ __forceinline__ float activate(float x, float up, uint32_t act) {
    constexpr float log2e = 1.4426950408889634f;
    if (act == LLAMINI_ACT_NONE) return x * up;
    constexpr float k = -0.79788456080286535587989211986876f * log2e;
    const float s = root_sigmoid(act == ACT_SILU ? x * (-0.5f * log2e) : x * fmaf(0.044715f * k, x * x, k));
    return (x * s) * (up * s);
}

template <typename T>
__global__ void __launch_bounds__(512) glu_i8_kernel(const GluArgs a) {
    __shared__ uint32_t red[64];
    const uint64_t row = blockIdx.x;
    const T* g = static_cast<const T*>(a.gate) + row * a.ld_gate;
    const T* u = a.up ? static_cast<const T*>(a.up) + row * a.ld_up : nullptr;
    uint32_t m = 0;
    float unused = 0.f;
    for (uint32_t i = threadIdx.x; i < a.cols; i += blockDim.x)
        m = max(m, abs_bits(activate(to_f32(g[i]), u ? to_f32(u[i]) : 1.f, a.act)));
    block_max_sum(m, unused, red);
    const RowScale s = row_scale(__uint_as_float(m));
    for (uint32_t i = threadIdx.x; i < a.cols; i += blockDim.x)
        a.q[row * a.ld_q + i] = (int8_t)quant1(activate(to_f32(g[i]), u ? to_f32(u[i]) : 1.f, a.act), s);
    if (threadIdx.x == 0) a.scale[row] = s.scale();
}

// The same with a row's values in the registers of G threads, read and
// activated once; the next row's loads are in flight meanwhile. Bound by memory and
// instruction issue (bf16 4096 x 11008 SiLU: 41.8 us, 5.39 TB/s; f32 2048 x 11008 33.1 us,
// 6.13 TB/s). Four CTAs an SM where a warp has a row of one piece a lane: 20000 x 256
// bf16 6.5 us, 7.3 with the three that more registers leave.
template <typename T, bool UP, bool WARP, uint32_t E, uint32_t V>
__global__ void __launch_bounds__(rows_threads<WARP, E, V, 16>(), V * E == 24 && V == 3 ? 2 : WARP && V == 1 ? 4 : 1) glu_i8_rows_kernel(const GluArgs a) {
    constexpr uint32_t R = WARP ? kWarpRows : 1;
    constexpr bool AHEAD = rows_ahead<E, V>();
    __shared__ uint32_t red[WARP ? 1 : 128];
    const uint32_t G = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31u : threadIdx.x;
    uint64_t row = (uint64_t)blockIdx.x * R + (WARP ? threadIdx.x >> 5 : 0);
    const uint64_t step = (uint64_t)gridDim.x * R;
    pdl_trigger();
    pdl_wait();
    Piece<T, E> g[V], u[V];
    auto load = [&](uint64_t at) {
        const T* pg = static_cast<const T*>(a.gate) + at * a.ld_gate;
        const T* pu = static_cast<const T*>(a.up) + at * a.ld_up;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
            load_piece<T, E>(g[j], pg, (t + j * G) * E, a.cols);
            if (UP) load_piece<T, E>(u[j], pu, (t + j * G) * E, a.cols);
        }
    };
    if (AHEAD && row < a.rows) load(row);
    for (uint32_t turn = 0; row < a.rows; row += step, turn++) {
        if (!AHEAD) load(row);
        float y[V][E];
        float top = 0.f, unused = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < V; j++) {
            piece_to_f32<T, E>(g[j], y[j]);
            float f[E];
            if (UP) piece_to_f32<T, E>(u[j], f);
            if (a.act == ACT_SILU) {                 // (one branch a piece, the same for all)
#pragma unroll
                for (uint32_t i = 0; i < E; i++) y[j][i] = activate(y[j][i], UP ? f[i] : 1.f, ACT_SILU);
            } else if (a.act == ACT_GELU) {
#pragma unroll
                for (uint32_t i = 0; i < E; i++) y[j][i] = activate(y[j][i], UP ? f[i] : 1.f, ACT_GELU);
            } else if (UP) {
#pragma unroll
                for (uint32_t i = 0; i < E; i++) y[j][i] *= f[i];
            }
#pragma unroll
            for (uint32_t i = 0; i < E; i++) top = max_abs(top, y[j][i]);
        }
        if (AHEAD && row + step < a.rows) load(row + step);
        uint32_t m = abs_bits(top);
        row_max_sum<WARP>(m, unused, red, turn);
        const RowScale s = row_scale(__uint_as_float(m));
        if (!s.plain) {
#pragma unroll
            for (uint32_t j = 0; j < V; j++)
#pragma unroll
                for (uint32_t i = 0; i < E; i++) y[j][i] = s.odd(y[j][i]);
        }
#pragma unroll
        for (uint32_t j = 0; j < V; j++) store_quant<E>(a.q + row * a.ld_q, (t + j * G) * E, a.cols, y[j], s.inv);
        if (t == 0) a.scale[row] = s.scale();
    }
}

// ---------------------------------------------------------------- weights

struct WeightArgs {
    const uint8_t* raw;
    int8_t* q;
    float* scale;
    uint64_t row_bytes, ld_q;
    uint32_t rows, cols;
    uint32_t seg_units;        // units of a segment of a row that fits shared memory
};

constexpr uint32_t kWSeg = 48 * 1024;      // raw bytes of a row staged at a time
constexpr uint32_t kWRow = 96 * 1024;      // longest row that is staged whole
constexpr uint32_t kWSlack = 64;           // behind it: the offset modulo 16, and words_at's read past a block
constexpr uint32_t kWThreads = 256;

// NW little-endian words from a 2-byte aligned address in shared memory (the
// aligned words around it; reads up to two bytes past the range).
template <int NW>
__device__ __forceinline__ void words_at(const uint8_t* p, uint32_t* w) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    const uint32_t* b = reinterpret_cast<const uint32_t*>(a & ~uintptr_t(3));
    const uint32_t s = (uint32_t)(a & 2u) * 8u;
    uint32_t prev = b[0];
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const uint32_t nx = b[i + 1];
        w[i] = __funnelshift_r(prev, nx, s);
        prev = nx;
    }
}
// Byte 0 .. 3 of a word as f32, exact: behind 0x4B it is the mantissa of 2^23 + b.
// `off` is 2^23, or more to subtract a bias on the way.
__device__ __forceinline__ float byte_f32(uint32_t word, int k, float off) {
    return __fsub_rn(__uint_as_float(__byte_perm(word, 0x4B000000u, 0x7440 | k)), off);
}
__device__ __forceinline__ float half_at(const uint8_t* p) {
    return __half2float(*reinterpret_cast<const __half*>(p));
}

// Elements 32 u .. 32 u + 31 of a row whose bytes (from the first block of
// the staged segment on) are at `row`, in their own order, bit-identical to
// gguf.c:409-594: products and sums are rounded as there (a fused multiply-add
// only where the product is exact).
template <uint32_t T>
__device__ __forceinline__ void unit_weights(const uint8_t* row, uint32_t u, float* y) {
    uint32_t w[8];
    constexpr float M = 8388608.0f;                  // 2^23
    constexpr uint32_t nib = 0x0F0F0F0Fu;
    if constexpr (T == GGML_TYPE_Q8_0) {
        const uint8_t* b = row + (size_t)u * 34;
        const float d = half_at(b);
        words_at<8>(b + 2, w);
#pragma unroll
        for (int i = 0; i < 32; i++) y[i] = __fmul_rn(byte_f32(w[i >> 2] ^ 0x80808080u, i & 3, M + 128.0f), d);
    } else if constexpr (T == GGML_TYPE_Q4_0) {
        const uint8_t* b = row + (size_t)u * 18;
        const float d = half_at(b);
        words_at<4>(b + 2, w);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            y[i] = __fmul_rn(byte_f32(w[i >> 2] & nib, i & 3, M + 8.0f), d);
            y[i + 16] = __fmul_rn(byte_f32((w[i >> 2] >> 4) & nib, i & 3, M + 8.0f), d);
        }
    } else if constexpr (T == GGML_TYPE_Q4_1) {
        // d q is exact (11 + 4 bits), so the fused sum rounds where gguf.c's does
        const uint8_t* b = row + (size_t)u * 20;
        const float d = half_at(b), m = half_at(b + 2);
        words_at<4>(b + 4, w);
#pragma unroll
        for (int i = 0; i < 16; i++) {
            y[i] = fmaf(byte_f32(w[i >> 2] & nib, i & 3, M), d, m);
            y[i + 16] = fmaf(byte_f32((w[i >> 2] >> 4) & nib, i & 3, M), d, m);
        }
    } else if constexpr (T == GGML_TYPE_Q5_0) {
        const uint8_t* b = row + (size_t)u * 22;
        const float d = half_at(b);
        words_at<5>(b + 2, w);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            // bits 4k .. 4k + 3 of the high-bit word, one to a byte, at bit 4
            const uint32_t a = w[0] >> (4 * k), c = w[0] >> (4 * k + 16);
            const uint32_t lo = (w[1 + k] & nib) | (((a & 1u) << 4) | ((a & 2u) << 11) | ((a & 4u) << 18) | ((a & 8u) << 25));
            const uint32_t hi = ((w[1 + k] >> 4) & nib) | (((c & 1u) << 4) | ((c & 2u) << 11) | ((c & 4u) << 18) | ((c & 8u) << 25));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y[4 * k + i] = __fmul_rn(byte_f32(lo, i, M + 16.0f), d);
                y[4 * k + i + 16] = __fmul_rn(byte_f32(hi, i, M + 16.0f), d);
            }
        }
    } else if constexpr (T == GGML_TYPE_Q4_K || T == GGML_TYPE_Q5_K) {
        constexpr bool five = T == GGML_TYPE_Q5_K;
        const uint8_t* b = row + (size_t)(u >> 3) * (five ? 176 : 144);
        const uint32_t j = u & 7u;
        const float d = half_at(b), dmin = half_at(b + 2);
        const uint8_t* sc = b + 4;
        uint32_t s6, m6;                             // gguf.c:391-399
        if (j < 4) {
            s6 = sc[j] & 63u;
            m6 = sc[j + 4] & 63u;
        } else {
            s6 = (sc[j + 4] & 15u) | ((uint32_t)(sc[j - 4] >> 6) << 4);
            m6 = (sc[j + 4] >> 4) | ((uint32_t)(sc[j] >> 6) << 4);
        }
        // d sc and d sc q are exact (11 + 6 + 5 bits): one rounding, at the difference
        const float ds = __fmul_rn(d, (float)s6), dm = __fmul_rn(dmin, (float)m6);
        words_at<8>(b + (five ? 48 : 16) + 32 * (j >> 1), w);
        uint32_t h[8];
        if constexpr (five) words_at<8>(b + 16, h);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            uint32_t v = (w[k] >> (4 * (j & 1u))) & nib;
            if constexpr (five) v |= ((h[k] >> j) & 0x01010101u) << 4;
#pragma unroll
            for (int i = 0; i < 4; i++) y[4 * k + i] = fmaf(ds, byte_f32(v, i, M), -dm);
        }
    } else if constexpr (T == GGML_TYPE_Q6_K) {
        const uint8_t* b = row + (size_t)(u >> 3) * 210;
        const uint32_t j = u & 7u, p = j >> 2, c = j & 3u;
        const float d = half_at(b + 208);
        uint32_t h[8];
        words_at<8>(b + 64 * p + 32 * (c & 1u), w);
        words_at<8>(b + 128 + 32 * p, h);
        const int8_t* sc = reinterpret_cast<const int8_t*>(b + 192 + 8 * p + 2 * c);
        const float d0 = __fmul_rn(d, (float)sc[0]), d1 = __fmul_rn(d, (float)sc[1]);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t v = ((w[k] >> (4 * (c >> 1))) & nib) | (((h[k] >> (2 * c)) & 0x03030303u) << 4);
#pragma unroll
            for (int i = 0; i < 4; i++) y[4 * k + i] = __fmul_rn(k < 4 ? d0 : d1, byte_f32(v, i, M + 32.0f));
        }
    }
}

__host__ __device__ constexpr uint32_t block_elems(uint32_t t) { return t >= GGML_TYPE_Q4_K ? 256 : 32; }
__host__ __device__ constexpr uint32_t block_bytes(uint32_t t) {
    return t == GGML_TYPE_Q4_0 ? 18 : t == GGML_TYPE_Q4_1 ? 20 : t == GGML_TYPE_Q5_0 ? 22 : t == GGML_TYPE_Q8_0 ? 34
         : t == GGML_TYPE_Q4_K ? 144 : t == GGML_TYPE_Q5_K ? 176 : 210;
}

// Segment `s0` (units) of a row into shared memory, at the same offset modulo
// 16 as in global memory so that its middle moves in 16-byte words; nothing
// outside the segment's bytes is read.
__device__ __forceinline__ const uint8_t* stage_segment(uint8_t* sm, const uint8_t* src, uint32_t n) {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15u);
    const uint32_t head = min(n, (16u - off) & 15u), vecs = (n - head) / 16, tail = n - head - vecs * 16;
    uint8_t* dst = sm + off;
    for (uint32_t i = threadIdx.x; i < head + tail; i += blockDim.x) {
        const uint32_t at = i < head ? i : head + vecs * 16 + (i - head);
        dst[at] = src[at];
    }
    const uint4* v = reinterpret_cast<const uint4*>(src + head);
    uint4* d = reinterpret_cast<uint4*>(dst + head);
    for (uint32_t i = threadIdx.x; i < vecs; i += blockDim.x) d[i] = v[i];
    __syncthreads();
    return dst;
}

template <uint32_t T>
__global__ void __launch_bounds__(kWThreads) weights_i8_kernel(const WeightArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ uint32_t red[64];
    constexpr uint32_t BE = block_elems(T), BB = block_bytes(T);
    const uint64_t row = blockIdx.x;
    const uint8_t* src = a.raw + row * a.row_bytes;
    int8_t* q = a.q + row * a.ld_q;
    const uint32_t units = a.cols / 32;
    const bool whole = units <= a.seg_units;
    uint32_t m = 0;
    float unused = 0.f;
    RowScale rs = {};
    for (uint32_t pass = 0; pass < 2; pass++) {
        for (uint32_t u0 = 0; u0 < units; u0 += a.seg_units) {
            const uint32_t nu = min(a.seg_units, units - u0), e0 = u0 * 32;
            const uint8_t* p = sm + (reinterpret_cast<uintptr_t>(src) & 15u);
            if (pass == 0 || !whole) {
                __syncthreads();                     // the segment before has been read
                p = stage_segment(sm, src + (uint64_t)e0 / BE * BB, nu * 32 / BE * BB);
            }
            for (uint32_t u = threadIdx.x; u < nu; u += kWThreads) {
                float y[32];
                unit_weights<T>(p, u, y);
#pragma unroll
                for (uint32_t i = 0; i < 32; i++) {
                    if (pass == 0) m = max(m, abs_bits(y[i]));
                    else q[e0 + u * 32 + i] = (int8_t)quant1(y[i], rs);
                }
            }
        }
        if (pass == 0) {
            block_max_sum(m, unused, red);
            rs = row_scale(__uint_as_float(m));
        }
    }
    if (threadIdx.x == 0) a.scale[row] = rs.scale();
}

// The same for rows that fit: a CTA walks groups of rows (back to back in memory),
// copies the next group's bytes while it works on this one's, and each thread
// keeps the U units it decodes in registers from the maximum to the rounding. tpr
// threads (whole warps) a row. Nothing is full: instructions (13 an element, half of them
// work of a row and thread) take 66 % of the issue slots, memory is at 55 % of the copy
// bandwidth, and a group's decoding, maximum and rounding wait for one another. Q8_0
// 4096 x 11008 26.0 us, 3.58 TB/s; without its stores 20.6, without its loads 23.0.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n"
                 ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void stage_async(uint8_t* sm, const uint8_t* src, uint32_t n) {
    const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15u);
    const uint32_t head = min(n, (16u - off) & 15u), vecs = (n - head) / 16, tail = n - head - vecs * 16;
    uint8_t* dst = sm + off;
    for (uint32_t i = threadIdx.x; i < vecs; i += blockDim.x) copy16(dst + head + i * 16, src + head + i * 16);
    for (uint32_t i = threadIdx.x; i < head + tail; i += blockDim.x) {
        const uint32_t at = i < head ? i : head + vecs * 16 + (i - head);
        dst[at] = src[at];
    }
}

template <uint32_t T, uint32_t U>
__global__ void __launch_bounds__(512, U == 1 ? 2 : 1) weights_i8_rows_kernel(const WeightArgs a, uint32_t tpr, uint32_t buf) {
    extern __shared__ __align__(16) uint8_t sm[];    // two buffers of `buf` bytes
    __shared__ uint32_t red[16];
    const uint32_t rows = blockDim.x / tpr, r = threadIdx.x / tpr, t = threadIdx.x - r * tpr;
    const uint32_t units = a.cols / 32, groups = (a.rows + rows - 1) / rows;
    pdl_trigger();
    pdl_wait();
    auto stage = [&](uint32_t g, uint32_t turn) {
        const uint64_t row0 = (uint64_t)g * rows;
        const uint32_t n = (uint32_t)min((uint64_t)rows, a.rows - row0);
        stage_async(sm + (turn & 1u) * buf, a.raw + row0 * a.row_bytes, (uint32_t)(n * a.row_bytes));
    };
    stage(blockIdx.x, 0);
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    for (uint32_t g = blockIdx.x, turn = 0; g < groups; g += gridDim.x, turn++) {
        if (g + gridDim.x < groups) stage(g + gridDim.x, turn + 1);
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 1;\n" ::: "memory");
        __syncthreads();
        const uint64_t row = (uint64_t)g * rows + r;
        const uint8_t* p = sm + (turn & 1u) * buf +
                           (uint32_t)(reinterpret_cast<uintptr_t>(a.raw + (uint64_t)g * rows * a.row_bytes) & 15u);
        float y[U][32], top = 0.f;
        if (row < a.rows) {
#pragma unroll
            for (uint32_t j = 0; j < U; j++) {
                const uint32_t u = t + j * tpr;
                if (u >= units) break;
                unit_weights<T>(p + r * (uint32_t)a.row_bytes, u, y[j]);
#pragma unroll
                for (uint32_t i = 0; i < 32; i++) top = max_abs(top, y[j][i]);
            }
        }
        uint32_t m = __reduce_max_sync(0xffffffffu, abs_bits(top));
        if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();                             // (and every thread has read this buffer)
        if (row >= a.rows) continue;
        const uint32_t nw = tpr / 32, lane = threadIdx.x & 31u;
        m = __reduce_max_sync(0xffffffffu, lane < nw ? red[r * nw + lane] : 0u);
        const RowScale rs = row_scale(__uint_as_float(m));
        int8_t* q = a.q + row * a.ld_q;
        const bool odd = t & 1u;
#pragma unroll
        for (uint32_t j = 0; j < U; j++) {
            const uint32_t u = t + j * tpr;
            if (!rs.plain) {
#pragma unroll
                for (uint32_t i = 0; i < 32; i++) y[j][i] = rs.odd(y[j][i]);
            }
            uint32_t w[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)
                w[i] = low_bytes(fmaf(y[j][4 * i], rs.inv, kRound), fmaf(y[j][4 * i + 1], rs.inv, kRound),
                                 fmaf(y[j][4 * i + 2], rs.inv, kRound), fmaf(y[j][4 * i + 3], rs.inv, kRound));
            // 32 bytes a unit: the even lane stores the first 16 of its own unit, the
            // odd one the second 16 of that, then the same for the odd lane's unit,
            // so that a store covers whole 32-byte sectors (lanes without a unit take part)
            uint32_t s1[4], s2[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t give = odd ? w[i] : w[4 + i];
                const uint32_t got = __shfl_xor_sync(0xffffffffu, give, 1);
                s1[i] = odd ? got : w[i];
                s2[i] = odd ? w[4 + i] : got;
            }
            int8_t* o = q + (u & ~1u) * 32 + (odd ? 16 : 0);
            if ((u & ~1u) < units) *reinterpret_cast<uint4*>(o) = make_uint4(s1[0], s1[1], s1[2], s1[3]);
            if ((u | 1u) < units) *reinterpret_cast<uint4*>(o + 32) = make_uint4(s2[0], s2[1], s2[2], s2[3]);
        }
        if (t == 0) a.scale[row] = rs.scale();
    }
}

template <uint32_t T>
bool launch_weights(const WeightArgs& a, cudaStream_t st) {
    // rows of up to 1024 units whose int8 rows start on 16 bytes
    const uint32_t units = a.cols / 32, U = units <= 512 ? 1 : 2, tpr = (units + 32 * U - 1) / (32 * U) * 32;
    if (tpr <= 512 && i8_aligned(a.q, 16) && a.ld_q % 16 == 0 && a.row_bytes <= kWRow) {
        uint32_t rows = tpr < 256 ? 256 / tpr : 1;   // about 256 threads a CTA
        while (rows > 1 && rows * a.row_bytes > kWRow / 4) rows--;
        const uint32_t buf = ((uint32_t)(rows * a.row_bytes) + kWSlack + 15u) & ~15u, smem = 2 * buf;
        auto* kernel = U == 1 ? weights_i8_rows_kernel<T, 1> : weights_i8_rows_kernel<T, 2>;
        static std::atomic<uint64_t> ready[2];
        if (!allow_smem(ready[U - 1], kernel, 2 * (kWRow + kWSlack + 16))) return false;
        // CTAs that run at once: by threads and shared memory, two by registers at 512 threads
        uint32_t occ = (200 * 1024) / (smem + 1024);
        if (occ * rows * tpr > 1024) occ = 1024 / (rows * tpr);
        if (occ < 1) occ = 1;
        const uint32_t groups = (a.rows + rows - 1) / rows, most = i8_sms() * occ;
        return LM_CUDA(launch_k(kernel, dim3(groups < most ? groups : most), dim3(rows * tpr), smem, st, a, tpr, buf));
    }
    const uint32_t smem = (uint32_t)(a.row_bytes < kWSeg ? a.row_bytes : kWSeg) + kWSlack;
    static std::atomic<uint64_t> ready{0};
    if (!allow_smem(ready, weights_i8_kernel<T>, kWSeg + kWSlack)) return false;
    weights_i8_kernel<T><<<a.rows, kWThreads, smem, st>>>(a);
    return LM_CUDA(cudaGetLastError());
}

bool act_type_ok(const char* who, uint32_t type) {
    if (act_bytes(type)) return true;
    set_error("%s: element type %u is not F32, F16 or BF16", who, type);
    return false;
}
bool cols_ok(const char* who, uint32_t cols) {
    if (cols >= 1 && cols <= kI8MaxCols) return true;
    set_error("%s: %u columns (1 to %u)", who, cols, kI8MaxCols);
    return false;
}
bool pitch_ok(const char* who, const char* what, u64 ld, uint32_t cols) {
    if (ld >= cols && ld <= (1ull << 40)) return true;
    set_error("%s: pitch %llu of %s for %u columns", who, (unsigned long long)ld, what, cols);
    return false;
}
bool rows_ok(const char* who, uint32_t rows) {
    if (rows <= 0x7FFFFFFFu) return true;
    set_error("%s: %u rows (at most 2^31 - 1)", who, rows);
    return false;
}
bool align_ok(const char* who, const void* const* ptrs, int n, size_t bytes) {
    for (int i = 0; i < n; i++)
        if (ptrs[i] && !i8_aligned(ptrs[i], bytes)) {
            set_error("%s: an array of %u-byte elements is not aligned to them", who, (unsigned)bytes);
            return false;
        }
    return true;
}

// CTAs of a kernel that walks `rows` rows, `per` at a time: as many as run at
// once, and no more than there are rows. occupancy: CTAs an SM by warps of a CTA,
// looked up once.
template <typename K>
uint32_t walkers(std::atomic<int>* occupancy, K* kernel, uint32_t threads, uint64_t rows, uint32_t per) {
    const uint32_t sms = i8_sms();
    const uint64_t want = (rows + per - 1) / per;
    if (want <= sms) return (uint32_t)want;
    std::atomic<int>& memo = occupancy[threads / 32];
    int occ = memo.load(std::memory_order_relaxed);
    if (occ == 0) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ, kernel, (int)threads, 0) != cudaSuccess || occ < 1) {
            cudaGetLastError();
            occ = 1;
        }
        memo.store(occ, std::memory_order_relaxed);
    }
    const uint64_t n = (uint64_t)sms * occ;
    return (uint32_t)(want < n ? want : n);
}
template <typename T> bool vec_rows(const void* p, uint64_t ld) {
    return !p || (i8_aligned(p, 16) && ld * sizeof(T) % 16 == 0);
}
template <typename T> bool vec_q(const int8_t* q, uint64_t ld) {
    return i8_aligned(q, vec_elems<T>()) && ld % vec_elems<T>() == 0;
}

// How a launch spreads its rows: a warp each, or CTAs of `threads`.
struct RowShape {
    uint32_t threads, per;
};

template <typename T, bool RESID, uint32_t E, bool WARP, uint32_t V>
bool launch_norm_rows(const NormArgs& a, const RowShape& r, cudaStream_t st) {
    static std::atomic<int> occupancy[33];
    const uint32_t grid = walkers(occupancy, norm_i8_rows_kernel<T, RESID, WARP, E, V>, r.threads, a.rows, r.per);
    return LM_CUDA(launch_k(norm_i8_rows_kernel<T, RESID, WARP, E, V>, dim3(grid), dim3(r.threads), 0, st, a));
}
template <typename T, bool UP, uint32_t E, bool WARP, uint32_t V>
bool launch_glu_rows(const GluArgs& a, const RowShape& r, cudaStream_t st) {
    static std::atomic<int> occupancy[33];
    const uint32_t grid = walkers(occupancy, glu_i8_rows_kernel<T, UP, WARP, E, V>, r.threads, a.rows, r.per);
    return LM_CUDA(launch_k(glu_i8_rows_kernel<T, UP, WARP, E, V>, dim3(grid), dim3(r.threads), 0, st, a));
}

// Vectors a thread for rows of nv 16-byte vectors (0: none fits; 10 + V: V a lane,
// a warp a row). Few and short rows want one vector a thread, for the shortest
// path through a row; long ones enough threads for two CTAs an SM and no idle lanes
// in the last round. us of bf16 norm with residual at V = 1, 2, 4: 4096 x 2048
// 11.8, 12.6, 13.1; 4096 x 4096 21.7, 22.6, 21.1. bf16 SiLU at V = 2, 3, 4: 4096 x
// 4864 19.4, 22.7, 20.8; 4096 x 11008 (3, 4, 6) 42.6, 51.2, 46.9; f32 (6, 8) 63.2, 68.5.
// Many short rows, a warp each: 20000 x 128 bf16 norm 8.2 against 10.1 us.
uint32_t rows_vectors(bool norm, uint32_t rows, uint32_t nv) {
    if (rows >= 1024 && nv <= 32) return 11;
    if (rows >= 1024 && nv <= 64) return 12;
    if (nv <= 256) return 1;
    if (nv <= 1024) return norm && rows >= 1024 && nv >= 512 ? 4 : 2;
    if (!norm && rows < 1024 && nv <= 2048) return 2;
    if (nv <= 1536) return 3;
    if (nv <= 2048) return 4;
    return nv <= 6 * 512 ? 6 : nv <= 8 * 512 ? 8 : 0;
}

// Calls LAUNCH for the shape that fits rows of `cols` elements; falls through
// when no shape does.
#define LM_I8_VEC_ROWS(NORM, LAUNCH, T, ...)                                                \
    do {                                                                                    \
        constexpr uint32_t E = vec_elems<T>();                                              \
        const uint32_t nv = (a.cols + E - 1) / E, v = rows_vectors(NORM, a.rows, nv);       \
        if (v == 0) break;                                                                  \
        const RowShape w = {32 * kWarpRows, kWarpRows}, r = {((nv + v - 1) / v + 31) / 32 * 32, 1}; \
        switch (v) {                                                                        \
        case 11: return LAUNCH<T, __VA_ARGS__, E, true, 1>(a, w, st);                       \
        case 12: return LAUNCH<T, __VA_ARGS__, E, true, 2>(a, w, st);                       \
        case 1: return LAUNCH<T, __VA_ARGS__, E, false, 1>(a, r, st);                       \
        case 2: return LAUNCH<T, __VA_ARGS__, E, false, 2>(a, r, st);                       \
        case 3: return LAUNCH<T, __VA_ARGS__, E, false, 3>(a, r, st);                       \
        case 4: return LAUNCH<T, __VA_ARGS__, E, false, 4>(a, r, st);                       \
        case 6: return LAUNCH<T, __VA_ARGS__, E, false, 6>(a, r, st);                       \
        case 8: return LAUNCH<T, __VA_ARGS__, E, false, 8>(a, r, st);                       \
        }                                                                                   \
    } while (0)
// The same one element at a time, where a pitch or base is not whole 16-byte
// vectors (4096 x 4097 bf16 norm: 62 us; 4096 x 4096 from vectors 21).
#define LM_I8_ODD_ROWS(LAUNCH, T, ...)                                                      \
    do {                                                                                    \
        const uint32_t n = a.cols;                                                          \
        const RowShape w = {32 * kWarpRows, kWarpRows}, r = {((n + 7) / 8 + 31) / 32 * 32, 1}, \
                       s = {((n + 15) / 16 + 31) / 32 * 32, 1};                             \
        if (a.rows >= 1024 && n <= 256) return LAUNCH<T, __VA_ARGS__, 1, true, 8>(a, w, st); \
        if (n <= 8192) return LAUNCH<T, __VA_ARGS__, 1, false, 8>(a, r, st);                \
        if (n <= 16384) return LAUNCH<T, __VA_ARGS__, 1, false, 16>(a, s, st);              \
    } while (0)

template <typename T, bool UP>
bool launch_glu(const GluArgs& a, cudaStream_t st) {
    if (vec_rows<T>(a.gate, a.ld_gate) && vec_rows<T>(a.up, a.ld_up) && vec_q<T>(a.q, a.ld_q))
        LM_I8_VEC_ROWS(false, launch_glu_rows, T, UP);
    LM_I8_ODD_ROWS(launch_glu_rows, T, UP);
    glu_i8_kernel<T><<<a.rows, 512, 0, st>>>(a);
    return LM_CUDA(cudaGetLastError());
}
template <typename T>
bool launch_glu(const GluArgs& a, cudaStream_t st) {
    return a.up ? launch_glu<T, true>(a, st) : launch_glu<T, false>(a, st);
}

template <typename T, bool RESID>
bool launch_norm(const NormArgs& a, cudaStream_t st) {
    if (vec_rows<T>(a.x, a.ld_x) && vec_rows<T>(a.resid, a.ld_resid) && vec_rows<T>(a.sum, a.ld_sum) && vec_q<T>(a.q, a.ld_q))
        LM_I8_VEC_ROWS(true, launch_norm_rows, T, RESID);
    LM_I8_ODD_ROWS(launch_norm_rows, T, RESID);
    norm_i8_kernel<T><<<a.rows, 512, 0, st>>>(a);
    return LM_CUDA(cudaGetLastError());
}
template <typename T>
bool launch_norm(const NormArgs& a, cudaStream_t st) {
    return a.resid ? launch_norm<T, true>(a, st) : launch_norm<T, false>(a, st);
}

}  // namespace
}  // namespace lm

extern "C" int llamini_weights_i8_device(u32 type, const void* d_blocks, u32 rows, u32 cols, i8* d_q, u64 ld_q,
                                         f32* d_scale, void* stream) {
    using namespace lm;
    const char* who = "weights_i8";
    TypeInfo ti;
    if (!type_info(type, &ti)) { set_error("%s: unsupported type %u", who, type); return -1; }
    if (!cols_ok(who, cols) || !rows_ok(who, rows) || !pitch_ok(who, "q", ld_q, cols)) return -1;
    if (cols % ti.block_elems != 0) {
        set_error("%s: %u columns are not whole blocks of type %u", who, cols, type);
        return -1;
    }
    if (rows == 0) return 0;
    const void* ptrs[] = {d_blocks, d_q, d_scale};
    const char* const names[] = {"blocks", "q", "scale"};
    if (!d_blocks || !d_q || !d_scale) { set_error("%s: null pointer", who); return -1; }
    const size_t align = type == GGML_TYPE_F32 ? 4 : 2;      // blocks start with, and are read in, 16-bit fields
    if (!align_ok(who, ptrs, 1, align) || !align_ok(who, ptrs + 2, 1, 4) || !i8_device_ptrs(who, ptrs, names, 3)) return -1;
    WeightArgs a;
    a.raw = static_cast<const uint8_t*>(d_blocks);
    a.q = reinterpret_cast<int8_t*>(d_q);
    a.scale = d_scale;
    a.row_bytes = type_bytes(type, cols);
    a.ld_q = ld_q;
    a.rows = rows; a.cols = cols;
    a.seg_units = kWSeg / ti.block_bytes * (ti.block_elems / 32);    // whole blocks to a segment
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    bool ok = false;
    GluArgs g = {};                                  // plain rows: the rounding of the gated activation without one
    g.gate = d_blocks;
    g.q = a.q; g.scale = a.scale;
    g.ld_gate = cols; g.ld_q = ld_q;
    g.rows = rows; g.cols = cols; g.act = LLAMINI_ACT_NONE;
    switch (type) {
    case GGML_TYPE_F32: ok = launch_glu<float>(g, st); break;
    case GGML_TYPE_F16: ok = launch_glu<__half>(g, st); break;
    case GGML_TYPE_Q4_0: ok = launch_weights<GGML_TYPE_Q4_0>(a, st); break;
    case GGML_TYPE_Q4_1: ok = launch_weights<GGML_TYPE_Q4_1>(a, st); break;
    case GGML_TYPE_Q5_0: ok = launch_weights<GGML_TYPE_Q5_0>(a, st); break;
    case GGML_TYPE_Q8_0: ok = launch_weights<GGML_TYPE_Q8_0>(a, st); break;
    case GGML_TYPE_Q4_K: ok = launch_weights<GGML_TYPE_Q4_K>(a, st); break;
    case GGML_TYPE_Q5_K: ok = launch_weights<GGML_TYPE_Q5_K>(a, st); break;
    case GGML_TYPE_Q6_K: ok = launch_weights<GGML_TYPE_Q6_K>(a, st); break;
    }
    return ok ? 0 : -1;
}

extern "C" int llamini_rms_norm_i8_device(u32 type, const void* d_x, u64 ld_x, const void* d_resid, u64 ld_resid,
                                          void* d_sum, u64 ld_sum, const f32* d_w, f32 eps, u32 rows, u32 cols,
                                          i8* d_q, u64 ld_q, f32* d_scale, void* stream) {
    using namespace lm;
    const char* who = "rms_norm_i8";
    if (!act_type_ok(who, type) || !cols_ok(who, cols) || !rows_ok(who, rows) || !pitch_ok(who, "x", ld_x, cols) ||
        (d_resid && !pitch_ok(who, "the residual", ld_resid, cols)) ||
        (d_sum && !pitch_ok(who, "the sum", ld_sum, cols)) || !pitch_ok(who, "q", ld_q, cols))
        return -1;
    if (!(eps >= 0.0f)) { set_error("%s: eps is negative or NaN", who); return -1; }
    if ((d_sum == d_x && d_x && ld_sum != ld_x) || (d_sum && d_sum == d_resid && ld_sum != ld_resid)) {
        set_error("%s: a sum stored over its input needs that input's pitch", who);
        return -1;
    }
    if (rows == 0) return 0;
    const void* ptrs[] = {d_x, d_resid, d_sum, d_w, d_q, d_scale};
    const char* const names[] = {"x", "resid", "sum", "w", "q", "scale"};
    if (!d_x || !d_w || !d_q || !d_scale) { set_error("%s: null pointer", who); return -1; }
    const void* f32s[] = {d_w, d_scale};
    if (!align_ok(who, ptrs, 3, act_bytes(type)) || !align_ok(who, f32s, 2, 4) || !i8_device_ptrs(who, ptrs, names, 6)) return -1;
    NormArgs a;
    a.x = d_x; a.resid = d_resid; a.sum = d_sum; a.w = d_w;
    a.q = reinterpret_cast<int8_t*>(d_q); a.scale = d_scale;
    a.ld_x = ld_x; a.ld_resid = ld_resid; a.ld_sum = ld_sum; a.ld_q = ld_q;
    a.rows = rows; a.cols = cols; a.eps = eps;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool ok = type == GGML_TYPE_F32 ? launch_norm<float>(a, st)
                  : type == GGML_TYPE_F16 ? launch_norm<__half>(a, st) : launch_norm<__nv_bfloat16>(a, st);
    return ok ? 0 : -1;
}

extern "C" int llamini_glu_i8_device(u32 type, const void* d_gate, u64 ld_gate, const void* d_up, u64 ld_up, u32 act,
                                     u32 rows, u32 cols, i8* d_q, u64 ld_q, f32* d_scale, void* stream) {
    using namespace lm;
    const char* who = "glu_i8";
    if (!act_type_ok(who, type) || !cols_ok(who, cols) || !rows_ok(who, rows) ||
        !pitch_ok(who, "gate", ld_gate, cols) || (d_up && !pitch_ok(who, "up", ld_up, cols)) ||
        !pitch_ok(who, "q", ld_q, cols))
        return -1;
    if (act > LLAMINI_ACT_NONE) { set_error("%s: unknown activation %u", who, act); return -1; }
    if (rows == 0) return 0;
    const void* ptrs[] = {d_gate, d_up, d_q, d_scale};
    const char* const names[] = {"gate", "up", "q", "scale"};
    if (!d_gate || !d_q || !d_scale) { set_error("%s: null pointer", who); return -1; }
    if (!align_ok(who, ptrs, 2, act_bytes(type)) || !align_ok(who, ptrs + 3, 1, 4) || !i8_device_ptrs(who, ptrs, names, 4)) return -1;
    GluArgs a;
    a.gate = d_gate; a.up = d_up;
    a.q = reinterpret_cast<int8_t*>(d_q); a.scale = d_scale;
    a.ld_gate = ld_gate; a.ld_up = ld_up; a.ld_q = ld_q;
    a.rows = rows; a.cols = cols; a.act = act;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool ok = type == GGML_TYPE_F32 ? launch_glu<float>(a, st)
                  : type == GGML_TYPE_F16 ? launch_glu<__half>(a, st) : launch_glu<__nv_bfloat16>(a, st);
    return ok ? 0 : -1;
}
