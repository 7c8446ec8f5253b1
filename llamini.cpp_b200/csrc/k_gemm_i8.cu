// k_gemm_i8.cu -- int8 matrix product with a scale for each token and channel:
//
//   out[m][n] = (sum_k a[m][k] w[n][k]) * a_scale[m] * w_scale[n] (+ bias[n])
//
// The sums are exact in 32-bit integers (at most 131071 columns, i8.cuh); the
// three f32 roundings after them (the sum to f32 and the two scales), the
// bias's and the output type's are all the rounding there is.
#include "i8.cuh"

namespace lm {
namespace {

struct GemmI8Args {
    const int8_t* a;
    const float* as;
    const int8_t* w;
    const float* ws;
    const float* bias;         // may be null
    void* out;
    uint64_t ld_a, ld_w, ld_out;
    uint32_t m, n, k;
};

// Rows of any pitch and alignment: 64 x 64 outputs a CTA, 64 columns of both
// operands at a time in shared memory as words of four, dp4a on 4 x 4 outputs
// a thread.
constexpr uint32_t kST = 64, kSW = kST / 4, kSPad = kSW + 1;

__device__ __forceinline__ void load_words(uint32_t (*dst)[kSPad], const int8_t* src, uint64_t ld, uint32_t r0,
                                           uint32_t rows, uint32_t k0, uint32_t k) {
    for (uint32_t i = threadIdx.x; i < kST * kSW; i += 256) {
        const uint32_t r = i / kSW, c = i % kSW;
        uint32_t v = 0;
        if (r0 + r < rows) {
            const uint8_t* p = reinterpret_cast<const uint8_t*>(src) + (uint64_t)(r0 + r) * ld;
#pragma unroll
            for (uint32_t b = 0; b < 4; b++)
                if (k0 + 4 * c + b < k) v |= (uint32_t)p[k0 + 4 * c + b] << (8 * b);
        }
        dst[r][c] = v;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) gemm_i8_any_kernel(const GemmI8Args g) {
    __shared__ uint32_t sa[kST][kSPad], sw[kST][kSPad];
    const uint32_t nt = (g.n + kST - 1) / kST;
    const uint32_t n0 = blockIdx.x % nt * kST, m0 = blockIdx.x / nt * kST;
    const uint32_t tx = threadIdx.x & 15u, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < g.k; k0 += kST) {
        load_words(sa, g.a, g.ld_a, m0, g.m, k0, g.k);
        load_words(sw, g.w, g.ld_w, n0, g.n, k0, g.k);
        __syncthreads();
#pragma unroll
        for (uint32_t c = 0; c < kSW; c++) {
            uint32_t x[4], y[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                x[i] = sa[ty + 16 * i][c];
                y[i] = sw[tx + 16 * i][c];
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) acc[i][j] = __dp4a((int)x[i], (int)y[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) {
        const uint32_t m = m0 + ty + 16 * i;
        if (m >= g.m) continue;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t n = n0 + tx + 16 * j;
            if (n >= g.n) continue;
            float v = (float)acc[i][j] * g.as[m] * g.ws[n];
            if (g.bias) v += g.bias[n];
            static_cast<T*>(g.out)[(uint64_t)m * g.ld_out + n] = from_f32<T>(v);
        }
    }
}

template <typename T>
bool launch_any(const GemmI8Args& g, cudaStream_t st) {
    const uint64_t tiles = (uint64_t)((g.m + kST - 1) / kST) * ((g.n + kST - 1) / kST);
    if (tiles > 0x7FFFFFFFull) {
        set_error("gemm_i8: %u x %u outputs are too many for one call", g.m, g.n);
        return false;
    }
    gemm_i8_any_kernel<T><<<(uint32_t)tiles, 256, 0, st>>>(g);
    return LM_CUDA(cudaGetLastError());
}

template <typename T>
bool launch(const GemmI8Args& g, cudaStream_t st) {
    return launch_any<T>(g, st);
}

}  // namespace
}  // namespace lm

extern "C" int llamini_gemm_i8_device(const i8* d_a, u64 ld_a, const f32* d_a_scale, u32 rows, const i8* d_w, u64 ld_w,
                                      const f32* d_w_scale, u32 n, u32 cols, const f32* d_bias, u32 out_type,
                                      void* d_out, u64 ld_out, void* stream) {
    using namespace lm;
    const char* who = "gemm_i8";
    const size_t ob = act_bytes(out_type);
    if (!ob) { set_error("%s: output type %u is not F32, F16 or BF16", who, out_type); return -1; }
    if (cols == 0 || cols > kI8MaxCols) { set_error("%s: %u columns (1 to %u)", who, cols, kI8MaxCols); return -1; }
    if (rows > 0x7FFFFFFFu || n > 0x7FFFFFFFu) { set_error("%s: %u x %u outputs", who, rows, n); return -1; }
    if (ld_a < cols || ld_w < cols || ld_out < n || ld_a > (1ull << 40) || ld_w > (1ull << 40) || ld_out > (1ull << 40)) {
        set_error("%s: a pitch is less than its row (a %llu, w %llu for %u columns; out %llu for %u)", who,
                  (unsigned long long)ld_a, (unsigned long long)ld_w, cols, (unsigned long long)ld_out, n);
        return -1;
    }
    if (rows == 0 || n == 0) return 0;
    if (!d_a || !d_a_scale || !d_w || !d_w_scale || !d_out) { set_error("%s: null pointer", who); return -1; }
    if (!i8_aligned(d_a_scale, 4) || !i8_aligned(d_w_scale, 4) || !i8_aligned(d_bias, 4) || !i8_aligned(d_out, ob)) {
        set_error("%s: scales, bias or output are not aligned to their elements", who);
        return -1;
    }
    const void* ptrs[] = {d_a, d_a_scale, d_w, d_w_scale, d_bias, d_out};
    if (!i8_device_ptrs(who, ptrs, 6)) return -1;
    GemmI8Args g;
    g.a = reinterpret_cast<const int8_t*>(d_a); g.as = d_a_scale;
    g.w = reinterpret_cast<const int8_t*>(d_w); g.ws = d_w_scale;
    g.bias = d_bias; g.out = d_out;
    g.ld_a = ld_a; g.ld_w = ld_w; g.ld_out = ld_out;
    g.m = rows; g.n = n; g.k = cols;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool ok = out_type == GGML_TYPE_F32 ? launch<float>(g, st)
                  : out_type == GGML_TYPE_F16 ? launch<__half>(g, st) : launch<__nv_bfloat16>(g, st);
    return ok ? 0 : -1;
}
