// i8.cuh -- what the 8-bit integer operators (k_i8.cu, k_gemm_i8.cu) share: the
// types of activations, the checks of their C entry points, and the rounding of
// a row of f32 values to int8.
//
// An int8 row stands for the values q[i] * scale with one f32 scale a row:
// scale = max|y| / 127 and q = y / scale rounded to the nearest integer, ties
// to even, so |q| <= 127 and -128 never appears. A row of zeros has scale 0. A
// row that holds a NaN or an infinity has scale NaN and q = 0: every value it
// stands for is NaN, so the fault stays visible.
#pragma once

#include "internal.h"
#include "llamini_b200.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

namespace lm {

// Sums of `cols` int8 products stay within 32 bits up to this length even when
// a caller's own rows hold -128: 131071 * 128 * 128 < 2^31.
constexpr uint32_t kI8MaxCols = 131071;

inline size_t act_bytes(uint32_t type) {
    return type == GGML_TYPE_F32 ? 4 : type == GGML_TYPE_F16 || type == LLAMINI_TYPE_BF16 ? 2 : 0;
}

// Whether every pointer of ptrs[0..n) (null ones are skipped) is memory that a
// kernel on the calling thread's current device may use: that device's own, or
// managed. A host pointer, or another device's, would fault in the kernel.
inline bool i8_device_ptrs(const char* who, const void* const* ptrs, int n) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: no usable CUDA device (this library has no CPU path)", who);
        return false;
    }
    for (int i = 0; i < n; i++) {
        if (!ptrs[i]) continue;
        cudaPointerAttributes a;
        if (cudaPointerGetAttributes(&a, ptrs[i]) != cudaSuccess) {
            cudaGetLastError();
            set_error("%s: no usable CUDA device (this library has no CPU path)", who);
            return false;
        }
        if (a.type == cudaMemoryTypeManaged) continue;
        if (a.type != cudaMemoryTypeDevice || a.device != dev) {
            set_error("%s: pointer argument %d is not memory of the current device (%d)", who, i + 1, dev);
            return false;
        }
    }
    return true;
}

inline bool i8_aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---------------------------------------------------------------- device

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// |y| as bits: their order as unsigned integers is the order of the
// magnitudes, infinity above every finite value and every NaN above that, so
// an integer maximum over a row also finds its NaNs.
__device__ __forceinline__ uint32_t abs_bits(float y) { return __float_as_uint(y) & 0x7FFFFFFFu; }

// The scale of a row whose largest magnitude has these bits, and how its
// elements become integers.
struct RowScale {
    float scale, inv;
    bool tiny, zero;
};
__device__ __forceinline__ RowScale row_scale(float amax) {
    RowScale r;
    const bool bad = !(amax < INFINITY);
    r.scale = bad ? NAN : __fdiv_rn(amax, 127.0f);
    // below 1.5e-36 the scale is subnormal or 127 / max overflows
    r.tiny = amax < 1.5e-36f;
    r.zero = bad || r.scale == 0.0f;
    r.inv = r.tiny || bad ? 0.0f : __fdiv_rn(127.0f, amax);
    return r;
}
// One element: y * (127 / max) instead of y / scale, one rounding apart, which
// only moves an element that lies within 2^-17 of halfway between two integers.
__device__ __forceinline__ int quant1(float y, const RowScale& r) {
    if (r.zero) return 0;
    if (r.tiny) return max(-127, min(127, __float2int_rn(__fdiv_rn(y, r.scale))));
    return __float2int_rn(y * r.inv);
}

// Block-wide maximum of unsigned integers and sum of floats; every thread gets
// both. red: 64 words of shared memory.
__device__ __forceinline__ void block_max_sum(uint32_t& m, float& s, uint32_t* red) {
    m = __reduce_max_sync(0xffffffffu, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const uint32_t nw = (blockDim.x + 31) >> 5, w = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31u) == 0) {
        red[w] = m;
        red[32 + w] = __float_as_uint(s);
    }
    __syncthreads();
    m = red[0];
    s = __uint_as_float(red[32]);
    for (uint32_t i = 1; i < nw; i++) {
        m = max(m, red[i]);
        s += __uint_as_float(red[32 + i]);
    }
}

}  // namespace lm
