// i8.cuh -- what the 8-bit integer operators (k_i8.cu, k_gemm_i8.cu) share: the
// types of activations, the checks of their C entry points, and the rounding of
// a row of f32 values to int8.
//
// An int8 row stands for the values q[i] * scale with one f32 scale a row:
// scale = max|y| / 127 and q = y * (127 / max|y|) rounded to the nearest integer,
// ties to even, both quotients rounded to f32, so |q| <= 127 and -128 never
// appears. (The reciprocal instead of y / scale moves only an element that lies
// within 2^-16 of halfway between two integers, among them exact ties, which it
// takes either way -- a Q8_0 row whose largest code is -128 has them at its block's
// +-64 -- and makes the rounding of y one fused multiply-add, the same everywhere. The
// norm's row kernels fold 1 / rms into the factor, one rounding more.) A row of
// zeros has scale 0.
// A row that holds a NaN or an infinity has scale NaN and q = 0: every value it
// stands for is NaN, so the fault stays visible. Where 127 / max|y| comes
// near f32's limit (it passes it below a max|y| of 3.7e-37; the change is at 1.5e-36) y
// and max|y| are multiplied by 2^100 first; where the scale rounds to 0 so does q.
#pragma once

#include "internal.h"
#include "llamini_b200.h"

#include <atomic>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <type_traits>

namespace lm {

// Sums of `cols` int8 products stay within 32 bits up to this length even when
// a caller's own rows hold -128: 131071 * 128 * 128 < 2^31.
constexpr uint32_t kI8MaxCols = 131071;

inline size_t act_bytes(uint32_t type) {
    return type == GGML_TYPE_F32 ? 4 : type == GGML_TYPE_F16 || type == LLAMINI_TYPE_BF16 ? 2 : 0;
}

// Whether every pointer of ptrs[0..n), called names[0..n) (null ones are skipped), is memory that a
// kernel on the calling thread's current device may use: that device's own, or
// managed. A host pointer, or another device's, would fault in the kernel.
inline bool i8_device_ptrs(const char* who, const void* const* ptrs, const char* const* names, int n) {
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        set_error("%s: no usable CUDA device (this library has no CPU path)", who);
        return false;
    }
    for (int i = 0; i < n; i++) {
        if (!ptrs[i]) continue;
        cudaPointerAttributes a;
        if (!LM_CUDA(cudaPointerGetAttributes(&a, ptrs[i]))) return false;
        if (a.type == cudaMemoryTypeManaged) continue;
        if (a.type != cudaMemoryTypeDevice || a.device != dev) {
            set_error("%s: %s is not memory of the current device (%d)", who, names[i], dev);
            return false;
        }
    }
    return true;
}

// SMs of the device (of the first one a call is made on: all of a box are alike).
inline uint32_t i8_sms() {
    static const uint32_t sms = [] {
        int dev = 0, n = 0;
        if (cudaGetDevice(&dev) != cudaSuccess ||
            cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2) {
            cudaGetLastError();
            n = 148;
        }
        return (uint32_t)n;
    }();
    return sms;
}

// The kernel's limit on dynamic shared memory, raised once a device. (Unasked a CTA gets
// 48 KB of static and dynamic shared memory together.)
template <typename K>
inline bool allow_smem(std::atomic<uint64_t>& done, K* kernel, size_t bytes) {
    int dev = 0;
    if (!LM_CUDA(cudaGetDevice(&dev))) return false;
    const uint64_t bit = 1ull << (dev & 63);             // (a device past the 63rd sets it at each call)
    if (dev < 64 && done.load(std::memory_order_acquire) & bit) return true;
    if (!LM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes))) return false;
    done.fetch_or(bit, std::memory_order_release);
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
// max(m, |y|), NaN when either is: one instruction an element.
__device__ __forceinline__ float max_abs(float m, float y) {
    float r;
    asm("{\n .reg .f32 t;\n abs.f32 t, %2;\n max.NaN.f32 %0, %1, t;\n}\n" : "=f"(r) : "f"(m), "f"(y));
    return r;
}

// Adding 1.5 * 2^23 leaves an f32 of magnitude below 2^22, rounded to the nearest
// integer (ties to even), in the low mantissa bits: the low byte is the int8.
constexpr float kRound = 12582912.0f;

// How the elements of a row with this largest magnitude become integers, and
// the row's scale (a division that only one thread of a row needs).
struct RowScale {
    float amax, inv, up;       // 127 / (amax up); up = 1, or 2^100 for tiny rows
    bool plain;                // finite and not tiny: q = y inv
    __device__ __forceinline__ float scale() const { return amax < INFINITY ? __fdiv_rn(amax, 127.0f) : NAN; }
    // what a row that is not plain multiplies by inv: nothing is left of one that
    // is not finite or whose scale rounds to zero
    __device__ __forceinline__ float odd(float y) const { return scale() > 0.0f ? y * up : 0.0f; }
};
__device__ __forceinline__ RowScale row_scale(float amax) {
    RowScale r;
    r.amax = amax;
    r.plain = amax >= 1.5e-36f && amax < INFINITY;
    r.up = amax < 1.5e-36f ? 0x1p100f : 1.0f;
    r.inv = r.plain || amax > 0.0f ? __fdiv_rn(127.0f, amax * r.up) : 0.0f;
    if (!(amax < INFINITY)) r.inv = 0.0f;
    return r;
}
__device__ __forceinline__ int quant1(float y, const RowScale& r) {
    return (int)(int8_t)__float_as_uint(fmaf(r.plain ? y : r.odd(y), r.inv, kRound));
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

// ---------------------------------------------------------------- rows in registers
//
// A row in pieces of E elements (16 bytes, or one element where pitches or bases
// are not whole 16 bytes) spread over G threads (a warp, or a whole CTA), up to V
// pieces a thread, piece j of thread t at t + j G.

template <typename T> constexpr uint32_t vec_elems() { return 16 / sizeof(T); }

// The 16 bytes of vector v as f32; elements from `cols` on are zero.
template <typename T>
__device__ __forceinline__ void vec_to_f32(const uint4& raw, float* f) {
    if constexpr (sizeof(T) == 4) {
        f[0] = __uint_as_float(raw.x); f[1] = __uint_as_float(raw.y);
        f[2] = __uint_as_float(raw.z); f[3] = __uint_as_float(raw.w);
    } else {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = p.x; f[2 * i + 1] = p.y;
            } else {                                 // bf16 is the upper half of f32
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ uint4 f32_to_vec(const float* f) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else
        return make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
}
// A piece as it lies in memory.
template <typename T, uint32_t E> struct Piece { uint4 v; };
template <typename T> struct Piece<T, 1> { T v; };

// Elements [at, at + E) of a row; past the row's end zeros, and nothing is read there.
template <typename T, uint32_t E>
__device__ __forceinline__ void load_piece(Piece<T, E>& p, const T* row, uint32_t at, uint32_t cols) {
    if constexpr (E == 1) {
        p.v = at < cols ? row[at] : from_f32<T>(0.f);
    } else {
        if (at + E <= cols) {
            p.v = *reinterpret_cast<const uint4*>(row + at);
            return;
        }
        p.v = make_uint4(0, 0, 0, 0);
        if (at < cols) {
            T e[E];
            *reinterpret_cast<uint4*>(e) = p.v;
            for (uint32_t i = 0; i < E; i++)
                if (at + i < cols) e[i] = row[at + i];
            p.v = *reinterpret_cast<uint4*>(e);
        }
    }
}
template <typename T, uint32_t E>
__device__ __forceinline__ void piece_to_f32(const Piece<T, E>& p, float* f) {
    if constexpr (E == 1) f[0] = to_f32(p.v);
    else vec_to_f32<T>(p.v, f);
}
template <typename T, uint32_t E>
__device__ __forceinline__ void store_piece(T* row, uint32_t at, uint32_t cols, const float* f) {
    if constexpr (E == 1) {
        if (at < cols) row[at] = from_f32<T>(f[0]);
    } else {
        const uint4 v = f32_to_vec<T>(f);
        if (at + E <= cols) {
            *reinterpret_cast<uint4*>(row + at) = v;
            return;
        }
        const T* e = reinterpret_cast<const T*>(&v);
        for (uint32_t i = 0; i < E; i++)
            if (at + i < cols) row[at + i] = e[i];
    }
}

__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
    const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
}

// E values of a row, times f (127 / max, or what maps onto it), to int8 at q + at.
template <uint32_t E>
__device__ __forceinline__ void store_quant(int8_t* q, uint32_t at, uint32_t cols, const float* v, float f) {
    if constexpr (E == 1) {
        if (at < cols) q[at] = (int8_t)__float_as_uint(fmaf(v[0], f, kRound));
    } else {
        uint32_t w[E / 4];
#pragma unroll
        for (uint32_t i = 0; i < E / 4; i++)
            w[i] = low_bytes(fmaf(v[4 * i], f, kRound), fmaf(v[4 * i + 1], f, kRound), fmaf(v[4 * i + 2], f, kRound),
                             fmaf(v[4 * i + 3], f, kRound));
        if (at + E <= cols) {
            if constexpr (E == 8) *reinterpret_cast<uint2*>(q + at) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(q + at) = w[0];
        } else {
            for (uint32_t i = 0; i < E; i++)
                if (at + i < cols) q[at + i] = (int8_t)(w[i >> 2] >> (8 * (i & 3u)));
        }
    }
}

// Maximum and sum over the threads of a row, a warp (WARP) or the CTA; every
// thread gets both, and each adds in the same order. `turn` alternates between
// two halves of red (128 words), so that one barrier a row is enough.
template <bool WARP>
__device__ __forceinline__ void row_max_sum(uint32_t& m, float& s, uint32_t* red, uint32_t turn) {
    m = __reduce_max_sync(0xffffffffu, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if constexpr (!WARP) {
        const uint32_t nw = blockDim.x >> 5, lane = threadIdx.x & 31u;
        uint32_t* r = red + (turn & 1u) * 64;
        if (lane == 0) {
            r[threadIdx.x >> 5] = m;
            r[32 + (threadIdx.x >> 5)] = __float_as_uint(s);
        }
        __syncthreads();
        m = lane < nw ? r[lane] : 0u;
        s = lane < nw ? __uint_as_float(r[32 + lane]) : 0.f;
        m = __reduce_max_sync(0xffffffffu, m);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
}

}  // namespace lm
