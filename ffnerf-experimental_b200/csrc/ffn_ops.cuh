// ffn_ops.cuh -- what the block operators (ffn_norm.cu, ffn_scan.cu, ffn_experts.cu) share: element
// types, wide loads and stores, argument checks.  Each operator file is a translation unit of its own.
#pragma once
#include <cstdint>
#include <string>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/ffnerf.h"

namespace ffn {

// Records the message that ffn_last_error(NULL) returns and gives the code back (ffn_capi.cu).
int op_fail(int code, const std::string& msg);

// Reads and clears the recurrence's share of the status word (ffn_scan.cu).
cudaError_t scan_status(int* v);

inline int op_launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? FFN_OK : op_fail(FFN_E_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// Streaming multiprocessors of the current device (the attribute query is cached by the runtime).
inline int op_sms() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        return 0;
    return n;
}

inline bool op_aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__nv_fp8_e4m3 v) { return static_cast<float>(v); }

template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as one access of N * sizeof(T) bytes (4, 8 or 16; or one element).
template <int BYTES> struct Raw;
template <> struct Raw<2> { using type = unsigned short; };
template <> struct Raw<4> { using type = unsigned int; };
template <> struct Raw<8> { using type = uint2; };
template <> struct Raw<16> { using type = uint4; };

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
    using R = typename Raw<sizeof(T) * N>::type;
    const R r = __ldg(reinterpret_cast<const R*>(p));
    return *reinterpret_cast<const Pack<T, N>*>(&r);
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& v) {
    using R = typename Raw<sizeof(T) * N>::type;
    *reinterpret_cast<R*>(p) = *reinterpret_cast<const R*>(&v);
}

// Maximum that keeps a NaN (fmaxf drops it): a row with a NaN has to get a NaN scale.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

constexpr float E4M3_MAX = 448.0f;

// The scale of values whose largest magnitude is `top`, and the factor that applies it.  A scale that
// would be zero is 1 (the values are then zero, or vanish); a factor that would be infinite (scales
// below 2^-128) is the largest finite one, so that a zero stays a zero.  A NaN stays a NaN.
__device__ __forceinline__ float e4m3_scale(float top) {
    const float s = __fdiv_rn(top, E4M3_MAX);
    return s == 0.0f ? 1.0f : s;
}
__device__ __forceinline__ float e4m3_inverse(float scale) {
    const float v = __fdiv_rn(1.0f, scale);
    return v > 3.402823466e38f ? 3.402823466e38f : v;
}

// Four fp32 values to four e4m3 bytes, nearest even, saturating at +-448; a NaN stays a NaN.
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

}  // namespace ffn
