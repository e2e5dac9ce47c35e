// jdg_devop.cuh — shared by the device operators (jdg_paged.cu, jdg_beam.cu): element types,
// vector loads and stores of 4 elements, and the host side of a call on a caller's stream.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/jdgpu.h"
#include "jdg_common.cuh"
#include "jdg_engine.h"

namespace jdg {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kDevSMs = 148;  // grid sizing only: nothing depends on the count being exact

inline int devop_size(int dt) { return dt == JD_F32 ? 4 : dt == JD_F16 || dt == JD_BF16 ? 2 : 0; }

// The stream a call is given must belong to the current device (function attributes and the
// caller's pointers do).  A stream in capture may not be asked for its device (that would end the
// capture); there the launch itself refuses a stream of another device.
inline int devop_stream(const char *who, cudaStream_t st, int *dev) {
    cudaError_t e = cudaGetDevice(dev);
    int sdev = *dev;
    if (e == cudaSuccess && st && st != cudaStreamLegacy && st != cudaStreamPerThread) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        e = cudaStreamIsCapturing(st, &cap);
        if (e == cudaSuccess && cap == cudaStreamCaptureStatusNone) e = cudaStreamGetDevice(st, &sdev);
    }
    if (e != cudaSuccess) {
        jdg_set_err(nullptr, "%s: no usable device or stream: %s", who, cudaGetErrorString(e));
        return JD_ECUDA;
    }
    if (sdev != *dev) {
        jdg_set_err(nullptr, "%s: the stream is not on the current device (%d vs %d)", who, sdev, *dev);
        return JD_EINVAL;
    }
    return JD_OK;
}

// Dynamic shared memory above 48 KB has to be allowed per kernel and device; done once for
// each (a mask of devices per kernel, no lock: setting it twice is harmless).
template <auto Kern>
inline int devop_smem(const char *who, int dev, int bytes) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return JD_OK;
    cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
        jdg_set_err(nullptr, "%s: cudaFuncSetAttribute(%d bytes) failed: %s", who, bytes, cudaGetErrorString(e));
        return JD_ECUDA;
    }
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return JD_OK;
}

// Launch, optionally as a programmatic dependent of the stream's previous kernel (which must be
// one of this call's own: the kernel then waits with griddepcontrol.wait where it needs it).
template <typename... KArgs, typename... Args>
inline int devop_launch(const char *who, bool pdl, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem,
                        cudaStream_t st, Args... args) {
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = pdl ? 1 : 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) {
        jdg_set_err(nullptr, "%s: launch failed: %s", who, cudaGetErrorString(e));
        return JD_ECUDA;
    }
    return JD_OK;
}

__device__ __forceinline__ void dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dep_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// two f32 at a time
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<const unsigned long long &>(a)), "l"(reinterpret_cast<const unsigned long long &>(b)),
          "l"(reinterpret_cast<const unsigned long long &>(c)));
    return r;
}

// 2^x, within 2 ulp
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// two packed elements of a 32-bit word (low half first)
__device__ __forceinline__ float2 unpack2(uint32_t w, const __half *) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, const __nv_bfloat16 *) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __half *) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, const __nv_bfloat16 *) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 4 consecutive elements, aligned to their 4 elements
__device__ __forceinline__ float4 ld4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <typename T>
__device__ __forceinline__ float4 ld4(const T *p) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = unpack2(w.x, p), b = unpack2(w.y, p);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void st4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
template <typename T>
__device__ __forceinline__ void st4(T *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(v.x, v.y, p), pack2(v.z, v.w, p));
}

// 16 bytes global -> shared, asynchronously; pred false writes zeros and reads nothing
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool pred) {
    const int n = pred ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace jdg
