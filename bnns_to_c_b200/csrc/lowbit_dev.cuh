// lowbit_dev.cuh - device and host helpers of the low-bit operators
// (q4_linear.cu, kv_cache.cu, kv_attend.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/bnn_lowbit.h"
#include "common.h"
#include "lowbit.h"

namespace bnn {
namespace lowbit {

// ---------------------------------------------------------------- host side
// makes a device current, and the caller's again at the end of the scope
struct DeviceScope {
    int prev = -1;
    cudaError_t err;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
    }
    ~DeviceScope() {
        int now = -1;
        if (prev >= 0 && cudaGetDevice(&now) == cudaSuccess && now != prev) cudaSetDevice(prev);
    }
};

inline int cuda_error(const char* what, cudaError_t e) {
    return set_error(BNN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}
// the device of a handle made with device = -1
inline int no_device(const char* what) {
    return set_error(BNN_ERR_CUDA, "%s: the handle was made without a device", what);
}
inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------- device side
struct Bf16 {
    using T = __nv_bfloat16;
    // a 4-bit code in the low mantissa bits of this half is kMagic's value + code, exactly
    static constexpr uint32_t kMagic = 0x43004300u;  // 128 in both halves
    static __device__ __forceinline__ float to_float(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
struct Fp16 {
    using T = __half;
    static constexpr uint32_t kMagic = 0x64006400u;  // 1024 in both halves
    static __device__ __forceinline__ float to_float(T v) { return __half2float(v); }
    static __device__ __forceinline__ T from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// 8 neighbouring 16-bit values p[0..7], those from n on as zeros
__device__ __forceinline__ uint4 load8(const uint16_t* p, int n, bool vec) {
    if (vec && n >= 8) return *reinterpret_cast<const uint4*>(p);
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store8(uint16_t* p, uint4 v, int n, bool vec) {
    if (vec && n >= 8) {
        *reinterpret_cast<uint4*>(p) = v;
        return;
    }
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
}
// the two 16-bit values of a word as floats
__device__ __forceinline__ float2 unpack2(uint32_t w, bool fp16) {
    if (fp16) return __half22float2(*reinterpret_cast<__half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, bool fp16) {
    if (fp16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float bf16_float(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

}  // namespace lowbit
}  // namespace bnn
