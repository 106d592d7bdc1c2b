// lowbit_dev.cuh - device and host helpers of the low-bit operators
// (q4_linear.cu, kv_cache.cu, kv_attend.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdlib>

#include "../../include/bnn_lowbit.h"
#include "common.h"
#include "lowbit.h"

namespace bnn {
namespace lowbit {

// ---------------------------------------------------------------- host side
// makes a device current, and the caller's again at the end of the scope
struct DeviceScope {
    int prev = -1;
    bool changed = false;
    cudaError_t err;
    explicit DeviceScope(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) {
            err = cudaSetDevice(device);
            changed = true;
        }
    }
    ~DeviceScope() {
        if (changed) cudaSetDevice(prev);
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
// Whether rows of `dim` elements, n of them `row` apart in each of `heads`
// heads `head` apart (each at least dim), share elements. Heads woven into
// rows, or rows into heads, are told at once; else each head's start is
// compared with the rows next to it.
inline bool rows_share(int64_t n, int64_t row, int64_t heads, int64_t head, int64_t dim) {
    if (n <= 1 || heads <= 1 || (__int128)row >= (__int128)(heads - 1) * head + dim || (__int128)head >= (__int128)(n - 1) * row + dim)
        return false;
    for (int64_t h = 1; h < heads; ++h) {
        const __int128 at = (__int128)h * head;
        if (at >= (__int128)n * row) break;  // behind the last row, which is dim wide at most
        const int64_t i = (int64_t)(at / row), behind = (int64_t)(at - (__int128)i * row);
        if (behind < dim || (i + 1 < n && row - behind < dim)) return true;
    }
    return false;
}
// Kernels here are launched as programmatic dependents of what is before them
// in the stream: they may start while it ends, and wait for it (grid_wait)
// before they touch anything that another kernel can have written or still
// reads. Every CTA waits, so that a kernel that has ended stands for all
// before it. BNN_PDL=0 in the environment turns this off, as for the engine.
inline bool pdl_on() {
    static const bool on = [] {
        const char* e = getenv("BNN_PDL");
        return !(e && e[0] == '0');
    }();
    return on;
}
template <class K, class... Args>
cudaError_t launch_cluster(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, bool early, int cluster_z, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (early && pdl_on()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster_z > 0) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = at[n].val.clusterDim.y = 1;
        at[n++].val.clusterDim.z = (unsigned)cluster_z;
    }
    cfg.attrs = at;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <class K, class... Args>
cudaError_t launch(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, bool early, const Args&... args) {
    return launch_cluster(kernel, grid, threads, smem, st, early, 0, args...);
}
inline int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---------------------------------------------------------------- device side
// (What other kernels write is read by plain loads behind the wait: a
// read-only load may be served, or moved, from before it.)
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void grid_launch() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }

// (a & b) | c in one instruction (the compiler makes two of two constants)
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
struct Bf16 {
    using T = __nv_bfloat16;
    // a 4-bit code in the low mantissa bits of this half is kMagic's value + code, exactly
    static constexpr uint32_t kMagic = 0x43004300u;  // 128 in both halves
    static __device__ __forceinline__ float to_float(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T from_float(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ float2 unpack(uint32_t w) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
        const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kMmaType = 1;  // operand type in a tcgen05 kind::f16 instruction descriptor
    static constexpr CUtensorMapDataType kTmaType = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // the four registers of an A fragment from its word: code - zero point,
    // z0 and z1 = magic + zero point of rows r and r + 8, twice
    static __device__ __forceinline__ void weights(uint32_t* a, uint32_t w, uint32_t z0, uint32_t z1) {
#pragma unroll
        for (int b = 0; b < 4; ++b) a[b] = sub2(and_or(w >> (4 * b), 0x000f000fu, kMagic), b & 1 ? z1 : z0);
    }
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {  // sums from 0
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};
struct Fp16 {
    using T = __half;
    static constexpr uint32_t kMagic = 0x64006400u;  // 1024 in both halves
    static __device__ __forceinline__ float to_float(T v) { return __half2float(v); }
    static __device__ __forceinline__ T from_float(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
    static __device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
        const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
        const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static constexpr uint32_t kMmaType = 0;  // operand type in a tcgen05 kind::f16 instruction descriptor
    static constexpr CUtensorMapDataType kTmaType = CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // as above; 10 mantissa bits also hold the next nibble, as 1024 + 16 *
    // code, so two of the three shifts are saved: / 16 - (64 + zero point)
    static __device__ __forceinline__ void weights(uint32_t* a, uint32_t w, uint32_t z0, uint32_t z1) {
        const uint32_t n1 = sub2(0x63806380u, z1);  // 960 - (1024 + zero point)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint32_t v = w >> (8 * b);
            a[2 * b] = sub2(and_or(v, 0x000f000fu, kMagic), z0);
            const uint32_t o = and_or(v, 0x00f000f0u, kMagic), s = 0x2c002c00u;  // 1 / 16
            const __half2 f = __hfma2(*reinterpret_cast<const __half2*>(&o), *reinterpret_cast<const __half2*>(&s),
                                      *reinterpret_cast<const __half2*>(&n1));
            a[2 * b + 1] = *reinterpret_cast<const uint32_t*>(&f);
        }
    }
    static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
    static __device__ __forceinline__ void mma0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {  // sums from 0
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};

// 8 neighbouring 16-bit values p[0..7], those from n on as zeros
__device__ __forceinline__ uint4 load8(const uint16_t* p, int n, bool vec) {
    if (vec && n >= 8) return *reinterpret_cast<const uint4*>(p);
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ uint2 load4(const uint16_t* p, int n) {
    uint32_t v[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) v[i >> 1] |= (uint32_t)p[i] << (16 * (i & 1));
    return make_uint2(v[0], v[1]);
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
// two floats at a time, each operation rounded to nearest as a single one is
__device__ __forceinline__ uint64_t both(float x, float y) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
    return v;
}
__device__ __forceinline__ float2 apart(uint64_t v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ float bf16_float(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// ---------------------------------------------------------------- mbarriers, TMA, tcgen05
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_arrive_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded: gives up after 2^22 rounds (seconds; a hand-off takes a
// microsecond) or when another wait of the CTA has, and sets the flag.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    for (int it = 0; it < (1 << 22); ++it) {
        uint32_t done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((it & 255) == 255 && *gave_up) return false;
    }
    *gave_up = 1;
    return false;
}
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(is));
    return is != 0;
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void t5_alloc(uint32_t smem_dst, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_dst), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void t5_free(uint32_t taddr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void t5_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void t5_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void t5_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}
// D (+)= A[tensor memory] * B[shared memory], 16-bit operands, K = 16, fp32 sums
__device__ __forceinline__ void t5_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
// 16 lanes x 32 columns: register 4i + {0, 1 | 2, 3} of lane (r, j) goes to
// lanes r | r + 8, columns 8i + 2j + {0, 1}
__device__ __forceinline__ void t5_st_16x256b_x4(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void t5_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// 16 columns of this thread's lane
__device__ __forceinline__ void t5_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

}  // namespace lowbit
}  // namespace bnn
