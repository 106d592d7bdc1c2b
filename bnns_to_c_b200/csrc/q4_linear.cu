// q4_linear.cu - the 4-bit linear layer of include/bnn_lowbit.h.
#include <new>

#include "lowbit_dev.cuh"

struct bnn_q4_layer {
    int device;
    int type;
    bnn::lowbit::Q4Geo geo;
    void* base;              // one allocation, in this order:
    const uint32_t* codes;   //   q4_words
    const uint16_t* scales;  //   q4_scales, in the layer's type
    const uint8_t* zeros;    //   q4_scales
    const float* bias;       //   [n_out] or nullptr
};

namespace bnn {
namespace lowbit {
namespace {

// ---------------------------------------------------------------- layout, once
// Padding: an input behind the last has code = zero point (weight 0), a row
// behind the last has scale 0.
__global__ void q4_layout_kernel(Q4Geo g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros, uint32_t* wo,
                                 uint16_t* so, uint8_t* zo) {
    const int64_t words = q4_words(g), step = (int64_t)gridDim.x * blockDim.x;
    const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t half = ((int64_t)g.K + 1) / 2;
    for (int64_t w = first; w < words; w += step) {
        const int i = (int)(w & 3), lane = (int)(w >> 2) & 31;
        const int64_t tk = w >> 7;
        const int tile = (int)(tk / g.kb), kb = (int)(tk % g.kb);
        uint32_t v = 0;
        for (int nib = 0; nib < 8; ++nib) {
            const int row = tile * 16 + q4_row(lane, nib), k = kb * 64 + q4_in(lane, i, nib);
            uint32_t q = 8;
            if (row < g.N) {
                if (k < g.K)
                    q = (codes[row * half + (k >> 1)] >> (4 * (k & 1))) & 15u;
                else if (zeros)
                    q = zeros[(int64_t)row * g.ng + min(k / g.group, g.ng - 1)] & 15u;
            }
            v |= q << (4 * (nib & 3) + 16 * (nib >> 2));
        }
        wo[w] = v;
    }
    for (int64_t s = first; s < (int64_t)g.tiles * 16 * g.ng; s += step) {
        const int row = (int)(s / g.ng), grp = (int)(s % g.ng);
        const int64_t at = q4_scale(g, row, grp);
        so[at] = row < g.N ? scales[s] : (uint16_t)0;
        zo[at] = row < g.N && zeros ? (uint8_t)(zeros[s] & 15u) : (uint8_t)8;
    }
}

struct Q4Params {
    Q4Geo g;
    const uint4* w;
    const uint32_t* s;  // pairs (row r, row r + 8)
    const uint16_t* z;  // pairs
    const float* bias;
    const uint16_t* x;
    int64_t xs;
    uint16_t* y;
    int64_t ys;
    int M;
    bool vec;  // rows of x are 16-byte aligned
};

// ---------------------------------------------------------------- rows on mma.sync
// One CTA makes a tile of 16 outputs for 8 * NT rows of x; its 8 warps take
// the 64-input blocks in turn and their sums are joined in shared memory.
// (q - z) is exact in 16 bits (|q - z| <= 15), so a group's sum of products
// has only the rounding of 32-bit sums, and its scale is applied to that sum.
constexpr int kQ4Warps = 8;

template <class A, int NT>
__global__ void __launch_bounds__(32 * kQ4Warps) q4_rows_kernel(const Q4Params p) {
    __shared__ float red[kQ4Warps][8 * NT][17];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = lane >> 2, j = lane & 3;
    const int tile = blockIdx.x, m0 = blockIdx.y * 8 * NT;
    const Q4Geo g = p.g;
    float acc[NT][4] = {};
    for (int kb = warp; kb < g.kb; kb += kQ4Warps) {
        const uint4 w4 = ldg_stream(p.w + ((int64_t)tile * g.kb + kb) * 32 + lane);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = kb * 64 + h * 32, grp = min(k / g.group, g.ng - 1);
            const int64_t at = ((int64_t)tile * g.ng + grp) * 8 + r;
            const uint32_t zz = p.z[at], ss = p.s[at];
            const uint32_t z0 = (zz & 0xffu) * 0x00010001u | A::kMagic, z1 = (zz >> 8) * 0x00010001u | A::kMagic;
            uint4 xv[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int m = m0 + t * 8 + r, kk = k + 8 * j;
                xv[t] = m < p.M && kk < g.K ? load8(p.x + m * p.xs + kk, g.K - kk, p.vec) : make_uint4(0, 0, 0, 0);
            }
            float c[NT][4] = {};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t v = w[h * 2 + i];
                uint32_t a[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    a[q] = A::sub2(((v >> (4 * q)) & 0x000f000fu) | A::kMagic, q & 1 ? z1 : z0);
#pragma unroll
                for (int t = 0; t < NT; ++t) A::mma(c[t], a, i ? xv[t].z : xv[t].x, i ? xv[t].w : xv[t].y);
            }
            const uint16_t sh0 = (uint16_t)ss, sh1 = (uint16_t)(ss >> 16);
            const float s0 = A::to_float(*reinterpret_cast<const typename A::T*>(&sh0));
            const float s1 = A::to_float(*reinterpret_cast<const typename A::T*>(&sh1));
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                acc[t][0] = fmaf(s0, c[t][0], acc[t][0]);
                acc[t][1] = fmaf(s0, c[t][1], acc[t][1]);
                acc[t][2] = fmaf(s1, c[t][2], acc[t][2]);
                acc[t][3] = fmaf(s1, c[t][3], acc[t][3]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) red[warp][t * 8 + 2 * j + (e & 1)][r + 8 * (e >> 1)] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 128 * NT; i += blockDim.x) {
        const int m = m0 + (i >> 4), n = tile * 16 + (i & 15);
        if (m >= p.M || n >= g.N) continue;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kQ4Warps; ++k) v += red[k][i >> 4][i & 15];
        if (p.bias) v += p.bias[n];
        const typename A::T o = A::from_float(v);
        p.y[m * p.ys + n] = *reinterpret_cast<const uint16_t*>(&o);
    }
}

template <class A, int NT>
cudaError_t q4_launch(const Q4Params& p, cudaStream_t st) {
    const dim3 grid((unsigned)p.g.tiles, (unsigned)cdiv64(p.M, 8 * NT));
    q4_rows_kernel<A, NT><<<grid, 32 * kQ4Warps, 0, st>>>(p);
    return cudaGetLastError();
}
template <class A>
cudaError_t q4_run(const Q4Params& p, cudaStream_t st) {
    if (p.M <= 8) return q4_launch<A, 1>(p, st);
    if (p.M <= 16) return q4_launch<A, 2>(p, st);
    return q4_launch<A, 4>(p, st);
}

int q4_create(bnn_q4_layer* L, const uint8_t* codes, const void* scales, const uint8_t* zeros, const float* bias) {
    const Q4Geo& g = L->geo;
    DeviceScope dev(L->device);
    if (dev.err != cudaSuccess) return cuda_error("bnn_q4_layer_create", dev.err);
    const auto up = [](int64_t n) { return (size_t)((n + 255) & ~(int64_t)255); };
    const size_t bw = up(q4_words(g) * 4), bs = up(q4_scales(g) * 2), bz = up(q4_scales(g)), bb = bias ? up((int64_t)g.N * 4) : 0;
    int rc = device_alloc(&L->base, bw + bs + bz + bb, "of a 4-bit layer");
    if (rc) return rc;
    char* at = (char*)L->base;
    L->codes = (const uint32_t*)at;
    L->scales = (const uint16_t*)(at + bw);
    L->zeros = (const uint8_t*)(at + bw + bs);
    L->bias = bias ? (const float*)(at + bw + bs + bz) : nullptr;
    // the caller's arrays (host or device memory) in device memory, for the layout kernel
    const int64_t half = ((int64_t)g.K + 1) / 2, ns = (int64_t)g.N * g.ng;
    const size_t rw = up(g.N * half), rs = up(ns * 2), rz = zeros ? up(ns) : 0;
    void* tmp = nullptr;
    if ((rc = device_alloc(&tmp, rw + rs + rz, "of a 4-bit layer's raw arrays"))) return rc;
    uint8_t *dw = (uint8_t*)tmp, *ds = dw + rw, *dz = ds + rs;
    cudaError_t e = cudaMemcpy(dw, codes, g.N * half, cudaMemcpyDefault);
    if (e == cudaSuccess) e = cudaMemcpy(ds, scales, ns * 2, cudaMemcpyDefault);
    if (e == cudaSuccess && zeros) e = cudaMemcpy(dz, zeros, ns, cudaMemcpyDefault);
    if (e == cudaSuccess && bias) e = cudaMemcpy((void*)L->bias, bias, (size_t)g.N * 4, cudaMemcpyDefault);
    if (e == cudaSuccess) {
        const int64_t blocks = cdiv64(q4_words(g), 256);
        q4_layout_kernel<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256>>>(
            g, dw, (const uint16_t*)ds, zeros ? dz : nullptr, (uint32_t*)L->codes, (uint16_t*)L->scales, (uint8_t*)L->zeros);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    cudaFree(tmp);
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_q4_layer_create", e);
}

}  // namespace
}  // namespace lowbit
}  // namespace bnn

using namespace bnn;
using namespace bnn::lowbit;

BNN_API int bnn_q4_layer_create(int device, int n_in, int n_out, int group, int type, const uint8_t* codes,
                                const void* scales, const uint8_t* zeros, const float* bias, bnn_q4_layer** out) {
    if (!out) return set_error(BNN_ERR_ARG, "NULL argument");
    *out = nullptr;
    if (!codes || !scales) return set_error(BNN_ERR_ARG, "NULL codes or scales");
    if (device < -1 || n_in <= 0 || n_out <= 0 || n_in > (1 << 24) || n_out > (1 << 24))
        return set_error(BNN_ERR_ARG, "device %d, %d inputs, %d outputs (1 .. 2^24)", device, n_in, n_out);
    if (group <= 0 || group % 32) return set_error(BNN_ERR_ARG, "group %d: a multiple of 32", group);
    if (type != BNN_BF16 && type != BNN_FP16) return set_error(BNN_ERR_ARG, "type %d: BNN_BF16 or BNN_FP16", type);
    auto* L = new (std::nothrow) bnn_q4_layer();
    if (!L) return set_error(BNN_ERR_OOM, "OOM");
    L->device = device;
    L->type = type;
    L->geo = q4_geo(n_in, n_out, group);
    const int rc = device < 0 ? BNN_OK : q4_create(L, codes, scales, zeros, bias);
    if (rc) {
        bnn_q4_layer_destroy(L);
        return rc;
    }
    *out = L;
    return BNN_OK;
}

BNN_API int bnn_q4_layer_run(const bnn_q4_layer* L, const void* d_x, int64_t x_stride, int rows, void* d_y,
                             int64_t y_stride, void* stream) {
    if (!L || rows < 0) return set_error(BNN_ERR_ARG, "bad arguments");
    const Q4Geo& g = L->geo;
    if (rows > 0 && (!d_x || !d_y)) return set_error(BNN_ERR_ARG, "NULL x or y");
    if (rows > 0 && (!aligned(d_x, 2) || !aligned(d_y, 2))) return set_error(BNN_ERR_ARG, "x and y: aligned to 2 bytes");
    if (rows > 1 && (x_stride < g.K || y_stride < g.N))
        return set_error(BNN_ERR_ARG, "strides %lld, %lld: at least %d, %d", (long long)x_stride, (long long)y_stride, g.K, g.N);
    if (rows > (1 << 19)) return set_error(BNN_ERR_ARG, "%d rows: at most 2^19", rows);
    if (L->device < 0) return no_device("bnn_q4_layer_run");
    if (rows == 0) return BNN_OK;
    DeviceScope dev(L->device);
    if (dev.err != cudaSuccess) return cuda_error("bnn_q4_layer_run", dev.err);
    Q4Params p{};
    p.g = g;
    p.w = (const uint4*)L->codes;
    p.s = (const uint32_t*)L->scales;
    p.z = (const uint16_t*)L->zeros;
    p.bias = L->bias;
    p.x = (const uint16_t*)d_x;
    p.xs = x_stride;
    p.y = (uint16_t*)d_y;
    p.ys = y_stride;
    p.M = rows;
    p.vec = aligned(d_x, 16) && (rows == 1 || x_stride % 8 == 0);
    const cudaError_t e = L->type == BNN_BF16 ? q4_run<Bf16>(p, (cudaStream_t)stream) : q4_run<Fp16>(p, (cudaStream_t)stream);
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_q4_layer_run", e);
}

BNN_API void bnn_q4_layer_destroy(bnn_q4_layer* L) {
    if (!L) return;
    if (L->base) {
        DeviceScope dev(L->device);
        cudaFree(L->base);
    }
    delete L;
}
