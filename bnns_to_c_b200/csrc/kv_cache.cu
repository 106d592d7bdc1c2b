// kv_cache.cu - the block-scaled key/value cache of include/bnn_lowbit.h:
// create, write (quantise as it is stored) and read.
#include <new>
#include <utility>

#include "kv_cache.h"
#include "lowbit_dev.cuh"

namespace bnn {
namespace lowbit {
namespace {

struct KvRows {
    KvGeo g;
    uint8_t* codes[2];    // keys, values
    uint16_t* scales[2];
    uint16_t* x[2];       // the caller's rows
    int64_t token[2], head[2];
    int n_tokens, n_seqs, width;
    const int32_t *table, *start, *off;
    bool vec[2], fp16;
};

// page and place in it of row t; false: the row has none
__device__ __forceinline__ bool kv_place(const KvRows& p, int t, int& page, int& tok) {
    const int b = p.off ? kv_seq(p.off, p.n_seqs, t) : t;
    if (b < 0) return false;
    const int64_t pos = (int64_t)p.start[b] + (p.off ? (int64_t)t - p.off[b] : 0);
    if (pos < 0 || pos > 0x7fffffff) return false;
    page = kv_page(p.g, p.table + (int64_t)b * p.width, p.width, (int)pos);
    tok = (int)pos & (p.g.pt - 1);
    return page >= 0;
}

// Both kernels: W = dp / 8 neighbouring lanes (32 for dp = 192) have one
// head of one token's keys or values, 8 numbers each: 16 bytes of the
// caller's row. Bound by those rows' bytes.
//
// The codes. x has at most 11 significant bits (24-bit sums are not at work
// here) and the scale 8, so x / scale is at least 2^-12 away from a border
// k + 1/2 that it does not hit exactly, far more than the rounding of the
// 32-bit quotient (2^-17 at 127): rounding that quotient to even gives the
// code of the exact quotient. The scale: max / top in 32 bits, then to 8
// bits; the exact quotient is, by the same argument with top for the scale,
// not within 2^-17 of a border of bf16 that it does not hit, so the two
// roundings give the one rounding of the definition.
template <int W>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvRows p) {
    const KvGeo g = p.g;
    const int i = threadIdx.x % W;  // numbers 8 * i .. of the head
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / W;
    const int which = blockIdx.y;
    const bool in = unit < (int64_t)p.n_tokens * g.heads;
    const int t = in ? (int)(unit / g.heads) : 0, head = in ? (int)(unit % g.heads) : 0;
    int page = 0, tok = 0;
    const bool there = in && kv_place(p, t, page, tok);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (there && 8 * i < g.dim) v = load8(p.x[which] + t * p.token[which] + head * p.head[which] + 8 * i, g.dim - 8 * i, p.vec[which]);
    float x[8];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;  // |x| as bits: an order that puts NaN above infinity above all numbers
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float2 f = unpack2(w[c], p.fp16);
        x[2 * c] = f.x;
        x[2 * c + 1] = f.y;
        top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
    // lanes of a group: group / 8 (a power of two), or all W of one group
    const int lanes = g.ng == 1 ? W : g.group / 8;
    for (int s = 1; s < lanes; s <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
    const int most = g.bits == 8 ? 127 : 7;
    const bool bad = top >= 0x7f800000u;
    const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(bad ? 0.0f : __uint_as_float(top), (float)most));
    const float s = __bfloat162float(sb);
    uint32_t code[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const float q = s > 0.0f && !bad ? rintf(__fdiv_rn(x[c], s)) : 0.0f;
        code[c] = (uint32_t)((int)fminf(fmaxf(q, -(float)most), (float)most) + most + 1);
    }
    if (!there || 8 * i >= g.dp) return;
    const int grp = g.ng == 1 ? 0 : 8 * i / g.group;
    if (grp < g.ng && (g.ng == 1 ? i == 0 : 8 * i % g.group == 0))
        p.scales[which][kv_scale(g, page, head, grp, tok)] = bad ? (uint16_t)0x7fff : *reinterpret_cast<const uint16_t*>(&sb);
    uint8_t* row = p.codes[which] + kv_row(g, page, head, tok);
    if (g.bits == 8) {
        const uint32_t a = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
        const uint32_t b = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
        if (which == 0) {
            *reinterpret_cast<uint2*>(row + kv_k_at(g, i)) = make_uint2(a, b);
        } else {
            *reinterpret_cast<uint32_t*>(row + kv_v_at(g, 2 * i)) = a;
            *reinterpret_cast<uint32_t*>(row + kv_v_at(g, 2 * i + 1)) = b;
        }
    } else if (which == 0) {
        uint32_t a = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) a |= code[c] << (4 * (c >> 1) + 16 * (c & 1));
        *reinterpret_cast<uint32_t*>(row + kv_k_at(g, i)) = a;
    } else {
        *reinterpret_cast<uint16_t*>(row + kv_v_at(g, 2 * i)) = (uint16_t)(code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12);
        *reinterpret_cast<uint16_t*>(row + kv_v_at(g, 2 * i + 1)) = (uint16_t)(code[4] | code[5] << 4 | code[6] << 8 | code[7] << 12);
    }
}

template <int W>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvRows p) {
    const KvGeo g = p.g;
    const int i = threadIdx.x % W;
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / W;
    const int which = blockIdx.y;
    if (unit >= (int64_t)p.n_tokens * g.heads || 8 * i >= g.dim) return;
    const int t = (int)(unit / g.heads), head = (int)(unit % g.heads);
    int page, tok;
    if (!kv_place(p, t, page, tok)) return;
    const int grp = g.ng == 1 ? 0 : 8 * i / g.group;
    const float s = bf16_float(p.scales[which][kv_scale(g, page, head, grp, tok)]);
    const uint8_t* row = p.codes[which] + kv_row(g, page, head, tok);
    uint32_t code[8];
    if (g.bits == 8) {
        uint2 v;
        if (which == 0) {
            v = *reinterpret_cast<const uint2*>(row + kv_k_at(g, i));
        } else {
            v.x = *reinterpret_cast<const uint32_t*>(row + kv_v_at(g, 2 * i));
            v.y = *reinterpret_cast<const uint32_t*>(row + kv_v_at(g, 2 * i + 1));
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) code[c] = ((c < 4 ? v.x : v.y) >> (8 * (c & 3))) & 255u;
    } else if (which == 0) {
        const uint32_t v = *reinterpret_cast<const uint32_t*>(row + kv_k_at(g, i));
#pragma unroll
        for (int c = 0; c < 8; ++c) code[c] = (v >> (4 * (c >> 1) + 16 * (c & 1))) & 15u;
    } else {
        const uint32_t v = *reinterpret_cast<const uint16_t*>(row + kv_v_at(g, 2 * i)) |
                           (uint32_t)*reinterpret_cast<const uint16_t*>(row + kv_v_at(g, 2 * i + 1)) << 16;
#pragma unroll
        for (int c = 0; c < 8; ++c) code[c] = (v >> (4 * c)) & 15u;
    }
    const int zero = g.bits == 8 ? 128 : 8;
    float x[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) x[c] = (float)((int)code[c] - zero) * s;  // 7 bits times 8: exact, rounded once below
    const uint4 o = make_uint4(pack2(x[0], x[1], p.fp16), pack2(x[2], x[3], p.fp16), pack2(x[4], x[5], p.fp16),
                               pack2(x[6], x[7], p.fp16));
    store8(p.x[which] + t * p.token[which] + head * p.head[which] + 8 * i, o, g.dim - 8 * i, p.vec[which]);
}

template <bool WRITE>
int kv_rows(const char* what, const bnn_kv_cache* c, const void* k, int64_t k_token, int64_t k_head, const void* v,
            int64_t v_token, int64_t v_head, int n_tokens, int n_seqs, const int32_t* table, int width,
            const int32_t* start, const int32_t* off, void* stream) {
    if (!c || n_tokens < 0 || n_seqs < 0 || width < 0) return set_error(BNN_ERR_ARG, "%s: bad arguments", what);
    const KvGeo& g = c->geo;
    if (!off && n_tokens != n_seqs)
        return set_error(BNN_ERR_ARG, "%s: %d tokens of %d sequences need offsets", what, n_tokens, n_seqs);
    const bool work = n_tokens > 0 && n_seqs > 0 && width > 0;
    if (work) {
        if (!k || !v || !table || !start) return set_error(BNN_ERR_ARG, "%s: NULL argument", what);
        if (!aligned(k, 2) || !aligned(v, 2) || !aligned(table, 4) || !aligned(start, 4) || !aligned(off, 4))
            return set_error(BNN_ERR_ARG, "%s: an array is not aligned to its type", what);
        if (!WRITE)  // rows of an output must not lie over one another
            for (const auto& s : {std::pair<int64_t, int64_t>(k_token, k_head), std::pair<int64_t, int64_t>(v_token, v_head)})
                if ((g.heads > 1 && s.second < g.dim) || (n_tokens > 1 && s.first < g.dim))
                    return set_error(BNN_ERR_ARG, "%s: strides %lld, %lld of an output: at least %d", what, (long long)s.first,
                                     (long long)s.second, g.dim);
    }
    if (c->device < 0) return no_device(what);
    if (!work) return BNN_OK;
    DeviceScope dev(c->device);
    if (dev.err != cudaSuccess) return cuda_error(what, dev.err);
    KvRows p{};
    p.g = g;
    p.codes[0] = c->kc, p.codes[1] = c->vc, p.scales[0] = c->ks, p.scales[1] = c->vs;
    p.x[0] = (uint16_t*)k, p.x[1] = (uint16_t*)v;
    p.token[0] = k_token, p.head[0] = k_head, p.token[1] = v_token, p.head[1] = v_head;
    p.n_tokens = n_tokens, p.n_seqs = n_seqs, p.width = width;
    p.table = table, p.start = start, p.off = off;
    p.fp16 = c->type == BNN_FP16;
    for (int w = 0; w < 2; ++w)
        p.vec[w] = aligned(p.x[w], 16) && (n_tokens == 1 || p.token[w] % 8 == 0) && (g.heads == 1 || p.head[w] % 8 == 0);
    const int W = g.dp == 64 ? 8 : g.dp == 128 ? 16 : 32;
    const int64_t blocks = cdiv64((int64_t)n_tokens * g.heads * W, 256);
    if (blocks > 0x7fffffff) return set_error(BNN_ERR_ARG, "%s: %d tokens are too many for one call", what, n_tokens);
    const dim3 grid((unsigned)blocks, 2);
    const cudaStream_t st = (cudaStream_t)stream;
    if (WRITE) {
        if (W == 8) kv_write_kernel<8><<<grid, 256, 0, st>>>(p);
        else if (W == 16) kv_write_kernel<16><<<grid, 256, 0, st>>>(p);
        else kv_write_kernel<32><<<grid, 256, 0, st>>>(p);
    } else {
        if (W == 8) kv_read_kernel<8><<<grid, 256, 0, st>>>(p);
        else if (W == 16) kv_read_kernel<16><<<grid, 256, 0, st>>>(p);
        else kv_read_kernel<32><<<grid, 256, 0, st>>>(p);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BNN_OK : cuda_error(what, e);
}

int kv_create(bnn_kv_cache* c) {
    const KvGeo& g = c->geo;
    DeviceScope dev(c->device);
    if (dev.err != cudaSuccess) return cuda_error("bnn_kv_cache_create", dev.err);
    cudaError_t e = cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, c->device);
    if (e == cudaSuccess) e = attend_setup(g);
    if (e != cudaSuccess) return cuda_error("bnn_kv_cache_create", e);
    const int rc = device_alloc(&c->base, c->bytes, "of a key/value cache");
    if (rc) return rc;
    const size_t bc = (size_t)(kv_code_bytes(g) + 255) & ~(size_t)255, bs = (size_t)(kv_scales(g) * 2 + 255) & ~(size_t)255;
    c->kc = (uint8_t*)c->base;
    c->vc = c->kc + bc;
    c->ks = (uint16_t*)(c->vc + bc);
    c->vs = (uint16_t*)((uint8_t*)c->ks + bs);
    // scales 0: every position reads back as zeros until it is written
    e = cudaMemset(c->base, 0, c->bytes);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_kv_cache_create", e);
}

}  // namespace
}  // namespace lowbit
}  // namespace bnn

using namespace bnn;
using namespace bnn::lowbit;

BNN_API int bnn_kv_cache_create(int device, int pages, int page_tokens, int kv_heads, int head_dim, int bits, int group,
                                int type, bnn_kv_cache** out) {
    if (!out) return set_error(BNN_ERR_ARG, "NULL argument");
    *out = nullptr;
    if (device < -1 || pages <= 0 || kv_heads <= 0 || kv_heads > 4096)
        return set_error(BNN_ERR_ARG, "device %d, %d pages, %d heads (1 .. 4096)", device, pages, kv_heads);
    if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)))
        return set_error(BNN_ERR_ARG, "pages of %d tokens: 16, 32, 64, 128 or 256", page_tokens);
    if (head_dim <= 0 || head_dim > 256 || head_dim % 8)
        return set_error(BNN_ERR_ARG, "head_dim %d: a multiple of 8, at most 256", head_dim);
    if (bits != 4 && bits != 8) return set_error(BNN_ERR_ARG, "%d bits: 4 or 8", bits);
    if (group == 0) group = head_dim;
    if (group != head_dim && group != 32 && group != 64 && group != 128)
        return set_error(BNN_ERR_ARG, "group %d: 32, 64, 128 or head_dim", group);
    if (type != BNN_BF16 && type != BNN_FP16) return set_error(BNN_ERR_ARG, "type %d: BNN_BF16 or BNN_FP16", type);
    auto* c = new (std::nothrow) bnn_kv_cache();
    if (!c) return set_error(BNN_ERR_OOM, "OOM");
    c->device = device;
    c->type = type;
    c->geo = kv_geo(pages, page_tokens, kv_heads, head_dim, bits, group);
    const auto up = [](int64_t n) { return (size_t)((n + 255) & ~(int64_t)255); };
    c->bytes = 2 * (up(kv_code_bytes(c->geo)) + up(kv_scales(c->geo) * 2));
    const int rc = device < 0 ? BNN_OK : kv_create(c);
    if (rc) {
        bnn_kv_cache_destroy(c);
        return rc;
    }
    *out = c;
    return BNN_OK;
}

BNN_API void bnn_kv_cache_destroy(bnn_kv_cache* c) {
    if (!c) return;
    if (c->base) {
        DeviceScope dev(c->device);
        cudaFree(c->base);
    }
    delete c;
}

BNN_API size_t bnn_kv_cache_bytes(const bnn_kv_cache* c) { return c ? c->bytes : 0; }

BNN_API int bnn_kv_cache_write(bnn_kv_cache* c, const void* d_k, int64_t k_token, int64_t k_head, const void* d_v,
                               int64_t v_token, int64_t v_head, int n_tokens, int n_seqs, const int32_t* d_table,
                               int table_pages, const int32_t* d_start, const int32_t* d_offsets, void* stream) {
    return kv_rows<true>("bnn_kv_cache_write", c, d_k, k_token, k_head, d_v, v_token, v_head, n_tokens, n_seqs, d_table,
                         table_pages, d_start, d_offsets, stream);
}

BNN_API int bnn_kv_cache_read(const bnn_kv_cache* c, void* d_k, int64_t k_token, int64_t k_head, void* d_v, int64_t v_token,
                              int64_t v_head, int n_tokens, int n_seqs, const int32_t* d_table, int table_pages,
                              const int32_t* d_start, const int32_t* d_offsets, void* stream) {
    return kv_rows<false>("bnn_kv_cache_read", c, d_k, k_token, k_head, d_v, v_token, v_head, n_tokens, n_seqs, d_table,
                          table_pages, d_start, d_offsets, stream);
}
