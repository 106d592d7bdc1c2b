// kv_cache.cu - the block-scaled key/value cache of include/bnn_lowbit.h:
// create, write (quantise as it is stored) and read.
#include <climits>
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
    int token[2], head[2];  // strides
    int n_tokens, n_seqs, width;
    const int32_t *table, *start, *off;
    bool vec[2];
    int tpc;              // tokens a CTA
    uint32_t head_magic;  // unit / heads = unit * head_magic >> 32 (heads > 1)
};

constexpr int kRowThreads = 256, kMaxTpc = 32;

// where head 0 of a token lies: bytes into the codes, scales; row -1: nowhere
struct KvPlace {
    int64_t row, scale;
};
// places of the CTA's tokens, a warp each
__device__ __forceinline__ void kv_places(const KvRows& p, KvPlace* place) {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < p.tpc; i += kRowThreads / 32) {
        const int t = blockIdx.x * p.tpc + i;
        KvPlace at = {-1, 0};
        if (t < p.n_tokens) {
            const int b = p.off ? kv_seq(p.off, p.n_seqs, t,
                                         [&](int lo, int step, int len) {
                                             return __popc(__ballot_sync(0xffffffffu, lane * step < len && p.off[lo + lane * step] <= t));
                                         })
                                : t;
            if (b >= 0) {
                const int64_t pos = (int64_t)p.start[b] + (p.off ? (int64_t)t - p.off[b] : 0);
                if (pos >= 0 && pos <= 0x7fffffff) {
                    const int page = kv_page(p.g, p.table + (int64_t)b * p.width, p.width, (int)pos);
                    if (page >= 0) {
                        at.row = kv_row(p.g, page, 0, (int)pos & (p.g.pt - 1));
                        at.scale = kv_scale(p.g, page, 0, 0, (int)pos & (p.g.pt - 1));
                    }
                }
            }
        }
        if (lane == 0) place[i] = at;
    }
    __syncthreads();
}

// Both kernels: W = dp / 8 neighbouring lanes (32 for dp = 192) have one head
// of one token, 8 numbers each: 16 bytes of the caller's row of keys and as
// many of values, one such unit at a time: many resident warps hide the
// loads better than more units a lane do (two at a time: 31.0 us against 28.8,
// and 4.9 against 3.7 for one token each of 64 sequences). A write's loads
// are on their way while the tokens' places are looked up.
// 17828 tokens, 8 heads of 128, 4 bits, groups of 32: written in 29 us, read in
// 23 (in a row of such launches): 3.2 and 4.1 TB/s. Bound by instructions
// (3.0 and 2.7 a clock of an SM's 4), not yet by the bytes (14.5 us each).
template <int W, int BITS>
struct KvLane {
    int i, dim_left;      // numbers 8 * i .. of a head; how many of them there are from there on
    int grp, k_at, v_at;  // its scale; bytes of a row
    bool owner;           // stores the group's scale
    int lanes;            // of a group
    __device__ __forceinline__ explicit KvLane(const KvGeo& g) {
        i = threadIdx.x % W;
        dim_left = g.dim - 8 * i;
        lanes = g.ng == 1 ? W : g.group / 8;  // a power of two, 4 at least
        grp = i >> (31 - __clz(lanes));
        owner = (i & (lanes - 1)) == 0 && grp < g.ng;
        k_at = kv_k_at(g, i), v_at = kv_v_at(g, 2 * i);
    }
};
// numbers 8 * i + 4 .. of a value lie this far behind 8 * i ..
template <int BITS>
__device__ __forceinline__ int kv_v_next(const KvGeo& g) { return g.dp / 32 * (BITS / 2); }

// unit n of the CTA: token and head
__device__ __forceinline__ bool kv_unit(const KvRows& p, int unit, int& local, int& head) {
    local = p.g.heads == 1 ? unit : (int)__umulhi((uint32_t)unit, p.head_magic);
    head = unit - local * p.g.heads;
    return local < p.tpc && (int64_t)blockIdx.x * p.tpc + local < p.n_tokens;
}

// Codes and scale of a group, of which this lane has the 8 numbers of v. x
// has at most 11 significant bits and the scale s has 8, so x / s is at
// least 2^-12 away from a border k + 1/2 of two codes that it does not hit
// exactly. x * (1 / s) is within 2^-15 of it: rounded to a grid of 2^-12 it
// is on its own side, or on the border where x / s is, and rounding that to
// even gives the code of the exact quotient. The scale: max * (1 / top) is
// within 2^-23 of max / top, which is at least 2^-16 away from any border of
// bf16 (none can be hit: 127 or 7 times an odd number of 9 bits has more than
// 11), so it rounds as the exact quotient does.
constexpr uint32_t kWhole = 0x4b400000u;  // 0x1.8p23f: on it, a whole number is in the low bits of a float
template <int W, int BITS, bool FP16>
__device__ __forceinline__ void kv_quantise(uint4 v, int lanes, uint32_t* code, uint16_t& scale) {
    constexpr int most = BITS == 8 ? 127 : 7;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    // |x| as bits, two at a time: an order that puts NaN above infinity above all numbers
    uint32_t big = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
    const auto over = [&](int s) { big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, s)); };
    over(1), over(2);
    if (lanes > 4) {
        over(4);
        if (W > 8 && lanes > 8) {
            over(8);
            if (W > 16 && lanes > 16) over(16);
        }
    }
    big = max(big & 0xffffu, big >> 16);
    const bool bad = big >= (FP16 ? 0x7c00u : 0x7f80u);
    const float top = bad ? 0.0f : unpack2(big, FP16).x;
    float x[8];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const float2 f = unpack2(w[c], FP16);
        x[2 * c] = f.x, x[2 * c + 1] = f.y;
    }
    const float grid = 0x1.8p11f, whole = 0x1.8p23f + (float)(most + 1);  // steps of 2^-12; of 1, and the stored offset
    __nv_bfloat16 sb = __float2bfloat16_rn(__fmul_rn(top, 1.0f / (float)most));
    float s = __bfloat162float(sb);
    if (s >= 0x1p-100f) {
        float inv;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
        for (int c = 0; c < 8; ++c) code[c] = __float_as_uint(__fadd_rn(__fadd_rn(__fmaf_rn(x[c], inv, grid), -grid), whole));
    } else {  // 1 / s may be out of range, and a subnormal scale far from max / top
        sb = __float2bfloat16_rn(__fdiv_rn(top, (float)most));
        s = __bfloat162float(sb);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            const float q = s > 0.0f && !bad ? rintf(__fdiv_rn(x[c], s)) : 0.0f;
            code[c] = kWhole + (uint32_t)((int)fminf(fmaxf(q, -(float)most), (float)most) + most + 1);
        }
    }
    scale = bad ? (uint16_t)0x7fff : *reinterpret_cast<const uint16_t*>(&sb);
}
// N codes side by side, code c at bit c * log2(base). Each one stands on
// kWhole, whose multiples drop out; multiply-adds, since the pipe of shifts
// and masks is what bounds the write.
template <int N, int STEP>
__device__ __forceinline__ uint32_t side_by_side(const uint32_t* code, uint32_t base, uint32_t off) {
    uint32_t w = code[(N - 1) * STEP];
#pragma unroll
    for (int c = N - 2; c >= 0; --c) asm("mad.lo.u32 %0, %0, %1, %2;" : "+r"(w) : "r"(base), "r"(code[c * STEP]));
    return w - off;
}
constexpr uint32_t whole_sum(int n, int bits) {  // kWhole * (1 + 2^bits + ...), n terms
    uint32_t s = 0;
    for (int i = 0; i < n; ++i) s = (s << bits) + kWhole;
    return s;
}
// a number that the compiler does not know, so that it does not make shifts of multiplications
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm("mov.b32 %0, %0;" : "+r"(v));
    return v;
}

template <int W, int BITS, bool FP16>
__global__ void __launch_bounds__(kRowThreads) kv_write_kernel(const KvRows p) {
    __shared__ KvPlace place[kMaxTpc];
    const KvGeo& g = p.g;
    const KvLane<W, BITS> me(g);
    const int units = p.tpc * g.heads, next = kv_v_next<BITS>(g);
    const int head_row = g.pt * g.row, head_scale = g.pt * g.ngp;  // from one head to the next
    uint16_t* x0[2];  // this lane's numbers of head 0 of the CTA's first token
#pragma unroll
    for (int which = 0; which < 2; ++which) x0[which] = p.x[which] + (int64_t)blockIdx.x * p.tpc * p.token[which] + 8 * me.i;
    const uint32_t base = opaque(BITS == 8 ? 256u : 16u);
    grid_wait();
    grid_launch();
    bool looked = false;
    for (int n0 = 0; n0 < units; n0 += kRowThreads / W) {
        uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        int local, head;
        if (kv_unit(p, n0 + threadIdx.x / W, local, head) && me.dim_left > 0)
#pragma unroll
            for (int which = 0; which < 2; ++which)
                v[which] = load8(x0[which] + (int64_t)local * p.token[which] + (int64_t)head * p.head[which], me.dim_left, p.vec[which]);
        if (!looked) kv_places(p, place);
        looked = true;
        const KvPlace at = local < p.tpc ? place[local] : KvPlace{-1, 0};
        const bool store = at.row >= 0 && 8 * me.i < g.dp;
        const int64_t row_at = at.row + (int64_t)head * head_row, scale_at = at.scale + (int64_t)head * head_scale + me.grp;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            uint32_t code[8];
            uint16_t scale;
            kv_quantise<W, BITS, FP16>(v[which], me.lanes, code, scale);
            if (!store) continue;
            if (me.owner) p.scales[which][scale_at] = scale;
            uint8_t* row = p.codes[which] + row_at;
            if (BITS == 8) {
                const uint32_t a = side_by_side<4, 1>(code, base, whole_sum(4, 8)), b = side_by_side<4, 1>(code + 4, base, whole_sum(4, 8));
                if (which == 0) {
                    *reinterpret_cast<uint2*>(row + me.k_at) = make_uint2(a, b);
                } else {
                    *reinterpret_cast<uint32_t*>(row + me.v_at) = a;
                    *reinterpret_cast<uint32_t*>(row + me.v_at + next) = b;
                }
            } else if (which == 0) {  // even numbers in the low half, odd ones in the high
                const uint32_t a = side_by_side<4, 2>(code, base, whole_sum(4, 4)), b = side_by_side<4, 2>(code + 1, base, whole_sum(4, 4));
                *reinterpret_cast<uint32_t*>(row + me.k_at) = __byte_perm(a, b, 0x5410);
            } else {
                const uint32_t a = side_by_side<8, 1>(code, base, whole_sum(8, 4));
                *reinterpret_cast<uint16_t*>(row + me.v_at) = (uint16_t)a;
                *reinterpret_cast<uint16_t*>(row + me.v_at + next) = (uint16_t)(a >> 16);
            }
        }
    }
}

template <int W, int BITS, bool FP16>
__global__ void __launch_bounds__(kRowThreads) kv_read_kernel(const KvRows p) {
    __shared__ KvPlace place[kMaxTpc];
    const KvGeo& g = p.g;
    const KvLane<W, BITS> me(g);
    const int units = p.tpc * g.heads, next = kv_v_next<BITS>(g);
    const int head_row = g.pt * g.row, head_scale = g.pt * g.ngp;  // from one head to the next
    uint16_t* x0[2];  // this lane's numbers of head 0 of the CTA's first token
#pragma unroll
    for (int which = 0; which < 2; ++which) x0[which] = p.x[which] + (int64_t)blockIdx.x * p.tpc * p.token[which] + 8 * me.i;
    grid_wait();
    grid_launch();
    kv_places(p, place);
    for (int n0 = 0; n0 < units; n0 += kRowThreads / W) {
        int local, head;
        if (!kv_unit(p, n0 + threadIdx.x / W, local, head) || me.dim_left <= 0) continue;
        const KvPlace at = place[local];
        if (at.row < 0) continue;
        const int64_t row_at = at.row + (int64_t)head * head_row, scale_at = at.scale + (int64_t)head * head_scale + me.grp;
        uint2 v[2];
        uint16_t sc[2];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const uint8_t* row = p.codes[which] + row_at;
            sc[which] = p.scales[which][scale_at];
            v[which] = make_uint2(0, 0);
            if (BITS == 8) {
                if (which == 0) {
                    v[0] = *reinterpret_cast<const uint2*>(row + me.k_at);
                } else {
                    v[1].x = *reinterpret_cast<const uint32_t*>(row + me.v_at);
                    v[1].y = *reinterpret_cast<const uint32_t*>(row + me.v_at + next);
                }
            } else if (which == 0) {
                v[0].x = *reinterpret_cast<const uint32_t*>(row + me.k_at);
            } else {
                v[1].x = *reinterpret_cast<const uint16_t*>(row + me.v_at) |
                         (uint32_t)*reinterpret_cast<const uint16_t*>(row + me.v_at + next) << 16;
            }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float s = bf16_float(sc[which]), zero = -(8388608.0f + (BITS == 8 ? 128.0f : 8.0f));
            uint32_t o[4];
#pragma unroll
            for (int c = 0; c < 8; c += 2) {
                // on 2^23 as a float; then 7 bits times 8: exact, rounded once below
                uint32_t b[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (BITS == 8) b[e] = __byte_perm(c < 4 ? v[which].x : v[which].y, 0x4b000000u, 0x7440 + (c & 3) + e);
                    else b[e] = and_or(v[which].x >> (which ? 4 * (c + e) : 2 * c + 16 * e), 15u, 0x4b000000u);
                const float2 x = apart(mul2(add2(both(__uint_as_float(b[0]), __uint_as_float(b[1])), both(zero, zero)), both(s, s)));
                o[c / 2] = pack2(x.x, x.y, FP16);
            }
            store8(x0[which] + (int64_t)local * p.token[which] + (int64_t)head * p.head[which], make_uint4(o[0], o[1], o[2], o[3]), me.dim_left, p.vec[which]);
        }
    }
}

template <int W, int BITS, bool FP16, bool WRITE>
cudaError_t kv_launch(const KvRows& p, dim3 grid, cudaStream_t st) {
    if constexpr (WRITE) return launch(kv_write_kernel<W, BITS, FP16>, grid, kRowThreads, 0, st, true, p);
    else return launch(kv_read_kernel<W, BITS, FP16>, grid, kRowThreads, 0, st, true, p);
}
template <int W, bool WRITE>
cudaError_t kv_width(const KvRows& p, bool fp16, dim3 grid, cudaStream_t st) {
    if (p.g.bits == 8) return fp16 ? kv_launch<W, 8, true, WRITE>(p, grid, st) : kv_launch<W, 8, false, WRITE>(p, grid, st);
    return fp16 ? kv_launch<W, 4, true, WRITE>(p, grid, st) : kv_launch<W, 4, false, WRITE>(p, grid, st);
}

template <bool WRITE>
int kv_rows(const char* what, const bnn_kv_cache* c, const void* k, int64_t k_token, int64_t k_head, const void* v,
            int64_t v_token, int64_t v_head, int n_tokens, int n_seqs, const int32_t* table, int width,
            const int32_t* start, const int32_t* off, void* stream) {
    if (!c || n_tokens < 0 || n_seqs < 0 || width < 0) return set_error(BNN_ERR_ARG, "%s: bad arguments", what);
    const KvGeo& g = c->geo;
    if (n_tokens > (1 << 30)) return set_error(BNN_ERR_ARG, "%s: %d tokens: at most 2^30", what, n_tokens);
    if (!off && n_tokens != n_seqs)
        return set_error(BNN_ERR_ARG, "%s: %d tokens of %d sequences need offsets", what, n_tokens, n_seqs);
    const bool work = n_tokens > 0 && n_seqs > 0 && width > 0;
    if (work) {
        if (!k || !v || !table || !start) return set_error(BNN_ERR_ARG, "%s: NULL argument", what);
        if (!aligned(k, 2) || !aligned(v, 2) || !aligned(table, 4) || !aligned(start, 4) || !aligned(off, 4))
            return set_error(BNN_ERR_ARG, "%s: an array is not aligned to its type", what);
        for (int64_t st : {k_token, k_head, v_token, v_head})
            if (st > INT_MAX || st < -INT_MAX) return set_error(BNN_ERR_ARG, "%s: a stride of 2^31 or more", what);
        if (!WRITE)  // rows of an output must not lie over one another
            for (const auto& s : {std::pair<int64_t, int64_t>(k_token, k_head), std::pair<int64_t, int64_t>(v_token, v_head)})
                if ((g.heads > 1 && s.second < g.dim) || (n_tokens > 1 && s.first < g.dim))
                    return set_error(BNN_ERR_ARG, "%s: strides %lld, %lld of an output: at least %d", what, (long long)s.first,
                                     (long long)s.second, g.dim);
                else if (rows_share(n_tokens, s.first, g.heads, s.second, g.dim))
                    return set_error(BNN_ERR_ARG, "%s: strides %lld, %lld put heads of an output over one another", what,
                                     (long long)s.first, (long long)s.second);
    }
    if (c->device < 0) return no_device(what);
    if (!work) return BNN_OK;
    DeviceScope dev(c->device);
    if (dev.err != cudaSuccess) return cuda_error(what, dev.err);
    KvRows p{};
    p.g = g;
    p.codes[0] = c->kc, p.codes[1] = c->vc, p.scales[0] = c->ks, p.scales[1] = c->vs;
    p.x[0] = (uint16_t*)k, p.x[1] = (uint16_t*)v;
    p.token[0] = (int)k_token, p.head[0] = (int)k_head, p.token[1] = (int)v_token, p.head[1] = (int)v_head;
    p.n_tokens = n_tokens, p.n_seqs = n_seqs, p.width = width;
    p.table = table, p.start = start, p.off = off;
    for (int w = 0; w < 2; ++w)
        p.vec[w] = aligned(p.x[w], 16) && (n_tokens == 1 || p.token[w] % 8 == 0) && (g.heads == 1 || p.head[w] % 8 == 0);
    const int W = g.dp == 64 ? 8 : g.dp == 128 ? 16 : 32;
    // four units a thread of a CTA, where every SM has several CTAs then
    p.tpc = 1;
    while (p.tpc < kMaxTpc && p.tpc * g.heads * W < 4 * kRowThreads && n_tokens / (2 * p.tpc) >= 8 * c->sms) p.tpc *= 2;
    p.head_magic = (uint32_t)((0x100000000ull + g.heads - 1) / g.heads);
    const dim3 grid((unsigned)cdiv64(n_tokens, p.tpc));
    const cudaStream_t st = (cudaStream_t)stream;
    const bool fp16 = c->type == BNN_FP16;
    const cudaError_t e = W == 8 ? kv_width<8, WRITE>(p, fp16, grid, st) : W == 16 ? kv_width<16, WRITE>(p, fp16, grid, st)
                                                                                   : kv_width<32, WRITE>(p, fp16, grid, st);
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
