// kv_attend.cu - attention of single query tokens over the key/value cache
// of include/bnn_lowbit.h.
//
// out = softmax(scale * q K^T) V for the rows (query heads) that share a kv
// head, in one pass over the keys and values with a running maximum and sum
// per row. The codes are decoded to fp16 in registers, exactly (7 bits), and
// multiplied on mma.sync m16n8k16 with the tokens in M (scores) and the
// channels in M (output), so that 8 query rows fill an instruction's N and
// no code passes through shared memory as anything but the bytes that came
// from the cache. tcgen05 would want its operands as 16-bit tiles in shared
// memory: eight to four times the bytes, for an operation that is bound by
// reading codes.
#include <climits>
#include <cmath>

#include "kv_cache.h"
#include "lowbit_dev.cuh"

namespace bnn {
namespace lowbit {
namespace {

constexpr int kWarps = 4;
constexpr int kMostInv = 127 + 118;  // exponent field of the largest 1 / unit: times 2^8 a float
constexpr int kSub = 16;  // tokens of an instruction
// 16-token blocks that a warp takes at a time: two where the sums leave it the
// registers and a row is short (of `row` bytes), so that shared memory holds
// enough steps: 64 ragged sequences in 4 bits 78 us against 85 of one at a
// time, but 100003 tokens in 8 bits, 128-byte rows, 62 against 48.
__host__ __device__ constexpr int attend_halves(int nt, int row) { return nt == 1 && row <= 64 ? 2 : 1; }

// CTAs of an attention kernel on an SM: as many as the registers allow, dp * nt
// sums over a CTA's warps among them
__host__ __device__ constexpr int attend_ctas(int dp, int nt) {
    return dp * nt <= 128 ? 4 : 2;
}

struct AttendParams {
    KvGeo g;
    const uint8_t *kc, *vc;
    const uint16_t *ks, *vs;
    const uint16_t* q;
    int64_t q_seq, q_head;
    uint16_t* out;
    int64_t o_seq, o_head;
    float* lse;
    bool fp16, q_vec, o_vec;  // rows of q are 16-byte, of out 8-byte aligned
    int n_grp;               // sequences; 1 for the prefix
    const int32_t* lengths;  // [n_grp], or nullptr: `length`
    int length;
    const int32_t* table;
    int width;
    int share;               // query heads per kv head
    int rg;                  // query rows per group and kv head (share; n_seqs * share for the prefix)
    int rt;                  // tiles of 8 * NT rows they make
    float scale_log2;        // scale * log2(e)
    bool partial;            // leave every item to the join kernel
    bool second;             // runs beside the prefix's kernel
    int2* owners;            // [group][kv head][tile]: first and last CTA of an item, for the join
    float* pacc;             // [slot][row][dp] means of the values with weights exp2(s - m)
    float2* pml;             // [slot][row] (m, sum of exp2(s - m))
    int stages;
};

// blocks of a group
__device__ __forceinline__ int grp_len(const AttendParams& p, int b) {
    const int n = p.lengths ? p.lengths[b] : p.length;
    const int64_t cap = (int64_t)p.width << p.g.sh;
    return n < 0 ? 0 : n > cap ? (int)cap : n;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
// 2^e for e <= 0; 0 below the range of normal numbers
__device__ __forceinline__ float pow2(int e) { return e < -126 ? 0.0f : __int_as_float((127 + e) << 23); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A block of 16 rows lies in shared memory as it does in the cache, but for
// the order of the eight 16-byte pieces of each 128-byte line, which a XOR
// with the line number spreads so that the lanes of one load (different
// rows, the same place in the row) meet different banks.
template <int ROW>
__device__ __forceinline__ int swz(int o) {
    constexpr int MUL = ROW >= 128 ? 1 : 2;
    return (o & ~0x70) | ((((o >> 4) ^ ((o >> 7) * MUL)) & 7) << 4);
}
// BYTES neighbouring bytes at `o` of such a block
template <int ROW, int BYTES>
__device__ __forceinline__ void lds_part(uint32_t* w, const uint8_t* base, int o) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(base + swz<ROW>(o + 16 * i));
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 8; ++i) {
            const uint2 v = *reinterpret_cast<const uint2*>(base + swz<ROW>(o + 8 * i));
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(base + swz<ROW>(o + 4 * i));
    }
}

// Codes as fp16 pairs. A byte or a nibble put into the mantissa of a power
// of two is that power plus the code and its offset, exactly; the subtraction
// leaves the code. (Sums of products could start at -(power + offset) *
// sum(q) instead, for the keys; that saves the subtraction, which is not what
// bounds this, and costs 4 of the 24 bits of the scores' sums.)
template <int LO>
__device__ __forceinline__ uint32_t bytes2(uint32_t w) {  // bytes LO and LO + 1 of w
    return Fp16::sub2(__byte_perm(w, 0x64646464u, LO ? 0x4342 : 0x4140), 0x64806480u);
}
// the four nibble pairs of a word: bits 0-3 of a half on 1024, bits 4-7, which
// are worth 1 there, on 64
__device__ __forceinline__ void nibbles4(uint32_t* a, uint32_t w) {
    const uint32_t v = w >> 8;
    a[0] = Fp16::sub2(and_or(w, 0x000f000fu, 0x64006400u), 0x64086408u);
    a[1] = Fp16::sub2(and_or(w, 0x00f000f0u, 0x54005400u), 0x54805480u);
    a[2] = Fp16::sub2(and_or(v, 0x000f000fu, 0x64006400u), 0x64086408u);
    a[3] = Fp16::sub2(and_or(v, 0x00f000f0u, 0x54005400u), 0x54805480u);
}

// Shared memory: prefix sums | row factors | (m, l) of the warps | q fragments
// | stages, later the warps' sums.
struct AttendSmem {
    int factor, ml, q, ring, stage, bytes;
};
__host__ __device__ inline AttendSmem attend_smem(const KvGeo& g, int n_grp, int nt, int stages) {
    const int rows = 8 * nt;
    AttendSmem s;
    s.factor = ((n_grp + 1) * 4 + 127) & ~127;
    s.ml = s.factor + 128 * ((rows * 4 + 127) / 128);
    s.q = s.ml + kWarps * rows * 8;
    s.ring = s.q + g.dp / 32 * nt * 512;
    s.stage = attend_halves(nt, g.row) * (2 * kSub * g.row + ((2 * g.ngp * kSub * 2 + 127) & ~127));
    const int ring = kWarps * stages * s.stage, merge = kWarps * rows * (g.dp + 8) * 4;
    s.bytes = s.ring + (ring > merge ? ring : merge);
    return s;
}

template <int N>
__device__ __forceinline__ void load_scales(float* f, const uint16_t* at) {  // N bf16, N a power of two, aligned
    if constexpr (N == 1) {
        f[0] = bf16_float(at[0]);
    } else {
        uint32_t w[N / 2];
        if constexpr (N == 2) w[0] = *reinterpret_cast<const uint32_t*>(at);
        if constexpr (N == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            w[0] = v.x, w[1] = v.y;
        }
        if constexpr (N == 8) {
            const uint4 v = *reinterpret_cast<const uint4*>(at);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// DP: head_dim rounded up; NT: tiles of 8 query rows; BPG: 32-blocks of
// channels that share a scale (8: all).
// The floor is the codes' bytes; decoding them holds it at 2.3 to 2.6 of an
// SM's 4 instructions a clock, half of them bit operations and conversions, at
// 16 warps of 127 registers an SM. 100003 tokens, 8 kv heads of 128 in 8 bits,
// 32 query heads: 48 us with the join (4.3 TB/s of codes). 179457 tokens of 64
// sequences, 64 query heads, in 4 bits and groups of 32: 78 us (2.7 TB/s). 16
// such sequences of 256 query heads in 8 bits (32 rows a tile, a unit for each
// row and group): 72 us, bound by fetching instructions too. The work is cut into one equal share a CTA, in blocks of tokens, whatever
// sequence they belong to; what is cut is joined by join_kernel.
template <int DP, int BITS, int NT, int BPG>
__global__ void __launch_bounds__(32 * kWarps, attend_ctas(DP, NT)) attend_kernel(const AttendParams p) {
    constexpr int NB = DP / 32, R = 8 * NT, ROW = DP * BITS / 8, CODES = kSub * ROW;
    constexpr int NG = (NB + BPG - 1) / BPG, NGP = NG <= 1 ? 1 : NG <= 2 ? 2 : NG <= 4 ? 4 : 8;
    constexpr int KP = ROW / 4, VP = ROW / 8;  // a lane's bytes of a key's, a value's row
    constexpr int HV = attend_halves(NT, ROW), KS = kSub * HV;  // 16-token blocks, tokens of a step
    constexpr int HALF = 2 * CODES + ((2 * NGP * kSub * 2 + 127) & ~127);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int2 warp_sum[kWarps];
    const KvGeo g = p.g;
    const AttendSmem at = attend_smem(g, p.n_grp, NT, p.stages);
    int* pre = reinterpret_cast<int*>(smem);
    float* factor = reinterpret_cast<float*>(smem + at.factor);
    float2* wml = reinterpret_cast<float2*>(smem + at.ml);
    uint4* qf = reinterpret_cast<uint4*>(smem + at.q);
    uint8_t* ring = smem + at.ring;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int r = lane >> 2, j = lane & 3;
    // The kernel for the sequences' own positions starts beside the prefix's,
    // which waits before it lets it start; it waits for it at its end.
    if (!p.second) grid_wait();
    grid_launch();

    // blocks before each group, counted in both sizes at once
    const int items = g.heads * p.rt;  // of a group
    int block;
    {
        const int per = (p.n_grp + 32 * kWarps - 1) / (32 * kWarps), b0 = tid * per, b1 = min(p.n_grp, b0 + per);
        const auto blocks = [&](int b) {
            const int n = grp_len(p, b);
            return make_int2((n + kBlock - 1) / kBlock, (n + kLong - 1) / kLong);
        };
        int2 sum = make_int2(0, 0);
        int most = 0;
        for (int b = b0; b < b1; ++b) {
            const int2 n = blocks(b);
            sum.x += n.x, sum.y += n.y;
            most = max(most, n.y);
        }
        int2 inc = sum;
        for (int s = 1; s < 32; s <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc.x, s), y = __shfl_up_sync(0xffffffffu, inc.y, s);
            if (lane >= s) inc.x += x, inc.y += y;
        }
        if (lane == 31) warp_sum[warp] = inc;
        const bool cut = __syncthreads_or(most > 1);
        int2 to = make_int2(inc.x - sum.x, inc.y - sum.y), all = make_int2(0, 0);
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) to.x += warp_sum[w].x, to.y += warp_sum[w].y;
            all.x += warp_sum[w].x, all.y += warp_sum[w].y;
        }
        const bool lng = !cut || split_long((int64_t)all.x * items, gridDim.x);
        block = lng ? kLong : kBlock;
        int at = lng ? to.y : to.x;
        for (int b = b0; b < b1; ++b) {
            pre[b] = at;
            const int2 n = blocks(b);
            at += lng ? n.y : n.x;
        }
        if (tid == 0) pre[p.n_grp] = lng ? all.y : all.x;
        __syncthreads();
    }
    const uint32_t units = (uint32_t)pre[p.n_grp] * (uint32_t)items;  // below 2^31: the host's check
    const int ctas = split_ctas(units, gridDim.x);
    const bool has = (int)blockIdx.x < ctas;
    const uint32_t u_end = has ? split_begin(units, blockIdx.x + 1, ctas) : 0;
    uint32_t u = has ? split_begin(units, blockIdx.x, ctas) : 0;

    // rows of groups with nothing in them, a warp each
    if (!p.partial) {
        const int q_heads = g.heads * p.share;
        for (int64_t row = (int64_t)blockIdx.x * kWarps + warp; row < (int64_t)p.n_grp * q_heads; row += gridDim.x * kWarps) {
            const int b = (int)((uint32_t)row / (uint32_t)q_heads), qh = (int)((uint32_t)row % (uint32_t)q_heads);
            if (pre[b + 1] != pre[b]) continue;
            for (int d = lane; d < g.dim; d += 32) p.out[b * p.o_seq + qh * p.o_head + d] = 0;
            if (p.lse && lane == 0) p.lse[row] = -INFINITY;
        }
    }

    int grp = 0;
    while (u < u_end) {
        // the item of block u, and the blocks of it that are this CTA's
        {
            int lo = grp, hi = p.n_grp;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((uint32_t)pre[mid] * (uint32_t)items <= u) lo = mid;
                else hi = mid;
            }
            grp = lo;
        }
        const int nb = pre[grp + 1] - pre[grp];
        const uint32_t in_grp = u - (uint32_t)pre[grp] * (uint32_t)items;
        const int item = (int)(in_grp / (uint32_t)nb), blk0 = (int)(in_grp % (uint32_t)nb);
        const int blk1 = (int)min((uint32_t)nb, blk0 + (u_end - u));
        const int head = item / p.rt, tile = item % p.rt;
        const int len = grp_len(p, grp);
        const int rows = min(R, p.rg - tile * R);
        const int row0 = grp * p.rg + tile * R;  // row i of the item: query row (row0 + i)
        if (blk0 == 0 && tid == 0)
            p.owners[(int64_t)grp * items + item] = make_int2(blockIdx.x, split_owner(units, u + nb - 1, ctas));

        // steps of KS tokens; the warps take them in turn
        const int end = min(blk1 * block, len), sub0 = blk0 * (block / KS), sub1 = (end + KS - 1) / KS;
        uint8_t* mine = ring + warp * p.stages * at.stage;
        const int32_t* row_table = p.table + (int64_t)grp * p.width;
        // copies of a step's tokens into a stage; bit h: its h-th 16 tokens have a page
        const auto fetch = [&](int sub, uint8_t* to) -> uint32_t {
            uint32_t got = 0;
#pragma unroll
            for (int h = 0; h < HV; ++h) {
                const int pos = sub * KS + h * kSub;
                const int page = pos < end ? kv_page(g, row_table, p.width, pos) : -1;
                if (page < 0) continue;
                got |= 1u << h;
                const int tok = pos & (g.pt - 1);
                const int64_t slot = ((int64_t)page * g.heads + head) * g.pt + tok, from = slot * ROW;
                const uint32_t dst = smem_addr(to) + h * HALF;
                static_assert(CODES % 512 == 0, "whole pieces for every lane");
#pragma unroll
                for (int c = 0; c < CODES / 512; ++c) {
                    const int o = (c * 32 + lane) * 16;
                    cp16(dst + swz<ROW>(o), p.kc + from + o);
                    cp16(dst + CODES + swz<ROW>(o), p.vc + from + o);
                }
                if (lane < 4 * NGP) {  // 32 * NGP bytes of scales of each
                    const int of = lane >= 2 * NGP, c = of ? lane - 2 * NGP : lane;
                    cp16(dst + 2 * CODES + lane * 16, (of ? p.vs : p.ks) + slot * NGP + 8 * c);
                }
            }
            return got;
        };
        // the first steps are on their way while q is made ready
        uint32_t there = 0;  // HV bits a stage
        int ahead = sub0 + warp;
        for (int s = 0; s < p.stages - 1; ++s, ahead += kWarps) {
            if (ahead < sub1) there |= fetch(ahead, mine + s * at.stage) << (HV * s);
            cp_commit();
        }

        // q as B fragments of fp16, each row scaled by a power of two that
        // puts its largest value in [2^9, 2^10): exact but for values
        // 2^-24 and less of the row's largest
        {
            uint4 v[R / kWarps];
#pragma unroll
            for (int k = 0; k < R / kWarps; ++k) {
                const int i = warp + k * kWarps;
                const int row = row0 + i, seq = row / p.share;
                v[k] = make_uint4(0, 0, 0, 0);
                if (i < rows && 8 * lane < g.dim)
                    v[k] = load8(p.q + seq * p.q_seq + (head * p.share + row - seq * p.share) * p.q_head + 8 * lane,
                                 g.dim - 8 * lane, p.q_vec);
            }
#pragma unroll
            for (int k = 0; k < R / kWarps; ++k) {
                const int i = warp + k * kWarps;
                const uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                float x[8];
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float2 f = unpack2(w[c], p.fp16);
                    x[2 * c] = f.x, x[2 * c + 1] = f.y;
                    top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
                }
                top = __reduce_max_sync(0xffffffffu, top);
                const int e = (int)(top >> 23);  // 127 + exponent of the largest; 255: not finite
                const int sh = top == 0 || e == 255 ? 0 : max(-126, min(126, 9 + 127 - e));
                const float up = __int_as_float((127 + sh) << 23);
                uint32_t h[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) h[c] = pack2(x[2 * c] * up, x[2 * c + 1] * up, true);
                if (lane < DP / 8) qf[((lane >> 2) * NT + (i >> 3)) * 32 + (i & 7) * 4 + (lane & 3)] = make_uint4(h[0], h[1], h[2], h[3]);
                // a row with an infinity or a NaN has only infinite scores and NaN: its softmax is NaN
                if (lane == 0) factor[i] = e == 255 ? NAN : p.scale_log2 * __int_as_float((127 - sh) << 23);
            }
        }
        __syncthreads();

        float acc[NB][2][NT][4], m[NT][2], l[NT][2], f[NT][2];
        // Sums of weight * scale * code are kept in a unit of a power of two for
        // each query row and scale group, so that a unit follows what the row
        // sees: neither a token without weight in it nor another row's values
        // move it. inv: 1 / unit beside exp2(s - m).
        float inv[NG][NT][2];
#pragma unroll
        for (int q = 0; q < NG; ++q)
#pragma unroll
            for (int t = 0; t < NT; ++t) inv[q][t][0] = inv[q][t][1] = __uint_as_float((uint32_t)kMostInv << 23);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][h][t][e] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[t][e] = -INFINITY, l[t][e] = 0.0f;
                f[t][e] = factor[t * 8 + 2 * j + e];
            }

        int st = 0, st_in = p.stages - 1;
        for (int sub = sub0 + warp; sub < sub1; sub += kWarps) {
            // the stage read a round ago is free: all lanes passed the barrier below
            there &= ~(((1u << HV) - 1) << (HV * st_in));
            if (ahead < sub1) there |= fetch(ahead, mine + st_in * at.stage) << (HV * st_in);
            ahead += kWarps;
            cp_commit();
            st_in = st_in + 1 == p.stages ? 0 : st_in + 1;
            switch (p.stages) {
                case 2: cp_wait<1>(); break;
                case 3: cp_wait<2>(); break;
                case 4: cp_wait<3>(); break;
                case 5: cp_wait<4>(); break;
                default: cp_wait<5>(); break;
            }
            __syncwarp();
            const uint8_t* step = mine + st * at.stage;
            const uint32_t have = there >> (HV * st) & ((1u << HV) - 1);
            st = st + 1 == p.stages ? 0 : st + 1;
            if (have) {
                // scores: tokens r and r + 8 in rows, query rows in columns
                float s[HV][NT][4], v0[HV][NGP], v1[HV][NGP];  // v0, v1: scales of the two tokens' values
#pragma unroll
                for (int h = 0; h < HV; ++h) {
                    const uint8_t* kb = step + h * HALF;
                    const uint16_t* sc = reinterpret_cast<const uint16_t*>(kb + 2 * CODES);  // [keys, values][token][NGP]
                    uint32_t k0[KP / 4], k1[KP / 4];
                    lds_part<ROW, KP>(k0, kb, r * ROW + j * KP);
                    lds_part<ROW, KP>(k1, kb, (r + 8) * ROW + j * KP);
                    float s0[NGP], s1[NGP];
                    load_scales<NGP>(s0, sc + r * NGP);
                    load_scales<NGP>(s1, sc + (r + 8) * NGP);
                    load_scales<NGP>(v0[h], sc + (kSub + r) * NGP);
                    load_scales<NGP>(v1[h], sc + (kSub + r + 8) * NGP);
                    float c[NT][4];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint4 qv[NT];
#pragma unroll
                        for (int t = 0; t < NT; ++t) qv[t] = qf[(b * NT + t) * 32 + lane];
                        uint32_t n0[4], n1[4];
                        if constexpr (BITS == 4) nibbles4(n0, k0[b]), nibbles4(n1, k1[b]);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t a[4];
                            if constexpr (BITS == 8) {
                                a[0] = bytes2<0>(k0[2 * b + x]), a[1] = bytes2<0>(k1[2 * b + x]);
                                a[2] = bytes2<2>(k0[2 * b + x]), a[3] = bytes2<2>(k1[2 * b + x]);
                            } else {
                                a[0] = n0[2 * x], a[1] = n1[2 * x], a[2] = n0[2 * x + 1], a[3] = n1[2 * x + 1];
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                if (b % BPG == 0 && x == 0) Fp16::mma0(c[t], a, qv[t].x, qv[t].y);
                                else Fp16::mma(c[t], a, x ? qv[t].z : qv[t].x, x ? qv[t].w : qv[t].y);
                            }
                        }
                        if (b == NB - 1 || b % BPG == BPG - 1) {  // the group's scale, on its sum of products
                            const float g0 = s0[b / BPG], g1 = s1[b / BPG];
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    s[h][t][e] = b < BPG ? (e < 2 ? g0 : g1) * c[t][e] : fmaf(e < 2 ? g0 : g1, c[t][e], s[h][t][e]);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[h][t][e] *= f[t][e & 1];
                }
                // tokens that are not there: behind the end, or without a page
                if (__builtin_expect(have != (1u << HV) - 1 || (sub + 1) * KS > len, 0)) {
#pragma unroll
                    for (int h = 0; h < HV; ++h) {
                        const int left = have >> h & 1u ? len - (sub * KS + h * kSub) : 0;
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[h][t][e] = r + (e < 2 ? 0 : 8) < left ? s[h][t][e] : -INFINITY;
#pragma unroll
                        for (int q = 0; q < NG; ++q) {
                            v0[h][q] = r < left ? v0[h][q] : 0.0f;
                            v1[h][q] = r + 8 < left ? v1[h][q] : 0.0f;
                        }
                    }
                }
                // The running maximum is lazy: raised when a score is 2^8 above
                // it, so most steps need no reduction over the lanes.
                bool raise = false;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(s[0][t][e], s[0][t][2 + e]);
                        if constexpr (HV == 2) x = fmaxf(x, fmaxf(s[1][t][e], s[1][t][2 + e]));
                        raise |= x > m[t][e] + 8.0f;
                    }
                if (__builtin_expect(__any_sync(0xffffffffu, raise), 0)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(s[0][t][e], s[0][t][2 + e]);
                            if constexpr (HV == 2) x = fmaxf(x, fmaxf(s[1][t][e], s[1][t][2 + e]));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            x = fmaxf(x, m[t][e]);
                            // inv takes the increase in whole powers of two, no fewer than it
                            // is, so that exp2(s - m) * inv never becomes less; the sums the rest
                            const float d = x == m[t][e] ? 0.0f : fminf(x - m[t][e], 252.0f), n = ceilf(d), part = exp2_fast(n - d);
                            m[t][e] = x;
                            l[t][e] *= part * pow2(-(int)n);
#pragma unroll
                            for (int q = 0; q < NG; ++q) {
                                const int to = (int)(__float_as_uint(inv[q][t][e]) >> 23) + (int)n, over = max(0, to - kMostInv);
                                inv[q][t][e] = __uint_as_float((uint32_t)(to - over) << 23);
                                const float corr = part * pow2(-over);
#pragma unroll
                                for (int b = q * BPG; b < (q + 1) * BPG && b < NB; ++b)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) acc[b][h][t][e] *= corr, acc[b][h][t][2 + e] *= corr;
                            }
                        }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float base = m[t][e] == -INFINITY ? 0.0f : m[t][e];
#pragma unroll
                        for (int h = 0; h < HV; ++h) {
                            s[h][t][e] = exp2_fast(s[h][t][e] - base);
                            s[h][t][2 + e] = exp2_fast(s[h][t][2 + e] - base);
                            l[t][e] += s[h][t][e] + s[h][t][2 + e];
                        }
                    }
                // The values' scales go with the weights, in the row's units,
                // rounded once to fp16: 2^-11 of each term at most, independent of
                // one another, next to a result of 8 or 11 bits. A unit is raised
                // when one is 2^15 or more, and puts it at 2^8: the largest of a
                // row and group is at least that, so that only those below 2^-22
                // of it lose bits (are 2^-33 of it off). At 2^11, raised more often,
                // 16 sequences of 32 rows a kv head took 77 us, at 2^8 71.
                uint32_t wt[HV][NG][NT][2];
                const auto weigh = [&] {
#pragma unroll
                    for (int h = 0; h < HV; ++h)
#pragma unroll
                        for (int q = 0; q < NG; ++q)
#pragma unroll
                            for (int t = 0; t < NT; ++t) {  // (weight * inv) * scale: no infinity on the way to a number
                                const uint64_t u = both(inv[q][t][0], inv[q][t][1]);
                                const float2 w0 = apart(mul2(mul2(both(s[h][t][0], s[h][t][1]), u), both(v0[h][q], v0[h][q])));
                                const float2 w1 = apart(mul2(mul2(both(s[h][t][2], s[h][t][3]), u), both(v1[h][q], v1[h][q])));
                                wt[h][q][t][0] = pack2(w0.x, w0.y, true);
                                wt[h][q][t][1] = pack2(w1.x, w1.y, true);
                            }
                };
                weigh();
                uint32_t most[4] = {};  // two halves each, none of them negative
#pragma unroll
                for (int h = 0; h < HV; ++h)
#pragma unroll
                    for (int q = 0; q < NG; ++q)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            uint32_t& x = most[((h * NG + q) * NT + t) & 3];
                            x = __vimax3_u16x2(x, wt[h][q][t][0], wt[h][q][t][1]);
                        }
                const uint32_t top = __vimax3_u16x2(__vmaxu2(most[0], most[1]), most[2], most[3]);
                if (__builtin_expect(__any_sync(0xffffffffu, (top + 0x08000800u) & 0x80008000u), 0)) {
#pragma unroll
                    for (int q = 0; q < NG; ++q)
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            uint32_t f[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                float x = 0.0f;  // (a NaN is passed over)
#pragma unroll
                                for (int h = 0; h < HV; ++h)  // 2^-8: the weights are at most 2^8
                                    x = fmaxf(x, fmaxf(s[h][t][e] * 0x1p-8f * v0[h][q], s[h][t][2 + e] * 0x1p-8f * v1[h][q]));
                                f[e] = __float_as_uint(x);
                            }
                            uint32_t x = __byte_perm(f[0], f[1], 0x7632);  // both at their upper 16 bits
                            x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, 16));
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                // the largest to 2^8 .. 2^9, unless it is below that already
                                const int was = (int)(__float_as_uint(inv[q][t][e]) >> 23);
                                const int now = min(was, 2 * 127 + 8 - 8 - (int)(x >> (16 * e + 7) & 255u));
                                inv[q][t][e] = __uint_as_float((uint32_t)now << 23);
                                const float corr = pow2(now - was);
#pragma unroll
                                for (int b = q * BPG; b < (q + 1) * BPG && b < NB; ++b)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) acc[b][h][t][e] *= corr, acc[b][h][t][2 + e] *= corr;
                            }
                        }
                    weigh();
                }
                // output: channels in rows, query rows in columns, the tokens summed
#pragma unroll
                for (int h = 0; h < HV; ++h) {
                    const uint8_t* vb = step + h * HALF + CODES;
                    uint32_t vw[4][(VP + 3) / 4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) lds_part<ROW, VP>(vw[t], vb, (2 * j + (t & 1) + 8 * (t >> 1)) * ROW + r * VP);
                    uint32_t wb[NT][2];
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        if (b % BPG == 0) {
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                wb[t][0] = movm_t(wt[h][b / BPG][t][0]);
                                wb[t][1] = movm_t(wt[h][b / BPG][t][1]);
                            }
                        }
                        uint32_t a[2][4];
                        if constexpr (BITS == 8) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {  // tokens 2j, 2j + 1; then 8 behind
                                const uint32_t lo = __byte_perm(vw[2 * x][b], vw[2 * x + 1][b], 0x5140);
                                const uint32_t hi = __byte_perm(vw[2 * x][b], vw[2 * x + 1][b], 0x7362);
                                a[0][2 * x] = bytes2<0>(lo), a[0][2 * x + 1] = bytes2<2>(lo);
                                a[1][2 * x] = bytes2<0>(hi), a[1][2 * x + 1] = bytes2<2>(hi);
                            }
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                uint32_t n[4];
                                nibbles4(n, __byte_perm(vw[2 * x][b >> 1], vw[2 * x + 1][b >> 1], b & 1 ? 0x7632 : 0x5410));
#pragma unroll
                                for (int c = 0; c < 4; ++c) a[c >> 1][2 * x + (c & 1)] = n[c];
                            }
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int t = 0; t < NT; ++t) Fp16::mma(acc[b][c][t], a[c], wb[t][0], wb[t][1]);
                    }
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncthreads();

        // join the warps: each leaves the mean of its values, which are in the
        // range of a float whatever the number of tokens, and its sum of weights
        float* sums = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 4);
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 8);
                l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 16);
                // a sum that is NaN with no maximum (all scores NaN) is not an empty one
                if (m[t][e] == -INFINITY && l[t][e] != 0.0f) m[t][e] = 0.0f;
                const int row = t * 8 + 2 * j + e;
                if (r == 0) wml[warp * R + row] = make_float2(m[t][e], l[t][e]);
                const float norm = l[t][e] == 0.0f ? 0.0f : 1.0f / l[t][e];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float unit = __uint_as_float((254u << 23) - __float_as_uint(inv[b / BPG][t][e]));
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<float2*>(sums + (warp * R + row) * (DP + 8) + 32 * b + 4 * r + 2 * h) =
                            make_float2(acc[b][h][t][e] * norm * unit, acc[b][h][t][2 + e] * norm * unit);
                }
            }
        __syncthreads();
        const bool whole = blk0 == 0 && blk1 == nb;
        const int64_t slot = whole ? 2 * (int64_t)gridDim.x + (int64_t)grp * items + item : 2 * (int64_t)blockIdx.x + (blk0 == 0);
        const bool direct = whole && !p.partial;
        // a thread a row: the warps' weights, in the place of their maxima
        if (tid < rows) {
            float top = -INFINITY, c[kWarps], sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wml[w * R + tid].x);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 ml = wml[w * R + tid];
                c[w] = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top) * ml.y;
                sum += c[w];
            }
            const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) wml[w * R + tid].x = c[w] * norm;
            const int row = row0 + tid;
            if (!direct) p.pml[slot * R + tid] = make_float2(top, sum);
            else if (p.lse)
                p.lse[(int64_t)(row / p.share) * g.heads * p.share + head * p.share + row % p.share] =
                    sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
        }
        __syncthreads();
        for (int n = tid; n < rows * (DP / 4); n += 32 * kWarps) {
            const int i = n / (DP / 4), d = n % (DP / 4) * 4;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float c = wml[w * R + i].x;
                const float4 x = *reinterpret_cast<const float4*>(sums + (w * R + i) * (DP + 8) + d);
                v.x = fmaf(c, x.x, v.x), v.y = fmaf(c, x.y, v.y), v.z = fmaf(c, x.z, v.z), v.w = fmaf(c, x.w, v.w);
            }
            if (!direct) {
                *reinterpret_cast<float4*>(p.pacc + (slot * R + i) * DP + d) = v;
            } else if (d < g.dim) {
                const int row = row0 + i, seq = row / p.share;
                uint16_t* to = p.out + seq * p.o_seq + (head * p.share + row - seq * p.share) * p.o_head + d;
                const uint32_t lo = pack2(v.x, v.y, p.fp16), hi = pack2(v.z, v.w, p.fp16);
                if (p.o_vec) {
                    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
                } else {
                    to[0] = (uint16_t)lo, to[1] = (uint16_t)(lo >> 16), to[2] = (uint16_t)hi, to[3] = (uint16_t)(hi >> 16);
                }
            }
        }
        __syncthreads();
        u += blk1 - blk0;
    }
    if (p.second) grid_wait();  // the join then follows both
}

// ---------------------------------------------------------------- join
// For each query row the parts of its items, of its own positions (and of the
// prefix), each a mean with the maximum and the sum of its weights. PER = 4: a
// CTA a row, whose warps share the parts, where there are few rows, of many
// parts each; PER = 1: a warp a row, which saves the join of the warps. Whole
// attentions: 64 ragged sequences of 64 heads 78 us with 1, 85 with 4; 82
// sequences of 64 heads behind 64 tokens 42 and 56; 96 of 16 behind 8190 44
// and 46.5; 48 of 16 behind 8190 34.6 and 33.2; 16 ragged ones of 64 28.7 and
// 27.0; one of 32 heads, 100003 tokens, 60 and 49.
struct JoinSide {
    const int2* owners;  // nullptr: this side has nothing
    const float* pacc;
    const float2* pml;
    const int32_t* lengths;
    int length;
    int rg, rt, R, ctas;
};
struct JoinParams {
    JoinSide side[2];  // own positions, prefix
    int rows;  // query rows
    int heads, share, dim, dp;
    int width[2];  // pages of the tables
    uint16_t* out;
    int64_t o_seq, o_head;
    float* lse;
    bool fp16, partial, o_vec;
};

constexpr int kJoinWarps = 4;

template <int PER>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const JoinParams p) {
    __shared__ __align__(16) float sums[PER][256];
    __shared__ float2 wml[PER];
    grid_wait();
    grid_launch();
    const int lane = threadIdx.x & 31, warp = PER == 1 ? 0 : threadIdx.x >> 5;  // of the row's
    const int q_heads = p.heads * p.share;
    constexpr int ROWS = kJoinWarps / PER;  // of a CTA at a time
    const int row0 = blockIdx.x * ROWS + (PER == 1 ? threadIdx.x >> 5 : 0);
    for (int n = row0; n < p.rows; n += gridDim.x * ROWS) {
        const int seq = n / q_heads, qh = n % q_heads, head = qh / p.share;
        const int row = seq * p.share + qh % p.share;  // of the kv head's query rows
        float m = -INFINITY, l = 0.0f, acc[8] = {};
        // on each side the item that the row is in, the row's place in it, and
        // the CTAs that have its parts
        int2 own[2];
        int item[2], i[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const JoinSide& s = p.side[w];
            own[w] = make_int2(0, -1), item[w] = i[w] = 0;
            if (!s.owners) continue;
            const int grp = row / s.rg, in = row % s.rg;
            i[w] = in % s.R, item[w] = (grp * p.heads + head) * s.rt + in / s.R;
            const int2 got = s.owners[item[w]];  // not written where the length is 0
            if ((s.lengths ? s.lengths[grp] : s.length) > 0 && p.width[w] > 0) own[w] = got;
        }
        if (!p.partial && own[0].x >= own[0].y) continue;  // the attention kernel has finished this row itself
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const JoinSide& s = p.side[w];
            // a lane reads the maximum and sum of a part, then all read its values
            for (int c = own[w].x + warp; c <= own[w].y; c += 32 * PER) {
                const int mine = c + lane * PER;
                const int64_t slot = own[w].x == own[w].y ? 2 * (int64_t)s.ctas + item[w] : 2 * (int64_t)mine + (mine == own[w].x);
                float2 ml = make_float2(-INFINITY, 0.0f);
                if (mine <= own[w].y) ml = s.pml[slot * s.R + i[w]];
                float top = ml.x;
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(top, m);
                const float a = m == -INFINITY ? 0.0f : exp2_fast(m - top);
                const float b = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);  // 0: this part saw nothing
                const float part = ml.x == -INFINITY ? 0.0f : b * ml.y;
                float sum = part;
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                m = top;
                sum += l * a;
                const float norm = sum == 0.0f ? 0.0f : 1.0f / sum, old = l * a * norm;
                l = sum;
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[k] *= old;
                // (a part that saw nothing has left zeros)
                const int parts = min(32, (own[w].y - c) / PER + 1);
#pragma unroll 8
                for (int q = 0; q < parts; ++q) {
                    const float f = __shfl_sync(0xffffffffu, part * norm, q);
                    const int64_t from = __shfl_sync(0xffffffffu, slot, q);
                    const float* x = s.pacc + (from * s.R + i[w]) * p.dp + 4 * lane;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (128 * k + 4 * lane < p.dp) {
                            const float4 v = *reinterpret_cast<const float4*>(x + 128 * k);
                            acc[4 * k] = fmaf(f, v.x, acc[4 * k]), acc[4 * k + 1] = fmaf(f, v.y, acc[4 * k + 1]);
                            acc[4 * k + 2] = fmaf(f, v.z, acc[4 * k + 2]), acc[4 * k + 3] = fmaf(f, v.w, acc[4 * k + 3]);
                        }
                }
            }
        }
        if constexpr (PER == 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int d = 128 * k + 4 * lane;
                if (d >= p.dim) continue;
                uint16_t* to = p.out + seq * p.o_seq + qh * p.o_head + d;
                const uint32_t lo = pack2(acc[4 * k], acc[4 * k + 1], p.fp16);
                const uint32_t hi = pack2(acc[4 * k + 2], acc[4 * k + 3], p.fp16);
                if (p.o_vec) {
                    *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
                } else {
                    to[0] = (uint16_t)lo, to[1] = (uint16_t)(lo >> 16), to[2] = (uint16_t)hi, to[3] = (uint16_t)(hi >> 16);
                }
            }
            if (p.lse && lane == 0) p.lse[(int64_t)seq * q_heads + qh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
            continue;
        }
        if (lane == 0) wml[warp] = make_float2(m, l);
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (128 * k + 4 * lane < p.dp)
                *reinterpret_cast<float4*>(&sums[warp][128 * k + 4 * lane]) = make_float4(acc[4 * k], acc[4 * k + 1], acc[4 * k + 2], acc[4 * k + 3]);
        __syncthreads();
        float top = -INFINITY, c[PER], sum = 0.0f;
#pragma unroll
        for (int w = 0; w < PER; ++w) top = fmaxf(top, wml[w].x);
#pragma unroll
        for (int w = 0; w < PER; ++w) {
            c[w] = wml[w].x == -INFINITY ? 0.0f : exp2_fast(wml[w].x - top) * wml[w].y;
            sum += c[w];
        }
        const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (int d = threadIdx.x; d < p.dim; d += 32 * PER) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < PER; ++w)
                if (c[w] != 0.0f) v = fmaf(c[w] * norm, sums[w][d], v);
            p.out[seq * p.o_seq + qh * p.o_head + d] = (uint16_t)pack2(v, 0.0f, p.fp16);
        }
        if (p.lse && threadIdx.x == 0)
            p.lse[(int64_t)seq * q_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host
// One attention kernel launch: tile of rows, CTAs, stages, and its part of
// the workspace. Depends on the handle and the call's sizes alone.
struct Plan {
    int n_grp, rg, nt, rt, ctas, stages, smem;
    int64_t slots;
    size_t own_bytes, acc_bytes, ml_bytes;
    size_t bytes() const { return own_bytes + acc_bytes + ml_bytes; }
};

Plan attend_plan(const bnn_kv_cache* c, int n_grp, int rg, bool partial) {
    const KvGeo& g = c->geo;
    Plan s{};
    s.n_grp = n_grp;
    s.rg = rg;
    const int most = g.dp <= 128 ? 4 : 2;  // registers: dp * nt sums over a warp's lanes
    s.nt = rg <= 8 ? 1 : rg <= 16 || most == 2 ? 2 : 4;
    s.rt = (int)cdiv64(rg, 8 * s.nt);
    const int per_sm = attend_ctas(g.dp, s.nt);
    s.ctas = (c->sms > 0 ? c->sms : 148) * per_sm;
    const int R = 8 * s.nt;
    s.stages = 2;
    while (s.stages < 6 && attend_smem(g, n_grp, s.nt, s.stages + 1).bytes <= 224 * 1024 / per_sm - 1024) ++s.stages;
    s.smem = attend_smem(g, n_grp, s.nt, s.stages).bytes;
    s.slots = 2 * (int64_t)s.ctas + (partial ? (int64_t)n_grp * g.heads * s.rt : 0);
    const auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    s.own_bytes = up((size_t)n_grp * g.heads * s.rt * 8);
    s.acc_bytes = up((size_t)s.slots * R * g.dp * 4);
    s.ml_bytes = up((size_t)s.slots * R * 8);
    return s;
}

// f(kernel) of a cache's kernel for nt row tiles
template <int DP, int BITS, int BPG, class F>
cudaError_t attend_rows(int nt, F&& f) {
    if (nt == 1) return f(attend_kernel<DP, BITS, 1, BPG>);
    if (nt == 2) return f(attend_kernel<DP, BITS, 2, BPG>);
    if constexpr (DP <= 128) return f(attend_kernel<DP, BITS, 4, BPG>);
    return cudaErrorInvalidValue;
}
template <int DP, int BITS, class F>
cudaError_t attend_group(const KvGeo& g, int nt, F&& f) {
    if (g.ng == 1) return attend_rows<DP, BITS, 8>(nt, f);
    if (g.group == 32) return attend_rows<DP, BITS, 1>(nt, f);
    if constexpr (DP > 64)
        if (g.group == 64) return attend_rows<DP, BITS, 2>(nt, f);
    if constexpr (DP > 128)
        if (g.group == 128) return attend_rows<DP, BITS, 4>(nt, f);
    return cudaErrorInvalidValue;
}
template <int BITS, class F>
cudaError_t attend_dim(const KvGeo& g, int nt, F&& f) {
    switch (g.dp) {
        case 64: return attend_group<64, BITS>(g, nt, f);
        case 128: return attend_group<128, BITS>(g, nt, f);
        case 192: return attend_group<192, BITS>(g, nt, f);
        default: return attend_group<256, BITS>(g, nt, f);
    }
}
template <class F>
cudaError_t attend_any(const KvGeo& g, int nt, F&& f) {
    return g.bits == 8 ? attend_dim<8>(g, nt, f) : attend_dim<4>(g, nt, f);
}

constexpr int kMaxSeqs = 16384;

int attend_check(const bnn_kv_cache* c, int n_seqs, int q_heads, int prefix_tokens) {
    if (!c || n_seqs < 0 || n_seqs > kMaxSeqs || prefix_tokens < 0)
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: bad arguments (0 .. %d sequences, a prefix of 0 or more tokens)", kMaxSeqs);
    if (q_heads <= 0 || q_heads % c->geo.heads || q_heads > 65536)
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: %d query heads are no multiple of %d kv heads", q_heads, c->geo.heads);
    return BNN_OK;
}

}  // namespace

cudaError_t attend_setup(const KvGeo& g) {
    // the kernels may use all of an SM's shared memory
    cudaError_t e = cudaSuccess;
    for (int nt = 1; nt <= (g.dp <= 128 ? 4 : 2) && e == cudaSuccess; nt *= 2)
        e = attend_any(g, nt, [](auto k) { return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, 226 * 1024); });
    return e;
}

}  // namespace lowbit
}  // namespace bnn

using namespace bnn;
using namespace bnn::lowbit;

BNN_API size_t bnn_kv_attend_work(const bnn_kv_cache* c, int n_seqs, int q_heads, int prefix_tokens) {
    if (attend_check(c, n_seqs, q_heads, prefix_tokens) || n_seqs == 0) return 0;
    const int share = q_heads / c->geo.heads;
    size_t n = attend_plan(c, n_seqs, share, prefix_tokens > 0).bytes();
    if (prefix_tokens > 0) n += attend_plan(c, 1, n_seqs * share, true).bytes();
    return n;
}

BNN_API int bnn_kv_attend(const bnn_kv_cache* c, const void* d_q, int64_t q_seq, int64_t q_head, int n_seqs, int q_heads,
                          const int32_t* d_lengths, const int32_t* d_table, int table_pages, const int32_t* d_prefix,
                          int prefix_pages, int prefix_tokens, float scale, void* d_out, int64_t o_seq, int64_t o_head,
                          float* d_lse, void* d_work, size_t work_bytes, void* stream) {
    int rc = attend_check(c, n_seqs, q_heads, prefix_tokens);
    if (rc) return rc;
    const KvGeo& g = c->geo;
    const bool prefix = prefix_tokens > 0;
    const float scale_log2 = scale * 1.4426950408889634f;
    if (table_pages < 0 || prefix_pages < 0 || !(scale_log2 - scale_log2 == 0.0f))
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: negative table width, or a scale that is not finite");
    if ((int64_t)table_pages * g.pt > INT_MAX - 256 || (int64_t)prefix_pages * g.pt > INT_MAX - 256)
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: a table of 2^31 tokens or more");
    if (n_seqs > 0 && q_heads > INT_MAX / n_seqs) return set_error(BNN_ERR_ARG, "bnn_kv_attend: %d sequences of %d heads", n_seqs, q_heads);
    if (n_seqs * (cdiv64((int64_t)table_pages * g.pt, kBlock) + cdiv64(prefix_tokens, kBlock)) > INT_MAX / q_heads)
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: %d sequences of up to %lld tokens are too many for one call", n_seqs,
                         (long long)table_pages * g.pt);
    if (prefix && (!d_prefix || (int64_t)prefix_pages * g.pt < prefix_tokens))
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: a prefix of %d tokens needs %lld pages", prefix_tokens,
                         (long long)cdiv64(prefix_tokens, g.pt));
    if (n_seqs > 0) {
        if (!d_q || !d_lengths || !d_out || (!d_table && table_pages > 0))
            return set_error(BNN_ERR_ARG, "bnn_kv_attend: NULL argument");
        if (!aligned(d_q, 2) || !aligned(d_out, 2) || !aligned(d_lengths, 4) || !aligned(d_table, 4) || !aligned(d_prefix, 4) ||
            !aligned(d_lse, 4))
            return set_error(BNN_ERR_ARG, "bnn_kv_attend: an array is not aligned to its type");
        if ((q_heads > 1 && o_head < g.dim) || (n_seqs > 1 && o_seq < g.dim))
            return set_error(BNN_ERR_ARG, "bnn_kv_attend: strides %lld, %lld of the output: at least %d", (long long)o_seq,
                             (long long)o_head, g.dim);
        if (rows_share(n_seqs, o_seq, q_heads, o_head, g.dim))
            return set_error(BNN_ERR_ARG, "bnn_kv_attend: strides %lld, %lld put heads of the output over one another", (long long)o_seq,
                             (long long)o_head);
        const size_t need = bnn_kv_attend_work(c, n_seqs, q_heads, prefix_tokens);
        if (!d_work || work_bytes < need || !aligned(d_work, 16))
            return set_error(BNN_ERR_ARG, "bnn_kv_attend: %zu bytes of workspace, 16-byte aligned, are needed (%zu given)", need,
                             d_work ? work_bytes : 0);
    }
    if (c->device < 0) return no_device("bnn_kv_attend");
    if (n_seqs == 0) return BNN_OK;
    DeviceScope dev(c->device);
    if (dev.err != cudaSuccess) return cuda_error("bnn_kv_attend", dev.err);
    const cudaStream_t st = (cudaStream_t)stream;
    const int share = q_heads / g.heads;

    AttendParams p{};
    p.g = g;
    p.kc = c->kc, p.vc = c->vc, p.ks = c->ks, p.vs = c->vs;
    p.q = (const uint16_t*)d_q, p.q_seq = q_seq, p.q_head = q_head;
    p.out = (uint16_t*)d_out, p.o_seq = o_seq, p.o_head = o_head, p.lse = d_lse;
    p.fp16 = c->type == BNN_FP16;
    p.q_vec = aligned(d_q, 16) && (n_seqs == 1 || q_seq % 8 == 0) && (q_heads == 1 || q_head % 8 == 0);
    p.o_vec = aligned(d_out, 8) && (n_seqs == 1 || o_seq % 4 == 0) && (q_heads == 1 || o_head % 4 == 0);
    p.share = share;
    p.scale_log2 = scale_log2;
    p.partial = prefix;
    JoinParams jp{};
    jp.rows = n_seqs * q_heads;
    jp.heads = g.heads, jp.share = share, jp.dim = g.dim, jp.dp = g.dp;
    jp.out = p.out, jp.o_seq = o_seq, jp.o_head = o_head, jp.lse = d_lse;
    jp.fp16 = p.fp16, jp.partial = prefix, jp.o_vec = p.o_vec;
    uint8_t* work = (uint8_t*)d_work;
    for (int side = prefix ? 1 : 0; side >= 0; --side) {
        const Plan s = side ? attend_plan(c, 1, n_seqs * share, true) : attend_plan(c, n_seqs, share, prefix);
        p.n_grp = s.n_grp, p.rg = s.rg, p.rt = s.rt, p.stages = s.stages;
        p.lengths = side ? nullptr : d_lengths;
        p.length = side ? prefix_tokens : 0;
        p.table = side ? d_prefix : d_table;
        p.width = side ? prefix_pages : table_pages;
        p.owners = (int2*)work;
        p.pacc = (float*)(work + s.own_bytes);
        p.pml = (float2*)(work + s.own_bytes + s.acc_bytes);
        work += s.bytes();
        p.second = prefix && side == 0 && pdl_on();
        // Started early, its CTAs would find the places of an SM taken by
        // those of the kernel before, and their shares are equal: 85 us
        // against 78 for 64 ragged sequences in 4 bits.
        const cudaError_t e = attend_any(g, s.nt, [&](auto k) { return launch(k, dim3(s.ctas), 32 * kWarps, s.smem, st, p.second, p); });
        if (e != cudaSuccess) return cuda_error("bnn_kv_attend", e);
        jp.side[side] = JoinSide{p.owners, p.pacc, p.pml, p.lengths, p.length, s.rg, s.rt, 8 * s.nt, s.ctas};
        jp.width[side] = p.width;
    }
    // no sequence can be longer than a block: none is cut
    if (!prefix && (int64_t)table_pages * g.pt <= kLong) return BNN_OK;
    const bool alone = jp.rows > 10 * c->sms;
    const int ctas = alone ? (int)cdiv64(jp.rows, kJoinWarps) : jp.rows;
    const cudaError_t e = launch(alone ? join_kernel<1> : join_kernel<kJoinWarps>, dim3((unsigned)min(ctas, c->sms * 12)), 32 * kJoinWarps, 0, st, true, jp);
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_kv_attend", e);
}
