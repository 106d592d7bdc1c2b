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
constexpr int kSub = 16;  // tokens a warp takes at a time

struct AttendParams {
    KvGeo g;
    const uint8_t *kc, *vc;
    const uint16_t *ks, *vs;
    const uint16_t* q;
    int64_t q_seq, q_head;
    uint16_t* out;
    int64_t o_seq, o_head;
    float* lse;
    bool fp16, q_vec;
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
    int32_t* pre;            // [n_grp + 1]: blocks before each group, for the join
    float* pacc;             // [slot][row][dp] sums of exp2(s - m) * value
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

// codes to fp16 pairs: a byte or nibble in the low mantissa bits of 1024
// gives 1024 + it, and the subtraction leaves the code, exactly
template <int LO>
__device__ __forceinline__ uint32_t pair8(uint32_t w) {  // bytes LO and LO + 1 of w
    return Fp16::sub2(__byte_perm(w, 0x64646464u, LO ? 0x4342 : 0x4140), 0x64806480u);
}
__device__ __forceinline__ uint32_t pair4(uint32_t w, int nib) {  // nibbles at 4 * nib of both halves
    return Fp16::sub2(and_or(w >> (4 * nib), 0x000f000fu, 0x64006400u), 0x64086408u);
}

template <int DP, int BITS>
struct AttendSmem {
    static constexpr int ROW = DP * BITS / 8;
    static constexpr int CODES = kSub * ROW;  // bytes of 16 rows
    __host__ __device__ static int stage(int ng) { return 2 * CODES + ((2 * ng * kSub * 2 + 127) & ~127); }
    __host__ __device__ static int qfrag(int nt) { return DP / 32 * nt * 512; }
    __host__ __device__ static int merge(int nt) { return kWarps * 8 * nt * (DP + 8) * 4; }
    // prefix sums | row factors | row (m, l) of the warps | q fragments | stages, later the warps' sums
    __host__ __device__ static int head(int n_grp, int nt) {
        return (((n_grp + 1) * 4 + 127) & ~127) + 128 * ((8 * nt * 4 + 127) / 128) + kWarps * 8 * nt * 8;
    }
    __host__ __device__ static int bytes(int n_grp, int nt, int ng, int stages) {
        const int ring = kWarps * stages * stage(ng), m = merge(nt);
        return head(n_grp, nt) + qfrag(nt) + (ring > m ? ring : m);
    }
};

template <int DP, int BITS, int NT>
__global__ void __launch_bounds__(32 * kWarps, DP <= 128 && NT == 1 ? 3 : 2) attend_kernel(const AttendParams p) {
    using S = AttendSmem<DP, BITS>;
    constexpr int NB = DP / 32, R = 8 * NT, ROW = S::ROW;
    constexpr int KP = ROW / 4, VP = ROW / 8;  // a lane's bytes of a key's, a value's row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int warp_sum[kWarps];
    const KvGeo g = p.g;
    int* pre = reinterpret_cast<int*>(smem);
    float* factor = reinterpret_cast<float*>(smem + (((p.n_grp + 1) * 4 + 127) & ~127));
    float2* wml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(factor) + 128 * ((R * 4 + 127) / 128));
    uint4* qf = reinterpret_cast<uint4*>(smem + S::head(p.n_grp, NT));
    uint8_t* ring = reinterpret_cast<uint8_t*>(qf) + S::qfrag(NT);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, j = lane & 3;

    // blocks before each group
    {
        const int per = (p.n_grp + 32 * kWarps - 1) / (32 * kWarps), b0 = tid * per, b1 = min(p.n_grp, b0 + per);
        int sum = 0;
        for (int b = b0; b < b1; ++b) sum += (grp_len(p, b) + kBlock - 1) / kBlock;
        int inc = sum;
        for (int s = 1; s < 32; s <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, inc, s);
            if (lane >= s) inc += o;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int at = inc - sum;
        for (int w = 0; w < warp; ++w) at += warp_sum[w];
        for (int b = b0; b < b1; ++b) {
            pre[b] = at;
            at += (grp_len(p, b) + kBlock - 1) / kBlock;
        }
        if (b0 < p.n_grp && b1 == p.n_grp) pre[p.n_grp] = at;
        __syncthreads();
    }
    if (blockIdx.x == 0)
        for (int b = tid; b <= p.n_grp; b += 32 * kWarps) p.pre[b] = pre[b];
    const int items = g.heads * p.rt;  // of a group
    const int64_t units = (int64_t)pre[p.n_grp] * items;
    const int ctas = split_ctas(units, gridDim.x);
    const bool has = (int)blockIdx.x < ctas;
    const int64_t u_end = has ? split_begin(units, blockIdx.x + 1, ctas) : 0;
    int64_t u = has ? split_begin(units, blockIdx.x, ctas) : 0;

    // groups with nothing in them
    if (!p.partial)
        for (int b = blockIdx.x; b < p.n_grp; b += gridDim.x) {
            if (pre[b + 1] != pre[b]) continue;
            for (int i = tid; i < g.heads * p.share * g.dim; i += 32 * kWarps) {
                const int head = i / g.dim, d = i % g.dim;
                p.out[b * p.o_seq + head * p.o_head + d] = 0;
                if (p.lse && d == 0) p.lse[(int64_t)b * g.heads * p.share + head] = -INFINITY;
            }
        }

    int grp = 0;
    while (u < u_end) {
        // the item of block u, and the blocks of it that are this CTA's
        {
            int lo = grp, hi = p.n_grp;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)pre[mid] * items <= u) lo = mid;
                else hi = mid;
            }
            grp = lo;
        }
        const int nb = pre[grp + 1] - pre[grp];
        const int64_t in_grp = u - (int64_t)pre[grp] * items;
        const int item = (int)(in_grp / nb), blk0 = (int)(in_grp % nb);
        const int blk1 = (int)min((int64_t)nb, blk0 + (u_end - u));
        const int head = item / p.rt, tile = item % p.rt;
        const int len = grp_len(p, grp);
        const int rows = min(R, p.rg - tile * R);
        const int64_t row0 = (int64_t)grp * p.rg + tile * R;  // row i of the item: query row (row0 + i)

        // q as B fragments of fp16, each row scaled by a power of two that
        // puts its largest value in [2^9, 2^10): exact but for values
        // 2^-24 and less of the row's largest
        for (int i = warp; i < R; i += kWarps) {
            float x[8] = {};
            if (i < rows && 8 * lane < g.dim) {
                const int64_t at = row0 + i;
                const uint4 v = load8(p.q + at / p.share * p.q_seq + (head * p.share + at % p.share) * p.q_head + 8 * lane,
                                      g.dim - 8 * lane, p.q_vec);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float2 f = unpack2(w[c], p.fp16);
                    x[2 * c] = f.x, x[2 * c + 1] = f.y;
                }
            }
            uint32_t top = 0;
#pragma unroll
            for (int c = 0; c < 8; ++c) top = max(top, __float_as_uint(x[c]) & 0x7fffffffu);
            top = __reduce_max_sync(0xffffffffu, top);
            const int e = (int)(top >> 23);  // 127 + exponent of the largest; 255: not finite
            const int sh = top == 0 || e == 255 ? 0 : max(-126, min(126, 9 + 127 - e));
            const float up = __int_as_float((127 + sh) << 23);
            if (lane < DP / 8) {
                uint4 v;
                v.x = pack2(x[0] * up, x[1] * up, true);
                v.y = pack2(x[2] * up, x[3] * up, true);
                v.z = pack2(x[4] * up, x[5] * up, true);
                v.w = pack2(x[6] * up, x[7] * up, true);
                qf[((lane >> 2) * NT + (i >> 3)) * 32 + (i & 7) * 4 + (lane & 3)] = v;
            }
            if (lane == 0) factor[i] = p.scale_log2 * __int_as_float((127 - sh) << 23);
        }
        __syncthreads();

        float acc[NB][2][NT][4], m[NT][2], l[NT][2], f[NT][2];
        uint32_t ev[NB];  // exponent field (bf16 bits) of the unit that acc is in, per 32 channels
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            ev[b] = 4u << 7;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][h][t][e] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[t][e] = -INFINITY, l[t][e] = 0.0f;
                f[t][e] = factor[t * 8 + 2 * j + e];
            }

        const int sub0 = blk0 * (kBlock / kSub), sub1 = min(blk1 * (kBlock / kSub), (len + kSub - 1) / kSub);
        const int stage_bytes = S::stage(g.ng);
        uint8_t* mine = ring + warp * p.stages * stage_bytes;
        const int32_t* row_table = p.table + (int64_t)grp * p.width;
        const int bpg = g.ng == 1 ? 8 : g.group / 32;  // 32-blocks a scale covers, a power of two

        // copies of one 16-token block into a stage; its page
        const auto fetch = [&](int sub, uint8_t* to) -> int {
            const int pos = sub * kSub, page = kv_page(g, row_table, p.width, pos);
            if (page < 0) return -1;
            const int tok = pos & (g.pt - 1);
            const int64_t at = kv_row(g, page, head, tok);
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
            static_assert(S::CODES % 512 == 0, "whole pieces for every lane");
#pragma unroll
            for (int c = 0; c < S::CODES / 512; ++c) {
                const int o = (c * 32 + lane) * 16;
                cp16(dst + swz<ROW>(o), p.kc + at + o);
                cp16(dst + S::CODES + swz<ROW>(o), p.vc + at + o);
            }
            if (lane < 4 * g.ng) {
                const int of = lane >= 2 * g.ng, c = of ? lane - 2 * g.ng : lane;
                const uint16_t* src = (of ? p.vs : p.ks) + kv_scale(g, page, head, c >> 1, tok) + 8 * (c & 1);
                cp16(dst + 2 * S::CODES + (of * g.ng * kSub + (c >> 1) * kSub + 8 * (c & 1)) * 2, src);
            }
            return page;
        };
        // pages of the blocks in flight, one bit each: there or not
        uint32_t there = 0;
        int ahead = sub0 + warp;
        for (int s = 0; s < p.stages - 1; ++s, ahead += kWarps) {
            if (ahead < sub1 && fetch(ahead, mine + s * stage_bytes) >= 0) there |= 1u << s;
            cp_commit();
        }
        int st = 0, st_in = p.stages - 1;
        for (int sub = sub0 + warp; sub < sub1; sub += kWarps) {
            // the stage read a round ago is free: all lanes passed the barrier below
            there &= ~(1u << st_in);
            if (ahead < sub1 && fetch(ahead, mine + st_in * stage_bytes) >= 0) there |= 1u << st_in;
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
            const uint8_t* kb = mine + st * stage_bytes;
            const bool page_there = there >> st & 1u;
            st = st + 1 == p.stages ? 0 : st + 1;
            if (page_there) {
                const uint8_t* vb = kb + S::CODES;
                const uint16_t* ksc = reinterpret_cast<const uint16_t*>(kb + 2 * S::CODES);
                const uint16_t* vsc = ksc + g.ng * kSub;
                // scores: tokens r and r + 8 in rows, query rows in columns
                float s[NT][4] = {};
                {
                    uint32_t k0[KP / 4], k1[KP / 4];
                    lds_part<ROW, KP>(k0, kb, r * ROW + j * KP);
                    lds_part<ROW, KP>(k1, kb, (r + 8) * ROW + j * KP);
                    float c[NT][4] = {};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint4 qv[NT];
#pragma unroll
                        for (int t = 0; t < NT; ++t) qv[t] = qf[(b * NT + t) * 32 + lane];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t a[4];
                            if constexpr (BITS == 8) {
                                a[0] = pair8<0>(k0[2 * b + h]), a[1] = pair8<0>(k1[2 * b + h]);
                                a[2] = pair8<2>(k0[2 * b + h]), a[3] = pair8<2>(k1[2 * b + h]);
                            } else {
                                a[0] = pair4(k0[b], 2 * h), a[1] = pair4(k1[b], 2 * h);
                                a[2] = pair4(k0[b], 2 * h + 1), a[3] = pair4(k1[b], 2 * h + 1);
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t) Fp16::mma(c[t], a, h ? qv[t].z : qv[t].x, h ? qv[t].w : qv[t].y);
                        }
                        if (b == NB - 1 || ((b + 1) & (bpg - 1)) == 0) {
                            // the group's scale, on its sum of products
                            const int grp_at = min(b / bpg, g.ng - 1) * kSub;
                            const float s0 = bf16_float(ksc[grp_at + r]), s1 = bf16_float(ksc[grp_at + r + 8]);
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                s[t][0] = fmaf(s0, c[t][0], s[t][0]), s[t][1] = fmaf(s0, c[t][1], s[t][1]);
                                s[t][2] = fmaf(s1, c[t][2], s[t][2]), s[t][3] = fmaf(s1, c[t][3], s[t][3]);
                                c[t][0] = c[t][1] = c[t][2] = c[t][3] = 0.0f;
                            }
                        }
                    }
                }
                const bool in0 = sub * kSub + r < len, in1 = sub * kSub + r + 8 < len;
                // The running maximum is one that was the maximum when it was
                // last raised: it is raised when a score is 2^8 above it, so
                // most blocks need no reduction over the lanes. exp2 of at
                // most 8 stays in fp16 and the ratio to the sum is the same.
                bool raise = false;
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[t][e] = in0 ? s[t][e] * f[t][e] : -INFINITY;
                        s[t][2 + e] = in1 ? s[t][2 + e] * f[t][e] : -INFINITY;
                        raise |= fmaxf(s[t][e], s[t][2 + e]) > m[t][e] + 8.0f;
                    }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(s[t][e], s[t][2 + e]);
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            x = fmaxf(x, m[t][e]);
                            const float corr = x == m[t][e] ? 1.0f : exp2_fast(m[t][e] - x);
                            m[t][e] = x;
                            l[t][e] *= corr;
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int h = 0; h < 2; ++h) acc[b][h][t][e] *= corr, acc[b][h][t][2 + e] *= corr;
                        }
                }
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float base = m[t][e] == -INFINITY ? 0.0f : m[t][e];
                        s[t][e] = exp2_fast(s[t][e] - base);
                        s[t][2 + e] = exp2_fast(s[t][2 + e] - base);
                        l[t][e] += s[t][e] + s[t][2 + e];
                    }
                // output: channels in rows, query rows in columns, the tokens
                // summed. The values' scales go with the weights: weight *
                // scale in units of a power of two near the largest scale so
                // far (bf16 scales reach beyond fp16), rounded once to fp16.
                // Error: 2^-12 of each term, independent of one another, next
                // to a result of 8 or 11 bits.
                uint32_t vw[4][(VP + 3) / 4];
#pragma unroll
                for (int t = 0; t < 4; ++t) lds_part<ROW, VP>(vw[t], vb, (2 * j + (t & 1) + 8 * (t >> 1)) * ROW + r * VP);
                uint32_t e_new = 0;
                uint32_t wb[NT][2];
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if ((b & (bpg - 1)) == 0 || b == 0) {
                        const int grp_at = min(b / bpg, g.ng - 1) * kSub;
                        const uint32_t u0 = in0 ? vsc[grp_at + r] : 0u, u1 = in1 ? vsc[grp_at + r + 8] : 0u;
                        const uint32_t big = max(u0 < 0x7f80u ? u0 : 0u, u1 < 0x7f80u ? u1 : 0u);
                        e_new = max(ev[b], min(__reduce_max_sync(0xffffffffu, big) & 0x7f80u, 253u << 7));
                        const float inv = __uint_as_float((254u << 23) - (e_new << 16));
                        const float w0 = bf16_float((uint16_t)u0) * inv, w1 = bf16_float((uint16_t)u1) * inv;
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            wb[t][0] = movm_t(pack2(s[t][0] * w0, s[t][1] * w0, true));
                            wb[t][1] = movm_t(pack2(s[t][2] * w1, s[t][3] * w1, true));
                        }
                    }
                    if (e_new != ev[b]) {
                        const int down = (int)((e_new - ev[b]) >> 7);
                        const float corr = down > 126 ? 0.0f : __int_as_float((127 - down) << 23);
                        ev[b] = e_new;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int t = 0; t < NT; ++t)
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[b][h][t][e] *= corr;
                    }
                    uint32_t a[2][4];
                    if constexpr (BITS == 8) {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {  // tokens 2j, 2j + 1; then 8 behind
                            const uint32_t lo = __byte_perm(vw[2 * x][b], vw[2 * x + 1][b], 0x5140);
                            const uint32_t hi = __byte_perm(vw[2 * x][b], vw[2 * x + 1][b], 0x7362);
                            a[0][2 * x] = pair8<0>(lo), a[0][2 * x + 1] = pair8<2>(lo);
                            a[1][2 * x] = pair8<0>(hi), a[1][2 * x + 1] = pair8<2>(hi);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t v = __byte_perm(vw[2 * x][b >> 1], vw[2 * x + 1][b >> 1], b & 1 ? 0x7632 : 0x5410);
                            a[0][2 * x] = pair4(v, 0), a[0][2 * x + 1] = pair4(v, 1);
                            a[1][2 * x] = pair4(v, 2), a[1][2 * x + 1] = pair4(v, 3);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int t = 0; t < NT; ++t) Fp16::mma(acc[b][h][t], a[h], wb[t][0], wb[t][1]);
                }
            }
            __syncwarp();
        }
        cp_wait<0>();
        __syncthreads();

        // join the warps
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
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float unit = __uint_as_float(ev[b] << 16);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<float2*>(sums + (warp * R + row) * (DP + 8) + 32 * b + 4 * r + 2 * h) =
                            make_float2(acc[b][h][t][e] * unit, acc[b][h][t][2 + e] * unit);
                }
            }
        __syncthreads();
        const bool whole = blk0 == 0 && blk1 == nb;
        const int64_t slot = whole ? 2 * (int64_t)gridDim.x + (int64_t)grp * items + item : 2 * (int64_t)blockIdx.x + (blk0 == 0);
        const bool direct = whole && !p.partial;
        for (int i = warp; i < rows; i += kWarps) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, wml[w * R + i].x);
            float c[kWarps], sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 ml = wml[w * R + i];
                c[w] = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - top);
                sum += ml.x == -INFINITY ? 0.0f : c[w] * ml.y;
            }
            const int64_t at = row0 + i, seq = at / p.share;
            const int qh = head * p.share + (int)(at % p.share);
            const float norm = direct ? (sum == 0.0f ? 0.0f : 1.0f / sum) : 1.0f;
            for (int d = 2 * lane; d < DP; d += 64) {
                float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w)
                    if (c[w] != 0.0f) {
                        const float2 x = *reinterpret_cast<const float2*>(sums + (w * R + i) * (DP + 8) + d);
                        v.x = fmaf(c[w], x.x, v.x), v.y = fmaf(c[w], x.y, v.y);
                    }
                v.x *= norm, v.y *= norm;
                if (direct) {
                    if (d < g.dim) {
                        const uint32_t o = pack2(v.x, v.y, p.fp16);
                        uint16_t* to = p.out + seq * p.o_seq + qh * p.o_head + d;
                        to[0] = (uint16_t)o, to[1] = (uint16_t)(o >> 16);
                    }
                } else {
                    *reinterpret_cast<float2*>(p.pacc + (slot * R + i) * DP + d) = v;
                }
            }
            if (lane == 0) {
                if (!direct) p.pml[slot * R + i] = make_float2(top, sum);
                else if (p.lse) p.lse[seq * g.heads * p.share + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
            }
        }
        __syncthreads();
        u += blk1 - blk0;
    }
}

// ---------------------------------------------------------------- join
// One CTA a query row: the parts of its items, of its own positions (and of
// the prefix), each a sum with its maximum, joined with their weights.
struct JoinSide {
    const int32_t* pre;  // nullptr: this side has nothing
    const float* pacc;
    const float2* pml;
    int n_grp, rg, rt, R, ctas;
};
struct JoinParams {
    JoinSide side[2];  // own positions, prefix
    int heads, share, dim, dp;
    uint16_t* out;
    int64_t o_seq, o_head;
    float* lse;
    bool fp16, partial;
};

__global__ void __launch_bounds__(128) join_kernel(const JoinParams p) {
    __shared__ float sums[4][256];
    __shared__ float2 wml[4];
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int q_heads = p.heads * p.share;
    const int64_t seq = blockIdx.x / q_heads;
    const int qh = blockIdx.x % q_heads, head = qh / p.share;
    float m = -INFINITY, l = 0.0f, acc[8] = {};
    for (int w = 0; w < 2; ++w) {
        const JoinSide s = p.side[w];
        if (!s.pre) continue;
        // this row in that side's items
        const int64_t row = seq * p.share + qh % p.share, grp = row / s.rg;
        const int in = (int)(row % s.rg), tile = in / s.R, i = in % s.R;
        const int items = p.heads * s.rt, item = head * s.rt + tile;
        const int nb = s.pre[grp + 1] - s.pre[grp];
        if (nb == 0) continue;
        const int64_t units = (int64_t)s.pre[s.n_grp] * items, u0 = (int64_t)s.pre[grp] * items + (int64_t)item * nb;
        const int n = split_ctas(units, s.ctas), c0 = split_owner(units, u0, n), c1 = split_owner(units, u0 + nb - 1, n);
        if (c0 == c1 && !p.partial) continue;
        for (int c = c0 + warp; c <= c1; c += 4) {
            const int64_t slot = c0 == c1 ? 2 * (int64_t)s.ctas + grp * items + item : 2 * (int64_t)c + (c == c0);
            const float2 ml = s.pml[slot * s.R + i];
            if (ml.x == -INFINITY) continue;  // this part saw nothing
            const float top = fmaxf(m, ml.x), a = m == -INFINITY ? 0.0f : exp2_fast(m - top), b = exp2_fast(ml.x - top);
            m = top;
            l = l * a + ml.y * b;
            const float* x = s.pacc + (slot * s.R + i) * p.dp;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k * 32 < p.dp) acc[k] = acc[k] * a + b * x[k * 32 + lane];
        }
        if (c0 == c1) continue;
    }
    // a row that the attention kernel has finished itself
    if (!p.partial) {
        const JoinSide s = p.side[0];
        const int64_t row = seq * p.share + qh % p.share, grp = row / s.rg;
        const int tile = (int)(row % s.rg) / s.R, items = p.heads * s.rt, item = head * s.rt + tile;
        const int nb = s.pre[grp + 1] - s.pre[grp];
        if (nb == 0) return;
        const int64_t units = (int64_t)s.pre[s.n_grp] * items, u0 = (int64_t)s.pre[grp] * items + (int64_t)item * nb;
        const int n = split_ctas(units, s.ctas);
        if (split_owner(units, u0, n) == split_owner(units, u0 + nb - 1, n)) return;
    }
    if (lane == 0) wml[warp] = make_float2(m, l);
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (k * 32 < p.dp) sums[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    float top = -INFINITY, c[4], sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, wml[w].x);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        c[w] = wml[w].x == -INFINITY ? 0.0f : exp2_fast(wml[w].x - top);
        sum += wml[w].x == -INFINITY ? 0.0f : c[w] * wml[w].y;
    }
    const float norm = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int d = threadIdx.x; d < p.dim; d += 128) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (c[w] != 0.0f) v = fmaf(c[w], sums[w][d], v);
        p.out[seq * p.o_seq + qh * p.o_head + d] = (uint16_t)pack2(v * norm, 0.0f, p.fp16);
    }
    if (p.lse && threadIdx.x == 0)
        p.lse[seq * q_heads + qh] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------- host
// One attention kernel launch: tile of rows, CTAs, stages, and its part of
// the workspace. Depends on the handle and the call's sizes alone.
struct Plan {
    int n_grp, rg, nt, rt, ctas, stages, smem;
    int64_t slots;
    size_t pre_bytes, acc_bytes, ml_bytes;
    size_t bytes() const { return pre_bytes + acc_bytes + ml_bytes; }
};

Plan attend_plan(const bnn_kv_cache* c, int n_grp, int rg, bool partial) {
    const KvGeo& g = c->geo;
    Plan s{};
    s.n_grp = n_grp;
    s.rg = rg;
    const int most = g.dp <= 128 ? 4 : 2;  // registers: dp * nt sums over a warp's lanes
    s.nt = rg <= 8 ? 1 : rg <= 16 || most == 2 ? 2 : 4;
    s.rt = (int)cdiv64(rg, 8 * s.nt);
    const int per_sm = g.dp <= 128 && s.nt == 1 ? 3 : 2;
    s.ctas = (c->sms > 0 ? c->sms : 148) * per_sm;
    const int R = 8 * s.nt, row = g.row;
    const int stage = 2 * kSub * row + ((2 * g.ng * kSub * 2 + 127) & ~127);
    const int head = (((n_grp + 1) * 4 + 127) & ~127) + 128 * ((R * 4 + 127) / 128) + kWarps * R * 8 + g.dp / 32 * s.nt * 512;
    const int merge = kWarps * R * (g.dp + 8) * 4;
    const int budget = 224 * 1024 / per_sm - 1024;
    int n = (budget - head) / (kWarps * stage);
    s.stages = n < 2 ? 2 : n > 6 ? 6 : n;
    const int ring = kWarps * s.stages * stage;
    s.smem = head + (ring > merge ? ring : merge);
    s.slots = 2 * (int64_t)s.ctas + (partial ? (int64_t)n_grp * g.heads * s.rt : 0);
    const auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    s.pre_bytes = up((size_t)(n_grp + 1) * 4);
    s.acc_bytes = up((size_t)s.slots * R * g.dp * 4);
    s.ml_bytes = up((size_t)s.slots * R * 8);
    return s;
}

template <int DP, int BITS, int NT>
cudaError_t attend_launch(const AttendParams& p, const Plan& s, cudaStream_t st) {
    attend_kernel<DP, BITS, NT><<<s.ctas, 32 * kWarps, s.smem, st>>>(p);
    return cudaGetLastError();
}
template <int DP, int BITS>
cudaError_t attend_rows(const AttendParams& p, const Plan& s, cudaStream_t st) {
    if (s.nt == 1) return attend_launch<DP, BITS, 1>(p, s, st);
    if (s.nt == 2) return attend_launch<DP, BITS, 2>(p, s, st);
    if constexpr (DP <= 128) return attend_launch<DP, BITS, 4>(p, s, st);
    return cudaErrorInvalidValue;
}
template <int BITS>
cudaError_t attend_dim(const AttendParams& p, const Plan& s, cudaStream_t st) {
    switch (p.g.dp) {
        case 64: return attend_rows<64, BITS>(p, s, st);
        case 128: return attend_rows<128, BITS>(p, s, st);
        case 192: return attend_rows<192, BITS>(p, s, st);
        default: return attend_rows<256, BITS>(p, s, st);
    }
}
cudaError_t attend_one(const AttendParams& p, const Plan& s, cudaStream_t st) {
    return p.g.bits == 8 ? attend_dim<8>(p, s, st) : attend_dim<4>(p, s, st);
}

// the kernels of a cache may use all of an SM's shared memory: set once, when the cache is made
template <int DP, int BITS>
cudaError_t attend_setup_rows() {
    constexpr int all = 226 * 1024;
    cudaError_t e = cudaFuncSetAttribute(attend_kernel<DP, BITS, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, all);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_kernel<DP, BITS, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, all);
    if constexpr (DP <= 128)
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attend_kernel<DP, BITS, 4>, cudaFuncAttributeMaxDynamicSharedMemorySize, all);
    return e;
}
template <int BITS>
cudaError_t attend_setup_dim(int dp) {
    switch (dp) {
        case 64: return attend_setup_rows<64, BITS>();
        case 128: return attend_setup_rows<128, BITS>();
        case 192: return attend_setup_rows<192, BITS>();
        default: return attend_setup_rows<256, BITS>();
    }
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

cudaError_t attend_setup(const KvGeo& g) { return g.bits == 8 ? attend_setup_dim<8>(g.dp) : attend_setup_dim<4>(g.dp); }

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
    if (table_pages < 0 || prefix_pages < 0 || !(scale - scale == 0.0f))
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: negative table width, or a scale that is not finite");
    if ((int64_t)table_pages * g.pt > INT_MAX - 256 || (int64_t)prefix_pages * g.pt > INT_MAX - 256)
        return set_error(BNN_ERR_ARG, "bnn_kv_attend: a table of 2^31 tokens or more");
    if ((int64_t)n_seqs * cdiv64((int64_t)table_pages * g.pt, kBlock) > INT_MAX)
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
    p.share = share;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.partial = prefix;
    JoinParams jp{};
    jp.heads = g.heads, jp.share = share, jp.dim = g.dim, jp.dp = g.dp;
    jp.out = p.out, jp.o_seq = o_seq, jp.o_head = o_head, jp.lse = d_lse;
    jp.fp16 = p.fp16, jp.partial = prefix;
    uint8_t* work = (uint8_t*)d_work;
    for (int side = prefix ? 1 : 0; side >= 0; --side) {
        const Plan s = side ? attend_plan(c, 1, n_seqs * share, true) : attend_plan(c, n_seqs, share, prefix);
        p.n_grp = s.n_grp, p.rg = s.rg, p.rt = s.rt, p.stages = s.stages;
        p.lengths = side ? nullptr : d_lengths;
        p.length = side ? prefix_tokens : 0;
        p.table = side ? d_prefix : d_table;
        p.width = side ? prefix_pages : table_pages;
        p.pre = (int32_t*)work;
        p.pacc = (float*)(work + s.pre_bytes);
        p.pml = (float2*)(work + s.pre_bytes + s.acc_bytes);
        work += s.bytes();
        const cudaError_t e = attend_one(p, s, st);
        if (e != cudaSuccess) return cuda_error("bnn_kv_attend", e);
        jp.side[side] = JoinSide{p.pre, p.pacc, p.pml, s.n_grp, s.rg, s.rt, 8 * s.nt, s.ctas};
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((int64_t)n_seqs * q_heads));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel, (const JoinParams)jp);
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_kv_attend", e);
}
