// q4_linear.cu - the 4-bit linear layer of include/bnn_lowbit.h.
#include <cmath>
#include <mutex>
#include <new>

#include <cuda.h>

#include "lowbit_dev.cuh"

struct bnn_q4_layer {
    int device;
    int type;
    bnn::lowbit::Q4Geo geo;
    void* base;              // one allocation, in this order:
    const uint32_t* codes;   //   q4_words
    const uint2* sz;         //   q4_scales / 2 times: scales and zero points of two rows
    const float* bias;       //   [n_out] or nullptr
    int mt;                  // for up to 8 rows: tiles of 16 outputs a CTA,
    int shares8;             //   CTAs that share K; for 9 to 16
    int shares16;
    bool exact;              // some weight (q - z) * s is outside the type's range
};

namespace bnn {
namespace lowbit {
namespace {

// ---------------------------------------------------------------- layout, once
// Padding: an input behind the last has code = zero point (weight 0), a row
// behind the last has scale 0. *exact is set where a weight (q - z) * s with a
// finite scale would round to an infinity of the type.
template <class A>
__global__ void q4_layout_kernel(Q4Geo g, const uint8_t* codes, const uint16_t* scales, const uint8_t* zeros,
                                 uint32_t* wo, uint16_t* szo, int* exact) {
    constexpr uint32_t magic = A::kMagic & 0xffffu;
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
                if (k < g.K) {
                    q = (codes[row * half + (k >> 1)] >> (4 * (k & 1))) & 15u;
                    const int64_t at = (int64_t)row * g.ng + k / g.group;
                    const float s = A::unpack(scales[at]).x, w = (float)((int)q - (zeros ? zeros[at] & 15 : 8)) * s;
                    if (isinf(A::to_float(A::from_float(w))) && !isinf(s)) *exact = 1;
                } else if (zeros)
                    q = zeros[(int64_t)row * g.ng + min(k / g.group, g.ng - 1)] & 15u;
            }
            v |= q << (4 * (nib & 3) + 16 * (nib >> 2));
        }
        wo[w] = v;
    }
    for (int64_t s = first; s < (int64_t)g.tiles * 16 * g.ng; s += step) {
        const int row = (int)(s / g.ng), grp = (int)(s % g.ng);
        const int64_t at = q4_scale(g, row, grp);
        uint16_t* to = szo + (at >> 1) * 4 + (at & 1);  // a pair of rows: two scales, two zero points
        to[0] = row < g.N ? scales[s] : (uint16_t)0;
        to[2] = (uint16_t)(magic | (row < g.N && zeros ? zeros[s] & 15u : 8u));
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// from the shared memory of CTA `rank` of the cluster
__device__ __forceinline__ float ld_cluster1(uint32_t addr, uint32_t rank) {
    uint32_t from;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(from));
    return v;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t from;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(from));
    return v;
}

struct Q4Params {
    Q4Geo g;
    const uint4* w;
    const uint2* sz;  // [tile][group][r]: scales of rows r and r + 8, then magic + zero point of both
    const float* bias;
    const uint16_t* x;
    int64_t xs;
    uint16_t* y;
    int64_t ys;
    int M;
    int shares;       // of K: CTAs of a cluster that make the same outputs
    int mt;           // tiles of 16 outputs a CTA, up to 8 rows
    int gshift;       // group = 32 << gshift, or -1
    bool exact;       // weights are not to be rounded to the type
    bool vec2, vec4, vec8;  // rows of x start 4-byte, 8-byte, 16-byte aligned
};

// ---------------------------------------------------------------- rows on mma.sync
// Few rows, or (in slices of 16) any number where the weights do not fit the
// type. A CTA makes MT tiles of 16 outputs for 8 * NT rows of x; its
// warps take chunks of U 64-input blocks in turn and their sums are joined in
// shared memory. The weights of the next chunk are on their way while one is
// multiplied: U * MT * 512 bytes a warp. A 16 x 64 block takes 83 instructions
// (and-or, shift and subtract). One row, launches in a row over layers that
// together are larger than the L2: 8192 x 8192 10.0 us (3.5 TB/s; one layer
// again and again 9.8), 4096 x 4096 4.1 us, 512 x 512 1.6 us. Neither the bytes
// nor the instructions (1.6 of 4 a clock in a lone cold launch, ALU 38%) bound
// it: a warp has one chunk on its way, and of 148 SMs 108 have two CTAs, 40 one.
// (q - z) is exact in 16 bits (|q - z| <= 15), so a group's sum of products
// has only the rounding of 32-bit sums, and its scale is applied to that sum.
// X: how x can be read: 2 = 8 bytes at a time, K a multiple of 64; 1 = 8 bytes
// at a time; 0 = value by value.
constexpr int kQ4Warps = 8;

// GM: what a scale covers: 0 = 32 inputs (or another odd multiple of 32), 1 = a
// block of 64, 2 = a chunk of U blocks.
template <int MT, int U, int GM>
struct Q4Chunk {
    uint4 w[U][MT];
    uint2 sz[GM == 0 ? 2 * U : GM == 1 ? U : 1][MT];
};

template <class A, int NT, int MT, int U, int GM, int X>
__global__ void __launch_bounds__(32 * kQ4Warps, 2) q4_rows_kernel(const Q4Params p) {
    extern __shared__ float red[];  // [warp][8 * NT][16 * MT + 1]
    constexpr int PITCH = 16 * MT + 1;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // known to be one number a warp
    const int r = lane >> 2, j = lane & 3;
    const int tile0 = blockIdx.x * MT, m0 = blockIdx.y * 8 * NT, rows = min(8 * NT, p.M - m0);
    const Q4Geo g = p.g;
    grid_launch();
    // Whole chunks first, U blocks at a time, the warps in turn; the blocks
    // that are left over one at a time. A few blocks go one at a time, too.
    const int share = p.shares > 1 ? (int)cluster_rank() : 0;
    // shares of whole chunks, which a scale may cover
    const int64_t chunks = (g.kb + U - 1) / U;
    const int first = (int)(chunks * share / p.shares) * U, blocks = min(g.kb, (int)(chunks * (share + 1) / p.shares) * U) - first;
    const int whole = blocks >= U * warps ? blocks / U : 0;
    int n = whole > warp ? (whole - warp + warps - 1) / warps : 0;
    int kb = warp * U;

    // rows of x behind the last are the first one again: a row has columns of
    // its own in the products, and these are not stored
    const uint16_t* xr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int m = t * 8 + r;
        xr[t] = p.x + (m < rows ? m0 + m : m0) * p.xs + (int64_t)first * 64 + 4 * j;
    }
    const uint4* wr[MT];
    const uint2* sr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int tile = min(tile0 + i, g.tiles - 1);  // a tile behind the last repeats it, unused
        wr[i] = p.w + ((int64_t)tile * g.kb + first) * 32 + lane;
        sr[i] = p.sz + (int64_t)tile * g.ng * 8 + r;
    }
    float acc[MT][NT][4] = {};
    using Chunk = Q4Chunk<MT, U, GM>;
    const auto fetch = [&](Chunk& c, int at, int count) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint4* w = wr[i] + (int64_t)at * 32;
#pragma unroll
            for (int u = 0; u < count; ++u) c.w[u][i] = __ldcs(w + u * 32);
        }
#pragma unroll
        for (int h = 0; h < (GM == 0 ? 2 * count : GM == 1 ? count : 1); ++h) {
            const int b = GM == 0 ? 2 * (first + at) + h : 2 * (first + at + h);  // 32-input block
            int grp = p.gshift >= 0 ? b >> p.gshift : b / (g.group >> 5);
            if (GM == 0) grp = min(grp, g.ng - 1);  // the second half of the last block may be padding alone
#pragma unroll
            for (int i = 0; i < MT; ++i) c.sz[h][i] = __ldg(sr[i] + grp * 8);
        }
    };
    const auto multiply = [&](const Chunk& q, int at, int count) {
        float c[MT][NT][4];
        const uint16_t* xp[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) xp[t] = xr[t] + (int64_t)at * 64;
#pragma unroll
        for (int u = 0; u < count; ++u) {
            uint2 xv[4][NT];
            const int left = g.K - (first + at + u) * 64 - 4 * j;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint16_t* x = xp[t] + u * 64 + e * 16;
                    if (X == 2 || (X == 1 && e * 16 < left)) xv[e][t] = *reinterpret_cast<const uint2*>(x);
                    else xv[e][t] = X == 0 ? load4(x, left - e * 16) : make_uint2(0, 0);
                }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint32_t w[4] = {q.w[u][i].x, q.w[u][i].y, q.w[u][i].z, q.w[u][i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint2 sz = q.sz[GM == 0 ? 2 * u + (e >> 1) : GM == 1 ? u : 0][i];
                    const uint32_t z0 = __byte_perm(sz.y, 0, 0x1010), z1 = __byte_perm(sz.y, 0, 0x3232);
                    uint32_t a[4];
                    A::weights(a, w[e], z0, z1);
                    const bool begins = GM == 0 ? e % 2 == 0 : GM == 1 ? e == 0 : u == 0 && e == 0;
                    const bool last = GM == 0 ? e % 2 == 1 : GM == 1 ? e == 3 : u == count - 1 && e == 3;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (begins) A::mma0(c[i][t], a, xv[e][t].x, xv[e][t].y);
                        else A::mma(c[i][t], a, xv[e][t].x, xv[e][t].y);
                    }
                    if (last) {
                        const float2 s = A::unpack(sz.x);
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            acc[i][t][0] = fmaf(s.x, c[i][t][0], acc[i][t][0]);
                            acc[i][t][1] = fmaf(s.x, c[i][t][1], acc[i][t][1]);
                            acc[i][t][2] = fmaf(s.y, c[i][t][2], acc[i][t][2]);
                            acc[i][t][3] = fmaf(s.y, c[i][t][3], acc[i][t][3]);
                        }
                    }
                }
            }
        }
    };
    {
        Chunk c0, c1;
        const int step = warps * U;
        if (n > 0) fetch(c0, kb, U);  // the weights are nobody's output: they need not wait
        grid_wait();
        while (n > 0) {
            if (n > 1) fetch(c1, kb + step, U);
            multiply(c0, kb, U);
            kb += step;
            if (--n == 0) break;
            if (n > 1) fetch(c0, kb + step, U);
            multiply(c1, kb, U);
            kb += step;
            --n;
        }
        for (kb = whole * U + warp; kb < blocks; kb += warps) {
            fetch(c0, kb, 1);
            multiply(c0, kb, 1);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                red[(warp * 8 * NT + t * 8 + 2 * j + (e & 1)) * PITCH + 16 * i + r + 8 * (e >> 1)] = acc[i][t][e];
    __syncthreads();
    const auto store = [&](int i, float v) {
        const int m = i / (16 * MT), o = i % (16 * MT), n = tile0 * 16 + o;
        if (m >= rows || n >= g.N) return;
        if (p.bias) v += p.bias[n];
        const typename A::T out = A::from_float(v);
        p.y[(m0 + m) * p.ys + n] = *reinterpret_cast<const uint16_t*>(&out);
    };
    const auto sum = [&](int i) {
        float v = 0.0f;
        for (int k = 0; k < warps; ++k) v += red[(k * 8 * NT + i / (16 * MT)) * PITCH + i % (16 * MT)];
        return v;
    };
    if (p.shares == 1) {
        for (int i = threadIdx.x; i < 128 * NT * MT; i += blockDim.x) store(i, sum(i));
    } else {
        // the CTAs of a cluster join their sums, a part of the outputs each, in the order of the shares
        __shared__ float mine[128 * NT * MT];
        for (int i = threadIdx.x; i < 128 * NT * MT; i += blockDim.x) mine[i] = sum(i);
        cluster_sync();
        const int part = (128 * NT * MT + p.shares - 1) / p.shares, end = min(128 * NT * MT, (share + 1) * part);
        for (int i = share * part + threadIdx.x; i < end; i += blockDim.x) {
            float v = 0.0f;
            for (int r = 0; r < p.shares; ++r) v += ld_cluster1(smem_addr(mine + i), r);
            store(i, v);
        }
        cluster_sync();  // nobody leaves while its sums are read
    }
}

// CTAs in clusters of c that run at a time with one on each of a B200's 148 SMs (as its
// occupancy calls say): clusters do not fill every GPC
constexpr int kAtOnce[9] = {0, 148, 148, 135, 132, 130, 132, 105, 120};

// Shares of K (of 16 blocks at least) for tiles of MT: the ones with the
// least estimated time. Two CTAs run on an SM; a warp's chunk costs 1.05 us
// where they do not, 1.3 (MT = 1) or 1.1 (MT = 2) where they do: it waits for
// memory. Blocks too few for a chunk for each warp go one at a time. A join
// costs 1.2 us. One row, 8192 x 1024: 2 shares 4.4 us, 4 shares 3.7; 16384 x
// 2048: 1 share 10.1, 2 shares 7.5; 4096 x 1024: 1 share 3.0, 2 shares 3.2.
double q4_rows_shares(const Q4Geo& g, int mt, int chunk_blocks, int* shares) {
    double best = 1e30;
    for (int c = 1; c <= 8; ++c) {
        if (c > 1 && g.kb < 16 * c) break;
        const int64_t ctas = cdiv64(g.tiles, mt) * c;
        const int blocks = (g.kb + c - 1) / c;
        const double chunk = ctas <= 148 ? 1.05 : mt == 1 ? 1.3 : 1.1;
        const bool alone = chunk_blocks == 1 || blocks < kQ4Warps * chunk_blocks;
        const double rounds = alone ? 0.6 * cdiv64(blocks, kQ4Warps) : chunk * cdiv64(blocks, kQ4Warps * chunk_blocks);
        const double us = 0.8 + (double)cdiv64(ctas, 2 * kAtOnce[c]) * (0.6 + rounds) + (c > 1 ? 1.2 : 0.0);
        if (us < best) best = us, *shares = c;
    }
    return best;
}

template <class A, int NT, int MT, int U, int GM, int X>
cudaError_t q4_launch(const Q4Params& p, cudaStream_t st) {
    const dim3 grid((unsigned)cdiv64(p.g.tiles, MT), (unsigned)cdiv64(p.M, 8 * NT), (unsigned)p.shares);
    const int warps = p.g.kb / p.shares < kQ4Warps ? p.g.kb / p.shares : kQ4Warps;
    return launch_cluster(q4_rows_kernel<A, NT, MT, U, GM, X>, grid, 32 * warps, warps * 8 * NT * (16 * MT + 1) * 4, st, true,
                          p.shares > 1 ? p.shares : 0, p);
}
template <class A, int NT, int MT, int U, int GM>
cudaError_t q4_forms(const Q4Params& p, cudaStream_t st) {
    if (!p.vec4 || p.g.K % 4) return q4_launch<A, NT, MT, U, GM, 0>(p, st);
    return p.g.K % 64 ? q4_launch<A, NT, MT, U, GM, 1>(p, st) : q4_launch<A, NT, MT, U, GM, 2>(p, st);
}
template <class A, int NT, int MT, int U>
cudaError_t q4_rows(const Q4Params& p, cudaStream_t st) {
    if (p.g.group % 64) return q4_forms<A, NT, MT, U, 0>(p, st);
    if (U == 1 || p.g.group % (64 * U)) return q4_forms<A, NT, MT, U, 1>(p, st);
    return q4_forms<A, NT, MT, U, U == 1 ? 1 : 2>(p, st);
}

// ---------------------------------------------------------------- tiles on tcgen05
// More rows. A CTA makes 128 outputs x NTOK rows of x (of K, or of a
// cluster's share of K): D[output][row] in tensor memory. The weights are the
// A operand: eight warps turn codes into (q - z) * s in 16 bits and store them
// into tensor memory as they come from their word (16x256b), so that shared
// memory carries x alone: B, 64 inputs a block, 128-byte swizzle, by TMA, or
// by eight warps where x is not aligned for it. With weights in shared
// memory, too, its 128 bytes a clock would hold an NTOK = 256 tile to two
// thirds of the rate. 2048 rows, 4096 x 4096: 53 us alone (1.30 PFLOP/s), 64
// in a long row of launches under the power cap (1.07; the 16-bit library
// product of that shape 52 then); tensor pipe busy 71% of the time, the rest
// the start and end of 256 CTAs in two rounds. 16 rows, 4096 to 16384: 15.6 us
// (layers in turn, larger than the L2 together), of 128 CTAs on 148 SMs, each a
// chain through tensor memory (2.2 of 4 instructions a clock, ALU 43% in a
// lone cold launch).
// Rounding a weight to 16 bits costs half a step of the type, 2^-8 (bf16; fp16
// 2^-11) of a product at most: the result is off by that much of sum |x w| at
// most, beside its own rounding, and typically, for independent products that
// do not cancel, by no more than its own rounding.
// Codes to tensor memory is a chain of about 800 clocks a stage (arithmetic,
// store, wait, hand over), so two groups of eight warps take the stages in
// turn. One thread's products start 70 to 100 clocks apart, so below NTOK =
// 256 (128 clocks a product) two threads take the stages in turn, with sums
// of their own that are added at the end.
constexpr int kGroups = 2, kWWarps = 8 * kGroups;
constexpr int kAhead = 4;   // 64-input blocks of a group whose codes are on their way
constexpr int kXWarps = 8;  // that load x where TMA cannot: kXWarps / S of them a stage
constexpr int q4_issuers(int ntok) { return ntok == 256 ? 1 : 2; }
constexpr int q4_tile_threads(int ntok) { return 32 * (kWWarps + q4_issuers(ntok) + kXWarps); }
// 64-input blocks a stage: handing one over costs about 300 clocks, more than
// the products of 64 inputs where NTOK is small
constexpr int q4_blocks(int ntok) { return ntok == 256 ? 1 : 2; }
constexpr int q4_stages(int ntok) { return ntok == 256 ? 6 : 4; }
__device__ unsigned int g_q4_wait_timeouts = 0;

struct Q4TileParams {
    Q4Params q;
    bool tma;
};

constexpr int kTileCols = 512;  // of tensor memory: NTOK sums an issuer, 32 a block of weights
// one CTA an SM: two would want the same columns
constexpr int q4_tile_smem(int ntok) {
    const int ring = q4_stages(ntok) * q4_blocks(ntok) * ntok * 128;
    return ring < 116 * 1024 ? 116 * 1024 : ring;
}

// 16 columns of this thread's lane, over the issuers
template <int NTOK, int ISS>
__device__ __forceinline__ void tile_sums(float* v, uint32_t at, int nk) {
    uint32_t r[16];
    t5_ld16(at, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
    if (ISS == 2 && nk > 1) {  // the second one had a stage
        t5_ld16(at + NTOK, r);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] += __uint_as_float(r[i]);
    }
}

template <class A, int NTOK, bool G32>
__global__ void __launch_bounds__(q4_tile_threads(NTOK), 1)
    q4_tiles_kernel(const Q4TileParams tp, const __grid_constant__ CUtensorMap map) {
    constexpr int S = q4_stages(NTOK), KB = q4_blocks(NTOK), BLOCK = NTOK * 128, STAGE = KB * BLOCK;
    constexpr int ISS = q4_issuers(NTOK), WW = kWWarps, XW = WW + ISS;  // warps: weights 0 ..; products WW ..; x XW ..
    constexpr int WCOL = NTOK * ISS;                                     // first column of the weights
    static_assert(WCOL + 32 * KB * S <= kTileCols && S % kGroups == 0 && S % ISS == 0, "stages");
    extern __shared__ __align__(1024) uint8_t ring[];
    __shared__ __align__(8) uint64_t bars[3 * S + 1];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up;
    const Q4Params& p = tp.q;
    const Q4Geo& g = p.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int tile0 = blockIdx.x * 8, m0 = blockIdx.y * NTOK;
    const int share = p.shares > 1 ? (int)cluster_rank() : 0;
    const int kb0 = (int)((int64_t)g.kb * share / p.shares), nkb = (int)((int64_t)g.kb * (share + 1) / p.shares) - kb0;
    const int nk = (nkb + KB - 1) / KB;  // stages; the last one may have fewer blocks
    const uint32_t full_w = smem_addr(bars), full_x = full_w + 8 * S, empty = full_x + 8 * S, done = empty + 8 * S;
    if (warp == WW) t5_alloc(smem_addr(&tmem_s), kTileCols);
    if (tid == 0) {
        for (int s = 0; s < S; ++s) {
            bar_init(full_w + 8 * s, 8);
            bar_init(full_x + 8 * s, tp.tma ? 1 : kXWarps / S);
            bar_init(empty + 8 * s, 1);
        }
        bar_init(done, ISS);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    t5_before();
    __syncthreads();
    t5_after();
    // Only now: a dependent that started before, took tensor memory that this
    // CTA waits for and then waited for this grid would hold up both.
    grid_launch();
    const uint32_t tmem = tmem_s;
    if (warp >= WW) grid_wait();  // the weights need not wait for the kernels before

    if (warp < WW) {
        // 16 outputs a warp: lanes 32 * (warp % 4) + 16 * (warp / 4 % 2) of tensor memory
        const int tile = min(tile0 + 2 * (warp & 3) + (warp >> 2 & 1), g.tiles - 1);
        const uint4* wp = p.w + ((int64_t)tile * g.kb + kb0) * 32 + lane;
        const uint2* sp = p.sz + (int64_t)tile * g.ng * 8 + (lane >> 2);
        const uint32_t to = tmem + WCOL + ((uint32_t)(32 * (warp & 3) + 16 * (warp >> 2 & 1)) << 16);
        const int first = warp >> 3;
        constexpr int AHEAD = kAhead / KB;  // stages
        uint4 w[kAhead];
        uint2 sz[kAhead][G32 ? 2 : 1];
        const auto fetch_block = [&](int slot, int kb) {
            w[slot] = __ldcs(wp + kb * 32);
#pragma unroll
            for (int h = 0; h < (G32 ? 2 : 1); ++h) {
                const int b = 2 * (kb0 + kb) + h;
                int grp = p.gshift >= 0 ? b >> p.gshift : b / (g.group >> 5);
                if (G32) grp = min(grp, g.ng - 1);
                sz[slot][h] = __ldg(sp + grp * 8);
            }
        };
        const auto fetch = [&](int slot, int it) {
#pragma unroll
            for (int k = 0; k < KB; ++k)
                if (it * KB + k < nkb) fetch_block(slot * KB + k, it * KB + k);
        };
        const auto weights = [&](uint32_t* v, int slot) {
            const uint32_t ww[4] = {w[slot].x, w[slot].y, w[slot].z, w[slot].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint2 q = sz[slot][G32 ? e >> 1 : 0];
                const uint32_t s0 = __byte_perm(q.x, 0, 0x1010), s1 = __byte_perm(q.x, 0, 0x3232);
                uint32_t f[4];
                A::weights(f, ww[e], __byte_perm(q.y, 0, 0x1010), __byte_perm(q.y, 0, 0x3232));
                v[4 * e] = A::mul2(f[0], s0), v[4 * e + 1] = A::mul2(f[2], s0);
                v[4 * e + 2] = A::mul2(f[1], s1), v[4 * e + 3] = A::mul2(f[3], s1);
            }
        };
        int it = first, s = first, ph = 1;  // ph: parity of the wait for a free stage; the first round passes
#pragma unroll
        for (int a = 0; a < AHEAD; ++a)
            if (it + a * kGroups < nk) fetch(a, it + a * kGroups);
        while (it < nk) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                if (it >= nk) break;
                uint32_t v[16];
                weights(v, a * KB);
                if (!__all_sync(0xffffffffu, bar_wait(empty + 8 * s, ph, &gave_up))) {
                    it = nk;
                    break;
                }
                t5_after();
                t5_st_16x256b_x4(to + 32 * KB * s, v);
                if (KB == 2 && it * KB + 1 < nkb) {
                    weights(v, a * KB + KB - 1);
                    t5_st_16x256b_x4(to + 32 * KB * s + 32, v);
                }
                if (it + AHEAD * kGroups < nk) fetch(a, it + AHEAD * kGroups);
                t5_wait_st();
                t5_before();
                __syncwarp();
                if (lane == 0) bar_arrive(full_w + 8 * s);
                it += kGroups;
                s += kGroups;
                if (s >= S) s -= S, ph ^= 1;
            }
        }
    } else if (warp < XW) {
        // The whole warp goes through the loop, so that addresses and
        // descriptors stay in uniform registers; one thread issues.
        const bool leader = elect_one();
        constexpr uint32_t idesc = (1u << 4) | (A::kMmaType << 7) | (A::kMmaType << 10) | ((uint32_t)(NTOK >> 3) << 17) | (8u << 24);
        const int issuer = warp - WW;
        const uint32_t d = tmem + NTOK * issuer;
        int s = issuer, ph = 0;
        for (int it = issuer; it < nk; it += ISS) {
            const bool there = bar_wait(full_x + 8 * s, ph, &gave_up) && bar_wait(full_w + 8 * s, ph, &gave_up);
            if (!__all_sync(0xffffffffu, there)) break;
            t5_after();
            if (leader) {
                // K-major, 128-byte swizzle: 8 rows of 128 bytes 1024 bytes apart
                const uint64_t b = (uint64_t)((smem_addr(ring) + s * STAGE) >> 4 & 0x3fffu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
#pragma unroll
                for (int k = 0; k < KB; ++k)
                    if (k == 0 || it * KB + k < nkb)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            t5_mma_ts(d, tmem + WCOL + 32 * (KB * s + k) + 8 * e, b + k * (BLOCK >> 4) + 2 * e, idesc, it >= ISS || k > 0 || e > 0);
                t5_commit(empty + 8 * s);
            }
            __syncwarp();
            s += ISS;
            if (s >= S) s -= S, ph ^= 1;
        }
        if (leader) t5_commit(done);
    } else if (tp.tma) {
        if (warp == XW && lane == 0) {
            int it = 0, s = 0, ph = 1;
            for (; it < nk; ++it) {
                if (!bar_wait(empty + 8 * s, ph, &gave_up)) break;
                const int n = min(KB, nkb - it * KB);
                bar_arrive_tx(full_x + 8 * s, n * BLOCK);
                for (int k = 0; k < n; ++k) tma_2d(smem_addr(ring) + s * STAGE + k * BLOCK, &map, (kb0 + it * KB + k) * 64, m0, full_x + 8 * s);
                if (++s == S) s = 0, ph ^= 1;
            }
            // copies that nothing waits for any more still have to land before the CTA ends
            if (it < nk)
                for (int o = it > S ? it - S : 0; o < it; ++o) {
                    int alone = 0;
                    bar_wait(full_x + 8 * (o % S), (o / S) & 1, &alone);
                }
        }
    } else {
        // 8 values of a row a lane, in words, shifted together where rows
        // start at odd places (2-byte loads: 36.8 us against 26.8 for 1174
        // rows, 6961 to 215), and value by value at the edges. A warp has a
        // stage of its own, so that it never waits for a round of it
        // further ahead than the next: a barrier tells only two rounds apart.
        const int s = (warp - XW) % S, part = (warp - XW) / S;
        constexpr int PARTS = kXWarps / S;
        for (int it = s; it < nk && part < PARTS; it += S) {
            if (!__all_sync(0xffffffffu, bar_wait(empty + 8 * s, (it / S & 1) ^ 1, &gave_up))) break;
            uint8_t* st = ring + s * STAGE;
            const int k0 = (kb0 + it * KB) * 64, values = min(KB, nkb - it * KB) * NTOK * 8;
#pragma unroll 1
            for (int i0 = lane + 32 * 4 * part; i0 < values; i0 += 32 * 4 * PARTS) {
                uint4 v[4];
                const uint16_t* x[4];
                int left[4];  // values of the row from there on
                bool inner = true;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const int i = i0 + 32 * a, m = m0 + (i >> 3) % NTOK, k = k0 + 64 * (i / (NTOK * 8)) + 8 * (i & 7);
                    x[a] = p.x + m * p.xs + k;
                    left[a] = m < p.M ? g.K - k : 0;
                    // the words around eight values at an odd place begin and end within x, too
                    const bool odd = reinterpret_cast<uintptr_t>(x[a]) & 2;
                    inner = inner && left[a] >= 8 && (!odd || ((m > 0 || k > 0) && (m + 1 < p.M || left[a] > 8)));
                }
                const bool all = __all_sync(0xffffffffu, inner);
                if (all && p.vec2) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(x[a]);
                        v[a] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else if (all) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const uint32_t odd = (uint32_t)reinterpret_cast<uintptr_t>(x[a]) >> 1 & 1;
                        const uint32_t* w = reinterpret_cast<const uint32_t*>(x[a] - odd);
                        const uint32_t w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[3 + odd];
                        v[a] = make_uint4(__funnelshift_r(w0, w1, 16 * odd), __funnelshift_r(w1, w2, 16 * odd),
                                          __funnelshift_r(w2, w3, 16 * odd), __funnelshift_r(w3, w4, 16 * odd));
                    }
                } else {
#pragma unroll
                    for (int a = 0; a < 4; ++a) v[a] = load8(x[a], left[a], false);
                }
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const int i = i0 + 32 * a, row = i >> 3, c = i & 7;
                    *reinterpret_cast<uint4*>(st + row * 128 + ((c ^ (row & 7)) << 4)) = v[a];
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) bar_arrive(full_x + 8 * s);
        }
    }
    __syncwarp();

    // results
    bool ok = true;
    if (warp < WW) {
        ok = __all_sync(0xffffffffu, bar_wait(done, 0, &gave_up));
        t5_after();
    }
    const int n = tile0 * 16 + 32 * (warp & 3) + lane;
    const int c0 = 16 * (warp >> 2);  // columns a warp: 16 of every 4 * WW
    constexpr int CSTEP = 4 * WW;
    if (p.shares == 1) {
        if (warp < WW && ok) {
            const float bias = p.bias && n < g.N ? p.bias[n] : 0.0f;
#pragma unroll 1
            for (int c = c0; c < NTOK; c += CSTEP) {
                float v[16];
                tile_sums<NTOK, ISS>(v, tmem + ((uint32_t)(32 * (warp & 3)) << 16) + c, nk);
                if (n < g.N) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (m0 + c + i < p.M) {
                            const typename A::T o = A::from_float(v[i] + bias);
                            p.y[(m0 + c + i) * p.ys + n] = *reinterpret_cast<const uint16_t*>(&o);
                        }
                }
            }
        }
    } else {
        // Each CTA joins NTOK / shares of the rows, in the order of the
        // shares: every one leaves its sums in its ring, and reads its
        // part of the others', 16 bytes at a time.
        float* sums = reinterpret_cast<float*>(ring);  // [row of x][128 outputs]
        if (warp < WW && ok) {
#pragma unroll 1
            for (int c = c0; c < NTOK; c += CSTEP) {
                float v[16];
                tile_sums<NTOK, ISS>(v, tmem + ((uint32_t)(32 * (warp & 3)) << 16) + c, nk);
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[(c + i) * 128 + 32 * (warp & 3) + lane] = v[i];
            }
        }
        cluster_sync();
        const int mine = (NTOK + p.shares - 1) / p.shares;
        for (int i = tid; i < mine * 32; i += q4_tile_threads(NTOK)) {
            const int c = share * mine + (i >> 5), o = 4 * (i & 31), m = m0 + c, out = tile0 * 16 + o;
            if (c >= NTOK || m >= p.M || out >= g.N) continue;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int r = 0; r < p.shares; ++r) {
                const float4 x = ld_cluster(smem_addr(sums + c * 128 + o), r);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (out + k < g.N) {
                    const typename A::T w = A::from_float(e[k] + (p.bias ? p.bias[out + k] : 0.0f));
                    p.y[m * p.ys + out + k] = *reinterpret_cast<const uint16_t*>(&w);
                }
        }
        cluster_sync();  // nobody leaves while its sums are read
    }
    t5_before();
    __syncthreads();
    if (warp == WW) {
        if (gave_up) {  // products may still be running
            int alone = 0;
            bar_wait(done, 0, &alone);
            if (lane == 0) atomicAdd(&g_q4_wait_timeouts, 1u);
        }
        t5_after();
        t5_free(tmem, kTileCols);
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)f;
        cudaGetLastError();
    });
    return fn;
}

template <class A, int NTOK, bool G32>
cudaError_t q4_tiles_launch(const Q4TileParams& p, const CUtensorMap& map, cudaStream_t st) {
    const dim3 grid((unsigned)cdiv64(p.q.g.tiles, 8), (unsigned)cdiv64(p.q.M, NTOK), (unsigned)p.q.shares);
    return launch_cluster(q4_tiles_kernel<A, NTOK, G32>, grid, q4_tile_threads(NTOK), q4_tile_smem(NTOK), st, true, p.q.shares, p, map);
}

// Rows a tile and shares of K: the pair with the least estimated clocks of
// the busiest SM: a 64-input block costs 560 (NTOK = 256), 290 or 220, and more
// where x is loaded by hand; a CTA 4000 to start and end, a joined one
// 1500 more.
void q4_tiles_choose(const Q4Params& p, int* ntok, int* shares) {
    double best = 1e30;
    for (int t = 32; t <= 256; t *= 2) {
        if (t > 32 && t / 2 >= p.M) break;
        const double tiles = (double)(cdiv64(p.g.tiles, 8) * cdiv64(p.M, t));
        const double stage = (t <= 64 ? 220 : t == 128 ? 290 : 560) * (p.vec8 ? 1.0 : p.vec2 ? 1 + t / 128.0 : 1 + t / 100.0);
        for (int c = 1; c <= 8; ++c) {
            if (c > 1 && p.g.kb < 8 * c) break;
            const double clocks = std::ceil(tiles * c / kAtOnce[c]) * ((double)p.g.kb / c * stage + 4000 + (c > 1 ? 1500 : 0));
            if (clocks < best) best = clocks, *ntok = t, *shares = c;
        }
    }
}

template <class A, bool G32>
cudaError_t q4_tiles(const Q4Params& p, cudaStream_t st) {
    Q4TileParams tp{};
    tp.q = p;
    int ntok = 32;
    q4_tiles_choose(p, &ntok, &tp.q.shares);
    CUtensorMap map{};
    EncodeTiledFn fn = p.vec8 ? encode_tiled() : nullptr;
    if (fn) {
        const cuuint64_t dims[2] = {(cuuint64_t)p.g.K, (cuuint64_t)p.M}, strides[1] = {(cuuint64_t)p.xs * 2};
        const cuuint32_t box[2] = {64, (cuuint32_t)ntok}, step[2] = {1, 1};
        tp.tma = p.xs * 2 < (1ll << 40) &&
                 fn(&map, A::kTmaType, 2, (void*)p.x, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    switch (ntok) {
        case 32: return q4_tiles_launch<A, 32, G32>(tp, map, st);
        case 64: return q4_tiles_launch<A, 64, G32>(tp, map, st);
        case 128: return q4_tiles_launch<A, 128, G32>(tp, map, st);
        default: return q4_tiles_launch<A, 256, G32>(tp, map, st);
    }
}
template <class A, bool G32>
cudaError_t q4_tiles_setup() {
    cudaError_t e = cudaFuncSetAttribute(q4_tiles_kernel<A, 32, G32>, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_tile_smem(32));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(q4_tiles_kernel<A, 64, G32>, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_tile_smem(64));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(q4_tiles_kernel<A, 128, G32>, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_tile_smem(128));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(q4_tiles_kernel<A, 256, G32>, cudaFuncAttributeMaxDynamicSharedMemorySize, q4_tile_smem(256));
    return e;
}

template <class A>
cudaError_t q4_run(const Q4Params& p, cudaStream_t st) {
    // Two tiles a CTA share their loads of x, and fewer inputs make a chunk;
    // one gives more CTAs. 8192 x 8192, one row: 9.9 us with two, 12.2 with
    // one; 4096 x 4096: 5.6 and 4.1; 4096 x 6144: 5.8 and 7.2.
    if (p.M <= 8) return p.mt == 2 ? q4_rows<A, 1, 2, 2>(p, st) : q4_rows<A, 1, 1, 4>(p, st);
    // 9 to 16 rows: reading x for every tile of 16 outputs is what costs in the
    // rows' kernel, starting in the tiles' (all 16 rows). 4096 x 4096: 9.0 us against 7.6,
    // 4096 x 16384 18.2 against 15.6, 1024 x 1024 3.0 against 4.3.
    if (p.exact || (p.M <= 16 && (int64_t)p.g.tiles * p.g.kb < 1 << 13)) return q4_rows<A, 2, 2, 1>(p, st);
    return p.g.group % 64 ? q4_tiles<A, true>(p, st) : q4_tiles<A, false>(p, st);
}

int q4_create(bnn_q4_layer* L, const uint8_t* codes, const void* scales, const uint8_t* zeros, const float* bias) {
    const Q4Geo& g = L->geo;
    DeviceScope dev(L->device);
    cudaError_t e = dev.err;
    if (e == cudaSuccess) e = q4_tiles_setup<Bf16, false>();
    if (e == cudaSuccess) e = q4_tiles_setup<Bf16, true>();
    if (e == cudaSuccess) e = q4_tiles_setup<Fp16, false>();
    if (e == cudaSuccess) e = q4_tiles_setup<Fp16, true>();
    if (e != cudaSuccess) return cuda_error("bnn_q4_layer_create", e);
    const auto up = [](int64_t n) { return (size_t)((n + 255) & ~(int64_t)255); };
    const size_t bw = up(q4_words(g) * 4), bs = up(q4_scales(g) * 4), bb = bias ? up((int64_t)g.N * 4) : 0;
    int rc = device_alloc(&L->base, bw + bs + bb, "of a 4-bit layer");
    if (rc) return rc;
    char* at = (char*)L->base;
    L->codes = (const uint32_t*)at;
    L->sz = (const uint2*)(at + bw);
    L->bias = bias ? (const float*)(at + bw + bs) : nullptr;
    // the caller's arrays (host or device memory) in device memory, for the layout kernel
    const int64_t half = ((int64_t)g.K + 1) / 2, ns = (int64_t)g.N * g.ng;
    const size_t rw = up(g.N * half), rs = up(ns * 2), rz = zeros ? up(ns) : 0;
    void* tmp = nullptr;
    if ((rc = device_alloc(&tmp, rw + rs + rz + 256, "of a 4-bit layer's raw arrays"))) return rc;
    uint8_t *dw = (uint8_t*)tmp, *ds = dw + rw, *dz = ds + rs;
    int *flag = (int*)(dz + rz), exact = 0;
    e = cudaMemset(flag, 0, sizeof(int));
    if (e == cudaSuccess) e = cudaMemcpy(dw, codes, g.N * half, cudaMemcpyDefault);
    if (e == cudaSuccess) e = cudaMemcpy(ds, scales, ns * 2, cudaMemcpyDefault);
    if (e == cudaSuccess && zeros) e = cudaMemcpy(dz, zeros, ns, cudaMemcpyDefault);
    if (e == cudaSuccess && bias) e = cudaMemcpy((void*)L->bias, bias, (size_t)g.N * 4, cudaMemcpyDefault);
    if (e == cudaSuccess) {
        const int64_t blocks = cdiv64(q4_words(g), 256);
        const auto kernel = L->type == BNN_BF16 ? q4_layout_kernel<Bf16> : q4_layout_kernel<Fp16>;
        kernel<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256>>>(g, dw, (const uint16_t*)ds, zeros ? dz : nullptr,
                                                                           (uint32_t*)L->codes, (uint16_t*)L->sz, flag);
        e = cudaGetLastError();
    }
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpy(&exact, flag, sizeof(int), cudaMemcpyDeviceToHost);
    L->exact = exact != 0;
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
    int two = 1;
    L->mt = q4_rows_shares(L->geo, 2, 2, &two) < q4_rows_shares(L->geo, 1, 4, &L->shares8) ? 2 : 1;
    if (L->mt == 2) L->shares8 = two;
    q4_rows_shares(L->geo, 2, 1, &L->shares16);
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
    p.sz = L->sz;
    p.bias = L->bias;
    p.x = (const uint16_t*)d_x;
    p.xs = x_stride;
    p.y = (uint16_t*)d_y;
    p.ys = y_stride;
    p.M = rows;
    p.mt = L->mt;
    p.exact = L->exact;
    p.shares = rows <= 8 ? L->shares8 : L->shares16;
    p.vec2 = aligned(d_x, 4) && (rows == 1 || x_stride % 2 == 0);
    p.vec4 = aligned(d_x, 8) && (rows == 1 || x_stride % 4 == 0);
    p.vec8 = aligned(d_x, 16) && (rows == 1 || x_stride % 8 == 0);
    p.gshift = -1;
    for (int i = 0; i < 20; ++i)
        if (g.group == 32 << i) p.gshift = i;
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

BNN_API int bnn_q4_device_error(int device, unsigned int* wait_timeouts) {
    if (!wait_timeouts) return set_error(BNN_ERR_ARG, "NULL argument");
    DeviceScope dev(device);
    if (dev.err != cudaSuccess) return cuda_error("bnn_q4_device_error", dev.err);
    const cudaError_t e = cudaMemcpyFromSymbol(wait_timeouts, g_q4_wait_timeouts, sizeof(unsigned int));
    return e == cudaSuccess ? BNN_OK : cuda_error("bnn_q4_device_error", e);
}
