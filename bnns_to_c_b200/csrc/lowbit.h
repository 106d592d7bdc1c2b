// lowbit.h - shared by the 4-bit linear layer (q4_linear.cu) and the
// key/value cache (kv_cache.cu): the layouts that their kernels agree on, as
// plain functions that a host compiler takes too (tests/san/lowbit_layout.cpp
// walks them), and small host helpers.
#pragma once
#include <cstddef>
#include <cstdint>

#ifdef __CUDACC__
#define LB_HD __host__ __device__ __forceinline__
#else
#define LB_HD inline
#endif

namespace bnn {
namespace lowbit {

// ---------------------------------------------------------------- 4-bit linear layer
// A tile is 16 output rows x 64 inputs, 512 bytes: lane (r = lane / 4,
// j = lane % 4) of a warp owns 16 of them, word i of its four being the part
// that it has of a 16 x 16 operand of the tensor cores: rows r and r + 8,
// inputs 16 * i + 4 * j + 0..3. That is the A fragment of an m16n8k16
// mma.sync (whose inputs may come in any order that x follows), and of
// tcgen05.st.16x256b, which puts the 16 rows into tensor memory with the
// inputs in their own order.
// Word: nibble p (bits 4p and 16 + 4p) holds the pair of inputs 2 * (p / 2)
// + {0, 1} of row r + 8 * (p % 2), so (word >> 4p) & 0x000f000f is register
// a_p of the fragment, two codes at the bottom of two 16-bit halves.
struct Q4Geo {
    int K, N, group, ng;  // inputs, outputs, inputs a scale, scales a row
    int tiles, kb;        // 16-row tiles, 64-input blocks
};
LB_HD Q4Geo q4_geo(int K, int N, int group) {
    Q4Geo g;
    g.K = K;
    g.N = N;
    g.group = group;
    g.ng = (int)(((int64_t)K + group - 1) / group);
    g.tiles = (int)(((int64_t)N + 15) / 16);
    g.kb = (int)(((int64_t)K + 63) / 64);
    return g;
}
LB_HD int64_t q4_words(const Q4Geo& g) { return (int64_t)g.tiles * g.kb * 128; }
LB_HD int64_t q4_word(const Q4Geo& g, int tile, int kb, int lane) { return (((int64_t)tile * g.kb + kb) * 32 + lane) * 4; }
// row and input of nibble `nib` (0..7) of word i of a lane, within the tile
LB_HD int q4_row(int lane, int nib) { return (lane >> 2) + 8 * (nib & 1); }
LB_HD int q4_in(int lane, int i, int nib) { return 16 * i + 4 * (lane & 3) + 2 * ((nib >> 1) & 1) + (nib >> 2); }
// place of a scale: [tile][group][r][row r, row r + 8]
LB_HD int64_t q4_scale(const Q4Geo& g, int row, int grp) {
    return (((int64_t)(row >> 4) * g.ng + grp) * 8 + (row & 7)) * 2 + ((row >> 3) & 1);
}
LB_HD int64_t q4_scales(const Q4Geo& g) { return (int64_t)g.tiles * g.ng * 16; }

// ---------------------------------------------------------------- key/value cache
// Codes: [page][kv head][token][row bytes], keys and values apart; scales
// (bf16): [page][kv head][token][ngp], a token's groups side by side, their
// number rounded up to a power of two. A row holds dp >= head_dim numbers (head_dim
// rounded up to 64, 128, 192 or 256; code 0 in the padding) in the order in
// which the attention's lanes take them: of each 32 numbers, lane quarter
// j = 0..3 takes 8 neighbouring keys, and lane eighth r = 0..7 takes 4
// neighbouring values; a lane's numbers of all the 32-blocks lie together.
// Codes are stored as code + 128 (a byte) or code + 8 (a nibble).
struct KvGeo {
    int pages, pt, heads, dim, dp, bits, group, ng, ngp;
    int row;  // bytes of a row of codes
    int sh;   // pt = 1 << sh
};
LB_HD KvGeo kv_geo(int pages, int pt, int heads, int dim, int bits, int group) {
    KvGeo g;
    g.pages = pages;
    g.pt = pt;
    g.heads = heads;
    g.dim = dim;
    g.dp = (dim + 63) / 64 * 64;
    g.bits = bits;
    g.group = group;
    g.ng = (dim + group - 1) / group;
    g.ngp = g.ng <= 1 ? 1 : g.ng <= 2 ? 2 : g.ng <= 4 ? 4 : 8;
    g.row = g.dp * bits / 8;
    g.sh = 0;
    while ((1 << g.sh) < pt) ++g.sh;
    return g;
}
LB_HD int64_t kv_code_bytes(const KvGeo& g) { return (int64_t)g.pages * g.heads * g.pt * g.row; }
LB_HD int64_t kv_scales(const KvGeo& g) { return (int64_t)g.pages * g.heads * g.pt * g.ngp; }
LB_HD int64_t kv_row(const KvGeo& g, int page, int head, int tok) { return (((int64_t)page * g.heads + head) * g.pt + tok) * g.row; }
LB_HD int64_t kv_scale(const KvGeo& g, int page, int head, int grp, int tok) {
    return (((int64_t)page * g.heads + head) * g.pt + tok) * g.ngp + grp;
}
// byte of the row where the 8 numbers 8 * i .. 8 * i + 7 of a key lie
// (8 bytes, or 4 with 4 bits: number c in nibble c / 2 + 4 * (c % 2))
LB_HD int kv_k_at(const KvGeo& g, int i) { return ((i & 3) * (g.dp / 32) + (i >> 2)) * g.bits; }
// byte of the row where the 4 numbers 4 * i .. 4 * i + 3 of a value lie
// (4 bytes, or 2 with 4 bits: number c in nibble c)
LB_HD int kv_v_at(const KvGeo& g, int i) { return ((i & 7) * (g.dp / 32) + (i >> 3)) * (g.bits / 2); }
// the page of position p in a row of `width` table entries; -1: none
LB_HD int kv_page(const KvGeo& g, const int32_t* table, int width, int p) {
    if (p < 0) return -1;
    const int at = p >> g.sh;
    if (at >= width) return -1;
    const int page = table[at];
    return page >= 0 && page < g.pages ? page : -1;
}
// sequence of row t: the last b in [0, n) with off[b] <= t; -1 where t is
// before the first or behind the last. 32 places are looked at together:
// below(lo, step, len) counts the l in 0 .. 31 with l * step < len and
// off[lo + l * step] <= t. Offsets that do not ascend give some b in [0, n).
template <class F>
LB_HD int kv_seq(const int32_t* off, int n, int t, F&& below) {
    if (t < off[0] || t >= off[n]) return -1;
    int lo = 0, len = n;
    while (len > 1) {
        const int step = (len + 31) / 32, k = below(lo, step, len);
        const int skip = (k > 0 ? k - 1 : 0) * step;
        lo += skip;
        len = len - skip < step ? len - skip : step;
    }
    return lo;
}

// ---------------------------------------------------------------- attention's split
// All the work is one line of blocks of tokens: sequence by sequence, within
// it item by item (kv head, tile of query rows), within that block by block;
// n CTAs take equal shares of it, the first ones a block more. So every CTA
// has the same work whatever the lengths, and an item is cut only where a
// share ends. A cut costs a CTA about what 256 tokens do, so blocks have as
// many, unless the shares are so long that 64 balance them better. They have
// as many, too, where no sequence is longer: then no item is cut.
constexpr int kBlock = 64, kLong = 256;
LB_HD bool split_long(int64_t blocks, int ctas) { return blocks < (int64_t)ctas * (2 * kLong / kBlock); }
// CTAs with a share: no more than blocks, so that none of them is empty
LB_HD int split_ctas(uint32_t units, int ctas) { return units < (uint32_t)ctas ? (int)units : ctas; }
LB_HD uint32_t split_begin(uint32_t units, int cta, int n) {
    const uint32_t q = units / (uint32_t)n, r = units % (uint32_t)n;
    return cta * q + ((uint32_t)cta < r ? (uint32_t)cta : r);
}
// the CTA that has block u (0 <= u < units)
LB_HD int split_owner(uint32_t units, uint32_t u, int n) {
    const uint32_t q = units / (uint32_t)n, r = units % (uint32_t)n, more = r * (q + 1);
    return (int)(u < more ? u / (q + 1) : r + (u - more) / q);
}

}  // namespace lowbit
}  // namespace bnn
