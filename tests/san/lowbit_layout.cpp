// Host-only walk over the index arithmetic that the low-bit kernels share
// (bnns_to_c_b200/csrc/lowbit.h). Test infrastructure:
// tests/test_lowbit_cpu.py compiles it with -fsanitize=address,undefined.
// Every place of a layout has to be inside its buffer and be taken exactly
// once; page tables and offsets of any content must give places inside the
// cache or none; the attention's split has to cover every block once.
// Prints one line per part; exits 1 at the first thing that is wrong.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../bnns_to_c_b200/csrc/lowbit.h"

using namespace bnn::lowbit;

#define CHECK(x)                                                   \
    do {                                                           \
        if (!(x)) {                                                \
            printf("line %d: %s\n", __LINE__, #x);                 \
            exit(1);                                               \
        }                                                          \
    } while (0)

static void linear(int K, int N, int group) {
    const Q4Geo g = q4_geo(K, N, group);
    std::vector<int> seen((size_t)g.tiles * 16 * g.kb * 64);
    for (int t = 0; t < g.tiles; ++t)
        for (int kb = 0; kb < g.kb; ++kb)
            for (int lane = 0; lane < 32; ++lane) {
                CHECK(q4_word(g, t, kb, lane) >= 0 && q4_word(g, t, kb, lane) + 4 <= q4_words(g));
                for (int i = 0; i < 4; ++i)
                    for (int nib = 0; nib < 8; ++nib) {
                        const int row = t * 16 + q4_row(lane, nib), k = kb * 64 + q4_in(lane, i, nib);
                        seen.at((size_t)row * g.kb * 64 + k)++;
                    }
            }
    for (int v : seen) CHECK(v == 1);
    std::vector<int> sc((size_t)q4_scales(g));
    for (int row = 0; row < g.tiles * 16; ++row)
        for (int grp = 0; grp < g.ng; ++grp) sc.at((size_t)q4_scale(g, row, grp))++;
    for (int v : sc) CHECK(v == 1);
}

static void cache(int pages, int pt, int heads, int dim, int bits, int group) {
    const KvGeo g = kv_geo(pages, pt, heads, dim, bits, group);
    CHECK(g.dp >= dim && g.dp % 64 == 0 && g.row * 8 == g.dp * bits && (1 << g.sh) == pt && g.ng * group >= dim);
    // a row: 8 numbers of a key, 4 of a value
    std::vector<int> k(g.row), v(g.row);
    for (int i = 0; i < g.dp / 8; ++i)
        for (int b = 0; b < bits; ++b) k.at(kv_k_at(g, i) + b)++;
    for (int i = 0; i < g.dp / 4; ++i)
        for (int b = 0; b < bits / 2; ++b) v.at(kv_v_at(g, i) + b)++;
    for (int b = 0; b < g.row; ++b) CHECK(k[b] == 1 && v[b] == 1);
    for (int i = 0; i < g.dp / 8; ++i) CHECK(kv_k_at(g, i) % bits == 0);
    for (int i = 0; i < g.dp / 4; ++i) CHECK(kv_v_at(g, i) % (bits / 2) == 0);
    std::vector<char> rows((size_t)kv_code_bytes(g)), sc((size_t)kv_scales(g));
    for (int p = 0; p < pages; ++p)
        for (int h = 0; h < heads; ++h)
            for (int t = 0; t < pt; ++t) {
                CHECK(kv_row(g, p, h, t) % g.row == 0);
                rows.at(kv_row(g, p, h, t))++;
                rows.at(kv_row(g, p, h, t) + g.row - 1)++;
                for (int q = 0; q < g.ng; ++q) sc.at(kv_scale(g, p, h, q, t))++;
                // the attention copies 16 tokens' rows and scales from here as 16-byte pieces
                if (t % 16 == 0) {
                    CHECK(kv_row(g, p, h, t) % 16 == 0 && kv_row(g, p, h, t) + 16 * g.row <= kv_code_bytes(g));
                    CHECK(kv_scale(g, p, h, 0, t) % 8 == 0 && kv_scale(g, p, h, 0, t) + 16 * g.ngp <= kv_scales(g));
                }
            }
    for (size_t i = 0; i < rows.size(); i += g.row) CHECK(rows[i] == 1 && rows[i + g.row - 1] == 1);
    // every scale has a place of its own; places behind a token's last group stay empty
    for (size_t i = 0; i < sc.size(); ++i) CHECK(sc[i] == ((int)(i % g.ngp) < g.ng));
}

static void pages() {
    std::mt19937 rng(1);
    const KvGeo g = kv_geo(7, 32, 2, 64, 8, 64);
    for (int n = 0; n < 20000; ++n) {
        const int width = (int)(rng() % 5);
        std::vector<int32_t> table(width);  // exactly sized: a read past it is a report
        for (auto& x : table) x = rng() % 3 ? (int)(rng() % 7) : (int)rng();
        const int p = rng() % 4 ? (int)(rng() % 200) : (int)rng();
        const int page = kv_page(g, table.data(), width, p);
        CHECK(page >= -1 && page < 7);
        if (p >= 0 && p / 32 < width && table[p / 32] >= 0 && table[p / 32] < 7) CHECK(page == table[p / 32]);
        else CHECK(page == -1);
    }
    for (int n = 0; n < 20000; ++n) {
        const int seqs = 1 + (int)(rng() % (n % 10 ? 9 : 3000));
        std::vector<int32_t> off(seqs + 1);
        const bool wild = rng() % 4 == 0;  // not ascending: any answer, but one inside
        int at = (int)(rng() % 5);
        for (auto& x : off) x = wild ? (int)rng() : (at += (int)(rng() % 4) * (rng() % 2));
        const int t = wild ? (int)rng() : (int)(rng() % (10 + 2 * seqs));
        const int b = kv_seq(off.data(), seqs, t, [&](int lo, int step, int len) {
            int k = 0;
            for (int l = 0; l < 32; ++l) k += l * step < len && off.at(lo + l * step) <= t;
            return k;
        });
        CHECK(b >= -1 && b < seqs);
        if (!wild) {
            if (b < 0) CHECK(t < off[0] || t >= off[seqs]);
            else CHECK(off[b] <= t && t < off[b + 1]);
        }
    }
}

static void split() {
    std::mt19937 rng(2);
    for (int n = 0; n < 3000; ++n) {
        const uint32_t units = 1 + rng() % 3000;
        const int ctas = split_ctas(units, 1 + (int)(rng() % 500));
        CHECK(ctas >= 1 && (uint32_t)ctas <= units);
        for (int c = 0; c < ctas; ++c) CHECK(split_begin(units, c, ctas) < split_begin(units, c + 1, ctas));
        for (int c = 0; c < ctas; ++c)
            for (uint32_t u = split_begin(units, c, ctas); u < split_begin(units, c + 1, ctas); ++u) CHECK(split_owner(units, u, ctas) == c);
        CHECK(split_begin(units, 0, ctas) == 0 && split_begin(units, ctas, ctas) == units);
    }
    const uint32_t many = 0x7fffffff;  // the most that a call takes
    CHECK(split_owner(many, many - 1, 592) == 591 && split_begin(many, 592, 592) == many && split_owner(many, 0, 592) == 0);
}

int main() {
    for (int K : {1, 31, 32, 63, 64, 65, 130, 512})
        for (int N : {1, 15, 16, 17, 100}) linear(K, N, 32), linear(K, N, 96), linear(K, N, 128);
    printf("linear\n");
    for (int dim : {8, 64, 72, 80, 128, 136, 192, 200, 256})
        for (int bits : {4, 8})
            for (int group : {32, 64, 128, dim}) cache(3, 16, 2, dim, bits, group), cache(2, 64, 3, dim, bits, group);
    printf("cache\n");
    pages();
    printf("pages\n");
    split();
    printf("split\n");
    return 0;
}
