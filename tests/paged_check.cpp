// CPU check of the paged pool's arithmetic (oh_paged_layout.h): every value of a
// page has a place of its own inside the page's block, every tile of the key axis
// is in one part, every row of every unit is in one piece, every piece and head
// has one block, and nothing goes past its bounds.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../ornithology_amd/csrc/oh_paged_layout.h"

#define CHECK(x)                                                              \
    do {                                                                      \
        if (!(x)) { fprintf(stderr, "%s:%d: %s\n", __FILE__, __LINE__, #x); exit(1); } \
    } while (0)

static unsigned seed = 1;
static int pick(int lo, int hi) {
    seed = seed * 1664525u + 1013904223u;
    return lo + (int)((seed >> 8) % (unsigned)(hi - lo + 1));
}

int main() {
    for (int hd : {64, 128, 256})
        for (int page : {32, 64, 128, 256})
            for (int unit : {8, 16, 0}) {                        // keys of 16 and 8 bits, values
                std::vector<char> used((size_t)page * hd, 0);
                for (int s = 0; s < page; s++)
                    for (int d = 0; d < hd; d++) {
                        const uint32_t at = unit ? pg_k_place(unit, hd, s, d) : pg_v_at(hd, s, d);
                        CHECK(at < used.size() && !used[at]);
                        used[at] = 1;
                    }
            }
    for (int k = 0; k < 20000; k++) {
        const int lo = 32 * pick(0, 300), hi = lo + pick(-40, 9000), least = pick(1, 600), most = pick(1, 256);
        const int parts = pg_parts(hi - lo, least, most);
        CHECK(parts >= 1 && parts <= most);
        int at = lo >> 5;
        for (int c = 0; c < parts; c++) {
            int t0, t1;
            pg_part(lo, hi, c, parts, &t0, &t1);
            CHECK(t0 == at && t1 >= t0);
            at = t1;
        }
        CHECK(at == (hi > lo ? (hi + 31) >> 5 : lo >> 5));
    }
    for (int k = 0; k < 3000; k++) {
        const int G = pick(1, 16), units = pick(1, 20), tr = pick(0, 1) ? 128 : 256, nkv = pick(1, 17), parts = pick(1, 5);
        std::vector<int64_t> f0(units), n(units);
        int64_t row = 0;
        for (int i = 0; i < units; i++) {
            f0[i] = row * G;
            const int r = pick(0, 3) ? pick(0, 3) : pick(0, 700);
            n[i] = (int64_t)r * G;
            row += r;
        }
        row += pick(0, 5);                                       // rows behind the last unit
        if (!row) continue;
        const int64_t pieces = pg_piece_count(row * G, units, tr), blocks = pg_blocks(pieces, nkv);
        std::vector<int> rows((size_t)(row * G), 0);
        for (int64_t x = 0; x < pieces; x++) {
            int u = -1;
            for (int i = 0; i < units && pg_first_piece(i, f0[i], tr) <= x; i++) u = i;
            if (u < 0) u = 0;
            int64_t from, to;
            if (!pg_piece_rows(x, u, f0[u], n[u], tr, &from, &to)) continue;
            CHECK(from >= f0[u] && to <= f0[u] + n[u] && to - from <= tr);
            for (int64_t r = from; r < to; r++) rows[(size_t)r]++;
        }
        for (int i = 0; i < units; i++)
            for (int64_t r = f0[i]; r < f0[i] + n[i]; r++) CHECK(rows[(size_t)r] == 1);
        for (int c = 0; c < parts; c++) {
            std::vector<int> seen((size_t)pieces * nkv, 0);
            for (int64_t x = 0; x < blocks; x++) {
                int h;
                int64_t p;
                pg_block_of(x, c, pieces, nkv, &h, &p);
                if (h >= nkv) continue;
                CHECK(h >= 0 && p >= 0 && p < pieces);
                seen[(size_t)(p * nkv + h)]++;
            }
            for (int s : seen) CHECK(s == 1);
        }
    }
    puts("ok");
    return 0;
}
