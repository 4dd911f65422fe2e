// oh_paged_layout.h - where things are in a paged pool, and how the key axis is
// cut: plain arithmetic, for the kernels and for the host's own check of it.
#pragma once
#include <stdint.h>
#ifdef __HIPCC__
#define OH_PG __host__ __device__ __forceinline__
#else
#define OH_PG inline
#endif

// element offsets in a (page, head) block's key and value parts of position
// `slot` of the page, dim d (units of u elements: 8 of 16 bits, 16 codes)
OH_PG uint32_t pg_k_place(int u, int hd, int slot, int d) {
    return (uint32_t)((slot >> 5) * 32 * hd + ((d / u) * 32 + (slot & 31)) * u + d % u);
}
OH_PG uint32_t pg_v_at(int hd, int slot, int d) {
    const int s = slot & 31;
    return (uint32_t)((slot >> 5) * 32 * hd + (((s >> 2) & 3) * hd + d) * 8 + 4 * (s >> 4) + (s & 3));
}

// parts of a stretch of n positions, each of at least `least` and at most `most` of them
OH_PG int pg_parts(int n, int least, int most) {
    const int p = (n + least - 1) / least;
    return p < 1 ? 1 : p < most ? p : most;
}
// the 32-position tiles [t0, t1) of part c of the positions [lo, hi), lo a multiple of 32
OH_PG void pg_part(int lo, int hi, int c, int parts, int *t0, int *t1) {
    const int T0 = lo >> 5, T = hi > lo ? ((hi + 31) >> 5) - T0 : 0;
    *t0 = T0 + (int)((int64_t)T * c / parts);
    *t1 = T0 + (int)((int64_t)T * (c + 1) / parts);
}

// Rows (times heads) are cut at multiples of tr and where units begin: the first
// piece of unit i, whose rows begin at f0, and the rows [from, to) of piece x if it
// is one of the unit's, which has n
OH_PG int64_t pg_first_piece(int i, int64_t f0, int tr) { return i + f0 / tr; }
OH_PG bool pg_piece_rows(int64_t x, int i, int64_t f0, int64_t n, int tr, int64_t *from, int64_t *to) {
    const int64_t skip = x - pg_first_piece(i, f0, tr);          // cuts behind the unit's first row
    if (skip < 0) return false;
    *from = skip > 0 ? (f0 / tr + skip) * tr : f0;
    *to = (f0 / tr + skip + 1) * tr;
    if (*to > f0 + n) *to = f0 + n;
    return *from < *to;
}
OH_PG int64_t pg_piece_count(int64_t rows, int units, int tr) { return (rows - 1) / tr + units; }

// A piece's block: blocks go to eight XCDs in turn, and the pieces of head h to
// those of them that have h's residue of g8 (a power of two up to 8 that
// divides the heads); parts begin at another of these
OH_PG int pg_heads_apart(int nkv) { return nkv % 8 == 0 ? 8 : nkv % 4 == 0 ? 4 : nkv % 2 == 0 ? 2 : 1; }
OH_PG int64_t pg_blocks(int64_t pieces, int nkv) {
    const int g8 = pg_heads_apart(nkv);
    return 8 * ((pieces * (nkv / g8) + 8 / g8 - 1) / (8 / g8));
}
// the head (past the last one: none) and the piece, counted from the last, of block x of part c
OH_PG void pg_block_of(int64_t x, int c, int64_t pieces, int nkv, int *head, int64_t *piece) {
    const int g8 = pg_heads_apart(nkv), xcd = (int)((x + (int64_t)g8 * c) % 8);
    const int64_t mine = x / 8 * (8 / g8) + xcd / g8;
    *head = (int)(mine / pieces) * g8 + xcd % g8;
    *piece = pieces - 1 - mine % pieces;
}
