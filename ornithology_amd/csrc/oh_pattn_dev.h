// oh_pattn_dev.h - what the attention kernels over a paged pool share: the
// batch's bounds, the parts of the key axis, operand conversion.
//
// o = sum_{t < lim} softmax_t(q . k_t * scale) v_t per row and head, lim the
// row's position + 1. Scores are taken in units of log2(e), so that the
// softmax is 2^(s - m). Products run on the matrix cores with 32-bit
// accumulators; f32 rows enter as sums of 16-bit terms, whose products with the
// codes are exact, and their weights as three bf16 terms (24 bits).
#pragma once
#include "oh_paged_dev.h"

#include <atomic>

// Operand vectors of the matrix instructions. Of the values: fp16 for fp16
// pools, else bf16, which has f32's range, so that a weight p * scale cannot
// leave it; codes are exact in either. Of the keys the same, but fp16 over
// codes for f32 and fp16 rows: two fp16 terms hold 22 bits of a query (scaled so
// that its largest dim is 2^14 or more, every dim above 2^-17 of that one
// does), one an fp16 query whole.
template <bool H> struct pg_vec { typedef pg_b8 v; typedef __bf16 e; };
template <> struct pg_vec<true> { typedef pg_h8 v; typedef _Float16 e; };
template <int RT, int CT> struct pg_ops {
    static constexpr bool Q8 = CT == OH_PT_Q8, KH = CT == OH_PT_F16 || (Q8 && RT != OH_PT_BF16), VH = CT == OH_PT_F16;
    typedef typename pg_vec<KH>::v kv;
    typedef typename pg_vec<VH>::v vv;
    typedef typename pg_vec<VH>::e ve;
    static constexpr int NQ = RT == OH_PT_F32 ? 2 : 1;
};

OH_DEV pg_f4 pg_mma16(pg_b8 a, pg_b8 b, pg_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
OH_DEV pg_f4 pg_mma16(pg_h8 a, pg_h8 b, pg_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
OH_DEV pg_f16 pg_mma32(pg_b8 a, pg_b8 b, pg_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
OH_DEV pg_f16 pg_mma32(pg_h8 a, pg_h8 b, pg_f16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// N terms of 8 values, each the rounding of what the ones before left
template <int N, class V>
OH_DEV void pg_split(const float (&x)[8], V (&out)[N]) {
    float r[8];
#pragma unroll
    for (int j = 0; j < 8; j++) r[j] = x[j];
#pragma unroll
    for (int t = 0; t < N; t++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            out[t][j] = (decltype(out[t][j] + out[t][j]))r[j];
            if (t + 1 < N) r[j] -= (float)out[t][j];
        }
}
// 8 codes as operand values
OH_DEV void pg_codes(uint32_t lo, uint32_t hi, pg_b8 *o) {
#pragma unroll
    for (int j = 0; j < 8; j++) (*o)[j] = (__bf16)(float)(int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
}
// (fp16: code + 128 under the exponent of 1024 is 1152 + code)
OH_DEV void pg_codes(uint32_t lo, uint32_t hi, pg_h8 *o) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - off,
             b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - off,
             c = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - off,
             d = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - off;
    *o = (pg_h8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The power of two by which a row whose largest |value| is `top` is multiplied
// before it is split into fp16 terms: top becomes 2^14 or more, below 2^15
OH_DEV int pg_row_exp(float top) { return top > 0.0f && top < INFINITY ? 14 - max(ilogbf(top), -100) : 0; }

// Values that are hidden from some row of a tile may be infinite or NaN
// (another request's leavings behind the end, a prompt's later tokens), and a
// weight of 0 times that is NaN: such tiles' values enter the products with 0
// in those places, and where there was one (`odd`), it is added afterwards to
// the rows that see it.
template <bool H>
OH_DEV void pg_only_finite(uint4 *w, bool *odd) {
    typedef unsigned short u2 __attribute__((ext_vector_type(2)));
    constexpr uint32_t E = H ? 0x7c007c00u : 0x7f807f80u;                  // exponents of all ones
    const u2 one = {1, 1}, zero = {0, 0};
    uint32_t *x = (uint32_t *)w, all = ~0u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u2 rest = __builtin_bit_cast(u2, (x[i] & E) ^ E);
        const uint32_t keep = __builtin_bit_cast(uint32_t, zero - __builtin_elementwise_min(rest, one));
        x[i] &= keep;
        all &= keep;
    }
    *odd |= all != ~0u;
}

// ---- the batch ------------------------------------------------------------------
// sequence s's rows and length, false (and reported) if they are not in range
OH_DEV bool pg_seq(const oh_pattn &a, int s, int *row, int *n, int *len) {
    const int r0 = a.b.start[s], r1 = a.b.start[s + 1], l = a.b.len[s];
    if (r0 < 0 || r1 < r0 || r1 > a.b.n_rows || r1 - r0 > a.b.max_new || l < 0 ||
        l > (int64_t)a.b.max_pages << a.pool.page_sh) {
        pg_report(a.pool, OH_PF_BATCH);
        return false;
    }
    *row = r0; *n = r1 - r0; *len = l;
    return true;
}
// positions of group i that its sequences share: whole pages within glen
OH_DEV int pg_shared(const oh_pattn &a, int i) {
    const int64_t most = (int64_t)a.b.max_pages << a.pool.page_sh;
    const int l = a.glen[i];
    if (l < 0 || l > most) { pg_report(a.pool, OH_PF_BATCH); return 0; }
    return (l >> a.pool.page_sh) << a.pool.page_sh;
}
// the positions that sequence s (of this lane) leaves to its group's prefix
OH_DEV int pg_prefix_of(const oh_pattn &a, int s) {
    int lo = 0, hi = a.n_group;
    if (!hi) return 0;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.gfirst[mid] <= s) lo = mid; else hi = mid;
    }
    const int f0 = a.gfirst[lo], f1 = a.gfirst[lo + 1];
    return s >= f0 && s < f1 && f0 >= 0 && f1 <= a.b.n_seq ? pg_shared(a, lo) : 0;
}
// Positions below this are visible to row `token` of the sequence whose rows end
// before `end`
OH_DEV int pg_lim(int len, int end, int token) { const int p = len - (end - token) + 1; return p > 0 ? p : 0; }

// A unit of work: the rows [row, row + n) of one sequence over its positions
// [lo, hi), or those of a group's sequences over the prefix they share
struct pg_unit { int row, n, lo, hi; const int32_t *pages; };

template <bool PREFIX>
OH_DEV bool pg_unit_at(const oh_pattn &a, int u, pg_unit *o) {
    if (PREFIX) {
        const int f0 = a.gfirst[u], f1 = a.gfirst[u + 1];
        int r0 = -1, r1 = -1;
        if (f0 >= 0 && f1 >= f0 && f1 <= a.b.n_seq) { r0 = a.b.start[f0]; r1 = a.b.start[f1]; }
        if (r0 < 0 || r1 < r0 || r1 > a.b.n_rows) { pg_report(a.pool, OH_PF_BATCH); return false; }
        o->row = r0; o->n = r1 - r0; o->lo = 0;
        o->hi = pg_shared(a, u);
        o->pages = a.b.table + (size_t)(f0 < a.b.n_seq ? f0 : 0) * a.b.max_pages;
        return true;
    }
    if (!pg_seq(a, u, &o->row, &o->n, &o->hi)) return false;
    o->lo = pg_prefix_of(a, u);
    o->pages = a.b.table + (size_t)u * a.b.max_pages;
    return true;
}
// what row `token` of a unit sees, as pg_lim
template <bool PREFIX>
OH_DEV int pg_unit_lim(const oh_pattn &a, const pg_unit &u, int token) {
    if (!PREFIX) return pg_lim(u.hi, u.row + u.n, token);
    const int s = pg_seq_of(a.pool, a.b, token);
    int row, n, len;
    if (s < 0 || !pg_seq(a, s, &row, &n, &len)) return 0;
    const int lim = pg_lim(len, row + n, token);
    return lim < u.hi ? lim : u.hi;
}

// A page list in a wave's registers, 64 entries at a time: an entry is a lane of
// one, where a load of its own would put a round trip to memory before every
// tile's loads
struct pg_list {
    const int32_t *pages;
    int n, first, mine;                                // entries, the first held one, this lane's
    OH_DEV void hold(int i) {
        first = i;
        const int at = i + (int)(threadIdx.x & 63);
        mine = at < n ? pages[at] : -1;
    }
    OH_DEV int get(int i) {                            // i: the same in the whole wave, never falling
        if (i - first >= 64) hold(i);
        return __builtin_amdgcn_readlane(mine, i - first);
    }
};

// where a part's result goes: of row `row` (of a unit: the row itself, or its
// place among a few rows' slots)
struct pg_slot { float *po; float2 *pml; };
OH_DEV pg_slot pg_slot_of(const oh_pattn &a, float *po, float2 *pml, int64_t row, int h, int parts, int c) {
    const int64_t at = (row * a.nh + h) * parts + c;
    return {po + at * a.pool.hd, pml + at};
}

OH_DEV void pg_part(const pg_unit &u, int c, int parts, int *t0, int *t1) { pg_part(u.lo, u.hi, c, parts, t0, t1); }

// ---- the kernels for many rows ---------------------------------------------------
// The rows (times heads) are cut at multiples of TR and where units begin; a
// block takes one such piece: rows [from, to) of unit u, for one kv head. The unit
// of a piece is the last one whose first piece is not behind it, and a batch of
// one prompt among many single tokens has few idle blocks. (Idle ones in turn
// with busy ones would leave half of the shader engines without work.) Last rows
// first: they see the most. An XCD, with an L2 of its own, has no other heads'
// pieces than it must.
template <bool PREFIX, int TR>
OH_DEV bool pg_piece(const oh_pattn &a, int pieces, pg_unit *u, int *kvh, int64_t *from, int64_t *to) {
    int64_t piece;
    pg_block_of(blockIdx.x, blockIdx.y, pieces, a.pool.nkv, kvh, &piece);
    if (*kvh >= a.pool.nkv) return false;
    auto first = [&](int i) { return (int64_t)a.b.start[PREFIX ? min(max(a.gfirst[i], 0), a.b.n_seq) : i] * a.G; };
    const int ui = max(pg_count(PREFIX ? a.n_group : a.b.n_seq, [&](int i) { return pg_first_piece(i, first(i), TR) <= piece; }) - 1, 0);
    if (!pg_unit_at<PREFIX>(a, ui, u)) return false;
    const int64_t F = (int64_t)u->n * a.G;
    return pg_piece_rows(piece, ui, (int64_t)u->row * a.G, F, TR, from, to) && (PREFIX ? u->hi > 0 : F > a.many);
}
// A kernel's dynamic LDS past 64 KB, asked for once on each device (each time
// takes a few us); asked: of this kernel, a bit for each device
inline hipError_t pg_allow_lds(const void *k, int bytes, std::atomic<uint64_t> *asked) {
    if (bytes <= 65536) return hipSuccess;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess || (dev < 64 && *asked >> dev & 1)) return e;
    e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess && dev < 64) *asked |= (uint64_t)1 << dev;
    return e;
}
// pieces, and blocks for them
inline int64_t pg_pieces(const oh_pattn *a, int units, int rows, int64_t *blocks) {
    const int64_t pieces = pg_piece_count((int64_t)a->b.n_rows * a->G, units, rows);
    *blocks = pg_blocks(pieces, a->pool.nkv);
    return pieces;
}

// the call f<rows, pool, head dim>(a, st) for a's types
#define PG_DIMS(f, R, C, a, st)                          \
    switch ((a)->pool.hd) {                              \
    case 64: return f<R, C, 64>(a, st);                  \
    case 128: return f<R, C, 128>(a, st);                \
    case 256: return f<R, C, 256>(a, st);                \
    default: return hipErrorNotSupported;                \
    }
#define PG_ROWS16(f, a, st)                                                         \
    if ((a)->pool.type == OH_PT_BF16) { PG_DIMS(f, OH_PT_BF16, OH_PT_BF16, a, st) } \
    if ((a)->pool.type == OH_PT_F16) { PG_DIMS(f, OH_PT_F16, OH_PT_F16, a, st) }    \
    if ((a)->type == OH_PT_BF16) { PG_DIMS(f, OH_PT_BF16, OH_PT_Q8, a, st) }        \
    PG_DIMS(f, OH_PT_F16, OH_PT_Q8, a, st)
#define PG_TYPES(f, a, st)                                                          \
    if ((a)->type == OH_PT_F32) { PG_DIMS(f, OH_PT_F32, OH_PT_Q8, a, st) }          \
    PG_ROWS16(f, a, st)
