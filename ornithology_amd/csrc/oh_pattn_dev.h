// oh_pattn_dev.h - what the attention kernels over a paged pool share: the
// batch's bounds, the parts of the key axis, operand conversion.
//
// o = sum_{t < lim} softmax_t(q . k_t * scale) v_t per row and head, lim the
// row's position + 1. Scores are taken in units of log2(e), so that the
// softmax is 2^(s - m). Products run on the matrix cores with 32-bit
// accumulators; rows of 32 bits (and 16-bit fp rows over codes) enter as sums
// of bf16 terms, whose products with the codes are exact: three terms hold 24
// bits, so nothing of an f32 row is lost.
#pragma once
#include "oh_paged_dev.h"

// operand vectors of the matrix instructions: fp16 for fp16 pools, else bf16
// (codes up to 127 are exact in either; bf16 has f32's range, so a weight
// p * scale cannot leave it)
template <int CT> struct pg_op { typedef pg_b8 v; typedef __bf16 e; };
template <> struct pg_op<OH_PT_F16> { typedef pg_h8 v; typedef _Float16 e; };

// terms of a query, and of a probability (times its value's scale)
template <int RT, int CT> constexpr int pg_nq() { return RT == OH_PT_F32 ? 3 : RT == OH_PT_F16 && CT == OH_PT_Q8 ? 2 : 1; }

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
OH_DEV pg_b8 pg_codes(uint32_t lo, uint32_t hi) {
    pg_b8 o;
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = (__bf16)(float)(int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
    return o;
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
// the positions that sequence s leaves to its group's prefix
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

// parts of a stretch of n positions: at most `most`, of at least 4 tiles each
// (a part's partial result is as large as two positions of a 16-bit pool)
constexpr int kPartMin = 128;
OH_DEV int pg_parts(int n, int most) {
    const int p = (n + kPartMin - 1) / kPartMin;
    return p < 1 ? 1 : p < most ? p : most;
}
// the 32-position tiles [t0, t1) of part c of a unit
OH_DEV void pg_part(const pg_unit &u, int c, int parts, int *t0, int *t1) {
    const int T0 = u.lo >> 5, T = u.hi > u.lo ? ((u.hi + 31) >> 5) - T0 : 0;
    *t0 = T0 + (int)((int64_t)T * c / parts);
    *t1 = T0 + (int)((int64_t)T * (c + 1) / parts);
}

// the call f<rows, pool, head dim>(a, st) for a's types
#define PG_DIMS(f, R, C, a, st)                          \
    switch ((a)->pool.hd) {                              \
    case 64: return f<R, C, 64>(a, st);                  \
    case 128: return f<R, C, 128>(a, st);                \
    case 256: return f<R, C, 256>(a, st);                \
    default: return hipErrorNotSupported;                \
    }
#define PG_TYPES(f, a, st)                                                          \
    if ((a)->pool.type == OH_PT_BF16) { PG_DIMS(f, OH_PT_BF16, OH_PT_BF16, a, st) } \
    if ((a)->pool.type == OH_PT_F16) { PG_DIMS(f, OH_PT_F16, OH_PT_F16, a, st) }    \
    if ((a)->type == OH_PT_F32) { PG_DIMS(f, OH_PT_F32, OH_PT_Q8, a, st) }          \
    if ((a)->type == OH_PT_BF16) { PG_DIMS(f, OH_PT_BF16, OH_PT_Q8, a, st) }        \
    PG_DIMS(f, OH_PT_F16, OH_PT_Q8, a, st)
