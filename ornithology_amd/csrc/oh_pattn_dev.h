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
// A unit of work: the rows [row, row + n) of one sequence (or of a group's
// sequences, for its prefix), over the positions [lo, hi) of a page list
struct pg_unit { int row, n, lo, hi; const int32_t *pages; };

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
// the group of sequence s, -1: none
OH_DEV int pg_group_of(const oh_pattn &a, int s) {
    int lo = 0, hi = a.n_group;
    if (!hi) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.gfirst[mid] <= s) lo = mid; else hi = mid;
    }
    return s >= a.gfirst[lo] && s < a.gfirst[lo + 1] ? lo : -1;
}
// parts of a stretch of n positions: at most `most`, of at least 4 tiles each
// (a part's partial result is as large as two positions of a 16-bit pool)
constexpr int kPartMin = 128;
OH_DEV int pg_parts(int n, int most) {
    const int p = (n + kPartMin - 1) / kPartMin;
    return p < 1 ? 1 : p < most ? p : most;
}
// what is visible to row `token` of a unit: positions below this
OH_DEV int pg_lim(const oh_pattn &a, int len, int end, int token) { const int p = len - (end - token) + 1; return p > 0 ? p : 0; }
