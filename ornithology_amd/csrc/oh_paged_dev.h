// oh_paged_dev.h - device helpers of the paged pool's kernels.
#pragma once
#include "oh_common.h"
#include "oh_paged.h"
#include "oh_paged_layout.h"

typedef __bf16 pg_b8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));

template <int T> struct pg_elem;                       // storage type of a row or pool element
template <> struct pg_elem<OH_PT_F32> { typedef float t; };
template <> struct pg_elem<OH_PT_F16> { typedef _Float16 t; };
template <> struct pg_elem<OH_PT_BF16> { typedef __bf16 t; };
template <> struct pg_elem<OH_PT_Q8> { typedef int8_t t; };

OH_DEV void pg_report(const oh_pool &p, int bit) { atomicOr(p.fault, bit); }

template <int CT>
OH_DEV uint32_t pg_k_at(int hd, int slot, int d) { return pg_k_place(CT == OH_PT_Q8 ? 16 : 8, hd, slot, d); }
OH_DEV uint8_t *pg_block(const oh_pool &p, int page, int head) {
    return p.mem + ((size_t)page * p.nkv + head) * p.block;
}

// How many of the indices [0, n) have p(i), for a p that holds up to some index
// and not behind it: 64 at a time, one to a lane, so that a search costs a round
// trip to memory and not one for each halving. The whole wave calls it.
template <class P>
OH_DEV int pg_count(int n, P p) {
    int c = 0;
    for (int i = 0; i < n; i += 64) {
        const int at = i + (int)(threadIdx.x & 63);
        const int k = (int)__popcll(__ballot(at < n && p(at)));
        c += k;
        if (k < 64) break;
    }
    return c;
}
// The sequence that row r (the same in the whole wave) belongs to, -1 if none
// does (and reported, but for rows behind the last sequence). A list that is not
// ascending leaves the other sequences' rows their own.
OH_DEV int pg_seq_of_wave(const oh_pool &p, const oh_pbatch &b, int r) {
    for (int i = 0; i < b.n_seq; i += 64) {
        const int at = i + (int)(threadIdx.x & 63);
        const uint64_t own = __ballot(at < b.n_seq && b.start[at] <= r && r < b.start[at + 1]);
        if (!own) continue;
        const int s = i + __builtin_ctzll(own);
        if (b.start[s + 1] <= b.n_rows) return s;
        pg_report(p, OH_PF_BATCH);
        return -1;
    }
    if (r < b.start[b.n_seq]) pg_report(p, OH_PF_BATCH);
    return -1;
}
// the same of a row of the lane's own
OH_DEV int pg_seq_of(const oh_pool &p, const oh_pbatch &b, int r) {
    int lo = 0, hi = b.n_seq;                          // the last s with start[s] <= r
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.start[mid] <= r) lo = mid; else hi = mid;
    }
    const int s0 = b.start[lo], s1 = b.start[lo + 1];
    if (r < s0 || r >= s1) {
        // rows behind the last sequence are nobody's; any other such row is a mistake
        if (r < b.start[b.n_seq]) pg_report(p, OH_PF_BATCH);
        return -1;
    }
    if (s1 > b.n_rows) { pg_report(p, OH_PF_BATCH); return -1; }
    return lo;
}

// N (8 or 4) values of a row at p, which is a multiple of their size
template <int N>
OH_DEV void pg_load(const float *p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const pg_f4 w = ldg((const pg_f4 *)(p + i));
        x[i] = w[0]; x[i + 1] = w[1]; x[i + 2] = w[2]; x[i + 3] = w[3];
    }
}
template <int N, class T>
OH_DEV void pg_load(const T *p, float (&x)[N]) {
    typedef T v __attribute__((ext_vector_type(N)));
    const v w = ldg((const v *)p);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = (float)w[i];
}
template <int N, class T>
OH_DEV void pg_store(T *p, const float (&x)[N]) {
    typedef T v __attribute__((ext_vector_type(N)));
    v w;
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = (T)x[i];
    *(v *)p = w;
}

// log2 of e
constexpr float kLog2e = 1.44269504088896340736f;
OH_DEV float pg_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
