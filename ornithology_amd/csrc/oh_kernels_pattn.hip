// oh_kernels_pattn.hip - attention of a ragged batch over a paged pool, and the
// joining of partial results.
#include "oh_pattn_dev.h"
#include <algorithm>

namespace {

// Few rows: a block takes up to 16 rows (row, head of one kv head's group) of
// a sequence and a part of its positions; its four waves take tiles of 32
// positions in turn and join at the end. Per tile a wave forms S^T = K Q^T
// (lane n = lane & 15 holds row n's scores of positions 4g..4g+3 and
// 16+4g..+3, g = lane >> 4), the probabilities, and O^T += V^T P^T with the
// probabilities where they are: the pool's value order matches.
template <int RT, int CT, int HD, bool PREFIX>
__global__ void __launch_bounds__(256)
pattn_few(oh_pattn a, int tiles_of_rows) {
    typedef typename pg_elem<RT>::t row_t;
    typedef pg_ops<RT, CT> ops;
    typedef typename ops::kv kop;
    typedef typename ops::vv vop;
    constexpr bool Q8 = CT == OH_PT_Q8;
    constexpr int NQ = ops::NQ, NP = RT == OH_PT_F32 ? 3 : 2, NS = HD / 32, ND = HD / 16;
    __shared__ float red[4][16][68];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    const int ui = (int)blockIdx.x / tiles_of_rows, rt = (int)blockIdx.x % tiles_of_rows, kvh = blockIdx.y, c = blockIdx.z;
    pg_unit u;
    if (!pg_unit_at<PREFIX>(a, ui, &u)) return;
    const int G = a.G, F = u.n * G;
    if (rt * 16 >= F || (!PREFIX && F > a.few) || (PREFIX && !u.hi)) return;
    const int parts = pg_parts(u.hi - u.lo, PREFIX ? a.gparts : a.parts);
    if (c >= parts) return;
    const int64_t all = a.gparts + a.sparts, pc = PREFIX ? c : a.gparts + c;
    const bool direct = !PREFIX && parts == 1 && u.lo == 0;
    int t0, t1;
    pg_part(u, c, parts, &t0, &t1);
    // this lane's row
    const int f = rt * 16 + n, tok = u.row + f / G, head = kvh * G + f % G;
    const bool valid = f < F;
    const int lim = valid ? pg_unit_lim<PREFIX>(a, u, tok) : 0;
    const row_t *src = (const row_t *)a.q.p + tok * a.q.rs + head * a.q.hs;
    kop qf[NQ][NS];
    float unit = a.scale;
    {
        float x[NS][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = valid ? (float)src[(Q8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g) + j] * a.sign : 0.0f;
                top = fmaxf(top, fabsf(x[i][j]));
            }
        if (NQ > 1) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const int e = pg_row_exp(top);
            unit = ldexpf(unit, -e);
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = ldexpf(x[i][j], e);
        }
#pragma unroll
        for (int i = 0; i < NS; i++) {
            kop t[NQ];
            pg_split<NQ>(x[i], t);
#pragma unroll
            for (int k = 0; k < NQ; k++) qf[k][i] = t[k];
        }
    }
    pg_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const int page_mask = (1 << a.pool.page_sh) - 1;
    for (int t = t0 + wave; t < t1; t += 4) {
        const int tb = 32 * t, page0 = u.pages[tb >> a.pool.page_sh];
        const bool bad = page0 < 0 || page0 >= a.pool.n_pages;   // its positions are seen by no row
        if (bad && lane == 0) pg_report(a.pool, OH_PF_PAGE);
        const uint8_t *blk = pg_block(a.pool, bad ? 0 : page0, kvh);
        const int slot = tb & page_mask;
        const int vis = bad ? 0 : lim - tb;                      // positions of the tile below this are visible
        const size_t tile = (size_t)(slot >> 5) * 32 * HD * (Q8 ? 1 : 2);
        const uint8_t *kp = blk + tile, *vp = blk + a.pool.v_off + tile;
        pg_f4 sc[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            sc[h] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
            if (Q8) {
#pragma unroll
                for (int i = 0; i < NS / 2; i++) {
                    const uint4 w = *(const uint4 *)(kp + ((4 * i + g) * 32 + 16 * h + n) * 16);
                    kop k0, k1;
                    pg_codes(w.x, w.y, &k0);
                    pg_codes(w.z, w.w, &k1);
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--) {          // the small terms first
                        sc[h] = pg_mma16(k0, qf[k][2 * i], sc[h]);
                        sc[h] = pg_mma16(k1, qf[k][2 * i + 1], sc[h]);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < NS; i++)
                    sc[h] = pg_mma16(*(const kop *)(kp + ((4 * i + g) * 32 + 16 * h + n) * 16), qf[0][i], sc[h]);
            }
        }
        float p[8];
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            pg_f4 ks = {1.0f, 1.0f, 1.0f, 1.0f};
            if (Q8) ks = *(const pg_f4 *)(blk + a.pool.ks_off + 4 * (slot + 16 * h + 4 * g));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float x = Q8 ? sc[h][i] * ks[i] * unit : sc[h][i] * unit;
                p[4 * h + i] = 16 * h + 4 * g + i < vis ? x : -INFINITY;
                mx = fmaxf(mx, p[4 * h + i]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m, mx);
        const float alpha = mn == m ? 1.0f : pg_exp2(m - mn);
        const float ref = mn == -INFINITY ? 0.0f : mn;           // (nothing seen, or keys of -inf)
        m = mn;
        l *= alpha;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            pg_f4 vs = {1.0f, 1.0f, 1.0f, 1.0f};
            if (Q8) vs = *(const pg_f4 *)(blk + a.pool.vs_off + 4 * (slot + 16 * h + 4 * g));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool see = 16 * h + 4 * g + i < vis;
                const float e = see ? pg_exp2(p[4 * h + i] - ref) : 0.0f;
                l += e;
                p[4 * h + i] = Q8 ? (see ? e * vs[i] : 0.0f) : e;
            }
        }
        vop pf[NP];
        pg_split<NP>(p, pf);
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] *= alpha;
        // Whole tiles hold finite values or ones that every row sees; where a
        // row of the tile sees only a part, what it does not see (another
        // request's leavings, a later token) may be infinite or NaN, and 0
        // times that is NaN: such tiles go row by row, with those values zero
        bool odd = false;
        vop vf[ND];
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
            if (Q8) {
                const uint4 w = *(const uint4 *)(vp + (g * HD + 16 * d + 2 * n) * 8);
                pg_codes(w.x, w.y, &vf[d]);
                pg_codes(w.z, w.w, &vf[d + 1]);
            } else {
                vf[d] = *(const vop *)(vp + (g * HD + 16 * d + n) * 16);
                vf[d + 1] = *(const vop *)(vp + (g * HD + 16 * (d + 1) + n) * 16);
            }
        }
        if (!Q8 && __any(valid && vis < 32)) {
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int j = 0; j < 8; j++) odd |= !isfinite((float)vf[d][j]);
            odd = __any(odd);
        }
        if (!odd) {
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int k = NP - 1; k >= 0; k--) o[d] = pg_mma16(vf[d], pf[k], o[d]);
        } else {
            for (int r = 0; r < 16; r++) {
                const int v = __shfl(vis, r);                    // row r's
                if (v <= 0) continue;
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    vop x;
#pragma unroll
                    for (int j = 0; j < 8; j++) x[j] = 16 * (j >> 2) + 4 * g + (j & 3) < v ? vf[d][j] : (typename ops::ve)0.0f;
                    pg_f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--) y = pg_mma16(x, pf[k], y);
                    if (n == r) o[d] += y;
                }
            }
        }
    }
    // the waves' results joined, 64 dims at a time
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (l != l) m = fmaxf(m, 0.0f);                    // a NaN score stays one
    if (g == 0) { sm[wave][n] = m; sl[wave][n] = l; }
    __syncthreads();
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w][n]);
#pragma unroll
    for (int w = 0; w < 4; w++) L += sm[w][n] == -INFINITY ? 0.0f : sl[w][n] * pg_exp2(sm[w][n] - M);
    const float mine = m == -INFINITY ? 0.0f : pg_exp2(m - M);
    const int64_t part = ((int64_t)tok * a.nh + head) * all + pc;
    if (!direct && wave == 0 && g == 0 && valid) a.pml[part] = make_float2(M, L);
    // thread x writes row x >> 4, dims 4 (x & 15) .. + 3 of the 64
    const int wr = threadIdx.x >> 4, wd = 4 * (threadIdx.x & 15), wf = rt * 16 + wr;
    const int wtok = u.row + wf / G, whead = kvh * G + wf % G;
    float Lw = 0.0f, Mw = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) Mw = fmaxf(Mw, sm[w][wr]);
#pragma unroll
    for (int w = 0; w < 4; w++) Lw += sm[w][wr] == -INFINITY ? 0.0f : sl[w][wr] * pg_exp2(sm[w][wr] - Mw);
    const float inv = direct ? (Lw > 0.0f || Lw != Lw ? 1.0f / Lw : 0.0f) : 1.0f;
#pragma unroll
    for (int q = 0; q < HD / 64; q++) {
        if (q) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                // dim within the 64: 8-bit values come two dims a lane
                const int dim = Q8 ? 32 * (d >> 1) + 2 * (4 * g + i) + (d & 1) : 16 * d + 4 * g + i;
                red[wave][n][dim] = mine == 0.0f ? 0.0f : o[4 * q + d][i] * mine;
            }
        __syncthreads();
        if (wf < F) {
            float y[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                y[i] = (red[0][wr][wd + i] + red[1][wr][wd + i] + red[2][wr][wd + i] + red[3][wr][wd + i]) * inv;
            if (direct) {
                row_t *to = (row_t *)a.out.p + wtok * a.out.rs + whead * a.out.hs + 64 * q + wd;
#pragma unroll
                for (int i = 0; i < 4; i++) to[i] = (row_t)y[i];
            } else {
                *(pg_f4 *)(a.po + (((int64_t)wtok * a.nh + whead) * all + pc) * HD + 64 * q + wd) = (pg_f4){y[0], y[1], y[2], y[3]};
            }
        }
    }
}

// Partial results joined: a wave takes one head of one row.
template <int RT, int HD>
__global__ void __launch_bounds__(256)
pattn_join(oh_pattn a) {
    typedef typename pg_elem<RT>::t row_t;
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int r = (int)(item / a.nh), h = (int)(item % a.nh);
    if (r >= a.b.n_rows) return;
    const int s = pg_seq_of(a.pool, a.b, r);
    int row0, rows, len;
    if (s < 0 || !pg_seq(a, s, &row0, &rows, &len)) return;
    const int lo = pg_prefix_of(a, s);
    const int parts = pg_parts(len - lo, rows * a.G <= a.few ? a.parts : a.mparts), gparts = lo ? pg_parts(lo, a.gparts) : 0;
    if (parts == 1 && !gparts) return;                 // written already
    const int64_t at = item * (a.gparts + a.sparts);
    const int np = gparts + parts;
    // part c of np: the prefix's, then the sequence's own
    float M = -INFINITY;
    for (int c = lane; c < np; c += 64) M = fmaxf(M, a.pml[at + (c < gparts ? c : a.gparts + c - gparts)].x);
#pragma unroll
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    float L = 0.0f, y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = 0.0f;
    for (int c = 0; c < np; c++) {
        const int64_t pc = at + (c < gparts ? c : a.gparts + c - gparts);
        const float2 ml = a.pml[pc];
        if (ml.x == -INFINITY) continue;               // nothing visible in it
        const float w = pg_exp2(ml.x - M);
        L = fmaf(ml.y, w, L);
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = fmaf(a.po[pc * HD + lane * E + e], w, y[e]);
    }
    const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
    row_t *to = (row_t *)a.out.p + r * a.out.rs + h * a.out.hs + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) to[e] = (row_t)(y[e] * inv);
}

template <int RT, int CT, int HD>
hipError_t go_few(const oh_pattn *a, hipStream_t st) {
    const int64_t tiles = (std::min((int64_t)a->b.max_new * a->G, (int64_t)a->few) + 15) / 16;
    if (tiles * a->b.n_seq > kMaxBlocks) return hipErrorInvalidConfiguration;
    if (a->n_group && !a->gmany) {
        const int64_t gtiles = ((int64_t)a->b.n_rows * a->G + 15) / 16;
        if (gtiles * a->n_group > kMaxBlocks) return hipErrorInvalidConfiguration;
        hipLaunchKernelGGL((pattn_few<RT, CT, HD, true>), dim3((unsigned)(gtiles * a->n_group), a->pool.nkv, a->gparts), dim3(256), 0, st, *a, (int)gtiles);
    }
    if (tiles)
        hipLaunchKernelGGL((pattn_few<RT, CT, HD, false>), dim3((unsigned)(tiles * a->b.n_seq), a->pool.nkv, a->parts), dim3(256), 0, st, *a, (int)tiles);
    return hipGetLastError();
}
template <int RT, int CT, int HD>
hipError_t go_join(const oh_pattn *a, hipStream_t st) {
    const int64_t blocks = ((int64_t)a->b.n_rows * a->nh + 3) / 4;
    if (blocks > kMaxBlocks) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((pattn_join<RT, HD>), dim3((unsigned)blocks), dim3(256), 0, st, *a);
    return hipGetLastError();
}

} // namespace

extern "C" hipError_t oh_launch_pattn_few(const oh_pattn *a, hipStream_t st) { PG_TYPES(go_few, a, st) }
extern "C" hipError_t oh_launch_pattn_join(const oh_pattn *a, hipStream_t st) { PG_TYPES(go_join, a, st) }
