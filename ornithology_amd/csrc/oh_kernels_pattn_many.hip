// oh_kernels_pattn_many.hip - attention over a paged pool where a sequence, or a
// group that shares a prefix, brings many rows.
//
// A block of NW waves takes 32 NW rows (row, head of one kv head's group) and
// a part of the positions, 64 at a time (32 of heads of 256): the tile's keys and
// values go through LDS once for all waves, as matrix operands in the pool's
// order (codes as 16-bit values), in two buffers, the next tile's loads in flight during this one's
// products. A wave holds 32 rows: S^T = K Q^T by 32x32x16 products (lane n =
// lane & 31 holds row n's scores of half the positions), the softmax, and
// O^T += V^T P^T with the probabilities where they are.
//
// Bound by the matrix cores and LDS: a product of 32 cycles takes 1 KB of LDS for
// its key or value operand, which is what LDS gives four SIMDs in that time. 8192
// tokens, 32 heads of 128 over 8, bf16: 0.71 ms, 770 TFLOP/s, where a library
// product of 8192^3 reaches 1140.
#include "oh_pattn_dev.h"
#include <algorithm>

namespace {

// A running maximum may be this much (a factor of 2^8) behind the largest
// score: weights stay far inside every operand type, 32-bit sums lose nothing,
// and the accumulators are scaled a few times a row instead of at every step
constexpr float kBehind = 8.0f;

// Positions a step, waves a block, and whether the waves take turns: of the two
// that share a SIMD one has its products while the other has its softmax. That
// takes eight waves, so two sets of accumulators in a SIMD's registers.
template <int RT, int CT, int HD> constexpr bool can_turn() { return HD < 256 && !(CT == OH_PT_Q8 && HD == 64); }
template <int RT, int CT, int HD, bool TURN> struct many_cfg {
    static constexpr bool TURNS = TURN;
    static constexpr int PER_SIMD = can_turn<RT, CT, HD>() || HD == 64 ? 2 : 1;    // waves
    static constexpr int T = HD == 256 ? 32 : 64, NW = TURNS ? 8 : 4, H = T / 32;
    static constexpr int TILE = T * HD * 2;            // keys, or values, of a step in LDS, as 16-bit operands
    static constexpr int LDS = 4 * TILE + 2 * (8 * T + 16);   // two of each; scales and whether there is a page
};

template <int RT, int CT, int HD, bool PREFIX, bool TURN>
__global__ void __launch_bounds__((64 * many_cfg<RT, CT, HD, TURN>::NW), (many_cfg<RT, CT, HD, TURN>::PER_SIMD))
pattn_many(oh_pattn a, int pieces) {
    typedef typename pg_elem<RT>::t row_t;
    typedef pg_ops<RT, CT> ops;
    typedef typename ops::kv kop;
    typedef typename ops::vv vop;
    typedef many_cfg<RT, CT, HD, TURN> cfg;
    constexpr bool Q8 = CT == OH_PT_Q8;
    constexpr int NW = cfg::NW, T = cfg::T, H = cfg::H, TILE = cfg::TILE, NT = 64 * NW, TR = 32 * NW;
    constexpr int NQ = ops::NQ, NP = RT == OH_PT_F16 && Q8 ? 2 : 1, NS = HD / 16, ND = HD / 32;
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const ldk = lds, *const ldv = lds + 2 * TILE;
    float *const lds_s = (float *)(lds + 4 * TILE);    // [2][keys' T, values' T]
    int *const lds_ok = (int *)(lds_s + 4 * T);        // [2][2]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, hf = lane >> 5;
    const int c = blockIdx.y, G = a.G;
    pg_unit u;
    int kvh;
    int64_t from, to;
    if (!pg_piece<PREFIX, TR>(a, pieces, &u, &kvh, &from, &to)) return;
    const int parts = pg_parts(u.hi - u.lo, PREFIX ? a.gleast : a.mleast, PREFIX ? a.gparts : a.mparts);
    if (c >= parts) return;
    const bool direct = !PREFIX && parts == 1 && u.lo == 0;
    int t0, t1;
    pg_part(u, c, parts, &t0, &t1);
    const int64_t f = from + wave * 32 + n;
    const int tok = (int)(f / G), head = kvh * G + (int)(f % G);
    const bool valid = f < to;
    // what the lane's row sees of the part; the last position that some row of the
    // block sees, and the first that some row does not
    int lim = valid ? min(pg_unit_lim<PREFIX>(a, u, tok), 32 * t1) : 0;
    int blim = lim, bmin = valid ? lim : 1 << 30;
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        blim = max(blim, __shfl_xor(blim, o));
        bmin = min(bmin, __shfl_xor(bmin, o));
    }
    __shared__ int wl[2][NW];
    if (lane == 0) { wl[0][wave] = blim; wl[1][wave] = bmin; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) { blim = max(blim, wl[0][w]); bmin = min(bmin, wl[1][w]); }
    if (!valid) lim = 1 << 30;                         // (no row: nothing to hide)
    blim = __builtin_amdgcn_readfirstlane(blim);
    bmin = __builtin_amdgcn_readfirstlane(bmin);
    const int p0 = 32 * t0, N = blim > p0 ? (blim - p0 + T - 1) / T : 0;       // steps

    kop qf[NQ][NS];
    float unit = a.scale;                              // of the row's scores as they come out of the products
    pg_f16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // ---- a step's keys and values: the 32-position tiles' bytes as they are in
    // the pool, 16 a thread at a time; where there is no page (behind the last
    // position, or a bad index) page 0's, which no row looks at
    constexpr int KB = 32 * HD * (Q8 ? 1 : 2), NL = H * KB / 16 / NT;          // bytes of a tile; loads per thread
    static_assert(H * KB == NL * 16 * NT, "whole loads");
    uint4 kr[NL], vr[NL];
    float scl = 0.0f;
    bool ok[H];
    const int page_mask = (1 << a.pool.page_sh) - 1;
    pg_list lk = {u.pages, a.b.max_pages, 0, 0};
    lk.hold(p0 >> a.pool.page_sh);
    pg_list lv = lk;
    bool bad = false;
    auto tile_at = [&](pg_list &list, int pos, bool *there) -> const uint8_t * {
        int page = -1;
        if (pos < blim) {
            page = list.get(pos >> a.pool.page_sh);
            if (page < 0 || page >= a.pool.n_pages) { page = -1; bad = true; }
        }
        *there = page >= 0;
        return pg_block(a.pool, page < 0 ? 0 : page, kvh) + (size_t)((pos & page_mask) >> 5) * KB;
    };
    bool odd = false, hide = false;                    // (hide: of the step whose values are in vr)
    auto fetch = [&](pg_list &list, int pos, uint32_t plane, uint4 (&r)[NL], bool keys = false) {
        const uint8_t *at[H];
        bool there[H];
#pragma unroll
        for (int h = 0; h < H; h++) at[h] = tile_at(list, pos + 32 * h, &there[h]);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int b = (tid + NT * i) * 16;
            r[i] = ldg((const uint4 *)((H == 1 || b < KB ? at[0] : at[H - 1]) + plane + b % KB));
        }
        if (keys) {
#pragma unroll
            for (int h = 0; h < H; h++) ok[h] = there[h];
        } else {
            hide = pos + T > bmin;
#pragma unroll
            for (int h = 0; h < H; h++) hide |= !there[h];
        }
        if (keys && Q8 && tid < 2 * T) {
            const int x = tid & (T - 1), p = pos + x;
            const uint8_t *blk = (x < 32 ? at[0] : at[H - 1]) - (size_t)((p & page_mask) >> 5) * KB;
            scl = ldg((const float *)(blk + (tid < T ? a.pool.ks_off : a.pool.vs_off) + 4 * (p & page_mask)));
        }
    };
    // keys: units (8 dims of one position) at (dim / 8 * 32 + position) * 16 of a
    // tile; values: units (8 positions of one dim) at (group * HD + dim) * 16
    auto stage_k = [&](int b) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = tid + NT * i;
            if (Q8) {
                const int h = e * 16 / KB, x = e % (KB / 16), ch = x >> 5, sl = x & 31;      // 16 dims ch of position sl
                kop *to = (kop *)(ldk + b * TILE + h * 64 * HD) + 2 * ch * 32 + sl;
                kop k0, k1;
                pg_codes(kr[i].x, kr[i].y, &k0);
                pg_codes(kr[i].z, kr[i].w, &k1);
                to[0] = k0;
                to[32] = k1;
            } else {
                *(uint4 *)(ldk + b * TILE + e * 16) = kr[i];
            }
        }
        if (Q8 && tid < 2 * T) lds_s[b * 2 * T + tid] = scl;
        if (tid == 0)
#pragma unroll
            for (int h = 0; h < H; h++) lds_ok[2 * b + h] = ok[h];
    };
    auto stage_v = [&](int b) {
        if (!Q8 && hide)
#pragma unroll
            for (int i = 0; i < NL; i++) pg_only_finite<ops::VH>(&vr[i], &odd);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = tid + NT * i;
            if (Q8) {
                vop v0, v1;
                pg_codes(vr[i].x, vr[i].y, &v0);
                pg_codes(vr[i].z, vr[i].w, &v1);
                vop *to = (vop *)(ldv + b * TILE) + 2 * e;
                to[0] = v0;
                to[1] = v1;
            } else {
                *(uint4 *)(ldv + b * TILE + e * 16) = vr[i];
            }
        }
    };

    // ---- products: S^T of step t, and O^T of the step before
    pg_f16 s[H];
    vop pf[NP][H][2];
    auto scores = [&](int t) {
        // operand row n is position 16 (n >> 3 & 1) + 8 (n >> 4) + (n & 7), so that
        // a lane's 8 scores of a product are one unit of the values
        const kop *at = (const kop *)(ldk + (t & 1) * TILE) + hf * 32 + 16 * ((n >> 3) & 1) + 8 * (n >> 4) + (n & 7);
#pragma unroll
        for (int h = 0; h < H; h++) {
#pragma unroll
            for (int v = 0; v < 16; v++) s[h][v] = 0.0f;
#pragma unroll
            for (int i = 0; i < NS; i++) {
                const kop kf = at[h * 4 * HD + i * 64];
#pragma unroll
                for (int k = NQ - 1; k >= 0; k--) s[h] = pg_mma32(kf, qf[k][i], s[h]);       // the small term first
            }
        }
    };
    auto values = [&](int t) {
        const vop *at = (const vop *)(ldv + (t & 1) * TILE) + hf * HD + n;
        auto unit_at = [&](int h, int k, int d) { return at[h * 4 * HD + 2 * k * HD + 32 * d]; };
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const vop vf = unit_at(h, k, d);
#pragma unroll
                    for (int x = NP - 1; x >= 0; x--) o[d] = pg_mma32(vf, pf[x][h][k], o[d]);
                }
    };

    // ---- the softmax of step t: weights from scores
    auto softmax = [&](int t) {
        const int pos = p0 + t * T, b = t & 1;
        const float *ks = lds_s + b * 2 * T, *vs = ks + T;
        int vis[H];                                    // positions of a tile below this are visible to the row
        bool some = false;
#pragma unroll
        for (int h = 0; h < H; h++) {
            vis[h] = __builtin_amdgcn_readfirstlane(lds_ok[2 * b + h]) ? lim - pos - 32 * h : 0;
            some |= vis[h] < 32;
        }
        const bool part = __any(some);
        if (Q8) {
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const pg_f4 kk = *(const pg_f4 *)(ks + 32 * h + 16 * (q & 1) + 8 * (q >> 1) + 4 * hf);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[h][4 * q + i] *= kk[i];
                }
        }
        if (part) {
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int v = 0; v < 16; v++)
                    if (16 * ((v >> 2) & 1) + 8 * (v >> 3) + (v & 3) >= vis[h] - 4 * hf) s[h][v] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int v = 0; v < 16; v++) mx = fmaxf(mx, s[h][v]);
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * unit;
        if (__any(mx > m + kBehind)) {
            const float mn = fmaxf(m, mx), alpha = mn == m ? 1.0f : pg_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) o[d][v] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.0f : m;   // (nothing seen yet, or keys of -inf)
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = pg_exp2(fmaf(s[h][8 * k + j], unit, -ref));
                    sum[j & 3] += p[j];
                }
                if (Q8) {
#pragma unroll
                    for (int q = 0; q < 2; q++) {
                        const pg_f4 vv = *(const pg_f4 *)(vs + 32 * h + 16 * q + 8 * k + 4 * hf);
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            // (a scale that the row does not see may be anything)
                            const bool see = !part || 16 * q + 8 * k + i < vis[h] - 4 * hf;
                            p[4 * q + i] = see ? p[4 * q + i] * vv[i] : 0.0f;
                        }
                    }
                }
                vop w[NP];
                pg_split<NP>(p, w);
#pragma unroll
                for (int x = 0; x < NP; x++) pf[x][h][k] = w[x];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };

    // Loads and products run one step past the end, on page 0's bytes and for
    // nothing: no branch splits the loops' registers.
    fetch(lk, p0, 0, kr, true);
    if (!cfg::TURNS) fetch(lv, p0, a.pool.v_off, vr);
    {
        float x[NS][8], top = 0.0f;
        const row_t *src = (const row_t *)a.q.p + (valid ? tok * a.q.rs + head * a.q.hs : u.row * a.q.rs) + 8 * hf;
#pragma unroll
        for (int i = 0; i < NS; i++)
            pg_load<8>(src + 16 * i, x[i]);
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = valid ? x[i][j] * a.sign : 0.0f;
                top = fmaxf(top, fabsf(x[i][j]));
            }
        if (NQ > 1) {
            const int e = pg_row_exp(fmaxf(top, __shfl_xor(top, 32)));
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
    stage_k(0);
    if (!cfg::TURNS) stage_v(0);
    __syncthreads();
    if (!cfg::TURNS) {
        for (int t = 0; t < N; t++) {
            fetch(lk, p0 + (t + 1) * T, 0, kr, true);
            fetch(lv, p0 + (t + 1) * T, a.pool.v_off, vr);
            scores(t);
            softmax(t);
            values(t);
            stage_k(~t & 1);
            stage_v(~t & 1);
            __syncthreads();
        }
    } else {
        // Half-steps, a barrier after each. The first four waves have their
        // products (O of step t - 1, S of step t) in half-step 2t and the softmax of
        // t in 2t + 1; the others half a step later. Half-step 2t requests the keys
        // of step t + 1 and the values of t; 2t + 1 puts them where those of two
        // steps before were, whose last readers were done in half-step 2t - 1.
        fetch(lv, p0, a.pool.v_off, vr);
        fetch(lk, p0 + T, 0, kr, true);
        if (wave < NW / 2) {
            scores(0);
            __syncthreads();
            for (int t = 0; t < N; t++) {
                softmax(t);
                stage_v(t & 1);
                stage_k(~t & 1);
                __syncthreads();
                fetch(lv, p0 + (t + 1) * T, a.pool.v_off, vr);
                fetch(lk, p0 + (t + 2) * T, 0, kr, true);
                values(t);
                scores(t + 1);
                __syncthreads();
            }
        } else {
            __syncthreads();
            scores(0);
            stage_v(0);
            stage_k(1);
            for (int t = 0; t < N; t++) {
                __syncthreads();
                fetch(lv, p0 + (t + 1) * T, a.pool.v_off, vr);
                fetch(lk, p0 + (t + 2) * T, 0, kr, true);
                softmax(t);
                __syncthreads();
                values(t);
                scores(t + 1);
                stage_v(~t & 1);
                stage_k(t & 1);
            }
        }
    }
    if (bad && tid == 0) pg_report(a.pool, OH_PF_PAGE);
    if (!Q8 && __syncthreads_or(odd)) {
        // dims 32 d + 8 q + 4 hf + i of the lane's row, over the steps that hid
        // something (one that did not has added its values: once more changes nothing)
        for (int p = bad || bmin < p0 ? p0 : p0 + (bmin - p0) / T * T; p < blim; p++) {
            const int page = u.pages[p >> a.pool.page_sh];
            if (p >= lim || !valid || page < 0 || page >= a.pool.n_pages) continue;
            const typename ops::ve *at = (const typename ops::ve *)(pg_block(a.pool, page, kvh) + a.pool.v_off) + pg_v_at(HD, p & page_mask, 4 * hf);
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const float y = (float)at[(32 * d + 8 * (v >> 2) + (v & 3)) * 8];
                    if (!isfinite(y)) o[d][v] += y;
                }
        }
    }
    l += __shfl_xor(l, 32);
    if (l != l) m = fmaxf(m, 0.0f);                    // a NaN score stays one
    if (!valid) return;
    // lane n's row: dims 32 d + 8 q + 4 hf .. + 3
    if (direct) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        row_t *to = (row_t *)a.out.p + tok * a.out.rs + head * a.out.hs + 4 * hf;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = o[d][4 * q + i] * inv;
                pg_store<4>(to + 32 * d + 8 * q, y);
            }
    } else {
        const pg_slot at = PREFIX ? pg_slot_of(a, a.gpo, a.gpml, tok, head, a.gparts, c) : pg_slot_of(a, a.mpo, a.mpml, tok, head, a.mparts, c);
        if (hf == 0) *at.pml = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *(pg_f4 *)(at.po + 32 * d + 8 * q + 4 * hf) = (pg_f4){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    }
}

template <int RT, int CT, int HD, bool PREFIX, bool TURN>
hipError_t launch(const oh_pattn *a, int units, int parts, hipStream_t st) {
    constexpr int NW = many_cfg<RT, CT, HD, TURN>::NW, lds = many_cfg<RT, CT, HD, TURN>::LDS;
    int64_t blocks;
    const int64_t pieces = pg_pieces(a, units, 32 * NW, &blocks);
    if (blocks > kMaxBlocks / 2) return hipErrorInvalidConfiguration;
    const auto k = pattn_many<RT, CT, HD, PREFIX, TURN>;
    static std::atomic<uint64_t> asked{0};
    const hipError_t e = pg_allow_lds((const void *)k, lds, &asked);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks, parts), dim3(64 * NW), lds, st, *a, (int)pieces);
    return hipGetLastError();
}
template <int RT, int CT, int HD, bool PREFIX>
hipError_t with_turns(const oh_pattn *a, int rows, int units, int parts, hipStream_t st) {
    if constexpr (can_turn<RT, CT, HD>())
        if (rows == 256) return launch<RT, CT, HD, PREFIX, true>(a, units, parts, st);
    return launch<RT, CT, HD, PREFIX, false>(a, units, parts, st);
}
template <int RT, int CT, int HD>
hipError_t go_rows(const oh_pattn *, int *rows) {
    *rows = can_turn<RT, CT, HD>() ? 256 : 128;
    return hipSuccess;
}
template <int RT, int CT, int HD>
hipError_t go_many(const oh_pattn *a, hipStream_t st) {
    hipError_t e = hipSuccess;
    if (a->n_group && a->gmany) e = with_turns<RT, CT, HD, true>(a, a->grows, a->n_group, a->gparts, st);
    if (e == hipSuccess && a->many >= 0) e = with_turns<RT, CT, HD, false>(a, a->mrows, a->b.n_seq, a->mparts, st);
    return e;
}

} // namespace

extern "C" hipError_t oh_pattn_many_rows(const oh_pattn *a, int *rows) {
    *rows = 128;
    if (a->type == OH_PT_F32) return hipSuccess;
    PG_ROWS16(go_rows, a, rows)
}
extern "C" hipError_t oh_launch_pattn_many(const oh_pattn *a, hipStream_t st) {
    if (a->type == OH_PT_F32) return oh_launch_pattn_f32(a, st);
    PG_ROWS16(go_many, a, st)
}
