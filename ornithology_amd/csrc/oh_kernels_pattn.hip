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
//
// Bound by memory where sequences are long or many (64 of up to 16000 positions,
// 8 heads of 128 in bf16: 265 us, 5.5 TB/s), by the chain of its loads where
// there is little to do: 13 us for one token after 4096 8-bit positions, of them
// 1.6 to find the item, 2 to request, 3 a tile of f32 rows, 2 to join the waves.
// One tile ahead for each wave, in registers and not through LDS (no wave shares
// another's): 16 to 32 KB in flight a wave.
//
// Work is dealt out in items: (part of the positions, 16 rows, kv head) of a
// prefix (`groups`: those of this kernel, before the sequences) or sequence. How
// many a unit has is known on the device only, where the lengths are.
struct few_item { int unit, rt, kvh, part; bool prefix; };
OH_DEV int few_items(const oh_pattn &a, int groups, int x, pg_unit *o) {
    pg_unit &u = *o;
    const bool prefix = x < groups;
    if (!(prefix ? pg_unit_at<true>(a, x, &u) : pg_unit_at<false>(a, x - groups, &u))) return 0;
    const int F = u.n * a.G;
    if (prefix ? !u.hi : F > a.few) return 0;
    return pg_parts(u.hi - u.lo, prefix ? a.gleast : a.least, prefix ? a.gparts : a.parts) * ((F + 15) / 16) * a.pool.nkv;
}
// item i, false if there are fewer. The whole wave calls it; a lane counts one of 64 units.
OH_DEV bool few_find(const oh_pattn &a, int groups, int i, few_item *o, pg_unit *u) {
    const int lane = threadIdx.x & 63, n = groups + a.b.n_seq;
    for (int x0 = 0, before = 0; x0 < n; x0 += 64) {
        pg_unit un = {0, 0, 0, 0, nullptr};
        const int x = x0 + lane, mine = x < n ? few_items(a, groups, x, &un) : 0;
        int sum = mine;                                // of the units up to and with this lane's
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(sum, d);
            if (lane >= d) sum += y;
        }
        const uint64_t ends = __ballot(before + sum > i);
        if (ends) {
            const int l = __builtin_ctzll(ends);
            const int left = i - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(mine, l));
            o->prefix = x0 + l < groups;
            o->unit = x0 + l - (o->prefix ? 0 : groups);
            u->row = __builtin_amdgcn_readlane(un.row, l);
            u->n = __builtin_amdgcn_readlane(un.n, l);
            u->lo = __builtin_amdgcn_readlane(un.lo, l);
            u->hi = __builtin_amdgcn_readlane(un.hi, l);
            const int64_t at = (int64_t)(un.pages - a.b.table);
            u->pages = a.b.table + ((int64_t)__builtin_amdgcn_readlane((int)(at >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)at, l));
            const int tiles = (u->n * a.G + 15) / 16;
            o->kvh = left % a.pool.nkv;
            o->rt = left / a.pool.nkv % tiles;
            o->part = left / a.pool.nkv / tiles;
            return true;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

template <int RT, int CT, int HD>
__global__ void __launch_bounds__(256)
pattn_few(oh_pattn a, int groups) {
    typedef typename pg_elem<RT>::t row_t;
    typedef pg_ops<RT, CT> ops;
    typedef typename ops::kv kop;
    typedef typename ops::vv vop;
    constexpr bool Q8 = CT == OH_PT_Q8;
    constexpr int NQ = ops::NQ, NP = RT == OH_PT_F32 ? 3 : 2, NS = HD / 32, ND = HD / 16;
    __shared__ float red[4][16][68];
    __shared__ float sm[4][16], sl[4][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    for (int item = blockIdx.x; ; item += gridDim.x) {
        few_item it;
        pg_unit u;
        if (!few_find(a, groups, item, &it, &u)) return;
        const bool prefix = it.prefix;
        const int rt = it.rt, kvh = it.kvh, c = it.part, G = a.G;
        const int F = u.n * G;
        const int parts = pg_parts(u.hi - u.lo, prefix ? a.gleast : a.least, prefix ? a.gparts : a.parts);
        // where row `tok`, head h of the item leaves its result
        auto slot = [&](int tok, int h) {
            return prefix ? pg_slot_of(a, a.gpo, a.gpml, tok, h, a.gparts, c)
                          : pg_slot_of(a, a.po, a.pml, (int64_t)it.unit * a.few_rows + tok - u.row, h, a.parts, c);
        };
        const bool direct = !prefix && parts == 1 && u.lo == 0;
        int t0, t1;
        pg_part(u, c, parts, &t0, &t1);
        // this lane's row
        const int f = rt * 16 + n, tok = u.row + f / G, head = kvh * G + f % G;
        const bool valid = f < F;
        const int lim = !valid ? 0 : prefix ? pg_unit_lim<true>(a, u, tok) : pg_unit_lim<false>(a, u, tok);
        // requests first: the page list, the queries, the first tile
        pg_list list = {u.pages, a.b.max_pages, 0, 0};
        list.hold(32 * t0 >> a.pool.page_sh);
        const row_t *src = (const row_t *)a.q.p + (valid ? tok * a.q.rs + head * a.q.hs : u.row * a.q.rs);
        float x[NS][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < NS; i++) pg_load<8>(src + (Q8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g), x[i]);
        pg_f4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        // A tile's keys and values as they are in the pool, requested a tile (of this
        // wave's) ahead: keys while the softmax and the values' products run, values
        // from the end of the products on
        constexpr int NU = HD / (Q8 ? 32 : 16);            // 16-byte units a lane and tile
        uint4 kr[NU], vr[NU];
        pg_f4 ks[2], vs[2], ks1[2], vs1[2];
        const int page_mask = (1 << a.pool.page_sh) - 1;
        bool bad = false, odd = false;
        const uint8_t *blk1;                               // of the next tile
        bool there, there1;
        auto tile_at = [&](int t) {
            const int page = list.get(32 * t >> a.pool.page_sh);
            there1 = page >= 0 && page < a.pool.n_pages;   // (if not, no row sees the tile)
            bad |= !there1;
            blk1 = pg_block(a.pool, there1 ? page : 0, kvh);
        };
        auto load_k = [&](int t) {
            const uint8_t *at = blk1 + (size_t)((32 * t & page_mask) >> 5) * 32 * HD * (Q8 ? 1 : 2) + (g * 32 + n) * 16;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < NU / 2; i++) kr[h * NU / 2 + i] = ldg((const uint4 *)(at + i * 2048 + h * 256));
            if (Q8) {
                const float *sc = (const float *)(blk1 + a.pool.ks_off) + (32 * t & page_mask) + 4 * g;
                const float *sv = (const float *)(blk1 + a.pool.vs_off) + (32 * t & page_mask) + 4 * g;
#pragma unroll
                for (int h = 0; h < 2; h++) { ks1[h] = ldg((const pg_f4 *)(sc + 16 * h)); vs1[h] = ldg((const pg_f4 *)(sv + 16 * h)); }
            }
        };
        auto load_v = [&](int t, const uint8_t *b) {
            const uint8_t *at = b + a.pool.v_off + (size_t)((32 * t & page_mask) >> 5) * 32 * HD * (Q8 ? 1 : 2) + g * HD * (Q8 ? 8 : 16) + n * 16;
#pragma unroll
            for (int i = 0; i < NU; i++) vr[i] = ldg((const uint4 *)(at + i * 256));
        };
        int t = t0 + wave;
        if (t < t1) {
            tile_at(t);
            load_k(t);
            load_v(t, blk1);
        }
        kop qf[NQ][NS];
        float unit = a.scale;
        {
#pragma unroll
            for (int i = 0; i < NS; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[i][j] = valid ? x[i][j] * a.sign : 0.0f;
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
        for (; t < t1; t += 4) {
            there = there1;
#pragma unroll
            for (int h = 0; h < 2; h++) { ks[h] = ks1[h]; vs[h] = vs1[h]; }
            const int tb = 32 * t, nt = t + 4 < t1 ? t + 4 : t;      // (at the end the same tile again, which is near)
            const int vis = there ? lim - tb : 0;                    // positions of the tile below this are visible
            pg_f4 sc[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                sc[h] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < NU / 2; i++) {
                    const uint4 w = kr[h * NU / 2 + i];
                    if (Q8) {
                        kop k0, k1;
                        pg_codes(w.x, w.y, &k0);
                        pg_codes(w.z, w.w, &k1);
#pragma unroll
                        for (int k = NQ - 1; k >= 0; k--) {          // the small term first
                            sc[h] = pg_mma16(k0, qf[k][2 * i], sc[h]);
                            sc[h] = pg_mma16(k1, qf[k][2 * i + 1], sc[h]);
                        }
                    } else {
                        sc[h] = pg_mma16(__builtin_bit_cast(kop, w), qf[0][i], sc[h]);
                    }
                }
            }
            tile_at(nt);
            load_k(nt);
            float p[8];
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = sc[h][i] * (Q8 ? ks[h][i] * unit : unit);
                    p[4 * h + i] = 16 * h + 4 * g + i < vis ? x : -INFINITY;
                    mx = fmaxf(mx, p[4 * h + i]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m, mx);
            if (__any(mn != m)) {
                const float alpha = mn == m ? 1.0f : pg_exp2(m - mn);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;
                m = mn;
            }
            const float ref = mn == -INFINITY ? 0.0f : mn;           // (nothing seen, or keys of -inf)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool see = 16 * h + 4 * g + i < vis;
                    const float e = see ? pg_exp2(p[4 * h + i] - ref) : 0.0f;
                    l += e;
                    p[4 * h + i] = Q8 ? (see ? e * vs[h][i] : 0.0f) : e;
                }
            vop pf[NP];
            pg_split<NP>(p, pf);
            if (!Q8 && __any(valid && vis < 32))
#pragma unroll
                for (int i = 0; i < NU; i++) pg_only_finite<ops::VH>(&vr[i], &odd);
#pragma unroll
            for (int i = 0; i < NU; i++) {
                if (Q8) {
                    vop v0, v1;
                    pg_codes(vr[i].x, vr[i].y, &v0);
                    pg_codes(vr[i].z, vr[i].w, &v1);
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--) {
                        o[2 * i] = pg_mma16(v0, pf[k], o[2 * i]);
                        o[2 * i + 1] = pg_mma16(v1, pf[k], o[2 * i + 1]);
                    }
                } else {
#pragma unroll
                    for (int k = NP - 1; k >= 0; k--) o[i] = pg_mma16(__builtin_bit_cast(vop, vr[i]), pf[k], o[i]);
                }
            }
            load_v(nt, blk1);
        }
        if (bad && lane == 0) pg_report(a.pool, OH_PF_PAGE);
        if (!Q8 && __any(odd)) {
            // the infinities and NaN of this wave's tiles, to the rows that see them:
            // dims 16 d + 4 g + i
            for (int t = t0 + wave; t < t1; t += 4)
                for (int p = 32 * t; p < 32 * t + 32 && p < u.hi; p++) {
                    const int page = u.pages[p >> a.pool.page_sh];
                    if (p >= lim || __any(valid && lim - 32 * t < 32) == 0 || page < 0 || page >= a.pool.n_pages) continue;
                    const typename ops::ve *at = (const typename ops::ve *)(pg_block(a.pool, page, kvh) + a.pool.v_off) + pg_v_at(HD, p & page_mask, 4 * g);
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float y = (float)at[(16 * d + i) * 8];
                            if (!isfinite(y)) o[d][i] += y;
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
        if (!direct && wave == 0 && g == 0 && valid) *slot(tok, head).pml = make_float2(M, L);
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
                    pg_store<4>((row_t *)a.out.p + wtok * a.out.rs + whead * a.out.hs + 64 * q + wd, y);
                } else {
                    *(pg_f4 *)(slot(wtok, whead).po + 64 * q + wd) = (pg_f4){y[0], y[1], y[2], y[3]};
                }
            }
        }
        __syncthreads();                                   // (the next item's results take the same place)
    }
}

// Partial results joined: a wave takes a head of a row and all of its parts, or,
// where there are few heads and many parts (SPLIT), a block's waves every fourth
// part each. A lane
// weighs a part of 64 at a time, so that the loads of the parts' sums wait for no
// exponential.
template <int RT, int HD, bool SPLIT>
__global__ void __launch_bounds__(256)
pattn_join(oh_pattn a) {
    typedef typename pg_elem<RT>::t row_t;
    constexpr int E = HD / 64, W = SPLIT ? 4 : 1, U = SPLIT ? 4 : 8;       // waves a head, parts requested together
    typedef float fe __attribute__((ext_vector_type(E)));
    __shared__ float ys[SPLIT ? 4 : 1][HD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = blockIdx.x;
    const int s = pg_seq_of_wave(a.pool, a.b, r);
    int row0, rows, len;
    if (s < 0 || !pg_seq(a, s, &row0, &rows, &len)) return;
    const int lo = pg_prefix_of(a, s);
    const bool few = rows * a.G <= a.few;
    const int parts = pg_parts(len - lo, few ? a.least : a.mleast, few ? a.parts : a.mparts), gparts = lo ? pg_parts(lo, a.gleast, a.gparts) : 0;
    if (parts == 1 && !gparts) return;                 // written already
    const int np = gparts + parts;
    for (int h = SPLIT ? blockIdx.y : 4 * blockIdx.y + wave; h < a.nh; h += (SPLIT ? 1 : 4) * gridDim.y) {
        // part c of np: the prefix's, then the sequence's own
        auto where = [&](int c) {
            return c < gparts ? pg_slot_of(a, a.gpo, a.gpml, r, h, a.gparts, c)
                   : few      ? pg_slot_of(a, a.po, a.pml, (int64_t)s * a.few_rows + r - row0, h, a.parts, c - gparts)
                              : pg_slot_of(a, a.mpo, a.mpml, r, h, a.mparts, c - gparts);
        };
        float M = -INFINITY;
        for (int c = lane; c < np; c += 64) M = fmaxf(M, where(c).pml->x);
#pragma unroll
        for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
        float L = 0.0f;
        fe y;
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = 0.0f;
        for (int c0 = 0; c0 < np; c0 += 64) {
            const int c = c0 + lane;
            const float2 ml = c < np ? *where(c).pml : make_float2(-INFINITY, 0.0f);
            const float w = ml.x == -INFINITY ? 0.0f : pg_exp2(ml.x - M);  // (0: nothing visible in it)
            if (w != 0.0f) L = fmaf(ml.y, w, L);
            const int n = min(64, np - c0);
            for (int i = SPLIT ? wave : 0; i < n; i += U * W) {            // the last ones again where there are fewer, for nothing
                fe x[U];
#pragma unroll
                for (int j = 0; j < U; j++) x[j] = *(const fe *)(where(min(c0 + i + W * j, np - 1)).po + lane * E);
#pragma unroll
                for (int j = 0; j < U; j++) {
                    const float wi = __shfl(w, (i + W * j) & 63);
                    if (i + W * j >= n) break;
#pragma unroll
                    for (int e = 0; e < E; e++) y[e] = fmaf(x[j][e], wi, y[e]);
                }
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) L += __shfl_xor(L, o);
        const float inv = L > 0.0f || L != L ? 1.0f / L : 0.0f;
        row_t *to = (row_t *)a.out.p + r * a.out.rs + h * a.out.hs;
        if (SPLIT) {
            *(fe *)&ys[wave][lane * E] = y;
            __syncthreads();
            for (int d = threadIdx.x; d < HD; d += 256) to[d] = (row_t)(((ys[0][d] + ys[1][d]) + (ys[2][d] + ys[3][d])) * inv);
            __syncthreads();                           // (ys is the next head's)
        } else {
#pragma unroll
            for (int e = 0; e < E; e++) to[lane * E + e] = (row_t)(y[e] * inv);
        }
    }
}

template <int RT, int CT, int HD>
hipError_t go_few(const oh_pattn *a, hipStream_t st) {
    const int groups = a->gmany ? 0 : a->n_group;
    // as many blocks as there can be items; where that is more than the card
    // holds a few times over they take several
    const int64_t tiles = (std::min((int64_t)a->b.max_new * a->G, (int64_t)a->few) + 15) / 16, gtiles = ((int64_t)a->b.n_rows * a->G + 15) / 16;
    const int64_t items = (tiles * a->b.n_seq * a->parts + gtiles * groups * a->gparts) * a->pool.nkv;
    const unsigned blocks = (unsigned)std::min<int64_t>(items, 1024);
    hipLaunchKernelGGL((pattn_few<RT, CT, HD>), dim3(blocks), dim3(256), 0, st, *a, groups);
    return hipGetLastError();
}
template <int RT, int CT, int HD>
hipError_t go_join(const oh_pattn *a, hipStream_t st) {
    // (a prompt's rows have mostly nothing to join: few blocks for them)
    if (a->b.n_rows > kMaxBlocks) return hipErrorInvalidConfiguration;
    const bool split = (int64_t)a->b.n_rows * a->nh <= 256 && std::max(a->parts, a->mparts) + (a->n_group ? a->gparts : 0) > 32;
    const int64_t blocks = split ? a->nh : (a->nh + 3) / 4, heads = std::min(blocks, std::max<int64_t>(1, (split ? 4096 : 2048) / a->b.n_rows));
    const auto k = split ? pattn_join<RT, HD, true> : pattn_join<RT, HD, false>;
    hipLaunchKernelGGL(k, dim3((unsigned)a->b.n_rows, (unsigned)heads), dim3(256), 0, st, *a);
    return hipGetLastError();
}

} // namespace

extern "C" hipError_t oh_launch_pattn_few(const oh_pattn *a, hipStream_t st) { PG_TYPES(go_few, a, st) }
extern "C" hipError_t oh_launch_pattn_join(const oh_pattn *a, hipStream_t st) { PG_TYPES(go_join, a, st) }
