// oh_kernels_pattn_f32.hip - attention over an 8-bit paged pool for f32 rows,
// where a sequence, or a group that shares a prefix, brings many of them.
//
// As oh_kernels_pattn_many.hip, but a query is two fp16 terms and a weight three
// bf16 ones, so that a key or value read from LDS serves two or three products.
// A wave can then hold 16 rows by 16x16x32 products without waiting for LDS,
// and two waves fit a SIMD's registers at a head dim of 256, where 32 rows a
// wave left one: its waits for LDS, for the step's loads and for the softmax
// were all in the open (403 us for five prompts of 1200 rows at most, 16 heads
// of 256 over 2; 332 so, 290 with 64 positions a step instead of 32: 89 GFLOP of
// scores and sums, 222 in terms). Bound by what the two waves cannot hide from
// each other: their products fill 40% of the matrix cores' time.
#include "oh_pattn_dev.h"
#include <algorithm>

namespace {

constexpr float kBehind = 8.0f;                        // (see oh_kernels_pattn_many.hip)

template <int HD> struct f32_cfg {
    static constexpr int T = 64, NW = 8, H = T / 32;
    static constexpr int TILE = T * HD * 2;            // keys, or values, of a step in LDS, as 16-bit operands
    static constexpr int LDS = 4 * TILE + 2 * (8 * T + 16);   // two of each; scales and whether there is a page
};

template <int HD, bool PREFIX>
__global__ void __launch_bounds__((64 * f32_cfg<HD>::NW), 2)
pattn_f32(oh_pattn a, int pieces) {
    typedef pg_ops<OH_PT_F32, OH_PT_Q8> ops;
    typedef typename ops::kv kop;
    typedef typename ops::vv vop;
    typedef f32_cfg<HD> cfg;
    constexpr int NW = cfg::NW, T = cfg::T, H = cfg::H, TILE = cfg::TILE, NT = 64 * NW, TR = 16 * NW;
    constexpr int NQ = ops::NQ, NP = 3, NS = HD / 32, ND = HD / 16;
    extern __shared__ __align__(16) uint8_t lds[];
    uint8_t *const ldk = lds, *const ldv = lds + 2 * TILE;
    float *const lds_s = (float *)(lds + 4 * TILE);    // [2][keys' T, values' T]
    int *const lds_ok = (int *)(lds_s + 4 * T);        // [2][2]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
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
    const int64_t f = from + wave * 16 + n;
    const int tok = (int)(f / G), head = kvh * G + (int)(f % G);
    const bool valid = f < to;
    // what the lane's row sees of the part; the last position that some row of the block sees
    int lim = valid ? min(pg_unit_lim<PREFIX>(a, u, tok), 32 * t1) : 0;
    int blim = lim;
#pragma unroll
    for (int o = 32; o; o >>= 1) blim = max(blim, __shfl_xor(blim, o));
    __shared__ int wl[NW];
    if (lane == 0) wl[wave] = blim;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) blim = max(blim, wl[w]);
    if (!valid) lim = 1 << 30;                         // (no row: nothing to hide)
    blim = __builtin_amdgcn_readfirstlane(blim);
    const int p0 = 32 * t0, N = blim > p0 ? (blim - p0 + T - 1) / T : 0;       // steps

    kop qf[NQ][NS];
    float unit = a.scale;                              // of the row's scores as they come out of the products
    pg_f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    // ---- a step's keys and values: the 32-position tiles' bytes as they are in
    // the pool, 16 a thread at a time; where there is no page (behind the last
    // position, or a bad index) page 0's, which no row looks at
    constexpr int KB = 32 * HD, NL = H * KB > 16 * NT ? H * KB / (16 * NT) : 1;      // bytes of a tile; loads per thread
    static_assert(H * KB == NL * 16 * NT || NL == 1, "whole loads");
    const bool loads = NL > 1 || 16 * tid < H * KB;    // (a head of 64 keeps half of the threads)
    uint4 kr[NL] = {}, vr[NL] = {};
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
    auto fetch = [&](pg_list &list, int pos, uint32_t plane, uint4 (&r)[NL], bool keys = false) {
        const uint8_t *at[H];
        bool there[H];
#pragma unroll
        for (int h = 0; h < H; h++) at[h] = tile_at(list, pos + 32 * h, &there[h]);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int b = 16 * (tid + NT * i);
            if (loads) r[i] = ldg((const uint4 *)((b < KB ? at[0] : at[H - 1]) + plane + b % KB));
        }
        if (keys)
#pragma unroll
            for (int h = 0; h < H; h++) ok[h] = there[h];
        if (keys && tid < 2 * T) {
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
            const int e = tid + NT * i, h = 16 * e / KB, x = e % (KB / 16), ch = x >> 5, sl = x & 31;        // 16 dims ch of position sl
            if (!loads) continue;
            kop *to = (kop *)(ldk + b * TILE + h * 64 * HD) + 2 * ch * 32 + sl;
            kop k0, k1;
            pg_codes(kr[i].x, kr[i].y, &k0);
            pg_codes(kr[i].z, kr[i].w, &k1);
            to[0] = k0;
            to[32] = k1;
        }
        if (tid < 2 * T) lds_s[b * 2 * T + tid] = scl;
        if (tid == 0)
#pragma unroll
            for (int h = 0; h < H; h++) lds_ok[2 * b + h] = ok[h];
    };
    auto stage_v = [&](int b) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            if (!loads) continue;
            vop v0, v1;
            pg_codes(vr[i].x, vr[i].y, &v0);
            pg_codes(vr[i].z, vr[i].w, &v1);
            vop *to = (vop *)(ldv + b * TILE) + 2 * (tid + NT * i);
            to[0] = v0;
            to[1] = v1;
        }
    };

    // ---- products: S^T of step t, and O^T of the step before
    pg_f4 s[H][2];                                     // positions 32 h + 16 u + 4 g + i of row n
    vop pf[NP][H];
    auto scores = [&](int t) {
        const kop *at = (const kop *)(ldk + (t & 1) * TILE) + g * 32 + n;
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                s[h][u] = (pg_f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const kop kf = at[h * 4 * HD + i * 128 + 16 * u];
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--) s[h][u] = pg_mma16(kf, qf[k][i], s[h][u]);       // the small term first
                }
            }
    };
    auto values = [&](int t) {
        const vop *at = (const vop *)(ldv + (t & 1) * TILE) + g * HD + n;
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const vop vf = at[h * 4 * HD + 16 * d];
#pragma unroll
                for (int x = NP - 1; x >= 0; x--) o[d] = pg_mma16(vf, pf[x][h], o[d]);
            }
    };
    auto softmax = [&](int t) {
        const int pos = p0 + t * T, b = t & 1;
        const float *ks = lds_s + b * 2 * T, *vs = ks + T;
        float mx = -INFINITY;
        bool see[H][2][4];
#pragma unroll
        for (int h = 0; h < H; h++) {
            // positions of a tile below this are visible to the row
            const int vis = (__builtin_amdgcn_readfirstlane(lds_ok[2 * b + h]) ? lim - pos - 32 * h : 0) - 4 * g;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const pg_f4 kk = *(const pg_f4 *)(ks + 32 * h + 16 * u + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    see[h][u][i] = 16 * u + i < vis;
                    s[h][u][i] = see[h][u][i] ? s[h][u][i] * (kk[i] * unit) : -INFINITY;
                    mx = fmaxf(mx, s[h][u][i]);
                }
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m + kBehind)) {
            const float mn = fmaxf(m, mx), alpha = mn == m ? 1.0f : pg_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.0f : m;   // (nothing seen yet, or keys of -inf)
#pragma unroll
        for (int h = 0; h < H; h++) {
            float p[8];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const pg_f4 vv = *(const pg_f4 *)(vs + 32 * h + 16 * u + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = pg_exp2(s[h][u][i] - ref);
                    l += e;
                    p[4 * u + i] = see[h][u][i] ? e * vv[i] : 0.0f;        // (a hidden scale may be anything)
                }
            }
            vop w[NP];
            pg_split<NP>(p, w);
#pragma unroll
            for (int x = 0; x < NP; x++) pf[x][h] = w[x];
        }
    };

    // Loads run one step past the end, on page 0's bytes and for nothing: no branch
    // splits the loop's registers.
    fetch(lk, p0, 0, kr, true);
    fetch(lv, p0, a.pool.v_off, vr);
    {
        float x[NS][8], top = 0.0f;
        const float *src = (const float *)a.q.p + (valid ? tok * a.q.rs + head * a.q.hs : u.row * a.q.rs) + 8 * g;
#pragma unroll
        for (int i = 0; i < NS; i++)
            pg_load<8>(src + 32 * i, x[i]);
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = valid ? x[i][j] * a.sign : 0.0f;
                top = fmaxf(top, fabsf(x[i][j]));
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        const int e = pg_row_exp(fmaxf(top, __shfl_xor(top, 32)));
        unit = ldexpf(unit, -e);
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] = ldexpf(x[i][j], e);
#pragma unroll
        for (int i = 0; i < NS; i++) {
            kop t[NQ];
            pg_split<NQ>(x[i], t);
#pragma unroll
            for (int k = 0; k < NQ; k++) qf[k][i] = t[k];
        }
    }
    stage_k(0);
    stage_v(0);
    __syncthreads();
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
    if (bad && tid == 0) pg_report(a.pool, OH_PF_PAGE);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (l != l) m = fmaxf(m, 0.0f);                    // a NaN score stays one
    if (!valid) return;
    // lane n's row: dims 16 d + 4 g .. + 3
    if (direct) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        float *out = (float *)a.out.p + tok * a.out.rs + head * a.out.hs + 4 * g;
#pragma unroll
        for (int d = 0; d < ND; d++) *(pg_f4 *)(out + 16 * d) = o[d] * inv;
    } else {
        const pg_slot at = PREFIX ? pg_slot_of(a, a.gpo, a.gpml, tok, head, a.gparts, c) : pg_slot_of(a, a.mpo, a.mpml, tok, head, a.mparts, c);
        if (g == 0) *at.pml = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < ND; d++) *(pg_f4 *)(at.po + 16 * d + 4 * g) = o[d];
    }
}

template <int HD, bool PREFIX>
hipError_t launch(const oh_pattn *a, int units, int parts, hipStream_t st) {
    constexpr int NW = f32_cfg<HD>::NW, lds = f32_cfg<HD>::LDS;
    int64_t blocks;
    const int64_t pieces = pg_pieces(a, units, 16 * NW, &blocks);
    if (blocks > kMaxBlocks / 2) return hipErrorInvalidConfiguration;
    const auto k = pattn_f32<HD, PREFIX>;
    static std::atomic<uint64_t> asked{0};
    const hipError_t e = pg_allow_lds((const void *)k, lds, &asked);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)blocks, parts), dim3(64 * NW), lds, st, *a, (int)pieces);
    return hipGetLastError();
}
template <int HD>
hipError_t go(const oh_pattn *a, hipStream_t st) {
    hipError_t e = hipSuccess;
    if (a->n_group && a->gmany) e = launch<HD, true>(a, a->n_group, a->gparts, st);
    if (e == hipSuccess && a->many >= 0) e = launch<HD, false>(a, a->b.n_seq, a->mparts, st);
    return e;
}

} // namespace

extern "C" hipError_t oh_launch_pattn_f32(const oh_pattn *a, hipStream_t st) {
    switch (a->pool.hd) {
    case 64: return go<64>(a, st);
    case 128: return go<128>(a, st);
    default: return go<256>(a, st);
    }
}
