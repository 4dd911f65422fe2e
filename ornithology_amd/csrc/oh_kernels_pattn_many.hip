// oh_kernels_pattn_many.hip - attention over a paged pool where a sequence, or a
// group that shares a prefix, brings many rows.
//
// A block of NW waves takes 32 NW rows (row, head of one kv head's group) and
// a part of the positions, 64 at a time: the tile's keys and values go through
// LDS once for all waves, as matrix operands in the pool's order (codes as
// bf16), in two buffers, the next tile's loads in flight during this one's
// products. A wave holds 32 rows: S^T = K Q^T by 32x32x16 products (lane n =
// lane & 31 holds row n's scores of half the positions), the softmax, and
// O^T += V^T P^T with the probabilities where they are.
#include "oh_pattn_dev.h"
#include <algorithm>

namespace {

constexpr int kT = 64;                                 // positions per step
// A running maximum may be this much (a factor of 2^8) behind the largest
// score: weights stay far inside every operand type, 32-bit sums lose nothing,
// and the accumulators are scaled a few times a row instead of at every step
constexpr float kBehind = 8.0f;

template <int HD> constexpr int tile_bytes() { return kT * HD * 2; }          // keys, or values, as 16-bit operands
template <int CT, int HD> constexpr int buf_bytes() { return 2 * tile_bytes<HD>() + (CT == OH_PT_Q8 ? 8 * kT : 0); }
// waves a block: eight where two fit a SIMD's registers and a step has a load for each thread
template <int RT, int CT, int HD> constexpr int waves() { return RT == OH_PT_F32 || HD == 256 || (CT == OH_PT_Q8 && HD == 64) ? 4 : 8; }

template <int RT, int CT, int HD, bool PREFIX, int NW = waves<RT, CT, HD>()>
__global__ void __launch_bounds__(64 * NW)
pattn_many(oh_pattn a, int tiles_of_rows) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_op<CT>::v opv;
    typedef typename pg_op<CT>::e ope;
    constexpr bool Q8 = CT == OH_PT_Q8;
    constexpr int NT = 64 * NW, TR = 32 * NW;
    constexpr int NQ = pg_nq<RT, CT>(), NP = RT == OH_PT_F32 ? 3 : RT == OH_PT_F16 && Q8 ? 2 : 1, NS = HD / 16, ND = HD / 32;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, hf = lane >> 5;
    // long rows first: the last row tiles of a prompt see the most
    const int unit = (int)blockIdx.x / tiles_of_rows, rt = tiles_of_rows - 1 - (int)blockIdx.x % tiles_of_rows;
    const int kvh = blockIdx.y, c = blockIdx.z;
    pg_unit u;
    if (!pg_unit_at<PREFIX>(a, unit, &u)) return;
    const int G = a.G, F = u.n * G;
    if (rt * TR >= F || (!PREFIX && F <= a.many) || (PREFIX && !u.hi)) return;
    const int parts = pg_parts(u.hi - u.lo, PREFIX ? a.gparts : a.mparts);
    if (c >= parts) return;
    const int64_t pc = PREFIX ? c : a.gparts + c;
    const bool direct = !PREFIX && parts == 1 && u.lo == 0;
    int t0, t1;
    pg_part(u, c, parts, &t0, &t1);
    const int f = rt * TR + wave * 32 + n, tok = u.row + f / G, head = kvh * G + f % G;
    const bool valid = f < F;
    int lim = valid ? pg_unit_lim<PREFIX>(a, u, tok) : 0;
    // the block's and the wave's last visible position
    int wlim = lim;
#pragma unroll
    for (int o = 32; o; o >>= 1) wlim = max(wlim, __shfl_xor(wlim, o));
    __shared__ int wl[NW];
    if (lane == 0) wl[wave] = wlim;
    __syncthreads();
    int blim = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) blim = max(blim, wl[w]);
    if (!valid) lim = 1 << 30;                         // (no row: nothing to hide)
    const int p0 = 32 * t0, p1 = min(32 * t1, blim);   // positions [p0, p1), in steps of kT

    opv qf[NQ][NS];
#pragma unroll
    for (int i = 0; i < NS; i++) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = 0.0f;
        if (valid) {
            const row_t *src = (const row_t *)a.q.p + tok * a.q.rs + head * a.q.hs + 16 * i + 8 * hf;
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (float)src[j] * a.sign;
        }
        opv t[NQ];
        pg_split<NQ>(x, t);
#pragma unroll
        for (int k = 0; k < NQ; k++) qf[k][i] = t[k];
    }
    pg_f16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // A step's keys and values: the two 32-position tiles' bytes, 16 a thread
    // at a time; where there is no page (behind the last position, or a bad
    // index) the block of page 0, which no row looks at
    constexpr int KB = 32 * HD * (Q8 ? 1 : 2), NL = 2 * KB / 16 / NT;          // bytes of a tile; loads per thread
    static_assert(2 * KB == NL * 16 * NT, "whole loads");
    uint4 kr[NL], vr[NL];
    float scl = 0.0f;
    const int page_mask = (1 << a.pool.page_sh) - 1;
    auto tile_at = [&](int pos, bool *ok) -> const uint8_t * {
        int page = -1;
        if (pos < p1) {
            page = u.pages[pos >> a.pool.page_sh];
            if (page < 0 || page >= a.pool.n_pages) { page = -1; if (tid == 0) pg_report(a.pool, OH_PF_PAGE); }
        }
        *ok = page >= 0;
        return pg_block(a.pool, page < 0 ? 0 : page, kvh);
    };
    const uint8_t *blk[2];
    bool ok[2];
    auto fetch = [&](int pos) {
#pragma unroll
        for (int h = 0; h < 2; h++) blk[h] = tile_at(pos + 32 * h, &ok[h]);
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int b = (tid + NT * i) * 16, h = b / KB, off = b % KB;
            const uint8_t *from = blk[h] + ((pos + 32 * h) & page_mask) / 32 * KB + off;
            kr[i] = *(const uint4 *)from;
            vr[i] = *(const uint4 *)(from + a.pool.v_off);
        }
        if (Q8 && tid < 2 * kT) {
            const int x = tid & (kT - 1), h = x >> 5;
            scl = *(const float *)(blk[h] + (tid < kT ? a.pool.ks_off : a.pool.vs_off) + 4 * ((pos + x) & page_mask));
        }
    };
    // into buffer b: K units (8 dims of one position) at (dim / 8 * 32 +
    // position) * 16 per tile, V units (8 positions of one dim) at (group * HD + dim) * 16
    auto stage = [&](int b) {
        uint8_t *K = lds + b * buf_bytes<CT, HD>(), *V = K + tile_bytes<HD>();
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int e = tid + NT * i;
            if (Q8) {
                const int h = e * 16 / KB, x = e % (KB / 16), ch = x >> 5, sl = x & 31;      // 16 dims ch of position sl
                uint8_t *kt = K + h * 64 * HD;
                *(pg_b8 *)(kt + ((2 * ch) * 32 + sl) * 16) = pg_codes(kr[i].x, kr[i].y);
                *(pg_b8 *)(kt + ((2 * ch + 1) * 32 + sl) * 16) = pg_codes(kr[i].z, kr[i].w);
                *(pg_b8 *)(V + e * 32) = pg_codes(vr[i].x, vr[i].y);
                *(pg_b8 *)(V + e * 32 + 16) = pg_codes(vr[i].z, vr[i].w);
            } else {
                *(uint4 *)(K + e * 16) = kr[i];
                *(uint4 *)(V + e * 16) = vr[i];
            }
        }
        if (Q8 && tid < 2 * kT) *(float *)(K + 2 * tile_bytes<HD>() + 4 * tid) = tid < kT ? scl * a.scale : scl;
    };

    bool now[2];
    if (p0 < p1) {
        fetch(p0);
        stage(0);
    }
    int b = 0;
    for (int pos = p0; pos < p1; pos += kT, b ^= 1) {
        now[0] = ok[0]; now[1] = ok[1];
        __syncthreads();                               // buffer b is whole, the other one free
        const bool more = pos + kT < p1;
        if (more) fetch(pos + kT);
        if (pos < wlim) {
            const uint8_t *K = lds + b * buf_bytes<CT, HD>(), *V = K + tile_bytes<HD>();
            const float *ks = (const float *)(K + 2 * tile_bytes<HD>()), *vs = ks + kT;
            pg_f16 s[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int v = 0; v < 16; v++) s[h][v] = 0.0f;
                // operand row n is position 16 (n >> 3 & 1) + 8 (n >> 4) + (n & 7), so that
                // a lane's 8 scores of a product are one unit of the values
                const uint8_t *at = K + h * 64 * HD + (hf * 32 + 16 * ((n >> 3) & 1) + 8 * (n >> 4) + (n & 7)) * 16;
#pragma unroll
                for (int i = 0; i < NS; i++) {
                    const opv kf = *(const opv *)(at + i * 1024);
#pragma unroll
                    for (int k = NQ - 1; k >= 0; k--) s[h] = pg_mma32(kf, qf[k][i], s[h]);
                }
            }
            // scores in units of log2(e), those that the row does not see at -inf
            const int vis0 = now[0] ? lim - pos : 0, vis1 = now[1] ? lim - pos - 32 : 0;     // visible ones of each tile
            const bool part = __any(vis0 < 32 || vis1 < 32);
            if (Q8) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const pg_f4 kk = *(const pg_f4 *)(ks + 32 * h + 16 * (q & 1) + 8 * (q >> 1) + 4 * hf);
#pragma unroll
                        for (int i = 0; i < 4; i++) s[h][4 * q + i] *= kk[i];
                    }
            }
            if (part) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int v = 0; v < 16; v++)
                        if (16 * ((v >> 2) & 1) + 8 * (v >> 3) + 4 * hf + (v & 3) >= (h ? vis1 : vis0)) s[h][v] = -INFINITY;
            }
            const float unit_scale = Q8 ? 1.0f : a.scale;        // (codes: in their scales)
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int v = 0; v < 16; v++) mx = fmaxf(mx, s[h][v]);
            mx = fmaxf(mx, __shfl_xor(mx, 32)) * unit_scale;
            if (__any(mx > m + kBehind)) {
                const float mn = fmaxf(m, mx), alpha = mn == m ? 1.0f : pg_exp2(m - mn);
                m = mn;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) o[d][v] *= alpha;
            }
            const float ref = m == -INFINITY ? 0.0f : m;         // (nothing seen yet, or keys of -inf)
            opv pf[NP][2][2];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    float p[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        p[j] = pg_exp2(fmaf(s[h][8 * k + j], unit_scale, -ref));
                        l += p[j];
                    }
                    if (Q8) {
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const pg_f4 vv = *(const pg_f4 *)(vs + 32 * h + 16 * q + 8 * k + 4 * hf);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                // (a scale that the row does not see may be anything)
                                const bool see = !part || 16 * q + 8 * k + 4 * hf + i < (h ? vis1 : vis0);
                                p[4 * q + i] = see ? p[4 * q + i] * vv[i] : 0.0f;
                            }
                        }
                    }
                    opv t[NP];
                    pg_split<NP>(p, t);
#pragma unroll
                    for (int x = 0; x < NP; x++) pf[x][h][k] = t[x];
                }
            // In a tile that some row sees a part of, values that are hidden from it
            // may be infinite or NaN, and 0 times that is NaN
            bool odd = false;
            if (!Q8 && part) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const opv vf = *(const opv *)(V + h * 64 * HD + ((2 * k + hf) * HD + 32 * d + n) * 16);
#pragma unroll
                            for (int j = 0; j < 8; j++) odd |= !isfinite((float)vf[j]);
                        }
                odd = __any(odd);
            }
            if (!odd) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int d = 0; d < ND; d++) {
                            const opv vf = *(const opv *)(V + h * 64 * HD + ((2 * k + hf) * HD + 32 * d + n) * 16);
#pragma unroll
                            for (int x = NP - 1; x >= 0; x--) o[d] = pg_mma32(vf, pf[x][h][k], o[d]);
                        }
            } else {
                // row by row, with what the row does not see as zero
#pragma unroll 1
                for (int r = 0; r < 32; r++) {
                    const int v0 = __shfl(vis0, r), v1 = __shfl(vis1, r);
                    asm volatile("" ::: "memory");               // (the values are read where they are used, not kept)
#pragma unroll
                    for (int d = 0; d < ND; d++) {
                        pg_f16 y;
#pragma unroll
                        for (int v = 0; v < 16; v++) y[v] = 0.0f;
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int k = 0; k < 2; k++) {
                                opv vf = *(const opv *)(V + h * 64 * HD + ((2 * k + hf) * HD + 32 * d + n) * 16);
#pragma unroll
                                for (int j = 0; j < 8; j++)
                                    if (16 * (j >> 2) + 8 * k + 4 * hf + (j & 3) >= (h ? v1 : v0)) vf[j] = (ope)0.0f;
#pragma unroll
                                for (int x = NP - 1; x >= 0; x--) y = pg_mma32(vf, pf[x][h][k], y);
                            }
                        if (n == r)
#pragma unroll
                            for (int v = 0; v < 16; v++) o[d][v] += y[v];
                    }
                }
            }
        }
        if (more) stage(b ^ 1);
    }
    l += __shfl_xor(l, 32);
    if (l != l) m = fmaxf(m, 0.0f);                    // a NaN score stays one
    if (!valid) return;
    // lane n's row: dims 32 d + 8 q + 4 hf .. + 3
    if (direct) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        row_t *to = (row_t *)a.out.p + tok * a.out.rs + head * a.out.hs + 4 * hf;
        typedef row_t r4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                r4 y;
#pragma unroll
                for (int i = 0; i < 4; i++) y[i] = (row_t)(o[d][4 * q + i] * inv);
                *(r4 *)(to + 32 * d + 8 * q) = y;
            }
    } else {
        const int64_t at = ((int64_t)tok * a.nh + head) * (a.gparts + a.sparts) + pc;
        if (hf == 0) a.pml[at] = make_float2(m, l);
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *(pg_f4 *)(a.po + at * HD + 32 * d + 8 * q + 4 * hf) = (pg_f4){o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]};
    }
}

template <int RT, int CT, int HD, bool PREFIX>
hipError_t launch(const oh_pattn *a, int64_t rows, int units, int parts, hipStream_t st) {
    constexpr int NW = waves<RT, CT, HD>(), lds = 2 * buf_bytes<CT, HD>();
    const int64_t tiles = (rows * a->G + 32 * NW - 1) / (32 * NW);
    if (tiles * units > kMaxBlocks / 2) return hipErrorInvalidConfiguration;
    const auto k = pattn_many<RT, CT, HD, PREFIX>;
    hipError_t e = hipFuncSetAttribute((const void *)k, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k, dim3((unsigned)(tiles * units), a->pool.nkv, parts), dim3(64 * NW), lds, st, *a, (int)tiles);
    return hipGetLastError();
}
template <int RT, int CT, int HD>
hipError_t go_many(const oh_pattn *a, hipStream_t st) {
    hipError_t e = hipSuccess;
    if (a->n_group && a->gmany) e = launch<RT, CT, HD, true>(a, a->b.n_rows, a->n_group, a->gparts, st);
    if (e == hipSuccess && a->many >= 0) e = launch<RT, CT, HD, false>(a, a->b.max_new, a->b.n_seq, a->mparts, st);
    return e;
}

} // namespace

extern "C" hipError_t oh_launch_pattn_many(const oh_pattn *a, hipStream_t st) { PG_TYPES(go_many, a, st) }
