// oh_kernels_paged.hip - rows into a paged pool and out of it.
//
// Append: per (row, head) of the keys, x / sqrt(mean(x^2) + eps) * w if there is
// a norm, the rotation of pairs (i, i + r/2) by the angle P * theta^(-2i/r),
// and the store, as 16-bit values or as codes rint(x * 127 / max|x|) with the
// scale max|x| / 127; values without norm and rotation; queries with both, to
// q_out. Bound by memory: rows are read once and written once, so a lane
// holds 8 values of a head (16 bytes of a 16-bit row), and a row's sines and
// cosines stay in its lanes' registers for all of the heads that a block takes
// (8191 f32 rows, 16 query and 2 key heads of 256: 67 us, 4.5 TB/s; one row 7 us,
// the chain of its loads).
#include "oh_paged_dev.h"
#include <algorithm>

namespace {

// (cos, sin) of frequency i at `pos`: the angles of the 1024-step and of the
// rest are added in 64 bits and rounded once, so far positions are as exact
// as near ones
OH_DEV float2 rope_cs(const oh_pool &p, int pos, int i) {
    const int half = p.rope_dim / 2;
    const double2 a = p.rope_hi[(size_t)(pos / kRopeStep) * half + i], b = p.rope_lo[(size_t)(pos % kRopeStep) * half + i];
    return make_float2((float)(a.x * b.x - a.y * b.y), (float)(a.y * b.x + a.x * b.y));
}

// the tables: entries [0, steps) of kRopeStep positions each, then those within one
__global__ void __launch_bounds__(256) rope_tables(double2 *t, int steps, int half, double theta) {
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int k = (int)(x / half), i = (int)(x % half);
    if (k >= steps + kRopeStep) return;
    const double angle = (double)(k < steps ? (int64_t)k * kRopeStep : k - steps) * pow(theta, -(double)i / half);
    t[x] = make_double2(cos(angle), sin(angle));
}

// the lanes of one head of one row
template <int HD> constexpr int head_lanes() { return HD / 8; }
template <int L, class F>
OH_DEV float lanes_fold(float v, F f) {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) v = f(v, __shfl_xor(v, o));
    return v;
}

// The place of row r: its sequence and position; false for padding and for rows
// that no sequence owns. All lanes of a wave call it; `row`: of this lane.
struct place { int s, pos; };
OH_DEV bool place_of(const oh_pool &p, const oh_pbatch &b, int row, place *o) {
    if (row >= b.n_rows) return false;
    o->s = pg_seq_of(p, b, row);
    if (o->s < 0) return false;
    o->pos = b.len[o->s] - (b.start[o->s + 1] - row);
    return o->pos >= 0;
}
// a position's page block for a head, and its slot in the page; null (and reported) if there is none
OH_DEV uint8_t *slot_of(const oh_pool &p, const oh_pbatch &b, const place &at, int head, int *slot) {
    const int pi = at.pos >> p.page_sh;
    if (pi >= b.max_pages) { pg_report(p, OH_PF_BATCH); return nullptr; }
    const int page = b.table[(size_t)at.s * b.max_pages + pi];
    if (page < 0 || page >= p.n_pages) { pg_report(p, OH_PF_PAGE); return nullptr; }
    *slot = at.pos & ((1 << p.page_sh) - 1);
    return pg_block(p, page, head);
}

// the 8 codes of a lane's values, and the head's scale
template <int HD>
OH_DEV float codes_of(float (&y)[8]) {
    float am = 0.0f;
    bool nan = false;                                  // a NaN is in no code: it goes into the scale
#pragma unroll
    for (int j = 0; j < 8; j++) { am = fmaxf(am, fabsf(y[j])); nan |= y[j] != y[j]; }
    if (nan) am = NAN;
    am = lanes_fold<head_lanes<HD>()>(am, [](float a, float b) { return a != a || b != b ? NAN : fmaxf(a, b); });
    // (below 2^-121 127 / max is infinite, and 0 times that no code: such heads are raised first)
    const float up = am < 0x1p-100f ? 0x1p100f : 1.0f, iv = am > 0.0f ? 127.0f / (am * up) : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] = fminf(fmaxf(rintf(y[j] * up * iv), -127.0f), 127.0f);
    return am / 127.0f;
}
OH_DEV uint2 pack_codes(const float (&y)[8]) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++) w[j >> 2] |= ((uint32_t)(int)y[j] & 0xffu) << (8 * (j & 3));
    return make_uint2(w[0], w[1]);
}

// Queries and keys: a block takes as many rows as its lanes hold heads, and
// `heads` of the nh + nkv heads of each.
template <int RT, int CT, int HD>
OH_DEV void append_qk(const oh_pappend &a, int block, int heads) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    constexpr int L = head_lanes<HD>(), R = 256 / L, U = 4;       // lanes a head, rows a block, heads requested together
    __shared__ float xs[256 * 8];
    const int tid = threadIdx.x, sub = tid % L, d0 = 8 * sub;
    const int nq = a.q.p ? a.nh : 0, all = nq + a.pool.nkv, groups = (all + heads - 1) / heads;
    const int r = block / groups * R + tid / L, h0 = block % groups * heads, h1 = min(h0 + heads, all);
    place at;
    bool ok = place_of(a.pool, a.b, r, &at);
    const int half = a.pool.rope_dim / 2;
    // the other value of a pair: 8 values at a time from another lane where r/2 is a
    // multiple of 8, else one by one
    const bool whole = half % 8 == 0;
    const int other = ((int)(tid & 63) + (d0 < half ? half / 8 : -(half / 8))) & 63;
    float2 cs[8];
#pragma unroll
    for (int j = 0; j < 8; j++) cs[j] = make_float2(1.0f, 0.0f);
    if (half && ok) {
        int pos[4];
#pragma unroll
        for (int x = 0; x < 4; x++) {
            pos[x] = x >= a.axes ? 0 : a.pos ? a.pos[x * a.pos_stride + r] : at.pos;
            if (pos[x] < 0 || pos[x] >= a.pool.max_pos) ok = false;
        }
        if (!ok) {
            if (sub == 0) pg_report(a.pool, OH_PF_POSITION);
        } else if (d0 < (whole ? half : 2 * half)) {             // (whole: a pair's other lane gets its own from here)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int d = d0 + j, i = d < half ? d : d - half;
                if (d >= 2 * half) continue;
                const int x = a.axes > 1 ? a.pool.rope_axis[i] : 0;
                cs[j] = rope_cs(a.pool, x == 0 ? pos[0] : x == 1 ? pos[1] : x == 2 ? pos[2] : pos[3], i);
            }
        }
    }
    if (whole)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = __shfl(cs[j].x, other), y = __shfl(cs[j].y, other);
            if (d0 >= half && d0 < 2 * half) cs[j] = make_float2(x, y);
        }
    for (int hb = h0; hb < h1; hb += U) {
        float y[U][8];
        if (ok) {
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int h = min(hb + k, h1 - 1);
                const oh_prows &in = h < nq ? a.q : a.k;
                pg_load<8>((const row_t *)in.p + r * in.rs + (h < nq ? h : h - nq) * in.hs + d0, y[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int h = hb + k;
            if (h >= h1) break;
            const float *w = h < nq ? a.q_norm : a.k_norm;
            if (w) {
                float ss = 0.0f, wt[8];
                pg_load<8>(w + d0, wt);
#pragma unroll
                for (int j = 0; j < 8; j++) ss = fmaf(y[k][j], y[k][j], ss);
                ss = lanes_fold<L>(ss, [](float x, float y) { return x + y; });
                const float inv = 1.0f / sqrtf(ss / HD + a.eps);
#pragma unroll
                for (int j = 0; j < 8; j++) y[k][j] = y[k][j] * inv * wt[j];
            }
            if (half) {
                float o[8];
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = __shfl(y[k][j], other);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) xs[tid * 8 + j] = y[k][j];
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int d = d0 + j;
                        o[j] = d < 2 * half ? xs[(tid - sub) * 8 + (d < half ? d + half : d - half)] : 0.0f;
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int d = d0 + j;
                    if (d < 2 * half) y[k][j] = d < half ? y[k][j] * cs[j].x - o[j] * cs[j].y : o[j] * cs[j].y + y[k][j] * cs[j].x;
                }
            }
            if (h < nq) {
                if (ok) pg_store<8>((row_t *)a.q_out.p + r * a.q_out.rs + h * a.q_out.hs + d0, y[k]);
                continue;
            }
            const float sc = CT == OH_PT_Q8 ? codes_of<HD>(y[k]) : 0.0f;
            int slot;
            uint8_t *blk = ok ? slot_of(a.pool, a.b, at, h - nq, &slot) : nullptr;
            if (!blk) continue;
            cache_t *to = (cache_t *)blk + pg_k_at<CT>(HD, slot, d0);
            if (CT == OH_PT_Q8) {
                *(uint2 *)to = pack_codes(y[k]);
                if (sub == 0) *(float *)(blk + a.pool.ks_off + 4 * slot) = sc;
            } else {
                pg_store<8>(to, y[k]);
            }
        }
    }
}

// Values: a block takes `span` rows (1 or 32) of one head, stretch by stretch of
// those that share a tile of 32 positions, puts them in the tile's order in LDS
// and stores that: whole units where all of their 8 positions are new.
template <int RT, int CT, int HD>
OH_DEV void append_v(const oh_pappend &a, int block, int span) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    constexpr int L = head_lanes<HD>(), R = 256 / L, NR = 32 / R > 0 ? 32 / R : 1;
    typedef cache_t unit_t __attribute__((ext_vector_type(8)));
    __shared__ __align__(16) cache_t tile[32 * HD];
    const int tid = threadIdx.x, sub = tid % L, d0 = 8 * sub, head = block % a.pool.nkv;
    const int r1 = min(block / a.pool.nkv * span + span, a.b.n_rows);
    // units of the tile that are 8 lanes apart would meet in the same LDS banks
    auto at_unit = [](int u) { return u ^ ((u >> 3) & 7); };
    for (int r = block / a.pool.nkv * span; r < r1;) {
        const int s = pg_seq_of(a.pool, a.b, r);
        if (s < 0) { r++; continue; }
        place at = {s, a.b.len[s] - (a.b.start[s + 1] - r)};
        const int left = min(a.b.start[s + 1], r1) - r;          // of the sequence, here
        if (at.pos < 0) { r += at.pos <= -left ? left : -at.pos; continue; }
        const int n = min(left, 32 - (at.pos & 31)), r0 = r;
        r += n;
        int slot;
        uint8_t *blk = slot_of(a.pool, a.b, at, head, &slot);
        if (!blk) continue;
        float y[NR][8];
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int i = min(k * R + tid / L, n - 1);
            pg_load<8>((const row_t *)a.v.p + (int64_t)(r0 + i) * a.v.rs + head * a.v.hs + d0, y[k]);
        }
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int i = k * R + tid / L, sl = (slot & 31) + i;
            const float sc = CT == OH_PT_Q8 ? codes_of<HD>(y[k]) : 0.0f;
            if (i >= n) continue;
            if (CT == OH_PT_Q8 && sub == 0) *(float *)(blk + a.pool.vs_off + 4 * (slot + i)) = sc;
#pragma unroll
            for (int j = 0; j < 8; j++)
                tile[at_unit(((sl >> 2) & 3) * HD + d0 + j) * 8 + 4 * (sl >> 4) + (sl & 3)] = CT == OH_PT_Q8 ? (cache_t)(int)y[k][j] : (cache_t)y[k][j];
        }
        __syncthreads();
        const uint32_t fresh = (uint32_t)((((uint64_t)1 << n) - 1) << (slot & 31));
        cache_t *to = (cache_t *)(blk + a.pool.v_off) + (slot >> 5) * 32 * HD;
#pragma unroll
        for (int k = 0; k < 4 * HD / 256; k++) {
            const int u = tid + 256 * k, g = u / HD;
            const uint32_t mine = ((fresh >> (4 * g)) & 15) | ((fresh >> (16 + 4 * g)) & 15) << 4;
            if (!mine) continue;
            const unit_t x = *(const unit_t *)(tile + at_unit(u) * 8);
            if (mine == 255) *(unit_t *)(to + u * 8) = x;
            else
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (mine >> j & 1) to[u * 8 + j] = x[j];
        }
        __syncthreads();
    }
}

template <int RT, int CT, int HD>
__global__ void __launch_bounds__(256)
paged_append(oh_pappend a, int qk_blocks, int heads, int span) {
    if ((int)blockIdx.x < qk_blocks) append_qk<RT, CT, HD>(a, blockIdx.x, heads);
    else append_v<RT, CT, HD>(a, blockIdx.x - qk_blocks, span);
}

// The stored rows of a batch, as values. Keys as they are stored, 8 values a
// lane; values of the rows that share a tile by way of LDS, which the tile's
// units go through whole.
template <int RT, int CT, int HD>
OH_DEV void read_k(const oh_pappend &a, int block) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    constexpr int L = head_lanes<HD>(), R = 256 / L;
    const int tid = threadIdx.x, sub = tid % L, d0 = 8 * sub, head = block % a.pool.nkv, r = block / a.pool.nkv * R + tid / L;
    place at;
    if (!place_of(a.pool, a.b, r, &at)) return;
    int slot;
    const uint8_t *blk = slot_of(a.pool, a.b, at, head, &slot);
    if (!blk) return;
    float y[8];
    pg_load<8>((const cache_t *)blk + pg_k_at<CT>(HD, slot, d0), y);
    if (CT == OH_PT_Q8) {
        const float sc = *(const float *)(blk + a.pool.ks_off + 4 * slot);
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] *= sc;
    }
    pg_store<8>((row_t *)a.k.p + r * a.k.rs + head * a.k.hs + d0, y);
}
template <int RT, int CT, int HD>
OH_DEV void read_v(const oh_pappend &a, int block, int span) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    typedef cache_t unit_t __attribute__((ext_vector_type(8)));
    constexpr int L = head_lanes<HD>(), R = 256 / L;
    __shared__ __align__(16) cache_t tile[32 * HD];
    const int tid = threadIdx.x, sub = tid % L, d0 = 8 * sub, head = block % a.pool.nkv;
    const int r1 = min(block / a.pool.nkv * span + span, a.b.n_rows);
    auto at_unit = [](int u) { return u ^ ((u >> 3) & 7); };     // (as in append_v)
    for (int r = block / a.pool.nkv * span; r < r1;) {
        const int s = pg_seq_of(a.pool, a.b, r);
        if (s < 0) { r++; continue; }
        place at = {s, a.b.len[s] - (a.b.start[s + 1] - r)};
        const int left = min(a.b.start[s + 1], r1) - r;
        if (at.pos < 0) { r += at.pos <= -left ? left : -at.pos; continue; }
        const int n = min(left, 32 - (at.pos & 31)), r0 = r;
        r += n;
        int slot;
        const uint8_t *blk = slot_of(a.pool, a.b, at, head, &slot);
        if (!blk) continue;
        const cache_t *from = (const cache_t *)(blk + a.pool.v_off) + (slot >> 5) * 32 * HD;
#pragma unroll
        for (int k = 0; k < 4 * HD / 256; k++) {
            const int u = tid + 256 * k;
            *(unit_t *)(tile + at_unit(u) * 8) = *(const unit_t *)(from + u * 8);
        }
        __syncthreads();
        for (int i = tid / L; i < n; i += R) {
            const int sl = (slot & 31) + i;
            const float sc = CT == OH_PT_Q8 ? *(const float *)(blk + a.pool.vs_off + 4 * (slot + i)) : 1.0f;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = (float)tile[at_unit(((sl >> 2) & 3) * HD + d0 + j) * 8 + 4 * (sl >> 4) + (sl & 3)];
                y[j] = CT == OH_PT_Q8 ? x * sc : x;
            }
            pg_store<8>((row_t *)a.v.p + (int64_t)(r0 + i) * a.v.rs + head * a.v.hs + d0, y);
        }
        __syncthreads();
    }
}
template <int RT, int CT, int HD>
__global__ void __launch_bounds__(256)
paged_read(oh_pappend a, int k_blocks, int span) {
    if ((int)blockIdx.x < k_blocks) read_k<RT, CT, HD>(a, blockIdx.x);
    else read_v<RT, CT, HD>(a, blockIdx.x - k_blocks, span);
}

// values go in stretches of 32 rows, but one by one where sequences bring few
int span_of(const oh_pappend *a) { return a->b.n_rows >= (int64_t)8 * a->b.n_seq ? 32 : 1; }

template <int RT, int CT, int HD>
hipError_t append(const oh_pappend *a, hipStream_t st) {
    constexpr int R = 256 / head_lanes<HD>();
    // as many heads a block as leave 1024 blocks, so that few rows spread over the
    // card and many rows form their sines and cosines once
    const int64_t all = (a->q.p ? a->nh : 0) + a->pool.nkv, chunks = ((int64_t)a->b.n_rows + R - 1) / R;
    const int64_t heads = std::min(all, std::max<int64_t>(1, chunks * all / 1024));
    const int64_t qk = chunks * ((all + heads - 1) / heads);
    const int span = span_of(a);
    const int64_t v = ((int64_t)a->b.n_rows + span - 1) / span * a->pool.nkv;
    if (qk + v > kMaxBlocks) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((paged_append<RT, CT, HD>), dim3((unsigned)(qk + v)), dim3(256), 0, st, *a, (int)qk, (int)heads, span);
    return hipGetLastError();
}
template <int RT, int CT, int HD>
hipError_t read(const oh_pappend *a, hipStream_t st) {
    constexpr int R = 256 / head_lanes<HD>();
    const int span = span_of(a);
    const int64_t k = ((int64_t)a->b.n_rows + R - 1) / R * a->pool.nkv, v = ((int64_t)a->b.n_rows + span - 1) / span * a->pool.nkv;
    if (k + v > kMaxBlocks) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((paged_read<RT, CT, HD>), dim3((unsigned)(k + v)), dim3(256), 0, st, *a, (int)k, span);
    return hipGetLastError();
}
template <int RT, int CT>
hipError_t go(const oh_pappend *a, bool back, hipStream_t st) {
    switch (a->pool.hd) {
    case 64: return back ? read<RT, CT, 64>(a, st) : append<RT, CT, 64>(a, st);
    case 128: return back ? read<RT, CT, 128>(a, st) : append<RT, CT, 128>(a, st);
    case 256: return back ? read<RT, CT, 256>(a, st) : append<RT, CT, 256>(a, st);
    default: return hipErrorNotSupported;
    }
}

hipError_t types(const oh_pappend *a, bool read, hipStream_t st) {
    const int r = a->type, c = a->pool.type;
    if (c == OH_PT_Q8)
        return r == OH_PT_F32 ? go<OH_PT_F32, OH_PT_Q8>(a, read, st) : r == OH_PT_BF16 ? go<OH_PT_BF16, OH_PT_Q8>(a, read, st)
                                                                                        : go<OH_PT_F16, OH_PT_Q8>(a, read, st);
    return c == OH_PT_BF16 ? go<OH_PT_BF16, OH_PT_BF16>(a, read, st) : go<OH_PT_F16, OH_PT_F16>(a, read, st);
}

} // namespace

extern "C" hipError_t oh_launch_paged_append(const oh_pappend *a, hipStream_t st) { return types(a, false, st); }
extern "C" hipError_t oh_launch_paged_read(const oh_pappend *a, hipStream_t st) { return types(a, true, st); }
extern "C" hipError_t oh_launch_rope_tables(double2 *t, int steps, int half, double theta, hipStream_t st) {
    const int64_t n = (int64_t)(steps + kRopeStep) * half;
    hipLaunchKernelGGL(rope_tables, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, t, steps, half, theta);
    return hipGetLastError();
}
