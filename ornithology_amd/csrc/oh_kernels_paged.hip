// oh_kernels_paged.hip - rows into a paged pool and out of it.
//
// Append: per (row, head) of the keys, x / sqrt(mean(x^2) + eps) * w if there is
// a norm, the rotation of pairs (i, i + r/2) by the angle P * theta^(-2i/r),
// and the store, as 16-bit values or as codes rint(x * 127 / max|x|) with the
// scale max|x| / 127; values without norm and rotation; queries with both, to
// q_out. A wave holds one head of one row.
#include "oh_paged_dev.h"

namespace {

// (cos, sin) of frequency i at `pos`: the angles of the 1024-step and of the
// rest are added in 64 bits and rounded once, so far positions are as exact
// as near ones
OH_DEV float2 rope_cs(const oh_pool &p, int pos, int i) {
    const int half = p.rope_dim / 2;
    const double2 a = p.rope_hi[(size_t)(pos / kRopeStep) * half + i], b = p.rope_lo[(size_t)(pos % kRopeStep) * half + i];
    return make_float2((float)(a.x * b.x - a.y * b.y), (float)(a.y * b.x + a.x * b.y));
}

OH_DEV float wave_sum_f32(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
OH_DEV float wave_max_f32(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

template <int RT, int CT, int HD>
__global__ void __launch_bounds__(256)
paged_append(oh_pappend a) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    constexpr int E = HD / 64;
    __shared__ float xs[4][HD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int nkv = a.pool.nkv, nq = a.q.p ? a.nh : 0, units = nq + 2 * nkv;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int r = (int)(item / units), u = (int)(item % units);
    if (r >= a.b.n_rows) return;
    const int s = pg_seq_of(a.pool, a.b, r);
    if (s < 0) return;
    const int len = a.b.len[s], pos = len - (a.b.start[s + 1] - r);
    if (pos < 0) return;                               // padding
    const bool isq = u < nq, isv = u >= nq + nkv;
    const int h = isq ? u : isv ? u - nq - nkv : u - nq;
    const oh_prows &in = isq ? a.q : isv ? a.v : a.k;
    const row_t *x = (const row_t *)in.p + r * in.rs + h * in.hs + lane * E;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = (float)x[e];
    if (!isv) {
        const float *w = isq ? a.q_norm : a.k_norm;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) ss = fmaf(y[e], y[e], ss);
            const float inv = 1.0f / sqrtf(wave_sum_f32(ss) / HD + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = y[e] * inv * w[lane * E + e];
        }
        const int half = a.pool.rope_dim / 2;
        if (half) {
#pragma unroll
            for (int e = 0; e < E; e++) xs[wave][lane * E + e] = y[e];
            __builtin_amdgcn_wave_barrier();
            bool bad = false;
            float z[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int d = lane * E + e;
                z[e] = y[e];
                if (d < 2 * half) {
                    const int i = d < half ? d : d - half;
                    const int pp = a.pos ? a.pos[a.pool.rope_axis[i] * a.pos_stride + r] : pos;
                    if (pp < 0 || pp >= a.pool.max_pos) { bad = true; continue; }
                    const float2 cs = rope_cs(a.pool, pp, i);
                    const float o = xs[wave][d < half ? d + half : d - half];
                    z[e] = d < half ? y[e] * cs.x - o * cs.y : o * cs.y + y[e] * cs.x;
                }
            }
            if (__any(bad)) {
                if (lane == 0) pg_report(a.pool, OH_PF_POSITION);
                return;
            }
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = z[e];
        }
    }
    if (isq) {
        row_t *o = (row_t *)a.q_out.p + r * a.q_out.rs + h * a.q_out.hs + lane * E;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = (row_t)y[e];
        return;
    }
    const int pi = pos >> a.pool.page_sh;
    if (pi >= a.b.max_pages) { if (lane == 0) pg_report(a.pool, OH_PF_BATCH); return; }
    const int page = a.b.table[(size_t)s * a.b.max_pages + pi], slot = pos & ((1 << a.pool.page_sh) - 1);
    if (page < 0 || page >= a.pool.n_pages) { if (lane == 0) pg_report(a.pool, OH_PF_PAGE); return; }
    uint8_t *blk = pg_block(a.pool, page, h);
    cache_t *to = (cache_t *)(blk + (isv ? a.pool.v_off : 0));
    if (CT == OH_PT_Q8) {
        float am = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) am = fmaxf(am, fabsf(y[e]));
        am = wave_max_f32(am);
        bool nan = false;                              // a NaN is in no code: it goes into the scale
#pragma unroll
        for (int e = 0; e < E; e++) nan |= y[e] != y[e];
        if (__any(nan)) am = NAN;
        const float iv = am > 0.0f ? 127.0f / am : 0.0f;
        if (lane == 0) *(float *)(blk + (isv ? a.pool.vs_off : a.pool.ks_off) + 4 * slot) = am / 127.0f;
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = fminf(fmaxf(rintf(y[e] * iv), -127.0f), 127.0f);
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane * E + e;
        to[isv ? pg_v_at(HD, slot, d) : pg_k_at<CT>(HD, slot, d)] = CT == OH_PT_Q8 ? (cache_t)(int)y[e] : (cache_t)y[e];
    }
}

// the stored rows of a batch, as values
template <int RT, int CT, int HD>
__global__ void __launch_bounds__(256)
paged_read(oh_pappend a) {
    typedef typename pg_elem<RT>::t row_t;
    typedef typename pg_elem<CT>::t cache_t;
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nkv = a.pool.nkv;
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int r = (int)(item / (2 * nkv)), u = (int)(item % (2 * nkv));
    if (r >= a.b.n_rows) return;
    const int s = pg_seq_of(a.pool, a.b, r);
    if (s < 0) return;
    const int pos = a.b.len[s] - (a.b.start[s + 1] - r);
    if (pos < 0) return;
    const int pi = pos >> a.pool.page_sh;
    if (pi >= a.b.max_pages) { if (lane == 0) pg_report(a.pool, OH_PF_BATCH); return; }
    const int page = a.b.table[(size_t)s * a.b.max_pages + pi], slot = pos & ((1 << a.pool.page_sh) - 1);
    if (page < 0 || page >= a.pool.n_pages) { if (lane == 0) pg_report(a.pool, OH_PF_PAGE); return; }
    const bool isv = u >= nkv;
    const int h = isv ? u - nkv : u;
    const uint8_t *blk = pg_block(a.pool, page, h);
    const cache_t *from = (const cache_t *)(blk + (isv ? a.pool.v_off : 0));
    const float sc = CT == OH_PT_Q8 ? *(const float *)(blk + (isv ? a.pool.vs_off : a.pool.ks_off) + 4 * slot) : 1.0f;
    const oh_prows &o = isv ? a.v : a.k;
    row_t *to = (row_t *)o.p + r * o.rs + h * o.hs;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane * E + e;
        const float x = (float)from[isv ? pg_v_at(HD, slot, d) : pg_k_at<CT>(HD, slot, d)];
        to[d] = (row_t)(CT == OH_PT_Q8 ? x * sc : x);
    }
}

template <int RT, int CT>
hipError_t go(const oh_pappend *a, bool read, hipStream_t st) {
    const int units = (read ? 0 : a->q.p ? a->nh : 0) + 2 * a->pool.nkv;
    const int64_t blocks = ((int64_t)a->b.n_rows * units + 3) / 4;
    if (blocks > kMaxBlocks) return hipErrorInvalidConfiguration;
    void (*k)(oh_pappend) = nullptr;
    switch (a->pool.hd) {
    case 64: k = read ? paged_read<RT, CT, 64> : paged_append<RT, CT, 64>; break;
    case 128: k = read ? paged_read<RT, CT, 128> : paged_append<RT, CT, 128>; break;
    case 256: k = read ? paged_read<RT, CT, 256> : paged_append<RT, CT, 256>; break;
    default: return hipErrorNotSupported;
    }
    hipLaunchKernelGGL(k, dim3((unsigned)blocks), dim3(256), 0, st, *a);
    return hipGetLastError();
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
