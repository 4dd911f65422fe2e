// oh_host_paged.cpp - the paged key/value pool of the C ABI: pools, and the
// checks of the calls that append to one, read it back and attend over it.
// No reference twin: the reference serves one sequence per session.
#include "oh_engine.h"
#include "oh_paged.h"

#include <new>

struct ornith_hip_paged {
    ornith_hip_ctx *ctx = nullptr;
    CtxRef ref;
    oh_pool pool;
    int axes = 1;                               // of the rotation
    void *mem = nullptr, *aux = nullptr;        // the pages; the rotation's tables and the fault word
};

namespace {

// the context's device for the calls of a scope, the caller's own after it
struct OnDevice {
    int was = -1;
    hipError_t e;
    explicit OnDevice(int device) {
        e = hipGetDevice(&was);
        if (e == hipSuccess && was != device) e = hipSetDevice(device);
        else if (e == hipSuccess) was = -1;
    }
    ~OnDevice() { if (was >= 0) (void)hipSetDevice(was); }
};

int type_bytes(uint32_t t) { return t == OH_PT_F32 ? 4 : t == OH_PT_F16 || t == OH_PT_BF16 ? 2 : t == OH_PT_Q8 ? 1 : 0; }

int batch_of(const char *who, const ornith_hip_paged *p, const ornith_hip_paged_batch *b, oh_pbatch *out) {
    if (!p || !b) { seterr("%s: null pool or batch", who); return ORNITH_HIP_ERR_FORMAT; }
    if (b->n_seq < 0 || b->n_rows < 0 || b->max_pages < 0 || b->max_new < 0 || b->max_len < 0) {
        seterr("%s: negative size (n_seq %d, n_rows %d, max_pages %d, max_new %d, max_len %d)", who, b->n_seq, b->n_rows, b->max_pages,
               b->max_new, b->max_len);
        return ORNITH_HIP_ERR_FORMAT;
    }
    if (b->n_seq && b->n_rows && (!b->seq_start || !b->kv_len || !b->pages)) {
        seterr("%s: null seq_start, kv_len or pages", who);
        return ORNITH_HIP_ERR_FORMAT;
    }
    *out = oh_pbatch{b->seq_start, b->kv_len, b->pages, b->n_seq, b->n_rows, b->max_pages, std::min(b->max_new, b->n_rows)};
    return ORNITH_HIP_OK;
}
// no rows at all: there is nothing to do; rows, but no place for them: refused
bool nothing(const oh_pbatch &b) { return !b.n_seq || !b.n_rows; }
int placed(const char *who, const ornith_hip_paged_batch *b) {
    if (b->max_new && b->max_pages) return ORNITH_HIP_OK;
    seterr("%s: %d rows of %d sequences, but max_new %d and max_pages %d", who, b->n_rows, b->n_seq, b->max_new, b->max_pages);
    return ORNITH_HIP_ERR_FORMAT;
}

// a launch's outcome; batches past its limits are the caller's to cut
int launched(const char *who, hipError_t e) {
    if (e == hipErrorInvalidConfiguration) {
        seterr("%s: more rows, heads or sequences than one launch takes", who);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    HCHK(e);
    return ORNITH_HIP_OK;
}

int rows_of(const char *who, const char *what, const ornith_hip_rows *r, uint32_t type, oh_prows *out) {
    if (!r || !r->p) { seterr("%s: null %s", who, what); return ORNITH_HIP_ERR_FORMAT; }
    const int e = type_bytes(type);
    if ((uintptr_t)r->p % 16 || r->row_stride * e % 16 || r->head_stride * e % 16 || r->row_stride < 0 || r->head_stride < 0) {
        seterr("%s: %s needs 16-byte aligned rows and heads (pointer %p, strides %lld and %lld elements of %d bytes)", who, what,
               (void *)r->p, (long long)r->row_stride, (long long)r->head_stride, e);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    *out = oh_prows{r->p, r->row_stride, r->head_stride};
    return ORNITH_HIP_OK;
}

// rows that are written: of their own each, so that no two of a launch's stores meet
int apart(const char *who, const char *what, const oh_prows &r, int64_t n_rows, int64_t heads, int hd) {
    if ((n_rows < 2 || r.rs >= hd) && (heads < 2 || r.hs >= hd)) return ORNITH_HIP_OK;
    seterr("%s: rows or heads of %s overlap (strides %lld and %lld, heads of %d)", who, what, (long long)r.rs, (long long)r.hs, hd);
    return ORNITH_HIP_ERR_FORMAT;
}

int row_type(const char *who, const ornith_hip_paged *p, uint32_t type) {
    if (type != OH_PT_F32 && type != OH_PT_F16 && type != OH_PT_BF16) {
        seterr("%s: rows of type %u (F32, F16 or BF16)", who, type);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    if (p->pool.type != OH_PT_Q8 && (int)type != p->pool.type) {
        seterr("%s: rows of type %u over a pool of type %d (a 16-bit pool takes rows of its own type)", who, type, p->pool.type);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    return ORNITH_HIP_OK;
}

// Which kernels take the batch, and in how many parts of the key axis: enough
// blocks to fill the card a few times over, so that sequences of different
// lengths even out, and no more parts than the longest list of pages can need.
// A sequence's rows times the heads of a group decide: up to kFewRows they go to
// the kernel for few rows; where all sequences have more, or could, to the one
// for many.
constexpr int kFewRows = 32;
// Parts of up to `most` positions for `units` pieces of work: as short as `least`,
// and longer where that would make more than `blocks` blocks.
int cut(int64_t most, int64_t units, int64_t blocks, int64_t least, int limit, int32_t *len) {
    const int64_t n = std::max<int64_t>(1, std::min<int64_t>(limit, blocks / std::max<int64_t>(1, units)));
    *len = (int32_t)std::min<int64_t>(INT32_MAX / 2, std::max(least, (most + n - 1) / n));
    return (int)std::max<int64_t>(1, (most + *len - 1) / *len);
}
void plan(const ornith_hip_paged *p, const oh_pbatch &b, int max_len, int nh, int n_group, oh_pattn *a) {
    const int nkv = p->pool.nkv, G = nh / nkv;
    const int64_t table = (int64_t)b.max_pages << p->pool.page_sh, most = max_len > 0 ? std::min<int64_t>(table, max_len) : table;
    const int64_t widest = (int64_t)b.max_new * G, all = (int64_t)b.n_rows * G;
    a->G = G;
    a->nh = nh;
    a->n_group = n_group;
    a->few = widest <= kFewRows || (b.n_seq > 1 && b.n_rows < (int64_t)b.n_seq * b.max_new) ? kFewRows : 0;
    a->many = widest <= kFewRows ? -1 : a->few;
    a->gmany = all > kFewRows;
    a->parts = a->mparts = a->gparts = 1;
    a->least = a->mleast = a->gleast = 1;
    a->few_rows = (int32_t)std::min<int64_t>(b.max_new, std::max(1, kFewRows / G));
    // Few rows: 128 positions are a tile for each wave of a block; two tiles where
    // there are many sequences and a block fills a CU (heads of 256), so that short
    // ones are done in one round of blocks: an item takes about 9 us and 3 for each
    // further tile
    if (a->few) a->parts = cut(most, (int64_t)b.n_seq * nkv, 8192, p->pool.hd == 256 && b.n_seq * nkv >= 64 ? 256 : 128, 256, &a->least);
    // Many rows: blocks of 256 rows where units have more than 128 (the wider
    // block would have idle waves otherwise). Two blocks for each CU, so that
    // their ends even out; of a prefix, whose blocks are all alike, one for three
    // of four CUs: the shader engines are not dealt blocks evenly (192 blocks of a
    // prefix of 8000 positions took 42 us, 252 shorter ones 64).
    int rows = 128;
    (void)oh_pattn_many_rows(a, &rows);
    a->mrows = widest > 128 ? rows : 128;
    a->grows = n_group && all / n_group > 128 ? rows : 128;
    if (a->many >= 0) a->mparts = cut(most, ((all - 1) / a->mrows + 1) * nkv, 512, 256, 32, &a->mleast);
    if (n_group && a->gmany) a->gparts = cut(most, ((all - 1) / a->grows + n_group) * nkv, a->grows < rows ? 512 : 192, 128, 64, &a->gleast);
    else if (n_group) a->gparts = cut(most, (int64_t)n_group * nkv, 512, 128, 64, &a->gleast);
}
// The partial results of a call: of the few-row sequences, of those with many
// rows, of the prefixes; none of a kernel that writes whole rows itself. ws null:
// the bytes alone.
uint64_t lay_out(oh_pattn *a, void *ws) {
    const bool groups = a->n_group > 0;
    const uint64_t n[3] = {a->few && (groups || a->parts > 1) ? (uint64_t)a->b.n_seq * a->few_rows * a->nh * a->parts : 0,
                           a->many >= 0 && (groups || a->mparts > 1) ? (uint64_t)a->b.n_rows * a->nh * a->mparts : 0,
                           groups ? (uint64_t)a->b.n_rows * a->nh * a->gparts : 0};
    const uint64_t all = n[0] + n[1] + n[2];
    a->po = (float *)ws;
    a->mpo = a->po + n[0] * a->pool.hd;
    a->gpo = a->mpo + n[1] * a->pool.hd;
    a->pml = (float2 *)(a->po + all * a->pool.hd);
    a->mpml = a->pml + n[0];
    a->gpml = a->mpml + n[1];
    return all * ((uint64_t)a->pool.hd * 4 + 8);
}

int heads(const char *who, const ornith_hip_paged *p, int nh) {
    if (nh < 1 || nh % p->pool.nkv) {
        seterr("%s: %d query heads over %d key heads", who, nh, p->pool.nkv);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    return ORNITH_HIP_OK;
}

int attend(const char *who, const ornith_hip_paged *p, const ornith_hip_paged_batch *b, int n_group, const int32_t *first,
           const int32_t *shared, int nh, uint32_t type, const ornith_hip_rows *q, const ornith_hip_rows *out, float scale, void *ws,
           uint64_t ws_bytes, void *stream) {
    oh_pattn a;
    memset(&a, 0, sizeof a);
    CHK(batch_of(who, p, b, &a.b));
    CHK(row_type(who, p, type));
    CHK(heads(who, p, nh));
    if (!std::isfinite(scale)) { seterr("%s: scale %g", who, (double)scale); return ORNITH_HIP_ERR_FORMAT; }
    if (n_group < 0 || n_group > b->n_seq || (n_group && (!first || !shared))) {
        seterr("%s: %d groups of %d sequences, or a null list", who, n_group, b->n_seq);
        return ORNITH_HIP_ERR_FORMAT;
    }
    if (nothing(a.b)) return ORNITH_HIP_OK;
    CHK(placed(who, b));
    if ((int64_t)a.b.n_rows * nh > INT32_MAX || (int64_t)a.b.n_seq * nh > INT32_MAX) CHK(launched(who, hipErrorInvalidConfiguration));
    CHK(rows_of(who, "q", q, type, &a.q));
    CHK(rows_of(who, "out", out, type, &a.out));
    CHK(apart(who, "out", a.out, b->n_rows, nh, p->pool.hd));
    if (a.out.p == a.q.p) { seterr("%s: out is q", who); return ORNITH_HIP_ERR_FORMAT; }
    a.pool = p->pool;
    a.type = (int)type;
    a.scale = fabsf(scale) * 1.44269504088896340736f;
    a.sign = scale < 0.0f ? -1.0f : 1.0f;
    a.gfirst = first; a.glen = shared;
    plan(p, a.b, b->max_len, nh, n_group, &a);
    const uint64_t need = lay_out(&a, ws);
    if (need > ws_bytes || (need && (!ws || (uintptr_t)ws % 16))) {
        seterr("%s: a 16-byte aligned workspace of %llu bytes is needed, %llu given", who, (unsigned long long)need, (unsigned long long)ws_bytes);
        return ORNITH_HIP_ERR_FORMAT;
    }
    OnDevice dev(p->ctx->device);
    HCHK(dev.e);
    const hipStream_t st = (hipStream_t)stream;
    if (a.many >= 0 || (n_group && a.gmany)) CHK(launched(who, oh_launch_pattn_many(&a, st)));
    if (a.few || (n_group && !a.gmany)) CHK(launched(who, oh_launch_pattn_few(&a, st)));
    if (need) CHK(launched(who, oh_launch_pattn_join(&a, st)));
    return ORNITH_HIP_OK;
}

int pool_new(ornith_hip_ctx *ctx, const ornith_hip_paged_cfg *c, ornith_hip_paged *p) {
    oh_pool &o = p->pool;
    memset(&o, 0, sizeof o);
    if (c->type != OH_PT_Q8 && c->type != OH_PT_F16 && c->type != OH_PT_BF16) {
        seterr("paged_new: pool type %u (ORNITH_HIP_KV_Q8, _F16 or _BF16)", c->type);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    if (c->hd != 64 && c->hd != 128 && c->hd != 256) {
        seterr("paged_new: head dim %d (64, 128 or 256)", c->hd);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    if (c->page_len != 32 && c->page_len != 64 && c->page_len != 128 && c->page_len != 256) {
        seterr("paged_new: pages of %d positions (32, 64, 128 or 256)", c->page_len);
        return ORNITH_HIP_ERR_UNSUPPORTED;
    }
    if (c->nkv < 1 || c->nkv > 65535 || c->n_pages < 1) {
        seterr("paged_new: %d key heads, %d pages", c->nkv, c->n_pages);
        return ORNITH_HIP_ERR_FORMAT;
    }
    if (c->rope_dim < 0 || c->rope_dim > c->hd || c->rope_dim % 2) {
        seterr("paged_new: rotation of %d of %d dims", c->rope_dim, c->hd);
        return ORNITH_HIP_ERR_FORMAT;
    }
    if (c->rope_dim && (!(c->rope_theta > 0.0f) || !std::isfinite(c->rope_theta) || c->max_pos < 1 || c->max_pos > (1 << 24))) {
        seterr("paged_new: rope_theta %g, max_pos %d (at most 2^24)", (double)c->rope_theta, c->max_pos);
        return ORNITH_HIP_ERR_FORMAT;
    }
    const int half = c->rope_dim / 2;
    for (int i = 0; c->rope_axis && i < half; i++) {
        if (c->rope_axis[i] > 3) { seterr("paged_new: axis %d of frequency %d (0 to 3)", c->rope_axis[i], i); return ORNITH_HIP_ERR_FORMAT; }
        p->axes = std::max(p->axes, c->rope_axis[i] + 1);
    }
    const uint32_t plane = (uint32_t)c->page_len * c->hd * type_bytes(c->type);
    o.nkv = c->nkv; o.hd = c->hd; o.type = (int32_t)c->type; o.n_pages = c->n_pages;
    while ((1 << o.page_sh) < c->page_len) o.page_sh++;
    o.v_off = plane;
    o.ks_off = 2 * plane;
    o.vs_off = o.ks_off + 4 * c->page_len;
    o.block = 2 * plane + (c->type == OH_PT_Q8 ? 8 * c->page_len : 0);
    o.rope_dim = c->rope_dim;
    o.max_pos = c->max_pos;
    const size_t bytes = (size_t)c->n_pages * c->nkv * o.block;
    HCHK(dev_malloc(ctx, &p->mem, bytes));
    o.mem = (uint8_t *)p->mem;
    HCHK(hipMemset(p->mem, 0, bytes));
    // the fault word, the rotation's (cos, sin) of kRopeStep positions each and of
    // those within one, the axes
    const int steps = half ? (c->max_pos + kRopeStep - 1) / kRopeStep : 0;
    const size_t tb = (size_t)(steps + (half ? kRopeStep : 0)) * half * sizeof(double2);
    HCHK(dev_malloc(ctx, &p->aux, 256 + tb + half + 1));
    uint8_t *aux = (uint8_t *)p->aux;
    HCHK(hipMemset(aux, 0, 256 + tb + half + 1));
    o.fault = (int32_t *)aux;
    o.rope_hi = (const double2 *)(aux + 256);
    o.rope_lo = o.rope_hi + (size_t)steps * half;
    o.rope_axis = aux + 256 + tb;
    if (half) HCHK(oh_launch_rope_tables((double2 *)(aux + 256), steps, half, c->rope_theta, nullptr));
    if (half && c->rope_axis) HCHK(hipMemcpy(aux + 256 + tb, c->rope_axis, half, hipMemcpyHostToDevice));
    HCHK(hipDeviceSynchronize());
    return ORNITH_HIP_OK;
}

} // namespace

extern "C" int ornith_hip_paged_new(ornith_hip_ctx *ctx, const ornith_hip_paged_cfg *cfg, ornith_hip_paged **out) {
    if (out) *out = nullptr;
    if (!ctx || !cfg || !out) { seterr("paged_new: null context, cfg or out"); return ORNITH_HIP_ERR_FORMAT; }
    OnDevice dev(ctx->device);
    HCHK(dev.e);
    ornith_hip_paged *p = nullptr;
    int r;
    try {
        p = new ornith_hip_paged;
        p->ctx = ctx;
        p->ref.hold(ctx);
        r = pool_new(ctx, cfg, p);
    } catch (const std::exception &) {
        seterr("paged_new: out of host memory");
        r = ORNITH_HIP_ERR_OOM;
    }
    if (r == ORNITH_HIP_OK) *out = p;
    else ornith_hip_paged_free(p);
    return r;
}

extern "C" void ornith_hip_paged_free(ornith_hip_paged *p) {
    if (!p) return;
    {
        OnDevice dev(p->ctx->device);
        if (p->mem) (void)hipFree(p->mem);
        if (p->aux) (void)hipFree(p->aux);
    }
    delete p;
}

extern "C" int ornith_hip_paged_faults(ornith_hip_paged *p, int32_t *faults) {
    if (!p || !faults) { seterr("paged_faults: null pool or result"); return ORNITH_HIP_ERR_FORMAT; }
    OnDevice dev(p->ctx->device);
    HCHK(dev.e);
    HCHK(hipDeviceSynchronize());
    const int32_t zero = 0;
    HCHK(hipMemcpy(faults, p->pool.fault, 4, hipMemcpyDeviceToHost));
    if (*faults) HCHK(hipMemcpy(p->pool.fault, &zero, 4, hipMemcpyHostToDevice));
    return ORNITH_HIP_OK;
}

extern "C" int ornith_hip_paged_append(ornith_hip_paged *p, const ornith_hip_paged_batch *b, int nh, uint32_t type,
                                       const ornith_hip_rows *k, const ornith_hip_rows *v, const ornith_hip_rows *q,
                                       const ornith_hip_rows *q_out, const float *q_norm, const float *k_norm, float eps,
                                       const int32_t *rope_pos, int64_t rope_stride, void *stream) {
    const char *who = "paged_append";
    oh_pappend a;
    memset(&a, 0, sizeof a);
    CHK(batch_of(who, p, b, &a.b));
    CHK(row_type(who, p, type));
    for (const float *w : {q_norm, k_norm})
        if ((uintptr_t)w % 16) { seterr("%s: norm weights at %p, not a multiple of 16 bytes", who, (const void *)w); return ORNITH_HIP_ERR_UNSUPPORTED; }
    if (!(eps >= 0.0f)) { seterr("%s: eps %g", who, (double)eps); return ORNITH_HIP_ERR_FORMAT; }
    if (nothing(a.b)) return ORNITH_HIP_OK;
    CHK(placed(who, b));
    CHK(rows_of(who, "k", k, type, &a.k));
    CHK(rows_of(who, "v", v, type, &a.v));
    if (q && q->p) {
        CHK(heads(who, p, nh));
        CHK(rows_of(who, "q", q, type, &a.q));
        CHK(rows_of(who, "q_out", q_out, type, &a.q_out));
        CHK(apart(who, "q_out", a.q_out, b->n_rows, nh, p->pool.hd));
        a.nh = nh;
    }
    a.pool = p->pool;
    a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps;
    a.pos = rope_pos; a.pos_stride = rope_stride; a.axes = p->axes;
    a.type = (int)type;
    OnDevice dev(p->ctx->device);
    HCHK(dev.e);
    return launched(who, oh_launch_paged_append(&a, (hipStream_t)stream));
}

extern "C" int ornith_hip_paged_read(const ornith_hip_paged *p, const ornith_hip_paged_batch *b, uint32_t type,
                                     const ornith_hip_rows *k, const ornith_hip_rows *v, void *stream) {
    const char *who = "paged_read";
    oh_pappend a;
    memset(&a, 0, sizeof a);
    CHK(batch_of(who, p, b, &a.b));
    CHK(row_type(who, p, type));
    if (nothing(a.b)) return ORNITH_HIP_OK;
    CHK(placed(who, b));
    CHK(rows_of(who, "k", k, type, &a.k));
    CHK(rows_of(who, "v", v, type, &a.v));
    CHK(apart(who, "k", a.k, b->n_rows, p->pool.nkv, p->pool.hd));
    CHK(apart(who, "v", a.v, b->n_rows, p->pool.nkv, p->pool.hd));
    a.pool = p->pool;
    a.type = (int)type;
    OnDevice dev(p->ctx->device);
    HCHK(dev.e);
    return launched(who, oh_launch_paged_read(&a, (hipStream_t)stream));
}

extern "C" int ornith_hip_paged_workspace(const ornith_hip_paged *p, const ornith_hip_paged_batch *b, int nh, uint32_t type,
                                          int n_group, uint64_t *bytes) {
    oh_pattn a;
    memset(&a, 0, sizeof a);
    if (!bytes) { seterr("paged_workspace: null result"); return ORNITH_HIP_ERR_FORMAT; }
    *bytes = 0;
    CHK(batch_of("paged_workspace", p, b, &a.b));
    CHK(row_type("paged_workspace", p, type));
    CHK(heads("paged_workspace", p, nh));
    if (n_group < 0) { seterr("paged_workspace: %d groups", n_group); return ORNITH_HIP_ERR_FORMAT; }
    if (nothing(a.b)) return ORNITH_HIP_OK;
    CHK(placed("paged_workspace", b));
    a.pool = p->pool;
    a.type = (int)type;
    plan(p, a.b, b->max_len, nh, n_group, &a);
    *bytes = lay_out(&a, nullptr);
    return ORNITH_HIP_OK;
}

extern "C" int ornith_hip_paged_attend(const ornith_hip_paged *p, const ornith_hip_paged_batch *b, int nh, uint32_t type,
                                       const ornith_hip_rows *q, const ornith_hip_rows *out, float scale, void *workspace,
                                       uint64_t workspace_bytes, void *stream) {
    return attend("paged_attend", p, b, 0, nullptr, nullptr, nh, type, q, out, scale, workspace, workspace_bytes, stream);
}

extern "C" int ornith_hip_paged_attend_prefix(const ornith_hip_paged *p, const ornith_hip_paged_batch *b, int n_group,
                                              const int32_t *prefix_first, const int32_t *prefix_len, int nh, uint32_t type,
                                              const ornith_hip_rows *q, const ornith_hip_rows *out, float scale, void *workspace,
                                              uint64_t workspace_bytes, void *stream) {
    return attend("paged_attend_prefix", p, b, n_group, prefix_first, prefix_len, nh, type, q, out, scale, workspace,
                  workspace_bytes, stream);
}
