"""GPU: the paged key/value pool (ornith_hip_paged_*) against its formulas in 64
bits (paged_ref): rows stored with norm and rotation, attention of ragged
batches, shared prefixes, at the sizes, strides and masks where it can go
wrong."""
import math

import pytest
import torch

import ornithology_amd as oa
import paged_ref as ref
from paged_ref import DT, Made, half_step

pytestmark = pytest.mark.gpu

KV = {"q8": oa.KV_Q8, "bf16": oa.KV_BF16, "f16": oa.KV_F16}
PAIRS = [("f32", "q8"), ("bf16", "q8"), ("f16", "q8"), ("bf16", "bf16"), ("f16", "f16")]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def close(got, want, tol):
    got = got.double()
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, at most {float(((got - want).abs() / tol).max()):.3g} tolerances"


def axes_of(n_axes, half):
    return [i % n_axes for i in range(half)]


# ---- append and read --------------------------------------------------------------

@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("hd,nh,nkv,page,rope,axes,norm,spec", [
    (256, 16, 2, 64, 64, 1, True, ([1], [1])),
    (256, 8, 1, 32, 256, 1, False, ([1, 1, 1], [4097, 33, 1])),
    (128, 6, 3, 64, 96, 3, True, ([70, 1, 0, 33, 5], [70, 129, 40, 65, 5])),
    (64, 4, 4, 128, 0, 1, True, ([31, 32, 33], [200, 32, 160])),
    (64, 10, 2, 256, 62, 2, False, ([300, 2, 3], [513, 2, 3])),
    (128, 32, 8, 32, 128, 1, False, ([1] * 40, list(range(1, 41)))),
])
def test_append_stores_and_rotates(hip_ctx, rows, cache, hd, nh, nkv, page, rope, axes, norm, spec):
    g, dt = gen(hd + nh + page), DT[rows]
    m = Made(*spec, page, extra_rows=3)
    theta, eps = 1e6, 1e-5
    pool = hip_ctx.paged_kv(m.n_pages, nkv, hd, page_len=page, type=KV[cache], rope_dim=rope, rope_theta=theta,
                            rope_axis=axes_of(axes, rope // 2) if axes > 1 else None)
    n, own = m.total, m.start[-1]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # heads of one fused buffer: [q | k | v] of a row side by side
    fused = rand(n, nh + 2 * nkv, hd).to(dt)
    q, k, v = fused[:, :nh], fused[:, nh:nh + nkv], fused[:, nh + nkv:]
    if own > 1:
        v[1] = 0                                            # a head of zeros has no scale
    kept = fused.clone()
    qw, kw = ((1 + 0.2 * rand(hd)) if norm else None for _ in range(2))
    pos = torch.randint(0, 1 << 20, (axes, n), generator=g, device="cuda", dtype=torch.int32)
    out = torch.full_like(q.contiguous(), 7.0)
    got = pool.append(m.batch, k, v, q=q, q_out=out, q_norm=qw, k_norm=kw, eps=eps, rope_pos=pos)
    assert got is out and torch.equal(fused, kept)
    assert (out[own:] == 7).all()                           # nobody's rows
    q, k, v = q[:own], k[:own], v[:own]
    u = 2.0 ** -24
    step = max(half_step(dt), 0.0)
    wants = []
    for x, w in ((q, qw), (k, kw)):
        y = ref.rotated(x, w, eps, pos[:, :own], axes_of(axes, rope // 2), theta)
        # |a cos| + |b sin| <= the pair's length; a norm's root, quotient and two
        # products, the rotation's three roundings and those of cos and sin; the
        # sum of squares walks over hd steps, half of which the root leaves
        most = (x.double() if w is None else ref.rotated(x, w, eps, pos[:, :own], [], theta)).abs().amax(-1, keepdim=True) * math.sqrt(2)
        wants.append((y, most * u * (10 + 2 * math.sqrt(hd))))
    close(out[:own], wants[0][0], step * wants[0][0].abs() + wants[0][1] + 1e-30)
    back = DT["f16" if cache == "f16" else "bf16" if cache == "bf16" else rows]
    ks, vs = (torch.full((n, nkv, hd), 5.0, dtype=back, device="cuda") for _ in range(2))
    pool.read(m.batch, back, ks, vs)
    assert (ks[own:] == 5).all() and (vs[own:] == 5).all()
    for got, (want, near) in ((ks[:own], wants[1]), (vs[:own], (v.double(), 0.0))):
        top = want.abs().amax(-1, keepdim=True)
        if cache == "q8":       # half a code of max / 127; the quotient, the scale and its product round too
            tol = top / 127 * (0.5 + 127 * 4 * u) + near * 2 + half_step(back) * (want.abs() + top / 254)
        else:
            tol = half_step(back) * want.abs() + near + 2.0 ** -25      # (fp16: subnormal steps)
        close(got, want, tol + 1e-30)
    pool.check()


@pytest.mark.parametrize("size", [2.0 ** -100, 1e-36, 3e-37, 1e-38, 1e-40])
def test_codes_of_small_heads(hip_ctx, size):
    g = gen(11)
    m = Made([40, 1], [40, 70], 32)
    pool = hip_ctx.paged_kv(m.n_pages, 2, 64, page_len=32, type=oa.KV_Q8)
    k, v = (torch.randn(m.total, 2, 64, generator=g, device="cuda").clamp(-1, 1) * size for _ in range(2))
    for x in (k, v):
        x[:, :, 5] = size                                   # (a head's largest)
        x[:, :, 7] = 0
    pool.append(m.batch, k, v)
    for got, x in zip(pool.read(m.batch, torch.float32), (k, v)):
        # half a code and the roundings of quotient, scale and product; a subnormal
        # scale is off by half of 2^-149 in each of up to 127 codes, and its product as much
        close(got, x.double(), size / 127 * (0.5 + 127 * 5 * 2.0 ** -24) + 128 * 2.0 ** -150)
        assert (got[:, :, 7] == 0).all()


def test_append_in_place_and_without_queries(hip_ctx):
    m = Made([3, 40], [10, 40], 32)
    pool = hip_ctx.paged_kv(m.n_pages, 2, 64, page_len=32, type=oa.KV_BF16, rope_dim=64, rope_theta=1e4)
    g = gen(1)
    q, k, v = (torch.randn(m.total, h, 64, generator=g, device="cuda").bfloat16() for h in (4, 2, 2))
    want = pool.append(m.batch, k, v, q=q)
    k0 = pool.read(m.batch, torch.bfloat16)[0]
    same = q.clone()
    assert pool.append(m.batch, k, v, q=same, q_out=same) is same and torch.equal(same, want)
    assert pool.append(m.batch, k, v) is None and torch.equal(pool.read(m.batch, torch.bfloat16)[0], k0)
    # positions by default are the cache's
    p = torch.tensor([m.positions()], dtype=torch.int32, device="cuda")
    assert torch.equal(pool.append(m.batch, k, v, q=q, rope_pos=p), want)
    pool.check()


# ---- attention -----------------------------------------------------------------------

SPECS = {
    "one": ([1], [1]),
    "one-31": ([1], [31]),
    "one-4097": ([1], [4097]),
    "decode": ([1] * 9, [1, 2, 31, 32, 33, 64, 500, 1025, 129]),
    "padded": ([1, 1, 2, 1, 4], [70, 0, 1, 0, 2]),
    "few": ([2, 3, 0, 5, 4], [2, 300, 77, 64, 1000]),
    "prompt-1000": ([1000], [1000]),
    "prompts": ([33, 64, 65, 1, 130], [33, 64, 65, 1, 130]),
    "mixed": ([257, 1, 1, 0, 1], [700, 3, 900, 10, 64]),
}


def run_attention(hip_ctx, rows, cache, hd, nh, nkv, page, spec, scale=None, groups=(), shared=0, seed=0, change=None, extra_pages=0):
    """Attention of a filled pool and its 64-bit result; change(k, v): the
    contents, edited before they are stored."""
    g, dt = gen(seed + hd + nh), DT[rows]
    m = Made(*spec, page, seed=seed, groups=groups, shared=shared, extra_rows=2, extra_pages=extra_pages)
    pool = hip_ctx.paged_kv(m.n_pages, nkv, hd, page_len=page, type=KV[cache])
    held = torch.float32 if cache == "q8" else DT[cache]
    # contents by position, those of shared pages alike
    k, v = (torch.randn(sum(m.lens), nkv, hd, generator=g, device="cuda").to(held) for _ in range(2))
    whole = shared // page * page
    for a, b in zip(groups[:-1], groups[1:]):
        for s in range(a + 1, b):
            for x in (k, v):
                x[m.all_start[s]:m.all_start[s] + whole] = x[m.all_start[a]:m.all_start[a] + whole]
    if change:
        change(m, k, v)
    if sum(m.lens):
        pool.append(m.whole, k, v)
        wide = torch.float32 if cache == "q8" else held
        k, v = pool.read(m.whole, wide)                     # (what is attended is what is stored)
    q = (torch.randn(m.total, nh, hd, generator=g, device="cuda") * 1.5).to(dt)
    out = torch.full_like(q, 9.0)
    if groups:
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        pool.attend_prefix(m.batch, q, i32(list(groups)), i32([shared] * (len(groups) - 1)), scale=scale, out=out)
    else:
        pool.attend(m.batch, q, scale=scale, out=out)
    own = m.start[-1]
    assert (out[own:] == 9).all()
    pool.check()
    return m, q, k, v, out[:own]


def verify(m, q, k, v, out, scale, rows):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    for s, (r, n) in enumerate(zip(m.rows, m.lens)):
        if not r:
            continue
        a, b = m.start[s], m.all_start[s]
        last = torch.arange(n - r, n, device="cuda")
        o, spread, reach = ref.attention(q[a:a + r].double(), k[b:b + n].double(), v[b:b + n].double(), last, scale)
        # weights are held in at least the rows' type
        tol = ref.attention_tolerance(o, spread, reach, DT[rows], q.shape[-1], n, 0.0 if rows == "f32" else half_step(DT[rows]))
        close(out[a:a + r], o, tol)


@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("hd,nh,nkv,page", [(256, 16, 2, 64), (128, 8, 8, 32), (128, 28, 4, 128), (64, 15, 3, 256), (64, 6, 1, 32)])
@pytest.mark.parametrize("spec", SPECS, ids=str)
def test_attend(hip_ctx, rows, cache, hd, nh, nkv, page, spec):
    verify(*run_attention(hip_ctx, rows, cache, hd, nh, nkv, page, SPECS[spec]), None, rows)


@pytest.mark.parametrize("rows,cache", [("f32", "q8"), ("bf16", "bf16"), ("f16", "q8")])
@pytest.mark.parametrize("spec", ["one-4097", "padded", "few", "mixed"])
def test_strided_rows_and_loose_bounds(hip_ctx, rows, cache, spec):
    m, q, k, v, out = run_attention(hip_ctx, rows, cache, 128, 8, 2, 64, SPECS[spec])
    held = k.dtype if cache == "q8" else DT[cache]
    pool = hip_ctx.paged_kv(m.n_pages, 2, 128, page_len=64, type=KV[cache])
    pool.append(m.whole, k.to(held), v.to(held))
    stored = pool.read(m.whole, k.dtype)
    own = m.start[-1]
    plain = pool.attend(m.batch, q)
    # one of three row buffers side by side; heads before rows
    side = torch.full((m.total, 3, 8, 128), 4.0, dtype=q.dtype, device="cuda")
    side[:, 1] = q
    heads = torch.full((8, m.total, 128), 4.0, dtype=q.dtype, device="cuda").transpose(0, 1)
    got = pool.attend(m.batch, side[:, 1], out=heads)
    assert got is heads and torch.equal(heads[:own], plain[:own]) and (heads[own:] == 4).all()
    pool.attend(m.batch, heads.copy_(q), out=side[:, 2])
    assert torch.equal(side[:own, 2], plain[:own]) and (side[:, 0] == 4).all() and (side[own:, 2] == 4).all()
    # the longest length is a hint, and max_new a bound that may be wide
    for max_new, max_len in ((max(m.rows), 1), (max(m.rows), 100), (m.total, 0), (m.total + 70, 1 << 20)):
        batch = oa.PagedBatch(*m.t, n_rows=m.total, max_new=max_new, max_len=max_len)
        verify(m, q, *stored, pool.attend(batch, q)[:own], None, rows)
    pool.check()


# ---- shared prefixes --------------------------------------------------------------------

GROUPS = {
    # rows, lengths, groups' first sequences, prefix
    "two": ([1, 1], [100, 90], (0, 2), 80),
    "answers": ([1] * 12, [530 + 3 * i for i in range(12)], (0, 12), 512),
    "three": ([1] * 20, [300 + 17 * i for i in range(20)], (0, 7, 8, 20), 289),
    "some": ([1, 2, 1, 40, 3, 1, 9], [333, 700, 290, 512, 257, 80, 20], (1, 5), 256),
    "pieces": ([130, 1, 64, 77], [900, 770, 900, 860], (0, 4), 768),
    "short": ([1, 1, 3], [20, 31, 9], (0, 3), 6),
    "only": ([2, 2, 5], [256, 258, 261], (0, 3), 256),
}


@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("hd,nh,nkv,page", [(256, 16, 2, 64), (128, 8, 8, 32), (128, 28, 4, 128), (64, 6, 1, 256)])
@pytest.mark.parametrize("group", GROUPS, ids=str)
def test_attend_prefix(hip_ctx, rows, cache, hd, nh, nkv, page, group):
    r, lens, groups, shared = GROUPS[group]
    verify(*run_attention(hip_ctx, rows, cache, hd, nh, nkv, page, (r, lens), groups=groups, shared=shared), None, rows)


# ---- masks --------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cache", PAIRS)
@pytest.mark.parametrize("hd,nh,nkv,page", [(128, 8, 2, 64), (256, 8, 1, 32), (64, 3, 3, 128)])
@pytest.mark.parametrize("spec", [([1, 1], [33, 600]), ([9, 3], [40, 200]), ([100], [300]), ([90, 1, 60], [90, 77, 400])], ids=str)
def test_what_is_hidden_is_not_seen(hip_ctx, rows, cache, hd, nh, nkv, page, spec):
    """Pages hold another request's infinities and NaN behind a sequence's end,
    and a prompt's later tokens are infinite or NaN: rows that do not see them
    are as if they were not there, rows that do are not finite."""
    g, dt = gen(5), DT[rows]
    m = Made(*spec, page)
    pool = hip_ctx.paged_kv(m.n_pages, nkv, hd, page_len=page, type=KV[cache])
    held = torch.float32 if cache == "q8" else DT[cache]
    n = m.n_pages
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    every = oa.PagedBatch(i32([page * i for i in range(n + 1)]), i32([page] * n), i32([[i] for i in range(n)]), n_rows=n * page, max_new=page)
    junk = torch.tensor([math.inf, math.nan, -math.inf, 1.0], device="cuda")[torch.randint(0, 4, (n * page, nkv, hd), generator=g, device="cuda")]
    pool.append(every, junk.to(held), junk.to(held))
    k, v = (torch.randn(sum(m.lens), nkv, hd, generator=g, device="cuda").to(held) for _ in range(2))
    pool.append(m.whole, k, v)
    q = torch.randn(m.total, nh, hd, generator=g, device="cuda").to(dt)
    wide = torch.float32 if cache == "q8" else held
    clean = pool.attend(m.batch, q)
    verify(m, q, *pool.read(m.whole, wide), clean, None, rows)
    # the last tokens of every sequence, if they are not all there is
    bad = [s for s in range(len(m.rows)) if m.rows[s] > 2]
    for x in (math.nan, math.inf):
        k2, v2 = k.clone(), v.clone()
        for s in bad:
            k2[m.all_start[s + 1] - 1] = math.nan
            v2[m.all_start[s + 1] - 2:m.all_start[s + 1]] = x
        pool.append(m.whole, k2, v2)
        out = pool.attend(m.batch, q)
        for s in range(len(m.rows)):
            a, b = m.start[s], m.start[s + 1] - (2 if s in bad else 0)
            assert torch.equal(out[a:b], clean[a:b])
            assert not torch.isfinite(out[b:m.start[s + 1]]).any()
    pool.check()


@pytest.mark.parametrize("rows,cache", [p for p in PAIRS if p[1] != "q8"])
@pytest.mark.parametrize("hd,nh,nkv", [(128, 8, 2), (256, 4, 1), (64, 4, 4)])
@pytest.mark.parametrize("spec", [([100], [300]), ([3], [250]), ([70, 1], [140, 133])], ids=str)
def test_an_infinite_value_that_every_row_sees(hip_ctx, rows, cache, hd, nh, nkv, spec):
    """It shares a tile with positions that are hidden from some rows."""
    def change(m, k, v):
        first = m.lens[0] - m.rows[0]
        v[first - 1, :, ::2] = math.inf
        v[first - 1, :, 1::2] = math.nan
    m, q, k, v, out = run_attention(hip_ctx, rows, cache, hd, nh, nkv, 64, spec, change=change)
    r = m.rows[0]
    assert (out[:r, :, ::2] == math.inf).all() and torch.isnan(out[:r, :, 1::2]).all()
    assert torch.isfinite(out[r:]).all()


def test_keys_of_minus_infinity_weigh_nothing(hip_ctx):
    def change(m, k, v):
        k[10:20] = -math.inf
    g = torch.Generator(device="cuda")
    m, q, k, v, out = run_attention(hip_ctx, "bf16", "bf16", 64, 4, 2, 32, ([1, 60], [100, 60]), change=change)
    # q of either sign: scores are NaN or infinite there; a row that does not see them is as before
    verify_some(m, q, k, v, out, 1)


def verify_some(m, q, k, v, out, s):
    a, b, r, n = m.start[s], m.all_start[s], m.rows[s], m.lens[s]
    last = torch.arange(n - r, n, device="cuda")
    o, spread, reach = ref.attention(q[a:a + r].double(), k[b:b + n].double(), v[b:b + n].double(), last, q.shape[-1] ** -0.5)
    close(out[a:a + r], o, ref.attention_tolerance(o, spread, reach, q.dtype, q.shape[-1], n, half_step(q.dtype)))


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
@pytest.mark.parametrize("rows,cache", [("f32", "q8"), ("bf16", "bf16"), ("f16", "q8")])
def test_scales(hip_ctx, rows, cache, scale):
    verify(*run_attention(hip_ctx, rows, cache, 64, 4, 2, 32, ([1, 70, 3], [100, 90, 65]), scale=scale), scale, rows)


@pytest.mark.parametrize("rows,cache", [("f32", "q8"), ("bf16", "bf16")])
@pytest.mark.parametrize("size", [1e-30, 1e30])
def test_values_far_from_one(hip_ctx, rows, cache, size):
    """Weights times scales of this size stay in range, queries as well."""
    def change(m, k, v):
        v *= size
        k /= 64
    m, q, k, v, out = run_attention(hip_ctx, rows, cache, 128, 4, 2, 32, ([1, 70], [333, 90]), change=change)
    verify(m, q, k, v, out, None, rows)


@pytest.mark.parametrize("rows,cache", [("f32", "q8"), ("bf16", "bf16")])
@pytest.mark.parametrize("hd,nh,nkv", [(64, 40, 1), (128, 5, 5), (64, 2, 1)])
def test_wide_groups_of_heads_and_wide_tables(hip_ctx, rows, cache, hd, nh, nkv):
    verify(*run_attention(hip_ctx, rows, cache, hd, nh, nkv, 32, ([1, 2, 1, 30], [700, 40, 1, 99]), extra_pages=3000), None, rows)


# ---- lists that are out of range ------------------------------------------------------

def filled(hip_ctx, spec, cache="q8", nkv=2, hd=64, page=32, **kw):
    m = Made(*spec, page, **kw)
    pool = hip_ctx.paged_kv(m.n_pages, nkv, hd, page_len=page, type=KV[cache], rope_dim=hd, rope_theta=1e4, max_pos=4096)
    g = gen(3)
    k, v = (torch.randn(m.all_start[-1], nkv, hd, generator=g, device="cuda").bfloat16() for _ in range(2))
    pool.append(m.whole, k, v)
    q = torch.randn(m.total, 2 * nkv, hd, generator=g, device="cuda").bfloat16()
    return m, pool, q


@pytest.mark.parametrize("what", ["page-low", "page-high", "len-long", "len-negative", "start-back", "start-past", "rows-many", "first-past", "shared-long"])
def test_bad_lists_are_reported(hip_ctx, what):
    """The sequence at fault is reported and left out; nothing is written outside
    and the other sequences' rows are as without it."""
    m, pool, q = filled(hip_ctx, ([1, 2, 70], [100, 90, 130]))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    first, shared = i32([0, 1]), i32([32])
    want = pool.attend_prefix(m.batch, q, first, shared)
    pool.check()
    start, length, table = m.t
    keep, kept = [0, 2], pool.read(m.whole, torch.bfloat16)
    hurt = {"page-low": (table[1], 1, -5), "page-high": (table[1], 1, m.n_pages), "len-long": (length, 1, 10 ** 6), "len-negative": (length, 1, -3),
            "start-back": (start, 2, 0), "start-past": (start, 3, m.total + 1), "rows-many": None, "first-past": (first, 1, 9), "shared-long": (shared, 0, 10 ** 6)}[what]
    batch = m.batch
    if what == "rows-many":
        batch, keep = oa.PagedBatch(*m.t, n_rows=m.total, max_new=2), [0, 1]
    else:
        x, i, bad = hurt
        x[i] = bad
        keep = {"start-back": [0], "start-past": [0, 1], "first-past": [1, 2], "shared-long": [1, 2]}.get(what, keep)
    out = torch.full_like(q, 3.0)
    pool.attend_prefix(batch, q, first, shared, out=out)
    for s in keep:
        a, b = m.start[s], m.start[s + 1]
        # (where the cut of the key axis changes, the sums' order does)
        assert (out[a:b].float() - want[a:b].float()).abs().max() < 0.03
    with pytest.raises(oa.HipError, match="page outside" if what.startswith("page") else "out of range"):
        pool.check()
    pool.check()                                             # (forgotten once told)
    if what in ("page-low", "page-high", "len-long", "start-past"):
        z = torch.zeros(m.total, 2, 64, dtype=torch.bfloat16, device="cuda")
        if what.startswith("page"):
            length[1] = 34                                   # the rows themselves are on the bad page
        pool.append(batch, z, z)
        with pytest.raises(oa.HipError):
            pool.check()
        if what.startswith("page"):
            table[1, 1], length[1] = m.table[1][1], 90
        elif what == "len-long":
            length[1] = 90
        else:
            start[3] = m.start[3]
        now = pool.read(m.whole, torch.bfloat16)
        rows = [m.all_start[s] + p for s in range(3) for p in range(m.lens[s] - (m.rows[s] if s != (2 if what == "start-past" else 1) else 0))]
        for x, y in zip(now, kept):
            assert torch.equal(x[rows], y[rows])
    pool.check()


def test_rotation_positions_out_of_range_are_reported(hip_ctx):
    m, pool, q = filled(hip_ctx, ([3], [3]))
    k = torch.ones(m.total, 2, 64, dtype=torch.bfloat16, device="cuda")
    before = pool.read(m.batch, torch.bfloat16)[0].clone()
    out = torch.full_like(q, 5.0)
    pool.append(m.batch, k, k, q=q, q_out=out, rope_pos=torch.tensor([[0, 4096, -1]], dtype=torch.int32, device="cuda"))
    with pytest.raises(oa.HipError, match="rotation position"):
        pool.check()
    after = pool.read(m.batch, torch.bfloat16)[0]
    assert torch.equal(after[0], k[0]) and torch.equal(after[1:3], before[1:3])
    assert not (out[0] == 5).all() and (out[1:] == 5).all()


# ---- refusals ----------------------------------------------------------------------------

def test_pools_that_are_refused(hip_ctx):
    for status, kw in ((3, dict(hd=96)), (3, dict(page_len=48)), (3, dict(type=oa.Q4_K)), (2, dict(nkv=0)), (2, dict(n_pages=0)),
                       (2, dict(rope_dim=65)), (2, dict(rope_dim=130)), (2, dict(rope_dim=64, max_pos=(1 << 24) + 1)), (2, dict(rope_dim=64, rope_theta=-1.0)),
                       (2, dict(rope_dim=8, rope_axis=[0, 1, 2, 4]))):
        with pytest.raises(oa.HipError) as e:
            hip_ctx.paged_kv(**{**dict(n_pages=2, nkv=2, hd=64), **kw})
        assert e.value.status == status, kw
    with pytest.raises(ValueError, match="axes for"):
        hip_ctx.paged_kv(2, 2, 64, rope_dim=8, rope_axis=[0, 1])
    with pytest.raises(oa.HipError) as e:
        hip_ctx.paged_kv(2 ** 31 - 1, 64, 256, page_len=256, type=oa.KV_BF16)
    assert e.value.status == 4                               # no memory for it, and nothing broken by that
    hip_ctx.paged_kv(2, 2, 64).free()


def test_calls_that_are_refused(hip_ctx):
    m, pool, q = filled(hip_ctx, ([1, 2], [10, 90]))
    k = torch.zeros(m.total, 2, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(oa.HipError, match="query heads"):
        pool.attend(m.batch, q[:, :3])
    with pytest.raises(oa.HipError, match="workspace"):
        pool.attend_prefix(m.batch, q, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), torch.tensor([32], dtype=torch.int32, device="cuda"),
                           workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    with pytest.raises(oa.HipError, match="groups"):
        pool.attend_prefix(m.batch, q, torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(oa.HipError, match="scale"):
        pool.attend(m.batch, q, scale=math.nan)
    with pytest.raises(oa.HipError, match="16-byte"):
        wide = torch.zeros(m.total, 4, 68, dtype=torch.bfloat16, device="cuda")
        pool.attend(m.batch, wide[..., :64])
    with pytest.raises(oa.HipError, match="16-byte"):
        flat = torch.zeros(m.total * 256 + 1, dtype=torch.bfloat16, device="cuda")
        pool.attend(m.batch, flat[1:].view(m.total, 4, 64))
    with pytest.raises(oa.HipError, match="eps"):
        pool.append(m.batch, k, k, eps=-1.0)
    with pytest.raises(oa.HipError, match="max_new"):
        pool.attend(oa.PagedBatch(*m.t, n_rows=m.total, max_new=0), q)
    with pytest.raises(oa.HipError, match="negative"):
        pool.attend(oa.PagedBatch(*m.t, n_rows=m.total, max_new=-1), q)
    half = hip_ctx.paged_kv(4, 2, 64, type=oa.KV_F16)
    with pytest.raises(oa.HipError, match="its own type"):
        half.append(m.batch, k, k)
    for bad in (dict(k=k.double(), v=k.double()), dict(k=k, v=k.half()), dict(k=k[:1], v=k), dict(k=k[..., :32], v=k), dict(k=k.cpu(), v=k)):
        with pytest.raises(ValueError):
            pool.append(m.batch, **bad)
    with pytest.raises(ValueError, match="rope_pos"):
        pool.append(m.batch, k, k, rope_pos=torch.zeros(1, m.total, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="q_norm"):
        pool.append(m.batch, k, k, q=q, q_norm=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="gradient"):
        pool.attend(m.batch, q.clone().requires_grad_())
    with pytest.raises(ValueError, match="int32"):
        oa.PagedBatch(m.t[0].long(), m.t[1], m.t[2], n_rows=m.total)
    # nothing to do is no mistake
    none = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert pool.attend(oa.PagedBatch(*m.t, n_rows=0), none).shape == (0, 4, 64)
    empty = [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 0)]
    assert pool.attend(oa.PagedBatch(empty[0], empty[1], torch.zeros(0, 3, dtype=torch.int32, device="cuda"), n_rows=m.total), q).shape == q.shape
    pool.free()
    with pytest.raises(ValueError, match="freed"):
        pool.attend(m.batch, q)


def test_outputs_that_overlap_are_refused(hip_ctx):
    m, pool, q = filled(hip_ctx, ([1, 2], [10, 90]))
    k = torch.zeros(m.total, 2, 64, dtype=torch.bfloat16, device="cuda")
    one, head = torch.zeros(1, 4, 64, dtype=q.dtype, device="cuda").expand(m.total, 4, 64), torch.zeros_like(q)[:, :1].expand_as(q)
    near = torch.zeros(m.total * 256 + 256, dtype=q.dtype, device="cuda").as_strided(q.shape, (256, 32, 1))
    for out in (one, head, near):
        with pytest.raises(oa.HipError, match="overlap"):
            pool.attend(m.batch, q, out=out)
        with pytest.raises(oa.HipError, match="overlap"):
            pool.append(m.batch, k, k, q=q, q_out=out)
        with pytest.raises(oa.HipError, match="overlap"):
            pool.read(m.batch, q.dtype, k=torch.empty_like(k), v=out[:, :2])
    with pytest.raises(oa.HipError, match="out is q"):
        pool.attend(m.batch, q, out=q)
    # inputs may: all rows and heads the same
    assert torch.equal(pool.attend(m.batch, one), pool.attend(m.batch, one.contiguous()))
    pool.check()


# ---- as they are used -----------------------------------------------------------------------

@pytest.mark.parametrize("rows,cache,hd,nh,nkv,page", [("f32", "q8", 256, 16, 2, 64), ("bf16", "bf16", 128, 8, 4, 32)])
def test_a_prompt_forked_and_continued(hip_ctx, rows, cache, hd, nh, nkv, page):
    """One prompt in two pieces, then three answers that share its whole pages,
    token by token: rotation, store and attention of every step against 64 bits."""
    g, dt, theta, eps = gen(11), DT[rows], 1e5, 1e-6
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    prompt, steps, n = 5 * page + 7, 6, 3
    whole = prompt // page
    pool = hip_ctx.paged_kv(40, nkv, hd, page_len=page, type=KV[cache], rope_dim=hd // 2, rope_theta=theta)
    qw, kw = 1 + 0.1 * rand(hd), 1 + 0.1 * rand(hd)
    axis = [0] * (hd // 4)
    wide = torch.float32 if cache == "q8" else DT[cache]

    def step(batch, positions):
        q, k, v = (rand(len(positions), h, hd).to(dt) for h in (nh, nkv, nkv))
        got = pool.append(batch, k, v, q=q, q_norm=qw, k_norm=kw, eps=eps)
        want = ref.rotated(q, qw, eps, i32([positions]), axis, theta)
        close(got, want, half_step(dt) * want.abs() + 2.0 ** -20)
        return got

    def check(q, out, table, length, n_rows):
        b = oa.PagedBatch(i32([0, length]), i32([length]), i32([table]), n_rows=length)
        k, v = pool.read(b, wide)
        last = torch.arange(length - n_rows, length, device="cuda")
        o, spread, reach = ref.attention(q.double(), k.double(), v.double(), last, hd ** -0.5)
        close(out, o, ref.attention_tolerance(o, spread, reach, dt, hd, length, 0.0 if rows == "f32" else half_step(dt)))

    pages = list(range(whole + 1))
    for a, b in ((0, 2 * page + 5), (2 * page + 5, prompt)):
        batch = oa.PagedBatch(i32([0, b - a]), i32([b]), i32([pages]), n_rows=b - a)
        q = step(batch, list(range(a, b)))
        check(q, pool.attend(batch, q), pages, b, b - a)
    # the prompt's last, partial page goes along as a copy of each answer's own
    tail = prompt - whole * page
    b = oa.PagedBatch(i32([0, tail]), i32([prompt]), i32([pages]), n_rows=tail)
    k, v = pool.read(b, wide)
    tables = [pages[:whole] + [20 + 3 * s, 21 + 3 * s] for s in range(n)]
    still = torch.zeros(1, n * tail, dtype=torch.int32, device="cuda")
    pool.append(oa.PagedBatch(i32([tail * s for s in range(n + 1)]), i32([prompt] * n), i32(tables), n_rows=n * tail),
                k.repeat(n, 1, 1), v.repeat(n, 1, 1), rope_pos=still)
    first, shared = i32([0, n]), i32([prompt])
    batch = oa.PagedBatch(i32(list(range(n + 1))), i32([prompt] * n), i32(tables), n_rows=n, max_new=1)
    for t in range(steps):
        batch.kv_len += 1
        q = step(batch, [prompt + t] * n)
        out = pool.attend_prefix(batch, q, first, shared)
        alone = pool.attend(batch, q)
        for s in range(n):
            check(q[s:s + 1], out[s:s + 1], tables[s], prompt + t + 1, 1)
            check(q[s:s + 1], alone[s:s + 1], tables[s], prompt + t + 1, 1)
    pool.check()


def test_a_sessions_attention(hip_ctx, tmp_path):
    """The keys and values that a session holds, in pages: a decode step's
    attention from there is the session's own."""
    import numpy as np

    import clibs
    path = str(tmp_path / "c1.gguf")
    clibs.write_c1_gguf(path)
    model = hip_ctx.load(path)
    s = model.session(200)
    s.eval(clibs.ids(0, "prompt", 100, 4096))
    s.step(7)
    q, gate, o, pos = s.attn()
    a, n = model.arch, s.pos
    assert pos == n - 1
    kq, ks, vq, vs = (torch.from_numpy(x).cuda() for x in s.kv(a["n_layers"] - 1))
    k, v = ((c.view(n, a["nkv"], a["hd"]).float() * x.view(n, a["nkv"], 1)) for c, x in ((kq, ks), (vq, vs)))
    m = Made([n], [n], 32)
    pool = hip_ctx.paged_kv(m.n_pages, a["nkv"], a["hd"], page_len=32)
    pool.append(m.batch, k, v)
    stored = pool.read(m.batch, torch.float32)
    assert all((x - y).abs().max() <= 2.0 ** -22 * y.abs().max() for x, y in zip(stored, (k, v)))
    one = oa.PagedBatch(torch.tensor([0, 1], dtype=torch.int32, device="cuda"), m.t[1], m.t[2], n_rows=1)
    got = pool.attend(one, torch.from_numpy(q).cuda().view(1, a["nh"], a["hd"]))
    want = o / (1 / (1 + np.exp(-gate.astype(np.float64))))
    last = torch.tensor([n - 1], device="cuda")
    e, spread, reach = ref.attention(torch.from_numpy(q).cuda().view(1, a["nh"], a["hd"]).double(), k.double(), v.double(), last, a["hd"] ** -0.5)
    tol = ref.attention_tolerance(e, spread, reach, torch.float32, a["hd"], n, 0.0)
    close(got, e, tol + 2.0 ** -20 * spread)
    assert np.allclose(got.cpu().numpy().ravel(), want, rtol=1e-4, atol=1e-5)
    s.free()
    model.free()


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("rows,cache", [("f32", "q8"), ("bf16", "bf16")])
def test_captured_steps(hip_ctx, rows, cache, prefix):
    """A decode step in a graph, replayed as the lists' contents change, between
    eager steps of another batch."""
    g, dt, hd, nkv, nh, n = gen(2), DT[rows], 128, 2, 8, 5
    m = Made([1] * n, [300 + 40 * s for s in range(n)], 32, groups=(0, n) if prefix else (), shared=256 if prefix else 0, extra_pages=2)
    pool = hip_ctx.paged_kv(m.n_pages + 20, nkv, hd, page_len=32, type=KV[cache], rope_dim=64)
    held = torch.float32 if cache == "q8" else DT[cache]
    k0, v0 = (torch.randn(m.all_start[-1], nkv, hd, generator=g, device="cuda").to(held) for _ in range(2))
    pool.append(m.whole, k0, v0)
    table = m.t[2]
    for s in range(n):
        for i in range(-(-m.lens[s] // 32), table.shape[1]):
            table[s, i] = m.n_pages + 2 * s + i % 2           # pages to grow into
    q, k, v = (torch.randn(n, h, hd, generator=g, device="cuda").to(dt) for h in (nh, nkv, nkv))
    first, shared = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, n], [256]))

    def step():
        r = pool.append(m.batch, k, v, q=q)
        return pool.attend_prefix(m.batch, r, first, shared) if prefix else pool.attend(m.batch, r)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in range(6):
        m.t[1].add_(1)
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda").to(dt))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(step(), got)                      # the same work, eagerly
        torch.cuda.synchronize()
    pool.check()


def test_two_streams_at_once(hip_ctx):
    """Calls on one pool from two streams, each with a workspace of its own, and
    from a thread's stream that is not the tensors' own."""
    m, pool, q = filled(hip_ctx, ([1] * 8, [900 + 50 * s for s in range(8)]))
    want = pool.attend(m.batch, q)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(20):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                o.append(pool.attend(m.batch, q))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, want) for x in o)
    pool.check()


def test_a_pool_past_32_bits(hip_ctx):
    """Pages at 4 GiB and behind hold what near ones do."""
    nkv, hd, page = 8, 256, 256
    n = 2500                                                 # 2 MiB a page: 4.9 GiB
    pool = hip_ctx.paged_kv(n, nkv, hd, page_len=page, type=oa.KV_BF16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    g = gen(9)
    k, v = (torch.randn(300, nkv, hd, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(300, 2 * nkv, hd, generator=g, device="cuda").bfloat16()
    outs = []
    for table in ([0, 1], [n - 1, 2100], [2050, n - 2]):
        b = oa.PagedBatch(i32([0, 300]), i32([300]), i32([table]), n_rows=300)
        pool.append(b, k, v)
        one = oa.PagedBatch(i32([0, 1]), i32([300]), i32([table]), n_rows=1)
        outs.append((*pool.read(b, torch.bfloat16), pool.attend(b, q), pool.attend(one, q[:1])))
    for o in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(o, outs[0]))
    assert torch.equal(outs[0][0], k) and torch.equal(outs[0][1], v)
    pool.check()
    pool.free()


def test_a_pool_outlives_its_context():
    ctx = oa.Context(0)
    m = Made([2], [40], 32)
    pool = ctx.paged_kv(m.n_pages, 2, 64, page_len=32, type=oa.KV_BF16)
    ctx.close()
    k = torch.ones(40, 2, 64, dtype=torch.bfloat16, device="cuda")
    pool.append(m.whole, k, k)
    assert torch.equal(pool.attend(m.batch, torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")), torch.ones(2, 4, 64, dtype=torch.bfloat16, device="cuda"))
    pool.check()
    pool.free()
