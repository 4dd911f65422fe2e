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
