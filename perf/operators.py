"""The paged key/value cache and the attention that reads it, as measurable cases.

A server keeps the keys and values of its requests in pages of one pool per
layer. Three operators work on it, each on a ragged batch: sequence s owns the
rows [start[s], start[s + 1]), the last of them at position length[s] - 1, and
``table[s]`` names its pages.

* "append": the rows' keys are rotated and stored with the values (8-bit codes
  with a scale per position and head, or 16-bit values), the queries rotated;
  the stored rows are read back;
* "attend": causal attention of the batch's rows over the pages: prompts,
  continued prompts, single tokens, and batches of both;
* "prefix": the same where groups of sequences share their first pages.

The plain forms keep the pool position by position; the library keeps its own
layout, filled once in ``prepare``, as a server's cache is filled by the steps
before.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MAX_POS = 1 << 20


def listed():
    return [
        # the attention layers of the 35B shape: one request's next token written (normed, rotated, 8-bit)
        {"name": "append 1 q8", "kind": "append", "nh": 16, "nkv": 2, "hd": 256, "rows": "f32", "cache": "q8", "page": 64,
         "mode": "decode", "n": 1, "context": 4097, "new": 1, "rope": 64, "theta": 1e7, "axes": 1, "norm": True, "offset": 0},
        # a full decode batch of a generic grouped-query model, far into long contexts
        {"name": "append 128 bf16", "kind": "append", "nh": 32, "nkv": 8, "hd": 128, "rows": "bf16", "cache": "bf16", "page": 64,
         "mode": "decode", "n": 128, "context": 1500, "new": 1, "rope": 128, "theta": 5e5, "axes": 1, "norm": False, "offset": 700000},
        # a long prompt's rows at the 35B shape
        {"name": "append prompt 8191 q8", "kind": "append", "nh": 16, "nkv": 2, "hd": 256, "rows": "f32", "cache": "q8", "page": 64,
         "mode": "prompt", "n": 1, "context": 8191, "new": 8191, "rope": 64, "theta": 1e7, "axes": 1, "norm": True, "offset": 0},
        # prompts with images: positions in time, height and width, lengths ragged
        {"name": "append images bf16 q8", "kind": "append", "nh": 32, "nkv": 8, "hd": 128, "rows": "bf16", "cache": "q8", "page": 32,
         "mode": "ragged", "n": 7, "context": 2311, "new": 2000, "rope": 128, "theta": 1e6, "axes": 3, "norm": True, "offset": 0},
        # the benchmark's decode step at the 35B shape: one token after 4096 positions
        {"name": "attend 1 x 4097 q8", "kind": "attend", "nh": 16, "nkv": 2, "hd": 256, "rows": "f32", "cache": "q8", "page": 64,
         "mode": "decode", "n": 1, "context": 4097, "new": 1},
        # a decode batch of a generic grouped-query model, contexts of very different lengths, two padding rows
        {"name": "attend 64 ragged bf16", "kind": "attend", "nh": 32, "nkv": 8, "hd": 128, "rows": "bf16", "cache": "bf16", "page": 64,
         "mode": "decode", "n": 64, "context": 16000, "new": 1, "padded": 2},
        # the largest: a prompt of 8192 tokens
        {"name": "attend prompt 8192 bf16", "kind": "attend", "nh": 32, "nkv": 8, "hd": 128, "rows": "bf16", "cache": "bf16", "page": 128,
         "mode": "prompt", "n": 1, "context": 8192, "new": 8192},
        # prompts continued from their 8-bit caches at the 35B shape
        {"name": "attend ragged f32 q8", "kind": "attend", "nh": 16, "nkv": 2, "hd": 256, "rows": "f32", "cache": "q8", "page": 64,
         "mode": "ragged", "n": 5, "context": 2777, "new": 1200},
        # a scheduler's mixed step: a piece of one prompt beside other requests' single tokens, small heads
        {"name": "attend mixed f16", "kind": "attend", "nh": 12, "nkv": 4, "hd": 64, "rows": "f16", "cache": "f16", "page": 32,
         "mode": "mixed", "n": 24, "context": 2500, "new": 512},
        # one system prompt before many requests, 35B shape
        {"name": "prefix 48 x 8000 q8", "kind": "prefix", "nh": 16, "nkv": 2, "hd": 256, "rows": "f32", "cache": "q8", "page": 64,
         "mode": "decode", "n": 48, "context": 8700, "new": 1, "shared": 8000, "groups": 1},
        # three of them, 16-bit cache
        {"name": "prefix 3 groups bf16", "kind": "prefix", "nh": 32, "nkv": 8, "hd": 128, "rows": "bf16", "cache": "bf16", "page": 64,
         "mode": "decode", "n": 60, "context": 9000, "new": 1, "shared": 8190, "groups": 3},
        # a few answers to one short prompt, drawn at once
        {"name": "prefix 4 x 500 f16 q8", "kind": "prefix", "nh": 8, "nkv": 2, "hd": 64, "rows": "f16", "cache": "q8", "page": 32,
         "mode": "decode", "n": 4, "context": 530, "new": 1, "shared": 500, "groups": 1},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    c = {"kind": rng.choice(("append", "attend", "attend", "prefix"))}
    c["nh"], c["nkv"], c["hd"] = rng.choice(((16, 2, 256), (32, 2, 256), (8, 2, 64), (32, 8, 128), (12, 4, 64), (12, 12, 64),
                                             (28, 4, 128), (15, 5, 64), (6, 1, 128), (16, 16, 128), (8, 4, 256)))
    c["rows"], c["cache"] = rng.choice((("f32", "q8"), ("f32", "q8"), ("bf16", "q8"), ("f16", "q8"), ("bf16", "bf16"), ("f16", "f16")))
    c["page"] = rng.choice((32, 64, 128, 256))
    if c["kind"] == "append":
        c["mode"] = rng.choice(("decode", "prompt", "ragged", "mixed"))
        c["n"] = _log(rng, 1, 128 if c["mode"] == "decode" else 6)
        c["context"] = _log(rng, 1, 4000 if c["mode"] == "prompt" else 2000)
        c["new"] = {"decode": 1, "prompt": c["context"]}.get(c["mode"]) or _log(rng, 1, c["context"])
        c["axes"], c["norm"] = rng.choice((1, 1, 3)), rng.random() < 0.5
        c["rope"] = rng.choice((c["hd"], c["hd"] // 2, c["hd"] // 4))
        c["theta"], c["offset"] = rng.choice((1e4, 5e5, 1e7)), 0 if rng.random() < 0.5 else _log(rng, 1, 900000)
        return c
    c["mode"] = rng.choice(("decode", "decode", "ragged", "mixed")) if c["kind"] == "prefix" else \
        rng.choice(("decode", "decode", "prompt", "ragged", "mixed"))
    most = 2e8 / (c["nkv"] * c["hd"])                       # cached positions of the batch
    c["n"] = _log(rng, 1 if c["kind"] == "attend" else 2, 100 if c["mode"] == "decode" else 12)
    c["context"] = _log(rng, 1 if c["kind"] == "attend" else 40, int(min(40000 if c["mode"] == "decode" else 4500, most / c["n"])))
    fit = max(1, int(5e8 / (c["n"] * c["nh"] * c["context"])))
    c["new"] = {"decode": 1, "prompt": c["context"]}.get(c["mode"]) or min(fit, _log(rng, 1, c["context"]))
    if c["mode"] == "prompt":
        c["n"] = max(1, min(c["n"], fit // c["context"]))
    if c["kind"] == "prefix":
        c["shared"] = min(c["context"] - 1, _log(rng, 33, c["context"]))
        c["new"] = min(c["new"], c["context"] - c["shared"])
        c["groups"] = rng.randint(1, min(3, c["n"]))
    return c


# ---- batches -------------------------------------------------------------------------

def _lengths(c):
    """([rows], [length]) of the case's sequences; the first one has the case's context."""
    rng = random.Random("%(n)d %(context)d %(new)d %(hd)d" % c)
    shared, rows, lens = c.get("shared", 0), [], []
    for s in range(c["n"]):
        new = {"decode": 1, "prompt": c["new"], "mixed": c["new"] if s == 0 else 1}.get(c["mode"]) or (c["new"] if s == 0 else rng.randint(1, c["new"]))
        low = max(shared + new, c["context"] // 16)
        length = c["context"] if s == 0 or c["mode"] == "prompt" else max(shared + new, _log(rng, max(1, low), max(low, c["context"])))
        if s >= c["n"] - c.get("padded", 0):
            length = 0                                      # a padding row, in no context
        rows.append(new)
        lens.append(length)
    return rows, lens


def _groups(c):
    """The first sequence of each group, and the number of sequences."""
    return [s * c["n"] // c["groups"] for s in range(c["groups"] + 1)]


def _pages(c, rng):
    """(table, pages of the pool): each sequence's pages, in no order; a group's shared whole pages once."""
    rows, lens = _lengths(c)
    need = [-(-n // c["page"]) for n in lens]
    of_group = {}
    if c["kind"] == "prefix":
        for a, b in zip(_groups(c)[:-1], _groups(c)[1:]):
            of_group.update({s: a for s in range(a, b)})
    whole = c.get("shared", 0) // c["page"]
    table = [[-1] * max(1, max(need)) for _ in need]
    places = [(s, i) for s, n in enumerate(need) for i in range(n) if not (of_group.get(s, s) != s and i < whole)]
    ids = list(range(len(places) + 3))
    rng.shuffle(ids)
    for (s, i), p in zip(places, ids):
        table[s][i] = p
    for s, a in of_group.items():
        table[s][:whole] = table[a][:whole]
    return table, len(ids)


def _quantised(x):
    """8-bit codes of rows of a head, and their scale."""
    most = x.abs().amax(-1, keepdim=True)
    codes = torch.round(x * torch.where(most > 0, 127.0 / most, torch.zeros_like(most))).clamp(-127, 127)
    return codes.to(torch.int8), most[..., 0] / 127.0


def _positions(c, rows, lens, dev):
    """Positions of the rotation: [axes, rows]. With three axes, text runs along
    all of them, and every 300 rows hold an image of 16 x 15 places."""
    p = torch.cat([torch.arange(n - r, n, device=dev) for r, n in zip(rows, lens)]) + c["offset"]
    if c["axes"] == 1:
        return p[None].int()
    i = p % 300
    image = i < 240
    return torch.stack([p - torch.where(image, i, 0), p - torch.where(image, i - i // 15, 0), p - torch.where(image, i - i % 15, 0)]).int()


def _axis(c):
    """The axis of each frequency: time, height and width in turn."""
    return [i % c["axes"] for i in range(c["rope"] // 2)]


def prepare(case, seed):
    c, dev, f = case, "cuda", TYPES[case["rows"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rows, lens = _lengths(c)
    table, n_pages = _pages(c, random.Random(seed))
    total = sum(rows)
    start = [sum(rows[:s]) for s in range(c["n"] + 1)]
    st = {"case": c, "total": total, "most_rows": max(rows), "most_len": max(lens), "n_pages": n_pages,
          "start": torch.tensor(start, dtype=torch.int32, device=dev), "length": torch.tensor(lens, dtype=torch.int32, device=dev),
          "table": torch.tensor(table, dtype=torch.int32, device=dev)}
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    # the pool: keys with a few strong channels, values of any sign
    shape = (n_pages * c["page"], c["nkv"], c["hd"])
    strong = 1.0 + 2.0 * (torch.rand(c["nkv"], c["hd"], generator=g, device=dev) > 0.95)
    pool = {"k": rand(*shape) * strong, "v": rand(*shape) + 0.3 * rand(c["nkv"], c["hd"])}
    for w in ("k", "v"):
        if c["cache"] == "q8":
            st[w + "_pool"], st[w + "_scale"] = _quantised(pool[w])
        else:
            st[w + "_pool"] = pool[w].to(TYPES[c["cache"]])
    st["q"] = (rand(total, c["nh"], c["hd"]) * 1.3).to(f)
    if c["kind"] == "append":
        st["k"] = (rand(total, c["nkv"], c["hd"]) * strong).to(f)
        st["v"] = rand(total, c["nkv"], c["hd"]).to(f)
        st["pos"] = _positions(c, rows, lens, dev)
        if c["norm"]:
            st["q_norm"], st["k_norm"] = (1.0 + 0.1 * rand(c["hd"]) for _ in range(2))
    if c["kind"] == "prefix":
        st["first"] = torch.tensor(_groups(c), dtype=torch.int32, device=dev)
        st["shared"] = torch.full((c["groups"],), c["shared"], dtype=torch.int32, device=dev)
    if own:
        _fill(st)
    return st


# ---- the library's calls ---------------------------------------------------------------

_ctx = []


def _fill(st):
    """The library's pool with the same contents: every page is written as a sequence of its own."""
    import ornithology_amd as oa
    if not _ctx:
        _ctx.append(oa.Context(0))
    c = st["case"]
    kind = {"q8": oa.KV_Q8, "bf16": oa.KV_BF16, "f16": oa.KV_F16}[c["cache"]]
    rope = dict(rope_dim=c["rope"], rope_theta=c["theta"], max_pos=MAX_POS, rope_axis=_axis(c)) if c["kind"] == "append" else {}
    st["cache"] = _ctx[0].paged_kv(st["n_pages"], c["nkv"], c["hd"], page_len=c["page"], type=kind, **rope)
    st["batch"] = oa.PagedBatch(st["start"], st["length"], st["table"], max_new=st["most_rows"], n_rows=st["total"])
    n, dev = st["n_pages"], st["q"].device
    whole = oa.PagedBatch(torch.arange(0, (n + 1) * c["page"], c["page"], dtype=torch.int32, device=dev),
                          torch.full((n,), c["page"], dtype=torch.int32, device=dev),
                          torch.arange(n, dtype=torch.int32, device=dev)[:, None], max_new=c["page"], n_rows=n * c["page"])
    k, v = ((st[w + "_pool"].float() * st[w + "_scale"][..., None]) if c["cache"] == "q8" else st[w + "_pool"] for w in ("k", "v"))
    still = torch.zeros(c.get("axes", 1), n * c["page"], dtype=torch.int32, device=dev)
    st["cache"].append(whole, k, v, rope_pos=still)


def _own_run(st):
    c, cache, batch = st["case"], st["cache"], st["batch"]
    if c["kind"] == "attend":
        return [cache.attend(batch, st["q"])]
    if c["kind"] == "prefix":
        return [cache.attend_prefix(batch, st["q"], st["first"], st["shared"])]
    q = cache.append(batch, st["k"], st["v"], q=st["q"], rope_pos=st["pos"], q_norm=st.get("q_norm"), k_norm=st.get("k_norm"), eps=1e-6)
    k, v = cache.read(batch, torch.float16 if c["cache"] == "f16" else torch.bfloat16)
    return [q, k, v]


# ---- plain forms -----------------------------------------------------------------------

def _row_places(st):
    """(sequence, position, pool row) of each of the batch's rows."""
    c, start = st["case"], st["start"].long()
    row = torch.arange(st["total"], device=start.device)
    s = torch.searchsorted(start, row, right=True) - 1
    p = st["length"].long()[s] - (start[s + 1] - row)
    at = st["table"].long()[s, p.clamp(min=0) // c["page"]] * c["page"] + p.clamp(min=0) % c["page"]
    return s, p, at


def _plain_rotated(x, w, st):
    c, half = st["case"], st["case"]["rope"] // 2
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    freq = c["theta"] ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    axis = torch.tensor(_axis(c), device=x.device)
    angle = st["pos"].double()[axis].T * freq               # far positions: 64 bits
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_append(st):
    c = st["case"]
    _, _, at = _row_places(st)
    q = _plain_rotated(st["q"], st.get("q_norm"), st).to(st["q"].dtype)
    k, v = _plain_rotated(st["k"], st.get("k_norm"), st), st["v"].float()
    out = [q]
    for w, x in (("k", k), ("v", v)):
        if c["cache"] == "q8":
            codes, scale = _quantised(x)
            st[w + "_pool"][at], st[w + "_scale"][at] = codes, scale
            out.append((st[w + "_pool"][at].float() * st[w + "_scale"][at][..., None]).bfloat16())
        else:
            st[w + "_pool"][at] = x.to(st[w + "_pool"].dtype)
            out.append(st[w + "_pool"][at])
    return out


def _plain_attend(st):
    c, dev = st["case"], st["q"].device
    n, nkv, hd, G, R, L = c["n"], c["nkv"], c["hd"], c["nh"] // c["nkv"], st["most_rows"], max(1, st["most_len"])
    s, p, _ = _row_places(st)
    j = torch.arange(st["total"], device=dev) - st["start"].long()[s]
    t = torch.arange(L, device=dev)
    at = st["table"].long().clamp(min=0)[:, t // c["page"]] * c["page"] + t % c["page"]        # [n, L]
    k, v = (st[w + "_pool"][at].float() for w in ("k", "v"))
    if c["cache"] == "q8":
        k, v = k * st["k_scale"][at][..., None], v * st["v_scale"][at][..., None]
    q = torch.zeros(n, R, c["nh"], hd, device=dev)
    q[s, j] = st["q"].float()
    last = torch.full((n, R), -1, device=dev)
    last[s, j] = p
    q = q.view(n, R, nkv, G, hd).permute(0, 2, 1, 3, 4).reshape(n * nkv, R * G, hd)
    k = k.permute(0, 2, 3, 1).reshape(n * nkv, hd, L)
    v = v.permute(0, 2, 1, 3).reshape(n * nkv, L, hd)
    x = torch.bmm(q, k.contiguous()).mul_(hd ** -0.5).view(n, nkv, R, G, L)
    seen = (t <= last[..., None])[:, None, :, None]
    x.masked_fill_(~seen, -math.inf)
    x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.bmm(x.view(n * nkv, R * G, L), v.contiguous()).view(n, nkv, R, G, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return [o.permute(0, 2, 1, 3, 4).reshape(n, R, c["nh"], hd)[s, j].to(st["q"].dtype)]


def run(state):
    if own:
        return _own_run(state)
    return _plain_append(state) if state["case"]["kind"] == "append" else _plain_attend(state)


# ---- what a pass cannot do without, and its exact results --------------------------------

def work(case):
    c = case
    rows, lens = _lengths(c)
    e, T = 4 if c["rows"] == "f32" else 2, sum(rows)
    position = c["nkv"] * (2 * c["hd"] + 8 if c["cache"] == "q8" else 4 * c["hd"])             # cached bytes
    if c["kind"] == "append":
        moved = T * c["hd"] * e * (2 * c["nh"] + 2 * c["nkv"])
        return {"bytes": moved + 2 * T * position + T * 4 * c["nkv"] * c["hd"], "flops": T * c["hd"] * 8.0 * (c["nh"] + 2 * c["nkv"])}
    held = sum(lens)
    if c["kind"] == "prefix":
        held -= (c["n"] - c["groups"]) * c["shared"]
    pairs = sum(r * (n - r) + r * (r + 1) // 2 if n else 0 for r, n in zip(rows, lens))
    return {"bytes": held * position + 2 * T * c["nh"] * c["hd"] * e, "flops": 4.0 * c["hd"] * c["nh"] * pairs}


def _exact_row_values(x, st):
    """Stored values of rows x in 64 bits, by the cache's type."""
    if st["case"]["cache"] != "q8":
        return x
    top = x.abs().max(dim=-1, keepdim=True).values
    step = top / 127
    return torch.where(top > 0, (x / torch.where(top > 0, step, top + 1)).round() * step, torch.zeros_like(x))


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["kind"] == "append":
        r = c["rope"]
        out = []
        for name in ("q", "k"):
            x = st[name].double()
            if st.get(name + "_norm") is not None:
                x = x / ((x * x).sum(-1, keepdim=True) / c["hd"] + 1e-6).sqrt() * st[name + "_norm"].double()
            y = x.clone()
            for i in range(r // 2):
                turn = st["pos"][i % c["axes"]].double() * math.exp(-2.0 * i / r * math.log(c["theta"]))
                co, si = turn.cos()[:, None], turn.sin()[:, None]
                y[..., i] = x[..., i] * co - x[..., i + r // 2] * si
                y[..., i + r // 2] = x[..., i] * si + x[..., i + r // 2] * co
            out.append(y)
        return [out[0], _exact_row_values(out[1], st), _exact_row_values(st["v"].double(), st)]
    G, page = c["nh"] // c["nkv"], c["page"]
    q = st["q"].double()
    o = torch.zeros_like(q)
    rows, lens = _lengths(c)
    begin = 0
    for s, (r, n) in enumerate(zip(rows, lens)):
        if n:
            places = (st["table"][s, :-(-n // page)].long()[:, None] * page + torch.arange(page, device=q.device)).reshape(-1)[:n]
            hidden = torch.arange(n, device=q.device)[None, :] > torch.arange(n - r, n, device=q.device)[:, None]
            for h in range(c["nh"]):
                kv = [st[w + "_pool"][places, h // G].double() * (st[w + "_scale"][places, h // G, None].double() if c["cache"] == "q8" else 1.0)
                      for w in ("k", "v")]
                x = q[begin:begin + r, h] @ kv[0].T.contiguous() / math.sqrt(c["hd"])
                o[begin:begin + r, h] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ kv[1]
        begin += r
    return [o]
