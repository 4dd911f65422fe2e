"""The paged operators in 64 bits, from their formulas, on lists and tensors the
tests make (the device's torch in float64; no code of the library)."""
import math

import torch

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype):
    """How far a rounding to dtype is off at most, relative to the value."""
    return torch.finfo(dtype).eps / 2


def half_least(dtype):
    """How far a rounding to dtype is off at most next to zero: half of its smallest
    subnormal, whatever the value's own size (fp16: 2^-25)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rotated(x, w, eps, pos, axis, theta):
    """Rows x [n, heads, hd] normed with weights w (None: not) and rotated:
    pos [axes, n], axis of each frequency."""
    x = x.double()
    if w is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = len(axis)
    if not half:
        return x
    freq = torch.tensor([theta ** (-i / half) for i in range(half)], dtype=torch.float64, device=x.device)
    angle = (pos[list(axis)].double().T * freq)[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., 2 * half:]], -1)


def attention(q, k, v, last, scale):
    """(o, spread, reach) of q [n, nh, hd] over one sequence's k, v [len, nkv, hd]
    (float64): row r sees positions 0..last[r]. spread: sum p |v|; reach: the
    largest sum |q_i k_i| * scale of a row's visible keys."""
    n, nh, _ = q.shape
    G = nh // k.shape[1]
    t = torch.arange(k.shape[0], device=q.device)
    hidden = t[None] > last[:, None]
    o, spread, reach = (torch.zeros_like(q) for _ in range(3))
    for h in range(nh):
        kh, vh = k[:, h // G], v[:, h // G]
        s = (q[:, h] @ kh.T.contiguous() * scale).masked_fill(hidden, -math.inf)
        top = s.amax(-1, keepdim=True) if k.shape[0] else s.new_full((n, 1), -math.inf)
        p = torch.where(hidden, 0.0, (s - top.clamp(min=-1e300)).exp())
        l = p.sum(-1, keepdim=True)
        p = torch.where(l > 0, p / l, torch.zeros_like(p))
        o[:, h], spread[:, h] = p @ vh, p @ vh.abs()
        r = (q[:, h].abs() @ kh.abs().T.contiguous() * abs(scale)).masked_fill(hidden, 0.0)
        reach[:, h] = r.amax(-1, keepdim=True) if k.shape[0] else 0.0
    return o, spread, reach


def attention_tolerance(o, spread, reach, dtype, hd, positions, weight_step):
    """Element by element: the output's rounding; each weight's rounding
    (weight_step, relative, on the sum of p |v|); and what 32-bit sums lose. A
    score is a sum of hd products (f32 queries: of three terms each), off by a
    rounding 2^-24 of the running sum at each step: steps that add as a random
    walk stay within 4 sqrt(steps) of them with what four standard deviations
    leave out. The softmax doubles a score's error (numerator and sum), its
    argument is rounded twice more, and the sums over positions walk likewise."""
    u = 2.0 ** -24
    score = 4 * math.sqrt(3 * hd) * u * reach + 4 * u * reach
    sums = 4 * math.sqrt(3 * max(1, positions)) * u
    return half_step(dtype) * o.abs() + half_least(dtype) + spread * (weight_step + 2 * score + sums + 16 * u) + 1e-30


class Made:
    """A batch: rows and lengths per sequence, pages in random order (shared: as
    many leading pages are the group's first sequence's), and its tensors."""

    def __init__(self, rows, lens, page, seed=0, groups=(), shared=0, extra_rows=0, extra_pages=0, stray=-1):
        import random

        import ornithology_amd as oa
        rng = random.Random(seed)
        self.rows, self.lens, self.page = list(rows), list(lens), page
        self.start = [sum(rows[:i]) for i in range(len(rows) + 1)]
        need = [-(-n // page) for n in lens]
        first = {s: a for a, b in zip(groups[:-1], groups[1:]) for s in range(a, b)}
        whole = shared // page
        cells = [(s, i) for s, n in enumerate(need) for i in range(n) if first.get(s, s) == s or i >= whole]
        ids = list(range(len(cells) + 2))
        rng.shuffle(ids)
        self.n_pages = len(ids)
        table = [[stray] * (max([1] + need) + extra_pages) for _ in need]
        for (s, i), p in zip(cells, ids):
            table[s][i] = p
        for s, a in first.items():
            table[s][:whole] = table[a][:whole]
        self.table = table
        self.total = self.start[-1] + extra_rows
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.t = i32(self.start), i32(self.lens), i32(table)
        self.batch = oa.PagedBatch(*self.t, n_rows=self.total, max_new=max(rows) if rows else 0)
        # every sequence's whole contents as rows, to fill and to read the pool
        self.all_start = [sum(lens[:i]) for i in range(len(lens) + 1)]
        self.whole = oa.PagedBatch(i32(self.all_start), self.t[1], self.t[2], n_rows=self.all_start[-1], max_new=max([0] + self.lens))

    def positions(self):
        """Of each row that a sequence owns."""
        return [n - r + j for r, n in zip(self.rows, self.lens) for j in range(r)]
