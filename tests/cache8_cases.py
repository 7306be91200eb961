"""Paged caches in all forms with awkward contents, and attention over them in 64 bits by definition."""
import math
import random

import torch

TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16, "f32": torch.float32}
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -126


def e4m3_grid():
    """All non-negative e4m3 numbers in ascending order: the i-th has the code i."""
    return [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8) if (8 + m) * 2.0 ** (e - 3) <= 448]


def quantise(x, form):
    """float32 rows -> (float64 values of the codes, float32 scales), by definition: the nearest number of the form, ties to even."""
    amax = x.abs().amax(-1)
    scale = torch.clamp_min((amax.double() / TOP[form]).float(), TINY)
    t = x.double() / scale.double().unsqueeze(-1)
    if form == "int8":
        code = torch.round(t)
    else:
        grid = torch.tensor(e4m3_grid(), dtype=torch.float64, device=x.device)
        a = t.abs().contiguous()
        hi = torch.searchsorted(grid, a).clamp(1, grid.numel() - 1)
        mid = (grid[hi - 1] + grid[hi]) / 2
        code = torch.where((a > mid) | ((a == mid) & (hi % 2 == 0)), grid[hi], grid[hi - 1]) * torch.where(t < 0, -1.0, 1.0)
    finite = torch.isfinite(x).all(-1)
    return (torch.where(finite.unsqueeze(-1), code, torch.zeros_like(code)),
            torch.where(finite, scale, torch.full_like(scale, math.nan)))


class Step:
    """requests: (tokens in the cache before the step, new tokens).  Pages in random order, unused table entries -1; a page's rows past
    the request's end hold what may be there: NaN (16 and 32 bits), code 0x7f and NaN scales (8 bits).  `shared`: groups as
    (requests, keys in common): the members' first keys are the first member's."""

    def __init__(self, requests, heads, kv, dim, form, act, page_size=16, seed=0, shared=(), pad=0, layers=2, layer=1, q_std=1.5,
                 k_std=0.6, v_std=1.0, table_wide=0, spare=2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        self.heads, self.kv, self.dim, self.form, self.act, self.layer, self.page_size = heads, kv, dim, form, act, layer, page_size
        self.requests, self.scale = requests, 1.0 / math.sqrt(dim)
        ends = [b + n for b, n in requests]
        need = [-(-e // page_size) for e in ends]
        order = list(range(sum(need) + spare))
        rng.shuffle(order)
        n_slots = len(requests) + 1
        slots = rng.sample(range(n_slots), len(requests))
        table = torch.full((n_slots, max(max(need) + 1, table_wide)), -1, dtype=torch.int32)
        k = [torch.randn((kv, e, dim), generator=gen, device="cuda") * k_std for e in ends]
        v = [torch.randn((kv, e, dim), generator=gen, device="cuda") * v_std for e in ends]
        for x in v:
            x *= torch.exp(torch.randn((kv, x.shape[1], 1), generator=gen, device="cuda"))
        for members, n in shared:
            for m in members[1:]:
                k[m][:, :n], v[m][:, :n] = k[members[0]][:, :n], v[members[0]][:, :n]
        shape = (len(order), layers, 2, kv, page_size)
        if form in TOP:
            self.pool = torch.full(shape + (dim,), 0x7f, dtype=torch.int8, device="cuda")
            self.scales = torch.full(shape, math.nan, device="cuda")
        else:
            self.pool = torch.full(shape + (dim,), math.nan, dtype=TYPES[form], device="cuda")
            self.scales = None
        self.k, self.v = [], []
        for r in range(len(requests)):
            both = []
            for which, x in ((0, k[r]), (1, v[r])):
                code, s = quantise(x, form) if form in TOP else (x.to(TYPES[form]), None)
                both.append(code.double() * s.double().unsqueeze(-1) if form in TOP else code.double())
                bits = code.float().to(TYPES[form]).view(torch.int8) if form in TOP else code
                for j in range(need[r]):
                    if which == 0:
                        table[slots[r], j] = order.pop()
                    page, live = int(table[slots[r], j]), min(page_size, ends[r] - j * page_size)
                    self.pool[page, layer, which, :, :live] = bits[:, j * page_size:j * page_size + live]
                    if s is not None:
                        self.scales[page, layer, which, :, :live] = s[:, j * page_size:j * page_size + live]
            self.k.append(both[0])
            self.v.append(both[1])
        if form in TOP:
            self.pool = self.pool.view(TYPES[form])
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.pos_list = [b + j for b, n in requests for j in range(n)] + [-1] * pad
        self.seq_list = [r for r, (_, n) in enumerate(requests) for _ in range(n)] + [0] * pad
        self.positions, self.seq, self.slots, self.table = ints(self.pos_list), ints(self.seq_list), ints(slots), table.cuda()
        self.n = len(self.pos_list)
        self.q = (torch.randn((self.n, heads * dim), generator=gen, device="cuda") * q_std).to(TYPES[act])
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def out(self):
        return torch.full_like(self.q, 77.0)

    def expected(self, window=0, hidden=()):
        """(results, bounds) in 64 bits; `hidden`: (request, key) pairs that have no page.

        The bound, with w the softmax's weights, A = sum w |v| and S = scale max_j sum_i |q_i k_ji|:
          half a step of the result's type, relative to the result;
          a weight's rounding: to half at 2^-11 (8-bit forms), to bfloat16 at 2^-8 (bfloat16 caches), in float else;
          a score's error e changes every weight by a factor within 1 +- 2 e: e = (d + 8) 2^-24 S for float sums in any order,
          2^-21 S for a float query in two halves and 2^-21 |s| for scores in units of log2 and their exponential;
          sums over n keys in float in any order: n 2^-23 A for the numerator and as much for the denominator;
          8-bit forms: a weight p_j vs_j in half is a multiple of 2^-24 of a unit, off by at most 2^-25 of it, where it is small.  The
          unit is chosen so that, with m = max p_j and c = max vs_j, the bound 2 m c (c rounded up to a power of two) is at least
          2^11 units when the unit is set, and the unit never shrinks, so a unit is at most 2^-10 m c.  The sum over n keys of
          codes up to C, divided by l >= m, is off by at most n C 2^-25 2^-10 c = n 2^-35 (C c), and C c is the largest value of a
          row of this scale (its largest element has the code C).  (It matters only where rows' scales differ by more than 2^20.)
        """
        g, d = self.heads // self.kv, self.dim
        want = torch.full((self.n, self.heads, d), 77.0, dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(want)
        p_err = {"int8": 2.0 ** -11, "e4m3": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 0.0}[self.form] if self.act == "bf16" else 2.0 ** -22
        half = torch.finfo(TYPES[self.act]).eps / 2
        gone = set(hidden)
        for t in range(self.n):
            pos, r = self.pos_list[t], self.seq_list[t]
            if pos < 0:
                continue
            lo = max(0, pos - window + 1) if window else 0
            keys = torch.tensor([j for j in range(lo, pos + 1) if (r, j) not in gone], dtype=torch.long, device="cuda")
            if keys.numel() == 0:
                want[t] = 0.0
                continue
            k, v = self.k[r][:, keys], self.v[r][:, keys]
            q = self.q[t].double().view(self.kv, g, d)
            s = torch.einsum("hgd,hkd->hgk", q, k) * self.scale
            big = (torch.einsum("hgd,hkd->hgk", q.abs(), k.abs()) * self.scale).amax(-1, keepdim=True)
            w = torch.softmax(s, -1)
            o = torch.einsum("hgk,hkd->hgd", w, v).reshape(self.heads, d)
            a = torch.einsum("hgk,hkd->hgd", w, v.abs()).reshape(self.heads, d)
            e = ((d + 8) * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -21) * big.reshape(self.heads, 1)
            want[t] = o
            floor = 0.0
            if self.form in TOP:
                floor = keys.numel() * 2.0 ** -35 * v.abs().amax((1, 2)).repeat_interleave(g).unsqueeze(-1)
            tol[t] = floor + half * o.abs() + (p_err + 2 * e + 2 * keys.numel() * 2.0 ** -23 + 2.0 ** -20) * a
        return want.view(self.n, -1), tol.view(self.n, -1)


def check(step, got, window=0, hidden=(), rows=None):
    want, tol = step.expected(window, hidden)
    got = got.double()
    if rows is not None:
        want, tol, got = want[rows], tol[rows], got[rows]
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(), tol[bad][:4].tolist())
