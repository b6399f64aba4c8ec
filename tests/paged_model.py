"""Plain models of the paged cache's operators: attention in 64 bits over explicit row lists, pages in Python ints."""
import math

import numpy as np
import torch

N_ROT = 64


def make_rows(fmt, x, n_rot=N_ROT):
    """f32 rows [n, dim] in a row format, by the store operators' rules."""
    n, dim = x.shape
    if fmt == "f32":
        return dict(raw=x.half().float().contiguous())
    if fmt == "row":
        scale = x.abs().amax(1, keepdim=True).clamp_min(1e-4) / 448.0
        return dict(codes=(x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scales=scale)
    nope = dim - n_rot
    b = x[:, :nope].reshape(n, nope // 64, 64)
    scale = torch.exp2(torch.ceil(torch.log2(b.abs().amax(2).clamp_min(1e-4) / 448.0)))
    codes = torch.zeros((n, dim), dtype=torch.uint8, device=x.device)
    codes[:, :nope] = (b / scale[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, nope)
    return dict(codes=codes, scales=scale.contiguous(), tail=x[:, nope:].contiguous() if n_rot else None)


def row_values(fmt, st, n_rot=N_ROT):
    """What the stored rows stand for, in 64 bits."""
    if fmt == "f32":
        return st["raw"].double()
    v = st["codes"].view(torch.float8_e4m3fn).double()
    if fmt == "row":
        return v * st["scales"].double()
    nope = v.shape[1] - n_rot
    v[:, :nope] *= st["scales"].double().repeat_interleave(64, 1)
    if n_rot:
        v[:, nope:] = st["tail"].double()
    return v


def visible(p, window, n_first):
    return [j for j in range(p + 1) if window == 0 or j > p - window or j < n_first]


def row_factors(fmt, st, n_rot=N_ROT):
    """r_j of every row, in 64 bits: 1 for f32 rows and for rows of ordinary size, which are held as f16 numbers; else the
    scale of a row, or the largest power of two that is at most its largest block scale, or its largest tail value / 256."""
    if fmt == "f32":
        return torch.ones(st["raw"].shape[0], dtype=torch.float64, device=st["raw"].device)
    if fmt == "row":
        r = st["scales"][:, 0].double()
        return torch.where((r < 2.0 ** -18) | (r > 2.0 ** 5), r, 1.0)
    top = st["scales"].amax(1)
    if n_rot:
        top = torch.maximum(top, st["tail"].abs().amax(1) / 256)
    r = torch.exp2(torch.floor(torch.log2(top.double())))
    return torch.where((top < 2.0 ** -17) | (top > 2.0 ** 5), r, 1.0)


def attention(q, rows, slots_of, positions, window, n_first, scale, sink, tail=0, factors=None):     # tail: how many of a row's last values are rounded to f16
    """q [T, H, D] (any type), rows [slots, D] f64, slots_of[t][j] the slot of row j of token t's sequence (None: hidden),
    positions[t].  Returns out, lse and the bounds of their errors (see the comments), all f64.

    The bounds count the roundings of an implementation that multiplies in f16 and adds in f32: weights to f16 (half a
    step: 2^-11 of each), the f32 tail, or a whole row of codes times a scale that is no power of two, to f16 (2^-11 of each value, in the row as value and, through the score, as
    key: a score off by d moves its weight by e^d - 1 <= 2 d and the normaliser by as much), f32 sums that may
    truncate (n additions are off by at most n 2^-23 of the sum of magnitudes: D for a score, the visible rows for an
    output; exp2 and the exponent's own rounding are below 2^-19 (|score| < 64)), and the output to bf16 (2^-8 of the value).
    f16's steps do not shrink below 2^-24, so a weight is also off by up to 2^-25 where the largest is 1: with weights held
    as w_j r_j relative to their largest W and rows as k_j / r_j (r_j = `factors`), that is 2^-25 W sum_j |k_j| / r_j
    of an output.  Values of a row with a tail are off by up to 2^-25 r_j in the same way."""
    T, H, D = q.shape
    out = torch.zeros((T, H, D), dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)
    for t in range(T):
        js = [j for j in visible(positions[t], window, n_first) if slots_of[t][j] is not None]
        extra = None if sink is None else sink.double()[:, None]
        if not js:
            if sink is not None:
                lse[t] = sink.double()
                lse_bound[t] = sink.double().abs() * 2.0 ** -20
            continue
        mine = torch.tensor([slots_of[t][j] for j in js], device=q.device)
        k = rows[mine]
        r = torch.ones_like(k[:, 0]) if factors is None else factors[mine]
        qd = q[t].double()
        s = qd @ k.t() * scale
        mag = qd.abs() @ k.abs().t() * abs(scale)
        d = mag * D * 2.0 ** -23 + 2.0 ** -19
        if tail:
            d = d + qd.abs().sum(1, keepdim=True) * r[None, :] * abs(scale) * 2.0 ** -25
            d = d + qd[:, D - tail:].abs() @ k[:, D - tail:].abs().t() * abs(scale) * 2.0 ** -11
        d = d.amax(1, keepdim=True)
        z = s if extra is None else torch.cat([s, extra], 1)
        lse[t] = torch.logsumexp(z, 1)
        w = torch.exp(s - lse[t][:, None])
        out[t] = w @ k
        spread = w @ k.abs()
        small = 2.0 ** -25 * (w * r).amax(1, keepdim=True) * (k.abs() / r[:, None]).sum(0)
        if tail:
            small = small + 2.0 ** -25 * (w @ r)[:, None]
        out_bound[t] = small + out[t].abs() * 2.0 ** -8 + spread * (2.0 ** -11 + (2.0 ** -11 if tail else 0.0) + 4 * d + len(js) * 2.0 ** -22) * 1.01 + 1e-30
        lse_bound[t] = 2 * d[:, 0] + len(js) * 2.0 ** -23 + lse[t].abs() * 2.0 ** -20
    return out, lse, out_bound, lse_bound


class Pages:
    """The page operators on Python lists, one step after the other."""

    def __init__(self, refs, table, lens, page_rows):
        self.refs, self.table, self.lens = [list(map(int, x)) if not isinstance(x[0], (list, np.ndarray)) else [list(map(int, r)) for r in x]
                                            for x in (refs, table, lens)]
        self.page_rows, self.moves, self.status = page_rows, [], 0

    def pages_of(self, rows):
        return -(-rows // self.page_rows)

    def _free(self):
        return [i for i, r in enumerate(self.refs) if r <= 0]

    def _held(self, s):
        return self.table[s][:self.pages_of(self.lens[s])]

    def _valid(self, s):
        return 0 <= self.lens[s] <= len(self.table[s]) * self.page_rows and all(0 <= p < len(self.refs) for p in self._held(s))

    def fork(self, pairs):
        n = len(self.table)
        targets = [b for _, b in pairs]
        ok = all(0 <= a < n and 0 <= b < n for a, b in pairs) and len(set(targets)) == len(targets)
        ok = ok and not any(a in targets for a, _ in pairs) and all(self._valid(a) for a, _ in pairs)
        if not ok:
            self.status = -1
            return
        free, need = self._free(), sum(self.lens[a] % self.page_rows != 0 for a, _ in pairs)
        if need > len(free):
            self.status = need - len(free)
            return
        for a, b in pairs:
            held, full = self._held(a), self.lens[a] // self.page_rows
            self.table[b] = held[:full] + [-1] * (len(self.table[b]) - full)
            for p in held[:full]:
                self.refs[p] += 1
            if len(held) > full:
                new = free.pop(0)
                self.moves.append((held[full], new))
                self.table[b][full] = new
                self.refs[new] = 1
            self.lens[b] = self.lens[a]

    def reserve(self, new_lens):
        want = [max(a, b) for a, b in zip(self.lens, new_lens)]
        if any(not 0 <= a <= w <= len(r) * self.page_rows for a, w, r in zip(self.lens, want, self.table)):
            self.status = -1
            return
        free = self._free()
        need = sum(self.pages_of(w) - self.pages_of(a) for a, w in zip(self.lens, want))
        if need > len(free):
            self.status = need - len(free)
            return
        for s, w in enumerate(want):
            for c in range(self.pages_of(self.lens[s]), self.pages_of(w)):
                self.table[s][c] = free.pop(0)
                self.refs[self.table[s][c]] = 1
            self.lens[s] = w

    def free(self, seqs):
        if any(not 0 <= s < len(self.table) or not self._valid(s) for s in seqs):
            self.status = -1
            return
        for s in set(seqs):
            for p in self._held(s):
                self.refs[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.lens[s] = 0

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        holes = [i for i in range(n) if self.refs[i] <= 0]
        for old in [i for i in range(n, len(self.refs)) if self.refs[i] > 0]:
            new = holes.pop(0)
            self.moves.append((old, new))
            self.table = [[new if p == old else p for p in r] for r in self.table]
            self.refs[new], self.refs[old] = self.refs[old], 0
        self.refs = [max(r, 0) for r in self.refs]
        return n
