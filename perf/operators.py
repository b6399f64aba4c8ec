"""The operators of the paged key-value cache: what is measured, and what each of them has to give.

Three operators over one cache of pages (row formats: the E4M3 byte cache with a scale per row or a
power-of-two scale per 64 values and an f32 tail, and f32 rows):

* ``decode``: attention of one new token per sequence over its pages, one row serving as key and value;
* ``window``: attention of the tokens of a prompt chunk, each over the last ``window`` rows up to its own
  position and the ``n_first`` first rows of its sequence;
* ``pages``: forking sequences, compacting the pool, and copying pages.

``run`` computes them from elementary torch operations in 32 bits, or with ``own`` through the package's
entry points.  ``exact`` restates the definitions in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

BLOCK64, ROW_AMAX, F32 = "fp8_block64", "fp8_row", "f32"
N_ROT = 64


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one session with the raw 128-row window the reference keeps: the smallest call, latency counts
        dict(name="decode one, 128 rows", op="decode", fmt=F32, heads=64, dim=512, page=64, seqs=1, longest=128,
             even=True, window=0, first=0, sink=True),
        # one session deep into a long document: only a split over the length fills the card
        dict(name="decode one, 131072 rows", op="decode", fmt=BLOCK64, heads=64, dim=512, page=64, seqs=1,
             longest=131072, even=True, window=0, first=0, sink=True),
        # a few sessions of very different age, odd lengths
        dict(name="decode 7, ragged", op="decode", fmt=BLOCK64, heads=64, dim=512, page=64, seqs=7, longest=9001,
             even=False, window=0, first=0, sink=True),
        # a serving batch on the byte cache with one scale per row
        dict(name="decode 64, ragged", op="decode", fmt=ROW_AMAX, heads=64, dim=512, page=64, seqs=64,
             longest=16384, even=False, window=0, first=0, sink=False),
        # a batch whose heads are split over ranks, with a window and first rows, small pages
        dict(name="decode 96, 16 heads, window", op="decode", fmt=F32, heads=16, dim=512, page=16, seqs=96,
             longest=5000, even=False, window=1024, first=4, sink=True),
        # the first chunk of a prompt, on f32 rows
        dict(name="window 512 tokens", op="window", fmt=F32, heads=64, dim=512, page=64, seqs=1, tokens=512, past=0,
             window=128, first=4, sink=True),
        # a chunk of 4096 tokens behind 4096 earlier ones, byte cache
        dict(name="window 4096 tokens", op="window", fmt=BLOCK64, heads=64, dim=512, page=64, seqs=1, tokens=4096,
             past=4096, window=128, first=4, sink=True),
        # chunks of several prompts together, odd lengths, some of one token only
        dict(name="window 9 prompts", op="window", fmt=ROW_AMAX, heads=64, dim=512, page=64, seqs=9, tokens=1531,
             past=777, window=128, first=1, sink=False),
        # heads of the narrow kind (128 wide) with a longer window
        dict(name="window 1000, 128 wide", op="window", fmt=F32, heads=64, dim=128, page=32, seqs=2, tokens=1000,
             past=500, window=512, first=16, sink=True),
        # one session forked into four, the layers of half the model: latency of a small change
        dict(name="fork 1 into 4", op="fork", layers=20, page=64, pool=512, seqs=16, forks=4, longest=1000, live=0.5),
        # a batch of sessions forked at once
        dict(name="fork 60", op="fork", layers=20, page=64, pool=1500, seqs=140, forks=60, longest=1000, live=0.6),
        # a pool with holes in it packed to its lower end
        dict(name="compact 1500 pages", op="compact", layers=20, page=64, pool=1500, seqs=100, forks=0, longest=1000,
             live=0.6),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "window", "window", "fork", "compact"])
    if op in ("fork", "compact"):
        case = dict(op=op, layers=_log_int(rng, 2, 20), page=rng.choice([16, 32, 64]), pool=_log_int(rng, 100, 1500),
                    longest=rng.randint(100, 1000), live=rng.choice([0.3, 0.5, 0.7]))
        sources = max(1, int(case["pool"] * case["live"] / (0.5 * _width(case) + 0.5)))
        case["forks"] = rng.randint(1, max(1, case["pool"] // 25)) if op == "fork" else 0
        case["seqs"] = sources + case["forks"]
        return case
    case = dict(op=op, fmt=rng.choice([BLOCK64, ROW_AMAX, F32]), heads=rng.choice([1, 5, 8, 16, 32, 48, 64, 96, 128]),
                dim=rng.choice([128, 256, 512, 512]), page=rng.choice([16, 32, 64, 128]))
    if op == "decode":
        seqs = _log_int(rng, 1, 64)
        case.update(seqs=seqs, longest=_log_int(rng, 1, min(131072, 400000 // seqs)), even=rng.random() < 0.3,
                    window=rng.choice([0, 0, 128, rng.randint(1, 3000)]), first=0, sink=rng.random() < 0.5)
    else:
        seqs = rng.randint(1, 9)
        case.update(seqs=seqs, tokens=_log_int(rng, seqs, 1500), past=rng.randint(0, 2000),
                    window=rng.choice([128, 128, rng.randint(1, 600)]), first=0, sink=rng.random() < 0.5)
    if case["window"]:
        case["first"] = rng.choice([0, 1, 4, rng.randint(1, 64)])
    return case


# ----------------------------------------------------------------------------------------------- inputs

def _lengths(case):
    """Rows per sequence and, for ``window``, the chunk's tokens per sequence: a part of the case, not of the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]
    if case["op"] == "decode":
        if case["even"]:
            return [case["longest"]] * n, [1] * n
        lens = [_log_int(rng, max(1, case["longest"] // 30), case["longest"]) for _ in range(n)]
        lens[rng.randrange(n)] = case["longest"]
        if n > 2:
            lens[rng.randrange(n)] = 1
        return lens, [1] * n
    cuts = sorted(rng.randint(0, case["tokens"]) for _ in range(n - 1))
    toks = [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    past = [case["past"] if n == 1 else rng.randint(0, case["past"]) for _ in range(n)]
    return [p + t for p, t in zip(past, toks)], toks


def _width(case):
    return (case["longest"] + case["page"] - 1) // case["page"]


def _held(case):
    """Rows of the sequences that hold pages before the call: together at most ``live`` of the pool."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    left, lens = int(case["pool"] * case["live"]), []
    for _ in range(case["seqs"] - case["forks"]):
        n = rng.randint(1, case["longest"])
        k = (n + case["page"] - 1) // case["page"]
        lens.append(n if k <= left else 0)
        left -= k if k <= left else 0
    return lens


def _sources(case):
    """The sequence each fork is taken from: one after the other, or one sequence for all of a few."""
    n = case["seqs"] - case["forks"]
    return [i % n if case["forks"] > 4 else 0 for i in range(case["forks"])]


def _cache_rows(fmt, x):
    """f32 rows [n, dim] in the cache's row format, by the store operators' rules."""
    n, dim = x.shape
    if fmt == F32:
        return dict(raw=x.half().float())
    if fmt == ROW_AMAX:
        scale = x.abs().amax(1, keepdim=True).clamp_min(1e-4) / 448.0
        return dict(codes=(x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scales=scale)
    nope = dim - N_ROT
    blocks = x[:, :nope].reshape(n, nope // 64, 64)
    scale = torch.exp2(torch.ceil(torch.log2(blocks.abs().amax(2).clamp_min(1e-4) / 448.0)))
    codes = torch.zeros((n, dim), dtype=torch.uint8, device=x.device)
    codes[:, :nope] = (blocks / scale[:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, nope)
    return dict(codes=codes, scales=scale, tail=x[:, nope:].contiguous())


def _prepare_attention(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    lens, toks = _lengths(case)
    page, dim, heads = case["page"], case["dim"], case["heads"]
    need = [(n + page - 1) // page for n in lens]
    spare = 3
    n_pages = sum(need) + spare
    x = torch.randn((n_pages * page, dim), generator=g, device=dev)
    # pages lie anywhere in the pool; entries behind a sequence's last page name no page
    order = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    st = dict(case=case, table=table, n_pages=n_pages, lens=lens, toks=toks,
              kv_len=torch.tensor(lens, dtype=torch.int32, device=dev), **_cache_rows(case["fmt"], x))
    del x
    n_q = sum(toks)
    st["q"] = torch.randn((n_q, heads, dim), generator=g, device=dev).bfloat16()
    st["sink"] = torch.randn((heads,), generator=g, device=dev) if case["sink"] else None
    start = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
    st["q_start"] = torch.from_numpy(start).to(dev)
    if own:
        from ds4cuda_b200 import ops
        kinds = {BLOCK64: ops.KV_FP8_BLOCK64, ROW_AMAX: ops.KV_FP8_ROW, F32: ops.KV_F32}
        st["cache"] = ops.PagedKv(kinds[case["fmt"]], page, N_ROT, codes=st.get("codes"), scales=st.get("scales"),
                                  tail=st.get("tail"), raw=st.get("raw"))
        st["workspace"] = ops.attn_workspace(heads, dim, dev)
    return st


def _prepare_pages(case, seed):
    """A pool in use: sequences of whole pages and a part of one, taken at random places."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    page, pool, layers = case["page"], case["pool"], case["layers"]
    width, seqs, forks = _width(case), case["seqs"], case["forks"]
    sources, held = seqs - forks, _held(case)
    lens = held + [0] * forks
    # per layer the codes, the scales and the tail of the byte cache, as 32-bit words
    arrays = []
    for _ in range(layers):
        for words in (page * 512 // 4, page * 7, page * N_ROT):
            arrays.append(torch.randint(-2 ** 31, 2 ** 31 - 1, (pool, words), generator=g, device=dev, dtype=torch.int32))
    free = list(range(pool))
    rng.shuffle(free)
    table = np.full((seqs, width), -1, dtype=np.int32)
    refs = np.zeros((pool,), dtype=np.int32)
    for b, n in enumerate(held):
        r = [free.pop() for _ in range((n + page - 1) // page)]
        table[b, :len(r)] = r
        refs[r] += 1
    pairs = list(zip(_sources(case), range(sources, seqs)))
    st = dict(case=case, arrays=arrays, table=torch.from_numpy(table).to(dev), refs=torch.from_numpy(refs).to(dev),
              lens=torch.tensor(lens, dtype=torch.int32, device=dev),
              pairs=torch.tensor(pairs, dtype=torch.int32, device=dev).reshape(-1, 2),
              host=dict(table=table, refs=refs, lens=lens, pairs=pairs))
    if own:
        from ds4cuda_b200 import ops
        st["pool"] = ops.PagePool(arrays, page, seqs, width)
        st["out"] = dict(refs_out=torch.empty_like(st["refs"]), table_out=torch.empty_like(st["table"]))
        if case["op"] == "fork":
            st["out"]["lens_out"] = torch.empty_like(st["lens"])
    return st


def prepare(case, seed):
    if case["op"] in ("decode", "window"):
        return _prepare_attention(case, seed)
    return _prepare_pages(case, seed)


# ------------------------------------------------------------------------------------------- plain forms

def _dequant(st, slots):
    """Rows at ``slots`` in f32."""
    fmt, dim = st["case"]["fmt"], st["case"]["dim"]
    if fmt == F32:
        return st["raw"][slots]
    x = st["codes"][slots].view(torch.float8_e4m3fn).float()
    if fmt == ROW_AMAX:
        return x * st["scales"][slots]
    nope = dim - N_ROT
    x[:, :nope] *= st["scales"][slots].repeat_interleave(64, 1)
    x[:, nope:] = st["tail"][slots]
    return x


def _slots(st, b, first, last):
    """Pool rows of rows ``first`` .. ``last`` - 1 of sequence ``b``."""
    page = st["case"]["page"]
    j = torch.arange(first, last, device=st["table"].device)
    return st["table"][b].long()[j // page] * page + j % page


def _softmax_rows(s, sink, rows):
    """Softmax weights over the last axis (``sink``: one more logit per head that has no row), times ``rows``."""
    m = s.amax(-1, keepdim=True)
    if sink is not None:
        m = torch.maximum(m, sink)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    if sink is not None:
        z = z + torch.exp(sink - m)
    return (p @ rows) / z


def _attend(st, b, q, p0):
    """q [n, heads, dim] at positions p0 .. p0 + n - 1 of sequence b."""
    case = st["case"]
    n, heads, dim = q.shape
    window = case["window"] or p0 + n
    lo = max(0, p0 - window + 1)
    first = min(case["first"], lo)
    slots = _slots(st, b, lo, p0 + n)
    if first:
        slots = torch.cat([_slots(st, b, 0, first), slots])
    rows = _dequant(st, slots)
    s = (q.reshape(n * heads, dim) @ rows.t()).reshape(n, heads, -1) / math.sqrt(dim)
    at = torch.arange(p0, p0 + n, device=q.device)[:, None]
    j = torch.cat([torch.arange(0, first, device=q.device), torch.arange(lo, p0 + n, device=q.device)])[None, :]
    seen = (j <= at) & ((j > at - window) | (j < case["first"]))
    s = s.masked_fill(~seen[:, None, :], float("-inf"))
    sink = None if st["sink"] is None else st["sink"][None, :, None]
    return _softmax_rows(s, sink, rows)


def _run_attention(st):
    outs, at = [], 0
    for b, (n, t) in enumerate(zip(st["lens"], st["toks"])):
        for c in range(0, t, 128):
            m = min(128, t - c)
            outs.append(_attend(st, b, st["q"][at + c:at + c + m].float(), n - t + c))
        at += t
    return torch.cat(outs).bfloat16()


def _run_fork(st):
    page, refs, table, lens = st["case"]["page"], st["refs"].clone(), st["table"].clone(), st["lens"].clone()
    src, dst = st["pairs"][:, 0].long(), st["pairs"][:, 1].long()
    full = st["lens"][src].long() // page
    part = (st["lens"][src] % page != 0)
    free = torch.nonzero(st["refs"] == 0)[:, 0]
    rank = torch.cumsum(part.int(), 0) - 1
    new = free[rank.clamp_min(0).long()]
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    shared = col < full[:, None]
    rows = torch.where(shared, table[src], -1)
    refs.index_add_(0, rows[shared].long(), torch.ones_like(rows[shared]))
    rows = torch.where(part[:, None] & (col == full[:, None]), new[:, None].int(), rows)
    refs[new[part]] = 1
    table[dst] = rows
    lens[dst] = lens[src]
    old = st["table"][src].long().gather(1, full.clamp_max(table.shape[1] - 1)[:, None])[:, 0]
    for a in st["arrays"]:
        a[new[part]] = a[old[part]]
    return refs, table, lens, st["arrays"]


def _run_compact(st):
    live = st["refs"] > 0
    n = live.sum()
    i = torch.arange(live.numel(), device=live.device)
    src = torch.nonzero(live & (i >= n))[:, 0]
    dst = torch.nonzero(~live & (i < n))[:, 0]
    to = i.clone()
    to[src] = dst
    table = torch.where(st["table"] >= 0, to[st["table"].clamp_min(0).long()].int(), st["table"])
    refs = st["refs"].clone()
    refs[dst] = st["refs"][src]
    refs[src] = 0
    for a in st["arrays"]:
        a[dst] = a[src]
    return refs, table, st["arrays"]


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from ds4cuda_b200 import ops
        if op == "decode":
            return ops.attn_decode_paged(st["q"], st["cache"], st["table"], st["kv_len"], window=case["window"],
                                         n_first=case["first"], sink=st["sink"], workspace=st["workspace"])
        if op == "window":
            return ops.attn_window_paged(st["q"], st["cache"], st["table"], st["kv_len"], st["q_start"],
                                         window=case["window"], n_first=case["first"], sink=st["sink"],
                                         workspace=st["workspace"])
        if op == "fork":
            refs, table, lens, _ = ops.pages_fork(st["pool"], st["refs"], st["table"], st["lens"], st["pairs"], **st["out"])
            return refs, table, lens, st["arrays"]
        refs, table, _ = ops.pages_compact(st["pool"], st["refs"], st["table"], **st["out"])
        return refs, table, st["arrays"]
    if op in ("decode", "window"):
        return _run_attention(st)
    return _run_fork(st) if op == "fork" else _run_compact(st)


# ------------------------------------------------------------------------------------------------- work

def _visible(case, n, t):
    """(rows a chunk of t tokens ending at row n - 1 touches, sum over its tokens of the rows each sees)."""
    window = case["window"] or n
    lo = max(0, n - t - window + 1)
    touched = (n - lo) + min(case["first"], lo) if t else 0
    seen = 0
    for p in range(n - t, n):
        a = max(0, p - window + 1)
        seen += p + 1 - a + min(case["first"], a)
    return touched, seen


def work(case):
    if case["op"] in ("decode", "window"):
        lens, toks = _lengths(case)
        dim, heads = case["dim"], case["heads"]
        row = {F32: 4 * dim, ROW_AMAX: dim + 4, BLOCK64: (dim - N_ROT) + (dim - N_ROT) // 64 * 4 + N_ROT * 4}[case["fmt"]]
        both = [_visible(case, n, t) for n, t in zip(lens, toks)]
        rows, seen = sum(r for r, _ in both), sum(s for _, s in both)
        return {"bytes": rows * row + 2 * sum(toks) * heads * dim * 2 + sum((r + case["page"] - 1) // case["page"] for r, _ in both) * 4,
                "flops": 4 * seen * heads * dim}
    page, pool, held = case["page"], case["pool"], _held(case)
    page_bytes = case["layers"] * (page * 512 + page * 28 + page * N_ROT * 4)
    if case["op"] == "fork":
        moved = sum(held[b] % page != 0 for b in _sources(case))
    else:
        used = sum((n + page - 1) // page for n in held)
        moved = used * (1 - used / pool)                     # live pages above the new end, on average
    return {"bytes": int(2 * moved * page_bytes) + 2 * 4 * (pool + case["seqs"] * _width(case)), "flops": 0}


# ------------------------------------------------------------------------------------------------ exact

def _e4m3_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        mag = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = float("nan") if (c & 127) == 127 else (-mag if c & 128 else mag)
    return v


def exact(case, seed):
    st = prepare(case, seed)
    dev = st["table"].device
    if case["op"] in ("decode", "window"):
        lens, toks = st["lens"], st["toks"]
        heads, dim, page = case["heads"], case["dim"], case["page"]
        values = torch.from_numpy(_e4m3_values()).to(dev)
        out = torch.zeros((sum(toks), heads, dim), dtype=torch.float64, device=dev)
        at = 0
        for b in range(len(lens)):
            n, t = lens[b], toks[b]
            if t == 0:
                continue
            window = case["window"] or n
            begin = max(0, n - t - window + 1)
            keep = list(range(min(case["first"], begin))) + list(range(begin, n))
            j = torch.tensor(keep, device=dev)
            slot = st["table"][b].long().index_select(0, torch.div(j, page, rounding_mode="floor")) * page + j.remainder(page)
            if case["fmt"] == F32:
                kv = st["raw"].index_select(0, slot).double()
            else:
                kv = values[st["codes"].index_select(0, slot).long()]
                sc = st["scales"].index_select(0, slot).double()
                if case["fmt"] == ROW_AMAX:
                    kv = kv * sc
                else:
                    for k in range((dim - N_ROT) // 64):
                        kv[:, 64 * k:64 * k + 64] *= sc[:, k:k + 1]
                    kv[:, dim - N_ROT:] = st["tail"].index_select(0, slot).double()
            # one token at a time over only the rows it sees
            for c in range(t):
                p = n - t + c
                a = max(0, p - window + 1)
                if a <= begin:
                    mine = kv[:len(keep) - (n - 1 - p)]
                else:
                    f = min(case["first"], a)               # first rows may lie before or inside the kept range
                    head = torch.nonzero(j < f)[:, 0]
                    lo = len(keep) - (n - a)
                    mine = torch.cat([kv[head], kv[lo:len(keep) - (n - 1 - p)]]) if f else kv[lo:len(keep) - (n - 1 - p)]
                logit = torch.einsum("hd,nd->hn", st["q"][at + c].double(), mine) / dim ** 0.5
                if st["sink"] is None:
                    lse = torch.logsumexp(logit, 1)
                else:
                    lse = torch.logsumexp(torch.cat([logit, st["sink"].double()[:, None]], 1), 1)
                out[at + c] = torch.einsum("hn,nd->hd", torch.exp(logit - lse[:, None]), mine)
            at += t
        return out
    # whole numbers: the tables from the definition, page by page; the pool's contents have no computed values
    h, page, pool = st["host"], case["page"], case["pool"]
    refs, table, lens = h["refs"].copy(), h["table"].copy(), list(h["lens"])
    if case["op"] == "fork":
        for src, dst in h["pairs"]:
            n = h["lens"][src]
            table[dst] = -1
            for c in range(n // page):
                table[dst, c] = h["table"][src, c]
                refs[table[dst, c]] += 1
            if n % page:
                new = next(i for i in range(pool) if refs[i] == 0)
                table[dst, n // page] = new
                refs[new] = 1
            lens[dst] = n
        return refs, table, np.asarray(lens, dtype=np.int32), [None] * len(st["arrays"])
    n = int((refs > 0).sum())
    holes = [i for i in range(n) if refs[i] == 0]
    for old in [i for i in range(n, pool) if refs[i] > 0]:
        new = holes.pop(0)
        table[h["table"] == old] = new
        refs[new], refs[old] = refs[old], 0
    return refs, table, [None] * len(st["arrays"])
