"""GPU tests of the paged cache: decode and chunk attention against the 64-bit model, page operators against the list
model, and the chain store -> attention -> fork -> free -> compact."""
import random

import pytest
import torch

import paged_model as model

pytestmark = pytest.mark.gpu

FMTS = ["f32", "row", "block"]


def kind(ops, fmt):
    return {"f32": ops.KV_F32, "row": ops.KV_FP8_ROW, "block": ops.KV_FP8_BLOCK64}[fmt]


class Case:
    """A cache with sequences of the given lengths in random pages; rows that belong to nobody hold NaN."""

    def __init__(self, ops, fmt, heads, dim, page, lens, toks=None, n_rot=64, seed=0, row_scale=None, q_scale=1.0, width=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.fmt, self.tail = fmt, {"f32": 0, "row": dim, "block": n_rot}[fmt]
        need = [-(-n // page) for n in lens]
        n_pages = sum(need) + 2
        x = torch.randn((n_pages * page, dim), generator=g, device="cuda")
        width = width or max(need + [1])
        order = torch.randperm(n_pages, generator=g, device="cuda").int().cpu().tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        owned = torch.zeros(n_pages * page, dtype=torch.bool)
        self.slots, at = [], 0
        for b, (n, k) in enumerate(zip(lens, need)):
            pages = order[at:at + k]
            at += k
            table[b, :k] = torch.tensor(pages, dtype=torch.int32)
            s = [pages[j // page] * page + j % page for j in range(n)]
            self.slots.append(s)
            owned[s] = True
            if row_scale is not None:
                for j, slot in enumerate(s):
                    x[slot] *= row_scale(j)
        self.st = model.make_rows(fmt, x, n_rot)
        self.rows = model.row_values(fmt, self.st, n_rot)
        self.factors = model.row_factors(fmt, self.st, n_rot)
        lost = ~owned.cuda()
        if fmt == "f32":
            self.st["raw"][lost] = float("nan")
        else:
            self.st["codes"][lost] = 0x7f
            self.st["scales"][lost] = float("nan")
            if fmt == "block" and n_rot:
                self.st["tail"][lost] = float("inf")
        self.kv = ops.PagedKv(kind(ops, fmt), page, n_rot, **self.st)
        self.table, self.kv_len = table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
        toks = [1] * len(lens) if toks is None else toks
        self.q = (torch.randn((sum(toks), heads, dim), generator=g, device="cuda") * q_scale).bfloat16()
        self.sink = torch.randn((heads,), generator=g, device="cuda")
        start = [0]
        for t in toks:
            start.append(start[-1] + t)
        self.q_start = torch.tensor(start, dtype=torch.int32, device="cuda")
        self.slots_of = [self.slots[b] for b, t in enumerate(toks) for _ in range(t)]
        self.positions = [lens[b] - t + i for b, t in enumerate(toks) for i in range(t)]

    def check(self, out, lse, window, n_first, sink, scale=None):
        want, want_lse, ob, lb = model.attention(self.q, self.rows, self.slots_of, self.positions, window, n_first,
                                                 self.q.shape[2] ** -0.5 if scale is None else scale, sink, self.tail,
                                                 self.factors)
        err = (out.double() - want).abs()
        assert bool((err <= ob).all()), f"out: worst {(err - ob).max().item():.3e} over its bound, nan {int(out.isnan().sum())}"
        if lse is not None:
            hidden = torch.isinf(want_lse)
            assert bool((torch.isinf(lse) == hidden).all())
            e = (lse.double() - want_lse).abs()[~hidden]
            assert bool((e <= lb[~hidden]).all()), f"lse: worst {(e - lb[~hidden]).max().item():.3e} over its bound"


DECODE = [  # heads, dim, page, lens, window, first, sink
    (64, 512, 64, [1], 0, 0, True),
    (64, 512, 64, [64, 65, 63, 128, 0, 1], 0, 0, False),
    (64, 512, 16, [1000, 3, 257], 0, 0, True),
    (1, 128, 1, [5, 130], 0, 0, False),
    (5, 256, 7, [100, 341, 2], 50, 3, True),
    (16, 384, 32, [700, 64, 129], 128, 4, True),
    (48, 512, 128, [300, 129], 1, 0, True),
    (96, 512, 64, [200, 1, 77], 0, 0, True),
    (128, 256, 64, [513, 500], 100, 500, False),
    (130, 128, 64, [90], 64, 1, True),
    (64, 512, 64, [9000], 0, 0, True),
    (8, 512, 64, [40] * 200, 0, 0, True),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,dim,page,lens,window,first,sink", DECODE)
def test_decode_against_64_bits(ops, fmt, heads, dim, page, lens, window, first, sink):
    c = Case(ops, fmt, heads, dim, page, lens, seed=heads + dim)
    s = c.sink if sink else None
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, window=window, n_first=first, sink=s, want_lse=True)
    c.check(out, lse, window, first, s)
    assert ops.device_status() == 0


WINDOW = [  # heads, dim, page, lens, toks, window, first, sink
    (64, 512, 64, [1], [1], 128, 4, True),
    (64, 512, 64, [300], [300], 128, 4, True),
    (64, 512, 64, [200, 90, 0, 131], [70, 90, 0, 1], 64, 1, False),
    (64, 512, 16, [150], [40], 0, 0, True),
    (16, 512, 64, [333, 50], [101, 50], 30, 7, True),
    (3, 128, 5, [91, 200, 64], [91, 3, 64], 17, 2, True),
    (1, 256, 64, [500], [200], 64, 0, False),
    (33, 384, 32, [77], [20], 128, 10, True),
    (128, 512, 64, [140, 20], [9, 20], 128, 4, True),
    (64, 128, 64, [260], [130], 100, 300, True),
    (40, 128, 64, [2000], [1900], 40, 3, True),          # more items than the tile list is cut for
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,dim,page,lens,toks,window,first,sink", WINDOW)
def test_window_against_64_bits(ops, fmt, heads, dim, page, lens, toks, window, first, sink):
    c = Case(ops, fmt, heads, dim, page, lens, toks, seed=heads + dim)
    s = c.sink if sink else None
    out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=window, n_first=first, sink=s, want_lse=True)
    c.check(out, lse, window, first, s)
    assert ops.device_status() == 0


def test_decode_block_rows_without_a_tail(ops):
    c = Case(ops, "block", 64, 256, 64, [150, 64], n_rot=0)
    c.tail = 0
    out = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len)
    c.check(out, None, 0, 0, None)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("scale", [lambda j: 1.0 + j / 40.0, lambda j: 30.0 if j == 200 else 0.01, lambda j: 1e-3 if j < 100 else 8.0])
def test_decode_maxima_that_grow_along_the_sequence(ops, fmt, scale):
    """The running maximum rises by more than its rescaling threshold, in early and in late tiles."""
    c = Case(ops, fmt, 64, 512, 64, [400, 333], row_scale=scale, q_scale=2.0)
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    c.check(out, lse, 0, 0, c.sink)


@pytest.mark.parametrize("fmt", FMTS)
def test_decode_query_scale_is_exact(ops, fmt):
    """A power of two moved from the query to the scale changes no bit, far beyond f16's range."""
    c = Case(ops, fmt, 16, 256, 64, [200, 70])
    a = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, scale=2.0 ** -4)
    for e in (-60, -20, 30, 60):
        b = ops.attn_decode_paged((c.q.float() * 2.0 ** e).bfloat16(), c.kv, c.table, c.kv_len, scale=2.0 ** (-4 - e))
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("mag", [1e-6, 1e4])
def test_decode_rows_far_from_one(ops, mag):
    for fmt in ("row", "block"):
        c = Case(ops, fmt, 16, 256, 64, [200, 70], row_scale=lambda j: mag)
        out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, scale=1.0 / mag / 16, want_lse=True)
        c.check(out, lse, 0, 0, None, scale=1.0 / mag / 16)


def test_entries_that_name_no_page_hide_their_rows(ops):
    c = Case(ops, "row", 64, 512, 16, [100, 50])
    c.table[0, 2], c.table[0, 4], c.table[1, 0] = -1, 1 << 30, c.kv.n_pages
    for j in list(range(32, 48)) + list(range(64, 80)):
        c.slots[0][j] = None
    for j in range(16):
        c.slots[1][j] = None
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, want_lse=True)
    c.check(out, lse, 0, 0, None)
    c.table.fill_(-1)
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    assert not out.any() and torch.allclose(lse, c.sink.expand_as(lse), rtol=1e-6, atol=0)
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, want_lse=True)
    assert not out.any() and bool((lse == -float("inf")).all())


def test_lengths_beyond_the_table_are_clamped(ops):
    c = Case(ops, "f32", 8, 128, 16, [64, 64])
    want = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len)
    got = ops.attn_decode_paged(c.q, c.kv, c.table, torch.tensor([1 << 30, 65], dtype=torch.int32, device="cuda"))
    assert torch.equal(want, got)
    got = ops.attn_decode_paged(c.q, c.kv, c.table, torch.tensor([-5, 64], dtype=torch.int32, device="cuda"))
    assert not got[0].any() and torch.equal(got[1], want[1])


def test_window_leaves_other_tokens_alone(ops):
    """A padded batch: tokens ahead of the first sequence and behind the last keep what the buffers held."""
    c = Case(ops, "block", 16, 512, 64, [90, 41], [30, 7])
    q = torch.full((50, 16, 512), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[5:42] = c.q
    out = torch.full_like(q, 7.0)
    ops.attn_window_paged(q, c.kv, c.table, c.kv_len, c.q_start + 5, window=20, n_first=2, out=out)
    c.check(out[5:42], None, 20, 2, None)
    assert bool((out[:5] == 7).all()) and bool((out[42:] == 7).all())


def test_chunk_longer_than_its_sequence(ops):
    """Tokens ahead of row 0 see nothing."""
    c = Case(ops, "f32", 64, 128, 64, [10], [10])
    q = torch.cat([c.q[:4], c.q])
    out, lse = ops.attn_window_paged(q, c.kv, c.table, c.kv_len, torch.tensor([0, 14], dtype=torch.int32, device="cuda"), want_lse=True)
    assert not out[:4].any() and bool((lse[:4] == -float("inf")).all())
    c.check(out[4:], lse[4:], 0, 0, None)


def test_nan_of_a_visible_row_stays_with_its_sequence(ops):
    c = Case(ops, "f32", 64, 512, 64, [70, 70])
    c.st["raw"][c.slots[0][69]] = float("nan")
    out = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len)
    assert bool(out[0].isnan().any(-1).all()) and not out[1].isnan().any()


def test_a_token_does_not_depend_on_its_neighbours_in_a_chunk(ops):
    """A chunk cut in two gives the tokens of the whole one (one token per item at 64 heads: the same bits)."""
    c = Case(ops, "block", 64, 512, 64, [300], [60])
    whole = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=128, n_first=4)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    a = ops.attn_window_paged(c.q[:23].contiguous(), c.kv, c.table, c.kv_len - 37, i32(0, 23), window=128, n_first=4)
    b = ops.attn_window_paged(c.q[23:].contiguous(), c.kv, c.table, c.kv_len, i32(0, 37), window=128, n_first=4)
    d = (torch.cat([a, b]).float() - whole.float()).abs()
    assert bool((d <= 2.0 ** -7 * whole.float().abs() + 2.0 ** -9).all())
    one = ops.attn_decode_paged(c.q[-1:].contiguous(), c.kv, c.table, c.kv_len, window=128, n_first=4)
    assert bool(((one - whole[-1:]).float().abs() <= 2.0 ** -7 * whole[-1:].float().abs() + 2.0 ** -9).all())


def test_captured_decode_follows_lengths_and_repeats_bits(ops):
    c = Case(ops, "block", 64, 512, 64, [500, 900, 64], width=20)
    ws, out = ops.attn_workspace(64, 512), torch.empty_like(c.q)
    ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, workspace=ws, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, workspace=ws, out=out)
    for lens in ([500, 900, 64], [1, 2, 0], [499, 130, 63], [500, 900, 64]):
        c.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        ws.fill_(0xff)
        want = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len)
        out.fill_(3.0)
        g.replay()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))


def test_two_streams_with_a_workspace_each(ops):
    a, b = Case(ops, "row", 64, 512, 64, [3000, 17]), Case(ops, "f32", 64, 512, 64, [2000], seed=5)
    wa, wb = ops.attn_decode_paged(a.q, a.kv, a.table, a.kv_len), ops.attn_decode_paged(b.q, b.kv, b.table, b.kv_len)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    ws = [ops.attn_workspace(64, 512), ops.attn_workspace(64, 512)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(sa):
            oa = ops.attn_decode_paged(a.q, a.kv, a.table, a.kv_len, workspace=ws[0])
        with torch.cuda.stream(sb):
            ob = ops.attn_decode_paged(b.q, b.kv, b.table, b.kv_len, workspace=ws[1])
        outs.append((oa, ob))
    torch.cuda.synchronize()
    for oa, ob in outs:
        assert torch.equal(oa, wa) and torch.equal(ob, wb)


# ---------------------------------------------------------------------------------------------------- pages

def pool_state(ops, rng, n_pages, n_seqs, width, page, layers=2, words=(24, 3), fill=0.6):
    g = torch.Generator(device="cuda").manual_seed(rng.randrange(1 << 30))
    arrays = [torch.randint(-2 ** 31, 2 ** 31 - 1, (n_pages, page * w), generator=g, device="cuda", dtype=torch.int32)
              for _ in range(layers) for w in words]
    free = list(range(n_pages))
    rng.shuffle(free)
    refs, table, lens = [0] * n_pages, [[-1] * width for _ in range(n_seqs)], [0] * n_seqs
    for b in range(n_seqs // 2):
        n = rng.randint(0, width * page)
        k = -(-n // page)
        if len(free) - k < n_pages * (1 - fill):
            continue
        lens[b] = n
        for c in range(k):
            table[b][c] = free.pop()
            refs[table[b][c]] += 1
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return ops.PagePool(arrays, page, n_seqs, width), t(refs), t(table), t(lens), model.Pages(refs, table, lens, page)


def same(m, before, pool, refs, table, lens=None, status=None):
    assert refs.tolist() == m.refs and table.tolist() == m.table
    if lens is not None:
        assert lens.tolist() == m.lens
    if status is not None:
        assert status.item() == m.status
    for a, old in zip(pool.arrays, before):
        want = old.clone()
        for src, dst in m.moves:
            want[dst] = old[src]
        assert torch.equal(a, want)


@pytest.mark.parametrize("seed,n_pages,n_seqs,width,page", [(0, 40, 10, 5, 4), (1, 300, 40, 9, 16), (2, 3000, 64, 40, 3),
                                                            (3, 7, 4, 3, 1), (4, 5000, 2500, 4, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_operators_against_lists(ops, seed, n_pages, n_seqs, width, page, in_place):
    rng = random.Random(seed)
    pool, refs, table, lens, m = pool_state(ops, rng, n_pages, n_seqs, width, page)

    def outs(**kw):
        return {} if in_place else {k: torch.full_like(v, 99) for k, v in kw.items()}

    for step in range(6):
        before = [a.clone() for a in pool.arrays]
        m.moves, m.status = [], 0
        what = ["fork", "free", "reserve", "compact"][rng.randrange(4)] if step else "fork"
        o = outs(refs_out=refs, table_out=table, lens_out=lens)
        if what == "fork":
            empty = [s for s in range(n_seqs) if m.lens[s] == 0]
            held = [s for s in range(n_seqs) if m.lens[s]] or [0]
            targets = [s for s in rng.sample(empty, rng.randint(0, len(empty))) if s not in held]
            pairs = [(rng.choice(held), b) for b in targets]
            m.fork(pairs)
            refs, table, lens, st = ops.pages_fork(pool, refs, table, lens, torch.tensor(pairs, dtype=torch.int32, device="cuda").reshape(-1, 2), **o)
        elif what == "free":
            seqs = [rng.randrange(n_seqs) for _ in range(rng.randint(0, n_seqs // 2))]
            m.free(seqs)
            refs, table, lens, st = ops.pages_free(pool, refs, table, lens, torch.tensor(seqs, dtype=torch.int32, device="cuda"), **o)
        elif what == "reserve":
            new = [rng.randint(0, width * page) if rng.random() < 0.2 else 0 for _ in range(n_seqs)]
            m.reserve(new)
            refs, table, lens, st = ops.pages_reserve(pool, refs, table, lens, torch.tensor(new, dtype=torch.int32, device="cuda"), **o)
        else:
            n = m.compact()
            o.pop("lens_out", None)
            refs, table, live = ops.pages_compact(pool, refs, table, **o)
            assert live.item() == n
            st = None
        same(m, before, pool, refs, table, lens, st)


def test_fork_refuses_bad_lists_and_a_full_pool_and_changes_nothing(ops):
    rng = random.Random(9)
    pool, refs, table, lens, m = pool_state(ops, rng, 30, 8, 6, 4, fill=0.99)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    lens[0], m.lens[0] = 6, 6                               # a part-filled last page, so that a fork needs one
    table[0, :2] = t([3, 5])
    m.table[0][:2] = [3, 5]
    refs[3] = refs[5] = 1
    m.refs[3] = m.refs[5] = 1
    before = [a.clone() for a in pool.arrays]
    bad = [[(0, 8)], [(-1, 7)], [(0, 0)], [(0, 6), (0, 6)], [(0, 6), (6, 7)], [(0, 6), (7, 0)], [(1 << 30, 6)]]
    for pairs in bad:
        m.status = 0
        m.fork(pairs)
        assert m.status == -1
        same(m, before, pool, *ops.pages_fork(pool, refs, table, lens, t(pairs)))
    table[0, 1] = m.table[0][1] = 30                         # an entry that names no page
    m.status = 0
    m.fork([(0, 6)])
    same(m, before, pool, *ops.pages_fork(pool, refs, table, lens, t([(0, 6)])))
    table[0, 1] = m.table[0][1] = 5
    lens[0] = m.lens[0] = 25                                 # more rows than the table has room for
    m.status = 0
    m.fork([(0, 6)])
    same(m, before, pool, *ops.pages_fork(pool, refs, table, lens, t([(0, 6)])))
    lens[0] = m.lens[0] = 6
    refs.fill_(1)
    m.refs = [1] * 30
    m.status = 0
    m.fork([(0, 6), (0, 7)])
    assert m.status == 2
    same(m, before, pool, *ops.pages_fork(pool, refs, table, lens, t([(0, 6), (0, 7)])))


def test_free_and_reserve_refuse_bad_lists(ops):
    rng = random.Random(11)
    pool, refs, table, lens, m = pool_state(ops, rng, 60, 8, 6, 4)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    before = [a.clone() for a in pool.arrays]
    for seqs in ([8], [-1], [0, 99]):
        m.status = 0
        m.free(seqs)
        same(m, before, pool, *ops.pages_free(pool, refs, table, lens, t(seqs)))
    for new in ([25] + [0] * 7, [2 ** 31 - 1] * 8):
        m.status = 0
        m.reserve(new)
        assert m.status == -1
        same(m, before, pool, *ops.pages_reserve(pool, refs, table, lens, t(new)))
    m.status = 0
    refs.fill_(1)
    m.refs = [1] * 60
    m.reserve([24] * 8)
    assert m.status > 0
    same(m, before, pool, *ops.pages_reserve(pool, refs, table, lens, t([24] * 8)))


@pytest.mark.parametrize("words,offset", [(4, 0), (3, 0), (1, 1), (9000, 0), (4097, 1)])
def test_pages_copy(ops, words, offset):
    """Widths that do and do not allow 128-bit access, pages larger than a unit, bases off their 16 bytes."""
    n = 20
    base = [torch.randint(-2 ** 31, 2 ** 31 - 1, (n * words + offset,), device="cuda", dtype=torch.int32) for _ in range(3)]
    arrays = [b[offset:].view(n, words) for b in base]
    pool = ops.PagePool(arrays, 1, 0, 1)
    old = [a.clone() for a in arrays]
    moves = [(0, 5), (0, 6), (19, 1), (7, 18), (2, 3)]
    pool = ops.PagePool(arrays, 1, 0, 1, max_list=len(moves))
    st = ops.pages_copy(pool, torch.tensor(moves, dtype=torch.int32, device="cuda"))
    assert st.item() == 0
    for a, o in zip(arrays, old):
        w = o.clone()
        for s, d in moves:
            w[d] = o[s]
        assert torch.equal(a, w)
    now = [a.clone() for a in arrays]
    for bad in ([(0, 20)], [(-1, 3)], [(0, 5), (1, 5)], [(0, 5), (5, 6)], [(4, 4)]):
        st = ops.pages_copy(pool, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        assert st.item() == -1 and all(torch.equal(a, o) for a, o in zip(arrays, now))
    assert ops.pages_copy(pool, torch.empty((0, 2), dtype=torch.int32, device="cuda")).item() == 0


# ------------------------------------------------------------------------------------------ used together

def test_a_serving_run(ops):
    """Reserve pages, store a prompt's rows through the framework's store op, attend to the chunk, decode, fork, let the fork go its own way, free the
    parent, compact, and go on: outputs equal the 64-bit model over the rows each sequence holds, and moving pages changes no bit."""
    D, H, page, n_pages, width = 512, 64, 16, 64, 12
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(1)
    codes = torch.zeros((n_pages * page, D), dtype=torch.uint8, device=dev)
    scales = torch.zeros((n_pages * page, 7), dtype=torch.float32, device=dev)
    tail = torch.zeros((n_pages * page, 64), dtype=torch.float32, device=dev)
    kv = ops.PagedKv(ops.KV_FP8_BLOCK64, page, 64, codes=codes, scales=scales, tail=tail)
    pool = ops.PagePool([codes, scales, tail], page, 3, width, n_pages=n_pages)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    refs, table, lens = torch.zeros(n_pages, dtype=torch.int32, device=dev), torch.full((3, width), -1, dtype=torch.int32, device=dev), i32(0, 0, 0)
    refs[:3] = 1                                               # somebody else's pages
    params = ops.rope_params_for_layer(2)

    def store(seq, first, n):
        kv_rows = torch.randn((n, D), generator=g, device=dev)
        pos = torch.arange(first, first + n, dtype=torch.int32, device=dev)
        slots = table[seq][(pos // page).long()] * page + pos % page
        ops.rope_fp8_store_rows(kv_rows, pos, params, 64, ops.FP8_BLOCK64_POW2, codes, scales, slots=slots.int().contiguous(), tail_out=tail)

    def query(n):
        q = torch.randn((n, H, D), generator=g, device=dev)
        pos = torch.arange(n, dtype=torch.int32, device=dev)
        return ops.rope_rows(q, pos, params, unit_rms=True).bfloat16()

    def slots_of(seq):
        t = table[seq].tolist()
        return [t[j // page] * page + j % page for j in range(lens[seq].item())]

    def check(q, out, seqs, positions, window, first):
        rows = model.row_values("block", dict(codes=codes, scales=scales, tail=tail))
        want, _, bound, _ = model.attention(q, rows, [slots_of(s) for s in seqs], positions, window, first, D ** -0.5, None, 64,
                                            model.row_factors("block", dict(scales=scales, tail=tail)))
        assert bool(((out.double() - want).abs() <= bound).all())

    refs, table, lens, st = ops.pages_reserve(pool, refs, table, lens, i32(100, 0, 41))
    assert st.item() == 0
    store(0, 0, 100)
    store(2, 0, 41)
    q = query(141)
    out = ops.attn_window_paged(q, kv, table, lens, i32(0, 100, 100, 141), window=32, n_first=4)
    check(q, out, [0] * 100 + [2] * 41, list(range(100)) + list(range(41)), 32, 4)

    refs, table, lens, st = ops.pages_fork(pool, refs, table, lens, i32(0, 1).reshape(1, 2))
    assert st.item() == 0 and lens.tolist() == [100, 100, 41]
    q = query(1).expand(3, H, D).contiguous()
    out = ops.attn_decode_paged(q, kv, table, lens)
    check(q, out, [0, 1, 2], [99, 99, 40], 0, 0)
    assert torch.equal(out[0], out[1])

    refs, table, lens, st = ops.pages_reserve(pool, refs, table, lens, lens + 1)
    for s in range(3):                                         # each its own next row
        store(s, lens[s].item() - 1, 1)
    out = ops.attn_decode_paged(q, kv, table, lens)
    check(q, out, [0, 1, 2], [100, 100, 41], 0, 0)
    assert not torch.equal(out[0], out[1])

    refs, table, lens, st = ops.pages_free(pool, refs, table, lens, i32(0, 0))
    refs[:3] = 0
    # the lengths decide where the tiles are cut, so bits are compared at the same lengths
    out = ops.attn_decode_paged(q, kv, table, lens)
    check(q[1:], out[1:], [1, 2], [100, 41], 0, 0)
    refs, table, n = ops.pages_compact(pool, refs, table)
    assert n.item() == int((refs > 0).sum()) and bool((refs[n.item():] == 0).all())
    again = ops.attn_decode_paged(q, kv, table, lens)
    assert torch.equal(again, out) and not again[0].any()
    assert ops.device_status() == 0


# ------------------------------------------------------------------------------- chunks whose rows are packed first

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,dim,page,lens,toks,window,first", [
    (64, 512, 16, [300, 1, 500, 70], [90, 1, 64, 70], 128, 4), (64, 256, 64, [200], [200], 33, 0), (20, 384, 7, [333, 90], [100, 33], 60, 20),
    (2, 128, 64, [400], [400], 128, 64), (100, 128, 32, [150], [90], 100, 200), (64, 128, 64, [40, 1500], [40, 700], 0, 0)])
def test_packed_chunks_against_64_bits(ops, fmt, heads, dim, page, lens, toks, window, first):
    """Rows of every size: plain ones, ones that need a factor, holes, and ends of runs inside a group of 16 rows."""
    c = Case(ops, fmt, heads, dim, page, lens, toks, seed=dim, row_scale=lambda j: (1.0, 1e-4 if fmt != "f32" else 1.0, 3.0)[j % 3])
    holes = [(0, 0)] + ([(0, 3)] if lens[0] > 5 * page else [])
    for b, k in holes:
        c.table[b, k] = -1
        for j in range(k * page, min((k + 1) * page, lens[b])):
            c.slots[b][j] = None
    ws = ops.attn_workspace(heads, dim)
    ws.fill_(0xff)                                       # NaN wherever something reads what nobody wrote
    out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=window, n_first=first, sink=c.sink, want_lse=True, workspace=ws)
    c.factors = pack_factors(c)
    c.tail = 0 if fmt == "f32" else c.tail
    c.check(out, lse, window, first, c.sink)
    assert ops.device_status() == 0


def pack_factors(c):
    """Of packed rows: 1, or the power of two at or below a row's largest value where that is outside [2^-9, 2^15]."""
    top = c.rows.nan_to_num(0.0).abs().amax(1)
    r = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300))))
    return torch.where((top > 0) & ((top < 2.0 ** -9) | (top > 2.0 ** 15)), r, torch.ones_like(r))


def test_nan_in_packed_rows_reaches_only_the_tokens_that_see_it(ops):
    c = Case(ops, "f32", 64, 128, 64, [200, 150], [200, 100])
    clean = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=32, n_first=2)
    for slot, value in ((c.slots[0][77], float("nan")), (c.slots[1][60], float("inf"))):
        c.st["raw"][slot, 5] = value
    out = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=32, n_first=2)
    sees = torch.zeros(300, dtype=torch.bool)
    sees[77:77 + 32] = True
    sees[200 + 10:200 + 10 + 32] = True
    bad = out.isnan().flatten(1).any(1).cpu()
    assert torch.equal(bad, sees)
    assert torch.equal(out[~sees.cuda()], clean[~sees.cuda()])


def test_packed_and_direct_chunks_agree(ops):
    """The same tokens in a call long enough to pack its rows and in calls that are not."""
    c = Case(ops, "block", 64, 512, 64, [400], [256])
    whole = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=128, n_first=4)
    for first in range(0, 256, 32):
        part = ops.attn_window_paged(c.q[first:first + 32].contiguous(), c.kv, c.table, c.kv_len - (224 - first),
                                     torch.tensor([0, 32], dtype=torch.int32, device="cuda"), window=128, n_first=4)
        d = (part.float() - whole[first:first + 32].float()).abs()
        assert bool((d <= 2.0 ** -7 * whole[first:first + 32].float().abs() + 2.0 ** -9).all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("spoil", ["first", "tail", "scale"])
@pytest.mark.parametrize("window", [20, 0])              # packed rows, and tiles straight from the cache
def test_rows_that_are_not_finite_reach_only_the_tokens_that_see_them(ops, fmt, spoil, window):
    """Four tokens of 16 heads share their tiles."""
    c = Case(ops, fmt, 16, 512, 64, [200, 90], [30, 11])
    call = lambda: ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=window, n_first=2)
    clean = call()
    old = None if fmt == "f32" else c.st["scales"].view(c.st["scales"].shape[0], -1).clone()
    slots = c.slots[0][181], c.slots[1][70]                                 # tokens 11 .. 30 see the first; 30 .. 40 (rows 79 .. 89) the second
    for slot, value in zip(slots, (float("nan"), float("inf"))):
        if fmt == "f32":
            c.st["raw"][slot, {"first": 0, "tail": 511, "scale": 200}[spoil]] = value
        elif spoil == "scale":
            c.st["scales"].view(c.st["scales"].shape[0], -1)[slot, 0] = value
        elif spoil == "tail" and fmt == "block":
            c.st["tail"][slot, 63] = value
        else:
            c.st["codes"][slot, 447 if spoil == "tail" else 0] = 0x7f
    out = call()
    sees = torch.zeros(41, dtype=torch.bool)
    sees[11:30] = True                                                      # (rows 181 .. 199, within 20 of the first)
    sees[30:41] = True
    assert torch.equal(out.isnan().flatten(1).any(1).cpu(), sees)
    # The others: to the bits where rows keep no factor.  The eight rows that are loaded with one whose scale is not finite keep theirs, and
    # weights times factors round elsewhere: within the bound of an output for either set of factors.
    if spoil == "scale" and fmt != "f32":
        keep = c.factors.clone()
        for b, j in ((0, 181), (1, 70)):
            for i in c.slots[b][j // 8 * 8:j // 8 * 8 + 8]:
                top = torch.cat([old[i], c.st["tail"][i].abs() / 256 if fmt == "block" else old[i]]).max().double()
                keep[i] = top if fmt == "row" else torch.exp2(torch.floor(torch.log2(top)))
        bound = 0
        for factors in (c.factors, keep):
            want, _, ob, _ = model.attention(c.q, c.rows, c.slots_of, c.positions, window, 2, 512 ** -0.5, None, c.tail, factors)
            bound = torch.maximum(ob, torch.as_tensor(bound, dtype=ob.dtype, device=ob.device))
        assert bool(((out.double() - want).abs() <= bound)[~sees.cuda()].all())
    else:
        assert torch.equal(out[~sees.cuda()], clean[~sees.cuda()])
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", ["row", "block"])
def test_every_tile_has_factors_of_its_own(ops, fmt):
    """Rows that need a factor in every tile, other ones in the next tile of the same buffer."""
    mags = (1e-6, 3e-6, 3e-5, 1e-5)
    c = Case(ops, fmt, 64, 512, 64, [6000, 4000, 900], row_scale=lambda j: mags[j // 64 % 4])
    scale = 1.0 / 3e-5 / 16
    for n_seqs in (1, 3):
        out, lse = ops.attn_decode_paged(c.q[:n_seqs], c.kv, c.table[:n_seqs], c.kv_len[:n_seqs], scale=scale, want_lse=True)
        for _ in range(3):
            again = ops.attn_decode_paged(c.q[:n_seqs], c.kv, c.table[:n_seqs], c.kv_len[:n_seqs], scale=scale)
            assert torch.equal(again, out)
    c.check(out, lse, 0, 0, None, scale=scale)


def test_bounds_of_sequences_that_are_not_ascending_stay_in_bounds(ops):
    """Device data that no host check sees: the call ends, and one whose last bound alone is too large counts as clamped."""
    c = Case(ops, "f32", 16, 128, 64, [90, 80, 100], [20, 30, 50])
    for bounds in ([0, 1 << 30, 50, 100], [-7, 90, 50, 100], [0, 20, 50, 1 << 30], [1 << 30, -5, 1 << 30, -5]):
        q_start = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        for window in (0, 24):
            out = torch.zeros_like(c.q)
            ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, q_start, window=window, n_first=2, out=out)
            short = torch.zeros_like(c.q[:60])
            ops.attn_window_paged(c.q[:60], c.kv, c.table, c.kv_len, q_start, window=window, n_first=2, out=short)
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    good = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, torch.tensor([0, 20, 50, 1 << 30], dtype=torch.int32, device="cuda"), window=24)
    c.check(good, None, 24, 0, None)


@pytest.mark.parametrize("fmt", ["row", "block"])
@pytest.mark.parametrize("toks", [0, 3, 70])
def test_rows_of_zeros_and_tiny_rows_keep_their_weight(ops, fmt, toks):
    """Such rows count in the softmax's sum, however small what they add to the output."""
    lens = [300, 90] if toks else [3000, 90]
    c = Case(ops, fmt, 16, 512, 64, lens, [toks, toks] if toks else None, row_scale=lambda j: (1.0, 0.0, 1e-34, 1e-20)[j % 4])
    scales = c.st["scales"].view(c.st["scales"].shape[0], -1)
    for b in range(2):
        for j, slot in enumerate(c.slots[b]):
            if j % 8 == 1:
                scales[slot] = 0.0                                          # whatever a store leaves for a row of zeros, zero is read as zero
                c.rows[slot] = 0.0
                c.factors[slot] = 1.0
            elif j % 8 == 2 and fmt == "row":
                scales[slot] = 1e-37
                c.rows[slot] = model.row_values(fmt, {k: v[slot:slot + 1] for k, v in c.st.items()}, 64)[0]
                c.factors[slot] = 1e-37
    if toks:
        out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, want_lse=True)
    else:
        out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, want_lse=True)
    if toks == 70:
        c.factors = pack_factors(c)
    c.check(out, lse, 0, 0, None)


@pytest.mark.parametrize("fmt", ["row", "f32"])
def test_rows_behind_four_gigabytes(ops, fmt):
    """Pages at the far end of a pool whose byte offsets need more than 32 bits, beside pages at its front."""
    dim, page = 512, 64
    n = (9 << 20) if fmt == "row" else (9 << 18)                            # 4.8 GB of rows
    order = [n // page - 1, 0, n // page - 2, 1, n // page // 2]
    g = torch.Generator(device="cuda").manual_seed(7)
    some = model.make_rows(fmt, torch.randn((len(order) * page, dim), generator=g, device="cuda"))
    slots = [p * page + r for p in order for r in range(page)]
    big = {k: torch.empty((n, v.shape[1]), dtype=v.dtype, device="cuda") for k, v in some.items()}
    for k, v in some.items():
        big[k][torch.tensor(slots, device="cuda")] = v
    kv = ops.PagedKv(kind(ops, fmt), page, 64, **big)
    table = torch.tensor([order], dtype=torch.int32, device="cuda")
    rows, factors = model.row_values(fmt, some), model.row_factors(fmt, some)
    length = 5 * page - 3
    for toks in (1, 150):
        q = torch.randn((toks, 64, dim), generator=g, device="cuda").bfloat16()
        kv_len = torch.tensor([length], dtype=torch.int32, device="cuda")
        if toks == 1:
            out = ops.attn_decode_paged(q, kv, table, kv_len)
        else:
            out = ops.attn_window_paged(q, kv, table, kv_len, torch.tensor([0, toks], dtype=torch.int32, device="cuda"), window=130, n_first=3)
        want, _, bound, _ = model.attention(q, rows, [list(range(length))] * toks, list(range(length - toks, length)), 0 if toks == 1 else 130,
                                            0 if toks == 1 else 3, dim ** -0.5, None, dim if fmt == "row" else 0, factors)
        assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("heads", [64, 8])
def test_captured_chunk_follows_the_cache_and_the_lengths(ops, heads):
    """A graph of a chunk's call (rows packed in the workspace), replayed after rows, lengths and bounds have changed."""
    c = Case(ops, "block", heads, 512, 64, [300, 200], [100, 80])
    ws, out = ops.attn_workspace(heads, 512), torch.zeros_like(c.q)
    call = lambda: ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=128, n_first=4, workspace=ws, out=out)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for change in (lambda: None, lambda: c.kv_len.sub_(31), lambda: c.st["scales"].mul_(2.0),
                   lambda: c.q_start.copy_(torch.tensor([20, 90, 150], dtype=torch.int32, device="cuda"))):
        change()
        out.fill_(5.0)
        want = call().clone()
        out.fill_(5.0)
        ws.fill_(0xff)
        graph.replay()
        assert torch.equal(out, want)
    assert bool((out[:20] == 5).all()) and bool((out[150:] == 5).all())


@pytest.mark.parametrize("window", [0, 7])
def test_chunk_longer_than_its_sequence_with_tokens_that_share_tiles(ops, window):
    c = Case(ops, "f32", 8, 128, 64, [10, 90], [10, 5])
    q = torch.cat([c.q[:4], c.q])
    out, lse = ops.attn_window_paged(q, c.kv, c.table, c.kv_len, torch.tensor([0, 14, 19], dtype=torch.int32, device="cuda"), window=window, want_lse=True)
    assert not out[:4].any() and bool((lse[:4] == -float("inf")).all())
    c.check(out[4:], lse[4:], window, 0, None)


def test_attention_refuses_what_does_not_fit_its_arguments(ops):
    c = Case(ops, "f32", 8, 128, 64, [10])
    for bad in (dict(window=1 << 32), dict(n_first=1 << 32), dict(window=-1), dict(workspace=torch.empty(1 << 20, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, **bad)
