"""GPU tests of the paged cache at its edges: workspaces in any state, items of many tiles, sizes and values at a rule's border."""
import random

import pytest
import torch

import paged_model as model
from ds4cuda_b200 import _lib
from test_gpu_paged import FMTS, Case, pack_factors, pool_state, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,lens,toks,window,first", [
    (64, [200, 90], [200, 90], 100, 3),                  # last tiles of 36 rows that reach past the rows and the 16 zeros behind them
    (16, [70, 300], [70, 20], 40, 0)])                   # four tokens share a tile's columns
def test_small_integers_left_in_the_workspace_reach_no_result(ops, fmt, heads, lens, toks, window, first):
    """As floats they are subnormal: the reciprocal of one is infinite.  Factors are looked at once one row of a call has a factor or
    no page."""
    c = Case(ops, fmt, heads, 512, 16, lens, toks, row_scale=lambda j: 1e-4 if j % 3 == 1 and fmt != "f32" else 1.0)
    c.table[0, 1] = -1
    for j in range(16, 32):
        c.slots[0][j] = None
    c.factors = pack_factors(c)
    c.tail = 0 if fmt == "f32" else c.tail
    ws = ops.attn_workspace(heads, 512)
    ws.zero_()
    clean = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=window, n_first=first, workspace=ws)
    for word in (1, 256, 1 << 20, 0x7f800000):
        ws.view(torch.int32).fill_(word)
        out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=window, n_first=first, want_lse=True, workspace=ws)
        c.check(out, lse, window, first, None)
        assert torch.equal(out, clean)
    assert ops.device_status() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dim", [128, 256, 384])
def test_packed_items_of_many_and_of_few_tiles_in_turn(ops, fmt, dim):
    """With up to 384 dims nothing but a barrier of its own keeps the drain of an item's accumulators apart from the products of the next
    one: long items ahead of short ones and the other way round, repeated."""
    c = Case(ops, fmt, 64, dim, 64, [900, 40, 700, 30, 1], [120, 40, 60, 30, 1], seed=dim)
    out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=600, n_first=5, sink=c.sink, want_lse=True)
    c.check(out, lse, 600, 5, c.sink)
    for _ in range(20):
        assert torch.equal(ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=600, n_first=5, sink=c.sink), out)
    assert ops.device_status() == 0


@pytest.mark.parametrize("heads", [64, 16])
def test_f32_rows_are_f16_numbers_on_every_path(ops, heads):
    """Values beyond f16's range and below its normal numbers: 65504 and subnormals, whether the call packs its rows first or not."""
    c = Case(ops, "f32", heads, 512, 64, [200, 120], [100, 100], row_scale=lambda j: 1e5 / 3 if j % 3 else 1.0)
    c.st["raw"].nan_to_num_(nan=0.0, posinf=9e4, neginf=-9e4)
    tiny = torch.tensor(c.slots[1], device="cuda")
    c.st["raw"][tiny] = torch.randn((120, 512), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 2e-6
    c.rows = c.st["raw"].clamp(-65504, 65504).half().double()
    assert bool((c.st["raw"].abs() > 65504).any()) and bool((c.rows[tiny] != c.st["raw"][tiny].double()).any())
    scale = 1e-5
    long = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=64, scale=scale)
    c.check(long, None, 64, 0, None, scale=scale)
    # the same tokens as sequences of their own, straight from the cache
    table = c.table.repeat_interleave(100, 0).contiguous()
    lens = torch.tensor([p + 1 for p in c.positions], dtype=torch.int32, device="cuda")
    short = ops.attn_decode_paged(c.q, c.kv, table, lens, window=64, scale=scale)
    c.check(short, None, 64, 0, None, scale=scale)
    assert heads < 64 or torch.equal(short, long)        # at 64 heads the same tiles in the same order


@pytest.mark.parametrize("n_pages,page,width,used,want", [
    (4, 4, 10, 0, [40, 0]),                              # one sequence that asks for more than the pool has
    (4, 4, 10, 3, [9, 40]), (1, 1, 7, 1, [7] * 2500), (50, 2, 40, 20, [80, 80])])
def test_reserve_counts_every_missing_page(ops, n_pages, page, width, used, want):
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    n = len(want)
    m = model.Pages([1] * used + [0] * (n_pages - used), [[-1] * width] * n, [0] * n, page)
    m.reserve(want)
    assert m.status > 0
    pool = ops.PagePool([], page, n, width, n_pages=n_pages)
    refs, table, lens = t(m.refs), t(m.table), t(m.lens)
    out = ops.pages_reserve(pool, refs, table, lens, t(want))
    assert out[3].item() == m.status
    assert out[0].tolist() == m.refs and out[1].tolist() == m.table and out[2].tolist() == m.lens


@pytest.mark.parametrize("toks", [None, [3, 2, 1] * 8])
def test_row_scales_below_f16s_normal_numbers_keep_their_bits(ops, toks):
    """Scales of 2^-17 to 2^-13 (rows of up to 2^-8 to 2^-4) and, beside them in a tile, larger ones; queries along a row, so that a
    scale that is off moves every score the same way."""
    lens = [1, 20, 3] * 8 if toks is None else [9, 20, 70] * 8
    c = Case(ops, "row", 16, 128, 4, lens, toks)
    g = torch.Generator(device="cuda").manual_seed(2)
    for slots in c.slots:
        at = torch.tensor(slots, device="cuda")
        c.st["scales"][at] = torch.exp2(torch.rand((len(slots), 1), generator=g, device="cuda") * 4 - 17)
        c.st["scales"][at[-1]] = 2.0 ** -17 * (1 + 2.0 ** -8)          # half a step off in f16
    c.rows = model.row_values("row", c.st)
    for t, slots in enumerate(c.slots_of):
        c.q[t] = torch.sign(c.rows[slots[-1]])[None].bfloat16()
    scale = 30.0 / max(c.rows[s[-1]].abs().sum().item() for s in c.slots)
    call = ops.attn_decode_paged if toks is None else ops.attn_window_paged
    args = (c.q, c.kv, c.table, c.kv_len) + (() if toks is None else (c.q_start,))
    out, lse = call(*args, scale=scale, want_lse=True)
    c.check(out, lse, 0, 0, None, scale=scale)


@pytest.mark.parametrize("how", ["whole", "cut, few parts", "cut, many parts", "packed", "no rows"])
def test_sinks_of_every_size(ops, how):
    """The largest and lowest f32 values and infinities count as what they are: a sink that outweighs all rows leaves an output of 0 and
    is the log-sum, a lowest one leaves the rows as they are, and without rows the log-sum is the sink to the bit."""
    top, inf = torch.finfo(torch.float32).max, float("inf")
    lens = {"whole": [100, 3], "cut, few parts": [1000] * 50, "cut, many parts": [20000, 5], "packed": [90, 90], "no rows": [0, 0]}[how]
    c = Case(ops, "f32", 16, 128, 64, lens, [80, 80] if how == "packed" else None, width=None if lens[0] else 8)
    sink = torch.tensor([-top, top, inf, -inf, -1e38, 1e38, -1e30, 1e30, 0.0, 3.0, -90.0, 90.0, 1e-45, -0.0, 2.5e38, -2.5e38], device="cuda")
    args = (c.q, c.kv, c.table, c.kv_len)
    call = lambda **kw: ops.attn_window_paged(*args, c.q_start, want_lse=True, **kw) if how == "packed" else ops.attn_decode_paged(*args, want_lse=True, **kw)
    out, lse = call(sink=sink)
    if how == "no rows":
        assert not out.any() and torch.equal(lse, sink.expand_as(lse))
        return
    bare, bare_lse = call()
    heavy, light = [1, 2, 5, 7, 14], [0, 3, 4, 6, 15]
    assert not out[:, heavy].any() and torch.equal(lse[:, heavy], sink[heavy].expand(len(c.q), 5))
    assert torch.equal(out[:, light], bare[:, light])
    assert torch.allclose(lse[:, light], bare_lse[:, light], rtol=0, atol=1e-5)
    rest = [8, 9, 10, 11, 12, 13]
    c.q, small = c.q[:, rest].contiguous(), sink[rest]
    c.check(out[:, rest], lse[:, rest], 0, 0, small)


@pytest.mark.parametrize("lens", [[100, 3], [20000, 5]])
def test_a_sink_that_is_not_a_number_spoils_its_head_only(ops, lens):
    c = Case(ops, "f32", 16, 128, 64, lens)
    c.sink[5] = float("nan")
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    others = [h for h in range(16) if h != 5]
    assert bool(out[:, 5].isnan().all()) and bool(lse[:, 5].isnan().all())
    assert not out[:, others].isnan().any() and not lse[:, others].isnan().any()


@pytest.mark.parametrize("heads,n_seqs", [(1024, 40), (64, 2)])          # whole items (more of them than are cut), and cut ones
def test_many_small_weights_add_up(ops, heads, n_seqs):
    """One row with a weight near 1 and 40000 of 2^-25.5 of it, which together are a thousandth.  A weight is held in f16 as 2^7 times what it
    is relative to its reference, so it is off by at most 2^-32 where it is small; the sum of 40000 by 1e-5."""
    n, dim, page = 40000, 128, 64
    g = torch.zeros((n // page * page, dim), device="cuda")
    g[:, 1] = 1.0
    g[0] = 0.0
    g[0, 0] = 1.0
    kv = ops.PagedKv(ops.KV_F32, page, raw=g)
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(n_seqs, 1)
    q = torch.zeros((n_seqs, heads, dim), device="cuda", dtype=torch.bfloat16)
    q[:, :, 0] = 1.0
    for length in (n, n - 777):
        kv_len = torch.full((n_seqs,), length, dtype=torch.int32, device="cuda")
        out, lse = ops.attn_decode_paged(q, kv, table, kv_len, scale=25.5 * 0.6931471805599453, want_lse=True)
        rest = (length - 1) * 2.0 ** -25.5
        want = rest / (1 + rest)
        # bf16's half step, the weights', and 2^-10 of it for the exponents' f32 roundings (25.5 is held to 2^-20) and the sums
        assert bool(((out[:, :, 1].double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -10) + length * 2.0 ** -32).all())
        assert bool(((out[:, :, 0].double() - 1 / (1 + rest)).abs() <= 2.0 ** -8 + 2.0 ** -10).all())
        assert not out[:, :, 2:].any()
    assert ops.device_status() == 0


# ------------------------------------------------------------------------------------- the caches that the store ops fill

@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("toks", [1, 40])
def test_attention_over_rows_the_store_ops_left(ops, fmt, toks):
    """kv rows -> norm, RoPE and quantiser of the framework -> attention; the rows are what the framework's own load op reads back."""
    D, H, page, n = 512, 16, 16, 90
    g = torch.Generator(device="cuda").manual_seed(5)
    order = torch.randperm(8, generator=g, device="cuda").int()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    slots = (order[(pos // page).long()] * page + pos % page).int()
    params, kv_rows = ops.rope_params_for_layer(3), torch.randn((n, D), generator=g, device="cuda") * 3
    w = 1 + 0.1 * torch.randn((D,), generator=g, device="cuda")
    slots_n, rows = 8 * page, torch.full((8 * page, D), float("nan"), dtype=torch.float64, device="cuda")
    if fmt == "f32":
        st = dict(raw=torch.full((slots_n, D), float("nan"), device="cuda"))
        ops.kv_rows_to_raw(kv_rows, pos, params, st["raw"], slots=slots, norm_w=w)
        rows[slots.long()] = st["raw"][slots.long()].double()
        kv = ops.PagedKv(ops.KV_F32, page, **st)
    else:
        mode = ops.FP8_ROW_AMAX if fmt == "row" else ops.FP8_BLOCK64_POW2
        st = dict(codes=torch.full((slots_n, D), 0x7f, dtype=torch.uint8, device="cuda"),
                  scales=torch.full((slots_n, 1 if fmt == "row" else 7), float("nan"), device="cuda"))
        if fmt == "block":
            st["tail"] = torch.full((slots_n, 64), float("nan"), device="cuda")
        ops.rope_fp8_store_rows(kv_rows, pos, params, 64, mode, st["codes"], st["scales"], slots=slots, norm_w=w, tail_out=st.get("tail"))
        rows[slots.long()] = ops.fp8_cache_load_rows(st["codes"], st["scales"], slots, 64, mode, tail=st.get("tail")).double()
        kv = ops.PagedKv(ops.KV_FP8_ROW if fmt == "row" else ops.KV_FP8_BLOCK64, page, 64, **st)
    assert not rows[slots.long()].isnan().any()
    q = torch.randn((toks, H, D), generator=g, device="cuda").bfloat16()
    table, kv_len = order[None].contiguous(), torch.tensor([n], dtype=torch.int32, device="cuda")
    sink = torch.randn((H,), generator=g, device="cuda")
    if toks == 1:
        out = ops.attn_decode_paged(q, kv, table, kv_len, window=50, n_first=3, sink=sink)
    else:
        out = ops.attn_window_paged(q, kv, table, kv_len, torch.tensor([0, toks], dtype=torch.int32, device="cuda"), window=50, n_first=3, sink=sink)
    want, _, bound, _ = model.attention(q, rows, [slots.tolist()] * toks, list(range(n - toks, n)), 50, 3, D ** -0.5, sink,
                                        {"f32": 0, "row": D, "block": 64}[fmt], model.row_factors(fmt, st))
    assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_single_rows_by_pages_of_one(ops, fmt):
    """A page of one row makes the table a list of rows: any order, the same row twice, rows of other sequences."""
    c = Case(ops, fmt, 64, 512, 1, [150, 70])
    picks = [c.slots[0][::-1] + c.slots[0][:30] + [c.slots[1][5]] * 40, c.slots[1][3:4], c.slots[1] + c.slots[0][10:90:2]]
    table = torch.full((3, max(map(len, picks))), -1, dtype=torch.int32)
    for b, p in enumerate(picks):
        table[b, :len(p)] = torch.tensor(p)
    c.table, c.kv_len = table.cuda(), torch.tensor([len(p) for p in picks], dtype=torch.int32, device="cuda")
    c.q = torch.cat([c.q, c.q[:1]])
    c.slots_of, c.positions = picks, [len(p) - 1 for p in picks]
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    c.check(out, lse, 0, 0, c.sink)


# ------------------------------------------------------------------------------------------------- work and its division

@pytest.mark.parametrize("fmt", FMTS)
def test_short_sequences_under_a_wide_table(ops, fmt):
    """A table as wide as the longest sequence may ever get: tiles are cut into runs by the room, lengths and first rows by what is there."""
    c = Case(ops, fmt, 64, 512, 16, [130, 1, 0, 64, 300, 5], width=1000)
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    c.check(out, lse, 0, 0, c.sink)
    w = Case(ops, fmt, 16, 512, 16, [130, 40, 64], [33, 40, 1], width=1000)
    out, lse = ops.attn_window_paged(w.q, w.kv, w.table, w.kv_len, w.q_start, sink=w.sink, want_lse=True)
    w.check(out, lse, 0, 0, w.sink)


@pytest.mark.parametrize("fmt", FMTS)
def test_more_items_than_are_cut(ops, fmt):
    c = Case(ops, fmt, 128, 128, 64, [1 + (37 * i) % 400 for i in range(300)])
    out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, want_lse=True)
    c.check(out, lse, 0, 0, c.sink)


@pytest.mark.parametrize("fmt", FMTS)
def test_the_most_sequences_a_call_takes(ops, fmt):
    c = Case(ops, fmt, 3, 128, 64, [1 + i % 70 for i in range(64)])
    which = torch.arange(4096) % 64
    table, lens, q = c.table[which].contiguous(), c.kv_len[which].contiguous(), c.q[which].contiguous()
    one = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len)
    c.check(one, None, 0, 0, None)
    out = ops.attn_decode_paged(q, c.kv, table, lens)
    assert torch.equal(out.view(64, 64, 3, 128), one.expand(64, 64, 3, 128))
    start = torch.arange(4097, dtype=torch.int32, device="cuda")
    chunk = ops.attn_window_paged(q, c.kv, table, lens, start)
    assert torch.equal(chunk.view(64, 64, 3, 128), chunk[:64].expand(64, 64, 3, 128))
    c.check(chunk[:64], None, 0, 0, None)
    with pytest.raises(_lib.Ds4Error):
        ops.attn_decode_paged(torch.cat([q, q[:1]]), c.kv, torch.cat([table, table[:1]]), torch.cat([lens, lens[:1]]))


def test_a_token_gives_the_same_bits_in_a_chunk_cut_elsewhere(ops):
    """One token per item, whole items, straight from the cache in each of these calls: the same order of the same sums."""
    c = Case(ops, "block", 64, 512, 64, [300], [60])
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    call = lambda rows, length: ops.attn_window_paged(c.q[rows].contiguous(), c.kv, c.table, i32(length), i32(0, rows.stop - rows.start), window=128, n_first=4)
    whole = call(slice(0, 60), 300)
    for cut in (1, 23, 59):
        assert torch.equal(torch.cat([call(slice(0, cut), 240 + cut), call(slice(cut, 60), 300)]), whole)
    one = ops.attn_decode_paged(c.q[-1:].contiguous(), c.kv, c.table, c.kv_len, window=128, n_first=4)
    assert torch.equal(one, whole[-1:])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,dim", [(64, 512), (64, 128), (8, 256)])
@pytest.mark.parametrize("scale", [lambda j: 1.0 + j / 40.0, lambda j: 30.0 if j % 90 == 80 else 0.01])
def test_packed_maxima_that_grow_along_the_rows(ops, fmt, heads, dim, scale):
    """The accumulators are rescaled between the tiles of packed items, and behind their last one."""
    c = Case(ops, fmt, heads, dim, 64, [400, 333], [180, 20], row_scale=scale, q_scale=2.0)
    out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=300, n_first=2, sink=c.sink, want_lse=True)
    c.factors = pack_factors(c) if fmt != "f32" else c.factors
    c.check(out, lse, 300, 2, c.sink)


@pytest.mark.parametrize("toks,heads,window", [(36000, 128, 1), (70000, 64, 1)])      # packed first, and straight from the cache
def test_queries_and_outputs_behind_four_gigabytes(ops, toks, heads, window):
    """With a window of one row a token's output is its own row, to bf16's bits."""
    g = torch.Generator(device="cuda").manual_seed(1)
    page, dim = 64, 512
    n = -(-toks // page) * page
    raw = torch.randn((n, dim), generator=g, device="cuda").half().float()
    order = torch.randperm(n // page, generator=g, device="cuda").int()
    kv = ops.PagedKv(ops.KV_F32, page, raw=raw)
    q = torch.empty((toks, heads, dim), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert q.numel() * 2 > 1 << 32
    out = ops.attn_window_paged(q, kv, order[None].contiguous(), torch.tensor([toks], dtype=torch.int32, device="cuda"),
                                torch.tensor([0, toks], dtype=torch.int32, device="cuda"), window=window)
    want = raw.view(n // page, page, dim)[order.long()].view(n, dim)[:toks].bfloat16()
    for at in range(0, toks, 5000):
        assert torch.equal(out[at:at + 5000], want[at:at + 5000, None].expand(-1, heads, -1))
    assert ops.device_status() == 0


# ------------------------------------------------------------------------------------------- streams, graphs, workspaces

@pytest.mark.parametrize("fmt", FMTS)
def test_decode_does_not_look_at_what_a_workspace_holds(ops, fmt):
    c = Case(ops, fmt, 64, 512, 64, [3000, 17, 0, 900])
    ws = ops.attn_workspace(64, 512)
    ws.zero_()
    clean, clean_lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, want_lse=True, workspace=ws)
    c.check(clean, clean_lse, 0, 0, None)
    for word in (1, 256, 0x7f800000, -1, 148):
        ws.view(torch.int32).fill_(word)
        out, lse = ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, want_lse=True, workspace=ws)
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


def test_captured_page_operators_follow_their_inputs(ops):
    """fork, reserve, free and compact in one graph, in place, replayed over two states of the pool, and with workspaces in any state."""
    rng = random.Random(4)
    pool, refs, table, lens, _ = pool_state(ops, rng, 32, 8, 6, 4)
    start = [t.clone() for t in (refs, table, lens, *pool.arrays)]
    t = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    pairs, new, gone = t([0, 6], [1, 7]), t(0, 0, 0, 0, 9, 0, 0, 24), t(2, 6)
    status = [t(5) for _ in range(3)]
    live = t(5)

    def chain():
        ops.pages_fork(pool, refs, table, lens, pairs, status=status[0])
        ops.pages_reserve(pool, refs, table, lens, new, status=status[1])
        ops.pages_free(pool, refs, table, lens, gone, status=status[2])
        ops.pages_compact(pool, refs, table, n_live=live)

    def reset():
        for a, b in zip((refs, table, lens, *pool.arrays), start):
            a.copy_(b)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        chain()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    changes = [lambda: None, lambda: new.fill_(24), lambda: pairs.copy_(t([0, 6], [0, 6])), lambda: start[2].clamp_(max=1)]
    seen = set()
    for change in changes:                               # (more pages than there are, a list that is refused, other lengths)
        change()
        results = []
        for run in (chain, graph.replay):
            reset()
            pool.workspace.fill_(0x41)
            run()
            results.append([x.clone() for x in (refs, table, lens, live, *status, *pool.arrays)])
        for a, b in zip(*results):
            assert torch.equal(a, b)
        seen.add(tuple(s.item() for s in status))
    assert len(seen) >= 3


def test_two_pools_on_two_streams(ops):
    t = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    made = []
    for seed in (1, 2):
        pool, refs, table, lens, m = pool_state(ops, random.Random(seed), 400, 40, 9, 16)
        empty = [s for s in range(40) if m.lens[s] == 0]
        held = [s for s in range(40) if m.lens[s]]
        pairs = [(held[i % len(held)], b) for i, b in enumerate(empty[:15])]
        before = [a.clone() for a in pool.arrays]
        m.fork(pairs)
        made.append((pool, refs, table, lens, t(pairs), m, before, torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for pool, refs, table, lens, pairs, m, before, stream in made:
        with torch.cuda.stream(stream):
            got.append(ops.pages_fork(pool, refs, table, lens, pairs))
    torch.cuda.synchronize()
    for (pool, *_, m, before, _), (refs, table, lens, st) in zip(made, got):
        same(m, before, pool, refs, table, lens, st)


# ---------------------------------------------------------------------------------------- arguments the headers allow

@pytest.mark.parametrize("toks", [None, [40, 7], [150, 30]])             # decode; a chunk straight from the cache or packed, by its heads
@pytest.mark.parametrize("heads,dim", [(64, 128), (16, 384), (64, 512)])
def test_queries_of_any_size_and_scales_of_any_sign(ops, toks, heads, dim):
    """A power of two moved from the query to the scale changes no bit; negative and zero scales are scales."""
    c = Case(ops, "block", heads, dim, 64, [200, 70], toks)
    call = ops.attn_decode_paged if toks is None else ops.attn_window_paged
    args = (c.kv, c.table, c.kv_len) + (() if toks is None else (c.q_start,))
    c.q[0, 0] = 0.0
    want, want_lse = call(c.q, *args, scale=-0.04, window=90, sink=c.sink, want_lse=True)
    c.check(want, want_lse, 90, 0, c.sink, scale=-0.04)
    for e in (-40, -9, 9, 40):
        out, lse = call((c.q.float() * 2.0 ** e).bfloat16(), *args, scale=-0.04 * 2.0 ** -e, window=90, sink=c.sink, want_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    out, lse = call(c.q, *args, scale=0.0, window=90, want_lse=True)
    c.check(out, lse, 90, 0, None, scale=0.0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("toks,heads", [(None, 64), ([40, 7], 64), ([150, 30], 64), ([40, 7], 5)])
def test_a_query_that_is_not_finite_spoils_its_head_only(ops, fmt, toks, heads):
    c = Case(ops, fmt, heads, 256, 64, [200, 70], toks)
    call = ops.attn_decode_paged if toks is None else ops.attn_window_paged
    args = (c.kv, c.table, c.kv_len) + (() if toks is None else (c.q_start,))
    clean, clean_lse = call(c.q, *args, window=90, want_lse=True)
    q = c.q.clone()
    q[0, 3, 200], q[-1, 2, 0] = float("nan"), float("inf")
    out, lse = call(q, *args, window=90, want_lse=True)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[-1, 2] = True
    assert bool(out[bad].isnan().any(-1).all())
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])


@pytest.mark.parametrize("mag", [1e-6, 1e-3, 30.0, 1e4])
@pytest.mark.parametrize("fmt", ["row", "block"])
@pytest.mark.parametrize("heads,n_rot", [(64, 64), (8, 0)])
def test_packed_rows_far_from_one(ops, mag, fmt, heads, n_rot):
    c = Case(ops, fmt, heads, 256, 16, [200, 70], [150, 60], n_rot=n_rot, row_scale=lambda j: mag)
    c.factors = pack_factors(c)
    if fmt == "block":
        c.tail = n_rot
    scale = 1.0 / mag / 16
    out, lse = ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=100, n_first=3, scale=scale, want_lse=True)
    c.check(out, lse, 100, 3, None, scale=scale)


def test_one_workspace_for_calls_one_behind_the_other(ops):
    """Cut, whole and packed calls of several shapes on one stream, each right behind the other."""
    cases = [Case(ops, "block", 64, 512, 64, [5000, 40]), Case(ops, "f32", 16, 128, 16, [100, 30], [90, 30]), Case(ops, "row", 64, 512, 64, [300], [200]),
             Case(ops, "f32", 64, 512, 64, [9000])]
    ws = ops.attn_workspace(64, 512)

    def call(c, **kw):
        if len(c.q) == len(c.kv_len):
            return ops.attn_decode_paged(c.q, c.kv, c.table, c.kv_len, sink=c.sink, **kw)
        return ops.attn_window_paged(c.q, c.kv, c.table, c.kv_len, c.q_start, window=70, sink=c.sink, **kw)

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    got = [[call(c, workspace=ws) for c in cases] for _ in range(8)]
    for outs in got:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FMTS)
def test_lengths_of_a_chunk_beyond_its_table_and_below_zero(ops, fmt):
    c = Case(ops, fmt, 16, 128, 16, [64, 48], [9, 5])
    args = (c.q, c.kv, c.table)
    for window in (0, 20):
        want = ops.attn_window_paged(*args, c.kv_len, c.q_start, window=window)
        c.check(want, None, window, 0, None)
        got = ops.attn_window_paged(*args, torch.tensor([2 ** 31 - 1, 48], dtype=torch.int32, device="cuda"), c.q_start, window=window)
        assert torch.equal(got, want)
        got = ops.attn_window_paged(*args, torch.tensor([-2 ** 31, 48], dtype=torch.int32, device="cuda"), c.q_start, window=window)
        assert not got[:9].any() and torch.equal(got[9:], want[9:])
    # the largest window and number of first rows are every row
    # (not to the bits of window=0: the room for packed rows goes by the window)
    c.check(ops.attn_window_paged(*args, c.kv_len, c.q_start, window=2 ** 31 - 1), None, 0, 0, None)
    c.check(ops.attn_window_paged(*args, c.kv_len, c.q_start, window=1, n_first=2 ** 31 - 1), None, 0, 0, None)


@pytest.mark.parametrize("n_pages,n_seqs,width,page", [(1, 2, 1, 1), (9, 5, 3, 2), (70000, 30000, 2, 3), (40, 6, 5, 1000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_page_lists_that_are_empty_and_pools_that_are_full_or_free(ops, n_pages, n_seqs, width, page, in_place):
    t = lambda v, *shape: torch.tensor(v, dtype=torch.int32, device="cuda").view(*(shape or (-1,)))
    words = torch.randint(-2 ** 31, 2 ** 31 - 1, (n_pages, 5), device="cuda", dtype=torch.int32)
    pool = ops.PagePool([words], page, n_seqs, width)
    refs, table, lens = [0] * n_pages, [[-1] * width for _ in range(n_seqs)], [0] * n_seqs
    m = model.Pages(refs, table, lens, page)
    state = [t(refs), t(table, n_seqs, width), t(lens)]

    def step(call, *lists):
        before, m.moves, m.status = words.clone(), [], 0
        outs = {} if in_place else dict(refs_out=torch.full_like(state[0], 99), table_out=torch.full_like(state[1], 99))
        if not in_place and call is not ops.pages_compact:
            outs["lens_out"] = torch.full_like(state[2], 99)
        got = call(pool, *state[:2], **outs) if call is ops.pages_compact else call(pool, *state, *lists, **outs)
        state[:2] = got[:2]
        if call is not ops.pages_compact:
            state[2] = got[2]
        return before, got

    def check(before, got, status=True):
        same(m, [before], pool, *state, got[3] if status else None)

    nothing = t([]).reshape(0, 2)
    for fill in (False, True):
        if fill:                                         # every page taken, from the first sequence on
            want = [min(width, max(0, n_pages - width * b)) * page for b in range(n_seqs)]
            done = step(ops.pages_reserve, t(want))
            m.reserve(want)
            check(*done)
        done = step(ops.pages_fork, nothing)
        m.fork([])
        check(*done)
        done = step(ops.pages_free, t([]))
        m.free([])
        check(*done)
        done = step(ops.pages_compact)
        assert done[1][2].item() == m.compact() and not m.moves
        check(*done, status=False)
    done = step(ops.pages_reserve, t([width * page] * n_seqs))
    m.reserve([width * page] * n_seqs)
    check(*done)
    done = step(ops.pages_free, t(list(range(n_seqs))[::-1] * 1))
    m.free(list(range(n_seqs)))
    check(*done)
