"""CPU tests of the paged cache's entry points: what they refuse, before anything is launched."""
import ctypes as C

import pytest

EINVAL = -22
PTR = 0x1000            # a 16-byte aligned address that nobody reads


@pytest.fixture(scope="module")
def lib():
    from ds4cuda_b200 import _lib, build
    build.build()
    return _lib.load()


def kv(**kw):
    from ds4cuda_b200 import _lib
    d = dict(row_format=_lib.KV_FP8_BLOCK64, head_dim=512, n_rot=64, page_rows=64, n_pages=10, codes=PTR, scales=PTR, tail=PTR, raw=None)
    d.update(kw)
    return _lib.PagedKvStruct(*[d[n] for n, _ in _lib.PagedKvStruct._fields_])


def decode(lib, cache=None, q=PTR, table=PTR, width=4, lens=PTR, n_seqs=2, heads=64, scale=1.0, sink=None, window=0, first=0, out=PTR,
           ws=PTR, ws_bytes=1 << 40):
    return lib.ds4b200_attn_decode_paged_bf16(q, C.byref(cache or kv()), table, width, lens, n_seqs, heads, scale, sink, window, first, out,
                                              None, ws, ws_bytes, None)


def window(lib, cache=None, q=PTR, n_tokens=5, q_start=PTR, n_seqs=2, heads=64, **kw):
    return lib.ds4b200_attn_window_paged_bf16(q, n_tokens, C.byref(cache or kv()), PTR, 4, PTR, q_start, n_seqs, heads, 1.0, None,
                                              kw.get("window", 128), 0, PTR, None, PTR, kw.get("ws_bytes", 1 << 40), None)


def test_attention_refusals(lib):
    from ds4cuda_b200 import _lib
    nan, inf = float("nan"), float("inf")
    for bad in (dict(q=None), dict(q=PTR + 8), dict(table=None), dict(lens=None), dict(out=None), dict(out=PTR + 2), dict(ws=None),
                dict(ws_bytes=1000), dict(width=0), dict(n_seqs=-1), dict(n_seqs=4097), dict(heads=0), dict(heads=1025), dict(scale=nan),
                dict(scale=inf), dict(window=-1), dict(first=-1)):
        assert decode(lib, **bad) == EINVAL, bad
        assert lib.ds4b200_last_error()
    for bad in (dict(row_format=3), dict(head_dim=64), dict(head_dim=192), dict(head_dim=640), dict(n_rot=32), dict(page_rows=0),
                dict(n_pages=-1), dict(n_pages=1 << 25, page_rows=64), dict(codes=None), dict(codes=PTR + 4), dict(scales=None),
                dict(tail=None), dict(row_format=_lib.KV_F32), dict(row_format=_lib.KV_F32, raw=PTR + 4), dict(row_format=_lib.KV_FP8_ROW, codes=None)):
        assert decode(lib, kv(**bad)) == EINVAL, bad
        assert window(lib, kv(**bad)) == EINVAL, bad
    wide = kv(page_rows=1 << 20, n_pages=4)
    assert decode(lib, wide, width=1 << 11) == EINVAL                        # positions would not fit 32 bits
    for bad in (dict(q=None), dict(q_start=None), dict(n_tokens=-1), dict(n_tokens=1 << 40), dict(n_seqs=4097), dict(ws_bytes=0)):
        assert window(lib, **bad) == EINVAL, bad
    assert decode(lib, n_seqs=0) == 0 and window(lib, n_tokens=0) == 0       # nothing to do, nothing launched
    assert lib.ds4b200_attn_workspace_bytes(0, 512) == EINVAL and lib.ds4b200_attn_workspace_bytes(64, 1024) == EINVAL
    assert lib.ds4b200_attn_workspace_bytes(64, 512) > 0


def test_page_refusals(lib):
    from ds4cuda_b200 import _lib

    def arrays(base=PTR, size=64, n=1):
        return (_lib.PageArray * max(1, n))(*[_lib.PageArray(base, size)] * n)

    big = 1 << 40

    def fork(a=None, n=1, pages=10, rows=4, ptr=PTR, seqs=3, width=4, pairs=PTR, n_pairs=2, status=PTR, ws=PTR, size=big):
        return lib.ds4b200_pages_fork(a or arrays(), n, pages, rows, ptr, PTR, PTR, PTR, PTR, PTR, seqs, width, pairs, n_pairs, status, ws, size, None)

    for bad in (dict(a=arrays(base=None)), dict(a=arrays(base=PTR + 2)), dict(a=arrays(size=0)), dict(a=arrays(size=6)), dict(n=-1), dict(n=193),
                dict(pages=-1), dict(pages=(1 << 20) + 1), dict(rows=0), dict(ptr=None), dict(seqs=-1), dict(width=0), dict(width=1 << 30), dict(pairs=None),
                dict(pairs=PTR + 4), dict(n_pairs=-1), dict(status=None), dict(ws=None), dict(ws=PTR + 4), dict(size=8)):
        assert fork(**bad) == EINVAL, bad
    assert lib.ds4b200_pages_copy(arrays(), 1, 10, None, 1, PTR, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_copy(arrays(), 1, 10, PTR, 1, PTR, PTR, 0, None) == EINVAL
    assert lib.ds4b200_pages_reserve(10, 4, PTR, PTR, PTR, PTR, PTR, PTR, None, 3, 4, PTR, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_reserve(10, 4, PTR, PTR, PTR, PTR, None, PTR, PTR, 3, 4, PTR, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_free(10, 4, PTR, PTR, PTR, PTR, PTR, PTR, 3, 4, None, 1, PTR, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_compact(arrays(), 1, 10, PTR, PTR, PTR, None, 3, 4, PTR, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_compact(arrays(), 1, 10, PTR, PTR, PTR, PTR, 3, 4, None, PTR, big, None) == EINVAL
    assert lib.ds4b200_pages_workspace_bytes((1 << 20) + 1, 1, 1) == EINVAL
    assert lib.ds4b200_pages_workspace_bytes(10, 3, 2) >= 100


def test_python_mirror_refuses_wrong_tensors():
    import torch
    from ds4cuda_b200 import ops
    with pytest.raises(ValueError):
        ops.PagedKv(ops.KV_F32, 3, raw=torch.zeros(4, 128))              # not whole pages
    with pytest.raises(ValueError):
        ops.PagedKv(ops.KV_F32, 2, raw=torch.zeros(4, 128))              # not on a GPU
    with pytest.raises(ValueError):
        ops.PagedKv(7, 2, codes=torch.zeros(4, 128, dtype=torch.uint8))
    with pytest.raises(ValueError):
        ops.PagedKv(ops.KV_FP8_ROW, 2, codes=torch.zeros(4, 128, dtype=torch.uint8), scales=torch.zeros(4, 2))


def test_list_model_of_the_pages():
    """The model itself, on a case worked out by hand."""
    import paged_model
    m = paged_model.Pages([1, 0, 1, 0, 0, 1], [[2, 5, -1], [-1] * 3, [0, -1, -1], [-1] * 3], [6, 0, 4, 0], 4)
    m.fork([(0, 1), (2, 3)])
    assert m.table == [[2, 5, -1], [2, 1, -1], [0, -1, -1], [0, -1, -1]] and m.refs == [2, 1, 2, 0, 0, 1]
    assert m.moves == [(5, 1)] and m.lens == [6, 6, 4, 4]
    m.free([0, 0])
    assert m.refs == [2, 1, 1, 0, 0, 0] and m.lens == [0, 6, 4, 4]
    m.reserve([9, 0, 0, 0])
    assert m.table[0] == [3, 4, 5] and m.refs == [2, 1, 1, 1, 1, 1]
    m.free([2])
    m.free([3])
    m.moves = []
    assert m.compact() == 5 and m.moves == [(5, 0)] and m.table[0] == [3, 4, 0]


@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_of_words_off_their_four_bytes_are_refused(lib, off):
    """Tables, lengths, lists, sinks and log-sums are read as words: an odd address is an error here, and no fault on the device."""
    bad = PTR + off
    dec = lambda **k: lib.ds4b200_attn_decode_paged_bf16(PTR, C.byref(kv()), k.get("table", PTR), 4, k.get("lens", PTR), 2, 64, 1.0, k.get("sink"), 0, 0,
                                                         PTR, k.get("lse"), PTR, 1 << 40, None)
    win = lambda **k: lib.ds4b200_attn_window_paged_bf16(PTR, 5, C.byref(kv()), k.get("table", PTR), 4, k.get("lens", PTR), k.get("start", PTR), 2, 64, 1.0,
                                                         k.get("sink"), 128, 0, PTR, k.get("lse"), PTR, 1 << 40, None)
    for k in ("table", "lens", "sink", "lse"):
        assert dec(**{k: bad}) == EINVAL and win(**{k: bad}) == EINVAL, k
        assert b"align" in lib.ds4b200_last_error()
    assert win(start=bad) == EINVAL
    for i in range(6):
        p = [PTR] * 6
        p[i] = bad
        assert lib.ds4b200_pages_fork(None, 0, 10, 4, *p, 3, 4, PTR, 2, PTR, PTR, 1 << 40, None) == EINVAL, i
        assert lib.ds4b200_pages_reserve(10, 4, *p, PTR, 3, 4, PTR, PTR, 1 << 40, None) == EINVAL, i
        assert lib.ds4b200_pages_free(10, 4, *p, 3, 4, PTR, 2, PTR, PTR, 1 << 40, None) == EINVAL, i
        if i < 4:
            assert lib.ds4b200_pages_compact(None, 0, 10, *p[:4], 3, 4, PTR, PTR, 1 << 40, None) == EINVAL, i
    assert lib.ds4b200_pages_reserve(10, 4, *[PTR] * 6, bad, 3, 4, PTR, PTR, 1 << 40, None) == EINVAL
    assert lib.ds4b200_pages_free(10, 4, *[PTR] * 6, 3, 4, bad, 2, PTR, PTR, 1 << 40, None) == EINVAL
