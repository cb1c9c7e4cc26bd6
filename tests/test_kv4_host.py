"""What the entries of the 4-bit cache refuse before anything touches a GPU."""
import ctypes

import pytest
import torch

from xpu_graph_b200 import lib, ops

BUF = ctypes.create_string_buffer(4096 + 16)
P = ctypes.c_void_p((ctypes.addressof(BUF) + 15) & ~15)
ODD = ctypes.c_void_p(P.value + 8)
H = lib.XG_F16


def test_cache_arguments():
    L = lib.load()

    def append(cache=P, pages=2, heads=1, page_size=16, stride=18 * 64, k=P, v=P, slots=P, tokens=1, d=64, dtype=lib.XG_F32):
        return L.xg_kv4_append(cache, pages, heads, page_size, stride, k, v, slots, tokens, d, d, d, d, d, dtype, None)

    assert append(d=96) == -2 and append(d=32) == -2
    for bad in ({"page_size": 24}, {"page_size": 0}, {"pages": -1}, {"heads": 0}, {"stride": 8}, {"stride": 18 * 64 - 16}, {"cache": ODD}, {"cache": None},
                {"tokens": -1}, {"k": None}, {"v": None}, {"slots": None}, {"dtype": 9}):
        assert append(**bad) == -1, bad
    assert append(heads=70000, stride=70000 * 18 * 64) < 0 and append(page_size=1 << 21, stride=1 << 32) < 0 and append(pages=1 << 33) < 0
    assert append(tokens=0) == 0 and append(tokens=0, k=None, v=None, slots=None) == 0 and append(pages=0, cache=None) == 0

    def read(k=P, v=P, slots=P, tokens=1, dtype=lib.XG_F32, page_size=16):
        return L.xg_kv4_read(P, 2, 1, page_size, 18 * 64, slots, tokens, 64, k, v, dtype, None)

    for bad in ({"k": None}, {"v": ODD}, {"slots": None}, {"tokens": -1}, {"dtype": 5}, {"page_size": 17}):
        assert read(**bad) == -1, bad
    assert read(tokens=0) == 0


def test_attention_arguments():
    L = lib.load()

    def attend(q=P, kv_heads=2, table=P, table_pages=3, lens=P, out=P, tokens=1, batch=1, q_heads=4, d=64, max_q=1, dtype=H, ws=None, ws_bytes=0, pages=2):
        return L.xg_kv4_attention(q, P, pages, kv_heads, 16, kv_heads * 18 * 64, table, table_pages, table_pages, lens, None, out, tokens, batch, q_heads, d, max_q,
                                  q_heads * d, d, 1.0, dtype, ws, ws_bytes, None)

    assert attend(dtype=lib.XG_F32) == -2 and attend(d=80) == -2
    for bad in ({"tokens": -1}, {"batch": -1}, {"q_heads": 0}, {"q_heads": 5}, {"max_q": -1}, {"table_pages": -1}, {"ws_bytes": -1}, {"q": None}, {"out": None},
                {"out": ODD}, {"lens": None}, {"table": None}):
        assert attend(**bad) == -1, bad
    assert attend(table_pages=1 << 27) < 0 and attend(tokens=1 << 32) < 0 and attend(batch=1 << 24) < 0
    # a workspace that is too small, missing, or not aligned
    need = L.xg_kv4_attention_workspace_bytes(1, 1, 4, 2, 64, 1, 16 * 1000)
    assert need > 0
    for ws, size in ((None, 0), (P, need - 1), (ODD, need), (None, need)):
        assert attend(table_pages=1000, ws=ws, ws_bytes=size) == -1
        assert "workspace" in lib.last_error()
    assert attend(tokens=0) == 0
    assert L.xg_kv4_attention_workspace_bytes(0, 1, 4, 2, 64, 1, 1000) == 0 and L.xg_kv4_attention_workspace_bytes(1, 1, 4, 2, 64, 1, 512) == 0


def test_page_arguments():
    L = lib.load()

    def copy(src, dst, base=P, pages=4, size=32, stride=32, count=None):
        n = len(src)
        a, b = (ctypes.c_int64 * n)(*src), (ctypes.c_int64 * n)(*dst)
        return L.xg_copy_pages(base, pages, size, stride, a, b, n if count is None else count, None)

    for src, dst in (([4], [0]), ([0], [4]), ([-1], [0]), ([0], [-1]), ([0, 1 << 40], [1, 2])):
        assert copy(src, dst) == -1
    assert copy([0], [1], base=None) == -1 and copy([0], [1], count=-1) == -1 and copy([0], [1], size=-1) == -1
    for bad in ({"base": ODD}, {"size": 24}, {"stride": 40}, {"stride": 16}):
        assert copy([0], [1], **bad) == -2, bad
    assert copy([0], [1], pages=1 << 32) < 0
    assert copy([], []) == 0 and copy([0], [1], size=0) == 0


def test_norm_and_rotation_arguments():
    L = lib.load()

    def rot(q=P, k=P, cos=P, sin=P, rows=4, rot=8, pos=P, axes=1, sections=None, q_out=P, k_out=P, tokens=1, q_heads=1, k_heads=1, d=8, dtype=H, w=H, t=H):
        s = None if sections is None else (ctypes.c_int64 * len(sections))(*sections)
        return L.xg_qk_norm_rope(q, k, None, None, 1e-6, cos, sin, rows, rot, pos, axes, tokens, s, q_out, k_out, tokens, q_heads, k_heads, d, d, d, d, d, dtype, w, t, None)

    for bad in ({"q": None}, {"k_out": None}, {"cos": None}, {"sin": None}, {"pos": None}, {"rot": 7}, {"rot": 10}, {"d": 0}, {"tokens": -1}, {"rows": -1},
                {"q_heads": -1}, {"dtype": 8}, {"w": lib.XG_BF16}, {"t": lib.XG_BF16}, {"axes": 0}, {"axes": 9}, {"axes": 2}, {"axes": 2, "sections": [1, 1]},
                {"axes": 2, "sections": [-1, 5]}, {"axes": 2, "sections": [3, 2]}):
        assert rot(**bad) == -1, bad
    assert rot(q_heads=70000) < 0 and rot(d=1 << 17, rot=8) < 0
    assert rot(tokens=0, q=None, k=None, cos=None, sin=None, pos=None, q_out=None, k_out=None) == 0


def test_page_lists():
    """copy_pages takes sequences and tensors of any integers that fit; a host tensor is not a cache."""
    for bad in ([1.5], ["1"], [1 << 70], [None] * 300):
        with pytest.raises((TypeError, OverflowError, ValueError)):
            ops._host_ints(bad)
    for n in (0, 1, 255, 256, 1000):
        assert torch.equal(ops._host_ints(list(range(n))), torch.arange(n)) and torch.equal(ops._host_ints(range(n)), torch.arange(n))
        assert torch.equal(ops._host_ints(tuple(range(n))), torch.arange(n))
    with pytest.raises((RuntimeError, NotImplementedError)):
        ops.copy_pages(torch.zeros(2, 16), [0], [1])


def test_a_row_for_each_sequence_where_there_are_no_starts():
    """Without q_starts sequence b's row is row b: more sequences than rows are refused before any launch."""
    L = lib.load()

    def attend(tokens, batch, max_q):
        need = L.xg_kv4_attention_workspace_bytes(tokens, batch, 4, 2, 64, max_q, 48)
        return L.xg_kv4_attention(P, P, 2, 2, 16, 2 * 18 * 64, P, 3, 3, P, None, P, tokens, batch, 4, 64, max_q, 256, 64, 1.0, H, P, max(need, 0), None)

    for tokens, batch, max_q in ((1, 2, 1), (1, 2, 100), (5, 4000, 1), (5, 4000, 100)):
        assert attend(tokens, batch, max_q) == -1, (tokens, batch, max_q)
        assert "row" in lib.last_error()
    assert attend(0, 2, 1) == 0


def test_page_lists_under_another_default_device():
    for n in (0, 2, 300):
        with torch.device("meta"):
            got = ops._host_ints(list(range(n)))
        assert got.device.type == "cpu" and torch.equal(got, torch.arange(n))


@pytest.mark.parametrize("n", [0, 2, 300])
def test_copy_pages_of_a_fake_cache(n):
    """Lists of any length with tensors that have no memory, as graph compilers trace them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        cache = torch.empty(1000, 4, 16, device="cuda")
        assert ops.copy_pages(cache, list(range(n)), range(n, 2 * n)) is None
        for bad in ([1.5], ["1"] * 300):
            with pytest.raises((TypeError, ValueError)):
                ops.copy_pages(cache, bad, bad)
