"""KV4Cache on the host: what forks, frees and compactions do to page lists and to the pages' contents, with page copies done on the
CPU."""
import random

import pytest
import torch

from xpu_graph_b200 import kv_cache


@pytest.fixture
def cache(monkeypatch):
    def copy_pages(t, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        t[torch.tensor(dst)] = t[torch.tensor(src)]

    monkeypatch.setattr(kv_cache.ops, "copy_pages", copy_pages)
    return kv_cache.KV4Cache(12, 1, 64, page_size=16, layers=2, device="cpu")


def test_pages_come_and_go(cache):
    a, b = cache.new(), cache.new()
    assert cache.extend(a, 17).tolist() == list(range(17))
    assert cache.extend(b, 3).tolist() == [32, 33, 34]
    assert cache.extend(a, 0).numel() == 0 and cache.extend(a, 15).tolist() == list(range(17, 32))
    assert cache.pages(a) == (0, 1) and cache.free_pages == 9
    table, lens = cache.tables([b, a])
    assert table.tolist() == [[2, -1], [0, 1]] and lens.tolist() == [3, 32]
    table, lens = cache.tables([])
    assert table.shape == (0, 0) and lens.shape == (0,)
    cache.free(a)
    assert cache.free_pages == 11
    with pytest.raises(MemoryError):
        cache.extend(b, 12 * 16)
    assert cache.length(b) == 3 and cache.free_pages == 11
    with pytest.raises(KeyError):
        cache.free(a)
    with pytest.raises(ValueError):
        cache.extend(b, -1)


def test_a_fork_shares_full_pages_and_copies_the_last(cache):
    a = cache.new()
    cache.extend(a, 40)
    cache.layers[1][2] = 7
    b = cache.fork(a)
    assert cache.pages(b)[:2] == cache.pages(a)[:2] and cache.pages(b)[2] not in cache.pages(a) and cache.length(b) == 40
    assert (cache.layers[1][cache.pages(b)[2]] == 7).all() and cache.free_pages == 8
    cache.free(a)
    assert cache.free_pages == 9
    cache.free(b)
    assert cache.free_pages == 12
    c = cache.new()
    cache.extend(c, 32)
    assert cache.pages(cache.fork(c)) == cache.pages(c)  # nothing to copy
    assert cache.pages(cache.fork(cache.new())) == ()


def test_any_order_of_them_keeps_every_sequence(cache):
    rng = random.Random(0)
    want = {}  # sequence -> a number per token, written to both layers' pages at the token's place
    stamp = 0
    for step in range(400):
        seq = rng.choice(list(want)) if want else None
        what = rng.random()
        if seq is None or what < 0.2:
            want[cache.new()] = []
        elif what < 0.6:
            n = rng.randint(0, 20)
            try:
                slots = cache.extend(seq, n).tolist()
            except MemoryError:
                continue
            for s in slots:
                stamp += 1
                for layer in cache.layers:
                    layer[s // 16, 0, 0, s % 16 * 4:s % 16 * 4 + 4] = torch.tensor([stamp >> 8 * i & 255 for i in range(4)], dtype=torch.uint8)
                want[seq].append(stamp)
        elif what < 0.75:
            try:
                want[cache.fork(seq)] = list(want[seq])
            except MemoryError:
                continue
        elif what < 0.9:
            cache.free(seq)
            del want[seq]
        else:
            used = cache.compact()
            assert used + cache.free_pages == 12 and all(p < used for s in want for p in cache.pages(s))
        for s, numbers in want.items():
            assert cache.length(s) == len(numbers)
            for layer in cache.layers:
                got = [int.from_bytes(bytes(layer[cache.pages(s)[i // 16], 0, 0, i % 16 * 4:i % 16 * 4 + 4].tolist()), "little") for i in range(len(numbers))]
                assert got == numbers


@pytest.mark.parametrize("bad", [dict(pages=0), dict(kv_heads=0), dict(head_dim=96), dict(page_size=24), dict(page_size=0), dict(layers=0)])
def test_refusals(bad):
    with pytest.raises(ValueError):
        kv_cache.KV4Cache(**{**dict(pages=4, kv_heads=1, head_dim=64, device="cpu"), **bad})


def test_a_fork_that_fails_leaves_the_pages_free(cache, monkeypatch):
    a = cache.new()
    cache.extend(a, 20)
    free, working = cache.free_pages, kv_cache.ops.copy_pages

    def failing(t, src, dst):
        raise RuntimeError("no copy")

    monkeypatch.setattr(kv_cache.ops, "copy_pages", failing)
    for _ in range(20):  # more often than there are pages
        with pytest.raises(RuntimeError, match="no copy"):
            cache.fork(a)
    assert cache.free_pages == free and cache.pages(a) == (0, 1)
    monkeypatch.setattr(kv_cache.ops, "copy_pages", working)
    b = cache.fork(a)
    assert cache.pages(b)[0] == 0 and cache.free_pages == free - 1
    cache.free(a), cache.free(b)
    assert cache.free_pages == 12


def test_an_extension_that_fails_changes_nothing(cache, monkeypatch):
    """The slots' tensor may fail to be made: the sequence is no longer than before, and its pages are free."""
    a = cache.new()
    cache.extend(a, 20)

    class Full:
        def __init__(self, *args, **kwargs):
            pass

        def to(self, *args, **kwargs):
            raise RuntimeError("out of memory")

    with monkeypatch.context() as m:
        m.setattr(kv_cache.torch, "tensor", Full)
        for _ in range(20):
            with pytest.raises(RuntimeError, match="out of memory"):
                cache.extend(a, 30)
    assert cache.length(a) == 20 and cache.pages(a) == (0, 1) and cache.free_pages == 10
    assert cache.extend(a, 13).tolist() == list(range(20, 33)) and cache.pages(a) == (0, 1, 2)
