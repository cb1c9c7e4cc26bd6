"""The 4-bit cache and its attention where calls are unusual: NaN in tokens that some rows see and others do not, more sequences than
one launch takes, pages that are no power of two and lie apart, lengths out of range, gradients asked for, calls at the same time."""
import math

import pytest
import torch

from tests.test_gpu_kv4 import _check_attention, _filled, _reference, _same, _table

pytestmark = pytest.mark.gpu


def _dev(x, dev):
    return torch.tensor(x, device=dev)


@pytest.mark.parametrize("d,group", [(64, 2), (128, 4), (256, 1)])
@pytest.mark.parametrize("new,at", [(5, 3), (90, 70), (300, 299), (300, 0)])
def test_a_nan_reaches_the_rows_that_see_it(cuda_device, d, group, new, at):
    """Keys or values of one new token and one head hold a NaN: rows before it are what they are without, rows from it on NaN."""
    from xpu_graph_b200 import lib, ops

    n, page, heads = new + 50, 32, 2
    table, lens, starts = _table([n], page, 12, cuda_device), _dev([n], cuda_device), _dev([0, new], cuda_device)
    q = torch.randn(new, heads * group, d, generator=torch.Generator().manual_seed(d)).bfloat16().to(cuda_device)
    token = 50 + at
    slot = table[0, token // page] * page + token % page
    g = torch.Generator(cuda_device).manual_seed(1)
    for side in ("keys", "values"):
        cache = _filled(12, heads, page, d, cuda_device)
        k, v = (torch.randn(1, heads, d, generator=g, device=cuda_device) for _ in range(2))
        (k if side == "keys" else v)[0, 1, d - 3] = math.nan  # the last group of channels of the second head
        ops.kv4_append(cache, k, v, slot[None])
        got = ops.kv4_attention(q, cache, table, lens, starts, new, d ** -0.5)
        ref = _reference(q, cache, table, [n], [0, new], d ** -0.5)  # (there the NaN is a 0)
        _check_attention(got[:at], tuple(x[:at] for x in ref), side, halves=new > 8)
        first = group  # rows of the other head
        _check_attention(got[:, :first], tuple(x[:, :first] for x in ref), side, halves=new > 8)
        assert torch.isnan(got[at:, first:, d - 64:]).all()
        if side == "keys":
            assert torch.isnan(got[at:, first:]).all()
    assert lib.tc_status() == 0


@pytest.mark.parametrize("new", [3, 70])
def test_a_row_of_q_that_is_not_finite(cuda_device, new):
    from xpu_graph_b200 import ops

    cache = _filled(6, 2, 64, 128, cuda_device)
    table, lens, starts = _table([200], 64, 6, cuda_device), _dev([200], cuda_device), _dev([0, new], cuda_device)
    q = torch.randn(new, 4, 128, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    ref = _reference(q, cache, table, [200], [0, new], 0.1)
    for bad in (math.nan, math.inf, -math.inf):
        p = q.clone()
        p[1, 2, 7] = bad
        got = ops.kv4_attention(p, cache, table, lens, starts, new, 0.1)
        assert not torch.isfinite(got[1, 2]).any()
        got[1, 2] = ref[0][1, 2].half()
        _check_attention(got, ref, f"{bad}", halves=new > 8)


def test_more_sequences_than_a_launch_takes(cuda_device):
    from xpu_graph_b200 import lib, ops

    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 41, (2500,), generator=g).tolist()
    lens[1023] = lens[1024] = lens[2048] = 0
    cache = _filled(sum(-(-n // 16) for n in lens) + 1, 1, 16, 64, cuda_device)
    table, n = _table(lens, 16, cache.shape[0], cuda_device), _dev(lens, cuda_device)
    q = torch.randn(2500, 2, 64, generator=g).bfloat16().to(cuda_device)
    got = ops.kv4_attention(q, cache, table, n, None, 1, 0.125)
    _check_attention(got, _reference(q, cache, table, lens, None, 0.125), "one row each")
    # none, one or two rows each, a few with many, rows in front of the first and behind the last
    new = torch.randint(0, 3, (2500,), generator=g)
    new[[7, 1030, 2499]] = 33
    starts = torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))) + 2
    q = torch.randn(int(starts[-1]) + 3, 2, 64, generator=g).bfloat16().to(cuda_device)
    for most in (33, 24, 2):  # both kernels, or the streaming one alone
        got = ops.kv4_attention(q, cache, table, n, starts.to(cuda_device), most, 0.125)
        _check_attention(got, _reference(q, cache, table, lens, starts.tolist(), 0.125), f"many {most}", halves=most == 33)
        assert not got[:2].any() and not got[starts[-1]:].any()
    assert lib.tc_status() == 0


@pytest.mark.parametrize("page,d", [(48, 128), (80, 64), (16, 256), (48, 256)])
def test_pages_of_any_size_that_lie_apart(cuda_device, page, d):
    """One layer of a cache whose pages hold several layers, 3 or 5 tiles a page: a stage's tiles end in different pages."""
    from xpu_graph_b200 import ops

    heads, group, lens, new = 2, 3, [500, 47, 49, 700], [1, 2, 40, 120]
    whole = torch.zeros(40 if page > 16 else 90, 3, heads, page // 16, 18 * d, dtype=torch.uint8, device=cuda_device)
    cache = whole[:, 1]
    pages = cache.shape[0]
    g = torch.Generator(cuda_device).manual_seed(d)
    k, v = (torch.randn(pages * page, heads, d, generator=g, device=cuda_device) for _ in range(2))
    ops.kv4_append(cache, k, v, torch.arange(pages * page, device=cuda_device))
    assert not whole[:, 0].any() and not whole[:, 2].any()
    table = _table(lens, page, pages, cuda_device)
    starts = [sum(new[:i]) for i in range(5)]
    q = torch.randn(starts[-1], heads * group, d, generator=g, device=cuda_device).half()
    got = ops.kv4_attention(q, cache, table, _dev(lens, cuda_device), _dev(starts, cuda_device), 120, d ** -0.5)
    _check_attention(got, _reference(q, cache, table, lens, starts, d ** -0.5), "apart", halves=True)
    got = ops.kv4_attention(q[:4], cache, table, _dev(lens, cuda_device), None, 1, d ** -0.5)
    _check_attention(got, _reference(q[:4], cache, table, lens, None, d ** -0.5), "apart")


def test_lengths_and_starts_out_of_range(cuda_device):
    """Negative lengths count as none; starts beyond the rows, or that go back, stay inside q and the result."""
    from xpu_graph_b200 import lib, ops

    cache = _filled(8, 2, 16, 64, cuda_device)
    table = torch.arange(8, device=cuda_device).view(2, 4)
    q = torch.randn(100, 4, 64, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    assert not ops.kv4_attention(q[:2], cache, table, _dev([-1, -(1 << 62)], cuda_device), None, 1, 0.1).any()
    assert not ops.kv4_attention(q, cache, table, _dev([-1, 0], cuda_device), _dev([0, 60, 100], cuda_device), 60, 0.1).any()
    lens = _dev([64, 1 << 62], cuda_device)
    for most in (1, 100):
        got = ops.kv4_attention(q, cache, table, lens, _dev([0, 3, 1 << 40], cuda_device), most, 0.1)
        want = ops.kv4_attention(q, cache, table, _dev([64, 64], cuda_device), _dev([0, 3, 100], cuda_device), most, 0.1)
        assert torch.equal(got, want)
        for starts in ([5, 3, 90], [-7, 100, 2], [200, 300, 400]):
            assert ops.kv4_attention(q, cache, table, lens, _dev(starts, cuda_device), most, 0.1).shape == q.shape
    # no sequence at all
    assert not ops.kv4_attention(q, cache, table[:0], lens[:0], lens.new_zeros(1), 100, 0.1).any()
    torch.cuda.synchronize()
    assert lib.tc_status() == 0


@pytest.mark.parametrize("d,group", [(64, 1), (128, 4), (256, 2)])
def test_one_sequence_with_rows_around_it(cuda_device, d, group):
    """However many of the rows are the sequence's, and whatever the hint says: its rows attend, the others are zeros."""
    from xpu_graph_b200 import lib, ops

    cache = _filled(60, 2, 32, d, cuda_device)
    table = _table([1700], 32, 60, cuda_device)
    q = torch.randn(300, 2 * group, d, generator=torch.Generator().manual_seed(d)).half().to(cuda_device)
    for n, lo, hi, most in ((1700, 5, 290, 300), (1700, 0, 300, 300), (333, 298, 300, 300), (90, 7, 8, 4000), (40, 10, 130, 120), (0, 3, 200, 300), (64, 9, 9, 300), (1700, 100, 300, 1)):
        got = ops.kv4_attention(q, cache, table, _dev([n], cuda_device), _dev([lo, hi], cuda_device), most, d ** -0.5)
        _check_attention(got, _reference(q, cache, table, [n], [lo, hi], d ** -0.5), f"{n} {lo} {hi} {most}", halves=most > 8)
        assert not got[:lo].any() and not got[hi:].any()
    assert lib.tc_status() == 0


def test_gradients_are_refused(cuda_device):
    """Serving operators: inputs that need a gradient run, going back through them does not."""
    from xpu_graph_b200 import ops

    cache = _filled(2, 1, 16, 64, cuda_device)
    k = torch.randn(3, 1, 64, device=cuda_device, requires_grad=True)
    slots = torch.arange(3, device=cuda_device)
    ops.kv4_append(cache.clone(), k, k, slots)
    q = torch.randn(1, 1, 64, device=cuda_device).half().requires_grad_()
    out = ops.kv4_attention(q, cache, slots[None, :1], _dev([3], cuda_device), None, 1, 0.1)
    with pytest.raises(RuntimeError):
        out.float().sum().backward()
    assert torch.equal(out, ops.kv4_attention(q.detach(), cache, slots[None, :1], _dev([3], cuda_device), None, 1, 0.1))


def test_two_streams_and_two_graphs_at_once(cuda_device):
    """Calls that split their keys (and so use workspaces) side by side, eagerly and as graphs from one memory pool."""
    from xpu_graph_b200 import lib, ops

    cache = _filled(200, 2, 64, 128, cuda_device)
    table = torch.arange(200, device=cuda_device)[None]
    lens = _dev([12800], cuda_device)
    g = torch.Generator().manual_seed(1)
    q = [torch.randn(r, 8, 128, generator=g).bfloat16().to(cuda_device) for r in (2, 40)]
    at = [_dev([0, len(x)], cuda_device) for x in q]

    def call(i):
        return ops.kv4_attention(q[i], cache, table, lens, at[i], len(q[i]), 0.1)

    want = [call(0), call(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(call(i))
        graphs.append(graph)
    for _ in range(3):
        for i in (1, 0, 0, 1):  # (one after the other: graphs of one pool share its memory)
            graphs[i].replay()
            assert _same(outs[i], want[i])
    assert lib.tc_status() == 0
