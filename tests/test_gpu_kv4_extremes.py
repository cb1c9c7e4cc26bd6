"""The 4-bit cache at the ends of what it holds: constants that fp16 rounds up, infinities in operands and results, weights and
query channels far below the largest."""
import math

import pytest
import torch

from tests.test_gpu_kv4 import _check_attention, _filled, _reference, _same, _table

pytestmark = pytest.mark.gpu


def _dev(x, dev):
    return torch.tensor(x, device=dev)


def _scales(cache):
    """Every pair's scale, keys' and values'."""
    d = cache.shape[-1] // 18
    return cache[..., 16 * d:].contiguous().view(torch.float16).unflatten(-1, (-1, 2))[..., 0].float()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_constants_that_fp16_rounds_up(cuda_device, d, dtype):
    """Tokens whose channels all hold one fp32 value: its fp16 least value may lie above it. Alone, over more than a tile, with ordinary
    tokens behind them; few and many new tokens."""
    from xpu_graph_b200 import lib, ops

    for constant in (0.3, 0.1, -0.3, 1000.3, 3e-6):
        for constants, others in ((1, 0), (33, 0), (33, 100), (100, 40)):
            n = constants + others
            cache = _filled(12, 2, 16, d, cuda_device)
            k = torch.full((constants, 2, d), constant, device=cuda_device)
            ops.kv4_append(cache, k, k, torch.arange(constants, device=cuda_device))
            assert (_scales(cache) >= 0).all()
            table = torch.arange(12, device=cuda_device)[None]
            for rows in (1, min(n, 90)):
                q = torch.randn(rows, 4, d, generator=torch.Generator().manual_seed(n)).to(dtype).to(cuda_device)
                got = ops.kv4_attention(q, cache, table, _dev([n], cuda_device), _dev([0, rows], cuda_device), rows, d ** -0.5)
                _check_attention(got, _reference(q, cache, table, [n], [0, rows], d ** -0.5), f"{constant} {constants} {others} {rows}", halves=rows > 8)
    assert lib.tc_status() == 0


@pytest.mark.parametrize("beside", ["zeros", "ordinary", "the other infinity", "60000 below"])
@pytest.mark.parametrize("d,group", [(64, 2), (128, 4), (256, 1)])
@pytest.mark.parametrize("new,at", [(5, 3), (90, 70), (300, 299), (300, 0)])
def test_infinities_are_held_as_the_largest_values(cuda_device, d, group, new, at, beside):
    """Keys or values of one new token and one head hold an infinity. Code 15 of such a group may stand for more than fp16 holds: rows
    before the token are what they are without it, rows from it on are finite and see the value."""
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
        x = k if side == "keys" else v
        if beside == "zeros":
            x[0, 1, d - 64:] = 0
        x[0, 1, d - 3] = math.inf
        if beside == "the other infinity":
            x[0, 1, d - 9] = -math.inf
        if beside == "60000 below":
            x[0, 1, d - 9] = -60000.0
        ops.kv4_append(cache, k, v, slot[None])
        got = ops.kv4_attention(q, cache, table, lens, starts, new, d ** -0.5)
        assert torch.isfinite(got).all(), side
        _check_attention(got, _reference(q, cache, table, [n], [0, new], d ** -0.5), side, halves=new > 8)
        if side == "values":
            assert (got[at:, group:, d - 3].abs() > 1.0).any()
    assert lib.tc_status() == 0


def test_infinities_read_back_in_fp16(cuda_device):
    """fp16 results end at fp16's largest value, where the same codes and scales stand for more in fp32."""
    from xpu_graph_b200 import ops

    x = torch.randn(6, 2, 128, generator=torch.Generator().manual_seed(0))
    x[0, 0, 3], x[1, 1, 70], x[2, 0, 5], x[2, 0, 6], x[3, 1, 0] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    x[4, 0, :64] = 0
    x[4, 0, 9] = math.inf
    x = x.to(cuda_device)
    cache = torch.zeros(1, 2, 1, 18 * 128, dtype=torch.uint8, device=cuda_device)
    slots = torch.arange(6, device=cuda_device)
    ops.kv4_append(cache, x, x.flip(0), slots)
    for got, full in zip(ops.kv4_read(cache, slots, torch.float16), ops.kv4_read(cache, slots, torch.float32)):
        assert not torch.isinf(got).any() and (full > 65520).any()
        assert _same(got, full.clamp(-65504.0, 65504.0).half())


@pytest.mark.parametrize("d,group", [(64, 2), (128, 4), (256, 1)])
@pytest.mark.parametrize("new", [1, 7, 90])
@pytest.mark.parametrize("sharp", [1.0, 4.0, 16.0])
def test_averages_of_infinities_in_fp16(cuda_device, d, group, new, sharp):
    """Rows whose weight lies on tokens with infinite values: the largest value, of either sign, by both kernels."""
    from xpu_graph_b200 import ops

    n = 200
    x = torch.zeros(n, 2, d, device=cuda_device)
    x[:, 0, ::2], x[:, 0, 1::2], x[:, 1, 5] = math.inf, -math.inf, math.inf
    cache = torch.zeros(7, 2, 2, 18 * d, dtype=torch.uint8, device=cuda_device)
    ops.kv4_append(cache, torch.randn(n, 2, d, generator=torch.Generator().manual_seed(0)).to(cuda_device), x, torch.arange(n, device=cuda_device))
    q = torch.randn(new, 2 * group, d, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    got = ops.kv4_attention(q, cache, torch.arange(7, device=cuda_device)[None], _dev([n], cuda_device), _dev([0, new], cuda_device), new, sharp * d ** -0.5).float()
    # weights that add to 1 within 200 roundings of 2^-11 at most, and fp32 sums
    assert ((got - x.repeat_interleave(group, 1)[:1].clamp(-65504, 65504)).abs() <= 2.0 ** -11 * 65504 * 2).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [60, 70])  # (up to 64 are streamed at head dim 64)
def test_many_keys_far_below_the_largest_score(cuda_device, rows, d, dtype):
    """One key 17.5 above 16383 others, whose weights of e^-17.5 make 0.04 % of the sum and, as the first value is 0, all of the result.
    A weight of 2^-18.2 beside a largest of 2^7 is 54 steps of fp16's smallest, half a step off at most: 2^-6.7. The result's own
    rounding is 2^-8 at most, the sums add less than 2^-12."""
    from xpu_graph_b200 import ops

    n = 16384
    cache = torch.zeros(n // 64, 1, 4, 18 * d, dtype=torch.uint8, device=cuda_device)
    k, v = torch.zeros(n, 1, d, device=cuda_device), torch.ones(n, 1, d, device=cuda_device)
    k[0], v[0] = 1.0, 0.0
    ops.kv4_append(cache, k, v, torch.arange(n, device=cuda_device))
    table = torch.arange(n // 64, device=cuda_device)[None]
    for around in (0, 150 * 256):  # rows of no sequence, with which the keys stay in one piece
        q = torch.ones(rows + around, 1, d, device=cuda_device, dtype=dtype)
        got = ops.kv4_attention(q, cache, table, _dev([n], cuda_device), _dev([0, rows], cuda_device), rows, 17.5 / d)[:rows, 0].double()
        weight = (n - rows + torch.arange(rows, device=cuda_device)[:, None].double()) * math.exp(-17.5)
        want = weight / (1 + weight)
        tol = 2.0 ** -32 / math.exp(-17.5) + torch.finfo(dtype).eps / 2 + 2.0 ** -12
        assert ((got - want).abs() <= tol * want).all(), (around, (got / want).amin().item(), (got / want).amax().item())


@pytest.mark.parametrize("new", [3, 70])
def test_a_channel_far_above_the_others(cuda_device, new):
    """fp16 queries with one channel 2^23 times the others', where the keys are zero: the others make the scores."""
    from xpu_graph_b200 import ops

    d, n = 128, 300
    g = torch.Generator().manual_seed(0)
    cache = torch.zeros(10, 2, 2, 18 * d, dtype=torch.uint8, device=cuda_device)
    k, v = torch.randn(320, 2, d, generator=g) * 500, torch.randn(320, 2, d, generator=g)
    k[..., :64] = 0
    ops.kv4_append(cache, k.to(cuda_device), v.to(cuda_device), torch.arange(320, device=cuda_device))
    q = torch.randn(new, 4, d, generator=g) * 2.0 ** -8
    q[..., :64] = 0
    q[..., 7] = 2.0 ** 15
    q = q.half().to(cuda_device)
    table = torch.arange(10, device=cuda_device)[None]
    got = ops.kv4_attention(q, cache, table, _dev([n], cuda_device), _dev([0, new], cuda_device), new, 0.5)
    _check_attention(got, _reference(q, cache, table, [n], [0, new], 0.5), "scores of small channels", halves=new > 8)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [3, 90])
def test_rows_of_any_size(cuda_device, d, new):
    """bf16 queries near the ends of what the type holds, with a scale that makes scores of ordinary size of them."""
    from xpu_graph_b200 import ops

    n = 300
    cache = _filled(10, 2, 32, d, cuda_device)
    table = torch.arange(10, device=cuda_device)[None]
    q = torch.randn(new, 4, d, generator=torch.Generator().manual_seed(d)).bfloat16().to(cuda_device)
    for power in (2.0 ** 99, 2.0 ** 103, 2.0 ** 112, 2.0 ** 122, 2.0 ** -95):
        got = ops.kv4_attention(q * power, cache, table, _dev([n], cuda_device), _dev([0, new], cuda_device), new, d ** -0.5 / power)
        _check_attention(got, _reference(q * power, cache, table, [n], [0, new], d ** -0.5 / power), f"{power}", halves=new > 8)


def test_few_pages_of_very_many(cuda_device):
    """One page among 2^27: what the checks of the numbers take goes by the numbers, not by the pages (2^27 bytes cleared take 20 ms)."""
    import time

    from xpu_graph_b200 import ops

    rows = torch.zeros(1 << 27, 16, dtype=torch.uint8, device=cuda_device)
    last = (1 << 27) - 1
    rows[last] = 7
    took = []
    for i in range(5):
        since = time.perf_counter()
        ops.copy_pages(rows, [last, last], [5 + i, 100 + i])
        took.append(time.perf_counter() - since)
    assert (rows[5:10] == 7).all() and (rows[100:105] == 7).all() and not rows[10:100].any() and not rows[:5].any()
    assert min(took) < 2e-3
    for src, dst in (([0, 1], [2, 2]), ([0, 1], [2, 0]), ([1 << 27], [0]), ([0], [-1])):
        with pytest.raises(ValueError):
            ops.copy_pages(rows, src, dst)
