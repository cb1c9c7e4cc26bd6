"""The 4-bit cache: kv4_append and kv4_read against the written-down quantisation bit for bit, kv4_attention against a softmax in 64
bits over the values that are read back, copy_pages."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _quantised(x):
    """Values, codes, scales and least values of [..., d], step by step as they are defined, in fp32 on the CPU."""
    y = x.detach().cpu().float().clamp(-65504.0, 65504.0).unflatten(-1, (-1, 64))
    least = y.amin(-1).half()  # (amin keeps NaN)
    scale = ((y.amax(-1) - least.float()) * torch.tensor(1 / 15)).half()
    code = ((y - least.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15)
    code = torch.where(scale[..., None] > 0, code, torch.zeros(()))
    return (code * scale.float()[..., None] + least.float()[..., None]).flatten(-2).to(x.dtype), code.flatten(-2), scale, least


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30))


def _new_cache(pages, heads, page, d, dev):
    g = torch.Generator(dev).manual_seed(pages)
    return torch.randint(0, 256, (pages, heads, page // 16, 18 * d), generator=g, device=dev, dtype=torch.uint8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,d,page", [(1, 1, 64, 16), (37, 3, 128, 32), (200, 2, 256, 64), (1000, 8, 128, 16), (5, 5, 64, 128)])
def test_append_and_read(cuda_device, tokens, heads, d, page, dtype):
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(tokens)
    pages = tokens // page + 4
    cache = _new_cache(pages, heads, page, d, cuda_device)
    before = cache.clone()
    packed = torch.randn(tokens, 3 * heads, d, generator=g) * torch.tensor([1e-3, 1.0, 300.0])[torch.randint(0, 3, (tokens, 3 * heads, 1), generator=g)]
    packed = packed.to(dtype).to(cuda_device)
    k, v = packed[:, heads:2 * heads], packed[:, 2 * heads:]
    slots = torch.randperm(pages * page, generator=g)[:tokens].to(cuda_device)
    assert ops.kv4_append(cache, k, v, slots) is None
    rk, rv = ops.kv4_read(cache, slots, dtype)
    assert _same(rk.cpu(), _quantised(k)[0]) and _same(rv.cpu(), _quantised(v)[0])
    # every other token is what it was
    rest = torch.tensor(sorted(set(range(pages * page)) - set(slots.tolist())), device=cuda_device)
    for a, b in zip(ops.kv4_read(cache, rest, torch.float32), ops.kv4_read(before, rest, torch.float32)):
        assert _same(a, b)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_places_in_a_tile(cuda_device, d):
    """The bytes lie where kv4_tile.cuh says."""
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(d)
    k, v = (torch.randn(32, 2, d, generator=g) for _ in range(2))
    cache = torch.zeros(3, 2, 1, 18 * d, dtype=torch.uint8, device=cuda_device)
    ops.kv4_append(cache, k.to(cuda_device), v.to(cuda_device), torch.arange(16, 48, device=cuda_device))
    raw = cache.cpu()
    assert not raw[0].any()
    for x, value in ((k, 0), (v, 1)):
        _, code, scale, least = _quantised(x)
        for token in range(32):
            r, t, c = token % 16, (token >> 1) & 3, (token & 1) + 2 * (token % 16 >> 3)
            for h in range(2):
                tile = raw[1 + token // 16, h, 0]
                pairs = tile[(16 + value) * d + r * (d // 16):][:d // 16].view(torch.float16).view(-1, 2)
                assert torch.equal(pairs[:, 0], scale[token, h]) and torch.equal(pairs[:, 1], least[token, h])
                for j in range(d // 8):
                    at = 8 * d + (4 * c + t) * (d // 2) + ((j % 8 ^ 2 * t) * (d // 64) + j // 8) * 4 if value else r * (d // 2) + (j % 4 * (d // 32) + j // 4) * 4
                    word = int.from_bytes(bytes(tile[at:at + 4].tolist()), "little")
                    assert [word >> 4 * i & 15 for i in range(8)] == code[token, h, 8 * j:8 * j + 8].int().tolist()


def test_values_out_of_the_ordinary(cuda_device):
    from xpu_graph_b200 import ops

    k = torch.randn(8, 1, 128)
    k[0, 0, :64] = 3.25  # a constant group
    k[1, 0, 5] = math.inf
    k[2, 0, 100] = -math.inf
    k[3, 0, 70] = math.nan
    k[4] = 0.0
    k[5] *= 1e-9  # a range below fp16's smallest
    k[6] *= 1e30
    k[7] = 100.0 + 0.001 * torch.randn(128)  # a range far below the values
    cache = torch.zeros(1, 1, 1, 18 * 128, dtype=torch.uint8, device=cuda_device)
    slots = torch.arange(8, device=cuda_device)
    for dtype in (torch.float32, torch.bfloat16):
        x = k.to(dtype).to(cuda_device)
        ops.kv4_append(cache, x, x.flip(0), slots)
        rk, rv = ops.kv4_read(cache, slots, dtype)
        want = _quantised(x)[0]
        assert _same(rk.cpu(), want) and _same(rv.cpu(), want.flip(0))
        assert torch.isnan(rk[3, 0, 64:]).all() and torch.isfinite(rk[3, 0, :64]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_skips_and_strides(cuda_device, dtype):
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(2)
    whole = _new_cache(12, 2, 16, 64, cuda_device).view(6, 2, 2, 1, 18 * 64)
    cache = whole[:, 1]  # pages of one layer, a page of another between them
    before = whole.clone()
    odd = torch.randn(6, 2 * 64 + 1, generator=g).to(dtype).to(cuda_device)[:, 1:].unflatten(1, (2, 64))
    heads_first = torch.randn(2, 6, 64, generator=g).to(dtype).to(cuda_device).transpose(0, 1)
    slots = torch.tensor([-1, 0, 95, 96, -(1 << 62), 17], device=cuda_device)
    wide = torch.stack((slots, slots), 1)
    ops.kv4_append(cache, odd, heads_first, wide[:, 0])
    rk, rv = ops.kv4_read(cache, slots, dtype)
    there = torch.tensor([False, True, True, False, False, True])
    for r, x in ((rk, odd), (rv, heads_first)):
        assert _same(r.cpu()[there], _quantised(x)[0][there]) and not r.cpu()[~there].any()
    assert torch.equal(whole[:, 0], before[:, 0])
    ops.kv4_append(cache, odd[:0], odd[:0], slots[:0])
    assert ops.kv4_read(cache, slots[:0], dtype)[0].shape == (0, 2, 64)
    assert not ops.kv4_read(cache[:0], slots, dtype)[0].any()


def test_cache_beyond_4_gib(cuda_device):
    from xpu_graph_b200 import ops

    pages = (1 << 32) // (8 * 4 * 18 * 128) + 9
    cache = torch.empty(pages, 8, 4, 18 * 128, dtype=torch.uint8, device=cuda_device)
    k = torch.randn(3, 8, 128, device=cuda_device)
    slots = torch.tensor([pages * 64 - 1, 5, pages * 64 - 64], device=cuda_device)
    cache[-1].zero_(), cache[0].zero_()
    ops.kv4_append(cache, k, k, slots)
    assert _same(ops.kv4_read(cache, slots, torch.float32)[0].cpu(), _quantised(k)[0])
    q = torch.randn(1, 8, 128, device=cuda_device).half()
    args = (torch.tensor([64], device=cuda_device), None, 1, 0.1)
    got = ops.kv4_attention(q, cache, torch.tensor([[pages - 1]], device=cuda_device), *args)
    assert torch.equal(got, ops.kv4_attention(q, cache[-1:].clone(), torch.tensor([[0]], device=cuda_device), *args))
    ops.copy_pages(cache, [pages - 1], [pages - 2])
    assert torch.equal(cache[-1], cache[-2])


# ---- attention -------------------------------------------------------------------------------------
def _filled(pages, heads, page, d, dev, seed=0, scale=1.0):
    from xpu_graph_b200 import ops

    g = torch.Generator(dev).manual_seed(seed)
    cache = torch.zeros(pages, heads, page // 16, 18 * d, dtype=torch.uint8, device=dev)
    k = torch.randn(pages * page, heads, d, generator=g, device=dev) * scale
    v = torch.randn(pages * page, heads, d, generator=g, device=dev) + torch.randn(1, heads, d, generator=g, device=dev)
    ops.kv4_append(cache, k, v, torch.arange(pages * page, device=dev))
    return cache


def _reference(q, cache, table, lens, starts, scale):
    """(out, tolerance without the final rounding's share): softmax in 64 bits over the values of the cache."""
    from xpu_graph_b200 import ops

    page, heads, d = 16 * cache.shape[2], cache.shape[1], cache.shape[3] // 18
    out, err_k, err_v = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(3))
    starts = list(range(len(lens) + 1)) if starts is None else starts
    group = q.shape[1] // heads
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        j = torch.arange(n, device=q.device)
        if n == 0 or hi == lo:
            continue
        ids = table[b, j // page]
        there = (ids >= 0) & (ids < cache.shape[0])
        k, v = (x.double().nan_to_num(0.0) for x in ops.kv4_read(cache, torch.where(there, ids * page + j % page, -1), torch.float32))
        k, v = (x.repeat_interleave(group, 1) for x in (k, v))
        qb = q[lo:hi].double()
        score = torch.einsum("ihd,jhd->hij", qb, k) * scale
        seen = there[None] & (j[None] <= (torch.arange(hi - lo, device=q.device) + n - (hi - lo))[:, None])
        score = score.masked_fill(~seen[None], -math.inf)
        p = torch.softmax(score, -1).nan_to_num(0.0)
        out[lo:hi] = torch.einsum("hij,jhd->ihd", p, v)
        size = torch.einsum("ihd,jhd->hij", qb.abs(), k.abs()).masked_fill(~seen[None], 0.0).amax(-1) * abs(scale)  # of the largest score's terms
        sums = torch.einsum("hij,jhd->ihd", p, v.abs())
        err_k[lo:hi] = sums * size.transpose(0, 1)[..., None]
        groups = v.unflatten(-1, (-1, 64))
        half_range = ((groups.amax(-1) - groups.amin(-1)) / 2)[..., None].expand_as(groups).flatten(-2)
        err_v[lo:hi] = sums + torch.einsum("hij,jhd->ihd", p, half_range)
    return out, err_k, err_v


def _check_attention(got, ref, what, halves=False):
    """Scores: fp32 sums of D products, the terms' size times 2^-20 at most (16 roundings of 2^-24: the tensor core's partial sums).
    They move a probability by a factor of e^(2 error). The probability times its value's scale goes into the second product as fp16,
    half a step of 2^-11 off, after the exponential (2^-20) and two fp32 products: that moves the value's distance from the middle of
    its group's range, at most half the range (8/7.5 of it, as the middle is taken at code 8). What is exact beside it is an fp32 sum.
    `halves`: keys and values in fp16 too (2^-11 each of the value)."""
    out, err_k, err_v = ref
    assert got.shape == out.shape
    u_k, u_v = (2.0 ** -11 + 2.0 ** -20, 2 * 2.0 ** -11 + 2.0 ** -19) if halves else (2.0 ** -20, 2.0 ** -11 * 8 / 7.5 + 2.0 ** -19)
    tol = out.abs() * torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -6) + 2 * u_k * err_k * (1 + 8 * u_k * err_k) + u_v * err_v + 1e-7
    bad = ~((got.double() - out).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, rows {sorted(set(bad.nonzero()[:, 0].tolist()))[:8]}"


def _table(lens, page, pages, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    most = max(1, max(-(-n // page) for n in lens))
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), most), -1, dtype=torch.int64)
    used = 0
    for b, n in enumerate(lens):
        count = -(-n // page)
        table[b, :count] = order[used:used + count]
        used += count
    assert used <= pages
    return table.to(dev)


ATTEND = [  # d, kv heads, group, page, lens, new tokens (None: one each, without starts)
    (64, 1, 1, 16, [1], None),
    (128, 2, 4, 16, [1, 15, 16, 17, 0, 100], None),
    (128, 8, 1, 64, [333], None),
    (256, 1, 3, 32, [70, 31, 32, 33], None),
    (64, 4, 8, 128, [1000, 1, 129, 128, 127], None),
    (128, 1, 16, 16, [200, 17], None),  # more query heads than one pass takes
    (128, 4, 5, 32, [5000, 3, 700], None),
    (128, 2, 4, 16, [20, 9, 0, 40, 64], [5, 3, 0, 1, 8]),
    (64, 2, 4, 32, [300, 7, 31], [7, 7, 2]),  # a sequence that is all new
    (256, 2, 1, 16, [90, 40], [4, 6]),
    (128, 1, 1, 16, [2, 3], [4, 5]),  # more rows than tokens: the first ones see nothing
    (128, 3, 2, 64, [9000, 8999], None),
    # many new tokens, alone and beside few
    (128, 2, 4, 16, [300, 100, 17, 0, 64, 70], [100, 40, 17, 0, 3, 64]),
    (64, 1, 1, 64, [513, 130], [513, 129]),
    (128, 1, 8, 32, [1500], [300]),
    (128, 4, 3, 16, [257, 77, 500], [86, 77, 85]),
    (64, 2, 5, 128, [3000, 64], [40, 64]),
    (128, 1, 4, 64, [6000, 700, 90], [100, 90, 80]),  # few rows, many keys
    (64, 2, 1, 32, [2500], [200]),
    (128, 1, 1, 16, [70, 0, 100], [90, 66, 130]),
    (256, 1, 2, 32, [150], [150]),
    (256, 2, 3, 64, [2000, 70, 300], [40, 2, 90]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,heads,group,page,lens,new", ATTEND)
def test_attention(cuda_device, d, heads, group, page, lens, new, dtype):
    from xpu_graph_b200 import lib, ops

    pages = sum(-(-n // page) for n in lens) + 3
    cache = _filled(pages, heads, page, d, cuda_device)
    table = _table(lens, page, pages, cuda_device)
    starts = None if new is None else [sum(new[:i]) for i in range(len(new) + 1)]
    g = torch.Generator().manual_seed(d + len(lens))
    tokens = len(lens) if new is None else starts[-1] + 2  # two rows of no sequence behind the last one
    q = (torch.randn(tokens, heads * group + 1, d, generator=g) * 1.5).to(dtype).to(cuda_device)[:, 1:]  # a slice of a wider tensor
    at = None if starts is None else torch.tensor(starts, device=cuda_device)
    got = ops.kv4_attention(q, cache, table, torch.tensor(lens, device=cuda_device), at, max(new or [1]), d ** -0.5)
    assert got.dtype == dtype and got.is_contiguous()
    _check_attention(got, _reference(q, cache, table, lens, starts, d ** -0.5), "attention", halves=max(new or [1]) > 8)
    if starts is not None:
        assert not got[starts[-1]:].any()
    assert lib.tc_status() == 0


def test_attention_sharp_and_flat(cuda_device):
    """Scores of hundreds, scores that are all alike, a negative and a zero scale."""
    from xpu_graph_b200 import ops

    lens = [700, 64]
    cache = _filled(12, 2, 64, 128, cuda_device, scale=6.0)
    table, n = _table(lens, 64, 12, cuda_device), torch.tensor(lens, device=cuda_device)
    q = torch.randn(2, 8, 128, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    for scale in (3.0, 0.0, -0.2, 1e-3):
        got = ops.kv4_attention(q, cache, table, n, None, 1, scale)
        _check_attention(got, _reference(q, cache, table, lens, None, scale), f"scale {scale}")


def test_attention_leaves_alone_what_is_not_there(cuda_device):
    """Tokens behind a sequence's end hold NaN, page numbers outside the cache hide their keys, a table wider than needed."""
    from xpu_graph_b200 import ops

    lens = [40, 18, 100, 33]
    cache = _filled(16, 2, 32, 128, cuda_device)
    table = torch.full((4, 9), 1 << 40, dtype=torch.int64, device=cuda_device)
    table[:, :4] = _table([128] * 4, 32, 16, cuda_device)
    nan = torch.full((128, 2, 128), math.nan, device=cuda_device)
    for b, n in enumerate(lens):
        j = torch.arange(n, 128, device=cuda_device)
        ops.kv4_append(cache, nan[:len(j)], nan[:len(j)], table[b, j // 32] * 32 + j % 32)
    table[2, 1] = -1
    table[3, 0] = 16
    q = torch.randn(4, 4, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device)
    n = torch.tensor(lens, device=cuda_device)
    got = ops.kv4_attention(q, cache, table, n, None, 1, 0.1)
    assert torch.isfinite(got).all()
    _check_attention(got, _reference(q, cache, table, lens, None, 0.1), "holes")
    table[1, :] = -5
    assert not ops.kv4_attention(q, cache, table, n, None, 1, 0.1)[1].any()
    # a length beyond the table's pages counts as the table's end
    wide = torch.tensor([40, 18, 100, 64], device=cuda_device)
    a = ops.kv4_attention(q, cache, table[:, :2], wide * 1000, None, 1, 0.1)
    assert _same(a, ops.kv4_attention(q, cache, table[:, :2], torch.full_like(wide, 64), None, 1, 0.1))
    # nothing cached at all
    assert not ops.kv4_attention(q, cache, table[:, :0], n, None, 1, 0.1).any()
    assert not ops.kv4_attention(q, cache[:0], table, n, None, 1, 0.1).any()
    assert ops.kv4_attention(q[:0], cache, table[:0], n[:0], None, 1, 0.1).shape == (0, 4, 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_of_many_new_tokens(cuda_device, dtype):
    """Holes, NaN behind the end, scores of hundreds, a negative and a zero scale, rows of q of any size and alignment."""
    from xpu_graph_b200 import lib, ops

    lens, starts = [333, 200], [0, 200, 350]
    cache = _filled(20, 2, 32, 128, cuda_device, scale=3.0)
    table = torch.cat((_table([352, 224], 32, 20, cuda_device), torch.full((2, 3), -7, device=cuda_device)), 1)
    nan = torch.full((32, 2, 128), math.nan, device=cuda_device)
    for b, n in enumerate(lens):
        j = torch.arange(n, -(-n // 32) * 32, device=cuda_device)
        ops.kv4_append(cache, nan[:len(j)], nan[:len(j)], table[b, j // 32] * 32 + j % 32)
    table[0, 3] = 20
    table[0, 10 - 1] = -1
    table[1, 0] = 1 << 33
    g = torch.Generator().manual_seed(1)
    q = torch.randn(350, 6 * 128 + 3, generator=g).to(dtype)[:, 3:].unflatten(1, (6, 128)).to(cuda_device)
    q = q * torch.tensor([1e-3, 1.0, 100.0]).to(dtype).to(cuda_device)[torch.arange(350, device=cuda_device) % 3][:, None, None]
    q[5] = 0
    n, at = torch.tensor(lens, device=cuda_device), torch.tensor(starts, device=cuda_device)
    for scale in (0.08, -0.05, 0.0):
        got = ops.kv4_attention(q, cache, table, n, at, 200, scale)
        assert torch.isfinite(got).all()
        _check_attention(got, _reference(q, cache, table, lens, starts, scale), f"scale {scale}", halves=True)
        assert torch.equal(got, ops.kv4_attention(q, cache, table, n, at, 200, scale))
    assert lib.tc_status() == 0


def test_attention_is_repeatable_and_any_hint_will_do(cuda_device):
    from xpu_graph_b200 import ops

    lens, starts = [900, 33, 5], [0, 3, 4, 6]
    cache = _filled(40, 2, 32, 128, cuda_device)
    table, n, at = _table(lens, 32, 40, cuda_device), torch.tensor(lens, device=cuda_device), torch.tensor(starts, device=cuda_device)
    q = torch.randn(6, 8, 128, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    one = ops.kv4_attention(q, cache, table, n, at, 3, 0.1)
    assert torch.equal(one, ops.kv4_attention(q, cache, table, n, at, 3, 0.1))
    for hint in (0, 1, 100000):
        _check_attention(ops.kv4_attention(q, cache, table, n, at, hint, 0.1), _reference(q, cache, table, lens, starts, 0.1), f"hint {hint}", halves=hint > 8)


def test_a_flat_average_over_a_long_history(cuda_device):
    """131072 keys of equal weight: the average is 1 / 360 of the values, where a bias of the sums would show."""
    from xpu_graph_b200 import ops

    n, g = 131072, torch.Generator(cuda_device).manual_seed(0)
    cache = torch.zeros(n // 64, 1, 4, 18 * 128, dtype=torch.uint8, device=cuda_device)
    v = torch.randn(n, 1, 128, generator=g, device=cuda_device)
    ops.kv4_append(cache, v, v, torch.arange(n, device=cuda_device))
    want = ops.kv4_read(cache, torch.arange(n, device=cuda_device), torch.float32)[1].double().mean(0)
    table = torch.arange(n // 64, device=cuda_device)[None]
    for rows in (1, 60):
        q = torch.zeros(rows, 1, 128, device=cuda_device).half()
        got = ops.kv4_attention(q, cache, table, torch.tensor([n + rows - 1], device=cuda_device).clamp(max=n), torch.tensor([0, rows], device=cuda_device), rows, 1.0)[-1]
        # independent roundings of 2^-11 at most of values of 1 around a mean of 0, over 360: below 2^-11 of the mean's size, twice for
        # keys in fp16; the result's own 2^-11; sums of 128 keys in fp32 with 2^-24 of up to 15 a step: below 2^-9 together
        assert ((got.double() - want).norm() / want.norm()).item() < 2.0 ** -9


# ---- pages -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("pages,shape,pairs", [(7, (2, 1, 18 * 64), 2), (1200, (1, 1, 18 * 64), 500), (64, (8, 4, 18 * 128), 30), (9, (16,), 4)])
def test_copy_pages(cuda_device, pages, shape, pairs):
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(pages)
    cache = torch.randint(0, 256, (pages, *shape), generator=g, dtype=torch.uint8).to(cuda_device)
    order = torch.randperm(pages, generator=g).tolist()
    src, dst = order[:pairs - 1] + order[:1], order[pairs:2 * pairs]  # one page goes to two places
    want = cache.clone()
    want[dst] = want[src]
    ops.copy_pages(cache, src, dst)
    assert torch.equal(cache, want)
    ops.copy_pages(cache, [], [])
    assert torch.equal(cache, want)


def test_copy_pages_of_one_layer_and_other_types(cuda_device):
    from xpu_graph_b200 import ops

    whole = torch.randn(10, 3, 40, 4, device=cuda_device)
    want = whole.clone()
    want[[7, 8], 1] = want[[2, 2], 1]
    ops.copy_pages(whole[:, 1], [2, 2], [7, 8])
    assert torch.equal(whole, want)


def test_refusals(cuda_device):
    from xpu_graph_b200 import lib, ops

    dev = cuda_device
    cache = torch.zeros(4, 2, 2, 18 * 64, dtype=torch.uint8, device=dev)
    x, slots = torch.zeros(3, 2, 64, device=dev), torch.arange(3, device=dev)

    def refused(error, op, *args):
        with pytest.raises(error):
            op(*args)

    refused(TypeError, ops.kv4_append, cache.int(), x, x, slots)
    refused(ValueError, ops.kv4_append, cache[0], x, x, slots)
    refused(ValueError, ops.kv4_append, cache.transpose(1, 2), x, x, slots)
    refused(ValueError, ops.kv4_append, cache, x[:, :1], x[:, :1], slots)
    refused(ValueError, ops.kv4_append, cache, x, x[:2], slots)
    refused(ValueError, ops.kv4_append, cache, x, x.half(), slots)
    refused(TypeError, ops.kv4_append, cache, x.double(), x.double(), slots)
    refused(TypeError, ops.kv4_append, cache, x, x, slots.int())
    refused(ValueError, ops.kv4_append, cache, x, x, slots[:2])
    refused(ValueError, ops.kv4_append, cache, x, x, slots.cpu())
    refused(lib.XgLibraryError, ops.kv4_append, torch.zeros(4, 2, 2, 18 * 96, dtype=torch.uint8, device=dev), torch.zeros(3, 2, 96, device=dev),
            torch.zeros(3, 2, 96, device=dev), slots)
    refused(TypeError, ops.kv4_read, cache, slots, torch.int32)
    refused(ValueError, ops.kv4_read, cache, slots[None], torch.float32)
    q, table, lens = torch.zeros(2, 4, 64, device=dev).half(), torch.zeros(2, 3, dtype=torch.int64, device=dev), torch.ones(2, dtype=torch.int64, device=dev)
    refused(lib.XgLibraryError, ops.kv4_attention, q.float(), cache, table, lens, None, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q[:, :3], cache, table, lens, None, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q[..., :32], cache, table, lens, None, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q, cache, table[:1], lens, None, 1, 1.0)
    refused(TypeError, ops.kv4_attention, q, cache, table.int(), lens, None, 1, 1.0)
    refused(TypeError, ops.kv4_attention, q, cache, table, lens.int(), None, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q[:1], cache, table, lens, None, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q, cache, table, lens, lens, 1, 1.0)
    refused(ValueError, ops.kv4_attention, q, cache, table, lens, None, -1, 1.0)
    refused(ValueError, ops.kv4_attention, q, cache, table.cpu(), lens, None, 1, 1.0)
    refused(ValueError, ops.copy_pages, cache, [0, 1], [2])
    refused(ValueError, ops.copy_pages, cache, [0, 1], [2, 2])
    refused(ValueError, ops.copy_pages, cache, [0, 1], [2, 0])
    refused(ValueError, ops.copy_pages, cache, [1], [1])
    refused(ValueError, ops.copy_pages, cache, [4], [0])
    refused(ValueError, ops.copy_pages, cache, [0], [-1])
    refused(ValueError, ops.copy_pages, cache, slots[:1], slots[1:2])
    refused(TypeError, ops.copy_pages, cache, torch.zeros(1), torch.ones(1))
    refused(lib.XgLibraryError, ops.copy_pages, torch.zeros(4, 3, dtype=torch.uint8, device=dev), [0], [1])
    assert not cache.any()


# ---- together ----------------------------------------------------------------------------------------
def _step(x, weights, cache, table, lens, starts, max_q, slots, positions, tables, heads, kv_heads, d):
    from xpu_graph_b200 import modules, ops

    w_qkv, w_o, wq, wk = weights
    qkv = ops.dense(x, w_qkv, True, None, None, "none").view(len(x), heads + 2 * kv_heads, d)
    q, k = modules.QKNormRopeModule()(qkv[:, :heads], qkv[:, heads:heads + kv_heads], wq, wk, 1e-6, *tables, positions)
    a = modules.CachedAttentionModule()(q, k, qkv[:, heads + kv_heads:], cache, slots, table, lens, starts, max_q)
    return ops.dense(a.flatten(1), w_o, True, None, None, "none")


def test_serving_steps(cuda_device):
    """A prompt in two chunks and decoding steps, the steps also as a replayed CUDA graph with a padding row and on another stream:
    the results of the same tokens are the same however they came in, within what a different split of the sums moves."""
    from xpu_graph_b200 import ops

    heads, kv_heads, d, page, hidden = 8, 2, 128, 16, 256
    g = torch.Generator().manual_seed(3)
    dev = cuda_device
    weights = [(torch.randn(n, m, generator=g) / math.sqrt(m)).bfloat16().to(dev) for n, m in (((heads + 2 * kv_heads) * d, hidden), (hidden, heads * d))]
    weights += [(1 + 0.1 * torch.randn(d, generator=g)).bfloat16().to(dev) for _ in range(2)]
    ang = torch.outer(torch.arange(128.0), 10000.0 ** (-torch.arange(0, d, 2.0) / d)).repeat(1, 2)
    tables = (ang.cos().to(dev), ang.sin().to(dev))
    x = torch.randn(60, hidden, generator=g).bfloat16().to(dev)
    table = torch.tensor([[3, 0, 5, 2], [0, 0, 0, 0]], device=dev)
    row = torch.tensor([3, 0, 5, 2], device=dev)
    cache = torch.zeros(6, kv_heads, page // 16, 18 * d, dtype=torch.uint8, device=dev)
    i = torch.arange(60, device=dev)
    slots = row[i // page] * page + i % page

    def chunk(lo, hi):
        return _step(x[lo:hi], weights, cache, table[:1], torch.tensor([hi], device=dev), torch.tensor([0, hi - lo], device=dev), hi - lo, slots[lo:hi], i[lo:hi],
                     tables, heads, kv_heads, d)

    want = torch.cat((chunk(0, 37), chunk(37, 60)))
    filled = cache.clone()
    # one token at a time from the 50th, beside a padding row, captured once
    state = {"x": torch.zeros(2, hidden, device=dev).bfloat16(), "lens": torch.zeros(2, dtype=torch.int64, device=dev),
             "slots": torch.full((2,), -1, device=dev), "pos": torch.zeros(2, dtype=torch.int64, device=dev)}

    def decode():
        return _step(state["x"], weights, cache, table, state["lens"], None, 1, state["slots"], state["pos"], tables, heads, kv_heads, d)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = decode()
    ops.kv4_append(cache, torch.zeros(10, kv_heads, d, device=dev), torch.zeros(10, kv_heads, d, device=dev), slots[50:])
    got = want.clone()
    for n in range(50, 60):
        state["x"][0], state["lens"][0], state["slots"][0], state["pos"][0] = x[n], n + 1, slots[n], n
        if n % 2:
            graph.replay()
            got[n] = out[0]
        else:
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                got[n] = decode()[0]
            torch.cuda.current_stream().wait_stream(side)
        assert not out[1].any()
    # the projections of 1, 23 and 37 rows may split their sums differently: a bf16 step of q, k, v, of an activation and of the output
    # each, and a code of the cache may fall to its neighbour (a step of a 15th of the range, on single channels)
    assert ((got.float() - want.float()).norm() / want.float().norm()).item() < 0.03
    k, f = (ops.kv4_read(c, slots, torch.float32)[0] for c in (cache, filled))
    assert ((k - f).norm() / f.norm()).item() < 0.03


def test_sequences_that_fork_and_move(cuda_device):
    """KV4Cache with the operators: forks that go on apart, frees and a compaction leave every sequence's attention as it is."""
    from xpu_graph_b200 import ops
    from xpu_graph_b200.kv_cache import KV4Cache

    dev, heads, d = cuda_device, 2, 64
    cache = KV4Cache(40, heads, d, page_size=32, device=dev)
    g = torch.Generator(dev).manual_seed(0)

    def grow(seq, n):
        k, v = (torch.randn(n, heads, d, generator=g, device=dev) for _ in range(2))
        ops.kv4_append(cache.layers[0], k, v, cache.extend(seq, n))

    seqs = [cache.new() for _ in range(3)]
    for seq, n in zip(seqs, (100, 64, 7)):
        grow(seq, n)
    seqs += [cache.fork(seqs[0]), cache.fork(seqs[1]), cache.fork(seqs[2])]
    for i, seq in enumerate(seqs):
        grow(seq, 3 + i)
    q = torch.randn(len(seqs), 4, d, generator=g, device=dev).bfloat16()

    def attend(which):
        table, lens = cache.tables([seqs[i] for i in which])
        return ops.kv4_attention(q[which], cache.layers[0], table, lens, None, 1, d ** -0.5)

    before = attend([0, 1, 2, 3, 4, 5])
    assert not torch.equal(before[0], before[3])
    cache.free(seqs[1])
    cache.free(seqs[0])
    assert cache.compact() + cache.free_pages == 40
    # (other sequences beside it, other cuts: roundings of fp16 times half a range of 3, and a bf16 step)
    after = attend([2, 3, 4, 5]).float()
    assert ((after - before[2:].float()).abs() <= 2.0 ** -11 * 6 + 2.0 ** -7 * after.abs()).all()


def test_operators_compile(cuda_device):
    """The operators inside a torch.compile graph, the mutation of the cache among them."""
    from xpu_graph_b200 import ops  # noqa: F401

    cache = torch.zeros(2, 1, 1, 18 * 64, dtype=torch.uint8, device=cuda_device)
    k, slots = torch.randn(4, 1, 64, device=cuda_device), torch.arange(4, device=cuda_device)
    q, lens = torch.randn(1, 2, 64, device=cuda_device).half(), torch.tensor([4], device=cuda_device)

    def f(cache, k, slots, q, lens, pages):
        torch.ops.xg_sm100.kv4_append(cache, k, k, slots)
        torch.ops.xg_sm100.copy_pages(cache, pages[:1], pages[1:])
        return torch.ops.xg_sm100.kv4_attention(q, cache, slots[1:2, None], lens, None, 1, 0.125) * 2, torch.ops.xg_sm100.kv4_read(cache, slots, torch.float32)[0]

    pages = torch.arange(2)
    other = cache.clone()
    want = f(cache, k, slots, q, lens, pages)
    got = torch.compile(f, backend="aot_eager")(other, k, slots, q, lens, pages)
    assert torch.equal(cache, other) and all(torch.equal(a, b) for a, b in zip(got, want))
