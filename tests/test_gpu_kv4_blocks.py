"""Attention over the 4-bit cache: no block of keys is left out or counted twice, however long the history and however it is cut."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,heads,group,rows,around", [(64, 1, 1, 1, 0), (128, 2, 4, 1, 0), (256, 1, 2, 3, 0), (128, 1, 4, 5, 0), (64, 1, 1, 90, 0), (128, 1, 4, 100, 0),
                                                       (128, 2, 1, 300, 0), (256, 1, 1, 70, 0), (64, 1, 4, 90, 10000), (128, 1, 2, 200, 20000), (256, 1, 1, 70, 20000)])
def test_every_block_of_keys_counts_once(cuda_device, d, heads, group, rows, around, dtype):
    """Queries of zeros average over all keys that they see; channel c of the values is 1 in the c-th block of 64 keys and 0 elsewhere, so
    that each channel shows its own block's share. `around`: rows of no sequence, with which keys stay in one piece."""
    from xpu_graph_b200 import ops

    n, page = 64 * d - 17, 32  # (the last block is no whole one)
    pages = -(-n // page)
    token = torch.arange(pages * page, device=cuda_device)
    v = (token[:, None] // 64 == torch.arange(d, device=cuda_device)).float()[:, None].expand(-1, heads, -1)
    k = torch.randn(len(token), heads, d, generator=torch.Generator(cuda_device).manual_seed(0), device=cuda_device)
    cache = torch.zeros(pages, heads, page // 16, 18 * d, dtype=torch.uint8, device=cuda_device)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    ops.kv4_append(cache, k, v, table[token // page] * page + token % page)
    q = torch.zeros(rows + around, heads * group, d, device=cuda_device, dtype=dtype)
    got = ops.kv4_attention(q, cache, table[None], torch.tensor([n], device=cuda_device), torch.tensor([0, rows], device=cuda_device), rows, 1.0)[:rows].double()
    seen = n - rows + 1 + torch.arange(rows, device=cuda_device)[:, None]
    first = 64 * torch.arange(d, device=cuda_device)[None]
    want = ((seen - first).clamp(0, 64).double() / seen)[:, None]
    # weights times scales, or values, half a step of fp16 off (2^-11): of the share of the groups' ranges that is averaged, at most their
    # middle and a sixteenth; of the share itself; and the result's own rounding. A block that is left out, or twice there, is off by
    # its share, 1 / d.
    tol = 2.0 ** -11 * 0.57 + want * (2.0 ** -10 + torch.finfo(dtype).eps / 2)
    assert tol.max() < 0.2 / d
    bad = (got - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} off, blocks {sorted(set(bad.nonzero()[:, 2].tolist()))[:8]}, rows {sorted(set(bad.nonzero()[:, 0].tolist()))[:8]}"
