"""The 4-bit cache at the ends of what it holds: constants that fp16 rounds up."""
import pytest
import torch

from tests.test_gpu_kv4 import _check_attention, _filled, _reference

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
