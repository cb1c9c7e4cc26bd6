"""Tensor memory and early launches: a kernel lets the next one in only once its own CTA holds its columns, or the next one could take
them and wait for a kernel that waits for it."""
import glob
import os
import re

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xpu_graph_b200", "csrc")
STEP = re.compile(r"ptx::tmem_alloc(?:_pair)?\(|__syncthreads\(\)|pdl_sync\(\)|pdl_trigger\(\)")


def test_columns_are_held_before_the_next_kernel_is_let_in():
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            source = re.sub(r"//[^\n]*", "", f.read())
        steps = [m.group(0) for m in STEP.finditer(source)]
        for i, step in enumerate(steps):
            if step.startswith("ptx::tmem_alloc"):
                seen += 1
                assert steps[i + 1] == "__syncthreads()", f"{os.path.basename(path)}: {steps[i + 1]} behind a tensor-memory allocation, before a barrier"
    assert seen >= 7


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tensor_memory_kernels_behind_one_another(cuda_device, d):
    """Attention over the cache, attention and dense layers in turn on one stream, each placed while the one before drains."""
    from xpu_graph_b200 import lib, ops

    g = torch.Generator(cuda_device).manual_seed(d)
    cache = torch.zeros(40, 2, 2, 18 * d, dtype=torch.uint8, device=cuda_device)
    k = torch.randn(40 * 32, 2, d, generator=g, device=cuda_device)
    ops.kv4_append(cache, k, k, torch.arange(40 * 32, device=cuda_device))
    table, lens = torch.arange(40, device=cuda_device).view(2, 20), torch.tensor([640, 640], device=cuda_device)
    starts = torch.tensor([0, 300, 600], device=cuda_device)
    q = torch.randn(600, 4, d, generator=g, device=cuda_device).bfloat16()
    w = (torch.randn(4 * d, 4 * d, generator=g, device=cuda_device) / (4 * d) ** 0.5).bfloat16()
    heads = q[:512, None].permute(1, 2, 0, 3)[..., :64].contiguous()

    def step():
        a = ops.kv4_attention(q, cache, table, lens, starts, 300, d ** -0.5)
        return a, ops.dense(a.flatten(1), w, True, None, None, "none"), ops.sdpa(heads, heads, heads, None, 0.125, True)

    want = step()
    torch.cuda.synchronize()
    for _ in range(20):
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert lib.tc_status() == 0
