"""xg_sm100::qk_norm_rope against its formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _formula(x, w, cos, sin, positions, sections):
    """Result and the magnitude of what is added for every element, in float64."""
    y = x.double()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
    rot = cos.shape[1]
    half = rot // 2
    pos = positions[None] if positions.dim() == 1 else positions
    axis = [a for a, n in enumerate(sections or [half]) for _ in range(n)]
    c = torch.zeros(x.shape[0], rot, dtype=torch.float64, device=x.device)
    s = torch.zeros_like(c)
    for i in range(rot):
        p = pos[axis[i % half]]
        ok = (p >= 0) & (p < cos.shape[0])
        c[:, i] = torch.where(ok, cos[p.clamp(0, cos.shape[0] - 1), i].double(), 0.0)
        s[:, i] = torch.where(ok, sin[p.clamp(0, cos.shape[0] - 1), i].double(), 0.0)
    c, s = c[:, None], s[:, None]
    a, b = y[..., :half], y[..., half:rot]
    lo, hi = a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:]
    mag = torch.cat(((a * c[..., :half]).abs() + (b * s[..., :half]).abs(), (b * c[..., half:]).abs() + (a * s[..., half:]).abs(), y[..., rot:].abs()), -1)
    return torch.cat((lo, hi, y[..., rot:]), -1), mag


def _check(got, want, what):
    ref, mag = want
    assert got.shape == ref.shape and got.is_contiguous(), what
    # one rounding to the type; before it fp32: the sum of D squares (at most D / lanes + 5 additions a lane, halved by the root),
    # the root, and five products and sums, together below 40 roundings of what is added
    tol = ref.abs() * torch.finfo(got.dtype).eps / 2 + mag * 40 * 2.0 ** -24 + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def _tables(n, rot, dev):
    ang = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1)))
    ang = torch.cat((ang, ang), 1)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


CASES = [  # tokens, q heads, k heads, D, rotated, sections
    (1, 1, 1, 64, 64, []),
    (16, 32, 8, 128, 128, []),
    (513, 4, 4, 64, 32, []),
    (130, 5, 1, 256, 256, [64, 32, 32]),
    (77, 8, 2, 128, 128, [16, 24, 24]),
    (33, 3, 2, 80, 80, [10, 15, 15]),  # sections that end inside a 16-byte piece
    (19, 2, 2, 96, 48, []),
    (21, 3, 1, 18, 6, [1, 2]),  # nothing is a multiple of 16 bytes
    (9, 2, 2, 7, 4, []),
    (40, 2, 0, 64, 64, []),  # queries alone
    (11, 2, 1, 64, 0, []),  # no rotation
    (3000, 12, 3, 128, 64, [8, 0, 24]),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,hq,hk,d,rot,sections", CASES)
def test_formula(cuda_device, tokens, hq, hk, d, rot, sections, dtype):
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(tokens + d)
    qkv = (torch.randn(tokens, hq + 2 * hk, d, generator=g) * 3).to(dtype).to(cuda_device)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype).to(cuda_device) for _ in range(2))
    cos, sin = _tables(200, rot, cuda_device)
    shape = (len(sections), tokens) if sections else (tokens,)
    pos = torch.randint(-3, 210, shape, generator=g).to(cuda_device)
    for a, b, tables in ((wq, wk, (cos, sin)), (None, wk.float(), (cos.to(dtype), sin.to(dtype))), (None, None, (cos, sin))):
        yq, yk = ops.qk_norm_rope(q, k, a, b, EPS, *tables, pos, sections)
        _check(yq, _formula(q, a, *tables, pos, sections), "q")
        _check(yk, _formula(k, b, *tables, pos, sections), "k")


def test_strides(cuda_device):
    """Heads before tokens, channels that are not contiguous, rows off the 16-byte grid, strided positions."""
    from xpu_graph_b200 import ops

    g = torch.Generator().manual_seed(5)
    cos, sin = _tables(64, 64, cuda_device)
    w = torch.randn(64, generator=g).to(cuda_device)
    base = torch.randn(4, 30, 64, generator=g).to(cuda_device)
    odd = torch.randn(30, 4 * 64 + 3, generator=g).to(cuda_device)[:, 3:].unflatten(1, (4, 64))
    pos = torch.randint(0, 64, (2, 60), generator=g).to(cuda_device)[:, ::2]
    for x in (base.transpose(0, 1), base.transpose(0, 1).contiguous().transpose(1, 2).contiguous().transpose(1, 2), odd):
        yq, yk = ops.qk_norm_rope(x, x[:, :2], w, w, EPS, cos, sin, pos, [20, 12])
        _check(yq, _formula(x, w, cos, sin, pos, [20, 12]), "q")
        _check(yk, _formula(x[:, :2], w, cos, sin, pos, [20, 12]), "k")


def test_no_tokens_and_refusals(cuda_device):
    from xpu_graph_b200 import ops

    q = torch.zeros(4, 2, 64, device=cuda_device)
    cos, sin = _tables(8, 64, cuda_device)
    pos = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    yq, yk = ops.qk_norm_rope(q[:0], q[:0], None, None, EPS, cos, sin, pos[:0], [])
    assert yq.shape == (0, 2, 64) and yk.shape == (0, 2, 64)

    def refused(error, *args):
        with pytest.raises(error):
            ops.qk_norm_rope(*args)

    refused(ValueError, q, q[:3], None, None, EPS, cos, sin, pos, [])
    refused(ValueError, q, q.half(), None, None, EPS, cos, sin, pos, [])
    refused(ValueError, q, q, cos[0, :3], None, EPS, cos, sin, pos, [])
    refused(ValueError, q, q, None, None, EPS, cos, sin[:4], pos, [])
    refused(ValueError, q[..., :32], q[..., :32], None, None, EPS, cos, sin, pos, [])
    refused(ValueError, q, q, None, None, EPS, cos, sin, pos[:3], [])
    refused(TypeError, q, q, None, None, EPS, cos, sin, pos.int(), [])
    refused(ValueError, q, q, None, None, EPS, cos, sin, pos, [16, 16])
    refused(ValueError, q, q, None, None, EPS, cos, sin, pos.expand(2, 4), [16, 15])
    refused(ValueError, q, q, None, None, EPS, cos, sin, pos.expand(2, 4), [40, -8])
    refused(ValueError, q, q, None, None, EPS, cos.cpu(), sin, pos, [])
    refused(TypeError, q.double(), q.double(), None, None, EPS, cos, sin, pos, [])


def test_backward_is_refused(cuda_device):
    from xpu_graph_b200 import ops

    q = torch.randn(4, 2, 64, device=cuda_device, requires_grad=True)
    cos, sin = _tables(8, 64, cuda_device)
    pos = torch.zeros(4, dtype=torch.int64, device=cuda_device)
    y = ops.qk_norm_rope(q, q.detach(), None, None, EPS, cos, sin, pos, [])[0]
    with pytest.raises(RuntimeError):
        y.sum().backward()
