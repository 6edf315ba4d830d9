"""Grouped int4 products of very small and very large columns, to the same bounds as those of ordinary ones (test_gpu_kv4.py)."""
import pytest
import torch

from test_gpu_kv4 import U, gen, rounded, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols,x_type", [(1, torch.float32), (3, torch.float32), (8, torch.float32), (2, torch.bfloat16), (8, torch.bfloat16)])
@pytest.mark.parametrize("size", [1e-35, 1e-33, 1e-30, 1e-20, 1e20, 1e34])
@pytest.mark.parametrize("offset", [False, True])
def test_columns_of_every_size(pkg, cols, x_type, size, offset):
    n, k, group, g = 96, 1344, 64, gen(cols)
    q = torch.randint(-8, 8, (n, k), device="cuda", generator=g)
    scale = (0.02 * torch.rand(n, k // group, device="cuda", generator=g) + 1e-3).half()
    off = (0.05 * torch.randn(n, k // group, device="cuda", generator=g)).half() if offset else None
    nib = (q & 15).to(torch.uint8).cpu().numpy()
    raw = lambda t: None if t is None else t.view(torch.int16).cpu().numpy()          # noqa: E731
    img = torch.from_numpy(pkg.ops.repack_w4_grouped(nib[:, 0::2] | nib[:, 1::2] << 4, raw(scale), raw(off), group)).cuda()
    x = (size * torch.randn(cols, k, device="cuda", generator=g, dtype=torch.float64)).to(x_type)
    y = torch.empty(cols, n, device="cuda")
    pkg.ops.gemv_w4_grouped(img.data_ptr(), x.data_ptr(), y.data_ptr(), n, k, group, ncols=cols, x_type=0 if x_type == torch.float32 else 1, has_offset=offset, stream=stream())
    rows = x.double()
    w = q.double() * scale.double().repeat_interleave(group, 1)
    weight = w.abs()
    if offset:
        o = off.double().repeat_interleave(group, 1)
        w, weight = w + o, weight + o.abs()
    want = rows @ w.T
    blocks = torch.nn.functional.pad(rows.abs(), (0, -k % 128)).view(cols, -1, 128).amax(-1).repeat_interleave(128, 1)[:, :k]
    bound = (-(-k // 32) + 18) * U * (rows.abs() @ weight.T) + (2.0 ** -20 if cols > 4 and x_type != torch.float32 else 2.0 ** -27) * (blocks @ weight.T)
    assert ((y.double() - want).abs() <= rounded(bound, want, torch.float32)).all(), ((y.double() - want).abs() / bound).max().item()
