"""qk_norm_rope and its gradients on rows as large as their type holds. Formula in 64
bits; tolerances as in test_norm_rope_gpu.py (half an ulp of the type and 32 float32 ulp
of the head's largest; gradients: of the terms' size). A gradient of such rows is as
small as 2^-128: below float32's normal numbers, where it is held to 2^-149."""

import pytest
import torch

from test_norm_rope_gpu import F32, HALF_ULP, bb, close, reference, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def rows(d, dtype):
    """Heads of one magnitude from the largest that the type holds down to ordinary ones,
    and heads of mixed magnitudes."""
    g = torch.Generator().manual_seed(3)
    top = 65504.0 if dtype == torch.float16 else 3.3e38
    sizes = [top * s for s in (1.0, 2.0 ** -3, 2.0 ** -4, 2.0 ** -20, 2.0 ** -60, 2.0 ** -66, 2.0 ** -120)]
    x = torch.rand(len(sizes) + 1, 2, d, generator=g, dtype=torch.float64) * 2 - 1
    x[:-1] *= torch.tensor(sizes, dtype=torch.float64)[:, None, None]
    x[-1] *= top * 2.0 ** (-80 * torch.rand(2, d, generator=g, dtype=torch.float64))
    return x.to(dtype).cuda()


@pytest.mark.parametrize("d,rot", [(16, 16), (64, 32), (128, 128), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_large_rows(d, rot, dtype, interleaved):
    x = rows(d, dtype)
    n = x.shape[0]
    w = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(4))).cuda()
    cos, sin = tables(n, rot)
    pos = torch.arange(n, device="cuda")
    yq, yk = bb().qk_norm_rope(x, x[:, :1], w, w, cos, sin, pos, interleaved=interleaved)
    want = reference(x, w, cos, sin, pos, 1e-6, interleaved)
    close(yq, want, dtype)
    close(yk, want[:, :1], dtype)


@pytest.mark.parametrize("d,rot", [(64, 32), (128, 128), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_large_rows(d, rot, dtype):
    x = rows(d, dtype)
    n = x.shape[0]
    w = (1 + 0.3 * torch.randn(d, generator=torch.Generator().manual_seed(4))).cuda()
    cos, sin = tables(n, rot)
    pos = torch.arange(n, device="cuda")
    g = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    leaf = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    y, _ = bb().qk_norm_rope(leaf[0], x[:, :0], leaf[1], w, cos, sin, pos)
    gx, gw = torch.autograd.grad(y, leaf, g)
    want = [x.double().requires_grad_(True), w.double().requires_grad_(True)]
    wx, ww = torch.autograd.grad(reference(want[0], want[1], cos, sin, pos, 1e-6, False), want, g.double())
    r = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    gmax = g.double().abs().amax(-1, keepdim=True)
    size = (x.double() * r).abs()
    scale = r * gmax * float(w.abs().max()) * 2 * (1 + size.amax(-1, keepdim=True))
    tol = HALF_ULP[dtype] * wx.abs() + 32 * F32 * scale + 2.0 ** -149 * 4
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -133  # half a step of its numbers below 2^-126
    assert bool(((gx.double() - wx).abs() <= tol).all())
    assert bool(((gw.double() - ww).abs() <= 64 * F32 * (2 * gmax * size).sum((0, 1))).all())


@pytest.mark.parametrize("d,rot", [(64, 32), (96, 48), (128, 64), (256, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_infinity_stays_in_its_pair(d, rot, dtype, interleaved):
    """An infinite element makes itself NaN and, where it is rotated, its partner; the rest
    of its head is 0. A head of infinite gradients makes no other weight's gradient NaN."""
    x = torch.randn(d, 1, d, generator=torch.Generator().manual_seed(6)).to(dtype).cuda()
    at = torch.arange(d, device="cuda")
    x[at, 0, at] = float("inf")
    w = torch.rand(d, device="cuda") + 0.5
    cos, sin = tables(d + 1, rot)
    pos = at + 1
    y, _ = bb().qk_norm_rope(x, x[:, :0], w, w, cos, sin, pos, interleaved=interleaved)
    want = reference(x, w, cos, sin, pos, 1e-6, interleaved)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert not torch.nan_to_num(y, nan=0.0).any()
    leaf = w.clone().requires_grad_(True)
    ones = torch.ones(1, 1, d, dtype=dtype, device="cuda")
    z, _ = bb().qk_norm_rope(ones, ones[:, :0], leaf, w, cos, sin, pos[:1], interleaved=interleaved)
    g = torch.zeros_like(z)
    g[..., d - 3] = float("inf")
    (gw,) = torch.autograd.grad(z, leaf, g)
    assert not bool(torch.isfinite(gw[d - 3])) and int((~torch.isfinite(gw)).sum()) == 1
