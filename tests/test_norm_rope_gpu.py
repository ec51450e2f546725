"""qk_norm_rope and its gradients against the formulas in 64 bits, the
gradients against differences, and what it refuses.

Tolerances. The kernel computes in float32 and rounds once: half an ulp of the
output type on every element (2^-8, 2^-11, 2^-24 of it), and for the float32
steps (a sum of up to 256 squares by halves, a reciprocal square root good to 2
ulp, three products, one rotation) less than 32 float32 ulp of the head's largest
element. Weight gradients sum n rows in float32: n of them split over at least
n / 256 chains lose less than 64 ulp of the sum of magnitudes.
"""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def bb():
    import breccia_b200
    return breccia_b200


def tables(rows, rot):
    f = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return a.cos().float().cuda(), a.sin().float().cuda()


def reference(x, w, cos, sin, pos, eps, interleaved):
    """float64 definition, differentiable."""
    x, w = x.double(), w.double()
    y = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    r = 2 * c.shape[-1]
    head, rest = y[..., :r], y[..., r:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = head.chunk(2, -1)
        head = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([head, rest], -1)


def close(got, want, dtype, scale=None):
    scale = want.abs().amax(-1, keepdim=True) if scale is None else scale
    err = (got.double() - want).abs()
    tol = HALF_ULP[dtype] * want.abs() + 32 * F32 * scale + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert got.dtype == dtype
    assert bool((err <= tol).all()), float((err - tol).max())


def inputs(tokens, hq, hk, d, dtype, wdtype, seed=0, mag=1.5):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(tokens, hq, d, generator=g) * mag).to(dtype).cuda()
    k = (torch.randn(tokens, hk, d, generator=g) * mag).to(dtype).cuda()
    wq = (1 + 0.3 * torch.randn(d, generator=g)).to(wdtype).cuda()
    wk = (1 + 0.3 * torch.randn(d, generator=g)).to(wdtype).cuda()
    return q, k, wq, wk


SHAPES = [  # tokens, hq, hk, d, rot
    (1, 32, 8, 128, 128), (1, 1, 1, 16, 16), (7, 3, 1, 64, 64), (65, 8, 2, 64, 32),
    (33, 5, 5, 80, 48), (130, 6, 3, 96, 96), (19, 4, 4, 256, 256), (9, 4, 1, 192, 64),
    (257, 16, 4, 128, 64), (2, 71, 2, 112, 112),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                          (torch.float32, torch.float32), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward(shape, dtype, wdtype, interleaved):
    t, hq, hk, d, rot = shape
    q, k, wq, wk = inputs(t, hq, hk, d, dtype, wdtype)
    cos, sin = tables(500, rot)
    pos = torch.randint(0, 500, (t,), generator=torch.Generator().manual_seed(1)).cuda()
    yq, yk = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos, eps=1e-5, interleaved=interleaved)
    close(yq, reference(q, wq, cos, sin, pos, 1e-5, interleaved), dtype)
    close(yk, reference(k, wk, cos, sin, pos, 1e-5, interleaved), dtype)


def test_packed_views_leading_shape_and_int32_positions():
    qkv = torch.randn(3, 11, 12 * 64, device="cuda").to(torch.bfloat16).view(3, 11, 12, 64)
    q, k = qkv[..., :8, :], qkv[..., 8:10, :]
    wq, wk = torch.rand(64, device="cuda") + .5, torch.rand(64, device="cuda") + .5
    cos, sin = tables(40, 64)
    pos = torch.arange(33, device="cuda", dtype=torch.int32).view(3, 11)
    yq, yk = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    assert yq.shape == q.shape and yk.shape == k.shape
    flat = pos.reshape(-1).long()
    close(yq.reshape(33, 8, 64), reference(q.reshape(33, 8, 64), wq, cos, sin, flat, 1e-6, False),
          torch.bfloat16)
    close(yk.reshape(33, 2, 64), reference(k.reshape(33, 2, 64), wk, cos, sin, flat, 1e-6, False),
          torch.bfloat16)


def test_odd_strides_alignment_and_broadcast():
    base = torch.randn(4 * 3 * 64 + 8, device="cuda")
    q = base[1:1 + 4 * 3 * 64].view(4, 3, 64)  # 4 bytes off a 16-byte boundary
    k = torch.randn(1, 1, 64, device="cuda").expand(4, 2, 64)  # one head for all
    w = torch.rand(65, device="cuda")[1:]
    cos, sin = tables(8, 64)
    pos = torch.tensor([7, 0, 0, 3], device="cuda")
    yq, yk = bb().qk_norm_rope(q, k, w, w, cos, sin, pos)
    close(yq, reference(q, w, cos, sin, pos, 1e-6, False), torch.float32)
    close(yk, reference(k, w, cos, sin, pos, 1e-6, False), torch.float32)
    t = torch.randn(64, 3, 4, device="cuda").permute(2, 1, 0)  # last axis strided
    yq, _ = bb().qk_norm_rope(t, k, w, w, cos, sin, pos)
    close(yq, reference(t, w, cos, sin, pos, 1e-6, False), torch.float32)


def test_zero_tokens_zero_heads_zeros_and_large():
    cos, sin = tables(4, 64)
    w = torch.ones(64, device="cuda")
    e = torch.empty(0, 2, 64, device="cuda")
    yq, yk = bb().qk_norm_rope(e, e, w, w, cos, sin, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert yq.shape == (0, 2, 64) and yk.shape == (0, 2, 64)
    none = torch.empty(3, 0, 64, device="cuda")
    q = torch.zeros(3, 2, 64, device="cuda")
    q[1] = 3e18
    q[2] = 1e-30
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    yq, yk = bb().qk_norm_rope(q, none, w, w, cos, sin, pos)
    assert yk.shape == (3, 0, 64)
    close(yq, reference(q, w, cos, sin, pos, 1e-6, False), torch.float32)
    x = q.clone().requires_grad_(True)
    yq, yk = bb().qk_norm_rope(x, none, w, w, cos, sin, pos)
    (yq[0].sum() + yk.sum()).backward()
    # at x = 0 the gradient is w / sqrt(eps)
    close(x.grad[0], torch.full((2, 64), 1e3, dtype=torch.float64, device="cuda"), torch.float32)
    assert not x.grad[1:].any()


def test_position_outside_the_table_is_nan_and_nan_stays_in_its_head():
    q, k, wq, wk = inputs(4, 2, 2, 64, torch.float32, torch.float32)
    cos, sin = tables(10, 64)
    q[3, 1, 5] = float("nan")
    pos = torch.tensor([3, 10, -1, 9], device="cuda")
    yq, yk = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    assert torch.isnan(yq[1:3]).all() and torch.isnan(yk[1:3]).all()
    assert torch.isnan(yq[3, 1]).all() and torch.isfinite(yq[3, 0]).all() and torch.isfinite(yk[3]).all()
    assert torch.isfinite(yq[0]).all()


@pytest.mark.parametrize("shape", [(1, 4, 1, 64, 64), (37, 8, 2, 128, 128), (301, 3, 1, 64, 32),
                                   (12, 2, 2, 256, 128), (50, 5, 2, 80, 48)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(shape, dtype, interleaved):
    t, hq, hk, d, rot = shape
    q, k, wq, wk = inputs(t, hq, hk, d, dtype, torch.float32, seed=3)
    cos, sin = tables(400, rot)
    pos = torch.randint(0, 400, (t,), generator=torch.Generator().manual_seed(2)).cuda()
    leaf = [x.detach().requires_grad_(True) for x in (q, k, wq, wk)]
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    yq, yk = bb().qk_norm_rope(*leaf, cos, sin, pos, interleaved=interleaved)
    got = torch.autograd.grad((yq, yk), leaf, (gq, gk))
    want_leaf = [x.detach().double().requires_grad_(True) for x in (q, k, wq, wk)]
    want = torch.autograd.grad(
        (reference(want_leaf[0], want_leaf[2], cos, sin, pos, 1e-6, interleaved),
         reference(want_leaf[1], want_leaf[3], cos, sin, pos, 1e-6, interleaved)),
        want_leaf, (gq.double(), gk.double()))
    for g, w, x, gy, weight in ((got[0], want[0], q, gq, wq), (got[1], want[1], k, gk, wk)):
        # terms of a head: r |gz w| and r |x r|^2-weighted means of it
        r = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        scale = r * gy.double().abs().amax(-1, keepdim=True) * float(weight.abs().max()) * \
            2 * (1 + (x.double() * r).abs().amax(-1, keepdim=True))
        close(g, w, dtype, scale)
    for g, w, x, gy in ((got[2], want[2], q, gq), (got[3], want[3], k, gk)):
        r = (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt()
        total = (2 * gy.double().abs().amax(-1, keepdim=True) * (x.double() * r).abs()).sum((0, 1))
        assert bool(((g.double() - w).abs() <= 64 * F32 * total).all())


def test_gradient_against_differences():
    q, k, wq, wk = inputs(3, 2, 1, 64, torch.float32, torch.float32, seed=5)
    cos, sin = tables(30, 32)
    pos = torch.tensor([4, 0, 29], device="cuda")
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    leaf = [x.clone().requires_grad_(True) for x in (q, k, wq, wk)]
    got = torch.autograd.grad(bb().qk_norm_rope(*leaf, cos, sin, pos), leaf, (gq, gk))

    def value(args):
        return float((reference(args[0], args[2], cos, sin, pos, 1e-6, False) * gq.double()).sum() +
                     (reference(args[1], args[3], cos, sin, pos, 1e-6, False) * gk.double()).sum())

    for n in range(4):
        step = torch.randn_like(leaf[n]).double()
        h = 1e-5
        args = [x.detach().double() for x in leaf]
        up, down = list(args), list(args)
        up[n], down[n] = args[n] + h * step, args[n] - h * step
        diff = (value(up) - value(down)) / (2 * h)  # second-order error: 1e-10 relative
        mine = float((got[n].double() * step).sum())
        size = float((got[n].double() * step).abs().sum())
        assert abs(mine - diff) <= 1e-5 * size


def test_gradients_only_of_what_asks_and_repeatable():
    q, k, wq, wk = inputs(700, 8, 2, 128, torch.bfloat16, torch.bfloat16, seed=8)
    cos, sin = tables(700, 128)
    pos = torch.arange(700, device="cuda")
    wq.requires_grad_(True)
    runs = []
    for _ in range(3):
        wq.grad = None
        yq, yk = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos)
        (yq.float().square().sum() + yk.float().sum()).backward()
        runs.append(wq.grad.clone())
    assert wk.grad is None and runs[0].dtype == torch.bfloat16
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_shared_tensor_and_non_contiguous_gradients():
    x = torch.randn(5, 2, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    cos, sin = tables(5, 64)
    pos = torch.arange(5, device="cuda")
    yq, yk = bb().qk_norm_rope(x, x, w, w, cos, sin, pos)  # one tensor on both sides
    g = torch.randn(64, 2, 5, device="cuda").permute(2, 1, 0)
    got = torch.autograd.grad((yq, yk), (x, w), (g, g[:1].expand(5, 2, 64)))
    x64, w64 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    y = reference(x64, w64, cos, sin, pos, 1e-6, False)
    want = torch.autograd.grad((y, y), (x64, w64), (g.double(), g[:1].expand(5, 2, 64).double()))
    for a, b in zip(got, want):
        assert float((a.double() - b).abs().max()) <= 1e-5 * float(b.abs().max())


def test_other_stream():
    q, k, wq, wk = inputs(4000, 8, 2, 128, torch.bfloat16, torch.bfloat16, seed=9)
    cos, sin = tables(4000, 128)
    pos = torch.arange(4000, device="cuda")
    want = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q2 = q * 2
        got = bb().qk_norm_rope(q2 / 2, k, wq, wk, cos, sin, pos)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_refusals():
    q, k, wq, wk = inputs(4, 2, 2, 64, torch.float32, torch.float32)
    cos, sin = tables(10, 64)
    pos = torch.arange(4, device="cuda")
    f = bb().qk_norm_rope
    with pytest.raises(TypeError):
        f(q.cpu(), k, wq, wk, cos, sin, pos)
    with pytest.raises(TypeError):
        f(q.double(), k.double(), wq, wk, cos, sin, pos)
    with pytest.raises(ValueError):
        f(q, k.bfloat16(), wq, wk, cos, sin, pos)
    with pytest.raises(ValueError):
        f(q[:3], k, wq, wk, cos, sin, pos)
    with pytest.raises(ValueError):
        f(q[..., :40], k[..., :40], wq[:40], wk[:40], cos[:, :16], sin[:, :16], pos)
    with pytest.raises(ValueError):
        f(q, k, wq[:32], wk, cos, sin, pos)
    with pytest.raises(TypeError):
        f(q, k, wq, wk.half(), cos, sin, pos)
    with pytest.raises(TypeError):
        f(q, k, wq, wk, cos.half(), sin, pos)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos, sin[:, :16], pos)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos[:, :12], sin[:, :12], pos)
    with pytest.raises(ValueError):
        f(q, k, wq, wk, cos, sin, pos[:3])
    with pytest.raises(TypeError):
        f(q, k, wq, wk, cos, sin, pos.float())
    big = torch.randn(2, 1, 512, device="cuda")
    with pytest.raises(ValueError):
        f(big, big, torch.ones(512, device="cuda"), torch.ones(512, device="cuda"), cos, sin, pos[:2])
