"""The attention block's operators refuse forward-mode tangents, whether gradients are
enabled or not, instead of dropping them; without a tangent a dual level changes nothing."""

import pytest
import torch
from torch.autograd import forward_ad

import breccia_b200 as bb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def block():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 4, 128, generator=g).to(torch.bfloat16).cuda()
    w = torch.ones(128, device="cuda")
    a = torch.rand(8, 64, generator=g).cuda()
    cache = bb.QuantizedKVCache(2, 16, 4, 128, bb.MXFP8BlockScaling())
    return x, w, a.cos(), a.sin(), torch.arange(5, device="cuda"), cache


def calls(x, w, cos, sin, pos, cache):
    """Each call, as a function of the tensor that may carry a tangent."""
    table = torch.zeros(5, 1, dtype=torch.int32, device="cuda")
    lens = torch.ones(5, dtype=torch.int32, device="cuda")
    return {
        "norm_q": lambda t: bb.qk_norm_rope(t, x, w, w, cos, sin, pos),
        "norm_k": lambda t: bb.qk_norm_rope(x, t, w, w, cos, sin, pos),
        "fused_v": lambda t: bb.qk_norm_rope_write(x, x, t, w, w, cos, sin, pos, cache, pos),
        "write_k": lambda t: cache.write(t, x, pos),
        "attend_q": lambda t: bb.cache_attention(t, cache, table, lens),
    }


NAMES = ["norm_q", "norm_k", "fused_v", "write_k", "attend_q"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(name, grad):
    args = block()
    call = calls(*args)[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(dual)


@pytest.mark.parametrize("name", NAMES)
def test_no_tangent_in_a_dual_level(name):
    args = block()
    call = calls(*args)[name]
    args[-1].write(args[0], args[0], args[4])
    want = call(args[0])
    with forward_ad.dual_level():
        got = call(args[0])
    for a, b in zip(want if isinstance(want, tuple) else (want,), got if isinstance(got, tuple) else (got,)):
        assert a is b is None or torch.equal(a, b)


def test_tangent_of_a_weight():
    x, w, cos, sin, pos, _ = block()
    with torch.no_grad(), forward_ad.dual_level():
        dual = forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises((RuntimeError, NotImplementedError)):
            bb.qk_norm_rope(x, x, dual, w, cos, sin, pos)
