"""QuantizedKVCache: written rows equal the oracle's casts of the same rows bit
for bit, read-back equals decode * scale, the fused norm + rotation + write
equals the two calls, and what they refuse.

The oracle's casts (oracle/cast.py) are pinned to the reference's own vectors,
so codes and scales are compared exactly; read-back is one float32 product and
one rounding, so it too is compared exactly.
"""

import numpy as np
import pytest
import torch

from oracle import cast as ocast

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def bb():
    import breccia_b200
    return breccia_b200


def recipe(name, d):
    b = bb()
    return {"block4": lambda: b.Float8BlockScaling("E4M3", block_k=d),
            "block5": lambda: b.Float8BlockScaling("E5M2", block_k=d),
            "mx4": lambda: b.MXFP8BlockScaling("E4M3"), "mx5": lambda: b.MXFP8BlockScaling("E5M2"),
            "nvfp4": lambda: b.NVFP4BlockScaling()}[name]()


RECIPES = ["block4", "block5", "mx4", "mx5", "nvfp4"]


def oracle_rows(x, r):
    """Code bytes and scales that a cached row of x (tokens, heads, d) holds."""
    with np.errstate(all="ignore"):
        q = ocast.cast(x.float().cpu().numpy(), r)
    data = q.data
    if r.name == "nvfp4":
        data = data[..., 0::2] | (data[..., 1::2] << 4)
    return torch.from_numpy(np.ascontiguousarray(data)).cuda(), torch.from_numpy(q.scale).cuda()


def oracle_values(x, r):
    with np.errstate(all="ignore"):
        return torch.from_numpy(ocast.dequantize(ocast.cast(x.float().cpu().numpy(), r))).cuda()


def rows_of(cache, side, slots):
    page, at = slots // cache.page_size, slots % cache.page_size
    return getattr(cache, side + "_data")[page, :, at], getattr(cache, side + "_scale")[page, :, at]


def same(a, b):
    a, b = a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)
    return a.shape == b.shape and torch.equal(a, b)


def values(tokens, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, heads, d, generator=g) * torch.exp(3 * torch.randn(tokens, heads, 1, generator=g))
    x[torch.rand(x.shape, generator=g) < 0.01] *= 40
    if tokens > 2:
        x[0, 0] = 0.0
        x[1, 0, :16] = 1e-12
    return x.to(dtype).cuda()


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (37, 3, 16), (130, 8, 64)])
def test_write_matches_the_casts(name, d, dtype, tokens, heads, page):
    r = recipe(name, d)
    pages = tokens // page + 3
    cache = bb().QuantizedKVCache(pages, page, heads, d, r)
    k, v = values(tokens, heads, d, dtype, 1), values(tokens, heads, d, dtype, 2)
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(3))[:tokens].cuda()
    cache.write(k, v, slots)
    for side, x in (("k", k), ("v", v)):
        codes, scales = rows_of(cache, side, slots)
        want_codes, want_scales = oracle_rows(x, r)
        assert same(codes, want_codes)
        assert same(scales, want_scales)
    used = torch.zeros(pages * page, dtype=torch.bool, device="cuda")
    used[slots] = True
    free = (~used).nonzero()[:, 0]
    for side in "kv":  # nothing else is written
        assert not any(t.view(torch.uint8).any() for t in map(torch.Tensor.contiguous,
                                                               rows_of(cache, side, free)))


@pytest.mark.parametrize("name", RECIPES)
def test_write_matches_cast_on_special_values(name):
    d = 128
    r = recipe(name, d)
    x = torch.randn(12, 2, d, device="cuda")
    x[0, 0, 3], x[1, 1, 64], x[2, 0, 127] = float("nan"), float("inf"), -float("inf")
    x[3] = 3e38
    x[4] = 1e-42
    x[5, 0] = -0.0
    x[6, 1, ::2] = 448.0
    cache = bb().QuantizedKVCache(1, 16, 2, d, r)
    slots = torch.arange(12, device="cuda")
    cache.write(x, x, slots)
    st = bb().cast(x, r)
    data = st.data.view(torch.uint8)
    if name == "nvfp4":
        data = data[..., 0::2] | (data[..., 1::2] << 4)
    for side in "kv":
        codes, scales = rows_of(cache, side, slots)
        assert same(codes, data) and same(scales, st.scale)
    k, _ = cache.read(torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                      torch.tensor([12], dtype=torch.int32, device="cuda"), 12, torch.float32)
    want = bb().dequantize(st)
    assert torch.equal(torch.isnan(k[0]), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(k[0], nan=0.0), torch.nan_to_num(want, nan=0.0))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
def test_read_back_ragged(name, d, out):
    r, page, heads = recipe(name, d), 16, 3
    lengths = [33, 0, 1, 16]
    cache = bb().QuantizedKVCache(9, page, heads, d, r)
    table = torch.full((4, 5), -1, dtype=torch.int32)
    order, at = torch.randperm(9, generator=torch.Generator().manual_seed(4)), 0
    for b, n in enumerate(lengths):
        m = -(-n // page)
        table[b, :m] = order[at:at + m].int()
        at += m
    table = table.cuda()
    dense = {}
    for b, n in enumerate(lengths):
        if n:
            k, v = (values(n, heads, d, torch.bfloat16, 10 * b + i) for i in (1, 2))
            t = torch.arange(n, device="cuda")
            cache.write(k, v, table[b].long()[t // page] * page + t % page)
            dense[b] = (oracle_values(k, r), oracle_values(v, r))
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    wide = torch.full((4, 9), -7, dtype=torch.int32, device="cuda")
    wide[:, 2:7] = table
    got = cache.read(wide[:, 2:7], lens, 35, out)  # a table with a row stride
    for i in range(2):
        assert got[i].shape == (4, 35, heads, d) and got[i].dtype == out
        for b, n in enumerate(lengths):
            assert not got[i][b, n:].any()
            if n:
                assert torch.equal(got[i][b, :n], dense[b][i].to(out))


def test_slots_outside_are_not_written_and_pages_outside_read_zero():
    cache = bb().QuantizedKVCache(2, 16, 2, 64, recipe("mx4", 64))
    x = torch.randn(5, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache.write(x, x, torch.tensor([-1, 32, 2 ** 40, -2 ** 40, 31], device="cuda"))
    cache.write(x, x, torch.tensor([-1, 32, 2 ** 31 - 1, -2 ** 31, 30], dtype=torch.int32, device="cuda"))
    assert cache.k_data[1, :, 14:].any() and not cache.k_data[0].any() and not cache.k_data[1, :, :14].any()
    table = torch.tensor([[1, 2, -1, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    k, v = cache.read(table, torch.tensor([200], dtype=torch.int32, device="cuda"), 100)
    assert k[0, 14:16].any() and not k[0, 16:].any() and not v[0, 16:].any()
    k, v = cache.read(table, torch.tensor([-3], dtype=torch.int32, device="cuda"), 40)
    assert not k.any() and not v.any()


def test_strided_inputs_and_empty_calls():
    r = recipe("block4", 128)
    cache = bb().QuantizedKVCache(4, 16, 2, 128, r)
    qkv = torch.randn(20, 7, 128, device="cuda", dtype=torch.float16)
    k, v = qkv[:, 3:5], qkv[:, 5:]
    slots = torch.arange(20, 40, device="cuda")
    cache.write(k, v, slots)
    for side, x in (("k", k), ("v", v)):
        codes, scales = rows_of(cache, side, slots)
        want = oracle_rows(x, r)
        assert same(codes, want[0]) and same(scales, want[1])
    odd = torch.randn(20 * 2 * 128 + 4, device="cuda", dtype=torch.float16)[3:-1].view(20, 2, 128)
    cache.write(odd, odd.transpose(0, 1).contiguous().transpose(0, 1), slots)
    assert same(rows_of(cache, "k", slots)[0], oracle_rows(odd, r)[0])
    assert same(rows_of(cache, "v", slots)[0], oracle_rows(odd, r)[0])
    cache.write(k[:0], v[:0], slots[:0])
    k, v = cache.read(torch.zeros(2, 0, dtype=torch.int32, device="cuda"),
                      torch.ones(2, dtype=torch.int32, device="cuda"), 3)
    assert k.shape == (2, 3, 2, 128) and not k.any()
    k, v = cache.read(torch.zeros(2, 1, dtype=torch.int32, device="cuda"),
                      torch.ones(2, dtype=torch.int32, device="cuda"), 0)
    assert k.shape == (2, 0, 2, 128)


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d,rot,interleaved", [(64, 32, True), (128, 128, False), (256, 256, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_fused_write_equals_the_two_calls(name, d, rot, interleaved, dtype):
    t, hq, hk = 29, 6, 3
    g = torch.Generator().manual_seed(7)
    qkv = torch.randn(t, hq + 2 * hk, d, generator=g).to(dtype).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    wq, wk = torch.rand(d, device="cuda") + .5, torch.rand(d, device="cuda") + .5
    a = torch.rand(64, rot // 2, device="cuda") * 6
    cos, sin = a.cos(), a.sin()
    pos = torch.randint(0, 64, (t,), generator=g).cuda()
    slots = torch.randperm(48, generator=g)[:t].cuda()
    slots[5], slots[6] = -1, 48
    r = recipe(name, d)
    one, two = (bb().QuantizedKVCache(3, 16, hk, d, r) for _ in range(2))
    got = bb().qk_norm_rope_write(q, k, v, wq, wk, cos, sin, pos, one, slots, interleaved=interleaved)
    yq, yk = bb().qk_norm_rope(q, k, wq, wk, cos, sin, pos, interleaved=interleaved)
    two.write(yk, v, slots)
    assert torch.equal(got, yq)
    for x, y in zip(one._buffers, two._buffers):
        assert same(x, y)


def test_offsets_past_32_bits():
    # 4.3 GB of codes on each side; only the last and the first page are used
    heads, page, d = 8, 64, 128
    pages = (1 << 32) // (heads * page * d) + 2
    cache = bb().QuantizedKVCache(pages, page, heads, d, recipe("mx4", d))
    x = torch.randn(64, heads, d, device="cuda", dtype=torch.bfloat16)
    y = torch.randn(64, heads, d, device="cuda", dtype=torch.bfloat16)
    at = torch.arange(64, device="cuda")
    cache.write(x, y, (pages - 1) * page + at)
    cache.write(y, x, at)
    table = torch.tensor([[pages - 1], [0]], dtype=torch.int32, device="cuda")
    k, v = cache.read(table, torch.full((2,), 64, dtype=torch.int32, device="cuda"), 64, torch.float32)
    for got, want in ((k[0], x), (v[0], y), (k[1], y), (v[1], x)):
        assert torch.equal(got, oracle_values(want, cache.recipe))
    q = torch.randn(2, 16, d, device="cuda", dtype=torch.bfloat16)
    ctx = torch.full((2,), 63, dtype=torch.int32, device="cuda")
    out = bb().cache_attention(q, cache, table, ctx)
    small = bb().QuantizedKVCache(2, page, heads, d, cache.recipe)
    small.write(x, y, page + at)
    small.write(y, x, at)
    want = bb().cache_attention(q, small, torch.tensor([[1], [0]], dtype=torch.int32, device="cuda"), ctx)
    assert torch.equal(out, want)


def test_refusals():
    b = bb()
    r = recipe("mx4", 128)
    with pytest.raises(ValueError):
        b.QuantizedKVCache(4, 24, 2, 128, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache(4, 8, 2, 128, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache(4, 16, 2, 96, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache(0, 16, 2, 128, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache(4, 16, 2, 64, b.Float8BlockScaling(block_k=128))
    with pytest.raises(TypeError):
        b.QuantizedKVCache(4, 16, 2, 128, b.Float8CurrentScaling())
    with pytest.raises(TypeError):
        b.QuantizedKVCache(4, 16, 2, 128, r, device="cpu")
    c = b.QuantizedKVCache(4, 16, 2, 128, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache.from_buffers(c.k_data, c.k_scale[..., :2].contiguous(), c.v_data, c.v_scale, r)
    with pytest.raises(TypeError):
        b.QuantizedKVCache.from_buffers(c.k_data, c.k_scale.float(), c.v_data, c.v_scale, r)
    with pytest.raises(ValueError):
        b.QuantizedKVCache.from_buffers(c.k_data[:, ::2], c.k_scale, c.v_data, c.v_scale, r)
    x = torch.randn(3, 2, 128, device="cuda", dtype=torch.bfloat16)
    s = torch.arange(3, device="cuda")
    with pytest.raises(ValueError):
        c.write(x[:, :1], x[:, :1], s)
    with pytest.raises(ValueError):
        c.write(x, x[:2], s)
    with pytest.raises(ValueError):
        c.write(x, x.half(), s)
    with pytest.raises(ValueError):
        c.write(x, x, s[:2])
    with pytest.raises(TypeError):
        c.write(x, x, s.float())
    with pytest.raises(TypeError):
        c.write(x.cpu(), x, s)
    with pytest.raises(RuntimeError):
        c.write(x.requires_grad_(True), x, s)
    x = x.detach()
    t, n = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        c.read(t.long(), n, 4)
    with pytest.raises(TypeError):
        c.read(t, n.long(), 4)
    with pytest.raises(ValueError):
        c.read(t, n.expand(2), 4)
    with pytest.raises(ValueError):
        c.read(t, n, -1)
    with pytest.raises(TypeError):
        c.read(t, n, 4, torch.float64)
    w = torch.ones(128, device="cuda")
    a = torch.zeros(4, 64, device="cuda")
    with pytest.raises(TypeError):
        b.qk_norm_rope_write(x.float(), x.float(), x.float(), w, w, a, a, s, c, s)
    with pytest.raises(ValueError):
        b.qk_norm_rope_write(x, x[:, :1], x, w, w, a, a, s, c, s)
    with pytest.raises(TypeError):
        b.qk_norm_rope_write(x, x, x, w, w, a, a, s, None, s)
    with pytest.raises(RuntimeError):
        b.qk_norm_rope_write(x, x, x, w.requires_grad_(True), w, a, a, s, c, s)
