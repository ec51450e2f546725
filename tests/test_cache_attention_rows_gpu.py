"""cache_attention with row counts of a cache head on both sides of every choice
that the entry point makes from them: the special cases of
test_cache_attention_gpu.py with 24 rows, with 72 (more than any recipe keeps on
the register path) and with 300 (two blocks of rows).

The reference is 64 bits on the values that the cache holds; a mask says place by
place what a row sees. Tolerances, from the kernels' own roundings. A score is a
float32 sum of d products, off by at most d 2^-24 of the sum of magnitudes (S: the
largest among the places that the row sees). A probability is off by that much
relatively, by the exponential's 2^-21, and by one rounding to f16: 2^-11 of it or,
below f16's normal numbers, 2^-31 of the row's largest (2^-20 on the register path of
block FP8, where it carries a scale that may lie 2^11 below the reference), or all of it
where that is less. Values on
tcgen05 in block FP8 are rounded to f16 once more: 2^-11 of them or, for E5M2's
smallest codes, 2^-24 of the token's largest. Sums are float32. So an output is within

    (2^-10 + 2 d 2^-24 S) sum p |v| + 2^-24 sum p max |v| + sum min(p, f max p) |v|

of the formula (f: 2^-31 or 2^-20), and half an ulp of its type; log-sum-exp is within
d 2^-24 S + 2^-20 (1 + |lse|).
"""

import math

import pytest
import torch

from test_cache_attention_gpu import HALF_ULP, RECIPES, Case, bb, recipe

pytestmark = pytest.mark.gpu

ROWS = [(6, 4), (18, 4), (75, 4)]  # draft, group: 24, 72, 300 rows


@pytest.fixture(scope="module", autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def causal(c):
    """What every row sees, (draft, context + draft) for each sequence."""
    t = c.draft
    tri = torch.ones(t, t, dtype=torch.bool, device="cuda").tril()
    return [torch.cat([tri.new_ones(t, n), tri], 1) for n in c.ctx]


def with_tree(c, tree):
    return [torch.cat([tree.new_ones(c.draft, n), tree[b] if tree.ndim == 3 else tree], 1)
            for b, n in enumerate(c.ctx)]


def rewrite(c, b, first, k=None, v=None):
    """Put other keys or values at the places from `first` on of sequence b."""
    page = c.cache.page_size
    n = (k if k is not None else v).shape[0]
    t = torch.arange(first, first + n, device="cuda")
    at = c.table[b].long()[t // page], t % page
    kk, vv = (x[b, first:first + n] for x in held(c))
    old = [buf[at[0], :, at[1]].clone() for buf in c.cache._buffers]
    c.cache.write(kk if k is None else k, vv if v is None else v, at[0] * page + at[1])
    for side, given in ((0, k), (2, v)):  # the side that stays keeps its codes and scales
        if given is None:
            for i in (side, side + 1):
                c.cache._buffers[i][at[0], :, at[1]] = old[i]


def held(c, dtype=torch.float32):
    return c.cache.read(c.table, c.context + c.draft, max(c.ctx) + c.draft, dtype)


def verify(c, got, see, scale=None, columns=None, rows=None):
    """Rows (all, or those of the mask (batch, draft)) and columns against the formula."""
    out, lse = got
    scale = c.d ** -0.5 if scale is None else scale
    block = c.cache.recipe.name == "block"
    floor = 2.0 ** (-20 if block and (c.draft * c.group <= 64 or c.d == 256) else -31)
    k, v = held(c)
    for b, m in enumerate(see):
        n = m.shape[1]
        kk, vv = (x[b, :n].double().repeat_interleave(c.group, 1).transpose(0, 1) for x in (k, v))
        q = c.q[b].double().transpose(0, 1)
        s = (q @ kk.transpose(1, 2) * scale).masked_fill(~m, -math.inf)
        big = (q.abs() @ kk.abs().transpose(1, 2) * abs(scale)).masked_fill(~m, 0).amax(-1)
        want_lse = torch.logsumexp(s, -1)
        p = torch.exp(s - want_lse[..., None].nan_to_num(neginf=0.0))
        # values that nobody sees may be anything
        whole = torch.where(m.any(0)[None, :, None], vv, torch.zeros_like(vv))
        vv = whole if columns is None else whole[..., columns]
        want, mass = p @ vv, p @ vv.abs()
        largest = p @ whole.abs().amax(-1, keepdim=True)
        low = torch.minimum(p, floor * p.amax(-1, keepdim=True)) @ vv.abs()
        o, l = out[b].double().transpose(0, 1), lse[b].double().transpose(0, 1)
        if columns is not None:
            o = o[..., columns]
        keep = torch.ones_like(m[:, 0]) if rows is None else rows[b]
        none = ~m.any(1)
        assert not o[:, none].any() and bool((l[:, none] == -math.inf).all())
        keep = keep & ~none
        tol = (2.0 ** -10 + 2 * c.d * 2.0 ** -24 * big[..., None]) * mass + \
            HALF_ULP[out.dtype] * want.abs() + 2.0 ** -24 + 2.0 ** -24 * largest + low
        err = (o - want).abs()
        assert bool((err <= tol)[:, keep].all()), (b, float((err / tol)[:, keep].nan_to_num(nan=math.inf).max()))
        ltol = d_tol(c.d, big, want_lse)
        lerr = (l - want_lse).abs()
        assert bool((lerr <= ltol)[:, keep].all()), (b, float((lerr - ltol)[:, keep].nan_to_num(nan=math.inf).max()))


def d_tol(d, big, lse):
    return d * 2.0 ** -24 * big + 2.0 ** -20 * (1 + lse.abs())


# ------------------------------------------------------------------ factors


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(name, d, draft, group, scale):
    c = Case(name, d, 1, group, [300, 2], draft, seed=21)
    verify(c, c.run(scale=scale), causal(c), scale)


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
def test_zero_and_tiny_queries_over_tiny_keys(name, draft, group):
    c = Case(name, 128, 1, group, [200, 3], draft, seed=22)
    g = torch.Generator().manual_seed(22)
    for b, n in enumerate(c.ctx):
        rewrite(c, b, 0, k=(1e-9 * torch.randn(n + draft, 1, 128, generator=g)).cuda())
    c.q[:, 0] = 0
    c.q[:, 1] *= 2.0 ** -40
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
def test_cache_as_the_constructor_leaves_it(name, draft, group):
    cache = Case(name, 128, 2, group, [1], draft, seed=23).cache
    for buf in cache._buffers:
        buf.zero_()
    g = torch.Generator().manual_seed(23)
    q = torch.randn(1, draft, 2 * group, 128, generator=g).to(torch.bfloat16).cuda()
    q[:, 1] *= 2.0 ** -30
    table = torch.zeros(1, 20, dtype=torch.int32, device="cuda")
    n = torch.tensor([200], dtype=torch.int32, device="cuda")
    out, lse = bb().cache_attention(q, cache, table, n, return_lse=True)
    want = torch.log(201.0 + torch.arange(draft, device="cuda"))[:, None].expand(draft, 2 * group)
    assert not out.any()
    assert float((lse[0] - want).abs().max()) <= 2.0 ** -20 * (1 + math.log(300))


@pytest.mark.parametrize("draft,group", ROWS)
def test_large_queries(draft, group):
    c = Case("mx4", 128, 1, group, [150, 2], draft, seed=24)
    c.q[0] *= 2.0 ** 60
    got = c.run(scale=2.0 ** -60)
    ref = Case("mx4", 128, 1, group, [150, 2], draft, seed=24)
    want = ref.run(scale=1.0)
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[1][0], want[1][0])


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("scale", [2.0 ** 12, -2.0 ** 30, 2.0 ** 80])
def test_large_scores(name, d, draft, group, scale):
    """Every row's weight lies on one place, and its score is beyond 2^18, 2^36, 2^86."""
    c = Case(name, d, 1, group, [300, 1], draft, seed=25)
    out, lse = c.run(scale=scale)
    k, v = held(c)
    for b, m in enumerate(causal(c)):
        n = m.shape[1]
        kk, vv = (x[b, :n].double().repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
        s = (c.q[b].double().transpose(0, 1) @ kk.transpose(1, 2) * scale).masked_fill(~m, -math.inf)
        top, at = s.topk(2, -1) if n > 1 else (s, torch.zeros_like(s, dtype=torch.int64))
        big = (c.q[b].double().abs().transpose(0, 1) @ kk.abs().transpose(1, 2) * abs(scale)).amax(-1)
        # rows whose second score is below the first by more than the scores' error and 64
        clear = top[..., 0] - top[..., 1] > 2 * d * 2.0 ** -24 * big + 64
        assert float(clear.double().mean()) > 0.5
        want = vv.gather(1, at[..., :1].expand(-1, -1, d))
        o, l = out[b].double().transpose(0, 1), lse[b].double().transpose(0, 1)
        assert bool(((o - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10)[clear].all())
        assert bool(((l - top[..., 0]).abs() <= d_tol(d, big, top[..., 0]))[clear].all())


# ------------------------------------------------------------------ masks


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("low", [-200.0, -90.0, 3.0])
def test_first_pages_outside_the_cache_and_low_scores(name, draft, group, low):
    """A share that begins in pages that nobody sees, over scores far below zero."""
    c = Case(name, 128, 1, group, [330, 200], draft, page=64, seed=31)
    g = torch.Generator().manual_seed(32)
    for b, n in enumerate(c.ctx):
        k = 1 + 0.05 * torch.randn(n + draft, 1, 128, generator=g)
        rewrite(c, b, 0, k=k.cuda())
    c.q.copy_((1 + 0.05 * torch.randn(c.q.shape, generator=g)) * (low / 128))
    see = causal(c)
    for b, pages in enumerate(([0, 1], [0, 1, 2])):
        for page in pages:
            c.table[b, page] = [-1, c.cache.num_pages][page % 2]
            see[b][:, page * 64:page * 64 + 64] = False
    verify(c, c.run(scale=1.0), see, 1.0)


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", [(300, 1), (140, 2)])
@pytest.mark.parametrize("ctx", [0, 5])
def test_trees_of_separate_blocks(name, draft, group, ctx):
    """Drafted tokens over several tiles, of which a row sees those of its own block."""
    c = Case(name, 128, 1, group, [ctx], draft, seed=33)
    g = torch.Generator().manual_seed(34)
    k = 1 + 0.05 * torch.randn(ctx + draft, 1, 128, generator=g)
    rewrite(c, 0, 0, k=k.cuda())
    c.q.copy_((1 + 0.05 * torch.randn(c.q.shape, generator=g)) * (-200 / 128))
    block = torch.arange(draft, device="cuda") // 70
    tree = (block[:, None] == block[None]).tril()
    tree[3] = False
    see = with_tree(c, tree)
    see[0][draft // 2:, :ctx] = True
    verify(c, c.run(scale=1.0, tree_mask=tree), see, 1.0)


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
def test_random_trees_and_missing_drafts(name, draft, group):
    c = Case(name, 64, 2, group, [0, 77, 128], draft, page=32, seed=35)
    tree = torch.rand(3, draft, draft, generator=torch.Generator().manual_seed(36)) < 0.3
    tree[:, 1] = False
    tree = tree.cuda()
    drafts = [draft, draft - 2, 1]
    see = with_tree(c, tree)
    for b, n in enumerate(drafts):
        see[b][n:] = False
        see[b][:, c.ctx[b] + n:] = False
    lens = torch.tensor(drafts, dtype=torch.int32, device="cuda")
    verify(c, c.run(tree_mask=tree, draft_lens=lens), see)


# ------------------------------------------------------------------ what is not finite


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("ctx", [21, 250])
def test_unseen_nan(name, draft, group, ctx):
    """NaN behind the end of a page, in other pages and in drafted tokens that a row
    does not see; rows that see a drafted NaN get it, and where values are NaN only
    in those columns."""
    d = 128
    c = Case(name, d, 2, group, [ctx, 40], draft, seed=37)
    tree = torch.eye(draft, dtype=torch.bool, device="cuda").repeat(2, 1, 1)
    tree[:, :, 0] = True
    tree[:, 0, :] = False
    tree[:, 4:, 3] = (torch.arange(4, draft, device="cuda") % 2 == 0)
    see = with_tree(c, tree)
    want = c.run(tree_mask=tree)
    verify(c, want, see)
    live = torch.zeros(c.cache.num_pages, c.cache.page_size, dtype=torch.bool, device="cuda")
    for b, n in enumerate(c.ctx):
        t = torch.arange(n + draft, device="cuda")
        live[c.table[b].long()[t // 16], t % 16] = True
    for buf in c.cache._buffers:
        buf[(~live)[:, None, :, None].expand_as(buf)] = float("nan") if buf.dtype == torch.float32 else 255
    got = c.run(tree_mask=tree)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    seeing = tree[0, :, 3]
    rows = torch.stack([~seeing, torch.ones_like(seeing)])
    page, at = int(c.table[0, (ctx + 3) // 16]), (ctx + 3) % 16
    for side in ("k", "v"):
        data, scale = getattr(c.cache, side + "_data"), getattr(c.cache, side + "_scale")
        keep = data[page, :, at].clone(), scale[page, :, at].clone()
        data[page, :, at] = 255
        scale[page, :, at] = float("nan") if scale.dtype == torch.float32 else 255
        out, lse = c.run(tree_mask=tree)
        assert torch.isnan(out[0, seeing]).all()
        data[page, :, at], scale[page, :, at] = keep
        verify(c, (out, lse), see, rows=rows)
    # some of a token's values only
    if name == "nvfp4":
        c.cache.v_scale[page, 1, at, 3] = 0x7F
        bad = torch.arange(48, 64, device="cuda")
    elif name.startswith("mx"):
        c.cache.v_data[page, 1, at, 77] = 255
        c.cache.v_data[page, 1, at, 78] = 127
        bad = torch.tensor([77, 78], device="cuda")
    else:
        c.cache.v_data[page, 1, at, 3] = 255
        bad = torch.tensor([3], device="cuda")
    out, lse = c.run(tree_mask=tree)
    odd = torch.zeros_like(out, dtype=torch.bool)
    odd[0, :, group:] = seeing[:, None, None] & torch.isin(torch.arange(d, device="cuda"), bad)
    assert torch.equal(torch.isnan(out), odd)
    fine = torch.tensor([i for i in range(d) if i not in bad.tolist()], device="cuda")
    if name == "nvfp4":
        c.cache.v_scale[page, 1, at, 3] = 0
    else:
        c.cache.v_data[page, 1, at, bad] = 0
    verify(c, (out, lse), see, columns=fine)


@pytest.mark.parametrize("draft,group", ROWS)
def test_infinite_values(draft, group):
    """E5M2 holds infinities: a row that sees one gets it in that column."""
    c = Case("mx5", 128, 1, group, [140], draft, seed=38)
    at = 140 + 2
    page, place = int(c.table[0, at // 16]), at % 16
    c.cache.v_data[page, 0, place, 5] = 0x7C
    c.cache.v_data[page, 0, place, 6] = 0xFC
    out, lse = c.run()
    c.cache.v_data[page, 0, place, 5:7] = 0
    assert bool((out[0, 2:, :, 5] == math.inf).all()) and bool((out[0, 2:, :, 6] == -math.inf).all())
    assert torch.isfinite(out[0, :2]).all()
    fine = torch.tensor([i for i in range(128) if i not in (5, 6)], device="cuda")
    verify(c, (out, lse), causal(c), columns=fine)


# ------------------------------------------------------------------ magnitudes


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("spread", [4.0, 6.0])
def test_values_and_keys_of_very_different_size(name, d, draft, group, spread):
    c = Case(name, d, 2, group, [700, 31], draft, seed=41, spread=spread)
    verify(c, c.run(scale=0.02), causal(c), 0.02)


@pytest.mark.parametrize("name", ["block4", "block5", "mx4", "mx5"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("draft,group", ROWS)
def test_values_near_the_largest_float(name, d, draft, group):
    c = Case(name, d, 1, group, [1500, 20], draft, seed=42)
    for b, n in enumerate(c.ctx):
        v = torch.randn(n + draft, 1, d, generator=torch.Generator().manual_seed(43)).clamp(-3, 3) * 1e38
        rewrite(c, b, 0, v=v.cuda())
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", ["block4", "block5", "mx4", "mx5"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("draft,group", ROWS)
def test_sum_does_not_depend_on_values(name, d, draft, group):
    """Values near the largest float beside tiny ones, tiles apart."""
    c = Case(name, d, 1, group, [400], draft, seed=42)
    v = torch.randn(400 + draft, 1, d, generator=torch.Generator().manual_seed(43)).clamp(-3, 3)
    v[:128] *= 1e38
    v[128:] *= 1e-12
    rewrite(c, 0, 0, v=v.cuda())
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("side", ["k", "v", "kv"])
@pytest.mark.parametrize("power", [12, 40])
def test_unseen_finite_values_do_not_reach_a_row(name, d, draft, group, side, power):
    """Drafted tokens with keys or values 2^power times the others', seen by a few rows
    or by none. (NVFP4's scales do not reach that far: its keys and values saturate.)"""
    c = Case(name, d, 1, group, [37, 0], draft, seed=44)
    g = torch.Generator().manual_seed(45)
    tree = torch.ones(draft, draft, dtype=torch.bool).tril()
    large = [1, draft // 2]
    tree[:, large] = False
    tree[large, large] = True
    tree[draft - 1, 1] = True
    for b, n in enumerate(c.ctx):
        for node in large:
            x = torch.randn(1, 1, d, generator=g).cuda() * 2.0 ** power
            rewrite(c, b, n + node, **{s: x for s in side})
    tree = tree.cuda()
    see = with_tree(c, tree)
    got = c.run(tree_mask=tree)
    verify(c, got, see)
    # the same to the last bit but the order of sums, whatever stands in those places
    few = ~tree[:, large].any(1)
    for b, n in enumerate(c.ctx):
        for node in large:
            x = torch.randn(1, 1, d, generator=g).cuda()
            rewrite(c, b, n + node, **{s: x for s in side})
    other = c.run(tree_mask=tree)
    verify(c, other, see)
    assert torch.allclose(got[1][:, few], other[1][:, few], rtol=2.0 ** -18, atol=2.0 ** -18)


@pytest.mark.parametrize("name", ["mx4", "mx5", "block4", "block5"])
@pytest.mark.parametrize("draft,group", ROWS)
def test_garbage_in_unseen_places(name, draft, group):
    """The largest scales that there are, where no row looks."""
    c = Case(name, 128, 1, group, [60, 0], draft, seed=46)
    tree = torch.ones(draft, draft, dtype=torch.bool, device="cuda").tril()
    tree[:, 2] = False
    see = with_tree(c, tree)
    verify(c, c.run(tree_mask=tree), see)
    for b, n in enumerate(c.ctx):
        page, at = int(c.table[b, (n + 2) // 16]), (n + 2) % 16
        for side in "kv":
            getattr(c.cache, side + "_scale")[page, :, at] = 3e38 if name.startswith("block") else 254
            getattr(c.cache, side + "_data")[page, :, at] = 0x77
    verify(c, c.run(tree_mask=tree), see)


@pytest.mark.parametrize("name", ["mx4", "mx5", "block4", "block5"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("draft,group", ROWS)
@pytest.mark.parametrize("power", [30, 90])
def test_large_values_with_little_weight(name, d, draft, group, power):
    """Tokens of the context whose values are 2^power times the others' and whose scores are
    so low that they do not count; and channel blocks 2^30 apart."""
    c = Case(name, d, 1, group, [500], draft, seed=47)
    g = torch.Generator().manual_seed(48)
    n = 500 + draft
    k = torch.randn(n, 1, d, generator=g)
    v = torch.randn(n, 1, d, generator=g)
    far = torch.rand(n, generator=g) < 0.1
    far[0], far[128:256] = True, power > 60  # a tile of them, too
    k[far] = -1.0
    v[far] *= 2.0 ** power
    if name.startswith("mx"):
        v[..., :32] *= 2.0 ** 30
    c.q.copy_(1 + 0.02 * torch.randn(c.q.shape, generator=g))
    rewrite(c, 0, 0, k=k.cuda(), v=v.cuda())
    verify(c, c.run(scale=1.0), causal(c), 1.0)


@pytest.mark.parametrize("name", ["mx4", "block4"])
def test_many_steps_of_sizes_apart(name):
    """Hardly any step's tokens go together, and a warp has more steps than it notes."""
    heads, d, ctx, page, n = 32, 64, 16400, 64, 3
    pages = -(-(ctx + 1) // page)
    cache = bb().QuantizedKVCache(n * pages, page, heads, d, recipe(name, d))
    g = torch.Generator("cuda").manual_seed(49)
    for b in range(n):
        x = torch.randn(2, ctx + 1, heads, d, generator=g, device="cuda")
        v = x[1] * torch.exp(6 * torch.randn(ctx + 1, heads, 1, generator=g, device="cuda"))
        t = torch.arange(ctx + 1, device="cuda")
        cache.write(x[0], v, b * pages * page + t)
    c = Case.__new__(Case)
    c.cache, c.ctx, c.draft, c.group, c.d, c.heads = cache, [ctx] * n, 1, 1, d, heads
    c.table = torch.arange(n * pages, dtype=torch.int32, device="cuda").view(n, pages)
    c.context = torch.tensor(c.ctx, dtype=torch.int32, device="cuda")
    c.q = (0.3 * torch.randn(n, 1, heads, d, generator=g, device="cuda")).bfloat16()
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("draft,group", ROWS)
def test_zeros_among_ordinary_values(name, d, draft, group):
    """Rows and channel blocks of zeros, keys and values, drafted ones too."""
    c = Case(name, d, 1, group, [600, 0], draft, seed=50)
    g = torch.Generator().manual_seed(51)
    for b, n in enumerate(c.ctx):
        n += draft
        k, v = torch.randn(n, 1, d, generator=g), torch.randn(n, 1, d, generator=g)
        v[torch.rand(n, generator=g) < 0.1] = 0
        k[torch.rand(n, generator=g) < 0.1] = 0
        v[torch.rand(n, generator=g) < 0.1, :, :32] = 0
        v[torch.rand(n, generator=g) < 0.05] *= 0.02
        rewrite(c, b, 0, k=k.cuda(), v=v.cuda())
    verify(c, c.run(), causal(c))


# ------------------------------------------------------------------ lengths, pages, order


@pytest.mark.parametrize("name", ["block4", "mx4", "nvfp4"])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("draft,group", [(18, 4), (75, 4)])
def test_long_contexts_split_over_blocks(name, page, draft, group):
    c = Case(name, 128, 2, group, [9001, 40, 20011], draft, page=page, seed=51, spare_columns=3)
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_row_counts_around_the_choices(name, d, rows):
    c = Case(name, d, 1, 1, [270, 0], rows, page=32, seed=52)
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
def test_many_sequences_to_a_block(name, draft, group):
    """More items than blocks, so that a block goes from one to the next."""
    c = Case(name, 128, 4, group, [(61 * i) % 397 for i in range(90)], draft, page=32, seed=53)
    verify(c, c.run(), causal(c))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft,group", ROWS)
def test_pages_outside_the_cache(name, draft, group):
    c = Case(name, 128, 2, group, [400, 50], draft, page=32, seed=54)
    see = causal(c)
    for b, page, to in ((0, 1, -1), (0, 2, c.cache.num_pages), (0, 9, -7), (1, 0, -1)):
        c.table[b, page] = to
        see[b][:, page * 32:page * 32 + 32] = False
    verify(c, c.run(), see)
    out, lse = bb().cache_attention(c.q, c.cache, c.table[:, :0], c.context, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("name", ["mx4", "block4", "nvfp4"])
@pytest.mark.parametrize("draft,group", ROWS)
def test_repeatable_other_stream_and_graph(name, draft, group):
    c = Case(name, 128, 2, group, [5000, 300], draft, page=64, seed=55)
    want = c.run()
    for _ in range(3):
        got = c.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = bb().cache_attention(c.q * 1, c.cache, c.table, c.context)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bb().cache_attention(c.q, c.cache, c.table, c.context)
    c.context.copy_(torch.tensor([4000, 77], dtype=torch.int32))  # lengths are read by the replay
    graph.replay()
    assert torch.equal(out, c.run()[0])
