"""cache_attention against softmax(scale q k^T) v in 64 bits on the values that
the cache holds.

Tolerances, from the kernel's own roundings. Codes and scales enter the products
exactly. A score is a float32 sum of d products: off by at most d 2^-24 of the
sum of magnitudes, S. A probability is off by that much relatively, by the
exponential's 2^-21, and by one f16 rounding, 2^-11; sums are float32. So the
output is within (2^-10 + 2 d 2^-24 S) sum p |v| of the formula, and half an ulp
of its type; log-sum-exp is within d 2^-24 S + 2^-20 (1 + |lse|).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


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


class Case:
    """A cache with `ctx[b]` + `draft` written tokens per sequence."""

    def __init__(self, name, d, heads, group, ctx, draft, page=16, dtype=torch.bfloat16, seed=0, spread=1.0,
                 spare_columns=0):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.draft, self.group, self.d, self.heads = ctx, draft, group, d, heads
        need = [-(-(n + draft) // page) for n in ctx]
        pages = sum(need) + 2
        self.cache = bb().QuantizedKVCache(pages, page, heads, d, recipe(name, d))
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(ctx), max(need) + spare_columns), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        self.table = self.table.cuda()
        for b, n in enumerate(ctx):
            n += draft
            size = torch.exp(spread * torch.randn(n, heads, 1, generator=g))
            k = (torch.randn(n, heads, d, generator=g) * size).to(torch.bfloat16).cuda()
            v = (torch.randn(n, heads, d, generator=g) * size.flip(0)).to(torch.bfloat16).cuda()
            t = torch.arange(n, device="cuda")
            self.cache.write(k, v, self.table[b].long()[t // page] * page + t % page)
        self.q = torch.randn(len(ctx), draft, heads * group, d, generator=g).to(dtype).cuda()
        self.context = torch.tensor(ctx, dtype=torch.int32, device="cuda")

    def run(self, **kw):
        return bb().cache_attention(self.q, self.cache, self.table, self.context, return_lse=True, **kw)

    def check(self, got, drafts=None, tree=None, scale=None, rows=None):
        out, lse = got
        b_, t_, hq, d = self.q.shape
        assert out.shape == self.q.shape and out.dtype == self.q.dtype
        assert lse.shape == (b_, t_, hq) and lse.dtype == torch.float32
        scale = d ** -0.5 if scale is None else scale
        n_max = max(self.ctx) + t_
        lens = self.context + t_
        k, v = self.cache.read(self.table, lens, n_max, torch.float32)
        for b, n in enumerate(self.ctx):
            have = t_ if drafts is None else drafts[b]
            live = n + have
            kk = k[b, :live].double().repeat_interleave(self.group, 1).transpose(0, 1)  # (hq, live, d)
            vv = v[b, :live].double().repeat_interleave(self.group, 1).transpose(0, 1)
            q = self.q[b].double().transpose(0, 1)  # (hq, t, d)
            s = q @ kk.transpose(1, 2) * scale
            big = (q.abs() @ kk.abs().transpose(1, 2) * abs(scale))
            see = torch.ones(t_, live, dtype=torch.bool, device="cuda")
            part = torch.ones(t_, t_, dtype=torch.bool, device="cuda").tril() if tree is None else \
                tree[b] if tree.ndim == 3 else tree
            see[:, n:] = part[:, :have]
            see[have:] = False
            s = s.masked_fill(~see, -math.inf)
            want_lse = torch.logsumexp(s, -1) if live else torch.full((hq, t_), -math.inf, device="cuda").double()
            p = torch.exp(s - want_lse[..., None].nan_to_num(neginf=0.0))
            want, mass = p @ vv, p @ vv.abs()
            big = big.masked_fill(~see, 0).amax(-1) if live else torch.zeros_like(want_lse)
            none = ~see.any(1)
            o, l = out[b].double().transpose(0, 1), lse[b].double().transpose(0, 1)
            assert not o[:, none].any() and bool((l[:, none] == -math.inf).all())
            err = (o - want).abs()
            tol = (2.0 ** -10 + 2 * d * 2.0 ** -24 * big[..., None]) * mass + \
                HALF_ULP[out.dtype] * want.abs() + 2.0 ** -24
            assert bool((err <= tol)[:, ~none].all()), (b, float((err - tol)[:, ~none].max()))
            lerr = (l - want_lse).abs()[:, ~none]
            ltol = (d * 2.0 ** -24 * big + 2.0 ** -20 * (1 + want_lse.abs()))[:, ~none]
            assert bool((lerr <= ltol).all()), (b, float((lerr - ltol).max()))


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(2, 4), (1, 1), (3, 7), (1, 24)])
def test_single_token(name, d, heads, group):
    c = Case(name, d, heads, group, [0, 1, 15, 16, 17, 63, 333], 1)
    c.check(c.run())


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("draft,group", [(2, 4), (5, 3), (17, 2), (64, 1), (40, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_drafted_tokens_causal(name, d, draft, group, dtype):
    c = Case(name, d, 2, group, [0, 3, 130, 47], draft, page=32, dtype=dtype, seed=2)
    drafts = [draft, 1, max(1, draft - 1), 0]
    lens = torch.tensor(drafts, dtype=torch.int32, device="cuda")
    c.check(c.run(draft_lens=lens), drafts)


@pytest.mark.parametrize("name", RECIPES)
@pytest.mark.parametrize("draft", [3, 16, 33])
@pytest.mark.parametrize("shared", [False, True])
def test_trees_with_empty_rows(name, draft, shared):
    c = Case(name, 128, 2, 4, [0, 5, 96, 250], draft, seed=3)
    g = torch.Generator().manual_seed(4)
    tree = torch.rand(draft, draft, generator=g) < 0.4 if shared else \
        torch.rand(4, draft, draft, generator=g) < 0.4
    tree[..., 1, :] = False  # sees no drafted token; with no context, nothing
    tree = tree.cuda()
    c.check(c.run(tree_mask=tree), tree=tree)


@pytest.mark.parametrize("name", ["block4", "mx4", "nvfp4"])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_long_contexts_split_over_blocks(name, page):
    c = Case(name, 128, 2, 4, [9001, 40, 20011], 1, page=page, seed=5, spare_columns=3)
    c.check(c.run())


@pytest.mark.parametrize("name", RECIPES)
def test_values_and_keys_of_very_different_size(name):
    c = Case(name, 128, 2, 2, [700, 31], 2, seed=6, spread=4.0)
    c.check(c.run(scale=0.02), scale=0.02)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales(scale):
    c = Case("block4", 64, 1, 4, [100, 2], 3, seed=7)
    c.check(c.run(scale=scale), scale=scale)


def test_large_and_tiny_queries():
    c = Case("block4", 64, 1, 4, [50, 2], 1, seed=8)
    c.q[0, 0, 0] *= 2.0 ** 60
    c.q[0, 0, 1] *= 2.0 ** -60
    c.q[0, 0, 2] = 0
    out, lse = c.run(scale=2.0 ** -60)
    ref = Case("block4", 64, 1, 4, [50, 2], 1, seed=8)
    want, want_lse = ref.run(scale=1.0)
    assert torch.equal(out[0, 0, 0], want[0, 0, 0]) and torch.equal(lse[0, 0, 0], want_lse[0, 0, 0])
    assert torch.allclose(lse[0, 0, 1:3], torch.full((2,), math.log(51), device="cuda"), atol=1e-5)


@pytest.mark.parametrize("name", RECIPES)
def test_what_is_not_seen_does_not_reach_a_row(name):
    """NaN codes and scales behind the end of a page, in other pages, and in drafted tokens that a row does not
    see; and the rows that see them do get them."""
    d, draft = 128, 6
    c = Case(name, d, 2, 4, [21, 40], draft, seed=9)
    tree = torch.eye(draft, dtype=torch.bool, device="cuda").repeat(2, 1, 1)
    tree[:, :, 0] = True
    tree[:, 0, :] = False  # row 0 sees only the context
    drafts = torch.tensor([draft, 4], dtype=torch.int32, device="cuda")
    want = c.run(tree_mask=tree, draft_lens=drafts)
    c.check(want, [draft, 4], tree)
    # everything not written by the two sequences
    live = torch.zeros(c.cache.num_pages, c.cache.page_size, dtype=torch.bool, device="cuda")
    for b, n in enumerate((21 + draft, 40 + 4)):
        t = torch.arange(n, device="cuda")
        live[c.table[b].long()[t // 16], t % 16] = True
    for buf in c.cache._buffers:
        dead = (~live)[:, None, :, None].expand_as(buf)
        buf[dead] = float("nan") if buf.dtype == torch.float32 else 255
    got = c.run(tree_mask=tree, draft_lens=drafts)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # drafted token 3 of sequence 0 becomes NaN in its values, then in its keys
    page, at = int(c.table[0, 24 // 16]), 24 % 16
    for side in ("v", "k"):
        data, scale = getattr(c.cache, side + "_data"), getattr(c.cache, side + "_scale")
        keep = data[page, :, at].clone(), scale[page, :, at].clone()
        data[page, :, at] = 255
        scale[page, :, at] = float("nan") if scale.dtype == torch.float32 else 255
        out, lse = c.run(tree_mask=tree, draft_lens=drafts)
        others = [0, 1, 2, 4, 5]
        # the step is then summed in another order
        assert torch.allclose(out[0, others].float(), want[0][0, others].float(), rtol=2.0 ** -7, atol=1e-3)
        assert torch.allclose(lse[0, others], want[1][0, others], rtol=1e-5)
        assert torch.equal(out[1], want[0][1])
        if not (side == "k" and name.startswith("mx4")) or torch.isnan(out[0, 3]).all():
            assert torch.isnan(out[0, 3]).all()
        data[page, :, at], scale[page, :, at] = keep
    # one code only, where a code can be NaN
    if name != "nvfp4":
        c.cache.v_data[page, 1, at, 77] = 255
        out, _ = c.run(tree_mask=tree, draft_lens=drafts)
        bad = torch.isnan(out)
        assert bad[0, 3, 4:, 77].all() and int(bad.sum()) == 4


def test_pages_outside_the_cache_are_not_seen():
    c = Case("mx4", 128, 2, 4, [64, 50], 1, seed=10)
    c.table[0, 1] = -1
    c.table[0, 2] = c.cache.num_pages
    out, lse = c.run()
    # what is left: tokens 0..15, 48..63 and the new one
    k, v = c.cache.read(c.table, c.context + 1, 65, torch.float32)
    keep = torch.tensor(list(range(16)) + list(range(48, 65)), device="cuda")
    kk, vv = (x[0, keep].double().repeat_interleave(4, 1).transpose(0, 1) for x in (k, v))
    s = (c.q[0].double().transpose(0, 1) @ kk.transpose(1, 2)) * 128 ** -0.5
    want = (torch.softmax(s, -1) @ vv).transpose(0, 1)
    assert float((out[0].double() - want).abs().max()) <= 2.0 ** -8 * float(vv.abs().max())
    short = bb().cache_attention(c.q, c.cache, c.table[:, :1].contiguous(), c.context)
    full = Case("mx4", 128, 2, 4, [15, 15], 1, seed=11)
    assert torch.isfinite(short).all() and full.cache.num_pages


def test_infinite_lengths_are_bounded_by_the_table():
    c = Case("block4", 64, 1, 2, [31, 15], 1, seed=12)
    big = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    out, lse = bb().cache_attention(c.q, c.cache, c.table, big, return_lse=True)
    assert torch.isfinite(out[0]).all()
    # a negative context counts as none: the token sees itself, at the first place
    assert torch.isfinite(out[1]).all() and torch.isfinite(lse[1]).all()


def test_many_sequences():
    ctx = [(37 * i) % 91 for i in range(70)]
    c = Case("block4", 64, 2, 4, ctx, 1, seed=13)
    c.check(c.run())


def test_repeatable_other_stream_and_graph():
    c = Case("mx4", 128, 4, 4, [5000, 300], 1, page=64, seed=14)
    want = c.run()
    for _ in range(3):
        got = c.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q = c.q * 1
        got = bb().cache_attention(q, c.cache, c.table, c.context)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = bb().cache_attention(c.q, c.cache, c.table, c.context)
    c.context.copy_(torch.tensor([4000, 77], dtype=torch.int32))  # lengths are read by the replay
    graph.replay()
    assert torch.equal(held, c.run()[0])


def test_three_dimensional_and_strided_queries():
    c = Case("nvfp4", 64, 2, 4, [100, 7], 1, seed=15)
    want = c.run()[0]
    assert torch.equal(bb().cache_attention(c.q[:, 0], c.cache, c.table, c.context), want[:, 0])
    wide = torch.zeros(2, 1, 12, 64, dtype=c.q.dtype, device="cuda")
    wide[:, :, 2:10] = c.q
    assert torch.equal(bb().cache_attention(wide[:, :, 2:10], c.cache, c.table, c.context), want)


def test_empty():
    c = Case("mx4", 64, 2, 2, [4], 1, seed=16)
    out = bb().cache_attention(c.q[:0], c.cache, c.table[:0], c.context[:0])
    assert out.shape == (0, 1, 4, 64)
    out, lse = bb().cache_attention(c.q, c.cache, c.table[:, :0], c.context, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


def test_refusals():
    f = bb().cache_attention
    c = Case("mx4", 64, 2, 2, [4, 5], 3, seed=17)
    q, t, n = c.q, c.table, c.context
    with pytest.raises(TypeError):
        f(q.float(), c.cache, t, n)
    with pytest.raises(TypeError):
        f(q.cpu(), c.cache, t, n)
    with pytest.raises(TypeError):
        f(q, None, t, n)
    with pytest.raises(ValueError):
        f(q[..., :3, :], c.cache, t, n)
    with pytest.raises(ValueError):
        f(q[..., :32], c.cache, t, n)
    with pytest.raises(TypeError):
        f(q, c.cache, t.long(), n)
    with pytest.raises(ValueError):
        f(q, c.cache, t[:1], n)
    with pytest.raises(TypeError):
        f(q, c.cache, t, n.long())
    with pytest.raises(ValueError):
        f(q, c.cache, t, n[:1])
    with pytest.raises(ValueError):
        f(q, c.cache, t, n, draft_lens=n[:1])
    with pytest.raises(TypeError):
        f(q, c.cache, t, n, tree_mask=torch.ones(3, 3, device="cuda"))
    with pytest.raises(ValueError):
        f(q, c.cache, t, n, tree_mask=torch.ones(2, 3, dtype=torch.bool, device="cuda"))
    with pytest.raises(RuntimeError):
        f(q.requires_grad_(True), c.cache, t, n)
