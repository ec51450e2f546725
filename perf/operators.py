"""Cases that measure the operators of the attention block around a quantised key/value cache.

Four kinds of pass, each as a serving or training program makes it:

* ``norm_rope``  -- root-mean-square norm of every query and key head and the position rotation, one
  call; with ``grad`` the training step's forward and backward.
* ``write``      -- keys and values quantised into a paged cache; with ``read`` they are read back too;
  with ``fused`` the norm and rotation run in the same call (a serving step).
* ``read``       -- the cache of a batch read back as dense keys and values (a prefix that is reused).
* ``attend``     -- attention of one token, or of a tree of drafted tokens, over the paged cache.

Recipes: ``block`` (FP8, one float32 scale per token and head), ``mxfp8`` (FP8, one power of two per 32
elements) and ``nvfp4`` (4-bit, one FP8 scale per 16). The plain forms are elementary torch operations in
float32. Cache buffers are (pages, kv heads, page size, bytes per row) codes and (pages, kv heads, page
size, scales per row) scales.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FP8 = {"E4M3": torch.float8_e4m3fn, "E5M2": torch.float8_e5m2}
_FP8_MAX = {"E4M3": 448.0, "E5M2": 57344.0}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one token of one stream: the smallest call, launch latency is all of it
        dict(name="norm_rope_1", op="norm_rope", grad=False, tokens=1, hq=32, hkv=8, d=128, rot=128,
             dtype="bf16", wdtype="bf16", interleaved=False, packed=True),
        # a long prompt, heads taken as views of the packed q/k/v projection
        dict(name="norm_rope_16384", op="norm_rope", grad=False, tokens=16384, hq=32, hkv=8, d=128,
             rot=128, dtype="bf16", wdtype="bf16", interleaved=False, packed=True),
        # a training step's forward and backward, odd token count, float32 weights
        dict(name="norm_rope_grad_8191", op="norm_rope", grad=True, tokens=8191, hq=32, hkv=8, d=128,
             rot=128, dtype="bf16", wdtype="f32", interleaved=False, packed=True),
        # a small training step in float32, 64-wide heads, interleaved pairs, half of the head rotated
        dict(name="norm_rope_grad_f32_509", op="norm_rope", grad=True, tokens=509, hq=16, hkv=4, d=64,
             rot=32, dtype="f32", wdtype="f32", interleaved=True, packed=False),
        # a serving step of 64 streams: norm, rotation and the quantised write of one token each
        dict(name="write_step_64", op="write", fused=True, read=False, tokens=64, hq=32, hkv=8, d=128,
             rot=128, dtype="bf16", recipe="mxfp8", fmt="E4M3", page=16),
        # a prompt written to the cache in FP8 with one scale per token and head
        dict(name="write_16384", op="write", fused=False, read=False, tokens=16384, hkv=8, d=128,
             dtype="bf16", recipe="block", fmt="E4M3", page=64),
        # an odd prompt written in 4 bits and read back by the prompt's own attention
        dict(name="write_read_nvfp4_4095", op="write", fused=False, read=True, tokens=4095, hkv=4,
             d=256, dtype="f16", recipe="nvfp4", fmt="E4M3", page=32),
        # a shared prefix of a ragged batch read back as dense keys and values
        dict(name="read_mxfp8_8x4096", op="read", batch=8, length=4096, hkv=8, d=128, dtype="bf16",
             recipe="mxfp8", fmt="E4M3", page=32),
        # one stream, one token, a short odd context: latency
        dict(name="attend_1x1023", op="attend", batch=1, draft=1, tree=False, lse=False, ctx=1023, hq=32,
             hkv=8, d=128, dtype="bf16", recipe="block", fmt="E4M3", page=16),
        # a full serving batch of single tokens over ragged contexts
        dict(name="attend_64x8192", op="attend", batch=64, draft=1, tree=False, lse=False, ctx=8192,
             hq=32, hkv=8, d=128, dtype="bf16", recipe="mxfp8", fmt="E4M3", page=64),
        # two long contexts in 4 bits, 8 query heads per key/value head
        dict(name="attend_2x131072_nvfp4", op="attend", batch=2, draft=1, tree=False, lse=True,
             ctx=131072, hq=64, hkv=8, d=128, dtype="bf16", recipe="nvfp4", fmt="E4M3", page=64),
        # large trees of drafted tokens over long contexts: the matrix products count
        dict(name="attend_tree_8x64x16384", op="attend", batch=8, draft=64, tree=True, lse=False,
             ctx=16384, hq=64, hkv=8, d=128, dtype="bf16", recipe="block", fmt="E4M3", page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _not(n, bad=3072):
    return n + 1 if n == bad else n


def draw(rng):
    """One more case of the ranges above: one token to long prompts and contexts, every recipe, both FP8
    formats, three head sizes, the head counts of dense, grouped and single key/value heads."""
    hq, hkv = rng.choice([(32, 8), (16, 4), (64, 8), (8, 8), (16, 2), (8, 1)])
    d = rng.choice([64, 128, 128, 256])
    recipe, fmt = rng.choice([("block", "E4M3"), ("block", "E5M2"), ("mxfp8", "E4M3"),
                              ("mxfp8", "E5M2"), ("nvfp4", "E4M3")])
    dtype, page = rng.choice(["bf16", "bf16", "f16"]), rng.choice([16, 32, 64, 128])
    op = rng.choice(["norm_rope", "norm_rope_grad", "write", "write_fused", "read", "attend", "attend",
                     "attend_tree", "attend_tree"])
    room = 32 * 128 * 16384 / (hq * d)  # tokens, so that q stays within the largest listed case's
    if op == "norm_rope":
        return dict(op="norm_rope", grad=False, tokens=_not(_log(rng, 1, min(16384, room))), hq=hq,
                    hkv=hkv, d=d, rot=rng.choice([d, d // 2]), dtype=rng.choice([dtype, "f32"]),
                    wdtype=rng.choice(["f32", "bf16"]), interleaved=rng.random() < 0.5,
                    packed=rng.random() < 0.7)
    if op == "norm_rope_grad":
        return dict(op="norm_rope", grad=True, tokens=_not(_log(rng, 64, min(8191, room / 4))), hq=hq,
                    hkv=hkv, d=d, rot=rng.choice([d, d // 2]), dtype=rng.choice([dtype, "f32"]),
                    wdtype="f32", interleaved=rng.random() < 0.5, packed=rng.random() < 0.7)
    if op == "write_fused":  # a power-of-two scale: a last-bit difference of the norm cannot move it
        return dict(op="write", fused=True, read=False, tokens=_not(_log(rng, 1, 512)), hq=hq, hkv=hkv,
                    d=d, rot=rng.choice([d, d // 2]), dtype=dtype, recipe="mxfp8", fmt=fmt, page=page)
    if op == "write":
        return dict(op="write", fused=False, read=recipe == "nvfp4" or rng.random() < 0.5,
                    tokens=_not(_log(rng, 1, min(16384, 8 * 128 * 16384 / (hkv * d)))), hkv=hkv, d=d,
                    dtype=dtype, recipe=recipe, fmt=fmt, page=page)
    if op == "read":
        length = _log(rng, 16, 8192)
        most = 8 * 4096 * 8 * 128 / (length * hkv * d)
        return dict(op="read", batch=_log(rng, 1, max(1, min(64, most))), length=_not(length), hkv=hkv,
                    d=d, dtype=dtype, recipe=recipe, fmt=fmt, page=page)
    if op == "attend":
        ctx = _log(rng, 1, 131072)
        most = 64 * 8192 * 8 * 128 / (ctx * hkv * d) / 2
        return dict(op="attend", batch=_log(rng, 1, max(1, min(64, most))), draft=1, tree=False,
                    lse=rng.random() < 0.5, ctx=_not(ctx), hq=hq, hkv=hkv, d=d, dtype=dtype,
                    recipe=recipe, fmt=fmt, page=page)
    ctx, nodes = _log(rng, 1, 32768), _log(rng, 2, 64)
    most = min(64 * 8192 * 8 * 128 / (ctx * hkv * d) / 2, 8 * 64 * 64 * 16384 * 128 / (ctx * nodes * hq * d) / 2)
    return dict(op="attend", batch=_log(rng, 1, max(1, min(32, most))), draft=nodes, tree=rng.random() < 0.8,
                lse=rng.random() < 0.5, ctx=_not(ctx), hq=hq, hkv=hkv, d=d, dtype=dtype, recipe=recipe,
                fmt=fmt, page=page)


def _row(case):
    """(code bytes, scales, bytes per scale) of one cached row."""
    d = case["d"]
    return {"block": (d, 1, 4), "mxfp8": (d, d // 32, 1), "nvfp4": (d // 2, d // 16, 1)}[case["recipe"]]


def _row_bytes(case):
    c, n, b = _row(case)
    return c + n * b


def _contexts(case):
    """Tokens in the cache before the drafted ones, per stream: ragged, the first the longest."""
    n = case["ctx"] if case["op"] == "attend" else case["length"]
    return [n - (b * 7919) % (n // 2 + 1) for b in range(case["batch"])]


def _drafts(case):
    t = case["draft"]
    return [t - (b * 3) % ((t + 1) // 2) for b in range(case["batch"])]


def work(case):
    d, e = case["d"], _DT[case["dtype"]].itemsize
    if case["op"] == "norm_rope":
        q = case["tokens"] * (case["hq"] + case["hkv"]) * d
        t = case["tokens"] * case["rot"] * 4
        # forward: one read, one write; backward: x and its gradient read, one gradient written
        return {"bytes": q * e * (5 if case["grad"] else 2) + t, "flops": q * (25 if case["grad"] else 8)}
    if case["op"] == "write":
        n = case["tokens"] * case["hkv"]
        by, fl = 2 * n * (d * e + _row_bytes(case)), 2 * n * d * 6
        if case["fused"]:
            by += 2 * case["tokens"] * case["hq"] * d * e + case["tokens"] * case["rot"] * 4
            fl += case["tokens"] * (case["hq"] + case["hkv"]) * d * 8
        if case["read"]:
            by += 2 * n * (_row_bytes(case) + d * e)
        return {"bytes": by, "flops": fl}
    ctx = _contexts(case)
    if case["op"] == "read":
        n = sum(ctx) * case["hkv"]
        m = case["batch"] * max(ctx) * case["hkv"]
        return {"bytes": 2 * (n * _row_bytes(case) + m * d * e), "flops": 2 * n * d}
    dr = _drafts(case)
    tokens = sum(c + t for c, t in zip(ctx, dr)) * case["hkv"]
    rows = case["batch"] * case["draft"] * case["hq"]
    by = tokens * 2 * _row_bytes(case) + rows * d * e * 2 + (rows * 4 if case["lse"] else 0)
    return {"bytes": by, "flops": sum(4 * d * case["hq"] * t * (c + t / 2) for c, t in zip(ctx, dr))}


# ------------------------------------------------------------------ inputs


def _tables(positions, rot, dev):
    f = torch.arange(rot // 2, device=dev, dtype=torch.float64) * (-2.0 / rot)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * (10000.0 ** f)[None]
    return a.cos().float(), a.sin().float()


def _paged_codes(case, g, pages):
    """A cache that holds keys or values: normal values with a spread per channel, quantised. Made in pieces,
    since a whole cache in float32 is several times its size."""
    c, n, _ = _row(case)
    h, s, d = case["hkv"], case["page"], case["d"]
    data = torch.empty(pages, h, s, c, dtype=torch.uint8, device="cuda")
    scale = torch.empty(pages, h, s, n, dtype=torch.float32 if case["recipe"] == "block" else torch.uint8,
                        device="cuda")
    spread = torch.rand(h, 1, d, generator=g, device="cuda") * 1.5 + 0.25
    step = max(1, (1 << 26) // (h * s * d))
    for at in range(0, pages, step):
        m = min(step, pages - at)
        x = torch.randn(m, h, s, d, generator=g, device="cuda") * spread
        codes, sc = _quantise(x, case["recipe"], case["fmt"])
        data[at:at + m] = codes
        scale[at:at + m] = sc
    return data, scale


def _empty_cache(case, pages):
    c, n, _ = _row(case)
    h, s = case["hkv"], case["page"]
    st = torch.float32 if case["recipe"] == "block" else torch.uint8
    return {k: torch.zeros(pages, h, s, c if "data" in k else n, device="cuda",
                           dtype=torch.uint8 if "data" in k else st)
            for k in ("k_data", "k_scale", "v_data", "v_scale")}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    st = dict(case)
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "norm_rope" or case.get("fused"):
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        if case.get("packed", True):
            qkv = (normal(t, hq + 2 * hkv, d) * 1.7).to(dt)
            st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            st["q"], st["k"] = (normal(t, hq, d) * 1.7).to(dt), (normal(t, hkv, d) * 1.7).to(dt)
        wd = _DT[case.get("wdtype", "bf16")]
        st["wq"], st["wk"] = (1 + 0.2 * normal(d)).to(wd), (1 + 0.2 * normal(d)).to(wd)
        top = max(t, 4096)
        st["cos"], st["sin"] = _tables(top, case["rot"], "cuda")
        st["positions"] = (torch.arange(t, device="cuda") if case["op"] == "norm_rope" else
                           torch.randint(0, top, (t,), generator=g, device="cuda"))
        if case.get("grad"):
            st["gq"], st["gk"] = normal(t, hq, d).to(dt), normal(t, hkv, d).to(dt)
            for k in ("q", "k", "wq", "wk"):
                st[k] = st[k].detach().requires_grad_(True)
    if case["op"] == "write":
        t, s = case["tokens"], case["page"]
        if not case["fused"]:
            st["k"], st["v"] = normal(t, case["hkv"], case["d"]).to(dt), normal(t, case["hkv"], case["d"]).to(dt)
        pages = -(-t // s) + 3
        st.update(_empty_cache(case, pages))
        order = torch.randperm(pages, generator=g, device="cuda")
        if case["fused"]:  # one token of each stream, anywhere in its page
            st["slots"] = torch.randperm(pages * s, generator=g, device="cuda")[:t]
        else:  # one stream's tokens, page after page
            at = torch.arange(t, device="cuda")
            st["slots"] = order[at // s] * s + at % s
        st["table"] = order[None, :-(-t // s)].to(torch.int32)
        st["lengths"] = torch.tensor([t], dtype=torch.int32, device="cuda")
        st["longest"] = t
    if case["op"] in ("read", "attend"):
        s, ctx = case["page"], _contexts(case)
        dr = _drafts(case) if case["op"] == "attend" else [0] * case["batch"]
        need = [-(-(c + t) // s) for c, t in zip(ctx, dr)]
        pages = sum(need) + 2
        st["k_data"], st["k_scale"] = _paged_codes(case, g, pages)
        st["v_data"], st["v_scale"] = _paged_codes(case, g, pages)
        order = torch.randperm(pages, generator=g, device="cuda").cpu()
        table = torch.full((case["batch"], max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        st["table"] = table.cuda()
        st["lengths"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        st["longest"] = max(ctx)
        if case["op"] == "attend":
            st["q"] = normal(case["batch"], case["draft"], case["hq"], case["d"]).to(dt)
            st["drafts"] = torch.tensor(dr, dtype=torch.int32, device="cuda")
            st["tree"] = None
            if case["tree"]:
                t = case["draft"]
                parent = (torch.rand(case["batch"], t, generator=g, device="cuda").cpu() *
                          torch.arange(t)).long()
                sees = torch.eye(t, dtype=torch.bool).repeat(case["batch"], 1, 1)
                b = torch.arange(case["batch"])
                for i in range(1, t):  # a node sees itself and what its parent sees
                    sees[:, i] |= sees[b, parent[:, i]]
                st["tree"] = sees.cuda()
    return st


# ------------------------------------------------------------------ plain forms


def _pow2(e):
    """2^e of whole numbers, from the bits (a power function may be a last bit off); e in -126..127."""
    return ((e.clamp(-126, 127).to(torch.int32) + 127) << 23).view(torch.float32)


def _to_grid(v, mantissa, least, most):
    """|v| saturated at `most`, to the nearest value with so many mantissa bits (exponents from `least` on);
    halves go toward zero. Signs are kept, and every step is exact in float32."""
    a = v.abs().clamp(max=most)
    _, e = torch.frexp(a)  # a = m 2^e, 1/2 <= m < 1
    e = (e - 1).clamp(min=least) - mantissa
    r = torch.ceil(a * _pow2(-e) - 0.5)
    return torch.copysign(r * _pow2(e), v) + 0.0


_GRID = {"E4M3": (3, -6, 448.0), "E5M2": (2, -14, 57344.0), "E2M1": (1, 0, 6.0)}


def _nibbles(val):
    """E2M1 values to codes, two to a byte, the even element in the low half."""
    m = val.abs()
    code = (2 * m.clamp(max=2) + (m - 2).clamp(0, 2) + (m - 4).clamp(0, 2) / 2).to(torch.uint8)
    code = torch.where(val < 0, code + 8, code)
    return code[..., 0::2] + code[..., 1::2] * 16


def _quantise(x, recipe, fmt):
    """Code bytes and scales of float32 rows (..., d)."""
    d = x.shape[-1]
    block = {"block": d, "mxfp8": 32, "nvfp4": 16}[recipe]
    y = x.reshape(*x.shape[:-1], d // block, block)
    amax = y.abs().amax(-1).clamp(min=1e-10)
    if recipe == "nvfp4":
        s = _to_grid(amax / 6.0, *_GRID["E4M3"])
        val = _to_grid(y / s.clamp(min=2.0 ** -9)[..., None], *_GRID["E2M1"]).reshape(x.shape)
        return _nibbles(val), s.to(_FP8["E4M3"]).view(torch.uint8)
    s = amax / _FP8_MAX[fmt]
    kept = s
    if recipe == "mxfp8":
        e = torch.round(torch.log2(s.double())).to(torch.int32)
        s = _pow2(e)
        kept = (e + 127).to(torch.uint8)
    val = _to_grid(y / s[..., None], *_GRID[fmt]).reshape(x.shape)
    return val.to(_FP8[fmt]).view(torch.uint8), kept


def _decode(data, scale, st):
    """float32 values (..., d) of code bytes and scales."""
    if st["recipe"] == "nvfp4":
        lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=data.device)
        v = torch.stack([lut[(data & 15).long()], lut[(data >> 4).long()]], -1).flatten(-2)
        s = scale.view(_FP8["E4M3"]).float()
    else:
        v = data.view(_FP8[st["fmt"]]).float()
        s = scale if st["recipe"] == "block" else _pow2(scale.to(torch.int32) - 127)
    n = s.shape[-1]
    return (v.reshape(*v.shape[:-1], n, -1) * s[..., None]).reshape(v.shape)


def _rotate(y, cos, sin, rot, interleaved, back=False):
    """The first `rot` values of every head turned by the token's angles (or back)."""
    if back:
        sin = -sin
    c, s = cos[:, None], sin[:, None]
    z = y.clone()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        z[..., 0:rot:2], z[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        z[..., :rot // 2], z[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return z


_EPS = 1e-6


def _norm_rope(x, w, st):
    x, w = x.detach().float(), w.detach().float()
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    p = st["positions"]
    return _rotate(x * r * w, st["cos"][p], st["sin"][p], st["rot"], st.get("interleaved", False))


def _norm_rope_back(x, w, gy, st):
    x, w, p = x.detach().float(), w.detach().float(), st["positions"]
    gz = _rotate(gy.float(), st["cos"][p], st["sin"][p], st["rot"], st["interleaved"], back=True)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    n = x * r
    h = gz * w
    return r * (h - n * (h * n).mean(-1, keepdim=True)), (gz * n).sum((0, 1))


def _store(st, k, v):
    page, at = st["slots"] // st["page"], st["slots"] % st["page"]
    for name, x in (("k", k), ("v", v)):
        codes, scale = _quantise(x.float(), st["recipe"], st["fmt"])
        st[name + "_data"][page, :, at] = codes
        st[name + "_scale"][page, :, at] = scale


def _held(st):
    """The cache as the values that it stands for: FP8 codes and power-of-two scales as those types."""
    r = {"k_data": st["k_data"].view(_FP8[st["fmt"]]), "v_data": st["v_data"].view(_FP8[st["fmt"]])}
    for k in ("k_scale", "v_scale"):
        r[k] = st[k] if st["recipe"] == "block" else st[k].view(torch.float8_e8m0fnu)
    return r


def _dense(st, which, length):
    """(batch, kv heads, length, d) float32 of the paged rows; what no table entry covers is whatever page 0 holds."""
    t = st["table"].clamp(min=0).long()
    data, scale = st[which + "_data"][t], st[which + "_scale"][t]  # (batch, pages, heads, page, ...)
    x = _decode(data, scale, st).transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])[:, :, :length]


def _read(st):
    n = st["longest"]
    live = (torch.arange(n, device="cuda")[None] < st["lengths"][:, None])[:, None, :, None]
    dt = _DT[st["dtype"]]
    return tuple(torch.where(live, _dense(st, w, n), 0.0).to(dt).transpose(1, 2) for w in ("k", "v"))


def _attend(st):
    q = st["q"].float()
    b, t, hq, d = q.shape
    g = hq // st["hkv"]
    n = st["table"].shape[1] * st["page"]
    k, v = _dense(st, "k", n), _dense(st, "v", n)
    at = torch.arange(n, device="cuda")[None] - st["lengths"][:, None]  # of the drafted tokens, from 0 on
    node, drafts = torch.arange(t, device="cuda"), st["drafts"]
    tree = st["tree"] if st["tree"] is not None else (node[:, None] >= node[None]).expand(b, t, t)
    seen = torch.gather(tree, 2, at.clamp(0, t - 1)[:, None].expand(b, t, n))
    seen = (at < 0)[:, None] | (seen & ((at >= 0) & (at < drafts[:, None]))[:, None])
    seen = seen & (node[None] < drafts[:, None])[:, :, None]  # (b, t, n)
    v = torch.where(seen.any(1)[:, None, :, None], v, 0.0)
    q = q.reshape(b, t, st["hkv"], g, d).permute(0, 2, 3, 1, 4).reshape(b, st["hkv"], g * t, d)
    s = (q @ k.transpose(2, 3)).reshape(b, st["hkv"], g, t, n) * (1 / math.sqrt(d))
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(b, st["hkv"], g * t, n) @ v).reshape(b, st["hkv"], g, t, d)
    o = o / torch.where(total == 0, 1.0, total)
    out = o.permute(0, 3, 1, 2, 4).reshape(b, t, hq, d).to(st["q"].dtype)
    if not st["lse"]:
        return out
    return out, (m + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(b, t, hq)


# ------------------------------------------------------------------ one pass


def _cache(st):
    """The handle of the cache that a serving program keeps beside its buffers."""
    import breccia_b200 as bb
    if "cache" not in st:
        recipe = {"block": lambda: bb.Float8BlockScaling(st["fmt"], block_k=st["d"]),
                  "mxfp8": lambda: bb.MXFP8BlockScaling(st["fmt"]),
                  "nvfp4": lambda: bb.NVFP4BlockScaling()}[st["recipe"]]()
        st["cache"] = bb.QuantizedKVCache.from_buffers(st["k_data"], st["k_scale"], st["v_data"],
                                                       st["v_scale"], recipe)
    return st["cache"]


def run(state):
    st = state
    if own:
        import breccia_b200 as bb
    if st["op"] == "norm_rope":
        if own:
            q, k = bb.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], st["positions"],
                                   eps=_EPS, interleaved=st["interleaved"])
            if not st["grad"]:
                return q, k
            return q, k, *torch.autograd.grad((q, k), (st["q"], st["k"], st["wq"], st["wk"]),
                                              (st["gq"], st["gk"]))
        dt = st["q"].dtype
        q, k = _norm_rope(st["q"], st["wq"], st).to(dt), _norm_rope(st["k"], st["wk"], st).to(dt)
        if not st["grad"]:
            return q, k
        gq, gwq = _norm_rope_back(st["q"], st["wq"], st["gq"], st)
        gk, gwk = _norm_rope_back(st["k"], st["wk"], st["gk"], st)
        return q, k, gq.to(dt), gk.to(dt), gwq.to(st["wq"].dtype), gwk.to(st["wk"].dtype)
    if st["op"] == "write":
        out = {}
        if own:
            if st["fused"]:
                out["q"] = bb.qk_norm_rope_write(st["q"], st["k"], st["v"], st["wq"], st["wk"], st["cos"],
                                                 st["sin"], st["positions"], _cache(st), st["slots"], eps=_EPS)
            else:
                _cache(st).write(st["k"], st["v"], st["slots"])
            if st["read"]:
                out["k"], out["v"] = _cache(st).read(st["table"], st["lengths"], st["longest"],
                                                     out_dtype=st["k"].dtype)
                return out
            return {**out, **_held(st)}
        k = st["k"]
        if st["fused"]:
            out["q"] = _norm_rope(st["q"], st["wq"], st).to(k.dtype)
            k = _norm_rope(k, st["wk"], st).to(k.dtype)
        _store(st, k, st["v"])
        if st["read"]:
            out["k"], out["v"] = _read(st)
            return out
        return {**out, **_held(st)}
    if st["op"] == "read":
        if own:
            return _cache(st).read(st["table"], st["lengths"], st["longest"], out_dtype=_DT[st["dtype"]])
        return _read(st)
    if own:
        return bb.cache_attention(st["q"], _cache(st), st["table"], st["lengths"], draft_lens=st["drafts"],
                                  tree_mask=st["tree"], return_lse=st["lse"])
    return _attend(st)


# ------------------------------------------------------------------ the definitions in 64 bits


def _two_to(e):
    """2^e of whole numbers in 64 bits, from the bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _fp8_values(fmt):
    bits, bias = (3, 7) if fmt == "E4M3" else (2, 15)
    def one(c):
        e, m = (c & 127) >> bits, c & ((1 << bits) - 1)
        v = math.ldexp(m, 1 - bias - bits) if e == 0 else math.ldexp((1 << bits) + m, e - bias - bits)
        if fmt == "E4M3" and c & 127 == 127:
            v = math.nan
        if fmt == "E5M2" and e == 31:
            v = math.nan if m else math.inf
        return -v if c & 128 else v
    return torch.tensor([one(c) for c in range(256)], dtype=torch.float64, device="cuda")


def _values64(data, scale, case):
    """Rows of one stream, (..., bytes) and (..., scales), as 64-bit values."""
    if case["recipe"] == "nvfp4":
        mag = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
        both = torch.cat([mag, -mag])
        x = torch.empty(*data.shape[:-1], 2 * data.shape[-1], dtype=torch.float64, device="cuda")
        x[..., 0::2], x[..., 1::2] = both[(data % 16).int()], both[(data // 16).int()]
        s = _fp8_values("E4M3")[scale.int()]
    else:
        x = _fp8_values(case["fmt"])[data.int()]
        s = scale.double() if case["recipe"] == "block" else _two_to(scale.int() - 127)
    return x * s.repeat_interleave(x.shape[-1] // s.shape[-1], -1)


def _norm_rope64(x, w, st, case):
    """The norm and the rotation, pairs as complex numbers."""
    y = torch.nn.functional.rms_norm(x, (case["d"],), w, _EPS)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"]][:, None]
    r = case["rot"]
    pairs = y[..., :r].unflatten(-1, (r // 2, 2)) if case.get("interleaved") else \
        y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
    z = z.flatten(-2) if case.get("interleaved") else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, y[..., r:]], -1)


def _nearest64(v, values):
    """The nearest of the format's values, halves toward zero."""
    values = values[torch.isfinite(values) & (values >= 0)].unique()
    mid = (values[1:] + values[:-1]) / 2
    a = v.abs().clamp(max=float(values[-1]))
    return torch.sign(v) * values[torch.searchsorted(mid, a)]  # a on a midpoint keeps the lower value


def _held64(x, case):
    """(values of the codes, scales) of rows x in 64 bits."""
    top = {"block": _FP8_MAX[case["fmt"]], "mxfp8": _FP8_MAX[case["fmt"]], "nvfp4": 6.0}[case["recipe"]]
    n = {"block": case["d"], "mxfp8": 32, "nvfp4": 16}[case["recipe"]]
    y = x.unflatten(-1, (-1, n))
    s = y.abs().amax(-1, keepdim=True).clamp(min=1e-10) / top
    if case["recipe"] == "mxfp8":
        s = _two_to(torch.round(torch.log2(s)))
    if case["recipe"] == "nvfp4":
        s = _nearest64(s, _fp8_values("E4M3"))
        grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
        return _nearest64(y / s.clamp(min=2.0 ** -9), grid).flatten(-2), s[..., 0]
    return _nearest64(y / s, _fp8_values(case["fmt"])).flatten(-2), s[..., 0]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "norm_rope":
        leaf = [st[k].detach().double().requires_grad_(case["grad"]) for k in ("q", "k", "wq", "wk")]
        q, k = _norm_rope64(leaf[0], leaf[2], st, case), _norm_rope64(leaf[1], leaf[3], st, case)
        if not case["grad"]:
            return q, k
        back = torch.autograd.grad((q, k), leaf, (st["gq"].double(), st["gk"].double()))
        return q.detach(), k.detach(), *back
    if case["op"] == "write":
        k, v, out = st["k"].double(), st["v"].double(), {}
        if case["fused"]:
            out["q"] = _norm_rope64(st["q"].double(), st["wq"].double(), st, case)
            k = _norm_rope64(k, st["wk"].double(), st, case).to(_DT[case["dtype"]]).double()
        if case["read"]:
            for name, x in (("k", k), ("v", v)):
                val, s = _held64(x, case)
                out[name] = (val * s.repeat_interleave(case["d"] // s.shape[-1], -1))[None]
            return out
        for name, x in (("k", k), ("v", v)):
            val, s = _held64(x, case)
            for part, y in (("_data", val), ("_scale", s)):
                # a byte of zero stands for 0, or as a power-of-two scale for 2^-127
                empty = 2.0 ** -127 if part == "_scale" and case["recipe"] == "mxfp8" else 0.0
                whole = torch.full(st[name + part].shape, empty, dtype=torch.float64, device="cuda")
                whole[st["slots"] // case["page"], :, st["slots"] % case["page"]] = y
                out[name + part] = whole
        return out
    table, rows = st["table"].cpu(), []
    if case["op"] == "attend" and work(case)["flops"] > 6e11:
        return None
    for b, n in enumerate(_contexts(case)):
        t = _drafts(case)[b] if case["op"] == "attend" else 0
        used = table[b, :-(-(n + t) // case["page"])].long().cuda()
        k, v = (_values64(st[w + "_data"][used], st[w + "_scale"][used], case).transpose(0, 1).flatten(1, 2)
                [:, :n + t] for w in ("k", "v"))
        if case["op"] == "read":
            rows.append([torch.nn.functional.pad(x.transpose(0, 1), (0, 0, 0, 0, 0, st["longest"] - n))
                         for x in (k, v)])
            continue
        q = st["q"][b].double().unflatten(1, (case["hkv"], -1))[:t]  # (t, kv heads, group, d)
        s = torch.einsum("thgd,hnd->hgtn", q, k) / math.sqrt(case["d"])
        hidden = torch.ones(t, t, dtype=torch.bool, device="cuda").tril().logical_not() \
            if st["tree"] is None else ~st["tree"][b, :t, :t]
        s[..., n:].masked_fill_(hidden, -math.inf)
        lse = torch.logsumexp(s, -1)
        o = torch.einsum("hgtn,hnd->thgd", torch.exp(s - lse[..., None]), v).flatten(1, 2)
        pad = case["draft"] - t
        rows.append([torch.nn.functional.pad(o, (0, 0, 0, 0, 0, pad)),
                     torch.nn.functional.pad(lse.permute(2, 0, 1).flatten(1), (0, 0, 0, pad), value=-math.inf)])
    both = [torch.stack(x) for x in zip(*rows)]
    if case["op"] == "read":
        return tuple(both)
    return tuple(both) if case["lse"] else both[0]
