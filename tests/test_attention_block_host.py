"""Host-side checks of the attention block's entry points: they refuse bad
arguments, and return for empty ones, before any CUDA call (no GPU here)."""

import ctypes

import pytest
import torch

import breccia_b200 as bb
from breccia_b200 import _lib

OK, NULL, SHAPE, ALIGN = _lib.BRC_OK, _lib.BRC_ERR_NULL, _lib.BRC_ERR_SHAPE, _lib.BRC_ERR_ALIGN
DTYPE, UNSUPPORTED, RANGE = _lib.BRC_ERR_DTYPE, _lib.BRC_ERR_UNSUPPORTED, _lib.BRC_ERR_RANGE

_RAW = (ctypes.c_uint8 * 512)()
P = ctypes.addressof(_RAW) + (-ctypes.addressof(_RAW) % 16)  # host memory: never read


def rope(**kw):
    a = _lib.NormRope(q=P, k=P, q_token=512, q_head=128, k_token=256, k_head=128, wq=P, wk=P, cos=P,
                      sin=P, positions=P, tokens=3, table_rows=8, hq=4, hk=2, d=128, rot=128,
                      dtype=_lib.DTYPE_BF16, w_dtype=_lib.DTYPE_F32, index64=1, interleaved=0,
                      eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def cache(**kw):
    c = _lib.KvCache(k_data=P, k_scale=P, v_data=P, v_scale=P, num_pages=4, heads=2, page_size=16,
                     head_dim=128, kind=_lib.STE_MXFP8, fmt=_lib.FP8_E4M3)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_ROPE = [
    (dict(q=None), NULL), (dict(wk=None), NULL), (dict(positions=None), NULL), (dict(cos=None), NULL),
    (dict(dtype=3), DTYPE), (dict(w_dtype=-1), DTYPE), (dict(tokens=-1), SHAPE), (dict(hq=-1), SHAPE),
    (dict(d=120), SHAPE), (dict(d=272), SHAPE), (dict(rot=8), SHAPE), (dict(rot=144), SHAPE),
    (dict(table_rows=0), SHAPE), (dict(q=P + 2), ALIGN), (dict(sin=P + 4), ALIGN),
    (dict(q_head=130), ALIGN), (dict(k_token=260), ALIGN),
]

BAD_CACHE = [
    (dict(k_data=None), NULL), (dict(v_scale=None), NULL), (dict(kind=7), DTYPE), (dict(fmt=2), DTYPE),
    (dict(num_pages=0), SHAPE), (dict(heads=0), SHAPE), (dict(page_size=24), SHAPE),
    (dict(page_size=8), SHAPE), (dict(head_dim=96), UNSUPPORTED), (dict(v_data=P + 8), ALIGN),
]


def norm(L, a):
    return L.brc_qk_norm_rope(ctypes.addressof(a) if a else None, P, P, None)


def norm_bwd(L, a, ws=P, n=1 << 40, gq=P, gk_token=256):
    return L.brc_qk_norm_rope_bwd(ctypes.addressof(a) if a else None, gq, P, 512, 128, gk_token, 128, P,
                                  P, P, P, ws, n, None)


def norm_write(L, a, c, v=P, v_token=256, slots=P, q_out=P):
    return L.brc_qk_norm_rope_write(ctypes.addressof(a) if a else None, v, v_token, 128, q_out,
                                    ctypes.addressof(c) if c else None, slots, 1, None)


def write(L, c, k=P, dtype=_lib.DTYPE_BF16, tokens=3, k_token=256, slots=P):
    return L.brc_kv_write(ctypes.addressof(c) if c else None, k, P, dtype, tokens, k_token, 128, 256,
                          128, slots, 0, None)


def read(L, c, table=P, pages=2, lengths=P, batch=1, length=5, out=P, dtype=_lib.DTYPE_BF16):
    return L.brc_kv_read(ctypes.addressof(c) if c else None, table, pages, pages, lengths, batch, length,
                         out, P, dtype, None)


def attend(L, c, q=P, dtype=_lib.DTYPE_BF16, batch=2, draft=3, hq=4, table=P, pages=2, context=P,
           tree_stride=0, out=P, ws=P, n=1 << 40):
    return L.brc_kv_attention(ctypes.addressof(c) if c else None, q, dtype, batch, draft, hq, table,
                              pages, pages, context, None, None, tree_stride, 0.1, out, None, ws, n, None)


@pytest.mark.parametrize("kw,want", BAD_ROPE, ids=str)
def test_norm_rope_arguments(kw, want):
    L, a = _lib.lib(), rope(**kw)
    assert norm(L, a) == want
    assert norm_bwd(L, a) == want
    assert norm_write(L, a, cache()) == want


def test_norm_rope_outputs():
    L = _lib.lib()
    assert norm(L, None) == norm_bwd(L, None) == norm_write(L, None, cache()) == NULL
    assert L.brc_qk_norm_rope(ctypes.addressof(rope()), None, P, None) == NULL
    assert L.brc_qk_norm_rope(ctypes.addressof(rope()), P + 8, P, None) == ALIGN
    assert norm_bwd(L, rope(), ws=None) == NULL
    assert norm_bwd(L, rope(), gq=None) == NULL
    assert norm_bwd(L, rope(), gk_token=4) == ALIGN
    assert norm_bwd(L, rope(), gq=P + 2) == ALIGN
    assert L.brc_qk_norm_rope_bwd_workspace(8) == L.brc_qk_norm_rope_bwd_workspace(512) == 0


def test_empty_norm_rope():
    L = _lib.lib()
    for a in (rope(tokens=0), rope(hq=0, hk=0, q=None, k=None)):
        assert norm(L, a) == OK
    assert norm_write(L, rope(tokens=0), cache()) == OK


@pytest.mark.parametrize("kw,want", BAD_CACHE, ids=str)
def test_cache_arguments(kw, want):
    L, c = _lib.lib(), cache(**kw)
    assert write(L, c) == want
    assert read(L, c) == want
    assert attend(L, c) == want
    assert norm_write(L, rope(hk=2), c) == want
    assert L.brc_kv_attention_workspace(ctypes.addressof(c), 1, 1, 4) == 0


def test_write_and_read():
    L, c = _lib.lib(), cache()
    assert write(L, None) == read(L, None) == NULL
    assert write(L, c, k=None) == write(L, c, slots=None) == NULL
    assert write(L, c, dtype=5) == DTYPE and write(L, c, tokens=-1) == SHAPE
    assert write(L, c, k=P + 4) == write(L, c, k_token=257) == ALIGN
    assert write(L, c, tokens=1 << 33) == RANGE
    assert write(L, c, tokens=0, k=None, slots=None) == OK
    assert read(L, c, table=None) == read(L, c, lengths=None) == read(L, c, out=None) == NULL
    assert read(L, c, batch=-1) == read(L, c, length=-1) == read(L, c, pages=-1) == SHAPE
    assert read(L, c, dtype=3) == DTYPE and read(L, c, out=P + 8) == ALIGN
    assert read(L, c, length=1 << 31) == read(L, c, batch=1 << 10, length=1 << 30) == RANGE
    assert read(L, c, batch=0) == read(L, c, length=0) == OK


def test_write_after_norm():
    L, c = _lib.lib(), cache()
    assert norm_write(L, rope(), None) == NULL
    assert norm_write(L, rope(dtype=_lib.DTYPE_F32, q_token=512), c) == DTYPE
    assert norm_write(L, rope(hk=1), c) == norm_write(L, rope(d=64, rot=64), c) == SHAPE
    for kw in (dict(v=None), dict(slots=None), dict(q_out=None)):
        assert norm_write(L, rope(), c, **kw) == NULL
    assert norm_write(L, rope(), c, v=P + 2) == norm_write(L, rope(), c, v_token=129) == ALIGN


def test_attention():
    L, c = _lib.lib(), cache()
    assert attend(L, None) == NULL
    for kw in (dict(q=None), dict(context=None), dict(out=None), dict(ws=None), dict(table=None)):
        assert attend(L, c, **kw) == NULL
    for kw in (dict(batch=-1), dict(draft=-1), dict(hq=0), dict(hq=3), dict(pages=-1), dict(tree_stride=-1)):
        assert attend(L, c, **kw) == SHAPE
    assert attend(L, c, dtype=_lib.DTYPE_F32) == DTYPE
    for kw in (dict(q=P + 2), dict(out=P + 8), dict(ws=P + 4)):
        assert attend(L, c, **kw) == ALIGN
    # rows, items and positions are counted in 32 bits
    for kw in (dict(draft=1 << 24, hq=2), dict(batch=1 << 24), dict(batch=1 << 20, draft=1 << 10, hq=2),
               dict(pages=1 << 27)):
        assert attend(L, c, **kw) == RANGE
    assert attend(L, c, batch=0, q=None, ws=None) == attend(L, c, draft=0, q=None, ws=None) == OK


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.ones(128)
    cs, pos = torch.ones(8, 64), torch.arange(3)
    with pytest.raises(TypeError):
        bb.qk_norm_rope(x, x, w, w, cs, cs, pos)
    with pytest.raises(TypeError):
        bb.QuantizedKVCache(4, 16, 2, 128, bb.MXFP8BlockScaling(), device="cpu")
    with pytest.raises(TypeError):
        bb.qk_norm_rope_write(x, x, x, w, w, cs, cs, pos, None, pos)
    with pytest.raises(TypeError):
        bb.cache_attention(x, None, None, None)
    z = torch.zeros(4, 2, 16, 128, dtype=torch.uint8)
    with pytest.raises(TypeError):
        bb.QuantizedKVCache.from_buffers(z, z, z, z, bb.MXFP8BlockScaling())
