"""The 4-bit page cache without a GPU: the format restatement the GPU tests compare with, what the Python wrappers refuse, what the C entry points refuse (all of it
before anything is launched)."""
import ctypes as C

import pytest
import torch

import _kv4 as R
from unimp_amd import _lib, ops

bf16, i32, i64 = torch.bfloat16, torch.int32, torch.int64


def test_format_by_hand():
    x = torch.tensor([[6., 5., 5.01, 3.5, 2.5, 1.75, 1.25, .75, .25, .2501, -6., -.1] + [0.] * 20])
    codes, scales = R.quantise(x)
    assert scales.tolist() == [[127]] and codes[0, :12].tolist() == [7, 6, 7, 6, 4, 4, 2, 2, 0, 1, 15, 8]
    assert R.held(torch.full((1, 32), 7.9))[0, 0] == 6 and R.held(torch.full((1, 32), 8.0))[0, 0] == 8       # saturates below the next exponent
    assert R.quantise(torch.zeros(1, 32))[1].item() == 2 and R.quantise(torch.full((1, 32), 1e-40))[1].item() == 2
    assert torch.isnan(R.held(torch.tensor([[float("inf")] + [1.] * 31]))).all()


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_page_layout_is_a_bijection(hd):
    """every byte of a page belongs to exactly one token's code pair or scale; packing token by token and whole pages agree"""
    assert ops.kv4_page_bytes(hd) == R.page_bytes(hd) == _lib.lib().unimp_kv4_page_bytes(hd)
    k, v = (torch.randn(32, hd, generator=torch.Generator().manual_seed(s)).to(bf16) for s in (0, 1))
    whole, single = R.pack(k, v), torch.zeros(R.page_bytes(hd), dtype=torch.uint8)
    for t in torch.randperm(32, generator=torch.Generator().manual_seed(2)).tolist():
        R.put(single, t, k[t], v[t])
    assert torch.equal(whole, single)
    a, b = R.unpack(whole, hd)
    assert torch.equal(a, R.held(k)) and torch.equal(b, R.held(v))
    assert torch.equal(R.held(a), a)                                # what is held quantises to itself


def test_other_head_dims():
    assert _lib.lib().unimp_kv4_page_bytes(96) == -1
    with pytest.raises(ValueError):
        ops.kv4_page_bytes(96)


def _pool(n=4, heads=2, hd=64):
    return torch.zeros((n, heads, R.page_bytes(hd)), dtype=torch.uint8)


def _bad(what, f):
    with pytest.raises(ValueError):
        f()
        pytest.fail(what)


def test_python_refusals():
    k = torch.zeros(3, 2, 64, dtype=bf16)
    s3 = torch.zeros(3, dtype=i64)
    _bad("heads", lambda: ops.kv4_write(k, k, _pool(heads=3), s3))
    _bad("page bytes of another head dim", lambda: ops.kv4_write(k, k, _pool(hd=80), s3))
    _bad("k and v differ", lambda: ops.kv4_write(k, k[:2], _pool(), s3))
    _bad("fp16", lambda: ops.kv4_write(k.half(), k.half(), _pool(), s3))
    _bad("int32 slots", lambda: ops.kv4_write(k, k, _pool(), s3.int()))
    _bad("strided slots", lambda: ops.kv4_write(k, k, _pool(), torch.zeros(6, dtype=i64)[::2]))
    _bad("pages not contiguous", lambda: ops.kv4_write(k, k, _pool(heads=4)[:, ::2], s3))
    _bad("a layered pool", lambda: ops.kv4_write(k, k, _pool()[None], s3))
    _bad("layers overlap", lambda: ops.kv4_read(_pool().expand(3, 4, 2, R.page_bytes(64)), s3, 64))
    qkv = torch.zeros(3, 3 * 128, dtype=bf16)
    app = lambda **kw: ops.kv4_rope_append(**{**dict(qkv2d=qkv, heads=2, head_stride=192, hd=64, offs=(0, 64, 128), rot=0, cos_rows=None, sin_rows=None, pages=_pool(),
                                                     slots=s3), **kw})
    _bad("offset outside the row", lambda: app(offs=(0, 64, 192)))
    _bad("odd rot", lambda: app(rot=3))
    _bad("no tables", lambda: app(rot=16))
    _bad("rot above the head dim", lambda: app(rot=66))
    _bad("tables of another shape", lambda: app(rot=64, cos_rows=torch.zeros(3, 16), sin_rows=torch.zeros(3, 16)))
    _bad("slots of another length", lambda: app(slots=s3[:2].contiguous()))
    z = lambda *s: torch.zeros(s, dtype=i32)
    ext = lambda **kw: ops.page_tables_extend(**{**dict(tables=z(4, 3), mapped=z(4), cached=z(4), new=z(4), free_pages=z(9), cursor=z(1), max_tokens=2), **kw})
    _bad("no columns", lambda: ext(tables=z(4, 0)))
    _bad("rows not in groups", lambda: ext(group=3))
    _bad("int64 lengths", lambda: ext(new=z(4).long()))
    _bad("shared length per row", lambda: ext(group=2, shared_len=z(4)))
    _bad("negative room", lambda: ext(max_tokens=-1))
    ro = lambda **kw: ops.kv4_reorder_beams(**{**dict(pages=_pool(), tables=z(4, 2), group=2, src_local=torch.zeros(4, dtype=i64), pos=torch.zeros(4, dtype=i64)), **kw})
    _bad("not a page size", lambda: ro(pages=torch.zeros(4, 2, 100, dtype=torch.uint8)))
    _bad("int32 sources", lambda: ro(src_local=z(4)))
    _bad("rows not in groups", lambda: ro(group=3))
    q = torch.zeros(3, 4, 64, dtype=bf16)
    at = lambda **kw: ops.kv4_attn_decode(**{**dict(q=q, pages=_pool(), tables=z(3, 2), lens=z(3), scale=1.0), **kw})
    _bad("five query heads on two", lambda: at(q=torch.zeros(3, 5, 64, dtype=bf16)))
    _bad("34 on two", lambda: at(q=torch.zeros(3, 34, 64, dtype=bf16)))
    _bad("fp32 q", lambda: at(q=q.float()))
    _bad("lens of other rows", lambda: at(lens=z(2)))
    _bad("tables of other rows", lambda: at(tables=z(2, 2)))
    _bad("alibi per key head", lambda: at(alibi=torch.zeros(2)))
    _bad("out of another shape", lambda: at(out=torch.zeros(3, 4, 80, dtype=bf16)))
    _bad("shared length of other groups", lambda: at(group=3, shared_len=z(3)))
    for f in (lambda: ops.kv4_write(k, k, _pool(), s3), app, ext, ro, at, lambda: ops.kv4_read(_pool(), s3, 64)):
        with pytest.raises(_lib.UnimpHipError):                     # all well, but no HIP device under the tensors
            f()


def test_c_refusals():
    L = _lib.lib()
    p, odd = C.c_void_p(1 << 20), C.c_void_p((1 << 20) + 8)         # never followed: refused before a launch
    ARG, SHAPE, ALIGN = 1, 2, 3
    w = lambda k=p, ts=128, pages=p, heads=2, hd=64, slots=p, n=5: L.unimp_kv4_write(k, p, ts, 64, 128, 64, pages, 4, heads, hd, slots, n, None)
    assert w(k=None) == w(slots=None) == ARG and w(hd=96) == w(heads=1 << 20) == w(n=1 << 40) == SHAPE and w(ts=100) == w(pages=odd) == w(k=odd) == ALIGN and w(n=0) == 0
    a = lambda rot=0, cos=None, hd=64, pages=p, rows=3: L.unimp_kv4_rope_append(p, 384, 192, rows, 2, hd, 0, 64, 128, rot, cos, cos, p, pages, 4, p, None)
    assert a(rot=32) == a(pages=None) == ARG and a(rot=66, cos=p) == a(rot=5, cos=p) == a(hd=72) == a(rows=70000) == SHAPE and a(pages=odd) == ALIGN and a(rows=0) == 0
    r = lambda layers=1, hd=64, n=5, k=p: L.unimp_kv4_read(p, 1 << 20, layers, 4, 2, hd, p, n, k, p, None)
    assert r(k=None) == ARG and r(layers=1 << 17) == r(hd=1) == r(n=1 << 40) == SHAPE and r(k=odd) == ALIGN and r(n=0) == 0
    t = lambda rows=4, width=3, group=1, out=C.c_void_p(1 << 21), cur=C.c_void_p(1 << 22), slots=p, n=5: L.unimp_page_tables_extend(
        p, rows, width, p, p, p, None, p, 9, p, group, None, out, cur, slots, n, p, None)
    assert t(out=p) == t(cur=p) == t(slots=None) == ARG and t(rows=0) == t(rows=65537) == t(width=0) == t(group=3) == t(group=0) == t(n=-1) == SHAPE
    b = lambda pages=p, hd=64, group=2, layers=1, stride=1 << 20: L.unimp_kv4_reorder_beams(pages, stride, layers, 4, 2, hd, p, 3, group, 2, p, p, None)
    assert b(pages=None) == ARG and b(hd=65) == b(group=17) == b(layers=1 << 17) == SHAPE and b(pages=odd) == b(stride=(1 << 20) + 4) == ALIGN and b(group=1) == 0

    def at(**kw):
        d = _lib.Kv4AttnDesc()
        for n, v in dict(q=p, q_row_stride=256, q_head_stride=64, pages=p, n_pages=4, kv_heads=2, hd=64, tables=p, table_stride=3, width=3, lens=p, rows=3, heads=4, scale=1.0,
                         out=p, o_row_stride=256, o_head_stride=64, group=1).items():
            setattr(d, n, kw.get(n, v))
        return L.unimp_kv4_attn_decode(C.byref(d), p, None)
    assert at(q=None) == at(lens=None) == at(out=None) == ARG and at(heads=5) == at(heads=34) == at(hd=32) == at(kv_heads=0) == at(rows=1 << 17) == at(width=-1) == SHAPE
    assert at(pages=odd) == ALIGN and at(rows=0) == 0
    assert L.unimp_struct_size(5) == C.sizeof(_lib.Kv4AttnDesc)


def test_packed_descriptor_is_the_struct():
    """the wrapper packs the descriptor by a format string: the same bytes as the ctypes mirror's"""
    vals = [11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 21, 22, 23, 0.375, 24, 25, 26, 27, 28, 29]
    d = _lib.Kv4AttnDesc(*vals)
    packed = ops._KV4_ATTN.pack(*vals)
    assert len(packed) == C.sizeof(d) or len(packed) == C.sizeof(d) - C.sizeof(d) % 8
    again = _lib.Kv4AttnDesc.from_buffer_copy(packed.ljust(C.sizeof(d), b"\0"))
    assert [getattr(again, n) for n, _ in d._fields_] == vals


def test_decode_session_refuses_other_caches():
    from types import SimpleNamespace
    from unimp_amd.decode import DecodeSession
    from unimp_amd.functional import Kv4Cache
    with pytest.raises(ValueError):
        DecodeSession(SimpleNamespace(lang_encoder=None), 4, False, kv_cache="int8")
    with pytest.raises(ValueError):
        Kv4Cache(SimpleNamespace(layers=[], kv=torch.zeros(1, 2, 1, 8, 2, 64, dtype=bf16)), [8], beams=17, max_new=4)
