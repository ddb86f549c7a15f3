"""Refusals of the paged serving path at the C boundary, and its oracle's own rules: no GPU."""
import ctypes

import pytest
import torch

from oracle import paged as ref


@pytest.fixture(scope="module")
def lib():
    from sparse_attention_b200_b200 import _lib
    return _lib.lib()


P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4100)
I64 = ctypes.c_int64


def _refused(lib, rc, word):
    from sparse_attention_b200_b200 import _lib
    assert rc == _lib.ERR_INVALID and word in lib.sparse_b200_last_error(), lib.sparse_b200_last_error()


def test_extend_pages_refuses(lib):
    good = dict(table=P, stride=8, width=8, seq=P, new=P, free=P, cap=4, count=P, seq_out=ctypes.c_void_p(8192),
                count_out=ctypes.c_void_p(8192), batch=2, total_q=4, total_pages=4)

    def call(**kw):
        a = {**good, **kw}
        return lib.sparse_b200_extend_pages(a["table"], I64(a["stride"]), a["width"], a["seq"], a["new"], a["free"], a["cap"],
                                            a["count"], a["seq_out"], P, P, P, P, P, a["count_out"], P, a["batch"],
                                            a["total_q"], a["total_pages"], None)
    for kw, word in ((dict(table=None), b"null"), (dict(batch=0), b"requests"), (dict(batch=4097), b"requests"),
                     (dict(total_q=-1), b"token"), (dict(total_pages=-1), b"negative"), (dict(width=0), b"table row"),
                     (dict(stride=4), b"table row"), (dict(width=1 << 24, stride=1 << 24), b"table row"),
                     (dict(seq_out=P), b"in place"), (dict(free=None), b"null")):
        _refused(lib, call(**kw), word)


def test_append_tokens_refuses(lib):
    good = dict(k=P, ks=128, kh=128, index=None, iscale=None, batch=2, hkv=2, total=4, pages=4, slots=P)

    def call(**kw):
        a = {**good, **kw}
        return lib.sparse_b200_append_tokens(a["k"], I64(a["ks"]), I64(a["kh"]), P, I64(128), I64(128), P, a["slots"], P, P, P, P,
                                             a["index"], a["iscale"], a["batch"], a["hkv"], a["total"], I64(a["pages"]), None)
    for kw, word in ((dict(k=None), b"null"), (dict(k=ODD), b"aligned"), (dict(ks=129), b"strides"), (dict(kh=4), b"strides"),
                     (dict(index=P), b"together"), (dict(batch=0), b"requests"), (dict(hkv=0), b"heads"),
                     (dict(pages=0), b"page"), (dict(total=-1), b"token"), (dict(slots=None), b"null")):
        _refused(lib, call(**kw), word)
    assert call(total=0) == 0


def test_select_pages_refuses(lib):
    good = dict(scores=P, batch=2, hidx=4, hkv=2, pages=9, total=4, topk=4, tile=1, sink=1, recent=1)

    def call(**kw):
        a = {**good, **kw}
        return lib.sparse_b200_select_pages(a["scores"], P, P, P, a["batch"], a["hidx"], a["hkv"], a["pages"], a["total"],
                                            a["topk"], a["tile"], a["sink"], a["recent"], 1, None)
    for kw, word in ((dict(scores=None), b"null"), (dict(hidx=3), b"multiple"), (dict(hkv=0), b"multiple"),
                     (dict(topk=0), b"at least one"), (dict(tile=0), b"tile"), (dict(tile=12), b"tile"), (dict(tile=256), b"tile"),
                     (dict(sink=-1), b"sink"), (dict(sink=3, recent=2), b"sink"), (dict(sink=2 ** 31 - 1, recent=2), b"sink"),
                     (dict(pages=0), b"page"), (dict(batch=5000), b"requests")):
        _refused(lib, call(**kw), word)
    assert call(total=0) == 0


def test_paged_attention_refuses(lib):
    good = dict(q=P, qt=128, qh=128, k=P, stride=8, width=8, ids=None, out=ctypes.c_void_p(8192), ws=None, batch=2, hq=8, hkv=2,
                total=4, pages=4, topk=3, tile=1, scale=0.1)

    def call(**kw):
        a = {**good, **kw}
        return lib.sparse_b200_paged_attention(a["q"], I64(a["qt"]), I64(a["qh"]), a["k"], P, P, P, P, I64(a["stride"]), a["width"],
                                               P, P, a["ids"], a["out"], None, a["ws"], I64(0), a["batch"], a["hq"], a["hkv"],
                                               a["total"], I64(a["pages"]), a["topk"], a["tile"], 1, 1,
                                               ctypes.c_float(a["scale"]), None)
    for kw, word in ((dict(q=None), b"null"), (dict(q=ODD), b"aligned"), (dict(ws=ODD), b"aligned"), (dict(qt=4), b"strides"),
                     (dict(hq=7), b"multiple"), (dict(hq=130), b"64"), (dict(hkv=0), b"multiple"), (dict(pages=0), b"fit"),
                     (dict(pages=1 << 24), b"fit"), (dict(width=0), b"table row"), (dict(stride=7), b"table row"),
                     (dict(ids=P, topk=0), b"at least one"), (dict(ids=P, tile=6), b"tile"), (dict(out=P), b"alias"),
                     (dict(scale=float("nan")), b"finite"), (dict(scale=float("inf")), b"finite"), (dict(batch=0), b"requests"),
                     (dict(total=-1), b"token")):
        _refused(lib, call(**kw), word)
    assert call(total=0) == 0
    assert lib.sparse_b200_paged_attention_workspace_bytes(7, 2, 1, 1, 0) < 0


def test_python_refuses_cpu_tensors():
    import sparse_attention_b200_b200 as sp
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32)
    pages = torch.zeros((1, 1, 128, 128), dtype=torch.uint8).view(torch.float8_e4m3fn)
    for bad in (lambda: sp.quantize_rows(q, 2), lambda: sp.extend_pages(one[None], one, one, one, one, total_q=1, total_pages=1),
                lambda: sp.select_pages(torch.zeros((1, 1, 1)), one, one, kv_heads=1, topk=1),
                lambda: sp.PagedCache.from_tensors(pages, pages, torch.ones((1, 1)), torch.ones((1, 1)))):
        with pytest.raises(sp.SparseB200Error):
            bad()


def test_list_rows_leave_every_request_room():
    for tile in (2, 4, 64, 128):
        for lens in ([1], [5, 0, 3, tile, tile + 1], [tile - 1] * 5, [0, 0, 2 * tile + 1]):
            cu, last = [0], -1
            for r, n in enumerate(lens):
                for i in range(-(-n // tile)):
                    row = ref.list_row(cu[-1], r, i, tile)
                    assert row > last
                    last = row
                cu.append(cu[-1] + n)
            assert last < cu[-1] // tile + len(lens)


def test_e4m3_rounding_of_the_oracle():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    finite = codes[~codes.isnan()]
    assert torch.equal(ref.round_e4m3(finite), finite)
    x = torch.cat([finite * 1.03, finite * 0.51, torch.linspace(-500, 500, 4001, dtype=torch.float64)])
    assert torch.equal(ref.round_e4m3(x).abs(), x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double().abs())
