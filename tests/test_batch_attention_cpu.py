"""What attention of a batch's rows and adjusted logits refuse before any device call, and the sizes of their workspaces."""
import ctypes
import math

import pytest

P = ctypes.c_void_p
GIB = 1 << 32


def _lib():
    from cpm.cu_amd import lib
    return lib.get()


def _attention(kind, **kw):
    a = dict(q=P(1 * GIB), qs=4096, k=P(100 * GIB), v=P(200 * GIB), pages=64, tables=P(4 * GIB), ts=None, blocks=8, offsets=P(5 * GIB), pos=P(6 * GIB), B=4, n=60, hq=32, hkv=2, scale=0.1, out=P(7 * GIB),
             os=4096, ws=P(8 * GIB), wb=1 << 40)
    a.update(kw)
    fn = _lib().batch_prompt_attention if kind == "prompt" else _lib().batch_decode_attention
    fn(a["q"], a["qs"], a["k"], a["v"], a["pages"], a["tables"], a["blocks"] if a["ts"] is None else a["ts"], a["blocks"], a["offsets"], a["pos"], a["B"], a["n"], a["hq"], a["hkv"], ctypes.c_float(a["scale"]), a["out"], a["os"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kind", ["prompt", "decode"])
@pytest.mark.parametrize("kw, match", [
    (dict(q=None), "null"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(tables=None), "null"), (dict(pos=None), "null"), (dict(out=None), "null"),
    (dict(n=-1), "n=-1"), (dict(n=1 << 24), "n=16777216"), (dict(B=0), "0 requests"), (dict(B=4097), "4097 requests"), (dict(blocks=0), "max_blocks=0"), (dict(blocks=(1 << 18) + 1), "max_blocks"),
    (dict(B=4096, blocks=1 << 17), "more than 268435456 entries"), (dict(ts=7), "tables closer"), (dict(ts=1 << 31), "tables closer"), (dict(out=P(4 * GIB + (3 << 22)), ts=1 << 20), "tables, offsets"), (dict(pages=0), "num_pages=0"), (dict(pages=1 << 23), "num_pages"), (dict(hkv=0), "0 KV heads"), (dict(hkv=3), "3 KV heads"), (dict(hq=0), "0 query heads"),
    (dict(hq=1025, hkv=1), "1025 query heads"), (dict(n=(1 << 24) - 1, hq=1024, qs=1 << 18, os=1 << 18), "beyond 32 bits"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(qs=4095), "closer"), (dict(os=4000), "closer"), (dict(qs=1 << 31), "further apart"), (dict(q=P(GIB + 8)), "16 bytes"), (dict(out=P(7 * GIB + 2)), "16 bytes"),
    (dict(qs=4100), "16 bytes"), (dict(k=P(100 * GIB + 4)), "16 bytes"), (dict(ws=P(8 * GIB + 8)), "16 bytes"), (dict(ws=None), "workspace of"), (dict(wb=100), "workspace of 100 bytes"),
    (dict(out=P(GIB + 4096 * 2)), "other rows of q"), (dict(out=P(GIB), os=8192), "other rows of q"), (dict(out=P(GIB + 8192), qs=8192 - 64, os=8192 - 64), "other rows of q"),
    (dict(out=P(100 * GIB + 4096)), "lie in the pools"), (dict(out=P(200 * GIB - 4096)), "lie in the pools"),
    (dict(out=P(4 * GIB)), "tables, offsets or positions"), (dict(pos=P(7 * GIB + 64)), "tables, offsets or positions"), (dict(offsets=P(7 * GIB + 64)), "tables, offsets or positions")], ids=str)
def test_attention_of_a_batch_refuses(kind, kw, match):
    with pytest.raises(ValueError, match=match):
        _attention(kind, **kw)


def test_offsets_are_needed():
    with pytest.raises(ValueError, match="null"):
        _attention("prompt", offsets=None)
    with pytest.raises(ValueError, match="60 rows of 4 requests need row_offsets"):
        _attention("decode", offsets=None)


@pytest.mark.parametrize("kind", ["prompt", "decode"])
def test_no_rows_need_nothing(kind):
    _attention(kind, n=0, q=None, out=None, k=None, v=None, tables=None, pos=None, offsets=None, ws=None, wb=0)


def test_workspaces():
    raw = _lib().raw
    for args in ((0, 8, 60, 32, 2), (4097, 8, 60, 32, 2), (4, 0, 60, 32, 2), (4, 8, -1, 32, 2), (4, 8, 60, 32, 3), (4, 8, 60, 32, 0)):
        assert raw.cpmcu_batch_prompt_attention_workspace_bytes(*args) == 0
        assert raw.cpmcu_batch_decode_attention_workspace_bytes(args[0], args[1], args[3], args[4]) == 0 or args[2] < 0
    # short tables: nothing is cut, a list is all there is; long ones: 896 pieces of 128 rows at most twice over, however many rows there are
    assert raw.cpmcu_batch_prompt_attention_workspace_bytes(1, 4, 1000, 32, 2) < 1 << 14
    assert raw.cpmcu_batch_prompt_attention_workspace_bytes(4096, 1 << 16, (1 << 24) - 1, 32, 2) < (1 << 27) + (1 << 22) + 64 * (1 << 21)
    assert raw.cpmcu_batch_decode_attention_workspace_bytes(4096, 1 << 16, 32, 2) < 1 << 25
    assert raw.cpmcu_adjust_logits_workspace_bytes(-1, 100) == raw.cpmcu_adjust_logits_workspace_bytes(5, 0) == raw.cpmcu_adjust_logits_workspace_bytes(5, (1 << 24) + 1) == 0


def _logits(**kw):
    a = dict(z=P(1 * GIB), zs=1000, n=8, V=1000, pen=P(2 * GIB), tok=P(3 * GIB), lens=P(4 * GIB), R=8, L=50, req=None, bi=P(5 * GIB), bv=P(6 * GIB), nb=4, al=P(7 * GIB), als=32, di=None, tm=None, mw=0,
             out=P(8 * GIB), os=1000, ids=P(9 * GIB), ws=P(10 * GIB), wb=1 << 30)
    a.update(kw)
    _lib().adjust_logits(a["z"], a["zs"], a["n"], a["V"], a["pen"], a["tok"], a["lens"], a["R"], a["L"], a["req"], a["bi"], a["bv"], a["nb"], a["al"], a["als"], a["di"], a["tm"], a["mw"], a["out"], a["os"], a["ids"],
                         a["ws"], a["wb"], None)


TREE = dict(di=P(11 * GIB), tm=P(12 * GIB), mw=1, R=1)


@pytest.mark.parametrize("kw, match", [
    (dict(z=None), "null"), (dict(out=None), "null"), (dict(n=-1), "n=-1"), (dict(n=1 << 24), "n=16777216"), (dict(V=0), "V=0"), (dict(V=(1 << 24) + 1), "V=16777217"), (dict(zs=999), "closer"), (dict(os=999), "closer"),
    (dict(z=P(GIB + 1)), "2 bytes"), (dict(R=0), "0 requests"), (dict(R=5), "8 rows of 5 requests"), (dict(pen=None), "tokens go with"), (dict(lens=None), "tokens go with"), (dict(L=0), "tokens go with"),
    (dict(bv=None), "biases"), (dict(nb=0), "0 biases"), (dict(nb=1025), "1025 biases"), (dict(als=31), "allowed closer"), (dict(als=-1), "allowed closer"),
    (dict(TREE, tm=None), "draft_ids go with"), (dict(TREE, R=8), "draft_ids go with"), (dict(TREE, req=P(13 * GIB)), "draft_ids go with"), (dict(TREE, pen=None, tok=None), "draft_ids go with"),
    (dict(TREE, n=129, mw=3), "129 nodes"), (dict(TREE, n=65, mw=1), "masks of 1 words"), (dict(ws=None), "workspace"), (dict(wb=8), "workspace of 8 bytes"), (dict(ws=P(10 * GIB + 4)), "workspace"),
    (dict(out=P(GIB + 2000)), "other logits"), (dict(out=P(GIB), os=2000), "other logits"), (dict(tok=P(8 * GIB + 64)), "memory of an argument"), (dict(al=P(8 * GIB)), "memory of an argument"),
    (dict(ids=P(3 * GIB)), "memory of an argument"), (dict(ids=P(4 * GIB + 28)), "memory of an argument"), (dict(ids=P(8 * GIB)), "ids in the memory"), (dict(ids=P(GIB + 16)), "ids in the memory")], ids=str)
def test_adjust_logits_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        _logits(**kw)


def test_more_threads_than_a_launch_has_are_refused():
    """A launch has fewer than 2^32 threads."""
    far = dict(q=P(1 << 50), out=P(1 << 52), qs=1 << 17, os=1 << 17, hq=1024, hkv=1024, wb=1 << 60)
    with pytest.raises(ValueError, match="prompt_attention: .* beyond a launch"):
        _attention("prompt", **dict(far, B=4096, n=(1 << 21) - 5))
    with pytest.raises(ValueError, match="decode_attention: .* beyond a launch"):
        _attention("decode", **dict(far, B=4096, n=4096))
    with pytest.raises(ValueError, match="adjust_logits: .* beyond a launch"):
        _logits(z=P(1 << 50), zs=5000, out=P(1 << 52), os=5000, n=(1 << 24) - 1, V=5000, R=1, al=None, ids=None, pen=None, tok=None, lens=None, bi=None, bv=None)


def test_texts_beyond_a_place_s_count_are_refused():
    """A place has 21 bits for its count."""
    with pytest.raises(ValueError, match="max_tokens=1048577"):
        _logits(L=(1 << 20) + 1)


def test_no_logits_need_nothing():
    _logits(n=0, z=None, out=None, ids=None, ws=None)


def test_more_requests_than_rows_may_be_are_refused():
    """A request's penalties are found by a 32-bit product."""
    for more in (dict(), dict(pen=None, tok=None, lens=None)):
        with pytest.raises(ValueError, match="16777216 requests outside"):
            _logits(R=1 << 24, req=P(13 * GIB), out=P(1 << 50), ids=P(1 << 52), **more)
    with pytest.raises(ValueError, match="715827883 requests outside"):
        _logits(R=715827883, req=P(13 * GIB), out=P(1 << 50), ids=P(1 << 52))
