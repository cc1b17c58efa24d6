"""Refusals of the 4-bit cache's, attention's and the linear layers' entry points that need
no GPU: arguments and, for host arrays, sequences, pages and past are checked before the
context is touched."""
import ctypes as C

import numpy as np
import pytest

from dismoen import DismoenError, KVCache, SeqBatch, lib
from dismoen._lib import (DmhAttention, DmhKvCache, DmhKvRows, DmhLinearRows, DmhLinearWeights,
                          DmhSeqBatch)

F_DEVICE = 1
_keep = []
CTX = (1, "ctx is NULL")  # what a call without a fault in its arguments ends with here


def ptr(n, at=0):
    a = np.zeros(n + 64, np.uint8)
    _keep.append(a)
    return (a.ctypes.data + 31) // 16 * 16 + at


def i32(*v):
    a = np.array(v, np.int32)
    _keep.append(a)
    return a.ctypes.data


def set_all(a, kw):
    for k, v in kw.items():
        assert hasattr(a, k), k
        setattr(a, k, v)
    return a


def cache(pages=(0, 1, 2, 3, 4, 5), past=(0, 20, 40), **kw):
    ids = None if pages is None else i32(*(list(pages) + [0] * 12)[:12])
    return set_all(DmhKvCache(kv_heads=2, dim=64, page_size=16, num_pages=6, max_pages=4,
                              codes=ptr(6 * 2 * 2 * 16 * 32), scales=ptr(6 * 2 * 2 * 16 * 2),
                              pages=ids, past=None if past is None else i32(*past)), kw)


def rows(**kw):
    return set_all(DmhKvRows(dtype=0, k=ptr(8 * 128 * 4), v=ptr(8 * 128 * 4), k_stride=128,
                             k_head_stride=64, v_stride=128, v_head_stride=64), kw)


def attention(**kw):
    return set_all(DmhAttention(dtype=0, q_heads=4, scale=0.125, q=ptr(8 * 256 * 4), gate=None,
                                o=ptr(8 * 256 * 4), q_stride=256, q_head_stride=64, o_stride=256,
                                o_head_stride=64), kw)


def batch(offsets=(0, 2, 5), total=6, max_len=4, slots_n=3, slots=None, fresh=None):
    return DmhSeqBatch(len(offsets) - 1, total, max_len, slots_n, i32(*offsets),
                       None if slots is None else i32(*slots),
                       None if fresh is None else i32(*fresh))


def call(name, a, c, b, flags=0):
    e = C.create_string_buffer(512)
    refs = [None if x is None else C.byref(x)
            for x in ((c, a, b) if name.startswith("dmh_kv") else (a, c, b))]
    rc = getattr(lib(), name)(None, *refs, flags, e, len(e))
    return rc, e.value.decode()


CALLS = {"dmh_kv_write": rows, "dmh_kv_read": rows, "dmh_attention_forward": attention}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("kw,code,text", [
    ({}, *CTX),
    ({"dim": 80}, 2, "dim 80"),
    ({"dim": 0}, 2, "dim 0"),
    ({"kv_heads": 0}, 2, "kv_heads 0"),
    ({"kv_heads": 1025}, 2, "kv_heads 1025"),
    ({"page_size": 8}, 2, "page_size 8"),
    ({"page_size": 48}, 2, "page_size 48"),
    ({"num_pages": 0}, 2, "num_pages 0"),
    ({"max_pages": 0}, 2, "max_pages 0"),
    ({"max_pages": 1 << 27}, 2, "2^30 positions"),
    ({"codes": None}, 1, "is NULL"),
    ({"scales": None}, 1, "is NULL"),
    ({"pages": None}, 1, "is NULL"),
    ({"past": None}, 1, "is NULL"),
    ({"codes": 24}, 1, "16-byte aligned"),
])
def test_cache_arguments(name, kw, code, text):
    rc, got = call(name, CALLS[name](), cache(**kw), batch())
    assert rc == code and text in got, got


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("c,b,text", [
    (dict(), dict(), CTX[1]),
    (dict(past=(0, -1, 0)), dict(), "sequence 1: its tokens"),
    (dict(past=(0, 62, 0)), dict(), "sequence 1: its tokens"),   # 62 + 3 of 64
    (dict(past=(0, 61, 0)), dict(), "a page outside|ctx is NULL"),
    (dict(past=(0, -1, 0)), dict(fresh=(0, 1)), CTX[1]),          # fresh: past does not count
    (dict(past=(-1, -1, -1)), dict(slots=(-1, -2)), CTX[1]),
    (dict(pages=(9,)), dict(), "sequence 0: a page outside"),
    (dict(pages=(-1,)), dict(), "sequence 0: a page outside"),
    (dict(), dict(offsets=(0, 2, 7)), "sequence 1: offsets"),
    (dict(), dict(slots=(0, 3)), "sequence 1: slot"),
], ids=str)
def test_cache_sequences(name, c, b, text):
    import re
    rc, got = call(name, CALLS[name](), cache(**c), batch(**b))
    assert rc == 1 and re.search(text, got), got


def test_shared_slots():
    """Two sequences of one slot may be read, not written."""
    b = dict(slots=(1, 1))
    assert "earlier sequence" in call("dmh_kv_write", rows(), cache(), batch(**b))[1]
    assert CTX[1] in call("dmh_kv_read", rows(), cache(), batch(**b))[1]
    assert CTX[1] in call("dmh_attention_forward", attention(), cache(), batch(**b))[1]


def test_pages_that_a_call_does_not_need():
    """Writing looks at the pages of its rows alone, attention at all up to them."""
    c = dict(pages=(77, 0, 1, 2), past=(20, 0, 0))
    b = dict(offsets=(0, 2))
    assert CTX[1] in call("dmh_kv_write", rows(), cache(**c), batch(**b))[1]
    assert CTX[1] in call("dmh_kv_read", rows(), cache(**c), batch(**b))[1]
    assert "a page outside" in call("dmh_attention_forward", attention(), cache(**c), batch(**b))[1]


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 5}, "unknown dtype"), ({"k": None}, "is NULL"), ({"v": None}, "is NULL"),
    ({"k_stride": 127}, "head lies in another"), ({"k_head_stride": 63}, "head lies in another"),
    ({"v_head_stride": 65}, "head lies in another"),  # behind the row's stride
    ({"k": 64 + 2}, "misaligned"),
])
def test_rows(kw, text):
    for name in ("dmh_kv_write", "dmh_kv_read"):
        rc, got = call(name, rows(**kw), cache(), batch())
        assert rc == 1 and text in got, got


def test_overlap():
    c = cache()
    for name in ("dmh_kv_write", "dmh_kv_read"):
        assert "must not overlap" in call(name, rows(k=c.codes + 64), c, batch())[1]
        assert "must not overlap" in call(name, rows(v=c.scales), c, batch())[1]
    r = rows()
    assert CTX[1] in call("dmh_kv_write", rows(k=r.k, v=r.k), c, batch())[1]
    assert "k and v" in call("dmh_kv_read", rows(k=r.k, v=r.k), c, batch())[1]
    # heads side by side in one row
    x = ptr(8 * 512 * 4)
    side = dict(k=x, v=x + 256, k_stride=256, v_stride=256, k_head_stride=128, v_head_stride=128)
    assert CTX[1] in call("dmh_kv_read", rows(**side), c, batch())[1]
    side["v"] = x + 252
    assert "k and v" in call("dmh_kv_read", rows(**side), c, batch())[1]
    a = attention()
    assert "o must not" in call("dmh_attention_forward", attention(o=a.q, q=a.q), c, batch())[1]
    assert "o must not" in call("dmh_attention_forward", attention(o=c.codes), c, batch())[1]
    assert "overlap" in call("dmh_kv_write", rows(), cache(scales=c.codes, codes=c.codes), batch())[1]


@pytest.mark.parametrize("kw,code,text", [
    ({"q_heads": 3}, 2, "q_heads 3"), ({"q_heads": 0}, 2, "q_heads 0"),
    ({"q_heads": 4098}, 2, "q_heads 4098"), ({"scale": 0.0}, 1, "scale"), ({"scale": -1.0}, 1, "scale"),
    ({"scale": float("nan")}, 1, "scale"), ({"scale": float("inf")}, 1, "scale"),
    ({"q": None}, 1, "is NULL"), ({"o": None}, 1, "is NULL"), ({"dtype": -1}, 1, "unknown dtype"),
    ({"o_stride": 255}, 1, "head lies"), ({"q_head_stride": 32}, 1, "head lies"),
    ({"gate": 64, "gate_stride": 10, "gate_head_stride": 64}, 1, "head lies"),
])
def test_attention_arguments(kw, code, text):
    rc, got = call("dmh_attention_forward", attention(**kw), cache(), batch())
    assert rc == code and text in got, got


def test_rows_past_32_bits():
    """Rows count tokens times query heads of a key head."""
    c = cache(kv_heads=1, past=(0, 0, 0), max_pages=1 << 26)
    big = dict(q_heads=4096, q=ptr(64), o=ptr(64, 16), dtype=0)
    strides = {k: 4096 * 64 for k in ("q_stride", "o_stride")}
    a = attention(**big, **strides)
    b = batch(offsets=(0, 1), total=1 << 18, max_len=1)
    a.o = a.q + (1 << 40)  # (never touched: the call is refused)
    rc, got = call("dmh_attention_forward", a, c, b, F_DEVICE)
    assert rc == 2 and "too many rows" in got, got
    b.total_tokens = (1 << 18) - 1
    assert CTX[1] in call("dmh_attention_forward", a, c, b, F_DEVICE)[1]


def test_nulls():
    for name, make in CALLS.items():
        assert call(name, None, cache(), batch())[0] == 1
        assert "cache is NULL" in call(name, make(), None, batch())[1]
        assert "batch is NULL" in call(name, make(), cache(), None)[1]
        # without rows no arrays are needed
        empty = DmhKvCache(2, 64, 16, 6, 4, None, None, None, None)
        assert CTX[1] in call(name, make(), empty, batch(offsets=(0, 0), total=0))[1]


# ---- linear layers -----------------------------------------------------------------------
def upload(**kw):
    w = set_all(DmhLinearWeights(8, 64, 32, ptr(32), ptr(256), None), kw)
    e, h = C.create_string_buffer(512), C.c_void_p()
    rc = lib().dmh_upload_linear(None, C.addressof(w), 0, C.byref(h), e, 512)
    return rc, e.value.decode()


@pytest.mark.parametrize("kw,code,text", [
    ({}, 1, "ctx or out is NULL"),
    ({"group_size": 48}, 2, "group_size 48"), ({"in_features": 80}, 2, "in_features 80"),
    ({"in_features": 0}, 2, "in_features 0"), ({"out_features": 0}, 2, "out_features 0"),
    ({"out_features": (1 << 24) + 1}, 2, "out_features"), ({"in_features": 1 << 21}, 2, "in_features"),
    ({"scales": None}, 1, "is NULL"), ({"packed": None}, 1, "is NULL"),
    ({"bias": 2}, 1, "misaligned"),
])
def test_linear_weights(kw, code, text):
    rc, got = upload(**kw)
    assert rc == code and text in got, got


@pytest.mark.parametrize("kw,text", [
    ({}, "ctx or the linear layer is NULL"), ({"dtype": 7}, "dtype must be known"),
    ({"dtype": 1, "out_dtype": 2}, "out_dtype"), ({"rows": -1}, "rows must be"),
    ({"rows": 1 << 30}, "rows must be"),
])
def test_linear_rows(kw, text):
    r = set_all(DmhLinearRows(0, 0, 2, ptr(512), 64, ptr(64), 8), kw)
    e = C.create_string_buffer(512)
    rc = lib().dmh_linear_forward(None, None, C.addressof(r), 0, e, 512)
    assert rc == 1 and text in e.value.decode()
    assert lib().dmh_linear_forward(None, None, None, 0, e, 512) == 1
    assert lib().dmh_free_linear(None, None) == 1


# ---- Python's own checks -------------------------------------------------------------------
class Block:
    device, handle = 0, None
    _lib = lib()


def arrays(**kw):
    a = {"codes": np.zeros((6, 2, 2, 16, 32), np.uint8), "scales": np.zeros((6, 2, 2, 16, 2), np.uint8),
         "pages": np.zeros((3, 4), np.int32), "past": np.zeros(3, np.int32)}
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,text", [
    ({"codes": np.zeros((6, 2, 16, 32), np.uint8)}, "codes must be"),
    ({"codes": np.zeros((6, 2, 2, 16, 32), np.int8)}, "codes must be a contiguous uint8"),
    ({"scales": np.zeros((6, 2, 2, 16, 4), np.uint8)}, "scales must be"),
    ({"scales": np.zeros((6, 2, 2, 16, 4), np.uint8)[..., ::2]}, "scales must be"),
    ({"pages": np.zeros((2, 4), np.int32)}, "pages must be"),
    ({"pages": np.zeros((3, 4), np.int64)}, "pages must be"),
    ({"pages": np.zeros(3, np.int32)}, "pages must be"),
    ({"past": np.zeros(3, np.uint32)}, "past must be"),
])
def test_python_arrays(kw, text):
    with pytest.raises(DismoenError, match=text):
        KVCache(Block, **arrays(**kw))


def test_python_rows():
    c = KVCache(Block, **arrays())
    off = np.array([0, 2], np.int32)
    b = SeqBatch(off, 2, 2, 3)
    k = np.zeros((2, 2, 64), np.float32)
    for bad, text in ((np.zeros((2, 2, 32), np.float32), "heads of 64"),
                      (np.zeros((2, 2, 128), np.float32)[..., ::2], "heads of 64"),
                      (np.zeros((2, 2, 64), np.float16), "heads of 64"),
                      (np.zeros((1, 2, 64), np.float32), "fewer rows")):
        with pytest.raises(DismoenError, match=text):
            c.write(k, bad, b)
    with pytest.raises(DismoenError, match="slots"):
        c.write(k, k, SeqBatch(off, 2, 2, 4))
    fixed = np.zeros((2, 2, 64), np.float32)
    fixed.flags.writeable = False
    with pytest.raises(DismoenError, match="read-only"):
        c.read(k, fixed, b)
    still = arrays()
    still["codes"].flags.writeable = False
    with pytest.raises(DismoenError, match="read-only"):
        KVCache(Block, **still)
    assert KVCache.shapes(6, 2, 16, 64) == ((6, 2, 2, 16, 32), (6, 2, 2, 16, 2))
