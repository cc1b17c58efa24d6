"""Refusals of the token mixer's entry points that need no GPU: arguments and,
for host arrays, the sequences are checked before the context is touched."""
import ctypes as C

import numpy as np
import pytest

from dismoen import lib
from dismoen._lib import DmhGatedDelta, DmhGatedNorm, DmhSeqBatch, DmhShortConv

F_DEVICE = 1
_keep = []


def ptr(a):
    _keep.append(a)
    return a.ctypes.data


def i32(*v):
    return ptr(np.array(v, np.int32))


def batch(offsets=(0, 2, 5), total=6, max_len=4, slots_n=3, slots=None, fresh=None):
    return DmhSeqBatch(len(offsets) - 1, total, max_len, slots_n, i32(*offsets),
                       None if slots is None else i32(*slots),
                       None if fresh is None else i32(*fresh))


def f32(n, at=0):
    return ptr(np.zeros(n + 8, np.float32)) + 4 * at


def conv(**kw):
    a = DmhShortConv(dtype=0, channels=8, width=4, silu=1, x=f32(48), x_stride=8, weight=f32(32),
                     bias=None, state=f32(72), y=f32(48), y_stride=8)
    return set_all(a, kw)


def delta(**kw):
    state = (ptr(np.zeros(3 * 2 * 64 + 8, np.float32)) + 15) // 16 * 16
    a = DmhGatedDelta(dtype=0, k_heads=1, v_heads=2, k_dim=8, v_dim=8, qk_norm=1, eps=1e-6,
                      scale=1.0, q=f32(48), k=f32(48), v=f32(96), a=f32(12), b=f32(12), q_stride=8,
                      k_stride=8, v_stride=16, a_stride=2, b_stride=2, a_log=f32(2), dt_bias=f32(2),
                      state=state, o=f32(96), o_stride=16)
    return set_all(a, kw)


def norm(**kw):
    a = DmhGatedNorm(dtype=0, stream_dtype=0, rows=3, groups=2, dim=4, post=1, gate_act=1, scale=1,
                     eps=1e-6, x=f32(24), gate=f32(24), residual=f32(24), stream=f32(24), y=f32(24),
                     x_stride=8, gate_stride=8, residual_stride=8, stream_stride=8, y_stride=8)
    return set_all(a, kw)


def set_all(a, kw):
    for k, v in kw.items():
        assert hasattr(a, k), k
        setattr(a, k, v)
    return a


def call(name, args, b=None, flags=0):
    e = C.create_string_buffer(512)
    f = getattr(lib(), f"dmh_{name}_forward")
    refs = [None if s is None else C.byref(s) for s in ([args] if name == "gated_norm" else [args, b])]
    rc = f(None, *refs, flags, e, len(e))
    return rc, e.value.decode()


CTX = (1, "ctx is NULL")  # what a call without a fault in its arguments ends with here


@pytest.mark.parametrize("kw,b,code,text", [
    ({}, {}, *CTX),
    ({"width": 2}, {}, *CTX),
    ({"bias": 64}, {}, *CTX),
    ({"dtype": 3}, {}, 1, "unknown dtype"),
    ({"channels": 0}, {}, 2, "channels 0"),
    ({"channels": (1 << 20) + 1}, {}, 2, "channels"),
    ({"width": 1}, {}, 2, "width 1"),
    ({"width": 5}, {}, 2, "width 5"),
    ({"x": None}, {}, 1, "is NULL"),
    ({"weight": None}, {}, 1, "is NULL"),
    ({"state": None}, {}, 1, "is NULL"),
    ({"y": None}, {}, 1, "is NULL"),
    ({"x_stride": 7}, {}, 1, "stride"),
    ({"y_stride": -8}, {}, 1, "stride"),
    ({"y_stride": 1 << 41}, {}, 1, "stride"),
])
def test_conv_arguments(kw, b, code, text):
    rc, got = call("short_conv", conv(**kw), batch(**b))
    assert rc == code and text in got, got


def test_conv_overlap():
    x = f32(200)
    assert "overlap" in call("short_conv", conv(x=x, y=x), batch())[1]
    assert "overlap" in call("short_conv", conv(x=x, y=x + 4 * 20), batch())[1]
    assert "overlap" in call("short_conv", conv(x=x, state=x + 4 * 47), batch())[1]
    # rows side by side in one buffer are apart
    assert CTX[1] in call("short_conv", conv(x=x, y=x + 32, x_stride=16, y_stride=16), batch())[1]
    assert "overlap" in call("short_conv", conv(x=x, y=x + 28, x_stride=16, y_stride=16),
                             batch())[1]
    assert "overlap" in call("short_conv", conv(x=x, y=x + 36, x_stride=16, y_stride=16),
                             batch())[1]


@pytest.mark.parametrize("name,make", [("short_conv", conv), ("gated_delta", delta)])
@pytest.mark.parametrize("b,text", [
    (dict(), CTX[1]),
    (dict(slots=(2, 0)), CTX[1]),
    (dict(slots=(-1, 0), offsets=(7, 9, 3)), "sequence 1: offsets"),  # skipped ones are not looked at
    (dict(slots=(-1, -5), offsets=(7, 9, 3)), CTX[1]),
    (dict(offsets=(0, 0, 0), slots=(1, 1)), CTX[1]),  # no rows: nothing is shared
    (dict(offsets=(0, 2, 7)), "sequence 1: offsets"),
    (dict(offsets=(-1, 2, 5)), "sequence 0: offsets"),
    (dict(offsets=(3, 2, 5)), "sequence 0: offsets"),
    (dict(offsets=(0, 4, 2, 5), slots=(0, -1, 1)), "sequence 2: offsets"),  # rows of sequence 0
    (dict(offsets=(0, 4, 2, 3, 5), slots=(0, -1, -1, 1)), "sequence 3: offsets"),
    (dict(offsets=(0, 4, 0, 0), slots=(0, -1, -1)), CTX[1]),  # padding
    (dict(offsets=(0, 5, 5)), "sequence 0: longer than max_seq_len"),
    (dict(slots=(0, 3)), "sequence 1: slot outside"),
    (dict(slots=(1, 1)), "sequence 1: names the state"),
    (dict(slots_n=1), "num_slots must be num_seqs"),
    (dict(slots_n=-1), "must not be negative"),
    (dict(total=-1), "must not be negative"),
    (dict(max_len=0), "max_seq_len must be positive"),
])
def test_sequences(name, make, b, text):
    rc, got = call(name, make(), batch(**b))
    assert rc == 1 and text in got, got


@pytest.mark.parametrize("name,make", [("short_conv", conv), ("gated_delta", delta)])
def test_batch_pointers(name, make):
    assert "batch is NULL" in call(name, make(), None)[1]
    assert "args is NULL" in call(name, None, batch())[1]
    b = batch()
    b.offsets = None
    assert "offsets is NULL" in call(name, make(), b)[1]
    # device arrays are not read on the host
    b.offsets = 64
    assert CTX[1] in call(name, make(), b, F_DEVICE)[1]


@pytest.mark.parametrize("kw,code,text", [
    ({}, *CTX),
    ({"a_log": None, "dt_bias": None}, *CTX),
    ({"dt_bias": None}, *CTX),
    ({"qk_norm": 0, "eps": float("nan")}, *CTX),
    ({"a_log": None}, 1, "dt_bias without a_log"),
    ({"dtype": -1}, 1, "unknown dtype"),
    ({"k_heads": 0}, 2, "k_heads 0"),
    ({"v_heads": 0}, 2, "v_heads 0"),
    ({"k_heads": 2, "v_heads": 3}, 2, "multiple"),
    ({"k_heads": 2, "v_heads": 1}, 2, "multiple"),
    ({"v_heads": 4097}, 2, "v_heads"),
    ({"k_dim": 12}, 2, "k_dim 12"),
    ({"k_dim": 264}, 2, "k_dim 264"),
    ({"k_dim": 0}, 2, "k_dim 0"),
    ({"v_dim": 4}, 2, "v_dim 4"),
    ({"v_dim": 512}, 2, "v_dim 512"),
    ({"scale": float("inf")}, 1, "scale"),
    ({"eps": -1e-6}, 1, "eps"),
    ({"eps": float("inf")}, 1, "eps"),
    ({"q": None}, 1, "is NULL"),
    ({"b": None}, 1, "is NULL"),
    ({"state": None}, 1, "is NULL"),
    ({"o": None}, 1, "is NULL"),
    ({"state": 4100}, 1, "16-byte"),
    ({"q_stride": 7}, 1, "stride"),
    ({"v_stride": 15}, 1, "stride"),
    ({"a_stride": 1}, 1, "stride"),
    ({"o_stride": 0}, 1, "stride"),
])
def test_delta_arguments(kw, code, text):
    rc, got = call("gated_delta", delta(**kw), batch())
    assert rc == code and text in got, got


def test_delta_overlap_and_size():
    for name in "qkvab":
        a = delta()
        a.o = getattr(a, name)
        assert "overlap" in call("gated_delta", a, batch())[1]
        a = delta()
        a.state = getattr(a, name) // 16 * 16
        assert "overlap" in call("gated_delta", a, batch())[1]
    a = delta()
    a.o = a.state
    assert "overlap" in call("gated_delta", a, batch())[1]
    b = batch()
    b.num_seqs = b.num_slots = 1 << 24
    rc, got = call("gated_delta", delta(), b, F_DEVICE)
    assert rc == 2 and "too many sequences" in got


@pytest.mark.parametrize("kw,code,text", [
    ({}, *CTX),
    ({"gate_act": 0, "gate": None, "residual": None, "y": None}, *CTX),
    ({"stream": None}, *CTX),
    ({"rows": 0}, *CTX),
    ({"dtype": 2, "stream_dtype": 2}, *CTX),
    ({"dtype": 2, "stream_dtype": 1}, 1, "stream_dtype"),
    ({"dtype": 0, "stream_dtype": 2}, 1, "stream_dtype"),
    ({"dtype": 5, "stream_dtype": 5}, 1, "dtype"),
    ({"rows": -1}, 2, "rows -1"),
    ({"groups": 0}, 2, "groups 0"),
    ({"dim": 0}, 2, "dim 0"),
    ({"dim": 8193}, 2, "dim 8193"),
    ({"gate_act": 3}, 1, "gate_act"),
    ({"eps": 0.0}, 1, "eps"),
    ({"eps": float("nan")}, 1, "eps"),
    ({"x": None}, 1, "is NULL"),
    ({"gate": None}, 1, "is NULL"),
    ({"stream": None, "y": None}, 1, "both NULL"),
    ({"x_stride": 7}, 1, "stride"),
    ({"y_stride": 7}, 1, "stride"),
    ({"residual_stride": 0}, 1, "stride"),
])
def test_norm_arguments(kw, code, text):
    rc, got = call("gated_norm", norm(**kw))
    assert rc == code and text in got, got


def test_norm_overlap():
    for out in ("stream", "y"):
        for name in ("x", "gate", "residual"):
            a = norm()
            setattr(a, out, getattr(a, name))
            text = call("gated_norm", a)[1]
            allowed = out == "stream" and name != "gate"  # in place
            assert (CTX[1] if allowed else "overlap") in text
            setattr(a, out, getattr(a, name) + 4)
            assert "overlap" in call("gated_norm", a)[1]
    a = norm()
    a.y = a.stream
    assert "overlap" in call("gated_norm", a)[1]


def test_operators_refuse_wrong_arrays():
    """The Python operators' own checks (shapes, types, sides), without a device."""
    from dismoen import DismoenError, GatedDelta, GatedNorm, SeqBatch, ShortConv

    class Blk:
        device, handle, _lib = 0, None, lib()

    def z(*s, t=np.float32):
        return np.zeros(s, t)

    off = np.array([0, 2, 5], np.int32)
    b = SeqBatch(off, 5, 4, 3)
    conv = ShortConv(Blk, z(8, 4))
    ok = (z(5, 8), z(3, 3, 8), b, z(5, 8))
    bad = [(z(5, 9), ok[1], b, ok[3]), (ok[0], z(3, 3, 8, t=np.float16), b, ok[3]),
           (ok[0], z(2, 3, 8), b, ok[3]), (z(4, 8), ok[1], b, ok[3]),
           (ok[0], ok[1], b, z(5, 8, t=np.float16)), (z(5, 16)[:, ::2], ok[1], b, ok[3]),
           (z(5, 8, t=np.float64), ok[1], b, ok[3]), (ok[0], z(3, 8, 3).swapaxes(1, 2), b, ok[3])]
    with pytest.raises(DismoenError, match="ctx is NULL"):
        conv(*ok)
    for args in bad:
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            conv(*args)
    for args in ((off.astype(np.int64), 5, 4, 3), (off[::2], 5, 4, 3)):
        with pytest.raises(DismoenError):
            SeqBatch(*args)
    with pytest.raises(DismoenError):
        SeqBatch(off, 5, 4, 3, slots=np.zeros(3, np.int32))
    delta = GatedDelta(Blk, 1, 2, 8, 8, a_log=z(2))
    args = [z(5, 1, 8), z(5, 1, 8), z(5, 2, 8), z(5, 2), z(5, 2), z(3, 2, 8, 8), b, z(5, 2, 8)]
    with pytest.raises(DismoenError, match="ctx is NULL"):
        delta(*args)
    for i, other in ((0, z(5, 2, 8)), (3, z(5, 1)), (5, z(3, 2, 8, 9)), (7, z(4, 2, 8)),
                     (2, z(5, 2, 8, t=np.float16))):
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            delta(*(args[:i] + [other] + args[i + 1:]))
    norm = GatedNorm(Blk, 4, 2, gate="silu", edge=True)
    x = z(3, 2, 4)
    with pytest.raises(DismoenError, match="ctx is NULL"):
        norm(x, z(3, 2, 4), z(3, 2, 4), gate=z(3, 2, 4))
    for kw in ({}, {"gate": z(3, 2, 5), "y": z(3, 2, 4)}, {"gate": z(3, 2, 4)},
               {"gate": z(4, 2, 4), "y": z(3, 2, 4)}):
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            norm(x, z(3, 2, 4), **kw)
    for kw in ({"gate": "relu"}, {"post": False, "gamma": z(4)}, {"edge_gamma": z(4)},
               {"gamma": z(5)}):
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            GatedNorm(Blk, 4, 2, **kw)


@pytest.mark.parametrize("name,make", [("short_conv", conv), ("gated_delta", delta)])
def test_rows_of_a_call(name, make):
    """Row numbers are 32 bits wide, with room for a step past the last one."""
    assert "below 2^30" in call(name, make(), batch(total=1 << 30))[1]
    # (addresses that rows of 64 bytes leave apart; not read on the host)
    far = {f: (2 + i) << 40 for i, f in enumerate(
        ["x", "y", "state"] if name == "short_conv" else [*"qkvabo", "state"])}
    assert CTX[1] in call(name, make(**far), batch(total=(1 << 30) - 1), F_DEVICE)[1]


def test_no_rows():
    """A call without rows needs no arrays (an empty tensor has no address)."""
    a = norm(rows=0, x=None, gate=None, residual=None, stream=None, y=None)
    assert CTX[1] in call("gated_norm", a)[1]
    for name, make, fields in (("short_conv", conv, "xy"), ("gated_delta", delta, "qkvabo")):
        a = make(**{f: None for f in fields})
        assert CTX[1] in call(name, a, batch((0, 0, 0), total=0))[1]


def test_batch_values_and_places():
    """Python's integers are wider than the call's, and a batch has a device."""
    from dismoen import DismoenError, SeqBatch, ShortConv

    class Blk:
        device, handle, _lib = 0, None, lib()

    off = np.array([0, 2, 5], np.int32)
    for args in ((off, 1 << 32, 4, 3), (off, 5, 1 << 31, 3), (off, 5, 4, (1 << 32) + 3),
                 (off, -1, 4, 3), (off[:0], 5, 4, 3)):
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            SeqBatch(*args)
    b = SeqBatch(off, 5, 4, 3)
    conv = ShortConv(Blk, np.zeros((8, 4), np.float32))
    args = [np.zeros((5, 8), np.float32), np.zeros((3, 3, 8), np.float32), b,
            np.zeros((5, 8), np.float32)]
    with pytest.raises(DismoenError, match="ctx is NULL"):
        conv(*args)
    b.device = 1
    with pytest.raises(DismoenError, match="batch"):
        conv(*args)


def test_port_block_refuses_wrong_arrays():
    torch = pytest.importorskip("torch")
    from dismoen import DismoenError, PortBlock

    class Blk:  # (a CPU tensor's device is -1)
        device, handle, _lib, dims = -1, None, lib(), {0: (8, 4, 2, 4, 4)}

    port = PortBlock(Blk, 0)
    ok = [torch.zeros(3, 8) for _ in range(4)]

    def run(i=None, other=None):
        a = list(ok)
        if i is not None:
            a[i] = other
        port(a[0], lambda v: v, *a[1:])

    with pytest.raises(DismoenError, match="ctx is NULL"):
        run()
    for i in range(4):
        for other in (torch.zeros(3, 8, dtype=torch.float16), torch.zeros(3, 9),
                      torch.zeros(3, 16)[:, ::2], torch.zeros(24), np.zeros((3, 8), np.float32)):
            with pytest.raises(DismoenError, match="CONFIG_ERROR.*must be contiguous float32"):
                run(i, other)
    with pytest.raises(DismoenError, match="CONFIG_ERROR"):
        run(3, torch.zeros(2, 8))
