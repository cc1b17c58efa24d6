"""The layer and the block made of the token mixer's operators: what they refuse, and
that a refused call has changed nothing, without a GPU."""

import ctypes as C

import numpy as np
import pytest

import test_mixer_refusals as T
from dismoen import (DismoenError, GatedDelta, GatedDeltaMixer, GatedNorm, PortBlock, SeqBatch,
                     ShortConv, lib)


def port_blk(**kw):
    """A block without a device (a CPU tensor's device is -1)."""
    return type("Blk", (), {"device": -1, "handle": None, "_lib": lib(), "dims": {}, **kw})


def test_port_block_needs_a_4_bit_layer():
    torch = pytest.importorskip("torch")
    blk = port_blk(dims={0: (8, 4, 2, 4, 4)}, gguf_dims={1: (8, 4, 2, 4, 4)})
    for layer in (1, 2):  # a GGUF layer, and none
        with pytest.raises(DismoenError, match=f"CONFIG_ERROR.*layer {layer} is not an uploaded"):
            PortBlock(blk, layer)
    port = PortBlock(blk, 0)
    a = [torch.zeros(3, 8) for _ in range(4)]

    def run():
        port(a[0], lambda v: v, *a[1:])

    with pytest.raises(DismoenError, match="ctx is NULL"):
        run()
    # the slot's layer of the moment: replaced by one of other rows, and freed
    blk.dims[0] = (16, 4, 2, 4, 4)
    with pytest.raises(DismoenError, match="CONFIG_ERROR.*replaced"):
        run()
    del blk.dims[0]
    with pytest.raises(DismoenError, match="CONFIG_ERROR.*not an uploaded"):
        run()


def test_port_block_refuses_other_rows_of_the_mixer():
    torch = pytest.importorskip("torch")
    port = PortBlock(port_blk(dims={0: (8, 4, 2, 4, 4)}), 0)
    rows = (6, 1, 8)
    for shape in ((6, 8), (6, 1, 8), (2, 3, 8), (1, 6, 8)):
        assert port._mixed(torch.zeros(shape), rows).shape == rows
    for out in (None, 1.0, torch.zeros(5, 8), torch.zeros(8, 6), torch.zeros(48), torch.zeros(())):
        with pytest.raises(DismoenError, match="CONFIG_ERROR.*mix must return 6 rows of 8"):
            port._mixed(out, rows)


class Counted:
    """The library without a device: which calls were to run, and the real checks of
    those that were only to be checked (which end at the missing context)."""
    CHECK = 0x80

    def __init__(self):
        self.ran = []

    def __getattr__(self, name):
        def call(*args):
            flags = args[-3]
            if not flags & self.CHECK:
                self.ran.append(name)
                return 0
            rc = getattr(lib(), name)(*args)
            text = C.string_at(args[-2])
            return 0 if rc and b"ctx is NULL" in text else rc
        return call


def test_mixer_refuses_before_anything_runs():
    hk, hv, dk, dv, rows = 1, 2, 8, 8, 5
    ch = 2 * hk * dk + hv * dv

    def z(*shape, t=np.float32):
        return np.zeros(shape, t)

    fake = Counted()
    blk = port_blk(_lib=fake)
    mixer = GatedDeltaMixer(blk, hk, hv, dk, dv, z(ch, 4), z(hv), z(hv), z(dv))
    batch = SeqBatch(np.array([0, 2, 5], np.int32), rows, 4, 3)
    ok = dict(mixed=z(rows, ch), z=z(rows, hv, dv), b=z(rows, hv), a=z(rows, hv),
              conv_state=z(3, 3, ch), state=z(3, hv, dk, dv), batch=batch, work=z(rows, ch),
              out=z(rows, hv, dv))
    mixer(**ok)
    assert fake.ran == ["dmh_short_conv_forward", "dmh_gated_delta_forward",
                        "dmh_gated_norm_forward"]
    for name, other in (("z", z(rows - 1, hv, dv)), ("z", z(rows, hv, dv, t=np.float16)),
                        ("a", z(rows, hv + 1)), ("b", z(rows - 1, hv)),
                        ("state", z(3, hv, dk, dv + 8)), ("state", z(2, hv, dk, dv)),
                        ("conv_state", z(3, 2, ch)), ("out", z(rows, hv, dv, t=np.float16)),
                        ("out", z(rows - 1, hv, dv)), ("work", z(rows - 1, ch)),
                        # what only the library sees: outputs on inputs
                        ("out", ok["work"][:, :hv * dv].reshape(rows, hv, dv, copy=False)),
                        ("out", ok["z"]), ("a", ok["out"][:, 0, :hv])):
        fake.ran.clear()
        with pytest.raises(DismoenError):
            mixer(**{**ok, name: other})
        assert not fake.ran, (name, other.shape)


def test_host_arrays_that_are_written_must_be_writable():
    """bytes, a broadcast value, a file mapped to be read: an operator that wrote there
    would change what others hold, or end the process."""
    blk = port_blk(_lib=Counted())
    batch = SeqBatch(np.array([0, 2, 5], np.int32), 5, 4, 3)

    def z(*shape):
        return np.zeros(shape, np.float32)

    def fixed(*shape):
        return np.frombuffer(bytes(4 * int(np.prod(shape))), np.float32).reshape(shape)

    conv, delta = ShortConv(blk, fixed(8, 4)), GatedDelta(blk, 1, 2, 8, 8, a_log=fixed(2))
    norm = GatedNorm(blk, 4, 2, gamma=fixed(4), edge=True)
    r, ins = fixed(5, 8), (fixed(5, 1, 8), fixed(5, 1, 8), fixed(5, 2, 8), fixed(5, 2), fixed(5, 2))
    conv(r, z(3, 3, 8), batch, z(5, 8))
    delta(*ins, z(3, 2, 8, 8), batch, z(5, 2, 8))
    norm(fixed(3, 2, 4), z(3, 2, 4), z(3, 2, 4), residual=fixed(3, 2, 4))
    for f in (lambda: conv(r, fixed(3, 3, 8), batch, z(5, 8)),
              lambda: conv(r, z(3, 3, 8), batch, fixed(5, 8)),
              lambda: conv(r, z(3, 3, 8), batch, np.broadcast_to(np.float32(0), (5, 8))),
              lambda: delta(*ins, fixed(3, 2, 8, 8), batch, z(5, 2, 8)),
              lambda: delta(*ins, z(3, 2, 8, 8), batch, fixed(5, 2, 8)),
              lambda: norm(fixed(3, 2, 4), fixed(3, 2, 4), z(3, 2, 4)),
              lambda: norm(fixed(3, 2, 4), None, fixed(3, 2, 4))):
        with pytest.raises(DismoenError, match="CONFIG_ERROR"):
            f()


def test_sequences_that_one_launch_holds():
    """The launch of the chunks counts units in eights: the last few below 2^23 are too
    many for it, and not for the one row by row."""
    for seqs, max_len, fits in (((1 << 23) - 1, 16, True), (1 << 23, 16, False),
                                ((1 << 23) - 1, 17, False), ((1 << 23) - 8, 17, True),
                                ((1 << 23) - 7, 17, False)):
        b = T.batch(max_len=max_len)
        b.num_seqs = b.num_slots = seqs
        # (addresses apart from each other, which the host does not read)
        far = {f: (2 + i) << 40 for i, f in enumerate([*"qkvabo", "state"])}
        rc, text = T.call("gated_delta", T.delta(v_heads=1, **far), b, T.F_DEVICE)
        assert ("ctx is NULL" if fits else "too many sequences") in text, (seqs, max_len, text)
