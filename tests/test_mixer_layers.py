"""The layer and the block made of the token mixer's operators: what they refuse, and
that a refused call has changed nothing, without a GPU."""

import pytest

from dismoen import DismoenError, PortBlock, lib


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
