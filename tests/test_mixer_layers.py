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


def test_port_block_refuses_other_rows_of_the_mixer():
    torch = pytest.importorskip("torch")
    port = PortBlock(port_blk(dims={0: (8, 4, 2, 4, 4)}), 0)
    rows = (6, 1, 8)
    for shape in ((6, 8), (6, 1, 8), (2, 3, 8), (1, 6, 8)):
        assert port._mixed(torch.zeros(shape), rows).shape == rows
    for out in (None, 1.0, torch.zeros(5, 8), torch.zeros(8, 6), torch.zeros(48), torch.zeros(())):
        with pytest.raises(DismoenError, match="CONFIG_ERROR.*mix must return 6 rows of 8"):
            port._mixed(out, rows)
