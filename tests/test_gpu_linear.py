"""Linear layers with 4-bit weights, against 64-bit products with the dequantiser's weights.

Tolerance: half a step of the output's type, plus roundings of 2^-24 of the sum of the
products' sizes: products are exact, a sum is taken 32 columns at a time (at most 6
roundings each) and over at most 8192 / 32 of these, in up to 16 waves and joined: 8 for
each part of x (of at most three) and each 128 columns of a wave's share cover sums that
grow one way; random ones stay far below.  STEPS counts 256 sums of one rounding each and
their inner 6, times three parts, at the largest size tested here (k of 4224: 132 sums)."""
import zlib

import numpy as np
import pytest
import torch

import mixer_ref as M
from dismoen import DismoenError, QuantLinear

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def gen(*seed):
    return torch.Generator().manual_seed(zlib.crc32(repr(seed).encode()))


def weights(g, n, k, group):
    q = torch.randint(-7, 8, (n, k), generator=g)
    scales = (torch.rand(n * k // group, generator=g) * 0.01 + 1e-3).half()
    flat = (q & 15).flatten().to(torch.uint8)
    packed = flat[0::2] | (flat[1::2] << 4)
    w = (q.view(n, -1, group).float() * scales.float().view(n, -1, 1)).bfloat16().double()
    return w.view(n, k), scales, packed


def check(got, x, w, bias, k):
    xd = x.double().cpu()
    want = xd @ w.T
    size = xd.abs() @ w.abs().T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    parts = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[x.dtype]
    M.close(got, want, size, parts * (k / 32 + 8) + 8)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (17, 96, 32), (50, 320, 64),
                                       (515, 4224, 32), (2048, 256, 256), (129, 1024, 128)])
@pytest.mark.parametrize("rows", [1, 3, 16, 17, 33, 64, 65, 200])
def test_linear(block, rows, n, k, group, t):
    g = gen(n, k, rows)
    w, scales, packed = weights(g, n, k, group)
    bias = torch.randn(n, generator=g) if rows % 2 else None
    x = torch.randn((rows, k), generator=g).to(t)
    lin = QuantLinear(block, n, k, scales.cuda(), packed.cuda(), group,
                      bias=None if bias is None else bias.cuda())
    for out in {t, torch.float32}:
        # strided rows: x from a wider projection, y into one
        wide = torch.full((rows + 1, k + 40), float("nan"), dtype=t, device="cuda")
        wide[:rows, 8:8 + k] = x
        y = torch.full((rows + 1, n + 5), 3.0, dtype=out, device="cuda")
        torch.cuda.synchronize()
        assert lin(wide[:rows, 8:8 + k], y[:rows, 2:2 + n]) is not None
        block.sync()
        check(y[:rows, 2:2 + n], x, w, bias, k)
        assert (y[rows:] == 3).all() and (y[:, :2] == 3).all() and (y[:, 2 + n:] == 3).all()
    lin.close()


@pytest.mark.parametrize("n,k,rows", [(1111, 544, 1300), (2401, 160, 2500), (33000, 64, 30),
                                      (1024, 96, 40), (1024, 128, 33), (4100, 32, 25)])
def test_rows_of_many_tiles(block, n, k, rows):
    """Many rows of x, and layers of many rows, of odd sizes."""
    g = gen("many")
    w, scales, packed = weights(g, n, k, 32)
    lin = QuantLinear(block, n, k, scales.cuda(), packed.cuda(), 32)
    for t in TYPES.values():
        x = torch.randn((rows, k), generator=g).to(t).cuda()
        y = torch.empty(rows, n, dtype=t, device="cuda")
        torch.cuda.synchronize()
        lin(x, y)
        block.sync()
        check(y, x, w, None, k)


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("n,k", [(32753, 32), (32768, 352), (33001, 1024), (32790, 1184), (32769, 1632),
                                 (40000, 2048), (32785, 2080), (32777, 4064), (32768, 4160)])
def test_few_rows_of_large_layers(block, n, k, t):
    """One to 17 rows of layers that take many tiles a workgroup, of whole and odd sizes: rows
    apart, rows that are not finite, and nothing written beside the results."""
    g = gen("large", n, k)
    w, scales, packed = weights(g, n, k, 32)
    bias = torch.randn(n, generator=g)
    lin = QuantLinear(block, n, k, scales.cuda(), packed.cuda(), 32, bias=bias.cuda())
    plain = QuantLinear(block, n, k, scales.cuda(), packed.cuda(), 32)
    for rows, out, layer in ((1, t, lin), (5, torch.float32, plain), (16, t, plain), (17, t, lin)):
        x = torch.randn((rows, k), generator=g).to(t)
        wide = torch.full((rows + 1, k + 40), float("nan"), dtype=t, device="cuda")
        wide[:rows, 8:8 + k] = x
        y = torch.full((rows + 1, n + 5), 3.0, dtype=out, device="cuda")
        torch.cuda.synchronize()
        layer(wide[:rows, 8:8 + k], y[:rows, 2:2 + n])
        block.sync()
        check(y[:rows, 2:2 + n], x, w, bias if layer is lin else None, k)
        assert (y[rows:] == 3).all() and (y[:, :2] == 3).all() and (y[:, 2 + n:] == 3).all()
        if rows == 5:
            clean = y.clone()
            wide[2, 8 + k - 1] = float("nan")
            torch.cuda.synchronize()
            layer(wide[:rows, 8:8 + k], y[:rows, 2:2 + n])
            block.sync()
            assert y[2, 2:2 + n].isnan().all()
            y[2] = clean[2]
            assert torch.equal(y, clean)
    lin.close()
    plain.close()


def test_rows_do_not_meet(block):
    """A row that is not finite makes its own results so, and no other's."""
    g = gen("nan")
    w, scales, packed = weights(g, 64, 256, 64)
    lin = QuantLinear(block, 64, 256, scales.cuda(), packed.cuda(), 64)
    for rows in (5, 40, 300):
        x = torch.randn((rows, 256), generator=g).bfloat16()
        clean, x[2, 100] = x.clone(), float("nan")
        y, z = (torch.empty(rows, 64, device="cuda") for _ in range(2))
        a, b = x.cuda(), clean.cuda()
        torch.cuda.synchronize()
        lin(a, y)
        lin(b, z)
        block.sync()
        assert y[2].isnan().all()
        keep = [i for i in range(rows) if i != 2]
        assert torch.equal(y[keep], z[keep])


def test_host_arrays(block):
    """numpy weights and rows give the device's bits."""
    g = gen("host")
    n, k, rows = 70, 160, 9
    w, scales, packed = weights(g, n, k, 32)
    bias = torch.randn(n, generator=g)
    x = torch.randn((rows, k), generator=g)
    y = torch.empty(rows, n, device="cuda")
    xd = x.cuda()
    dev = QuantLinear(block, n, k, scales.cuda(), packed.cuda(), 32, bias=bias.cuda())
    torch.cuda.synchronize()
    dev(xd, y)
    block.sync()
    host = QuantLinear(block, n, k, scales.numpy(), packed.numpy(), 32, bias=bias.numpy())
    out = np.full((rows, n), 2, np.float32)
    host(x.numpy(), out)
    assert np.array_equal(out, y.cpu().numpy())


def test_refused_weights(block):
    """What the dequantiser refuses, the upload refuses with its text."""
    g = gen("bad")
    _, scales, packed = weights(g, 8, 64, 32)
    bad = packed.clone()
    bad[100] = 0x18
    def changed(i, v):
        s = scales.clone()
        s[i] = v
        return s

    for s, p, text in ((scales, bad, "reserved nibble"),
                       (changed(5, 0.0), packed, "non-positive at group 5"),
                       (changed(3, float("inf")), packed, "NaN or Inf at group 3"),
                       (changed(7, -1.0), packed, "non-positive at group 7")):
        with pytest.raises(DismoenError, match=text) as e:
            QuantLinear(block, 8, 64, s.numpy(), p.numpy(), 32)
        assert e.value.code == 5
    QuantLinear(block, 8, 64, scales.numpy(), packed.numpy(), 32).close()


def test_from_a_quant_model(block, tmp_path):
    from dismoen import formats
    g = gen("file")
    w, scales, packed = weights(g, 96, 128, 32)
    path = str(tmp_path / "model.bin")
    formats.write_quant_file(path, "m", [("a.weight", [96, 128], scales.numpy().view(np.uint16),
                                          packed.numpy())], 32)
    with formats.scan_quant_file(path) as index:
        lin = QuantLinear.from_quant_model(block, index, "a.weight")
        with pytest.raises(DismoenError, match="not in the quant model"):
            QuantLinear.from_quant_model(block, index, "b.weight")
    x, y = torch.randn((4, 128), generator=g).cuda(), torch.empty(4, 96, device="cuda")
    torch.cuda.synchronize()
    lin(x, y)
    block.sync()
    check(y, x, w, None, 128)


@pytest.mark.parametrize("rows", [1, 16, 20, 400])
@pytest.mark.parametrize("n", [200, 20000, 33000])
def test_largest_values(block, n, rows):
    """The largest fp32 value, which has no bf16 above it; infinities stay in their row."""
    if n * rows > 4 << 20:
        n = 1500
    g = gen("largest", n)
    w, scales, packed = weights(g, n, 160, 32)
    lin = QuantLinear(block, n, 160, scales.cuda(), packed.cuda(), 32)
    for t in TYPES.values():
        x = torch.randn((rows, 160), generator=g).to(t)
        x[0, 77] = torch.finfo(t).max
        x[rows - 1, 3] = -torch.finfo(t).max
        y, z = (torch.empty(rows, n, device="cuda") for _ in range(2))
        a, b = x.cuda(), x.cuda()
        b[0, 100] = float("inf")
        torch.cuda.synchronize()
        lin(a, y)
        lin(b, z)
        block.sync()
        check(y, x, w, None, 160)
        assert not z[0].isfinite().any() and torch.equal(y[1:], z[1:])
    lin.close()


def test_too_many_rows(block):
    """More tiles than a launch holds are refused before anything is read."""
    import ctypes as C

    from dismoen._lib import DmhLinearRows
    g = gen("too many")
    _, scales, packed = weights(g, 1000, 64, 32)
    lin = QuantLinear(block, 1000, 64, scales.cuda(), packed.cuda(), 32)
    e = C.create_string_buffer(512)
    r = DmhLinearRows(2, 2, (1 << 30) - 1, 1 << 44, 64, 1 << 46, 1000)  # (addresses of nothing)
    rc = block._lib.dmh_linear_forward(block.handle, lin._l, C.addressof(r), 1, e, 512)
    assert rc == 2 and b"too many rows" in e.value


@pytest.mark.parametrize("rows", [3, 40, 700])
@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
def test_captured(rows, t):
    """Replays take new rows and give the bits of the same call made at once; one that needs
    memory which a capture cannot make is refused."""
    from dismoen import MoEBlock
    g = gen("captured", rows)
    with MoEBlock(0) as blk:
        w, scales, packed = weights(g, 2100, 256, 32)
        lin = QuantLinear(blk, 2100, 256, scales.cuda(), packed.cuda(), 32)
        x, y = torch.zeros(rows, 256, dtype=t, device="cuda"), torch.zeros(rows, 2100, device="cuda")
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        mark = torch.zeros(1, device="cuda")
        torch.cuda.synchronize()
        if rows == 700 and t is not torch.bfloat16:
            blk.set_stream(stream.cuda_stream)
            with torch.cuda.graph(graph, stream=stream):
                with pytest.raises(DismoenError, match="before the capture"):
                    lin(x, y)
                mark.add_(1)
            blk.set_stream(None)
            graph = torch.cuda.CUDAGraph()
        lin(x, y)
        blk.sync()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(DismoenError, match="being captured"):
                QuantLinear(blk, 2100, 256, scales.numpy(), packed.numpy(), 32)
            lin(x, y)
        blk.set_stream(None)
        for _ in range(3):
            x.copy_(torch.randn((rows, 256), generator=g))
            y.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone()
            torch.cuda.synchronize()
            lin(x, y)
            blk.sync()
            assert torch.equal(got, y)
            check(y, x, w, None, 256)
        del graph
        lin.close()
        with pytest.raises(DismoenError, match="linear layer is NULL"):
            lin(x, y)
