"""Linear layers whose weights take more threads to re-tile than a launch has."""
import pytest
import torch

import mixer_ref as M
from dismoen import MoEBlock, QuantLinear

pytestmark = pytest.mark.gpu


def test_more_weights_than_a_launch_has_threads_for():
    """2^24 x 2^13 weights, a thread for 32 of them: 2^32.  Sums of 8192 columns in 32s, as in
    test_gpu_linear: 256 + 8 for each of bf16's one part, and 8."""
    n, k, group = 1 << 24, 1 << 13, 256
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("needs 150 GB")
    g = torch.Generator().manual_seed(5)
    q = torch.randint(-7, 8, (64, k), generator=g)
    flat = (q & 15).to(torch.uint8)
    rows = (flat[:, 0::2] | (flat[:, 1::2] << 4)).cuda()
    packed = torch.full((n, k // 2), 0x21, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, k // group), 0.5, dtype=torch.float16, device="cuda")
    some = [0, 1, 15, 16, (1 << 23) - 1, 1 << 23, n - 17, n - 16, n - 1]
    some += [i * (n // 64) + 77 for i in range(64 - len(some))]
    packed[some], scales[some] = rows, 0.25
    x = torch.randn((2, k), generator=g).bfloat16().cuda()
    y = torch.empty((2, n), dtype=torch.float32, device="cuda")
    with MoEBlock(0) as blk:
        lin = QuantLinear(blk, n, k, scales.view(-1), packed.view(-1), group)
        del packed
        torch.cuda.synchronize()
        lin(x, y)
        blk.sync()
        lin.close()
    xd, w = x.double().cpu(), q.double() * 0.25
    M.close(y[:, some], xd @ w.T, xd.abs() @ w.abs().T, 272)
    rest = torch.tensor([1.0, 2.0], dtype=torch.float64).repeat(k // 2) * 0.5
    other = [i for i in range(2, n, n // 61) if i not in some]
    M.close(y[:, other], (xd @ rest)[:, None].expand(2, len(other)),
            (xd.abs() @ rest)[:, None], 272)
    torch.cuda.empty_cache()
