"""What a call of attention needs before it is captured: a call of the same heads and number
of sequences, whatever the lengths of either."""
import pytest
import torch

from dismoen import CacheAttention, MoEBlock
from test_gpu_cache import TYPES, Cache, gen, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES.values(), ids=TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (12, 2, 128), (8, 8, 256), (40, 1, 96)])
def test_single_tokens_before_prompts(heads, kv_heads, dim, t):
    """Single tokens are enough before prompts are captured; replays give the bits of the call."""
    g = gen("capture", heads, dim)
    lens = [150, 1, 70]
    with MoEBlock(0) as blk:
        c = Cache(blk, g, [100, 40, 7], lens, kv_heads, dim, 16)
        c.fill(blk, [torch.randn((2, p + n, kv_heads, dim), generator=g).to(t).cuda()
                     for p, n in zip(c.past, c.rows)])
        rows = sum(lens)
        q = rand(g, rows, heads, dim, t=t)
        out, one = torch.zeros_like(q), torch.zeros_like(q[:3])
        attend, batch, single = CacheAttention(blk, heads), c.batch(), c.batch([1, 1, 1])
        torch.cuda.synchronize()
        attend(q, c.cache, single, one)
        blk.sync()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        blk.set_stream(stream.cuda_stream)
        with torch.cuda.graph(graph, stream=stream):
            attend(q, c.cache, batch, out)
        blk.set_stream(None)
        for i in range(3):
            q.copy_(rand(g, *q.shape, t=t))
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            blk.sync()
            replayed = out.clone()
            attend(q, c.cache, single, one)  # in the same memory
            out.zero_()
            torch.cuda.synchronize()
            attend(q, c.cache, batch, out)
            blk.sync()
            assert torch.equal(replayed, out) and bool((out != 0).any())
        del graph
