"""Reading a KV cache back on the stream that wrote it."""
import pytest
import torch

import dli
from support import one_node_graph

pytestmark = pytest.mark.gpu


def normal(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


@pytest.mark.parametrize("format", ["", "fp8"])
@pytest.mark.parametrize("foreign", [True, False])
def test_read_waits_for_the_stream_that_wrote(format, foreign):
    """Tokens written over others behind a long queue of work: the read on the same stream sees the new
    ones, whatever torch's current stream is."""
    e = dli.Engine().load_plugin()
    e.configure_kv_cache(block_size=16, max_seq_len=64, format=format)
    graph = one_node_graph("attention", ["q", "k", "v", "p"], attrs={"causal": True, "kv_cache": "c"})
    q, p = normal((2, 4, 20, 64), 1), torch.tensor([3, 9]).cuda()
    busy = torch.randn((4096, 4096), device="cuda")
    old, new = ({"q": q, "k": normal((2, 2, 20, 64), s), "v": normal((2, 2, 20, 64), s + 1), "p": p}
                for s in (2, 4))
    e.run(graph, new)
    torch.cuda.synchronize()
    want = [x.clone() for x in e.read_kv_cache("c", 5, 20)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        e.run(graph, old)
        torch.cuda.synchronize()
        current = torch.cuda.current_stream() if foreign else side
        with torch.cuda.stream(side):
            for _ in range(20):
                busy @ busy
        with torch.cuda.stream(current):
            out = e.run(graph, new, stream=side.cuda_stream)
            got = e.read_kv_cache("c", 5, 20, stream=side.cuda_stream)
        side.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.cuda.current_stream().cuda_stream != side.cuda_stream
        del out
