"""Steps of a cache that are replayed from a graph, and left."""

import pytest
import torch

from rbf_attention_b200 import lm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB = 130


def test_a_replayed_step_that_is_left():
    """The replay filled a block and put the next one's rows in its place: what is left of the sequences is nothing, and answers
    from the cache are those of a fresh one."""
    torch.manual_seed(0)
    model = lm.CausalLM(VOCAB, 128, 2, 2, 300, attention_type="rbf_triton", num_registers=0).to(DEV, torch.bfloat16)
    ids = torch.randint(0, VOCAB, (2, 40), generator=torch.Generator().manual_seed(1)).to(DEV)
    cache = model.new_cache(2, 300)
    tokens = ids[:, :20].clone()

    def step():                             # 20 tokens: a block fills up and the next one begins
        x, pending = model.token_emb(tokens), None
        for i, block in enumerate(model.blocks):
            x, pending = block.forward_cached(x, cache, i, False, pending)

    with torch.no_grad():
        model.forward_cached(ids[:, :10], cache)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            cache.begin(20)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
        torch.cuda.current_stream().wait_stream(stream)
        graph.replay()
        cache.end()
        before = cache.read(0)
        cache.begin(20)
        graph.replay()
        cache.abort()
        # either the tokens are as they were, or the sequences are empty
        for s in range(2):
            n = cache.length(s)
            if n:
                assert torch.equal(cache.read(0, [s], n)[0], before[0][s:s + 1, :, :n])
        assert [cache.length(s) for s in range(2)] == [0, 0] and cache.free_pages == cache.num_pages
        assert torch.equal(model.generate(ids, 30, cache=cache), model.generate(ids, 30, cache=model.new_cache(2, 300)))
        cache.free([0, 1])
        model.forward_cached(ids, cache)
        cache.begin(20)                     # nothing has run: the caller knows
        cache.abort(written=False)
        assert [cache.length(s) for s in range(2)] == [40, 40]
        cache.begin(20)
        cache.abort(written=True)
        assert [cache.length(s) for s in range(2)] == [0, 0]
