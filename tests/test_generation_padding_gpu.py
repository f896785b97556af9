"""Padded batches of a model with a cache."""

import pytest
import torch
import torch.nn.functional as F

from rbf_attention_b200 import lm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB, LIMIT = 130, 600


@pytest.mark.parametrize("all_logits", [False, True])
@pytest.mark.parametrize("pos,xsa", [("rope", False), ("rope", True), ("learned", False)])
def test_padding_may_reach_behind_the_positions(pos, xsa, all_logits):
    """Only real tokens need a place."""
    torch.manual_seed(0)
    model = lm.CausalLM(VOCAB, d_model=128, num_layers=2, num_heads=2, max_seq_len=LIMIT, pos_emb_type=pos, num_registers=2,
                        attention_type="rbf_triton")
    for block in model.blocks:
        block.attn.apply_xsa = xsa
    model = model.to(DEV, torch.bfloat16).requires_grad_(False)
    ids, new = torch.randint(0, VOCAB, (2, LIMIT), generator=torch.Generator().manual_seed(1)).to(DEV), [LIMIT, 70]
    padded = F.pad(ids, (0, 37), value=VOCAB - 1)
    caches = [model.new_cache(2, LIMIT) for _ in range(2)]
    want = model.forward_cached(ids, caches[0], new, all_logits=all_logits)
    got = model.forward_cached(padded, caches[1], new, all_logits=all_logits)
    if all_logits:
        assert got.shape[1] == padded.shape[1]
        for b, n in enumerate(new):
            assert torch.equal(got[b, :n], want[b, :n])
    else:
        assert torch.equal(got, want)
    for layer in range(2):
        assert all(torch.equal(a, b) for a, b in zip(caches[0].read(layer), caches[1].read(layer)))
