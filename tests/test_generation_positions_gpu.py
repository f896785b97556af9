"""Answers that end where the model's positions do."""

import pytest
import torch

from rbf_attention_b200 import lm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VOCAB, LIMIT = 130, 600


def _model(pos, registers=2):
    torch.manual_seed(0)
    model = lm.CausalLM(VOCAB, d_model=128, num_layers=2, num_heads=2, max_seq_len=LIMIT, pos_emb_type=pos, num_registers=registers,
                        attention_type="rbf_triton")
    return model.to(DEV, torch.bfloat16).requires_grad_(False)


def _ids(B, T):
    return torch.randint(0, VOCAB, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)


@pytest.mark.parametrize("pos", ["rope", "learned"])
def test_the_last_answer_needs_no_position(pos):
    """The last id is not read again: a prompt as long as the positions has one, a shorter one as many more."""
    model = _model(pos)
    ids = _ids(2, LIMIT)
    assert torch.equal(model.generate(ids, 1)[:, 0], model.forward_cached(ids, model.new_cache(2, LIMIT)).argmax(-1))
    out = model.generate(ids[:, :LIMIT - 3], 4)
    cache = model.new_cache(2, LIMIT)
    assert torch.equal(out, model.generate(ids[:, :LIMIT - 3], 4, cache=cache))
    assert cache.length(0) == LIMIT + model.num_registers
    with pytest.raises(ValueError, match="positions end"):
        model.generate(ids[:, :LIMIT - 3], 5)


def test_no_page_is_taken_for_it():
    model = _model("rope", registers=0)
    asked = []
    new_cache = model.new_cache
    model.new_cache = lambda *args: asked.append(new_cache(*args)) or asked[-1]
    model.generate(_ids(2, 250), 7)
    assert asked[0].num_pages == 2 and asked[0].free_pages == 0
