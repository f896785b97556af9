"""float32 weights under autocast, as the reference trains, with a cache of the caller's own in the type that autocast computes in."""

import pytest
import torch

from rbf_attention_b200 import lm
from rbf_attention_b200.cache import PagedCache
from test_generation_gpu import DEV, VOCAB, _bound, _ids, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,pos,xsa", [("rbf_triton", "rope", False), ("rbf_triton", "learned", True), ("rbf_non_softmax", "rope", True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_answers_under_autocast(dtype, kind, pos, xsa):
    """Portions against the model's forward: its roundings, and keys and values that are held in steps of 1/127 of a block's largest
    magnitude - of some four root mean squares, so off by 4 / 127 / sqrt(12) = 0.9 % of them."""
    model = _model(kind, pos, registers=2, dtype=torch.float32, xsa=xsa)
    ids = _ids(2, 60)
    with torch.autocast("cuda", dtype=dtype):
        cache = PagedCache(len(model.blocks), 2, 64, 2, 62, dtype=dtype, device=DEV)
        first = model.forward_cached(ids[:, :40], cache, all_logits=True)
        rest = torch.cat([model.forward_cached(ids[:, t:t + 1], cache, all_logits=True) for t in range(40, 60)], 1)
        want = model(ids)[0]
        answers = model.generate(ids[:, :10], 5, cache=PagedCache(len(model.blocks), 2, 64, 2, 62, dtype=dtype, device=DEV))
    assert first.dtype == rest.dtype == dtype and answers.shape == (2, 5) and int(answers.max()) < VOCAB
    bound = _bound(model.to(dtype)) + 0.01
    for got, ref in ((first, want[:, :40]), (rest, want[:, 40:])):
        assert (got.double() - ref.double()).norm() <= bound * ref.double().norm()
