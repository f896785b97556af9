"""The policy loss under ``create_graph``: the gradient is there, linked to the logits, and refuses to be differentiated, also as one
term among others - a gradient returned as a constant would make a penalty on it add nothing."""

import pytest
import torch

from rbf_attention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _case(dtype):
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(30, 50, device=DEV, generator=g).to(dtype)
    t = torch.randint(0, 50, (30,), device=DEV, generator=g)
    lp = torch.log_softmax(x.float(), -1).gather(1, t[:, None])[:, 0]
    return x.requires_grad_(True), t, lp + 0.1, torch.randn(30, device=DEV, generator=g), lp - 0.1


def _loss(leaf, t, old, adv, ref):
    return ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.2)[0]


@pytest.mark.parametrize("registered", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_second_order_is_refused(dtype, registered, monkeypatch):
    if registered:
        monkeypatch.setattr(ops, "_direct", lambda *tensors: False)
    leaf, *rest = _case(dtype)
    (want,) = torch.autograd.grad(_loss(leaf, *rest), leaf)
    (linked,) = torch.autograd.grad(_loss(leaf, *rest), leaf, create_graph=True)
    assert not want.requires_grad and linked.requires_grad and torch.equal(linked, want)
    with pytest.raises(RuntimeError, match="Trying to backward through"):
        (leaf.sum() + linked.float().square().sum()).backward()
    factor = torch.ones((), device=DEV, requires_grad=True)
    (linked,) = torch.autograd.grad(_loss(leaf, *rest) * factor, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="Trying to backward through"):
        torch.autograd.grad(linked.float().square().sum(), factor)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_the_node_holds(dtype):
    """The gradient is handed out once, with and without a retained graph, and goes through the hooks of saved tensors."""
    leaf, *rest = _case(dtype)
    (want,) = torch.autograd.grad(_loss(leaf, *rest), leaf)
    loss = _loss(leaf, *rest)
    (first,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf, retain_graph=True)
    loss = _loss(leaf, *rest)
    (again,) = torch.autograd.grad(loss, leaf)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf)
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.clone(), lambda t: t):
        loss = _loss(leaf, *rest)
    (hooked,) = torch.autograd.grad(loss, leaf)
    assert packed and all(torch.equal(want, g) for g in (first, again, hooked))


def test_the_logits_memory_is_free_once_they_are_dropped():
    """bfloat16 and float32 keep the gradient, not the logits; after the backward the graph keeps nothing."""
    source = torch.randn(64, 4096, device=DEV, requires_grad=True)
    _, t, old, adv, ref = _case(torch.float32)
    t, old, adv, ref = (x.repeat(3)[:64] for x in (t, old, adv, ref))
    before = torch.cuda.memory_allocated()
    for dtype in (torch.float32, torch.float16):        # a graph that nobody goes back through leaves nothing behind
        loss = _loss(source.to(dtype) * 1.0, t, old, adv, ref)
        del loss
        assert torch.cuda.memory_allocated() == before
    loss = _loss(source * 1.0, t, old, adv, ref)
    size = source.numel() * 4
    assert torch.cuda.memory_allocated() - before < 1.5 * size
    loss.backward()
    assert torch.cuda.memory_allocated() - before < 1.5 * size       # the leaf's gradient
