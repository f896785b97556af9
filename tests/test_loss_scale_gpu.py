"""Losses of float16 logits under a loss scale: the factor comes before the gradient is rounded, so that elements below float16's
smallest numbers survive. Element by element against 64 bits."""

import math

import pytest
import torch

from rbf_attention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOW, HIGH, KL = 0.2, 0.3, 0.05


def _logits(rows, cols, pad, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.empty(rows, cols + pad, dtype=torch.float16, device=DEV)
    for r in range(0, rows, 2048):
        x[r:r + 2048] = torch.randn(x[r:r + 2048].shape, device=DEV, generator=g) * 2.5
    x = x[:, :cols]
    t = torch.randint(0, cols, (rows,), device=DEV, generator=g)
    t[::2] = x.argmax(-1)[::2]
    t[torch.rand(rows, device=DEV, generator=g) < 0.1] = -100
    t[0] = 0
    return x, t, g


def _chunks(x, t):
    for r in range(0, x.shape[0], 512):
        z = x[r:r + 512].detach().double()
        yield slice(r, r + 512), torch.softmax(z, -1), torch.nn.functional.one_hot(t[r:r + 512].clamp(min=0), x.shape[1])


def _policy_case(rows, cols, pad=0, seed=0):
    x, t, g = _logits(rows, cols, pad, seed)
    lp = torch.empty(rows, dtype=torch.float64, device=DEV)
    for rs, p, one in _chunks(x, t):
        lp[rs] = (p * one).sum(-1).log()
    step = 0.3 * torch.randn(rows, device=DEV, generator=g)
    for border in (math.log(1 - LOW), math.log(1 + HIGH)):      # ratios are not within rounding of where the clipping starts
        step = torch.where((step - border).abs() < 0.01, step + 0.03, step)
    old = (lp - step).float()
    ref = (lp + 0.3 * torch.randn(rows, device=DEV, generator=g)).float()
    return x, t, lp, old, ref, torch.randn(rows, device=DEV, generator=g)


def _check_rows(grad, x, t, slope, size, factor):
    """grad against factor * slope * (onehot - p). An element is rounded once: half a step is 2^-11 of it, or 2^-25 where it is below
    2^-14. The log-probability, with it the slope (whose terms add up to ``size``) and p are off by some steps of fp32 of the
    size of the largest logit, as in test_policy_loss_gpu.py: twice that each."""
    off = 8 * 2.0**-24 * (x.double().abs().max().item() + math.log(x.shape[1]) + 1)
    keep = t != -100
    assert not grad[~keep].any()
    for rs, p, one in _chunks(x, t):
        want = torch.where(keep[rs, None], factor * slope[rs, None] * (one - p), 0.0)
        bound = want.abs() * 2.0**-11 + 2.0**-25 + 4 * off * abs(factor) * size[rs, None] * (p + one)
        err = (grad[rs].double() - want).abs()
        assert (err <= bound).all(), (rs, (err / bound).max().item())


def _policy_slopes(t, lp, old, ref, adv):
    keep = t != -100
    r, away = (lp - old.double()).exp(), (ref.double() - lp).exp()
    plain, clipped = r * adv.double(), r.clamp(1 - LOW, 1 + HIGH) * adv.double()
    slope = KL * (1 - away) - torch.where(plain <= clipped, plain, 0.0)
    size = KL * (1 + away) + plain.abs()
    return torch.where(keep, slope, 0.0) / keep.sum(), torch.where(keep, size, 0.0) / keep.sum()


def _policy(leaf, t, old, ref, adv):
    return ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, clip_low=LOW, clip_high=HIGH, kl_weight=KL)[0]


@pytest.mark.parametrize("rows,cols,pad", [(16384, 50257, 0), (4096, 1000, 0), (4096, 1001, 23), (3, 7, 0), (1, 1, 0), (1, 70001, 0),
                                           (70000, 40, 1)])
@pytest.mark.parametrize("factor", [65536.0, -24.0])
def test_policy_loss_under_a_loss_scale(rows, cols, pad, factor):
    x, t, lp, old, ref, adv = _policy_case(rows, cols, pad, seed=rows + cols)
    leaf = x.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(_policy(leaf, t, old, ref, adv) * factor, leaf)
    _check_rows(grad, x, t, *_policy_slopes(t, lp, old, ref, adv), factor)


def test_rows_of_other_layouts():
    x, t, lp, old, ref, adv = _policy_case(300, 501, 6, seed=1)
    want = _policy_slopes(t, lp, old, ref, adv)
    tokens = torch.stack([t, t + 1], 1)[:, 0]
    for leaf in (x[:, :], torch.cat([x[:, :1], x], 1)[:, 1:], x.t().contiguous().t()):
        leaf = leaf.detach().requires_grad_(True)
        (grad,) = torch.autograd.grad(_policy(leaf, tokens, old, ref, adv) * 4096.0, leaf)
        _check_rows(grad, x, t, *want, 4096.0)
    wide = torch.zeros(300, 501, dtype=torch.float16, device=DEV, requires_grad=True)       # broadcast rows
    leaf = wide[:1].detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(_policy(leaf.expand(300, 501), t, old, ref, adv), leaf)
    assert grad.shape == (1, 501) and grad.isfinite().all()


def test_the_registered_operator_the_factor_and_the_graph():
    x, t, lp, old, ref, adv = _policy_case(200, 333, 2, seed=2)
    leaf = x.detach().requires_grad_(True)
    loss = _policy(leaf, t, old, ref, adv)
    (direct,) = torch.autograd.grad(loss * 65536.0, leaf)
    loss2, _, stats = torch.ops.rbf_attn_b200.policy_loss_fwd(leaf, t, old, adv, ref, None, LOW, HIGH, KL, -100, True)
    (other,) = torch.autograd.grad(loss2 * 65536.0, leaf)
    assert torch.equal(loss, loss2) and torch.equal(direct, other) and stats.shape == (200, 2)
    assert torch.equal(torch.ops.rbf_attn_b200.loss_gradient(x, t, stats.detach(), torch.tensor(65536.0, device=DEV), -100), direct)
    # an infinite scale leaves numbers that a scaler recognises
    (grad,) = torch.autograd.grad(_policy(leaf, t, old, ref, adv) * math.inf, leaf)
    keep = t != -100
    assert not grad[keep].isfinite().any() and not grad[~keep].any()
    # the backward reads the logits again
    changed = (x * 1).requires_grad_(True)
    between = changed * 1
    loss = _policy(between, t, old, ref, adv)
    with torch.no_grad():
        between.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


@pytest.mark.parametrize("registered", [False, True])
def test_second_order_is_refused(registered, monkeypatch):
    x, t, lp, old, ref, adv = _policy_case(30, 50, seed=3)
    if registered:
        monkeypatch.setattr(ops, "_direct", lambda *tensors: False)
    leaf = x.detach().requires_grad_(True)
    (want,) = torch.autograd.grad(_policy(leaf, t, old, ref, adv), leaf)
    (linked,) = torch.autograd.grad(_policy(leaf, t, old, ref, adv), leaf, create_graph=True)
    assert linked.requires_grad and torch.equal(linked, want)
    with pytest.raises(RuntimeError, match="Trying to backward through"):
        (leaf.sum() + linked.square().sum()).backward()


def test_captured_and_replayed():
    x, t, lp, old, ref, adv = _policy_case(64, 1000, seed=4)
    leaf, factor = x.detach().clone().requires_grad_(True), torch.tensor(1024.0, device=DEV)

    def run():
        return torch.autograd.grad(_policy(leaf, t, old, ref, adv) * factor, leaf)[0]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
    torch.cuda.current_stream().wait_stream(stream)
    for seed in (5, 6):
        x2, t2, _, old2, ref2, adv2 = _policy_case(64, 1000, seed=seed)
        with torch.no_grad():
            for to, value in zip((leaf, t, old, ref, adv, factor), (x2, t2, old2, ref2, adv2, torch.tensor(8.0 * seed, device=DEV))):
                to.copy_(value)
        graph.replay()
        assert torch.equal(out, run())


def test_refusals():
    x, t, lp, old, ref, adv = _policy_case(8, 20, seed=7)
    stats, factor = torch.zeros(8, 2, device=DEV), torch.ones((), device=DEV)
    gradient = torch.ops.rbf_attn_b200.loss_gradient
    assert not gradient(x, t, stats, factor, -100).any()
    assert gradient(x[:0], t[:0], stats[:0], factor, -100).shape == (0, 20)
    for args in ((x.float(), t, stats, factor), (x.bfloat16(), t, stats, factor), (x, t.int(), stats, factor), (x, t[:4], stats, factor),
                 (x, t, stats[:4], factor), (x, t, stats.half(), factor), (x, t, stats.t().contiguous().t(), factor),
                 (x, t, stats, factor.expand(2)), (x, t, stats.cpu(), factor), (x.cpu(), t.cpu(), stats.cpu(), factor)):
        with pytest.raises((ValueError, RuntimeError)):
            gradient(*args, -100)
