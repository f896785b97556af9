"""Cross entropy of float16 logits under a loss scale: the factor comes before the gradient is rounded. Element by element against
64 bits."""

import math

import pytest
import torch

from rbf_attention_b200 import lm, ops
from test_loss_scale_gpu import DEV, _check_rows, _chunks, _logits

pytestmark = pytest.mark.gpu


def _slopes(t):
    """d(mean loss)/d(log-probability): the loss is minus their mean."""
    weight = (t != -100).double() / (t != -100).sum()
    return -weight, weight


def _without_infinities(grad, x, t, slope, factor):
    """float16's largest number is 65504 and its steps there are 32: from 65520 on a value rounds to infinity, which is asserted, and
    replaced by the value. (One row under a factor of 65536 has its token's element there.)"""
    out = grad.double()
    for rs, p, one in _chunks(x, t):
        want = factor * slope[rs, None] * (one - p)
        over = want.abs() >= 65520
        assert torch.equal(out[rs][over], want[over].sign() * math.inf)
        out[rs] = torch.where(over, want, out[rs])
    return out


@pytest.mark.parametrize("rows,cols,pad", [(16384, 50257, 0), (16384, 50304, 0), (4096, 1000, 0), (4096, 1001, 23), (3, 7, 0), (1, 1, 0),
                                           (1, 70001, 0), (70000, 40, 8)])
@pytest.mark.parametrize("factor", [65536.0, -24.0])
def test_under_a_loss_scale(rows, cols, pad, factor):
    x, t, _ = _logits(rows, cols, pad, seed=rows + cols)
    leaf = x.detach().requires_grad_(True)
    loss = ops.cross_entropy(leaf, t)
    (grad,) = torch.autograd.grad(loss * factor, leaf)
    slope, size = _slopes(t)
    _check_rows(_without_infinities(grad, x, t, slope, factor), x, t, slope, size, factor)
    with torch.no_grad():
        assert torch.equal(ops.cross_entropy(leaf, t), loss)
    assert torch.equal(ops._cross_entropy_fwd(x, t, -100)[0], loss)         # as without the statistics


def test_a_model_in_float16_under_a_scaler():
    """What the usual loop does: scale, backward, unscale. The projection's gradient against 64 bits of the same logits: each of its
    sums over the rows has every term's rounding (2^-11, or 2^-25 of the scaled sum below 2^-14) and its own."""
    torch.manual_seed(0)
    rows, cols, width = 8192, 5000, 64
    h = torch.randn(rows, width, device=DEV).half()
    weight = (torch.randn(cols, width, device=DEV) * 0.3).half().requires_grad_(True)
    t = torch.randint(0, cols, (rows,), device=DEV)
    scale = 65536.0
    logits = h @ weight.t()
    scaler = torch.amp.GradScaler(init_scale=scale)
    scaler.scale(lm.cross_entropy(logits, t)).backward()
    z = logits.detach().double()
    d = (torch.softmax(z, -1) - torch.nn.functional.one_hot(t, cols)) / rows
    want = d.t() @ h.double()
    bound = (d.abs() * 2.0**-11 * 1.05 + 2.0**-25 / scale).t() @ h.double().abs() + want.abs() * 2.0**-11 + 2.0**-25 / scale
    # the products' sums in fp32: rows terms of half a step of 2^-24 each, in any order
    bound += rows * 2.0**-24 * (d.abs().t() @ h.double().abs())
    assert ((weight.grad.double() / scale - want).abs() <= bound).all()


def test_the_registered_operator_the_graph_and_ignored_rows(monkeypatch):
    x, t, _ = _logits(200, 333, 2, seed=2)
    leaf = x.detach().requires_grad_(True)
    loss = ops.cross_entropy(leaf, t)
    (direct,) = torch.autograd.grad(loss * 65536.0, leaf)
    (linked,) = torch.autograd.grad(ops.cross_entropy(leaf, t) * 65536.0, leaf, create_graph=True)
    assert torch.equal(linked, direct)
    with pytest.raises(RuntimeError, match="Trying to backward through"):
        (leaf.sum() + linked.float().square().sum()).backward()
    monkeypatch.setattr(ops, "_direct", lambda *tensors: False)
    other = ops.cross_entropy(leaf, t)
    assert torch.equal(other, loss) and torch.equal(torch.autograd.grad(other * 65536.0, leaf)[0], direct)
    t[:] = -100
    nothing = ops.cross_entropy(leaf, t)
    assert nothing.isnan() and not torch.autograd.grad(nothing, leaf)[0].any()
    empty = x[:0].detach().requires_grad_(True)
    loss = ops.cross_entropy(empty, t[:0])
    assert torch.autograd.grad(loss, empty)[0].shape == (0, 333)
    with pytest.raises(ValueError):
        torch.ops.rbf_attn_b200.cross_entropy_rows(x.float(), t, -100)


def test_columns_of_minus_infinity_and_rows_that_are_not_finite():
    x, t, _ = _logits(50, 640, 0, seed=3)
    x, t = x.clone(), t.clamp(max=599)
    t[t < 0] = -100
    x[:, 600:] = -math.inf
    leaf = x.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(ops.cross_entropy(leaf, t) * 1024.0, leaf)
    assert not grad[:, 600:].any() and grad.isfinite().all()
    x[7], x[8, 5] = -math.inf, math.nan
    t[7], t[8] = 3, 4
    leaf = x.detach().requires_grad_(True)
    (grad,) = torch.autograd.grad(ops.cross_entropy(leaf, t), leaf)
    assert grad[7:9].isnan().all() and grad[9:].isfinite().all()
