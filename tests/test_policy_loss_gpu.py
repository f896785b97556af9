"""Log-probabilities of tokens and the clipped policy loss with its gradient, against the formulas in 64 bits."""

import math

import pytest
import torch

from rbf_attention_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(rows, cols, dtype, seed=0, std=2.0, pad=0, ignored=0.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    memory = torch.randn(rows, cols + pad, device=DEV, generator=g).mul(std).to(dtype)
    x = memory[:, :cols]
    t = torch.randint(0, cols, (rows,), device=DEV, generator=g)
    t[torch.rand(rows, device=DEV, generator=g) < ignored] = -100
    if rows:
        t[rows // 2] = cols - 1
    lp = _log_probs(x, t).float()
    old = lp + 0.3 * torch.randn(rows, device=DEV, generator=g)
    ref = lp + 0.3 * torch.randn(rows, device=DEV, generator=g)
    adv = torch.randn(rows, device=DEV, generator=g)
    return x, t, old, ref, adv


def _counts(x, t):
    return (t != -100) & (t >= 0) & (t < x.shape[1])


def _log_probs(x, t):
    keep = _counts(x, t)
    lp = torch.log_softmax(x.double(), -1).gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    return torch.where(keep, lp, 0.0)


def _reference(x, t, old, ref, adv, low, high, kl, weights=None):
    z = x.detach().double().requires_grad_(True)
    keep = _counts(x, t)
    lp = torch.log_softmax(z, -1).gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0][keep]
    r, a = (lp - old.double()[keep]).exp(), adv.double()[keep]
    value = -torch.minimum(r * a, r.clamp(1 - low, 1 + high) * a)
    if ref is not None:
        gap = ref.double()[keep] - lp
        value = value + kl * (gap.exp() - gap - 1)
    w = weights.double()[keep] if weights is not None else torch.full_like(lp, 1.0) / keep.sum()
    loss = (w * value).sum()
    loss.backward()
    return loss.detach(), z.grad


# lp is a difference of numbers of the size of the largest logit and of log(cols): some steps of fp32 of that size (8 bound the
# exponent's two units in the last place, the sum and the logarithm).
def _lp_bound(x):
    return 8 * 2.0**-24 * (x.detach().double().abs().max().item() + math.log(x.shape[1]) + 1)


def _check(x, t, old, ref, adv, low=0.2, high=0.3, kl=0.05, weights=None):
    leaf = x.detach().requires_grad_(True)
    loss, lp = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, weights=weights, clip_low=low, clip_high=high, kl_weight=kl)
    assert not lp.requires_grad and loss.dtype == torch.float32
    loss.backward()
    want, grad = _reference(x, t, old, ref, adv, low, high, kl, weights)
    off = _lp_bound(x)
    assert (lp.double() - _log_probs(x, t)).abs().max() <= off
    keep = _counts(x, t)
    w = weights.double().abs()[keep] if weights is not None else torch.full((int(keep.sum()),), 1.0 / max(int(keep.sum()), 1), device=DEV)
    # d(loss)/d(lp) is at most e^|lp - old| |A| + kl (1 + e^|ref - lp|); the values' own rounding is 2^-23 of the same terms
    steep = (adv.abs() * 4 + (kl * 5 if ref is not None else 0))[keep].double()
    assert (loss.double() - want).abs() <= (w * steep).sum() * (off + 2.0**-22) + 2.0**-24 * want.abs()
    # a row's gradient: w slope (onehot - p): relative errors of the slope and of p (both off by lp's error), then the rounding
    half = torch.finfo(x.dtype).eps / 2
    rel = ((leaf.grad.double() - grad).norm() / grad.norm().clamp(min=1e-300)).item()
    # below 2^-14 the numbers of float16 are 2^-24 apart, so each element is off by up to 2^-25 whatever its size: 2^-25 sqrt(elements)
    # in the norm. (Many long rows are there: 1 / 300 rows / 50000 columns.)
    small = 2.0**-25 * math.sqrt(keep.sum().item() * x.shape[1]) / grad.norm().clamp(min=1e-300).item() if x.dtype == torch.float16 else 0.0
    assert rel <= half + 16 * off + small, rel
    assert not leaf.grad[~keep].any()
    with torch.no_grad():
        again, lp2 = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, weights=weights, clip_low=low, clip_high=high, kl_weight=kl)
    assert torch.equal(lp, lp2) and torch.equal(again, loss)
    assert torch.equal(ops.token_log_probs(x, t), lp)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 50257), (3, 7), (40, 8), (33, 1000), (700, 1023), (5, 130001)])
def test_sizes(rows, cols, dtype):
    _check(*_case(rows, cols, dtype, seed=rows + cols, ignored=0.2 if rows > 1 else 0.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [1, 3, 8, 47])
def test_rows_of_any_alignment(dtype, pad):
    x, *rest = _case(60, 501, dtype, seed=pad, pad=pad)
    _check(x, *rest)
    _check(torch.cat([x[:, :1], x], 1)[:, 1:], *rest)
    _check(x.t().contiguous().t(), *rest)


@pytest.mark.parametrize("dtype", TYPES)
def test_without_the_kl_term_and_with_weights(dtype):
    x, t, old, ref, adv = _case(90, 300, dtype, seed=5)
    _check(x, t, old, None, adv, kl=0.0)
    w = torch.rand(90, device=DEV) - 0.3
    _check(x, t, old, ref, adv, weights=w, kl=1.0)
    _check(x, t, old, None, adv, weights=w, kl=0.0, low=0.0, high=0.0)


def test_clipped_rows_have_the_gradient_of_the_rest():
    """Ratios far out on either side, both signs of the advantage and none."""
    x, t, old, ref, adv = _case(48, 200, torch.float32, seed=6, ignored=0.0)
    lp = _log_probs(x, t).float()
    old = lp - torch.tensor([1.0, -1.0, 0.05, 0.0], device=DEV).repeat(12)
    adv = torch.tensor([1.0, -1.0, 0.0], device=DEV).repeat_interleave(4).repeat(4)
    _check(x, t, old, ref, adv)
    _check(x, t, old, None, adv, kl=0.0)
    leaf = x.clone().requires_grad_(True)
    ops.policy_loss(leaf, t, old, adv)[0].backward()
    ratio = (lp - old).exp()
    still = ((adv > 0) & (ratio > 1.2)) | ((adv < 0) & (ratio < 0.8)) | (adv == 0)
    assert still.any() and (~still).any()
    assert not leaf.grad[still].any() and leaf.grad[~still].any(-1).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_columns_of_minus_infinity_and_tokens_outside(dtype):
    x, t, old, ref, adv = _case(50, 640, dtype, seed=7)
    x = x.clone()
    t = t.clamp(max=599)
    x[:, 600:] = -math.inf
    t[:6] = torch.tensor([-1, 640, 2**40, -100, 0, 599], device=DEV)
    old = ref = _log_probs(x, t).float()
    _check(x, t, old + 0.1, ref - 0.1, adv)
    x[7], x[8, 5] = -math.inf, math.nan
    t[7], t[8] = 3, 4
    leaf = x.clone().requires_grad_(True)
    loss, lp = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.1)
    loss.backward()
    assert loss.isnan() and lp[7].isnan() and lp[8].isnan() and leaf.grad[7:9].isnan().all()
    assert leaf.grad[9:].isfinite().all() and lp[9:].isfinite().all()


def test_no_row_that_counts():
    x, t, old, ref, adv = _case(9, 70, torch.bfloat16, seed=8)
    t[:] = -100
    leaf = x.clone().requires_grad_(True)
    loss, lp = ops.policy_loss(leaf, t, old, adv)
    loss.backward()
    assert loss.isnan() and not lp.any() and not leaf.grad.any()
    loss, _ = ops.policy_loss(x, t, old, adv, weights=old)
    assert loss == 0
    for n in (0,):
        empty = x[:n].clone().requires_grad_(True)
        loss, lp = ops.policy_loss(empty, t[:n], old[:n], adv[:n])
        loss.backward()
        assert loss.isnan() and lp.shape == (0,) and empty.grad.shape == (0, 70)
        assert ops.token_log_probs(x[:n], t[:n]).shape == (0,)


@pytest.mark.parametrize("pad", [0, 5])
def test_scaled_loss_and_differences(pad):
    """The gradient against differences of the loss in 64 bits, under an outer factor."""
    x, t, old, ref, adv = _case(6, 40, torch.float32, seed=9, pad=pad, ignored=0.0)
    old = old + 0.02
    leaf = x.detach().requires_grad_(True)
    loss, _ = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.3)
    (loss * -2.5).backward()
    step = 1e-5
    for r in range(6):
        for c in (0, int(t[r]), 39):
            sides = []
            for s in (step, -step):
                z = x.double().clone()
                z[r, c] += s
                sides.append(_reference(z, t, old, ref, adv, 0.2, 0.2, 0.3)[0])
            slope = -2.5 * (sides[0] - sides[1]) / (2 * step)
            assert abs(leaf.grad[r, c].double() - slope) <= 1e-5 + 1e-4 * abs(slope), (r, c)


def test_through_the_registered_operator_and_a_second_backward():
    x, t, old, ref, adv = _case(30, 333, torch.bfloat16, seed=10, pad=2)
    leaf = x.detach().requires_grad_(True)
    loss, _ = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.1)
    (direct,) = torch.autograd.grad(loss * 3, leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf)
    args = (leaf, t, old, adv, ref, None, 0.2, 0.2, 0.1, -100, True)
    loss2, lp2, _ = torch.ops.rbf_attn_b200.policy_loss_fwd(*args)
    (other,) = torch.autograd.grad(loss2 * 3, leaf)
    assert torch.equal(loss, loss2) and torch.equal(direct, other)
    loss3, _ = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.1)
    (linked,) = torch.autograd.grad(loss3, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second-order|does not require grad|backward"):
        linked.sum().backward()


def test_runs_are_bitwise_alike():
    x, t, old, ref, adv = _case(900, 2000, torch.float16, seed=11)
    seen = []
    for _ in range(3):
        leaf = x.clone().requires_grad_(True)
        loss, lp = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.1)
        loss.backward()
        seen.append((loss.detach(), lp, leaf.grad))
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_captured_and_replayed():
    x, t, old, ref, adv = _case(64, 1000, torch.bfloat16, seed=12)
    leaf = x.clone().requires_grad_(True)

    def run():
        loss, lp = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=0.1)
        return loss, lp, torch.autograd.grad(loss, leaf)[0]

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = run()
    torch.cuda.synchronize()
    for seed in (13, 14):
        for to, value in zip((leaf, t, old, ref, adv), _case(64, 1000, torch.bfloat16, seed=seed)):
            with torch.no_grad():
                to.copy_(value)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, run()))


def test_refusals():
    x, t, old, ref, adv = _case(8, 20, torch.float32, seed=15)
    good = dict(logits=x, tokens=t, old_log_probs=old, advantages=adv, ref_log_probs=ref, weights=old, clip_low=0.1, clip_high=0.1,
                kl_weight=0.1)
    ops.policy_loss(**good)
    for change in ({"logits": x[0]}, {"logits": x.double()}, {"logits": x.cpu()}, {"logits": x[:4]}, {"logits": x[:, :0]},
                   {"tokens": t.int()}, {"tokens": t[:, None]}, {"tokens": t.cpu()}, {"old_log_probs": old.half()},
                   {"old_log_probs": old[:4]}, {"advantages": adv.double()}, {"advantages": adv.cpu()}, {"ref_log_probs": ref[:, None]},
                   {"weights": old.bfloat16()}, {"clip_low": -0.1}, {"clip_high": float("nan")}, {"ref_log_probs": None}):
        for leaf in (False, True):
            call = {**good, **change}
            if leaf:
                call["logits"] = call["logits"].detach().requires_grad_(True)
            with pytest.raises((ValueError, RuntimeError)):
                ops.policy_loss(**call)
    for change in ({"logits": x[0]}, {"tokens": t.int()}, {"tokens": t[:3]}, {"logits": x.double()}):
        with pytest.raises((ValueError, RuntimeError)):
            ops.token_log_probs(**{"logits": x, "tokens": t, **change})
    leaf = x.clone().requires_grad_(True)
    for name in ("old_log_probs", "advantages", "ref_log_probs", "weights"):
        with pytest.raises(RuntimeError, match=f"{name}.*detach"):
            ops.policy_loss(**{**good, "logits": leaf, name: good[name].clone().requires_grad_(True)})


def test_two_losses_of_one_leaf_and_accumulated_gradients():
    x, t, old, ref, adv = _case(40, 300, torch.bfloat16, seed=16)
    leaf = x.clone().requires_grad_(True)
    one, _ = ops.policy_loss(leaf, t, old, adv)
    two, _ = ops.policy_loss(leaf, t, old, adv, ref_log_probs=ref, kl_weight=1.0)
    (one * 0.5 + two * 0.25).backward()
    want = 0.5 * _reference(x, t, old, None, adv, 0.2, 0.2, 0.0)[1] + 0.25 * _reference(x, t, old, ref, adv, 0.2, 0.2, 1.0)[1]
    # two gradients rounded, scaled and rounded, added and rounded: five half steps at most, of numbers that may cancel by half
    half = torch.finfo(x.dtype).eps / 2
    assert (leaf.grad.double() - want).norm() <= 10 * half * want.norm()
    again, _ = ops.policy_loss(leaf, t, old, adv)
    before = leaf.grad.clone()
    again.backward()
    single = _reference(x, t, old, None, adv, 0.2, 0.2, 0.0)[1]
    assert ((leaf.grad.double() - before.double()) - single).norm() <= 4 * half * (before.double().norm() + single.norm())


def test_strided_rows_of_the_statistics():
    x, t, old, ref, adv = _case(30, 100, torch.float16, seed=17)
    wide = torch.stack([old, ref, adv], 1)
    tokens = torch.stack([t, t + 1], 1)[:, 0]
    a = ops.policy_loss(x, t, old, adv, ref_log_probs=ref, kl_weight=0.2)
    b = ops.policy_loss(x, tokens, wide[:, 0], wide[:, 2], ref_log_probs=wide[:, 1], kl_weight=0.2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("rows", [8192, 8193, 20000])
def test_many_rows_are_counted_alike(rows):
    """Few rows are counted by every block, many by a kernel of their own."""
    x, t, old, ref, adv = _case(rows, 33, torch.float32, seed=18)
    _check(x, t, old, ref, adv)


@pytest.mark.parametrize("rows", [297, 460])
@pytest.mark.parametrize("cols,dtype", [(29001, torch.float32), (57857, torch.float16), (115711, torch.bfloat16), (57857, torch.float32)])
def test_long_rows_at_every_way_of_holding_them(rows, cols, dtype):
    """Rows just above what two blocks on an SM hold, just below and above what one does, more of them than run at once."""
    _check(*_case(rows, cols, dtype, seed=rows + cols))
