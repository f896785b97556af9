"""Rows of logits around the longest that two blocks of an SM keep in shared memory (115200 bytes each) and the longest that one does
(226 KB): losses and gradients do not depend on how a row is held."""

import pytest
import torch

from rbf_attention_b200 import ops
from test_policy_loss_gpu import _case, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [250, 300, 900])
@pytest.mark.parametrize("cols,dtype", [(28800, torch.float32), (28801, torch.float32), (28804, torch.float32), (28928, torch.float32),
                                        (57600, torch.bfloat16), (57601, torch.float16), (57608, torch.bfloat16),
                                        (57856, torch.float32), (57857, torch.float32)])
def test_policy_loss(rows, cols, dtype):
    _check(*_case(rows, cols, dtype, seed=rows + cols))


@pytest.mark.parametrize("cols,dtype", [(28800, torch.float32), (28804, torch.float32), (28928, torch.float32), (57600, torch.bfloat16),
                                        (57608, torch.bfloat16), (57856, torch.float16)])
def test_cross_entropy(cols, dtype):
    """Each element within half a step, 2^-25 in float16, and the exponential's 2^-18."""
    x, t, *_ = _case(400, cols, dtype, seed=cols)
    leaf, ref = x.detach().requires_grad_(True), x.double().requires_grad_(True)
    loss, want = ops.cross_entropy(leaf, t), torch.nn.functional.cross_entropy(ref, t, ignore_index=-100)
    loss.backward()
    want.backward()
    assert abs(loss.item() - want.item()) <= 2e-6 * abs(want.item()) + 1e-6
    half, least = torch.finfo(dtype).eps / 2, 2.0**-25 if dtype == torch.float16 else 0.0
    # near its token's probability of one an element is a difference: 2^-18 of 1 / rows
    assert ((leaf.grad.double() - ref.grad).abs() <= (half + 2.0**-18) * ref.grad.abs() + least + 2.0**-18 / 320 * (ref.grad < 0)).all()
