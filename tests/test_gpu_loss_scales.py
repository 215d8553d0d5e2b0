"""Losses of fp32 rows whose column scales are far from 1, or not finite."""
import math

import pytest
import torch

from ternaryllm_amd import ops

from tests import losses
from tests.test_gpu_loss import device_weight, spread

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def graded(weight, x, t, s, g):
    """Losses of cross entropy and their gradients, in float64 on the CPU."""
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    return [y.detach().cpu().double() for y in (loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()))]


@pytest.mark.parametrize("far", [-100, -70, 60, 122])
@pytest.mark.parametrize("M,K,N", [(5, 72, 333), (60, 72, 333), (300, 40, 9000)])
def test_scales_far_from_one(M, K, N, far):
    """Rows 2^-far and scales 2^far times ordinary ones: the same losses, and gradients 2^far and 2^-far times theirs."""
    up = 2.0 ** far
    w, s = losses.head(K, N, F32, M)
    x, t, g = losses.rows(M, K, F32, M), torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(M)), spread(M, N)
    ref = losses.Reference(x, w, s, *losses.targets(t, N), grad=g)
    loss, dx, ds = graded(device_weight(w), x / up, t, s * up, g)
    dx_bound, ds_bound = ref.gradient_bounds()
    assert ((loss - ref.loss).abs() <= ref.loss_bound()).all()
    # (what comes near fp32's smallest numbers is off by half of those, 2^-150, instead: of each row's share of a sum in its products and the sum)
    least = 2.0 ** -150
    assert ((dx / up - ref.dx).abs() <= dx_bound + losses.U * ref.dx.abs() + (3 * N + 8) * least / up).all()
    assert ((ds * up - ref.ds).abs() <= ds_bound + losses.U * ref.ds.abs() + (3 * M + 8) * least * up).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("M", [5, 60])
def test_a_scale_that_is_not_finite_has_no_gradient(M, dtype):
    """A column's logits of -inf times that scale: 0 times infinity is in every gradient of the rows, whatever their type and how many they are."""
    K, N = 64, 300
    w = losses.head(K, N, dtype, 4)[0]
    w[:, 7], w[0, 7] = 0, -1
    x, t = losses.rows(M, K, dtype, 4).abs().clamp(min=1), torch.arange(M) + 20
    t[2] = -100
    s = torch.full((N,), 0.1)
    s[7] = math.inf
    loss, dx, _ = graded(device_weight(w), x, t, s, torch.ones(M))
    counts = t != -100
    assert loss.isfinite().all() and dx[counts].isnan().all() and (dx[2] == 0).all()
