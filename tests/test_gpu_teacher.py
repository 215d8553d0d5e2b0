"""A teacher's rows at the edges: temperatures, and entries so unlikely that fp32 has no probability for them."""
import math

import pytest
import torch

from ternaryllm_amd import ops

from tests import losses
from tests.test_gpu_loss import check, device_weight, some_teacher, spread

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heat", [1e-6, 1e-3, 50.0, 1e6])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N", [(17, 257, 129), (130, 136, 777)])
def test_temperatures_far_from_one(M, K, N, dtype, heat):
    w, s = losses.head(K, N, dtype, M)
    x, g = losses.rows(M, K, dtype, M), spread(M, N)
    ids, logits = some_teacher(M, N, 6, K)
    ref = losses.Reference(x, w, s, *losses.teacher(ids, logits, N, heat), heat=heat, grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, temperature=heat, back=ops.BackWeight(weight))
    got, scales = torch.autograd.grad(loss, (dx, ds), g.cuda())
    check(ref, loss, got)
    # (as check takes the rows' gradient: sums of a heat of 10^6 leave fp16, and what is past the middle between its largest number and the next step rounds to infinity)
    scales, most, bound = scales.cpu().double(), torch.finfo(dtype).max * (1 + torch.finfo(dtype).eps / 4), ref.gradient_bounds()[1]
    past = (scales.abs() == math.inf) & (scales.sign() == ref.ds.sign()) & (ref.ds.abs() + bound >= most)
    assert (past | ((scales - ref.ds).abs() <= bound + torch.finfo(dtype).eps / 2 * ref.ds.abs() + 2.0 ** -25)).all()


@pytest.mark.parametrize("M", [6, 70])
def test_an_unlikely_entry_that_is_no_column(M):
    """Its probability is 0 in fp32, and the row has no loss all the same; an entry of -inf may have any id."""
    w, s = losses.head(64, 200, torch.float16)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    x = losses.rows(M, 64, torch.float16).cuda().requires_grad_()
    ids, logits = torch.randint(0, 200, (M, 4), generator=torch.Generator().manual_seed(1)), torch.randn((M, 4), generator=torch.Generator().manual_seed(2))
    for row, (number, logit) in enumerate([(200, -1000.0), (-1, -200.0), (1 << 40, -3e38), (-5, -math.inf), (7, -1000.0)]):
        ids[row, 2], logits[row, 2] = number, logit
    loss = ops.distillation(weight, x, ids.cuda(), logits.cuda(), s.cuda(), back=back)
    gx, = torch.autograd.grad(loss.sum(), x)
    assert loss[:3].isnan().all() and gx[:3].isnan().all() and loss[3:].isfinite().all() and gx[3:].isfinite().all()
