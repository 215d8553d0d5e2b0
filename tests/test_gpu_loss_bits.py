"""Losses of fp32 rows that have all of fp32's bits, and of some near the end of its range."""
import pytest
import torch

from ternaryllm_amd import ops

from tests import losses
from tests.test_gpu_loss import device_weight, some_targets, some_teacher, spread
from tests.test_gpu_loss_scales import graded

pytestmark = pytest.mark.gpu

F32 = torch.float32
# few rows, and many in tiles of 128 and of 256 columns; lengths that are no whole pieces; pieces of the vocabulary
SIZES = [(5, 72, 333), (48, 301, 1000), (60, 301, 333), (200, 64, 5003), (300, 72, 9000), (1025, 130, 12000)]


def step(M, K, N, x, s, up=1.0, top=0):
    w = losses.thin_head(K, N, 4, M)
    g, weight = spread(M, N), device_weight(w)
    dx, ds = (x * up).cuda().requires_grad_(), (s / up).cuda().requires_grad_()
    if top:
        ids, logits = some_teacher(M, N, top, K)
        ref = losses.Reference(x, w, s, *losses.teacher(ids, logits, N, 2.0), heat=2.0, grad=g)
        loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, temperature=2.0, back=ops.BackWeight(weight))
    else:
        t = some_targets(M, N, K)
        ref = losses.Reference(x, w, s, *losses.targets(t, N), grad=g)
        loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    got = [y.detach().cpu().double() for y in (loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()))]
    dx_bound, ds_bound = ref.gradient_bounds()
    assert ((got[0] - ref.loss).abs() <= ref.loss_bound()).all()
    assert ((got[1] * up - ref.dx).abs() <= dx_bound).all()
    assert ((got[2] / up - ref.ds).abs() <= ds_bound + losses.U * ref.ds.abs()).all()
    return got


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_rows_of_all_bits(M, K, N, top):
    step(M, K, N, losses.long_rows(M, K, M), losses.long_scales(N, M), top=top)


def test_rows_of_all_bits_in_parts():
    """More rows than the workspace of a backward pass takes at a time."""
    step(1700, 16, 16500, losses.long_rows(1700, 16), losses.long_scales(16500))


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("M,K,N", SIZES[:4])
def test_rows_near_the_end_of_the_range(M, K, N, top):
    """Up to 2^120, where scaled bf16 parts leave fp32's range, with scales that make ordinary logits of them."""
    step(M, K, N, losses.long_rows(M, K, M), losses.long_scales(N, M), 2.0 ** 118, top)


@pytest.mark.parametrize("M,K,N", [(6, 72, 333), (70, 72, 333), (70, 72, 5003)])
def test_rows_beside_such_rows_keep_their_bits(M, K, N):
    w, s = losses.thin_head(K, N, 4, M), losses.long_scales(N, M) * 2.0 ** -118
    x, t, g, weight = losses.long_rows(M, K, M), some_targets(M, N, K), spread(M, N), device_weight(w)
    plain = graded(weight, x, t, s, g)
    large = [3, M - 2]
    x[large] *= 2.0 ** 118
    got = graded(weight, x, t, s, g)
    others = [m for m in range(M) if m not in large]
    assert torch.equal(got[0][others], plain[0][others]) and torch.equal(got[1][others], plain[1][others])
    alone = graded(weight, x[large], t[large], s, g[large])
    assert ((got[0][large] - alone[0]).abs() <= 1e-4).all() and got[1][large].isfinite().all() and got[2].isfinite().all()
