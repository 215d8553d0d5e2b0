"""Losses of logits so large that fp32 holds them to whole numbers or worse: what such a number is rounded by must not become an exponential of its own."""
import pytest
import torch

from ternaryllm_amd import ops

from tests import losses
from tests.test_gpu_loss import device_weight, some_teacher, spread

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("heat", [None, 1.0, 3.0, 0.7])
@pytest.mark.parametrize("dtype,up", [(F16, 2.0 ** 12), (F32, 2.0 ** 12), (F32, 2.0 ** 70)])
@pytest.mark.parametrize("M,K,N", [(5, 200, 777), (48, 200, 777), (80, 200, 777), (80, 64, 9001)])
def test_one_logit_leads(M, K, N, dtype, up, heat):
    """Logits of 2^30 (and 2^88) of which one leads by far: its probability is 1, and all others' 0."""
    w, s = losses.head(K, N, F32, M)
    x, g = losses.rows(M, K, dtype, M), spread(M, N)
    s = s * 2.0 ** 14
    if heat is None:
        t = torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(M))
        best = (x.double() @ torch.as_tensor(w).double() * s.double()).argmax(-1)
        t[::2] = best[::2]                                       # (rows that are sure of what is wanted have no gradient)
        wanted, counts = losses.targets(t, N)
    else:
        ids, logits = some_teacher(M, N, 6, K)
        wanted, counts = losses.teacher(ids, logits, N, heat)
    x = (x.double() * up).to(dtype)
    ref = losses.Reference(x, w, s, wanted, counts, heat=heat or 1.0, grad=g)
    most = ref.z.topk(2, -1).values
    clear = most[:, 0] - most[:, 1] > 100 + 4 * ref.off          # (rows whose two largest logits fp32 tells apart)
    assert clear.sum() >= 0.8 * M
    wanted, counts = wanted * clear[:, None], counts & clear     # the others count for nothing
    if heat is None:
        t = torch.where(clear, t, -100)
    else:
        logits[~clear] = -float("inf")
    ref = losses.Reference(x, w, s, wanted, counts, heat=heat or 1.0, grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    if heat is None:
        loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    else:
        loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, temperature=heat, back=ops.BackWeight(weight))
    got = [y.detach().cpu().double() for y in (loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()))]
    assert ((got[0] - ref.loss).abs() <= ref.loss_bound()).all()
    sure = torch.nn.functional.one_hot(ref.z.argmax(-1), N).double()
    assert (ref.probabilities[clear] - sure[clear]).abs().max() < 2.0 ** -100
    # a probability of 1 and of 0 is no less; what is wanted is off by its roundings, and what is made of both by those of products and sums
    ref.probabilities, ref.off = sure, torch.zeros_like(ref.off)
    dx_bound, ds_bound = ref.gradient_bounds()
    assert ((got[1] - ref.dx).abs() <= dx_bound).all()
    assert ((got[2] - ref.ds).abs() <= ds_bound + losses.U * ref.ds.abs()).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("up", [2.0 ** 3, 2.0 ** 14, 2.0 ** 20])
@pytest.mark.parametrize("M", [3, 60])
def test_two_logits_share_the_lead(M, up, dtype):
    """Two columns that are alike, far above all others: half of the probability is each one's, and a row that wants either has lost the logarithm of 2 and no more."""
    K, N = 64, 500
    w = losses.head(K, N, F32, M)[0]
    w[:, 7], w[:, 400] = 1, 1
    x = losses.rows(M, K, dtype, M).abs() + 1
    weight, s = device_weight(w), torch.full((N,), up).cuda()
    t = torch.tensor([7, 400] * M)[:M].cuda()
    with torch.no_grad():
        loss = ops.cross_entropy(weight, x.cuda(), t, s).cpu().double()
        one = ops.distillation(weight, x.cuda(), t[:, None], torch.zeros((M, 1)).cuda(), s).cpu().double()
    z = (x.double() @ torch.as_tensor(w).double()) * up
    most = z.topk(3, -1).values
    assert (most[:, 0] == most[:, 1]).all() and (most[:, 1] - most[:, 2] > 100).all()
    # (both passes' sums and logits are exact but for the factor that makes exponents of 2 of them, the same for both columns; a logarithm and a product are left)
    assert ((loss - 0.6931471805599453).abs() <= 8 * losses.U).all() and torch.equal(one, loss)
