"""Cross entropy and distillation of a ternary head against float64 on the CPU (tests/losses.py): rows and sizes at the edges of tiles, pieces and fragments."""
import math

import pytest
import torch

from ternaryllm_amd import ops, packing

from tests import losses

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32
# rows, K, N
SIZES = [(1, 64, 100), (1, 5, 1), (2, 200, 7), (3, 1, 16), (17, 257, 129), (48, 512, 1000), (49, 64, 130), (64, 300, 5003), (130, 136, 777), (257, 1000, 513),
         (5, 72, 16385), (60, 40, 33000)]


def device_weight(w):
    return ops.DeviceWeight(packing.PackedWeight.from_dense(torch.as_tensor(w)), "cuda")


def spread(M, seed):
    return 0.25 + torch.rand(M, generator=torch.Generator().manual_seed(seed + 3))


def some_targets(M, N, seed):
    t = torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(seed + 4))
    t[0], t[-1] = N - 1, 0
    if M > 2:
        t[1::5] = -100
    return t


def some_teacher(M, N, top, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed + 5)
    ids = torch.randint(0, N, (M, top), generator=g)                 # (some are there twice)
    logits = (3 * torch.randn((M, top), generator=g)).to(dtype)
    if M > 2:
        logits[1::5] = -math.inf                                     # rows without a teacher
        ids[1::5] = -7
        logits[2, top // 2:] = -math.inf if top > 1 else logits[2, 0]
    return ids, logits


def check(ref, loss, dx=None, ds=None, scale_dtype=None):
    assert loss.dtype == F32 and ((loss.detach().cpu().double() - ref.loss).abs() <= ref.loss_bound()).all()
    if dx is None:
        return
    dx_bound, ds_bound = ref.gradient_bounds()
    # (a result past the largest number of its type rounds to infinity: from the middle between that number and the next power of two's step on)
    got, most = dx.cpu().double(), torch.finfo(ref.dtype).max * (1 + torch.finfo(ref.dtype).eps / 4)
    past = (got.abs() == math.inf) & (got.sign() == ref.dx.sign()) & (ref.dx.abs() + dx_bound >= most)
    assert dx.dtype == ref.dtype and (past | ((got - ref.dx).abs() <= dx_bound)).all()
    assert (dx.cpu()[~ref.counts] == 0).all()
    if ds is not None:
        half = torch.finfo(scale_dtype).eps / 2
        assert ds.dtype == scale_dtype and ((ds.cpu().double() - ref.ds).abs() <= ds_bound + half * ref.ds.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("scale_dtype", [F16, F32, None])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_cross_entropy(M, K, N, dtype, scale_dtype):
    w, s = losses.head(K, N, scale_dtype or F32, M, scaled=scale_dtype is not None)
    x, t, g = losses.rows(M, K, dtype, M), some_targets(M, N, K), spread(M, N)
    ref = losses.Reference(x, w, s, *losses.targets(t, N), grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), None if s is None else s.cuda().requires_grad_()
    loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    wanted = [dx] if ds is None else [dx, ds]
    grads = torch.autograd.grad(loss, wanted, g.cuda())
    check(ref, loss, *grads, *([None, None] if ds is None else [scale_dtype])[:2 - len(grads) + 1])
    with torch.no_grad():                                            # the same bits without a gradient
        assert torch.equal(ops.cross_entropy(weight, x.cuda(), t.cuda(), None if s is None else s.cuda()), loss)


@pytest.mark.parametrize("top,heat", [(1, 1.0), (5, 2.0), (64, 0.5), (130, 1.0)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("M,K,N", [(1, 64, 100), (17, 257, 129), (48, 512, 1000), (49, 64, 130), (130, 136, 777), (60, 40, 33000)])
def test_distillation(M, K, N, dtype, top, heat):
    w, s = losses.head(K, N, dtype, M)
    x, g = losses.rows(M, K, dtype, M), spread(M, N)
    ids, logits = some_teacher(M, N, top, K, F16 if top == 5 else F32)
    ref = losses.Reference(x, w, s, *losses.teacher(ids, logits, N, heat), heat=heat, grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, temperature=heat, back=ops.BackWeight(weight))
    check(ref, loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()), dtype)


def test_one_entry_is_cross_entropy():
    w, s = losses.head(128, 500, F16)
    weight, x, t = device_weight(w), losses.rows(70, 128, F16).cuda(), some_targets(70, 500, 1).clamp(min=0).cuda()
    loss = ops.cross_entropy(weight, x, t, s.cuda())
    assert torch.equal(ops.distillation(weight, x, t[:, None], torch.full((70, 1), -3.0).cuda(), s.cuda()), loss)


@pytest.mark.parametrize("M", [3, 40, 70])
def test_gradients_are_those_of_differences(M):
    """Along a direction, of what moves the loss by differences that float64 resolves."""
    w, s = losses.head(96, 300, F32, 4)
    x, ids_logits, g = losses.rows(M, 96, F32, 4), some_teacher(M, 300, 6, 4), spread(M, 4)
    wanted, counts = losses.teacher(*ids_logits, 300, 1.5)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.distillation(weight, dx, ids_logits[0].cuda(), ids_logits[1].cuda(), ds, temperature=1.5, back=ops.BackWeight(weight))
    got = torch.autograd.grad(loss, (dx, ds), g.cuda())
    gen = torch.Generator().manual_seed(9)
    for i, at in enumerate((x, s)):
        along = torch.randn(at.shape, generator=gen, dtype=torch.float64)
        step = 1e-5
        moved = []
        for sign in (1, -1):
            there = [x.double(), s.double()]
            there[i] = there[i] + sign * step * along
            moved.append(float((losses.Reference(*(there[0], w, there[1]), wanted, counts, heat=1.5).loss * g.double()).sum()))
        want = (moved[0] - moved[1]) / (2 * step)
        ref = losses.Reference(x, w, s, wanted, counts, heat=1.5, grad=g)
        bound = float((ref.gradient_bounds()[i] * along.abs()).sum()) + 1e-6 * float((torch.stack([ref.dx.abs().sum(), ref.ds.abs().sum()])[i]))
        assert abs(float((got[i].cpu().double() * along).sum()) - want) <= bound


def test_rows_that_are_not_finite_stay_by_themselves():
    for M in (4, 60):
        w, s = losses.head(64, 200, F16)
        x, t = losses.rows(M, 64, F16), some_targets(M, 200, 2)
        t[:] = torch.arange(M)
        bad = x.clone()
        bad[1, 3], bad[2, 5] = math.nan, math.inf
        t[3] = -100
        bad[3] = math.nan                                            # a row that counts for nothing
        weight = device_weight(w)
        back = ops.BackWeight(weight)
        dx, ds = bad.cuda().requires_grad_(), s.cuda().requires_grad_()
        loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=back)
        gx, gs = torch.autograd.grad(loss.sum(), (dx, ds))
        ref = losses.Reference(x, w, s, *losses.targets(t, 200))
        fine = torch.tensor([i not in (1, 2) for i in range(M)])
        assert loss[1:3].isnan().all() and gx[1:3].isnan().all() and gs.isnan().all() and loss[3] == 0 and (gx[3] == 0).all()
        assert ((loss.detach().cpu().double() - ref.loss).abs() <= ref.loss_bound())[fine].all()
        assert ((gx.cpu().double() - ref.dx).abs() <= ref.gradient_bounds()[0])[fine].all()


def test_targets_and_ids_that_are_no_columns():
    w, s = losses.head(64, 200, F16)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    for M in (6, 70):
        t = torch.randint(0, 200, (M,))
        t[1], t[2], t[3] = 200, -1, 1 << 40
        x = losses.rows(M, 64, F16).cuda().requires_grad_()
        loss = ops.cross_entropy(weight, x, t.cuda(), s.cuda(), back=back)
        gx, = torch.autograd.grad(loss.sum(), x)
        assert loss[1:4].isnan().all() and gx[1:4].isnan().all() and loss[4:].isfinite().all() and gx[4:].isfinite().all() and gx[0].isfinite().all()
        ids, logits = torch.randint(0, 200, (M, 3)), torch.randn((M, 3))
        ids[1, 2], ids[2, 0], logits[3, 1], logits[4, 1] = 200, -1, math.nan, math.inf
        loss = ops.distillation(weight, x, ids.cuda(), logits.cuda(), s.cuda(), back=back)
        gx, = torch.autograd.grad(loss.sum(), x)
        assert loss[1:5].isnan().all() and gx[1:5].isnan().all() and loss[5:].isfinite().all() and gx[5:].isfinite().all()


@pytest.mark.parametrize("M", [5, 80])
def test_large_logits_and_scales(M):
    """Logits of thousands, scales whose largest is far above the others, and gradients of the losses of any size."""
    w, _ = losses.head(64, 400, F32)
    s = torch.exp2(torch.arange(400) % 23 - 12.0)
    x, t, g = losses.rows(M, 64, F16), torch.randint(0, 400, (M,), generator=torch.Generator().manual_seed(1)), torch.exp2(torch.arange(M) % 30 - 20.0)
    ref = losses.Reference(x, w, s, *losses.targets(t, 400), grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    check(ref, loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()), F32)


def test_strides_and_another_stream():
    w, s = losses.head(72, 333, F16)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    for M in (9, 90):
        x, t, g = losses.rows(M, 72, F16, M), some_targets(M, 333, M), spread(M, M)
        plain = x.cuda().requires_grad_()
        loss = ops.cross_entropy(weight, plain, t.cuda(), s.cuda(), back=back)
        gx, = torch.autograd.grad(loss, plain, g.cuda())
        wide = torch.full((M, 200), math.nan, dtype=F16, device="cuda")
        for view in (wide[:, 8:80], wide[:, 3:75], wide[:, 56:200:2]):
            view.copy_(x)
            other = torch.cuda.Stream()
            other.wait_stream(torch.cuda.current_stream())
            leaf = view.detach().requires_grad_()
            with torch.cuda.stream(other):
                again = ops.cross_entropy(weight, leaf, t.cuda().expand(2, M)[1], s.cuda(), back=back)
                gy, = torch.autograd.grad(again, leaf, g.cuda())
            torch.cuda.current_stream().wait_stream(other)
            assert torch.equal(again, loss) and torch.equal(gx, gy)
        # a gradient that is one value for all rows
        assert torch.equal(torch.autograd.grad(ops.cross_entropy(weight, plain, t.cuda(), s.cuda(), back=back).sum(), plain)[0],
                           torch.autograd.grad(ops.cross_entropy(weight, plain, t.cuda(), s.cuda(), back=back), plain, torch.ones(M).cuda())[0])


def test_without_rows():
    w, s = losses.head(64, 100, F16)
    weight = device_weight(w)
    x, s = torch.zeros((0, 64), dtype=F16).cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.cross_entropy(weight, x, torch.zeros(0, dtype=torch.int64).cuda(), s, back=ops.BackWeight(weight))
    gx, gs = torch.autograd.grad(loss.sum(), (x, s))
    assert loss.shape == (0,) and gx.shape == (0, 64) and (gs == 0).all()
    assert ops.distillation(weight, x, torch.zeros((0, 3), dtype=torch.int64).cuda(), torch.zeros((0, 3)).cuda(), s, back=ops.BackWeight(weight)).shape == (0,)


@pytest.mark.parametrize("M", [7, 100])
def test_a_captured_step(M):
    """Replayed over other rows, with the program's own eager work between the replays."""
    w, s = losses.head(128, 1000, F16)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    x, t, g = (torch.zeros((M, 128), dtype=F16).cuda(), torch.zeros(M, dtype=torch.int64).cuda(), spread(M, 1).cuda())
    s = s.cuda()
    ids, logits = torch.zeros((M, 4), dtype=torch.int64).cuda(), torch.zeros((M, 4)).cuda()

    def step():
        leaf, scale = x.detach().requires_grad_(), s.detach().requires_grad_()
        both = ops.cross_entropy(weight, leaf, t, scale, back=back) + ops.distillation(weight, leaf, ids, logits, scale, back=back)
        return both.detach(), *torch.autograd.grad(both, (leaf, scale), g)

    def fill(seed):
        x.copy_(losses.rows(M, 128, F16, seed))
        t.copy_(some_targets(M, 1000, seed))
        for to, new in zip((ids, logits), some_teacher(M, 1000, 4, seed)):
            to.copy_(new)

    fill(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(2, 6):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)
