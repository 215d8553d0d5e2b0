"""Losses of more than 48 rows at the edges of the tiles that they are multiplied in: rows of 32, 64 and 128, columns of 64 to 256, pieces of the vocabulary,
rows in several parts."""
import pytest
import torch

from ternaryllm_amd import ops

from tests import losses
from tests.test_gpu_loss import check, device_weight, some_targets, some_teacher, spread

pytestmark = pytest.mark.gpu


def step(M, K, N, dtype, top, heat=1.0, scaled=True, seed=0):
    w, s = losses.head(K, N, dtype, seed, scaled=scaled)
    x, g = losses.rows(M, K, dtype, seed), spread(M, seed)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), None if s is None else s.cuda().requires_grad_()
    if top:
        ids, logits = some_teacher(M, N, top, seed)
        ref = losses.Reference(x, w, s, *losses.teacher(ids, logits, N, heat), heat=heat, grad=g)
        loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, temperature=heat, back=ops.BackWeight(weight))
    else:
        t = some_targets(M, N, seed)
        ref = losses.Reference(x, w, s, *losses.targets(t, N), grad=g)
        loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    grads = torch.autograd.grad(loss, [dx] if ds is None else [dx, ds], g.cuda())
    check(ref, loss, *grads, *([None] if ds is None else []), *([dtype] if ds is not None else []))


# few and many tiles of every kind; the last ones take the tallest
SIZES = [(63, 64, 250), (65, 256, 4096), (96, 264, 300), (128, 512, 8200), (129, 1030, 70), (300, 24, 9000), (400, 320, 20001), (1025, 128, 12000)]


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_tiles(M, K, N, dtype, top):
    step(M, K, N, dtype, top, 1.5 if top else 1.0, seed=M)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_in_parts(dtype):
    """More rows than the workspace of a backward pass takes at a time."""
    step(4500 if dtype == torch.float16 else 1700, 16, 16500, dtype, 2, seed=5)


@pytest.mark.parametrize("top", [200, 1000])
def test_teachers_of_many_entries(top):
    """Among so few columns that a wave has some of every row, and most ids are there more than once."""
    step(70, 40, 300, torch.float16, top, 0.7, seed=top)
    step(200, 16, 5000, torch.float32, top, 1.0, seed=top)


def test_all_entries_in_one_place():
    """Every row's teacher names the same 64 neighbouring columns, the last of the vocabulary."""
    M, K, N = 150, 64, 1000
    w, s = losses.head(K, N, torch.float16, 3)
    x, g = losses.rows(M, K, torch.float16, 3), spread(M, 3)
    ids = torch.stack([N - 1 - torch.randperm(64, generator=torch.Generator().manual_seed(m)) for m in range(M)])
    logits = torch.randn((M, 64), generator=torch.Generator().manual_seed(8))
    ref = losses.Reference(x, w, s, *losses.teacher(ids, logits, N, 1.0), grad=g)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, back=ops.BackWeight(weight))
    check(ref, loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()), torch.float16)


def test_weights_whose_rows_repeat():
    """Merged arrays may name a row several times: such a weight has more planes of codes than one, its transpose too."""
    K, N, M = 40, 90, 60
    from ternaryllm_amd import packing
    w = torch.from_numpy(losses.head(K, N, torch.float32, 6)[0])
    twice = w.clone()
    twice[::3] *= 2
    columns = [torch.cat([torch.nonzero(twice[:, n] == v)[:, 0].repeat_interleave(abs(v)) for v in (-1, -2)] + []) for n in range(N)], \
              [torch.cat([torch.nonzero(twice[:, n] == v)[:, 0].repeat_interleave(abs(v)) for v in (1, 2)]) for n in range(N)]
    arrays = []
    for side in columns:
        ends = torch.tensor([len(c) for c in side]).cumsum(0).tolist()
        arrays += [torch.cat(side).int().numpy(), torch.tensor([[a, b] for a, b in zip([0, *ends[:-1]], ends)]).int().flatten().numpy()]
    try:
        packed = packing.PackedWeight.from_tiled_csc(arrays[0], arrays[1], arrays[2], arrays[3], N, K, K)
    except ValueError:
        pytest.skip("the packer takes no repeated rows from tiled arrays")
    if packed.header.code_planes < 2 or not (packed.to_dense() == twice.numpy()).all():
        pytest.skip("no room for further planes of codes")
    weight = ops.DeviceWeight(packed, "cuda")
    for rows in (5, M):
        x, t, g = losses.rows(rows, K, torch.float16), some_targets(rows, N, 1), spread(rows, 1)
        ref = losses.Reference(x, twice, None, *losses.targets(t, N), grad=g)
        dx = x.cuda().requires_grad_()
        loss = ops.cross_entropy(weight, dx, t.cuda(), back=ops.BackWeight(weight))
        check(ref, loss, *torch.autograd.grad(loss, dx, g.cuda()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("top", [0, 7])
@pytest.mark.parametrize("M", [1, 3, 24, 25])
def test_few_rows_over_the_longest_vocabularies(M, top, dtype):
    """And the fewest rows of which logits are not kept."""
    step(M, 16, 65537 + 5, dtype, top, 2.0 if top else 1.0, seed=M)
    step(M, 24, 65536, dtype, top, seed=M)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("M", [5, 60])
def test_wanted_columns_of_no_probability(M, dtype):
    """A column whose scale takes its logits to -inf: rows that want it have an infinite loss, the others what they have without it."""
    K, N = 64, 300
    w, _ = losses.head(K, N, dtype, 4)
    w[:, 7], w[0, 7] = 0, -1
    x = losses.rows(M, K, dtype, 4).abs().clamp(min=1)
    s = torch.full((N,), 0.1)
    s[7] = float("inf")
    without = s.clone()
    without[7] = 1e30
    weight = device_weight(w)
    ids = torch.arange(M)[:, None] % 5 + torch.tensor([4, 20])           # (some rows' first is 7)
    logits = torch.randn((M, 2), generator=torch.Generator().manual_seed(1))
    hit = (ids == 7).any(-1)
    for rate in (lambda of: ops.distillation(weight, x.cuda(), ids.cuda(), logits.cuda(), of.cuda()), lambda of: ops.cross_entropy(weight, x.cuda(), ids[:, 0].cuda(), of.cuda())):
        got, want = rate(s).cpu(), rate(without).cpu()
        assert hit.any() and (got[hit] == float("inf")).all() and (want[hit] > 1e20).all()
        assert torch.equal(got[~hit], want[~hit]) and got[~hit].isfinite().all()
