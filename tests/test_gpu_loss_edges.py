"""Losses of a ternary head in calls that the documentation allows beside the ordinary: more rows than a launch has, a backward pass twice, rows and gradients of any
stride, several streams and threads at a time, the same bits every time."""
import threading

import pytest
import torch

from ternaryllm_amd import TernaryLinear, ops

from tests import losses
from tests.test_gpu_loss import check, device_weight, some_targets, some_teacher, spread

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("top", [0, 4])
def test_more_rows_than_a_launch_takes(dtype, top):
    M, K, N = 33000, 24, 70
    w, s = losses.head(K, N, dtype, 1)
    x, g = losses.rows(M, K, dtype, 1), spread(M, 1)
    weight = device_weight(w)
    dx, ds = x.cuda().requires_grad_(), s.cuda().requires_grad_()
    if top:
        gen = torch.Generator().manual_seed(3)
        ids, logits = torch.randint(0, N, (M, top), generator=gen), torch.randn((M, top), generator=gen)
        logits[::7] = -float("inf")
        there = (logits > -float("inf")).any(-1)
        wanted = torch.zeros((M, N), dtype=torch.float64).scatter_add_(1, ids, torch.softmax(logits.double(), -1).nan_to_num(0.0))
        ref = losses.Reference(x, w, s, wanted, there, grad=g)
        loss = ops.distillation(weight, dx, ids.cuda(), logits.cuda(), ds, back=ops.BackWeight(weight))
    else:
        t = some_targets(M, N, 1)
        wanted = torch.nn.functional.one_hot(t.clamp(min=0), N).double() * (t >= 0)[:, None]
        ref = losses.Reference(x, w, s, wanted, t >= 0, grad=g)
        loss = ops.cross_entropy(weight, dx, t.cuda(), ds, back=ops.BackWeight(weight))
    check(ref, loss, *torch.autograd.grad(loss, (dx, ds), g.cuda()), dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("M,N", [(1, 40), (30, 5003), (60, 333), (300, 17000)])
def test_the_same_bits_every_time(M, N, dtype):
    w, s = losses.head(72, N, dtype, M)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    x, t, g = losses.long_rows(M, 72, M).to(dtype).cuda().requires_grad_(), some_targets(M, N, M).cuda(), spread(M, M).cuda()
    ids, logits = (y.cuda() for y in some_teacher(M, N, 9, M))
    s = s.cuda().requires_grad_()
    first = None
    for _ in range(4):
        loss = ops.cross_entropy(weight, x, t, s, back=back) + ops.distillation(weight, x, ids, logits, s, temperature=2.0, back=back)
        got = [loss.detach(), *torch.autograd.grad(loss, (x, s), g, retain_graph=True)]
        again = torch.autograd.grad(loss, (x, s), g)             # (a second time from what the first left)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first)) and all(torch.equal(a, b) for a, b in zip(again, got[1:]))


@pytest.mark.parametrize("M", [5, 90])
def test_gradients_of_any_stride_and_one_of_two(M):
    w, s = losses.head(40, 200, F16, 2)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    x, t, g = losses.rows(M, 40, F16, 2), some_targets(M, 200, 2).cuda(), spread(2 * M, 2)[::2].cuda()
    both = [x.cuda().requires_grad_(), s.cuda().requires_grad_()]
    want = torch.autograd.grad(ops.cross_entropy(weight, both[0], t, both[1], back=back), both, g)
    strided = spread(2 * M, 2).cuda()[::2]
    got = torch.autograd.grad(ops.cross_entropy(weight, both[0], t, both[1], back=back), both, strided)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for i in (0, 1):
        loss = ops.cross_entropy(weight, both[0], t, both[1], back=back)
        only, = torch.autograd.grad(loss, both[i], g)
        assert torch.equal(only, want[i])
    # rows that need no gradient, and scales that do: no transposed codes
    loss = ops.cross_entropy(weight, x.cuda(), t, both[1])
    assert torch.equal(torch.autograd.grad(loss, both[1], g)[0], want[1])


@pytest.mark.parametrize("M", [9, 200])
def test_threads_and_streams_at_once(M):
    w, s = losses.head(64, 3000, F16, 3)
    weight = device_weight(w)
    back = ops.BackWeight(weight)
    s = s.cuda()
    inputs = [(losses.rows(M, 64, F16, i).cuda(), some_targets(M, 3000, i).cuda(), spread(M, i).cuda()) for i in range(4)]

    def step(x, t, g):
        leaf, scale = x.detach().requires_grad_(), s.detach().requires_grad_()
        loss = ops.cross_entropy(weight, leaf, t, scale, back=back)
        return [loss.detach(), *torch.autograd.grad(loss, (leaf, scale), g)]

    want = [step(*i) for i in inputs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = step(*inputs[i])
                stream.synchronize()
                wrong.extend(i for a, b in zip(got, want[i]) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_module_that_takes_another_state():
    """The transposed codes go with the weight: another state's are made anew."""
    heads = [TernaryLinear(64, 300, bias=False, reference_buffers=False, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    x, t = losses.rows(6, 64, F16).cuda().requires_grad_(), some_targets(6, 300, 1).cuda()
    want = [torch.autograd.grad(h.cross_entropy(x, t).sum(), x)[0] for h in heads]
    heads[0].load_state_dict(heads[1].state_dict())
    assert torch.equal(torch.autograd.grad(heads[0].cross_entropy(x, t).sum(), x)[0], want[1]) and not torch.equal(*want)
    # rows of any shape
    y = losses.rows(6, 64, F16).cuda().view(2, 3, 64).requires_grad_()
    loss = heads[0].cross_entropy(y, t.view(2, 3))
    assert loss.shape == (2, 3) and torch.equal(torch.autograd.grad(loss.sum(), y)[0].view(6, 64), want[1])
    assert heads[0].cross_entropy(x[0], t[0]).shape == ()
