"""Continuations of one prompt in a decoder, and what they are worth: forks of a sequence attended together, tokens rated, a teacher compared with, against the
fp32 restatement of the whole model; the head's module on its own."""
import pytest
import torch

from ternaryllm_amd import TernaryLinear, ops

from tests import losses
from tests.test_gpu_decoder import TINY_TOL, _reference_logits
from tests.test_gpu_paged_decoder import model, tokens_of  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def forked(model, prompt, count, page=16, dtype=torch.float16, pages=80):
    """A prompt and `count` sequences that go on from all of its tokens but the last."""
    cache = model.paged_cache(pages, page, dtype)
    first = cache.open()
    model.extend(cache, [(first, prompt[:-1])])
    return cache, [cache.fork(first) for _ in range(count)]


@pytest.mark.parametrize("page", [16, 64])
def test_continuations_match_the_reference(model, cuda, page):
    prompt, *answers = tokens_of(model, (101, 1, 7, 30, 12, 2), cuda)
    cache, seqs = forked(model, prompt, len(answers), page)
    assert cache.free_pages >= 80 - -(-101 // page)
    whole = [torch.cat([prompt, t]) for t in answers]
    want = [_reference_logits(model, t[None])[0] for t in whole]
    scale = max(w.abs().max().item() for w in want)
    chunks = [(s, torch.cat([prompt[-1:], t])) for s, t in zip(seqs, answers)]
    got = model.score(cache, chunks)
    for rated, w, t in zip(got, want, answers):
        logs = torch.log_softmax(w.float(), -1)[100:-1].gather(1, t[:, None])[:, 0]
        assert rated.dtype == torch.float32 and rated.shape == t.shape
        assert (rated - logs).abs().max() <= 2 * TINY_TOL * scale        # (of a logit, and of the logarithm of their sum)
    # a token more for all of them
    more = tokens_of(model, (1, 1, 1, 1, 1), cuda)
    logits = model.extend(cache, list(zip(seqs, more)))
    for y, t, m in zip(logits, whole, more):
        w = _reference_logits(model, torch.cat([t, m])[None])[0, -1]
        assert (y.float() - w).abs().max().item() <= TINY_TOL * scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_forks_give_what_sequences_of_their_own_give(model, cuda, dtype):
    prompt, *answers = tokens_of(model, (140, 5, 9, 1), cuda)
    cache, seqs = forked(model, prompt, 3, dtype=dtype)
    apart = model.paged_cache(80, 16, dtype)
    alone = [apart.open() for _ in answers]
    for s in alone:
        model.extend(apart, [(s, prompt[:-1])])
    for step in range(3):
        chunks = [torch.cat([prompt[-1:], t]) if step == 0 else t[:1] for t in answers]
        got = model.extend(cache, list(zip(seqs, chunks)))
        want = model.extend(apart, list(zip(alone, chunks)))
        assert cache.prefix([(s, 1) for s in seqs]) is not None and apart.prefix([(s, 1) for s in alone]) is None
        scale = want.float().abs().max().item()
        assert (got.float() - want.float()).abs().max().item() <= (TINY_TOL if dtype == torch.float16 else 2.0 ** -3) * scale


def test_divergence_from_a_teacher(model, cuda):
    prompt, *answers = tokens_of(model, (80, 6, 1, 20), cuda)
    cache, seqs = forked(model, prompt, 3)
    chunks = [(s, torch.cat([prompt[-1:], t])) for s, t in zip(seqs, answers)]
    g = torch.Generator().manual_seed(3)
    teacher = [(torch.randint(0, 320, (t.numel(), 8), generator=g).to(cuda), (3 * torch.randn((t.numel(), 8), generator=g)).to(cuda)) for _, t in chunks]
    got = model.divergence(cache, chunks, teacher, temperature=2.0)
    for y, (_, t), (ids, logits), a in zip(got, chunks, teacher, answers):
        z = _reference_logits(model, torch.cat([prompt, a])[None])[0, 79:].cpu().double()
        wanted, _ = losses.teacher(ids.cpu(), logits.cpu(), 320, 2.0)
        gap = (torch.special.xlogy(wanted, wanted) - wanted * torch.log_softmax(z / 2.0, -1)).sum(-1) * 4
        assert y.shape == t.shape and (y.cpu() - gap).abs().max() <= 4 * 2 * TINY_TOL * float(z.abs().max()) / 2


def test_a_pass_that_raises_leaves_forks_as_they_were(model, cuda):
    prompt, answer = tokens_of(model, (60, 5), cuda)
    cache, (a, b) = forked(model, prompt, 2)
    want = model.extend(cache, [(a, answer), (b, answer)])
    for s in (a, b):
        cache.truncate(s, 59)
    before = cache.free_pages
    with pytest.raises(ValueError):
        model.divergence(cache, [(a, answer), (b, answer)], [(torch.zeros((5, 0), dtype=torch.long).cuda(), torch.zeros((5, 0)).cuda())] * 2)
    with pytest.raises(ValueError):
        model.divergence(cache, [(a, answer)], [])
    assert cache.length(a) == cache.length(b) == 59 and cache.free_pages <= before
    assert torch.equal(model.extend(cache, [(a, answer), (b, answer)]), want)


def test_a_captured_pass_over_forks(model, cuda):
    """Captured once for three sequences of one group; replayed over other groups and lengths it gives the eager bits."""
    prompt, other = tokens_of(model, (100, 130), cuda)
    cache, seqs = forked(model, prompt, 3)
    cache2 = cache.open()
    model.extend(cache, [(cache2, other)])
    more = [cache2, cache.fork(cache2), cache.fork(cache2)]
    tokens = torch.zeros(3, dtype=torch.long, device=cuda)
    batch = ops.PageBatch(torch.zeros((3, 20), dtype=torch.int32, device=cuda), torch.arange(4, dtype=torch.int32, device=cuda),
                          torch.zeros(3, dtype=torch.int32, device=cuda), 1)
    prefix = ops.PagePrefix(torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda), 1 << 30)

    def fill(numbers, token):
        tokens.fill_(token)
        tokens[1] += 1
        chunks = [(s, 1) for s in numbers]
        now, groups = cache.extend(chunks), cache.prefix(chunks)
        batch.table[:, :now.table.shape[1]] = now.table
        batch.lengths.copy_(now.lengths)
        prefix.groups.copy_(groups.groups)
        prefix.shared.copy_(groups.shared)

    fill(seqs, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.extend_batch(cache, tokens, batch, prefix)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.extend_batch(cache, tokens, batch, prefix)
    for i, numbers in enumerate((seqs, more, seqs, more)):
        fill(numbers, 20 + i)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, model.extend_batch(cache, tokens, batch, prefix))


def test_the_heads_module(cuda):
    """A step of two heads that are tuned by their scales, and a state that is loaded in between."""
    w, s = losses.head(128, 500, torch.float16, 1)
    linear = TernaryLinear(128, 500, bias=False, weight=w, scale=s, reference_buffers=False).to(cuda)
    linear.w_scale.requires_grad_()
    x, t = losses.rows(60, 128, torch.float16, 1), torch.randint(0, 500, (5, 12), generator=torch.Generator().manual_seed(1))
    for _ in range(2):
        leaf = x.to(cuda).view(5, 12, 128).requires_grad_()
        loss = linear.cross_entropy(leaf, t.to(cuda))
        assert loss.shape == (5, 12)
        gx, gs = torch.autograd.grad(loss.sum(), (leaf, linear.w_scale))
        ref = losses.Reference(x, linear.ternary_weight, linear.w_scale.detach().cpu(), *losses.targets(t.flatten(), 500))
        bounds = ref.gradient_bounds()
        assert ((loss.detach().cpu().double().flatten() - ref.loss).abs() <= ref.loss_bound()).all()
        assert ((gx.cpu().double().view(60, 128) - ref.dx).abs() <= bounds[0]).all()
        assert ((gs.cpu().double() - ref.ds).abs() <= bounds[1] + 2.0 ** -11 * ref.ds.abs() + 2.0 ** -25).all()
        other = TernaryLinear(128, 500, bias=False, weight=losses.head(128, 500, torch.float16, 7)[0], scale=losses.head(128, 500, torch.float16, 8)[1],
                              reference_buffers=False)
        linear.w_scale.requires_grad_(False)
        linear.load_state_dict(other.state_dict())
        linear.w_scale.requires_grad_()
    ids, logits = t[:, :1, None].expand(5, 12, 3).to(cuda), torch.zeros((5, 12, 3), device=cuda)
    with torch.no_grad():                                        # one id three times is the target
        a = linear.distillation(x.to(cuda).view(5, 12, 128), ids, logits)
        b = linear.cross_entropy(x.to(cuda).view(5, 12, 128), ids[..., 0])
    assert ((a - b).abs() <= 1e-5 * b.abs() + 1e-5).all()


def test_losses_are_differentiable_once_and_notice_changes(cuda):
    w, s = losses.head(64, 100, torch.float32)
    weight = ops.DeviceWeight(__import__("ternaryllm_amd").packing.PackedWeight.from_dense(torch.as_tensor(w)), "cuda")
    back = ops.BackWeight(weight)
    x, t, s = losses.rows(6, 64, torch.float32).cuda().requires_grad_(), torch.arange(6).cuda(), s.cuda()
    loss = ops.cross_entropy(weight, x, t, s, back=back)
    first, = torch.autograd.grad(loss.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(first.sum(), x)
    loss = ops.cross_entropy(weight, x, t, s, back=back)
    want, = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    again, = torch.autograd.grad(loss.sum(), x)
    assert torch.equal(want, again)
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(loss.sum(), x)
    loss = ops.cross_entropy(weight, x, t, s, back=back)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(loss.sum(), x)
    # by the scales alone, without the transposed codes; in a graph with other operators; accumulated
    scale = s.clone().requires_grad_()
    loss = ops.cross_entropy(weight, x.detach(), t, scale)
    gs, = torch.autograd.grad(loss.mean(), scale)
    assert gs.isfinite().all()
    mix = torch.eye(64, device="cuda").requires_grad_()
    for _ in range(2):
        (ops.cross_entropy(weight, x.detach() @ mix, t, s, back=back).mean() * 0.5).backward()
    plain = x.detach().requires_grad_()
    g, = torch.autograd.grad(ops.cross_entropy(weight, plain, t, s, back=back).mean(), plain)
    want = x.detach().t() @ g
    assert ((mix.grad - want).abs() <= 1e-4 * want.abs().max()).all()


def test_captures_that_would_meet_an_eager_graph_are_refused(cuda):
    """On the host, in front of any launch.  The capture goes on with another leaf."""
    w, s = losses.head(64, 100, torch.float16)
    linear = TernaryLinear(64, 100, bias=False, weight=w, scale=s, reference_buffers=False).to(cuda)
    x, t = losses.rows(60, 64, torch.float16).cuda(), torch.arange(60).cuda()
    leaf = x.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    fresh = linear.__class__(64, 100, bias=False, weight=w, scale=s, reference_buffers=False).to(cuda)
    alive = linear.cross_entropy(leaf, t)
    want, = torch.autograd.grad(alive.sum(), leaf, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="lives outside"):
            linear.cross_entropy(leaf, t)
        with pytest.raises(RuntimeError, match="transposed"):
            fresh.cross_entropy(x.detach().requires_grad_(), t)
        other = x.detach().requires_grad_()
        out, = torch.autograd.grad(linear.cross_entropy(other, t), other, torch.ones(60, device=cuda))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_captures_whose_operands_lead_to_an_eager_graph_are_refused(cuda):
    """Rows that were worked out in the captured graph from a leaf that an eager one holds; a leaf of the captured graph's own goes on."""
    w, s = losses.head(64, 100, torch.float16)
    linear = TernaryLinear(64, 100, bias=False, weight=w, scale=s, reference_buffers=False).to(cuda)
    x, t = losses.rows(60, 64, torch.float16).cuda(), torch.arange(60).cuda()
    leaf = x.clone().requires_grad_()
    alive = linear.cross_entropy(leaf * 0.5, t)
    want, = torch.autograd.grad(alive.sum(), leaf, retain_graph=True)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(RuntimeError, match="lives outside"):
            linear.cross_entropy(leaf * 0.5, t)
        other = x.detach().requires_grad_()
        out, = torch.autograd.grad(linear.cross_entropy(other * 0.5, t), other, torch.ones(60, device=cuda))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del alive
