"""A decoder over a paged cache: chunks and single tokens of several sequences in one pass, against the fp32 restatement of the whole model."""
import pytest
import torch

from tests.test_gpu_decoder import TINY_TOL, _reference_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda):
    from ternaryllm_amd import TernaryConfig, TernaryLlamaDecoder
    cfg = TernaryConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=4, vocab_size=320,
                        max_position_embeddings=200, sparsity=0.66)
    return TernaryLlamaDecoder(cfg, seed=5, device=cuda, pack_threads=2)


def tokens_of(model, lengths, cuda):
    g = torch.Generator().manual_seed(9)
    return [torch.randint(0, model.config.vocab_size, (n,), generator=g).to(cuda) for n in lengths]


# passes over three sequences of 70, 33 and 130 tokens: (tokens of each in the pass)
PASSES = [[(70, 0, 0)], [(30, 5, 130), (40, 28, 0)], [(69, 32, 1), (1, 1, 100), (0, 0, 29)], [(16, 16, 16), (1, 1, 1), (53, 16, 113)]]


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("passes", PASSES)
def test_passes_match_the_reference(model, cuda, passes, page):
    text = tokens_of(model, (70, 33, 130), cuda)
    want = [_reference_logits(model, t[None])[0] for t in text]
    scale = max(w.abs().max().item() for w in want)
    cache = model.paged_cache(40, page)
    for _ in range(2):                                           # the second time in pages that the first gave back, in another order
        numbers = [cache.open() for _ in text]
        for step in passes:
            chunks = [(i, n) for i, n in enumerate(step) if n]
            logits = model.extend(cache, [(numbers[i], text[i][cache.length(numbers[i]):cache.length(numbers[i]) + n]) for i, n in chunks])
            for (i, _), got in zip(chunks, logits):
                worst = (got.float() - want[i][cache.length(numbers[i]) - 1]).abs().max().item() / scale
                assert worst <= TINY_TOL, (step, i, worst)
        for n in numbers:
            cache.close(n)
    assert cache.free_pages == 40


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_a_prompt_at_once_and_token_by_token(model, cuda, dtype):
    """The same cache rows, so the same logits up to what the order of the passes rounds."""
    text, = tokens_of(model, (50,), cuda)
    cache = model.paged_cache(20, 16, dtype)
    a, b = cache.open(), cache.open()
    at_once = model.extend(cache, [(a, text)]).float()
    for t in text:
        stepwise = model.extend(cache, [(b, t[None])]).float()
    scale = at_once.abs().max().item()
    # rows of 8 bits: a value that rounds to its other neighbour, 2^-3 of it, where the passes' own roundings differ
    assert (at_once - stepwise).abs().max().item() <= (TINY_TOL if dtype == torch.float16 else 2.0 ** -3) * scale


def test_truncated_tokens_are_forgotten(model, cuda):
    text, other = tokens_of(model, (60, 60), cuda)
    cache = model.paged_cache(20, 16)
    s, fresh = cache.open(), cache.open()
    model.extend(cache, [(s, text)])
    cache.truncate(s, 37)
    got = model.extend(cache, [(s, other[:9])])
    want = model.extend(cache, [(fresh, torch.cat([text[:37], other[:9]]))])
    assert (got.float() - want.float()).abs().max() <= TINY_TOL * want.float().abs().max()


def test_a_captured_step_serves_other_sequences_and_lengths(model, cuda):
    """Steps of three sequences captured once; between the replays the batch's tensors take other values.  Every replay gives the eager bits."""
    text = tokens_of(model, (70, 33, 130), cuda)
    cache = model.paged_cache(60, 16)
    numbers = [cache.open() for _ in text]
    model.extend(cache, [(n, t[:20]) for n, t in zip(numbers, text)])
    columns = 10
    table, starts, lengths = torch.zeros((3, columns), dtype=torch.int32, device=cuda), torch.arange(4, dtype=torch.int32, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda)
    tokens = torch.zeros(3, dtype=torch.long, device=cuda)
    from ternaryllm_amd import ops
    batch = ops.PageBatch(table, starts, lengths, 1)

    def take(order, at):
        new = cache.extend([(numbers[i], 1) for i in order])
        table.zero_()
        table[:, :new.table.shape[1]] = new.table
        lengths.copy_(new.lengths)
        tokens.copy_(torch.stack([text[i][at] for i in order]))

    take((0, 1, 2), 20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        model.extend_batch(cache, tokens, batch)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.extend_batch(cache, tokens, batch)
    for at, order in ((21, (2, 0, 1)), (22, (0, 1, 2)), (23, (1, 2, 0)), (24, (1, 0, 2))):
        take(order, at)
        eager = model.extend_batch(cache, tokens, batch).clone()
        rows = cache._rows.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, eager) and torch.equal(cache._rows, rows)


def test_the_contiguous_cache_takes_over(model, cuda):
    text = tokens_of(model, (40, 40), cuda)
    cache = model.paged_cache(20, 32)
    numbers = [cache.open() for _ in text]
    logits = model.extend(cache, [(n, t) for n, t in zip(numbers, text)])
    assert model.adopt(cache, numbers) == 40
    st = model._decode_state(2)
    st["token"].copy_(logits.argmax(-1))
    st["pos"].fill_(40)
    st["mask"].copy_((torch.arange(model.max_seq_len, device=cuda) <= 40)[None, None, None])
    token = st["token"].clone()
    got = model._decode_step(st["token"], st["pos"], st["mask"]).float()
    want = model.extend(cache, [(n, t[None]) for n, t in zip(numbers, token)]).float()
    assert (got - want).abs().max() <= TINY_TOL * want.abs().max()
    with pytest.raises(ValueError):
        model.adopt(cache, [numbers[0], cache.open()])


def test_norms_that_are_not_as_built_and_refusals(model, cuda):
    text, = tokens_of(model, (30,), cuda)
    cache = model.paged_cache(8, 16)
    a, b = cache.open(), cache.open()
    want = model.extend(cache, [(a, text)]).float()
    calls = []
    hook = model.norm.register_forward_hook(lambda *_: calls.append(1))
    got = model.extend(cache, [(b, text)]).float()
    hook.remove()
    assert calls and (got - want).abs().max() <= TINY_TOL * want.abs().max()
    with pytest.raises(ValueError):
        model.extend(cache, [])
    with pytest.raises(ValueError):
        model.extend(cache, [(a, text[:0])])
    with pytest.raises(ValueError):
        model.extend(cache, [(a, text.repeat(6))])
    with pytest.raises(RuntimeError):
        model.extend(cache, [(a, text.repeat(4))])               # more pages than there are
    assert cache.length(a) == cache.length(b) == 30


def test_a_pass_that_raises_can_be_made_again(model, cuda):
    """A layer that raises, behind others that have written their pages: lengths and pages are as before it, and so are the logits of the next try."""
    text, other = tokens_of(model, (60, 45), cuda)
    cache = model.paged_cache(12, 16)
    a, b = cache.open(), cache.open()
    model.extend(cache, [(a, text[:20]), (b, other[:5])])
    free = cache.free_pages
    hook = model.layers[1].o_proj.register_forward_pre_hook(lambda *_: (_ for _ in ()).throw(RuntimeError("stopped")))
    try:
        with pytest.raises(RuntimeError, match="stopped"):
            model.extend(cache, [(a, other[:30]), (b, text[:40])])
    finally:
        hook.remove()
    assert (cache.length(a), cache.length(b), cache.free_pages) == (20, 5, free)
    got = model.extend(cache, [(a, text[20:]), (b, other[5:])])
    fresh = model.paged_cache(12, 16)
    numbers = fresh.open(), fresh.open()
    model.extend(fresh, [(numbers[0], text[:20]), (numbers[1], other[:5])])
    want = model.extend(fresh, [(numbers[0], text[20:]), (numbers[1], other[5:])])
    assert torch.equal(got, want)


def test_the_first_pass_may_be_the_captured_one(cuda):
    """Nothing of a pass is left to be made on the host at its first call, in a decoder made on the GPU or moved there."""
    from ternaryllm_amd import TernaryConfig, TernaryLlamaDecoder
    cfg = TernaryConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2, vocab_size=128,
                        max_position_embeddings=100, sparsity=0.66)
    for model in (TernaryLlamaDecoder(cfg, seed=5, device=cuda, pack_threads=2), TernaryLlamaDecoder(cfg, seed=5, device="cpu", pack_threads=2).to(cuda)):
        cache = model.paged_cache(10, 16)
        text = torch.arange(6, device=cuda)
        batch = cache.extend([(cache.open(), 4), (cache.open(), 2)])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model.extend_batch(cache, text, batch)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            got = logits.clone()
            assert torch.equal(model.extend_batch(cache, text, batch), got)
