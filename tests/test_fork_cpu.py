"""Sequences of a paged cache that go on from the same tokens, on the host alone: which pages they hold, which are copied, which stand in a group."""
import ctypes
import random

import pytest
import torch

from ternaryllm_amd import PagedCache, _lib, ops


def stamp(cache, batch, seq, first, last, value):
    """Writes `value` where tokens first .. last - 1 of a sequence of the batch are kept."""
    for j in range(first, last):
        cache._rows[:, :, int(batch.table[seq, j // cache.page_size]), :, j % cache.page_size] = value
        if cache._exponents is not None:
            cache._exponents[:, :, int(batch.table[seq, j // cache.page_size]), :, j % cache.page_size] = value


def held(cache, number):
    batch = cache.whole([number])
    n = cache.length(number)
    return [float(cache._rows[0, 1, int(batch.table[0, j // cache.page_size]), 0, j % cache.page_size, 3]) for j in range(n)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_forks_keep_their_tokens(dtype):
    """Random opens, forks, extensions, truncations and closes against lists of what each sequence holds."""
    rng = random.Random(4)
    cache = PagedCache(2, 60, 1, 16, 16, dtype, device="cpu")
    text, value = {}, 0
    for _ in range(150):
        what = rng.choice(["open", "fork", "extend", "extend", "extend", "cut", "close"])
        some = rng.choice(list(text)) if text else None
        if what == "open" and len(text) < 8:
            text[cache.open()] = []
        elif what == "fork" and text and len(text) < 10:
            text[cache.fork(some)] = list(text[some])
        elif what == "extend" and text:
            chunks = [(s, rng.randint(0, 40)) for s in rng.sample(list(text), rng.randint(1, len(text)))]
            before = {s: held(cache, s) for s in text}
            try:
                batch = cache.extend(chunks)
            except RuntimeError:
                assert all(held(cache, s) == before[s] for s in text)
                continue
            for i, (s, n) in enumerate(chunks):
                value = value % 100 + 1
                stamp(cache, batch, i, len(text[s]), len(text[s]) + n, value)
                text[s] += [float(value)] * n
        elif what == "cut" and text:
            n = rng.randint(0, len(text[some]))
            cache.truncate(some, n)
            text[some] = text[some][:n]
        elif what == "close" and len(text) > 2:
            cache.close(some)
            del text[some]
        for s, want in text.items():
            assert held(cache, s) == want
        pages = {p for s in text for p in cache._sequences[s][0]}
        assert len(pages) + cache.free_pages == 60 and not pages & set(cache._free)
        assert cache._forks == sum(len(cache._sequences[s][0]) for s in text) - len(pages)
    for s in list(text):
        cache.close(s)
    assert cache.free_pages == 60 and cache._forks == 0


def test_pages_that_end_inside_are_copied_once_for_each_but_the_last():
    cache = PagedCache(1, 10, 1, 16, 16, device="cpu")
    a = cache.open()
    cache.extend([(a, 40)])
    others = [cache.fork(a) for _ in range(3)]
    assert cache.free_pages == 7
    cache.extend([(s, 1) for s in [a, *others]])
    assert cache.free_pages == 4                                 # (one of the four goes on in the page itself)
    tails = [cache._sequences[s][0][2] for s in [a, *others]]
    assert len(set(tails)) == 4
    fork = cache.fork(a)
    with pytest.raises(RuntimeError, match="needed"):
        cache.extend([(fork, 8), (a, 16 * 4)])                   # a copy and five pages of four
    assert cache.length(fork) == 41 and cache._sequences[fork][0] == cache._sequences[a][0]


def groups_of(cache, chunks):
    prefix = cache.prefix(chunks)
    return None if prefix is None else (prefix.groups.tolist(), prefix.shared.tolist())


def test_groups():
    cache = PagedCache(1, 200, 1, 16, 16, device="cpu")
    a, alone = cache.open(), cache.open()
    cache.extend([(a, 200), (alone, 90)])
    assert groups_of(cache, [(a, 1), (alone, 1)]) is None        # nothing is shared
    b, c = cache.fork(a), cache.fork(a)
    chunks = [(a, 1), (b, 3), (alone, 1), (c, 1)]
    cache.extend(chunks)
    assert groups_of(cache, chunks) == ([0, 2, 4], [192, 192, 0, 0])
    chunks = [(alone, 2), (c, 1), (a, 1), (b, 1)]
    cache.extend(chunks)
    assert groups_of(cache, chunks) == ([0, 1, 4], [0, 192, 192, 192])
    # what was only a few tokens is no group; what shares less than half of a group's is none of it
    cache.truncate(c, 40)
    near = cache.fork(c)
    assert groups_of(cache, [(c, 0), (near, 0)]) is None
    assert groups_of(cache, [(a, 0), (b, 0), (c, 0)]) == ([0, 2, 3], [192, 192, 0])
    cache.truncate(b, 130)
    assert groups_of(cache, [(a, 0), (b, 0)]) == ([0, 2], [128, 128])
    # rows of a chunk are no part of what is in front of it
    chunks = [(a, 100), (cache.fork(a), 0)]
    cache.extend(chunks)
    assert groups_of(cache, chunks) == ([0, 2], [192, 192])
    for s in (b, c, near, chunks[1][0]):
        cache.close(s)
    assert groups_of(cache, [(a, 0), (alone, 0)]) is None and cache._forks == 0


def test_prefixes_that_are_none():
    q = torch.zeros((3, 4, 64), dtype=torch.float16)
    pages = ops.Pages(torch.zeros((5, 2, 16, 64), dtype=torch.float16), torch.zeros((5, 2, 16, 64), dtype=torch.float16))
    i32 = dict(dtype=torch.int32)
    batch = ops.PageBatch(torch.zeros((2, 2), **i32), torch.zeros(3, **i32), torch.zeros(2, **i32), 1)
    good = ops.PagePrefix(torch.tensor([0, 2], **i32), torch.zeros(2, **i32))
    for bad in (good._replace(groups=good.groups.long()), good._replace(shared=good.shared[:1]), good._replace(groups=good.groups[:0]),
                good._replace(shared=torch.zeros((2, 1), **i32)), good._replace(groups=torch.zeros(4, **i32)[::2])):
        with pytest.raises(ValueError):
            ops.paged_attention(q, pages, batch, prefix=bad)
    with pytest.raises(RuntimeError, match="GPU"):               # taken, up to the GPU that is not there
        ops.paged_attention(q, pages, batch, prefix=good)


@pytest.mark.parametrize("seqs,shared,heads,kv,apart", [
    (4, 512, 32, 32, True), (64, 8192, 32, 8, True), (64, 600, 32, 8, True), (32, 1400, 32, 8, True), (16, 1400, 32, 8, True),
    (32, 600, 32, 8, False), (32, 256, 32, 8, False), (2, 512, 32, 8, False), (64, 64, 32, 8, False)])
def test_shared_tokens_are_read_apart_where_that_takes_less(seqs, shared, heads, kv, apart):
    """What the two forms took is in the comment of the rule; the workspace shows which is chosen."""
    at = ctypes.c_void_p(256)
    pages = _lib.Pages(at, at, None, None, kv * 32 * 128, 32 * 128, 128, 10000, 32, kv, 128, _lib.TL_F16)
    batch = _lib.PageBatch(at, at, at, shared // 32 + 3, shared // 32 + 3, seqs)
    prefix = _lib.PagePrefix(at, at, 1, shared)
    need = [ctypes.c_int64(0), ctypes.c_int64(0)]
    assert _lib.lib().tl_paged_attention_workspace(seqs, heads, pages, batch, 1, need[0]) == 0
    assert _lib.lib().tl_paged_attention_shared_workspace(seqs, heads, pages, batch, prefix, 1, need[1]) == 0
    assert (need[1].value != need[0].value) == apart
