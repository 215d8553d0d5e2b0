"""Attention of groups of sequences that begin alike against float64 on the CPU: sizes at the edges of pages, rounds of keys, units and parts."""
import math

import pytest
import torch

from ternaryllm_amd import ops

from tests import paged, prefixes
from tests.test_gpu_paged import attention_bound, fresh_pages, on_gpu, random

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 128), (8, 2, 128), (14, 2, 64), (4, 4, 256), (3, 1, 64), (40, 2, 128), (6, 3, 256)]
ONE, MANY = [(1, 1)], [(1, 30), (1, 1), (1, 65), (1, 64), (1, 200)]
BATCHES = [
    ([(64, ONE * 2)], 16), ([(63, ONE * 3)], 16), ([(0, ONE * 2), (65, [(1, 3)])], 16), ([(200, MANY), (128, ONE * 20)], 32),
    ([(1000, [(3, 5), (0, 40), (2, 700), (1, 1)]), (70, [(4, 4)] * 9), (10, [(1, 300), (2, 2)])], 64), ([(2600, [(1, 9)] * 70)], 256),
    ([(320, [(7, 20), (5, 5)]), (129, [(40, 90), (1, 1), (33, 64)])], 16)]


def check(groups, heads, kv, hd, page, kind, *, front=0, behind=0, most=None, seed=1, widest=None, spoiled=True):
    seqs = prefixes.Shared(groups, page, front=front, behind=behind, seed=seed, widest=widest)
    pages = fresh_pages(seqs, kv, hd, kind, seed=seed, spoiled=spoiled)
    seqs.copied(*pages)
    q = random((seqs.tokens, heads + 3, hd), seed + 9)[:, 1:1 + heads]
    out = torch.full((seqs.tokens, heads * hd), 3.0, dtype=torch.float16, device="cuda")
    wide = random((seqs.tokens, heads + 3, hd), seed + 9).cuda()
    ops.paged_attention(wide[:, 1:1 + heads], on_gpu(pages), seqs.batch(ops, most=most), out=out, prefix=seqs.prefix(ops))
    got = out.cpu().view(seqs.tokens, heads, hd)
    k, v = (paged.values(*t) for t in zip(pages[:2], pages[2:]))
    want = paged.attention(q, k, v, seqs, 1 / math.sqrt(hd))
    inside = ~want.isnan().any(-1).any(-1)
    assert (got[~inside] == 3.0).all() and int(inside.sum()) == int(seqs.starts[-1]) - front
    bound = attention_bound(q, k, v, want, max(length for _, length in seqs.both), 1 / math.sqrt(hd))
    assert ((got.double() - want).abs() <= bound)[inside].all()


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("groups,page", BATCHES)
def test_groups(kind, heads, kv, hd, groups, page):
    check(groups, heads, kv, hd, page, kind)


@pytest.mark.parametrize("groups,page", BATCHES[3:5])
def test_rows_of_no_sequence_stay_as_they_are(groups, page):
    check(groups, 8, 2, 128, page, "float16", front=2, behind=5, most=1, widest=80)


@pytest.mark.parametrize("heads,kv,hd", [(32, 32, 128), (32, 8, 128), (7, 1, 64)])
def test_long_prefixes_and_many_groups(heads, kv, hd):
    """Keys shared out among many workgroups, and more groups than a wave looks at at once."""
    check([(9000, [(1, 3), (1, 700), (1, 64)])], heads, kv, hd, 64, "float16", spoiled=False)
    check([(40 + g, [(1, 1 + g % 5)] * (1 + g % 3)) for g in range(150)], 4, 2, hd, 32, "float16", spoiled=False)


def test_the_same_bits_every_time_and_without_groups_what_the_plain_call_gives():
    seqs = prefixes.Shared([(300, [(1, 40)] * 9), (70, [(2, 9)] * 3)], 32)
    pages = fresh_pages(seqs, 2, 128, "float16")
    seqs.copied(*pages)
    q, dev, batch = random((seqs.tokens, 8, 128), 3).cuda(), on_gpu(pages), seqs.batch(ops)
    got = ops.paged_attention(q, dev, batch, prefix=seqs.prefix(ops))
    for _ in range(5):
        assert torch.equal(ops.paged_attention(q, dev, batch, prefix=seqs.prefix(ops)), got)
    plain = ops.paged_attention(q, dev, batch)
    none = ops.PagePrefix(torch.zeros(1, dtype=torch.int32).cuda(), torch.zeros(12, dtype=torch.int32).cuda())
    for prefix in (none, seqs.prefix(ops, most=None), seqs.prefix(ops, most=300)):       # (so few that they are not read apart)
        assert torch.equal(ops.paged_attention(q, dev, batch, prefix=prefix), plain)


def test_groups_that_do_not_hold():
    """Numbers that are wrong make rows NaN at most, and no other group's."""
    seqs = prefixes.Shared([(300, [(1, 40)] * 4), (128, [(2, 9)] * 3), (64, [(1, 5)] * 2)], 32)
    pages = fresh_pages(seqs, 2, 64, "float16")
    seqs.copied(*pages)
    q, dev, batch = random((seqs.tokens, 4, 64), 3).cuda(), on_gpu(pages), seqs.batch(ops)
    good = ops.paged_attention(q, dev, batch)
    prefix = seqs.prefix(ops)
    whole = ops.paged_attention(q, dev, batch, prefix=prefix)
    assert ((whole - good).abs() <= 0.01).all()
    first = slice(0, 4)
    for shared in (prefix.shared.clone().fill_(1 << 30), -prefix.shared, prefix.shared + 10000):
        mine = prefix.shared.clone()
        mine[first] = shared[first]
        y = ops.paged_attention(q, dev, batch, prefix=prefix._replace(shared=mine))
        assert y[first].isnan().all() and torch.equal(y[4:], whole[4:])
    mine = prefix.shared.clone()
    mine[2] = 128                                                # (not what the rest of its group has)
    y = ops.paged_attention(q, dev, batch, prefix=prefix._replace(shared=mine))
    assert y[2].isnan().all() and torch.equal(y[:2], whole[:2]) and torch.equal(y[3:], whole[3:])
    # groups that fall, or name sequences that there are none of
    for groups in ([0, 4, 2, 9], [-5, 4, 7, 100], [3, 3, 3, 3], [9, 9, 9, 9], [1 << 30, -1, 5, 0]):
        y = ops.paged_attention(q, dev, batch, prefix=prefix._replace(groups=torch.tensor(groups, dtype=torch.int32).cuda()))
        assert y.shape == good.shape
    # pages that are none, of the prefix and of one sequence alone
    table = batch.table.clone()
    table[0, 1] = 100000
    y = ops.paged_attention(q, dev, batch._replace(table=table), prefix=prefix)
    assert y[:4].isnan().all() and torch.equal(y[4:], whole[4:])
    table = batch.table.clone()
    table[3, 9] = -1
    y = ops.paged_attention(q, dev, batch._replace(table=table), prefix=prefix)
    assert y[3].isnan().all() and torch.equal(y[:3], whole[:3]) and torch.equal(y[4:], whole[4:])
    # more tokens than the table holds, of one sequence
    lengths = batch.lengths.clone()
    lengths[1] = 1 << 20
    y = ops.paged_attention(q, dev, batch._replace(lengths=lengths), prefix=prefix)
    assert y[1].isnan().all() and torch.equal(y[0], whole[0]) and torch.equal(y[2:], whole[2:])


@pytest.mark.parametrize("where", [0, 1])
def test_what_is_not_finite_in_a_sequence_of_its_own_stays_there(where):
    seqs = prefixes.Shared([(300, [(3, 40)] * 4)], 32)
    pages = fresh_pages(seqs, 1, 128, "float16", spoiled=False)
    seqs.copied(*pages)
    q, batch = random((seqs.tokens, 4, 128), 3).cuda(), seqs.batch(ops)
    whole = ops.paged_attention(q, on_gpu(pages), batch, prefix=seqs.prefix(ops))
    token = 338                                                  # of sequence 1: its rows are tokens 337 to 339
    pages[where][int(seqs.table[1, token // 32]), 0, token % 32, 7] = math.nan if where == 0 else math.inf
    y = ops.paged_attention(q, on_gpu(pages), batch, prefix=seqs.prefix(ops))
    assert torch.equal(y[:4], whole[:4]) and torch.equal(y[6:], whole[6:]) and not y[4:6].isfinite().all(-1).any()


def test_a_captured_call_serves_other_groups():
    pool = ops.Pages(*(random((200, 2, 32, 64), i).cuda() for i in range(2)))
    shapes = [([(300, [(1, 40)] * 4), (64, [(2, 9)] * 4)], 0), ([(64, [(1, 3)] * 3), (500, [(1, 200), (4, 4), (1, 1), (2, 9), (1, 8)])], 0),
              ([(0, [(1, 100)] * 4), (640, [(2, 2)] * 4)], 0)]
    q = torch.zeros((12, 8, 64), dtype=torch.float16).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = ops.PageBatch(torch.zeros((8, 24), **i32), torch.zeros(9, **i32), torch.zeros(8, **i32), 4)
    prefix = ops.PagePrefix(torch.zeros(3, **i32), torch.zeros(8, **i32), 1 << 30)

    def fill(i):
        seqs = prefixes.Shared(shapes[i][0], 32, widest=24, seed=i, spare=0)
        batch.table.copy_(seqs.table.clamp(min=0))
        batch.starts.copy_(seqs.starts)
        batch.lengths.copy_(seqs.lengths)
        prefix.groups.copy_(torch.tensor(seqs.groups, dtype=torch.int32))
        prefix.shared.copy_(torch.tensor(seqs.shared, dtype=torch.int32) // 32 * 32)     # (whole pages, which are the same ones)
        q.copy_(random(q.shape, i))

    out, again = (torch.zeros((12, 512), dtype=torch.float16, device="cuda") for _ in range(2))
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.paged_attention(q, pool, batch, out=out, prefix=prefix)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_attention(q, pool, batch, out=out, prefix=prefix)
    for i in (1, 2, 0, 1):
        fill(i)
        graph.replay()
        torch.cuda.synchronize()
        rows = int(batch.starts[-1])
        ops.paged_attention(q, pool, batch, out=again, prefix=prefix)
        assert torch.equal(out[:rows], again[:rows])
        assert ((out[:rows] - ops.paged_attention(q, pool, batch)[:rows]).abs() <= 0.01).all()
