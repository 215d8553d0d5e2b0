"""The operators of a paged cache against float64 on the CPU (tests/paged.py): sizes at the edges of pages, tiles, fragments and parts."""
import math

import pytest
import torch

from ternaryllm_amd import ops

from tests import paged

pytestmark = pytest.mark.gpu


def frequencies(pairs, theta=10000.0):
    return theta ** (-torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))


def random(shape, seed, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def fresh_pages(seqs, kv, hd, kind, seed=0, spoiled=True):
    """Pages on the CPU of random rows; where no sequence has a row, values that are not finite."""
    shape = (seqs.pages, kv, seqs.page_size, hd)
    k, v = random(shape, seed + 1), random(shape, seed + 2)
    ke = ve = None
    if kind == "e4m3":
        k, v = ((100 * t.float()).clamp(-448, 448).to(torch.float8_e4m3fn) for t in (k, v))
        ke, ve = (torch.randint(118, 123, shape[:3], generator=torch.Generator().manual_seed(seed + i), dtype=torch.uint8) for i in (3, 4))
    if spoiled:
        used = torch.zeros(shape[0], shape[2], dtype=torch.bool)
        for b, (_, length) in enumerate(seqs.both):
            for j in range(length):
                used[int(seqs.table[b, j // seqs.page_size]), j % seqs.page_size] = True
        for t, bad in ((k, math.nan), (v, math.inf if kind != "e4m3" else math.nan)):
            where = (~used)[:, None, :, None].expand(shape)
            if kind == "e4m3":
                t.view(torch.uint8)[where] = 0x7f
            else:
                t[where] = bad
    return ops.Pages(k, v, ke, ve)


def on_gpu(pages):
    return ops.Pages(*(None if t is None else t.cuda() for t in pages))


# ---------------------------------------------------------------- rotated heads
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,hd,pairs,norm", [
    (1, 1, 1, 8, 4, True), (1, 32, 32, 128, 64, False), (3, 5, 1, 64, 32, True), (7, 12, 4, 96, 20, True), (5, 3, 3, 80, 5, False), (2, 64, 8, 128, 64, True),
    (2, 2, 1, 256, 1, True), (2, 3, 2, 512, 256, True), (3, 2, 2, 192, 0, True), (65, 9, 3, 128, 31, True)])
def test_rope_heads(dtype, interleaved, tokens, heads, kv, hd, pairs, norm):
    qkv = random((tokens, heads + 2 * kv, hd), tokens * hd + pairs, dtype)
    q, k = qkv[:, :heads], qkv[:, heads:heads + kv]
    weights = [1 + 0.2 * random((hd,), 7 + i, torch.float32) for i in range(2)] if norm else [None, None]
    weights = [None if w is None else w.to(dtype) for w in weights]
    positions = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(pairs))
    positions[0] = 0 if tokens == 1 else 1048575
    f, factor, eps = frequencies(pairs), 1.25, 1e-5
    dev = qkv.cuda()
    dq, dk = dev[:, :heads], dev[:, heads:heads + kv]
    on = [None if w is None else w.cuda() for w in weights]
    how = dict(factor=factor, interleaved=interleaved, q_norm=on[0], k_norm=on[1], eps=eps)
    got = ops.rope_heads(dq, dk, positions.cuda(), f.cuda(), **how)
    for x, w, y in zip((q, k), weights, got):
        x = paged.normed(x, w, eps)
        want = paged.rotated(x, positions, f, interleaved, factor)
        assert y.dtype == dtype and y.is_contiguous()
        assert ((y.cpu().double() - want).abs() <= paged.rope_bound(x, paged.partners(x, pairs, interleaved), max(1.0, factor), dtype, want)).all()
    # the same bits in place, and of one operand alone
    alone = ops.rope_heads(dq, None, positions.cuda(), f.cuda(), **how)
    assert alone[1] is None and torch.equal(alone[0], got[0])
    ops.rope_heads(dq, dk, positions.cuda(), f.cuda(), q_out=dq, k_out=dk, **how)
    assert torch.equal(dq, got[0]) and torch.equal(dk, got[1]) and torch.equal(dev[:, heads + kv:].cpu(), qkv[:, heads + kv:])


def test_rope_heads_without_tokens():
    q, k = ops.rope_heads(torch.zeros((0, 4, 64), device="cuda"), torch.zeros((0, 2, 64), device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"),
                          frequencies(32).cuda())
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_rope_heads_keeps_what_is_not_finite_in_its_own_head():
    q = torch.randn((3, 4, 64)).half()
    q[1, 2, 5], q[2, 0, 3] = math.nan, math.inf
    y, _ = ops.rope_heads(q.cuda(), None, torch.arange(3, device="cuda"), frequencies(32).cuda(), q_norm=torch.ones(64).half().cuda())
    bad = ~torch.isfinite(y.cpu())
    assert bad[1, 2].any() and bad[2, 0].any()
    bad[1, 2] = bad[2, 0] = False
    assert not bad.any()


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_norms_of_fp32_heads_of_any_magnitude(hd, eps):
    """Squares that overflow or vanish in fp32 are no reason for a head of finite values not to be normalised.  Heads of every magnitude side by side in a wave."""
    sizes = [3e37, 1e25, 2e18, 1.0, 1e-12, 1e-19, 1e-25, 1e-38]
    x = random((3, len(sizes), hd), hd, torch.float32).clamp(-5, 5) * torch.tensor(sizes)[:, None]
    w = 1 + 0.2 * random((hd,), 5, torch.float32)
    f, at = frequencies(hd // 2), torch.tensor([0, 17, 900000])
    want = paged.normed(x, w, eps)
    bound = paged.rope_bound(want, paged.partners(want, hd // 2, False), 1.0, torch.float32, want)
    got, _ = ops.rope_heads(x.cuda(), None, at.cuda(), f.cuda(), q_norm=w.cuda(), eps=eps)
    assert ((got.cpu().double() - paged.rotated(want, at, f, False, 1.0)).abs() <= bound).all()
    # and on the way into pages, of which they are the keys
    seqs = paged.Sequences([(3, 3)], 16)
    pages = on_gpu(fresh_pages(seqs, len(sizes), hd, "float16", spoiled=False))
    ops.rope_to_pages(None, x.cuda(), torch.zeros_like(x).cuda(), pages, seqs.batch(ops), k_norm=w.cuda(), eps=eps)
    keys = ops.read_pages(pages, seqs.batch(ops), 3)[0].cpu().double()
    assert ((keys - want).abs() <= bound + 2.0 ** -11 * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_norms_of_heads_with_an_infinity(dtype):
    """Its root is infinite: what is finite beside it becomes 0, itself NaN."""
    x = random((2, 3, 64), 3, dtype)
    x[0, 1, 7], x[1, 2, 40] = math.inf, -math.inf
    got = ops.rope_heads(x.cuda(), None, None, None, q_norm=torch.ones(64).to(dtype).cuda())[0].cpu()
    want = paged.normed(x, torch.ones(64), 1e-6)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(got).sum()) == 2
    for row in (got[0, 1], got[1, 2]):
        assert (row[~torch.isnan(row)] == 0).all()


# ---------------------------------------------------------------- into pages and back
BATCHES = [
    ([(1, 1)], 16), ([(1, 17)], 16), ([(3, 3), (0, 5), (1, 40), (16, 16), (17, 33)], 16), ([(2, 130), (0, 0), (5, 64)], 64), ([(40, 40), (1, 257)], 256),
    ([(5, 3), (2, 2)], 32)]  # (the last: more rows than tokens)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("both,page", BATCHES)
@pytest.mark.parametrize("heads,kv,hd,pairs,interleaved,norm", [(4, 2, 128, 64, False, True), (3, 3, 64, 32, True, False), (2, 1, 256, 24, False, True), (1, 1, 80, 3, False, False)])
def test_rope_to_pages_and_back(dtype, kind, both, page, heads, kv, hd, pairs, interleaved, norm):
    seqs = paged.Sequences(both, page, front=2, behind=3, seed=len(both))
    q, k, v = random((seqs.tokens, heads + 2 * kv, hd), hd + page, dtype).split((heads, kv, kv), dim=1)
    v = (v * torch.exp2(torch.arange(seqs.tokens)[:, None, None] % 9 - 4.0)).to(dtype)
    weight = (1 + 0.2 * random((hd,), 5, torch.float32)).to(dtype) if norm else None
    f = frequencies(pairs)
    pages = on_gpu(fresh_pages(seqs, kv, hd, kind, seed=3, spoiled=False))
    before = ops.Pages(*(None if t is None else t.clone() for t in pages))
    q_out = torch.full((seqs.tokens, heads, hd), 7.0, dtype=dtype, device="cuda")
    on = None if weight is None else weight.cuda()
    how = dict(interleaved=interleaved, q_norm=on, k_norm=on)
    batch = seqs.batch(ops)
    got = ops.rope_to_pages(q.cuda(), k.cuda(), v.cuda(), pages, batch, f.cuda(), q_out=q_out, **how)
    assert got is q_out
    positions = torch.zeros(seqs.tokens, dtype=torch.int64)
    inside = torch.zeros(seqs.tokens, dtype=torch.bool)
    for b, (n, length) in enumerate(both):
        first = int(seqs.starts[b])
        positions[first:first + n] = torch.arange(length - n, length)
        inside[first:first + n] = True
    xq, xk = (paged.normed(t, weight, 1e-6) for t in (q, k))
    want_q, want_k = (paged.rotated(t, positions, f, interleaved, 1.0) for t in (xq, xk))
    q_bound = paged.rope_bound(xq, paged.partners(xq, pairs, interleaved), 1.0, dtype, want_q)
    assert ((q_out.cpu().double() - want_q).abs() <= q_bound)[inside].all() and (q_out[~inside.cuda()] == 7).all()
    # what the pages hold: the rows that have a place, and everything else as it was
    held = paged.values(pages.k.cpu(), None if pages.k_exponents is None else pages.k_exponents.cpu()), \
        paged.values(pages.v.cpu(), None if pages.v_exponents is None else pages.v_exponents.cpu())
    slack = paged.rope_bound(xk, paged.partners(xk, pairs, interleaved), 1.0, torch.float32, want_k)
    touched = torch.zeros((seqs.pages, page), dtype=torch.bool)
    for row, b, at, number, slot in seqs.rows():
        touched[number, slot] = True
        if kind == "float16":
            assert ((held[0][number, :, slot] - want_k[row]).abs() <= slack[row] + 2.0 ** -11 * want_k[row].abs()).all()
            assert torch.equal(held[1][number, :, slot], v[row].half().double())
        else:
            # a value is off by half a step of three bits, or of the row's smallest: 2^-4 of it, 2^-10 of the power of two
            grain = 2.0 ** (paged.exponents_of(want_k[row])[:, None] - 10)
            assert ((held[0][number, :, slot] - want_k[row]).abs() <= torch.maximum(want_k[row].abs() * 2.0 ** -4, 2 * grain) + slack[row]).all()
            assert torch.equal(held[1][number, :, slot], paged.byte_values(v[row].double()))
    for now, then in zip(pages, before):
        if now is not None:
            now, then = (t.cpu().view(torch.uint8).transpose(1, 2) for t in (now, then))
            assert torch.equal(now[~touched], then[~touched])
    # and read back, into new tensors and into a cache of another layout
    for out in (torch.float16, torch.float32):
        back = [torch.full((kv, seqs.tokens, hd), 5.0, dtype=out, device="cuda").transpose(0, 1) for _ in range(2)]
        ops.read_pages(pages, batch, seqs.tokens, k_out=back[0], v_out=back[1])
        fresh = ops.read_pages(pages, batch, seqs.tokens, out)
        rows = {row for row, *_ in seqs.rows()}
        for row in range(seqs.tokens):
            if not inside[row]:
                assert (back[0][row] == 5).all() and (back[1][row] == 5).all()
            elif row not in rows:
                assert torch.isnan(back[0][row]).all() and torch.isnan(back[1][row]).all()
        for row, b, at, number, slot in seqs.rows():
            for t, n, h in zip(back, fresh, held):
                assert torch.equal(t[row].cpu(), h[number, :, slot].to(out)) and torch.equal(n[row], t[row])


@pytest.mark.parametrize("positions", [None, "given"])
def test_rope_to_pages_without_queries_and_with_positions(positions):
    seqs = paged.Sequences([(4, 9)], 16)
    k, v = random((4, 2, 64), 1), random((4, 2, 64), 2)
    where = None if positions is None else torch.tensor([5, 900000, 0, 17])
    pages = on_gpu(fresh_pages(seqs, 2, 64, "float16", spoiled=False))
    assert ops.rope_to_pages(None, k.cuda(), v.cuda(), pages, seqs.batch(ops), frequencies(32).cuda(), None if where is None else where.cuda()) is None
    at = torch.arange(5, 9) if where is None else where
    alone, _ = ops.rope_heads(k.cuda(), None, at.cuda(), frequencies(32).cuda())
    back = ops.read_pages(pages, seqs.batch(ops), 4)
    assert torch.equal(back[0], alone) and torch.equal(back[1].cpu(), v)


def test_bytes_at_the_ends_of_their_range():
    """Rows of zeros, of the smallest and largest numbers, of infinities and NaN."""
    rows = torch.zeros((9, 1, 64), dtype=torch.float32)
    rows[1, 0, 3] = 1e-30
    rows[2] = torch.linspace(-65504, 65504, 64)
    rows[3, 0, :3] = torch.tensor([math.inf, -math.inf, 1.0])
    rows[4, 0, :2] = torch.tensor([math.nan, 3.0])
    rows[5, 0, :4] = torch.tensor([448.0, 447.0, -8.5, 0.0146484375])
    rows[6, 0, :2] = torch.tensor([448.0001, 1.0])
    rows[7] = 6e-8
    rows[8, 0, :2] = torch.tensor([3e38, -70000.0])
    seqs = paged.Sequences([(9, 9)], 16)
    pages = on_gpu(fresh_pages(seqs, 1, 64, "e4m3", spoiled=False))
    ops.rope_to_pages(None, rows.cuda(), rows.cuda(), pages, seqs.batch(ops))
    want = paged.byte_values(rows.double())
    for got in ops.read_pages(pages, seqs.batch(ops), 9, torch.float32):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=-1.0), torch.nan_to_num(want, nan=-1.0))
        assert torch.isfinite(got[:4]).all() and torch.isnan(got[4, 0, 0]) and got[4, 0, 1] == 3
    for got in ops.read_pages(pages, seqs.batch(ops), 9):   # every value is a finite fp16 number
        assert torch.isfinite(got[[0, 1, 2, 3, 5, 6, 7, 8]]).all()


# ---------------------------------------------------------------- attention
def attention_bound(q, k, v, want, longest, scale):
    """Probabilities are rounded to 11 bits (2^-11 of the largest value, and 2^-25 a key below fp16's normal range), the result once more; a score
    is a sum of head_dim exact products in fp32, off by head_dim * 2^-24 of the largest sum of magnitudes, which the softmax takes twice; the
    exponentials, their sum and the rescaling of sums have a few steps of fp32 each."""
    k, v = (torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0) for t in (k, v))
    score = 2 * scale * q.shape[-1] * 2.0 ** -24 * (q.double().norm(dim=-1).max() * k.norm(dim=-1).max())
    return (2.0 ** -11 + longest * 2.0 ** -25 + score + 64 * 2.0 ** -24) * v.abs().max() + 2.0 ** -11 * want.abs() + 2.0 ** -25


def check_attention(both, heads, kv, hd, page, kind, *, front=0, behind=0, most=None, scale=None, seed=1, widest=None):
    seqs = paged.Sequences(both, page, front=front, behind=behind, seed=seed, widest=widest)
    pages = fresh_pages(seqs, kv, hd, kind, seed=seed)
    q = random((seqs.tokens, heads + 3, hd), seed + 9)[:, 1:1 + heads]
    out = torch.full((seqs.tokens, heads * hd), 3.0, dtype=torch.float16, device="cuda")
    wide = random((seqs.tokens, heads + 3, hd), seed + 9).cuda()
    ops.paged_attention(wide[:, 1:1 + heads], on_gpu(pages), seqs.batch(ops, most=most), scale=scale, out=out)
    got = out.cpu().view(seqs.tokens, heads, hd)
    s = 1 / math.sqrt(hd) if scale is None else scale
    k, v = paged.values(pages.k, pages.k_exponents), paged.values(pages.v, pages.v_exponents)
    want = paged.attention(q, k, v, seqs, s)
    inside = torch.zeros(seqs.tokens, dtype=torch.bool)
    inside[front:seqs.tokens - behind if behind else None] = True
    assert (got[~inside] == 3).all()
    bound = attention_bound(q, k, v, want, max(length for _, length in both), s)
    assert ((got.double() - want).abs() <= bound)[inside].all()


SHAPES = [(1, 1, 128), (8, 2, 128), (14, 2, 64), (4, 4, 256), (3, 1, 64), (40, 2, 128), (5, 5, 64)]


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("both,page", [
    ([(1, 1)], 16), ([(1, 15), (1, 16), (1, 17)], 16), ([(1, 700), (1, 63), (1, 64), (1, 65), (0, 30), (1, 1)], 32), ([(1, 1300)], 256)])
def test_one_row_of_each_sequence(kind, heads, kv, hd, both, page):
    check_attention(both, heads, kv, hd, page, kind)


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("both,page", [
    ([(2, 2)], 16), ([(5, 130), (16, 16), (0, 0), (1, 90), (17, 63)], 16), ([(64, 64), (65, 400)], 64), ([(130, 131), (1, 257), (3, 3)], 128)])
def test_chunks(kind, heads, kv, hd, both, page):
    check_attention(both, heads, kv, hd, page, kind, front=1, behind=2)


# 128 rows to a workgroup: a table with room for 64 K tokens, and rows enough for the host to expect as much work
@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd,page", [(16, 2, 128, 256), (14, 2, 64, 256), (16, 16, 128, 64), (32, 1, 64, 16)])
def test_tall_workgroups(kind, heads, kv, hd, page):
    check_attention([(130, 131), (1, 257), (0, 5), (129, 400), (9, 5)], heads, kv, hd, page, kind, front=1, behind=1, widest=65536 // page)


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_that_see_nothing(kind, hd):
    """More rows than tokens: the first see nothing and are 0."""
    check_attention([(5, 2), (3, 0), (70, 66), (2, 2)], 2, 1, hd, 16, kind)


@pytest.mark.parametrize("heads,kv,hd", [(8, 2, 128), (2, 2, 64), (4, 1, 256)])
def test_a_long_sequence_is_shared_out(heads, kv, hd):
    check_attention([(1, 9000), (1, 100), (3, 5000)], heads, kv, hd, 64, "float16")


def test_many_sequences():
    both = [(i % 3, (i * 37) % 90 + 2) for i in range(1500)]
    check_attention(both, 2, 1, 64, 16, "float16")


@pytest.mark.parametrize("most", [0, 1, 3, 100])
def test_the_hint_changes_no_result(most):
    check_attention([(3, 200), (1, 80), (40, 300)], 8, 2, 128, 16, "float16", most=most)


def test_scale():
    check_attention([(3, 200), (1, 80)], 8, 2, 128, 16, "float16", scale=0.3)
    check_attention([(3, 200), (1, 80)], 8, 2, 128, 16, "e4m3", scale=1e-3)


@pytest.mark.parametrize("most", [1, 70])
def test_pages_and_lengths_that_are_none(most):
    """A page number out of range, or a length that the table does not hold: the sequence is NaN, nothing else is touched."""
    seqs = paged.Sequences([(1, 300), (1, 40), (2, 300)], 16)
    pages = on_gpu(fresh_pages(seqs, 2, 64, "float16"))
    q = random((4, 4, 64), 3).cuda()
    good = ops.paged_attention(q, pages, seqs.batch(ops, most=most))
    for number in (-1, seqs.pages, 1 << 30):
        batch = seqs.batch(ops, most=most)
        batch.table[2, 11] = number
        got = ops.paged_attention(q, pages, batch)
        assert torch.equal(got[:2], good[:2]) and torch.isnan(got[2:]).all()
        k, v = random((4, 2, 64), 5).cuda(), random((4, 2, 64), 6).cuda()
        then = [t.clone() for t in pages[:2]]
        batch.table[2, 18] = number                 # the page of the sequence's last two rows
        ops.rope_to_pages(None, k, v, ops.Pages(*then), batch)
        kept = ops.read_pages(ops.Pages(*then), batch, 4)
        assert torch.equal(kept[0][:2], k[:2]) and torch.isnan(kept[0][2:]).all()
    batch = seqs.batch(ops, most=most)
    batch.lengths[2] = 19 * 16 + 1
    got = ops.paged_attention(q, pages, batch)
    assert torch.equal(got[:2], good[:2]) and torch.isnan(got[2:]).all()


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
def test_a_length_that_the_table_does_not_hold_is_no_length(kind):
    """Nothing of such a sequence is written or read, the rows whose pages the table does have neither; the others are as ever."""
    seqs = paged.Sequences([(3, 40), (9, 60), (2, 2)], 16)
    pages, batch = on_gpu(fresh_pages(seqs, 2, 64, kind, spoiled=False)), seqs.batch(ops)
    k, v = random((seqs.tokens, 2, 64), 5).cuda(), random((seqs.tokens, 2, 64), 6).cuda()
    good, want = ops.Pages(*(None if t is None else t.clone() for t in pages)), ops.Pages(*(None if t is None else t.clone() for t in pages))
    ops.rope_to_pages(None, k, v, want, batch)
    read = ops.read_pages(want, batch, seqs.tokens)
    batch.lengths[1] = batch.table.shape[1] * 16 + 1              # its rows are tokens 56 to 64: the table ends at 63
    ops.rope_to_pages(None, k, v, good, batch)
    written = {number for _, b, _, number, _ in seqs.rows() if b != 1}
    for now, then, done in zip(good, pages, want):
        if now is not None:
            for number in range(seqs.pages):
                expected = done if number in written else then
                assert torch.equal(now[number].view(torch.uint8), expected[number].view(torch.uint8)), number
    back = ops.read_pages(want, batch, seqs.tokens)
    for t, r in zip(back, read):
        assert torch.isnan(t[3:12]).all() and torch.equal(t[:3], r[:3]) and torch.equal(t[12:], r[12:])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("most", [1, 100])                        # 16 rows a workgroup, and 64
def test_values_that_are_not_finite_among_the_new_tokens(hd, most):
    """A key or a value that is not finite reaches the rows that see it and no others, of its sequence or of another."""
    seqs = paged.Sequences([(100, 200), (3, 90)], 16)
    for kind in ("float16", "e4m3"):
        pages = fresh_pages(seqs, 1, hd, kind, spoiled=False)
        held = [paged.values(*t) for t in zip(pages[:2], pages[2:])]
        q = random((seqs.tokens, 2, hd), 3)
        want = paged.attention(q, *held, seqs, 1 / math.sqrt(hd))
        bound = attention_bound(q, *held, want, 200, 1 / math.sqrt(hd))
        for which, token in ((0, 170), (1, 170), (1, 191), (1, 127), (1, 199), (1, 100), (0, 101)):
            now = list(t if t is None else t.clone() for t in pages)
            where = int(seqs.table[0, token // 16]), 0, token % 16, 5
            if kind == "e4m3":
                now[which].view(torch.uint8)[where] = 0x7f
            else:
                now[which][where] = math.nan if which == 0 else math.inf
            got = ops.paged_attention(q.cuda(), on_gpu(ops.Pages(*now)), seqs.batch(ops, most=most)).cpu().view(seqs.tokens, 2, hd)
            good = torch.ones(seqs.tokens, dtype=torch.bool)
            good[token - 100:100] = False                         # row i is token 100 + i
            assert ((got.double() - want).abs() <= bound)[good].all(), (kind, which, token)
            assert not torch.isfinite(got[token - 100:100]).all(-1).any(), (kind, which, token)


@pytest.mark.parametrize("both,heads,kv,hd", [([(1, 300), (1, 33)], 4, 2, 128), ([(20, 90), (3, 3)], 2, 1, 64), ([(20, 90)], 1, 1, 256)])
@pytest.mark.parametrize("low,high", [(-32, -16), (-24, -10), (-15, -15)])
def test_bytes_of_small_exponents(both, heads, kv, hd, low, high):
    """fp16 holds values of exponents under -15 to half of its 2^-24: so does what is read back in it, so do the attention's keys and values.  fp32 holds all."""
    seqs = paged.Sequences(both, 16, seed=4)
    pages = fresh_pages(seqs, kv, hd, "e4m3", seed=2, spoiled=False)
    ke, ve = (torch.randint(127 + low, 128 + high, pages.k.shape[:3], generator=torch.Generator().manual_seed(i), dtype=torch.uint8) for i in range(2))
    pages = pages._replace(k_exponents=ke, v_exponents=ve)
    k, v = paged.values(pages.k, ke), paged.values(pages.v, ve)
    device = on_gpu(pages)
    whole = paged.Sequences([(n, n) for _, n in both], 16, seed=4)
    assert torch.equal(whole.table, seqs.table)
    for dtype in (torch.float16, torch.float32):
        for t, held in zip(ops.read_pages(device, whole.batch(ops), whole.tokens, dtype), (k, v)):
            want = torch.cat([whole.held(b, held) for b in range(len(both))])
            assert torch.equal(t.cpu(), want.to(dtype)) and (dtype == torch.float16 or torch.equal(t.cpu().double(), want))
    q = (2.0 ** -high * random((seqs.tokens, heads, hd), 9).float()).clamp(-60000, 60000).half()      # scores that tell keys apart
    scale = 1 / math.sqrt(hd) / 100
    got = ops.paged_attention(q.cuda(), device, seqs.batch(ops), scale=scale).cpu().double().view(q.shape)
    want = paged.attention(q, k, v, seqs, scale)
    bound = attention_bound(q, k, v, want, max(n for _, n in both), scale)
    bound = bound + 2.0 ** -25 + 2 * scale * 2.0 ** -25 * q.double().abs().sum(-1).max() * v.abs().max()   # of a value, and of a score's keys, twice
    assert ((got - want).abs() <= bound).all()


# so many query heads on a key head that a workgroup of 64, 128 or 16 rows has those of one token only
@pytest.mark.parametrize("heads,hd,most,widest", [(40, 64, 20, None), (40, 128, 20, None), (33, 256, 20, None), (80, 64, 20, 65536), (80, 128, 20, 65536), (16, 128, 1, None), (11, 64, 0, None),
                                                  (16, 256, 1, None)])
@pytest.mark.parametrize("kind", ["float16", "e4m3"])
def test_later_tokens_that_are_not_finite_beside_rows_of_one_token(heads, hd, most, widest, kind):
    """The chunk's later tokens share the last tile of an earlier row, and weigh nothing in it, whatever they hold."""
    seqs = paged.Sequences([(20, 100), (7, 7)], 16, widest=None if widest is None else widest // 16)
    pages = fresh_pages(seqs, 1, hd, kind, spoiled=False)
    held = [paged.values(*t) for t in zip(pages[:2], pages[2:])]
    q = random((seqs.tokens, heads, hd), 3)
    want = paged.attention(q, *held, seqs, 1 / math.sqrt(hd))
    bound = attention_bound(q, *held, want, 100, 1 / math.sqrt(hd))
    for which, token in ((1, 90), (1, 99), (0, 85), (1, 97)):
        now = list(t if t is None else t.clone() for t in pages)
        where = int(seqs.table[0, token // 16]), 0, token % 16, 5
        if kind == "e4m3":
            now[which].view(torch.uint8)[where] = 0x7f
        else:
            now[which][where] = math.nan if which == 0 else math.inf
        got = ops.paged_attention(q.cuda(), on_gpu(ops.Pages(*now)), seqs.batch(ops, most=most)).cpu().view(seqs.tokens, heads, hd)
        good = torch.ones(seqs.tokens, dtype=torch.bool)
        good[token - 80:20] = False                               # row i is token 80 + i
        assert ((got.double() - want).abs() <= bound)[good].all(), (which, token)
        assert not torch.isfinite(got[token - 80:20]).all(-1).any(), (which, token)


def test_no_sequences_and_no_rows():
    pages = ops.Pages(*(torch.zeros((2, 1, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2)))
    i32 = dict(dtype=torch.int32, device="cuda")
    none = ops.PageBatch(torch.zeros((0, 1), **i32), torch.zeros(1, **i32), torch.zeros(0, **i32), 0)
    assert ops.paged_attention(torch.zeros((0, 1, 64), dtype=torch.float16, device="cuda"), pages, none).shape == (0, 64)
    out = torch.full((2, 64), 3.0, dtype=torch.float16, device="cuda")
    ops.paged_attention(torch.zeros((2, 1, 64), dtype=torch.float16, device="cuda"), pages, none, out=out)
    empty = ops.PageBatch(torch.zeros((3, 1), **i32), torch.zeros(4, **i32), torch.zeros(3, **i32), 0)
    ops.paged_attention(torch.zeros((2, 1, 64), dtype=torch.float16, device="cuda"), pages, empty, out=out)
    assert (out == 3).all()


def test_a_peak_over_a_long_plain():
    """One key above 60000 that are alike, each with 1.7e-5 of its weight, below fp16's normal range, and all of them together with as much."""
    n = 60001
    seqs = paged.Sequences([(1, n)], 256)
    for kind in ("float16", "e4m3"):
        pages = fresh_pages(seqs, 1, 64, kind, spoiled=False)
        k = torch.zeros(pages.k.shape)
        k[int(seqs.table[0, 100]), 0, 7, 0] = 11.0
        v = torch.ones(pages.v.shape)
        v[int(seqs.table[0, 100]), 0, 7] = 3.0
        ke = None if kind == "float16" else torch.full(pages.k.shape[:3], 127, dtype=torch.uint8)
        dtype = torch.float16 if kind == "float16" else torch.float8_e4m3fn
        q = torch.zeros((1, 1, 64), dtype=torch.float16)
        q[0, 0, 0] = 8.0                                          # a score of 11, and 0
        got = ops.paged_attention(q.cuda(), on_gpu(ops.Pages(k.to(dtype), v.to(dtype), ke, ke)), seqs.batch(ops)).cpu().double()
        weight = 1 / (1 + (n - 1) * math.exp(-11))
        # the plain's probabilities are rounded to fp16's smallest step, 2^-24, in the sums above and below the line alike: 2^-25 of 1.67e-5 each
        slack = 2.0 ** -25 / math.exp(-11) + 2.0 ** -10
        assert (got - (3 * weight + 1 - weight)).abs().max() <= 3 * slack


@pytest.mark.parametrize("depth", [14.0, 17.5, 18.5])
@pytest.mark.parametrize("rows,most,hd,widest", [(1, 1, 64, None), (3, 40, 64, None), (2, 40, 256, None), (3, 140, 64, 1 << 22)])   # of 16, 64 and 128 rows a workgroup
def test_a_plain_far_below_its_peaks_keeps_its_weight(rows, most, hd, widest, depth):
    """Four keys `depth` above 2^20 others that are alike, over which one workgroup goes alone (of so many sequences that each has one; all have the same pages).
    fp16's lower end takes 2^-25 a key where the largest probability is 2^7 at least, of a row that weighs that or more.  The sums are fp32 and lose by additions of
    little to much, half a step (2^-24) each: a lane's sum takes 8 keys at a time of its sixteenth of them all (16 rows), or 16 of its quarter; sums of values take 32
    a time, of which the instruction may cut off a whole step (2^-23), of a quarter of the keys or of all.  Twice each, as values reach 2.  Beside it the
    result's rounding."""
    n, page, seqs = 1 << 20, 1024, 520
    k, v = (torch.zeros((n // page, 1, page, hd), dtype=torch.float16, device="cuda") for _ in range(2))
    v.fill_(1.0)
    k[0, 0, 5:128:32, 0], v[0, 0, 5:128:32] = depth, -2.0         # (every wave has one)
    i32 = dict(dtype=torch.int32, device="cuda")
    table = torch.arange(n // page, **i32)[None].repeat(seqs, 1)
    if widest is not None:
        table = torch.cat([table, torch.zeros((seqs, (widest - n) // page), **i32)], 1)
    batch = ops.PageBatch(table, rows * torch.arange(seqs + 1, **i32), torch.full((seqs,), n, **i32), most)
    q = torch.zeros((rows * seqs, 1, hd), dtype=torch.float16, device="cuda")
    q[..., 0] = 8.0                                               # scores of `depth`, and 0
    got = ops.paged_attention(q, ops.Pages(k, v), batch, scale=0.125).cpu().double().view(seqs, rows, hd)
    plain = (n - rows + 1 - 4 + torch.arange(rows, dtype=torch.float64)) * math.exp(-depth)
    want = ((plain - 8.0) / (plain + 4.0))[None, :, None]
    sums = n / 16 / 8 * 2.0 ** -24 + n / 4 / 32 * 2.0 ** -23 if most == 1 else n / 4 / 16 * 2.0 ** -24 + n / 32 * 2.0 ** -23
    slack = 3 * n * 2.0 ** -32 + 2 * sums + 2.0 ** -11 * want.abs() + 2.0 ** -16
    assert ((got - want).abs() <= slack).all(), (got[0, :, 0], want[0, :, 0])


# 16, 64 and 128 rows to a workgroup, and one sequence cut into pieces
LARGE_SCORES = [([(1, 90), (1, 33)], 4, 2, 128, None), ([(20, 90), (1, 33)], 4, 2, 64, None), ([(40, 130), (3, 3)], 16, 1, 128, 65536), ([(2, 7000)], 2, 1, 64, None),
                ([(70, 4000)], 2, 1, 256, None)]


@pytest.mark.parametrize("both,heads,kv,hd,widest", LARGE_SCORES)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("kind", ["float16", "e4m3"])
def test_scores_as_large_as_they_get(both, heads, kv, hd, widest, sign, kind):
    """Finite queries and keys whose scores reach 2^31 and more.  Every score is one product, the two largest keys of three have the same, the third is below
    by far more than a softmax sees: a row is the mean of the values of the two that it sees, up to its rounding and a few of fp32."""
    seqs = paged.Sequences(both, 16, seed=2, widest=None if widest is None else widest // 16)
    pages = fresh_pages(seqs, kv, hd, kind, seed=5, spoiled=False)
    for c, scale in ((30000.0, 1.0), (57344.0, 1.0), (41000.0, 0.37), (33333.0, 2.5), (9000.0, 0.125), (60000.0, 1e6)):
        keys = torch.zeros(pages.k.shape)
        keys[..., 0] = sign * 57344.0
        where = torch.arange(keys[..., 0].numel()).view(keys.shape[:3]) % 3 == 0   # (in the order of the pages: somewhere in each sequence)
        keys[..., 0][where] = 53248.0 if sign == 1 else -61440.0
        if kind == "e4m3":
            now = pages._replace(k=(keys / 256).to(torch.float8_e4m3fn), k_exponents=torch.full(keys.shape[:3], 127 + 8, dtype=torch.uint8))
        else:
            now = pages._replace(k=keys.half())
        q = torch.zeros((seqs.tokens, heads, hd), dtype=torch.float16)
        q[..., 0] = c
        got = ops.paged_attention(q.cuda(), on_gpu(now), seqs.batch(ops), scale=scale).cpu().double().view(q.shape)
        held = [paged.values(*t) for t in zip(now[:2], now[2:])]
        assert torch.equal(held[0], keys.double())
        want = paged.attention(q, *held, seqs, scale)
        assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -16 * held[1].abs().max()).all(), (c, scale)


@pytest.mark.parametrize("both,heads,kv,hd,widest", LARGE_SCORES)
@pytest.mark.parametrize("height", [2.0 ** 10, 2.0 ** 11, 3000.0, 2.0 ** 12, -2.0 ** 12, 2.0 ** 14, 2.0 ** 17, -2.0 ** 17])
def test_small_differences_of_large_scores(both, heads, kv, hd, widest, height):
    """Scores of `height` and up to 10 more, in steps of a half that fp32 holds exactly, growing along the sequence.  Beside the bound of any scores, references
    below 4096 are rounded by 2^-12 as exponents of 2, once in each of two sums that meet."""
    seqs = paged.Sequences(both, 16, seed=2, widest=None if widest is None else widest // 16)
    pages = fresh_pages(seqs, kv, hd, "float16", seed=5, spoiled=False)
    k = torch.zeros(pages.k.shape)
    k[..., 0] = height / 16
    for b, (_, length) in enumerate(both):
        for j in range(length):
            k[int(seqs.table[b, j // 16]), :, j % 16, 1] = 0.5 * (20 * j // length)
    q = torch.zeros((seqs.tokens, heads, hd), dtype=torch.float16)
    q[..., 0], q[..., 1] = 16.0, 1.0
    now = pages._replace(k=k.half())
    assert torch.equal(now.k.float(), k)
    got = ops.paged_attention(q.cuda(), on_gpu(now), seqs.batch(ops), scale=1.0).cpu().double().view(q.shape)
    want = paged.attention(q, now.k.double(), now.v.double(), seqs, 1.0)
    zero = torch.zeros((1, 1))
    bound = attention_bound(zero, zero, now.v.double(), want, max(length for _, length in both), 1.0)   # (of scores that are exact)
    assert ((got - want).abs() <= bound + 2 * 2.0 ** -12 * now.v.double().abs().max()).all()


@pytest.mark.parametrize("kind", ["float16", "e4m3"])
@pytest.mark.parametrize("most", [1, 200])
def test_pages_of_other_strides(kind, most):
    """Slots before heads, and keys and values of a layer in one tensor."""
    seqs = paged.Sequences([(2, 70), (1, 33), (3, 150)], 32)
    pages = fresh_pages(seqs, 2, 128, kind)
    q = random((seqs.tokens, 8, 128), 4).cuda()
    want = ops.paged_attention(q, on_gpu(pages), seqs.batch(ops, most=most))
    n, kv, page, hd = pages.k.shape
    raw = torch.uint8 if kind == "e4m3" else torch.float16
    both = torch.zeros((n, page, 2, kv, hd), dtype=raw, device="cuda")
    views = [both[:, :, i].transpose(1, 2).view(pages.k.dtype) if kind == "e4m3" else both[:, :, i].transpose(1, 2) for i in range(2)]
    for view, t in zip(views, (pages.k, pages.v)):
        view.view(raw).copy_(t.view(raw).cuda())
    other = ops.Pages(*views, *(None if t is None else t.cuda() for t in pages[2:]))
    assert torch.equal(ops.paged_attention(q, other, seqs.batch(ops, most=most)), want)
    k, v = random((seqs.tokens, 2, 128), 5).cuda(), random((seqs.tokens, 2, 128), 6).cuda()
    plain = on_gpu(pages)
    for p in (plain, other):
        ops.rope_to_pages(None, k, v, p, seqs.batch(ops))
    a, b = ops.read_pages(plain, seqs.batch(ops), seqs.tokens), ops.read_pages(other, seqs.batch(ops), seqs.tokens)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for view, t in zip(views, plain[:2]):
        bits = torch.uint8 if kind == "e4m3" else torch.int16   # (what no sequence has is not a number)
        assert torch.equal(view.view(bits), t.view(bits))


@pytest.mark.parametrize("most", [1, 200])
def test_pages_that_lie_far_apart(most):
    """Offsets past 32 bits: pages of 5 GB."""
    seqs = paged.Sequences([(1, 30), (2, 20)], 16, spare=0)
    pages = fresh_pages(seqs, 2, 64, "float16")
    step = (5 << 30) // 2
    pool = torch.empty(4 * step, dtype=torch.float16, device="cuda")
    far = ops.Pages(*(torch.as_strided(pool, pages.k.shape, (step, 16 * 64, 64, 1), i * 2 * 16 * 64) for i in range(2)))
    for view, t in zip(far, pages[:2]):
        view.copy_(t.cuda())
    q = random((3, 4, 64), 4).cuda()
    assert seqs.pages == 4 and torch.equal(ops.paged_attention(q, far, seqs.batch(ops, most=most)), ops.paged_attention(q, on_gpu(pages), seqs.batch(ops, most=most)))
    k, v = random((3, 2, 64), 5).cuda(), random((3, 2, 64), 6).cuda()
    ops.rope_to_pages(None, k, v, far, seqs.batch(ops))
    back = ops.read_pages(far, seqs.batch(ops), 3)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)


def test_more_rows_than_one_launch_takes():
    """A launch has fewer than 2^32 threads: 2^24 workgroups of 256."""
    n = (1 << 24) + 5
    q = torch.randn((n, 1, 16), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    f, at = frequencies(8).cuda(), torch.arange(n, device="cuda")
    got, _ = ops.rope_heads(q, None, at, f)
    edges = (0, 1, 1000, (1 << 23) - 3, (1 << 23) + 3, (1 << 24) - 2, n)
    for a, b in zip(edges, edges[1:]):
        assert torch.equal(ops.rope_heads(q[a:b], None, at[a:b], f)[0], got[a:b]), (a, b)
    # into pages: one sequence, its pages in reverse order; and more rows out of them, of a sequence four times as long
    count = -(-4 * n // 1024)
    i32 = dict(dtype=torch.int32, device="cuda")
    pages = ops.Pages(*(torch.zeros((count, 1, 1024, 16), dtype=torch.float16, device="cuda") for _ in range(2)))
    batch = ops.PageBatch(torch.arange(count - 1, -1, -1, **i32)[None], torch.tensor([0, n], **i32), torch.tensor([n], **i32), n)
    ops.rope_to_pages(None, q, q, pages, batch, f)
    held = [t.flip(0).reshape(-1, 1, 16) for t in pages[:2]]
    assert torch.equal(held[0][:n], got) and torch.equal(held[1][:n], q) and not held[0][n:].any() and not held[1][n:].any()
    m = 4 * n
    pages.v.copy_(torch.randn(pages.v.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(2), dtype=torch.float16))
    k, v = ops.read_pages(pages, batch._replace(starts=torch.tensor([0, m], **i32), lengths=torch.tensor([m], **i32)), m)
    assert torch.equal(k, held[0][:m]) and torch.equal(v, pages.v.flip(0).reshape(-1, 1, 16)[:m])


def test_two_streams_at_once():
    """Calls on two streams do not share what they work in: each gives the bits that it gives alone."""
    seqs = [paged.Sequences([(1, 3000 + 100 * i), (1, 500)], 64, seed=i) for i in range(2)]
    pages = [on_gpu(fresh_pages(s, 2, 128, "float16", seed=i)) for i, s in enumerate(seqs)]
    qs, batches = [random((2, 8, 128), i).cuda() for i in range(2)], [s.batch(ops) for s in seqs]
    alone = [ops.paged_attention(q, p, b) for q, p, b in zip(qs, pages, batches)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attention(qs[i], pages[i], batches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, alone[i]) for g in got[i])


def test_two_graphs_of_one_stream_replayed_on_two():
    seqs = paged.Sequences([(1, 4000), (1, 700)], 64)
    pages, batch = on_gpu(fresh_pages(seqs, 2, 128, "float16")), seqs.batch(ops)
    qs = [random((2, 8, 128), i).cuda() for i in range(2)]
    want = [ops.paged_attention(q, pages, batch) for q in qs]
    graphs, outs = [], []
    for q in qs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(ops.paged_attention(q, pages, batch))
    streams = [torch.cuda.Stream() for _ in qs]
    for turn in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want)), turn


def test_the_same_bits_every_time():
    both = [(1, (i * 997) % 4000 + 1) for i in range(40)]
    seqs = paged.Sequences(both, 16)
    pages, batch, q = on_gpu(fresh_pages(seqs, 2, 128, "float16")), seqs.batch(ops), random((40, 8, 128), 2).cuda()
    first = ops.paged_attention(q, pages, batch)
    assert all(torch.equal(ops.paged_attention(q, pages, batch), first) for _ in range(20))


class _NoShortWay:
    def __getattr__(self, name):
        return lambda *args: None


def test_the_short_way_and_the_general_one(monkeypatch):
    """The same bits, whichever of the two takes a call."""
    seqs = paged.Sequences([(2, 30), (1, 70), (5, 5)], 16)
    qkv = random((seqs.tokens, 8, 64), 1).cuda()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    w, f, at = random((64,), 2).cuda(), frequencies(32).cuda(), torch.arange(seqs.tokens, device="cuda")

    def all_of_them():
        got = []
        for kind in ("float16", "e4m3"):
            pages = on_gpu(fresh_pages(seqs, 2, 64, kind, spoiled=False))
            got += ops.rope_heads(q, k, at, f, q_norm=w, factor=1.5)
            got.append(ops.rope_to_pages(q, k, v, pages, seqs.batch(ops), f, interleaved=True, k_norm=w))
            got.append(ops.rope_to_pages(q, k, v, pages, seqs.batch(ops), f, at, k_norm=w))
            got += [t.view(torch.uint8) for t in pages if t is not None]
            got += ops.read_pages(pages, seqs.batch(ops), seqs.tokens) + ops.read_pages(pages, seqs.batch(ops), seqs.tokens, torch.float32)
            got.append(ops.paged_attention(q, pages, seqs.batch(ops)))
            got.append(ops.paged_attention(q, pages, seqs.batch(ops), scale=0.5, out=torch.empty((seqs.tokens, 256), dtype=torch.float16, device="cuda")))
        return got

    short = all_of_them()
    monkeypatch.setattr(ops, "_short", _NoShortWay)
    general = all_of_them()
    assert len(short) == len(general) and all(torch.equal(a, b) for a, b in zip(short, general))


def test_no_derivative_is_lost_on_the_short_way():
    from tests.test_paged_cpu import check_no_derivative_is_lost, parts
    q, k, pages, batch = parts()
    to = lambda t: None if t is None else t.cuda()
    check_no_derivative_is_lost(q.cuda(), k.cuda(), ops.Pages(*map(to, pages)), ops.PageBatch(*map(to, batch[:3]), 1), torch.zeros(3, dtype=torch.int64).cuda(),
                                torch.ones(32, dtype=torch.float64).cuda(), torch.ones(64).half().cuda())
