"""What the operators of a paged cache refuse, without a GPU: the tensor-level checks, and the library's own in front of a launch."""
import ctypes
import math

import pytest
import torch

from tests import paged
from ternaryllm_amd import _lib, ops


def parts(kind="float16", kv=2, page=16, hd=64, seqs=2, tokens=3, heads=4):
    dtype = torch.float16 if kind == "float16" else torch.float8_e4m3fn
    k, v = (torch.zeros((5, kv, page, hd)).to(dtype) for _ in range(2))
    exps = (None, None) if kind == "float16" else (torch.zeros((5, kv, page), dtype=torch.uint8), torch.zeros((5, kv, page), dtype=torch.uint8))
    batch = ops.PageBatch(torch.zeros((seqs, 2), dtype=torch.int32), torch.zeros(seqs + 1, dtype=torch.int32), torch.zeros(seqs, dtype=torch.int32), 1)
    return torch.zeros((tokens, heads, hd), dtype=torch.float16), torch.zeros((tokens, kv, hd), dtype=torch.float16), ops.Pages(k, v, *exps), batch


def test_nothing_runs_without_a_gpu():
    q, k, pages, batch = parts()
    with pytest.raises(RuntimeError):
        ops.rope_heads(q, k, torch.zeros(3, dtype=torch.int64), torch.ones(32, dtype=torch.float64))
    with pytest.raises(RuntimeError):
        ops.rope_to_pages(q, k, k, pages, batch)
    with pytest.raises(RuntimeError):
        ops.read_pages(pages, batch, 3)
    with pytest.raises(RuntimeError):
        ops.paged_attention(q, pages, batch)


@pytest.mark.parametrize("change", [
    lambda p: p._replace(v=p.v[:4]), lambda p: p._replace(v=p.v.float()), lambda p: p._replace(k=p.k.float(), v=p.v.float()),
    lambda p: p._replace(k_exponents=torch.zeros((5, 2, 16), dtype=torch.uint8)), lambda p: p._replace(v=p.v.transpose(1, 2).contiguous().transpose(1, 2)),
    lambda p: p._replace(k=p.k[0], v=p.v[0]), lambda p: p._replace(k=p.k.to(torch.float8_e4m3fn), v=p.v.to(torch.float8_e4m3fn))])
def test_pages_that_are_none(change):
    q, k, pages, batch = parts()
    with pytest.raises(ValueError):
        ops.paged_attention(q, change(pages), batch)
    with pytest.raises(ValueError):
        ops.read_pages(change(pages), batch, 3)
    with pytest.raises(ValueError):
        ops.rope_to_pages(q, k, k, change(pages), batch)


@pytest.mark.parametrize("change", [
    lambda p: p._replace(k_exponents=None), lambda p: p._replace(v_exponents=None), lambda p: p._replace(k_exponents=p.k_exponents[:4]),
    lambda p: p._replace(k_exponents=p.k_exponents.int()), lambda p: p._replace(v_exponents=p.v_exponents.transpose(1, 2).contiguous().transpose(1, 2))])
def test_exponents_that_are_none(change):
    q, _, pages, batch = parts("e4m3")
    with pytest.raises(ValueError):
        ops.paged_attention(q, change(pages), batch)


@pytest.mark.parametrize("change", [
    lambda b: b._replace(table=b.table.long()), lambda b: b._replace(starts=b.starts.long()), lambda b: b._replace(lengths=b.lengths.long()),
    lambda b: b._replace(starts=b.starts[:-1]), lambda b: b._replace(lengths=b.lengths[:-1]), lambda b: b._replace(table=b.table[0]),
    lambda b: b._replace(table=b.table.t().contiguous().t()), lambda b: b._replace(starts=torch.zeros(6, dtype=torch.int32)[::2])])
def test_batches_that_are_none(change):
    q, k, pages, batch = parts()
    with pytest.raises(ValueError):
        ops.paged_attention(q, pages, change(batch))
    with pytest.raises(ValueError):
        ops.rope_to_pages(q, k, k, pages, change(batch))


def test_heads_and_outputs_that_do_not_fit():
    q, k, pages, batch = parts()
    at, f = torch.zeros(3, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    bad = [
        lambda: ops.rope_heads(q[0], None, at, f), lambda: ops.rope_heads(q, k[:2], at, f), lambda: ops.rope_heads(q, k.float(), at, f),
        lambda: ops.rope_heads(q, k, None, f), lambda: ops.rope_heads(q, k, at.int(), f), lambda: ops.rope_heads(q, k, at[:2], f),
        lambda: ops.rope_heads(q, k, at, f.float()), lambda: ops.rope_heads(q, k, at, f[None]), lambda: ops.rope_heads(q.bfloat16(), None, at, f),
        lambda: ops.rope_heads(q, k, at, f, q_norm=torch.ones(64)), lambda: ops.rope_heads(q, k, at, f, k_norm=torch.ones(32).half()),
        lambda: ops.rope_heads(q, k, at, f, q_out=k), lambda: ops.rope_heads(q, k, at, f, q_out=q.float()),
        lambda: ops.rope_heads(q.transpose(1, 2), None, at, f), lambda: ops.rope_to_pages(q, k, k[:2], pages, batch),
        lambda: ops.rope_to_pages(q[:2], k, k, pages, batch), lambda: ops.rope_to_pages(q, k[:, :1], k[:, :1], pages, batch),
        lambda: ops.rope_to_pages(q, q, q, pages, batch), lambda: ops.read_pages(pages, batch, 3, torch.bfloat16),
        lambda: ops.read_pages(pages, batch, 3, k_out=k), lambda: ops.read_pages(pages, batch, 3, k_out=k, v_out=k.float()),
        lambda: ops.read_pages(pages, batch, 2, k_out=k, v_out=k.clone()), lambda: ops.paged_attention(q[..., :32], pages, batch),
        lambda: ops.paged_attention(q[0], pages, batch), lambda: ops.paged_attention(q, pages, batch, out=q), lambda: ops.paged_attention(q.bfloat16(), pages, batch),
        lambda: ops.paged_attention(q, pages, batch, out=torch.zeros((3, 256)))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_no_backward_pass():
    q, k, pages, batch = parts()
    at, f = torch.zeros(3, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    w = torch.ones(64).half().requires_grad_()
    for call in (lambda x: ops.rope_heads(x, k, at, f), lambda x: ops.rope_to_pages(None, x[:, :2], k, pages, batch), lambda x: ops.paged_attention(x, pages, batch),
                 lambda x: ops.rope_heads(q, k, at, f, k_norm=w)):
        with pytest.raises(RuntimeError, match="backward"):
            call(q.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
            call(q.clone().requires_grad_())


def derived_calls(q, k, pages, batch, at, f, w):
    """(operand, call of it) of every floating operand of every operator."""
    return [(q, lambda x: ops.rope_heads(x, k, at, f)), (k, lambda x: ops.rope_heads(q, x, at, f)), (f, lambda x: ops.rope_heads(q, k, at, x)),
            (w, lambda x: ops.rope_heads(q, k, at, f, q_norm=x)), (q, lambda x: ops.rope_heads(q, k, at, f, q_out=x)),
            (q, lambda x: ops.rope_to_pages(x, k, k, pages, batch, f)), (k, lambda x: ops.rope_to_pages(q, x, k, pages, batch, f)),
            (k, lambda x: ops.rope_to_pages(q, k, x, pages, batch, f)), (f, lambda x: ops.rope_to_pages(q, k, k, pages, batch, x)),
            (pages.k, lambda x: ops.rope_to_pages(q, k, k, pages._replace(k=x), batch, f)), (pages.v, lambda x: ops.rope_to_pages(q, k, k, pages._replace(v=x), batch)),
            (w, lambda x: ops.rope_to_pages(q, k, k, pages, batch, f, k_norm=x)), (pages.k, lambda x: ops.read_pages(pages._replace(k=x), batch, 3)),
            (pages.v, lambda x: ops.read_pages(pages._replace(v=x), batch, 3)), (k, lambda x: ops.read_pages(pages, batch, 3, k_out=x, v_out=k)),
            (q, lambda x: ops.paged_attention(x, pages, batch)), (pages.k, lambda x: ops.paged_attention(q, pages._replace(k=x), batch)),
            (pages.v, lambda x: ops.paged_attention(q, pages._replace(v=x), batch)), (q, lambda x: ops.paged_attention(q, pages, batch, out=x.view(3, -1)))]


def check_no_derivative_is_lost(q, k, pages, batch, at, f, w):
    from torch.autograd import forward_ad
    for i, (t, call) in enumerate(derived_calls(q, k, pages, batch, at, f, w)):
        with pytest.raises(RuntimeError, match="backward"):
            call(t.detach().clone().requires_grad_())
            pytest.fail(f"call {i} lost a gradient")
        with torch.no_grad(), forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangents"):
            call(forward_ad.make_dual(t.detach().clone(), torch.ones_like(t)))
            pytest.fail(f"call {i} lost a tangent")


def test_no_derivative_is_lost():
    q, k, pages, batch = parts()
    check_no_derivative_is_lost(q, k, pages, batch, torch.zeros(3, dtype=torch.int64), torch.ones(32, dtype=torch.float64), torch.ones(64).half())


def test_outputs_that_overlap_operands():
    at, f = torch.zeros(3, dtype=torch.int64), torch.ones(32, dtype=torch.float64)
    rows = torch.zeros((5, 6, 64), dtype=torch.float16)
    q, k = rows[:3, :4], rows[:3, 4:]
    for out in (rows[1:4, :4], rows[:3, 1:5], rows[:3, 2:]):
        with pytest.raises(ValueError):
            ops.rope_heads(q, k, at, f, q_out=out)
    with pytest.raises(ValueError):
        ops.rope_heads(q, k, at, f, q_out=q, k_out=q[:, 2:])
    # taken, up to the GPU that is not there: in place, and beside each other in other rows
    other = torch.zeros((3, 6, 64), dtype=torch.float16)
    for outs in ({"q_out": q, "k_out": k}, {"q_out": other[:, :4], "k_out": other[:, 4:]}):
        with pytest.raises(RuntimeError):
            ops.rope_heads(q, k, at, f, **outs)


def test_rows_read_back_lie_apart():
    _, _, pages, batch = parts()
    both = torch.zeros((6, 4, 64), dtype=torch.float16)
    for k, v in ((both[:3, :2], both[:3, :2]), (both[:3, :2], both[1:4, :2]), (both[:3, :2], both[:3, 1:3])):
        with pytest.raises(ValueError):
            ops.read_pages(pages, batch, 3, k_out=k, v_out=v)
    for k, v in ((both[:3, :2], both[3:, :2]), (both[:3, :2], both[:3, 2:])):
        with pytest.raises(RuntimeError):                         # taken, up to the GPU that is not there
            ops.read_pages(pages, batch, 3, k_out=k, v_out=v)


def test_rows_alike_overlap():
    """Against the places themselves, over layouts of every order."""
    pool = torch.arange(4000)
    taken = set()
    for token, head, offsets in ((64, 16, (0, 16, 48, 64, 8, 130)), (16, 64, (0, 16, 64, 48, 24)), (32, 80, (0, 16, 8, 96)), (16, 96, (0, 32, 48, 112)), (96, 32, (0, 16, 64, 80, 1))):
        for tokens, heads in ((3, 2), (1, 4), (4, 1), (2, 5), (1, 1)):
            x = pool.as_strided((tokens, heads, 16), (token, head, 1))
            for offset in offsets:
                y = pool.as_strided((tokens, heads, 16), (token, head, 1), offset)
                real = bool(set(x.flatten().tolist()) & set(y.flatten().tolist()))
                assert ops._alike_overlap(x, y) == ops._alike_overlap(y, x) == real, (token, head, tokens, heads, offset)
                taken.add(real)
    assert taken == {True, False}


class Raw:
    """The library's structures over addresses that are never followed: every call here is refused before a launch."""

    def __init__(self, **changes):
        at = 1 << 20
        self.pages = _lib.Pages(at, at, None, None, 2 * 16 * 64, 16 * 64, 64, 5, 16, 2, 64, _lib.TL_F16)
        self.batch = _lib.PageBatch(at, at, at, 2, 2, 2)
        self.q = _lib.HeadRows(at, 256, 64, at, 256, 64, None, 4)
        self.k = _lib.HeadRows(at, 128, 64, at, 128, 64, None, 2)
        self.v = _lib.HeadRows(at, 128, 64, None, 0, 0, None, 2)
        self.rotation = _lib.Rotation(at, at, 32, 0, 1.0, 1e-6)
        self.args = {"dtype": _lib.TL_F16, "tokens": 3, "head_dim": 64, "scale": 0.125, "out": at, "workspace": at, "bytes": 1 << 40, "heads": 4, "most": 1,
                     "q_token": 256, "k_out": at, "out_token": 128}
        for name, value in changes.items():
            where, _, field = name.partition("__")
            if field:
                setattr(getattr(self, where), field, value)
            elif where in self.args:
                self.args[where] = value
            else:
                setattr(self, where, value)

    def heads(self):
        return _lib.lib().tl_rope_heads(self.q, self.k, self.args["dtype"], self.args["tokens"], self.args["head_dim"], self.rotation, None)

    def to_pages(self):
        return _lib.lib().tl_rope_to_pages(self.q, self.k, self.v, self.args["dtype"], self.args["tokens"], self.rotation, self.pages, self.batch, None)

    def read(self):
        return _lib.lib().tl_read_pages(self.pages, self.batch, self.args["tokens"], self.args["dtype"], self.args["k_out"], self.args["out"],
                                        self.args["out_token"], 64, None)

    def attend(self):
        a = self.args
        return _lib.lib().tl_paged_attention(1 << 20, a["q_token"], 64, a["dtype"], a["tokens"], a["heads"], self.pages, self.batch, a["most"], a["scale"],
                                             a["out"], a["workspace"], a["bytes"], None)


ARG, SHAPE, DTYPE, ALIGN, UNSUPPORTED, SIZE = -1, -2, -3, -4, -5, -8


@pytest.mark.parametrize("call,changes,code", [
    ("heads", {"dtype": 2}, DTYPE), ("heads", {"head_dim": 60}, UNSUPPORTED), ("heads", {"head_dim": 520}, UNSUPPORTED), ("heads", {"head_dim": 0}, UNSUPPORTED),
    ("heads", {"tokens": -1}, SHAPE), ("heads", {"tokens": 1 << 40}, SHAPE), ("heads", {"rotation": None}, ARG), ("heads", {"rotation__pairs": 33}, SHAPE),
    ("heads", {"rotation__pairs": -1}, SHAPE), ("heads", {"rotation__frequencies": None}, ARG), ("heads", {"rotation__positions": None}, ARG),
    ("heads", {"q__x": None}, ARG), ("heads", {"q__y": None}, ARG), ("heads", {"k__heads": -1}, SHAPE), ("heads", {"q__x": (1 << 20) + 8}, ALIGN),
    ("heads", {"q__x_token": 257}, ALIGN), ("heads", {"k__y_head": 4}, ALIGN), ("heads", {"q__norm_weight": 8}, ALIGN),
    ("to_pages", {"dtype": 7}, DTYPE), ("to_pages", {"pages": None}, ARG), ("to_pages", {"batch": None}, ARG), ("to_pages", {"pages__k": None}, ARG),
    ("to_pages", {"k__heads": 3}, SHAPE), ("to_pages", {"v__heads": 0}, SHAPE), ("to_pages", {"v__norm_weight": 16}, ARG), ("to_pages", {"rotation__pairs": 33}, SHAPE),
    ("to_pages", {"batch__starts": None}, ARG), ("to_pages", {"batch__lengths": None}, ARG), ("to_pages", {"batch__table": None}, ARG),
    ("read", {"dtype": 2}, DTYPE), ("read", {"out_token": 129}, ALIGN), ("read", {"k_out": 8}, ALIGN), ("read", {"tokens": -3}, SHAPE),
    ("read", {"pages__page_size": 8}, SHAPE), ("read", {"pages__page_size": 48}, SHAPE), ("read", {"pages__page_size": 2048}, SHAPE), ("read", {"pages__pages": 0}, SHAPE),
    ("read", {"pages__pages": 1 << 40}, SHAPE), ("read", {"pages__kv_heads": 0}, SHAPE), ("read", {"pages__head_dim": 72}, SHAPE), ("read", {"pages__head_dim": 528}, SHAPE),
    ("read", {"pages__slot_stride": 32}, SHAPE), ("read", {"pages__page_stride": 0}, SHAPE), ("read", {"pages__head_stride": -64}, SHAPE),
    ("read", {"pages__slot_stride": 1 << 28}, SHAPE), ("read", {"pages__head_stride": 1025}, ALIGN), ("read", {"pages__v": 24}, ALIGN),
    ("read", {"pages__dtype": 0}, DTYPE), ("read", {"pages__dtype": 2}, ARG), ("read", {"pages__k_exponents": 16}, None), ("read", {"batch__seqs": -1}, SHAPE),
    ("read", {"batch__table_stride": 1}, SHAPE), ("read", {"batch__table_pages": -1}, SHAPE), ("read", {"batch__table_pages": 1 << 30, "batch__table_stride": 1 << 30}, SHAPE),
    ("attend", {"dtype": 0}, UNSUPPORTED), ("attend", {"dtype": 2}, DTYPE), ("attend", {"heads": 3}, SHAPE), ("attend", {"heads": 0}, SHAPE),
    ("attend", {"pages__head_dim": 96, "pages__slot_stride": 96}, UNSUPPORTED), ("attend", {"out": None}, ARG), ("attend", {"workspace": None}, ARG),
    ("attend", {"workspace": 8}, ALIGN), ("attend", {"bytes": 100}, SIZE), ("attend", {"scale": 0.0}, ARG), ("attend", {"scale": -1.0}, ARG),
    ("attend", {"scale": math.nan}, ARG), ("attend", {"scale": 2e30}, ARG), ("attend", {"batch__table_pages": 1 << 23, "batch__table_stride": 1 << 23}, SHAPE), ("attend", {"scale": math.inf}, ARG), ("attend", {"most": -1}, ARG), ("attend", {"q_token": 100}, ALIGN),
    ("attend", {"out": (1 << 20) + 2}, ALIGN)])
def test_the_library_refuses(call, changes, code):
    if code is None:                                # exponents beside fp16 pages: one alone is refused as well
        changes = {**changes, "pages__v_exponents": 16}
        code = ARG
    raw = Raw(**changes)
    assert getattr(raw, call)() == code
    assert _lib.lib().tl_last_error()


@pytest.mark.parametrize("call,changes", [
    ("read", {"pages__slot_stride": 1 << 60}), ("to_pages", {"pages__slot_stride": (1 << 60) + 64}), ("attend", {"pages__slot_stride": 1 << 60}),
    ("heads", {"q__x_head": 1 << 62}), ("heads", {"k__y_head": 1 << 63 - 1}), ("to_pages", {"v__x_head": 1 << 63 - 1}), ("to_pages", {"q__y_head": (1 << 62) + 64})])
def test_strides_whose_products_leave_64_bits(call, changes):
    assert getattr(Raw(**changes), call)() == SHAPE


@pytest.mark.parametrize("call", ["heads", "to_pages", "read", "attend"])
def test_no_rows_need_no_addresses(call):
    raw = Raw(tokens=0, q__x=None, q__y=None, k__x=None, k__y=None, v__x=None, rotation__positions=None, k_out=None, out=None, workspace=None)
    assert getattr(raw, call)() == 0
    if call != "heads":
        assert getattr(Raw(batch__seqs=0, batch__table=None, batch__lengths=None, batch__starts=None), call)() == 0


def test_workspace_size():
    need, raw = ctypes.c_int64(0), Raw()

    def ask(tokens=3, heads=4, pages=raw.pages, batch=raw.batch, most=1, to=ctypes.byref(need)):
        return _lib.lib().tl_paged_attention_workspace(tokens, heads, pages, batch, most, to)

    assert ask() == 0 and need.value > 0
    assert ask(to=None) == ask(pages=None) == ask(batch=None) == ask(most=-1) == ask(tokens=-1) == ARG
    assert ask(heads=3) == SHAPE


def test_what_the_plain_forms_hold():
    """The 8-bit grid of the plain form is torch's, row exponents are the least, and a sequence's rows come out of any order of pages."""
    x = torch.randn((50, 64), generator=torch.Generator().manual_seed(1), dtype=torch.float64) * torch.exp2(torch.arange(50.0))[:, None].double() * 2.0 ** -30
    e = paged.exponents_of(x)
    assert ((x.abs().amax(-1) <= 448 * 2.0 ** e) | (e == 8)).all() and ((x.abs().amax(-1) > 448 * 2.0 ** (e - 1)) | (e == -32)).all()
    small = e < 8
    codes = (x / 2.0 ** e[:, None]).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(paged.byte_values(x)[small], (codes * 2.0 ** e[:, None])[small])
    seqs = paged.Sequences([(2, 40), (1, 16), (0, 0)], 16)
    pool = torch.zeros((seqs.pages, 1, 16, 1))
    for _, b, at, page, slot in seqs.rows():
        pool[page, 0, slot, 0] = 100 * b + at
    assert seqs.held(0, pool)[38:].flatten().tolist() == [38, 39] and seqs.held(1, pool)[15].item() == 115 and seqs.held(2, pool).shape == (0, 1, 1)


# ---------------------------------------------------------------- what the host keeps
def test_sequences_hold_the_pages_that_they_need():
    from ternaryllm_amd import PagedCache
    cache = PagedCache(2, 6, 2, 64, 16, device="cpu")
    a, b = cache.open(), cache.open()
    batch = cache.extend([(a, 17), (b, 3)])
    assert batch.starts.tolist() == [0, 17, 20] and batch.lengths.tolist() == [17, 3] and batch.most_rows == 17 and batch.table.shape == (2, 2)
    assert all(t.dtype == torch.int32 for t in batch[:3]) and cache.free_pages == 3
    held = set(batch.table[0].tolist()) | {batch.table[1, 0].item()}
    assert len(held) == 3 and held <= set(range(6))
    again = cache.extend([(b, 1), (a, 15)])                      # b first; both within their pages
    assert again.lengths.tolist() == [4, 32] and cache.free_pages == 3 and again.table[1].tolist() == batch.table[0].tolist()
    with pytest.raises(RuntimeError):
        cache.extend([(a, 48), (b, 13)])                          # four pages of three; nothing changes
    assert cache.free_pages == 3 and cache.length(a) == 32 and cache.length(b) == 4
    cache.truncate(a, 16)
    assert cache.free_pages == 4 and cache.length(a) == 16
    whole = cache.whole([a, b])
    assert whole.starts.tolist() == [0, 16, 20] and whole.lengths.tolist() == [16, 4]
    cache.close(a)
    assert cache.free_pages == 5
    c = cache.open()
    assert c not in (a, b) and cache.length(c) == 0 and cache.extend([(c, 0), (b, 0)]).most_rows == 0
    for bad in ([], [(a, 1)], [(b, 1), (b, 1)], [(b, -1)]):
        with pytest.raises(ValueError):
            cache.extend(bad)
    for length in (-1, 5):
        with pytest.raises(ValueError):
            cache.truncate(b, length)
    assert cache.length(b) == 4


def state_of(cache):
    return list(cache._free), {s: (list(held), n) for s, (held, n) in cache._sequences.items()}


def test_a_batch_that_cannot_be_made_takes_no_pages(monkeypatch):
    from ternaryllm_amd import PagedCache
    cache = PagedCache(1, 9, 2, 64, 16, device="cpu")
    a, b = cache.open(), cache.open()
    cache.extend([(a, 20), (b, 1)])
    before = state_of(cache)

    def none(*_):
        raise RuntimeError("no memory")

    with monkeypatch.context() as m:
        m.setattr(ops, "PageBatch", none)
        with pytest.raises(RuntimeError, match="no memory"):
            cache.extend([(a, 20), (b, 40)])
    assert state_of(cache) == before


@pytest.mark.parametrize("shape,dtype,why", [((128, 4), torch.float16, RuntimeError), ((256, 4), torch.float32, RuntimeError), ((256, 4), torch.float16, None)])
def test_a_pass_that_raises_leaves_the_sequences_as_they_were(shape, dtype, why):
    """Refused before it begins -- heads of 32, a decoder of fp32 -- or raising on the way, as every pass does here, where there is no GPU."""
    from ternaryllm_amd import PagedCache, TernaryConfig, TernaryLlamaDecoder
    cfg = TernaryConfig(hidden_size=shape[0], intermediate_size=128, num_hidden_layers=2, num_attention_heads=shape[1], num_key_value_heads=shape[1], vocab_size=64,
                        max_position_embeddings=200, sparsity=0.66)
    model = TernaryLlamaDecoder(cfg, seed=5, device="cpu", dtype=dtype, pack_threads=2)
    cache = PagedCache(2, 12, shape[1], cfg.head_dim, 16, device="cpu")
    a, b, c = cache.open(), cache.open(), cache.open()
    cache.extend([(a, 20), (b, 3), (c, 33)])
    cache.close(c)
    before, text = state_of(cache), torch.arange(40)
    with pytest.raises(why or Exception):
        model.extend(cache, [(b, text), (a, text[:13])])
    assert state_of(cache) == before
    for bad in (text.float(), text.bool(), text[None], text[:0], text.to(torch.uint8)):
        with pytest.raises(ValueError):
            model.extend(cache, [(a, text[:3]), (b, bad)])
    with pytest.raises(ValueError if why is None else why):          # another decoder's cache
        other = PagedCache(1, 12, shape[1], cfg.head_dim, 16, device="cpu")
        model.extend(other, [(other.open(), text)])
    assert state_of(cache) == before


@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_layers_of_a_paged_cache(dtype):
    from ternaryllm_amd import PagedCache
    cache = PagedCache(3, 4, 2, 32, 32, dtype, device="cpu")
    layers = [cache.layer(i) for i in range(3)]
    for p in layers:
        assert p.k.dtype == p.v.dtype == dtype and p.k.shape == p.v.shape == (4, 2, 32, 32) and (p.k_exponents is None) == (dtype == torch.float16)
        if p.k_exponents is not None:
            assert p.k_exponents.shape == p.v_exponents.shape == (4, 2, 32) and p.k_exponents.is_contiguous()
    assert len({p.k.data_ptr() for p in layers} | {p.v.data_ptr() for p in layers}) == 6


@pytest.mark.parametrize("change", [{"dtype": torch.float32}, {"page_size": 24}, {"page_size": 8}, {"page_size": 2048}, {"pages": 0}, {"layers": 0}, {"head_dim": 40}])
def test_paged_caches_that_are_refused(change):
    from ternaryllm_amd import PagedCache
    with pytest.raises(ValueError):
        PagedCache(**{**dict(layers=1, pages=2, kv_heads=1, head_dim=64, device="cpu"), **change})


SCALINGS = [
    None, {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 2.5, "original_max_position_embeddings": 1000, "beta_fast": 20, "beta_slow": 2, "attention_factor": 0.75}]


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("rotary,theta", [(128, 10000.0), (64, 500000.0), (20, 10000.0)])
def test_rope_frequencies(scaling, rotary, theta):
    from ternaryllm_amd.attention import rope_frequencies
    got, factor = rope_frequencies(rotary, theta, scaling)
    assert got.dtype == torch.float64 and got.shape == (rotary // 2,)
    kind = (scaling or {}).get("rope_type", "default")
    for i in range(rotary // 2):                                  # dimension by dimension, from the definition
        f = theta ** (-2 * i / rotary)
        if kind == "linear":
            f /= scaling["factor"]
        if kind == "llama3":
            length, wave = scaling["original_max_position_embeddings"], 2 * math.pi / f
            if wave > length / scaling["low_freq_factor"]:
                f /= scaling["factor"]
            elif wave >= length / scaling["high_freq_factor"]:
                part = (length / wave - scaling["low_freq_factor"]) / (scaling["high_freq_factor"] - scaling["low_freq_factor"])
                f = (1 - part) * f / scaling["factor"] + part * f
        if kind == "yarn":
            edges = [rotary * math.log(scaling["original_max_position_embeddings"] / (2 * math.pi * n)) / (2 * math.log(theta))
                     for n in (scaling.get("beta_fast", 32), scaling.get("beta_slow", 1))]
            low, high = max(math.floor(edges[0]), 0), min(math.ceil(edges[1]), rotary - 1)
            ramp = min(max((i - low) / (high - low), 0.0), 1.0)
            f = f / scaling["factor"] * ramp + f * (1 - ramp)
        assert abs(got[i].item() / f - 1) < 1e-12
    assert factor == (1.0 if kind != "yarn" else scaling.get("attention_factor") or 0.1 * math.log(scaling["factor"]) + 1)


@pytest.mark.parametrize("scaling", [s for s in SCALINGS if s and s["rope_type"] != "default"])
def test_rope_frequencies_are_those_of_transformers(scaling):
    utils = pytest.importorskip("transformers.modeling_rope_utils")
    transformers = pytest.importorskip("transformers")
    from ternaryllm_amd.attention import rope_frequencies
    try:
        cfg = transformers.LlamaConfig(hidden_size=1024, num_attention_heads=8, max_position_embeddings=65536, rope_parameters={"rope_theta": 10000.0, **scaling})
        cfg.rope_parameters
    except Exception:
        pytest.skip("a release whose configurations have no rope_parameters")
    want, factor = utils.ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    got, mine = rope_frequencies(128, 10000.0, scaling)
    # theirs are fp32 throughout: a power, a quotient and a weighted mean
    assert (got / want.double() - 1).abs().max() < 2.0 ** -20 and abs(mine - factor) < 1e-6


def test_rope_frequencies_refuses():
    from ternaryllm_amd.attention import rope_frequencies
    for args in ((0, 1e4), (7, 1e4), (8, 1e4, {"rope_type": "no such"})):
        with pytest.raises(ValueError):
            rope_frequencies(*args)


YARNS = [{"mscale": 1.0, "mscale_all_dim": 1.0}, {"mscale": 0.707, "mscale_all_dim": 1.2}, {"mscale": 0.5}, {"mscale_all_dim": 0.5}, {"mscale": 0.8, "mscale_all_dim": 0.0},
         {"mscale": 0.8, "mscale_all_dim": 0.6, "attention_factor": 1.5}, {"truncate": False}, {"truncate": True}, {"truncate": False, "mscale": 0.7, "mscale_all_dim": 0.9}]


@pytest.mark.parametrize("more", YARNS)
@pytest.mark.parametrize("scale", [0.5, 1.0, 8.0])
def test_yarn_takes_all_that_a_configuration_says(more, scale):
    from ternaryllm_amd.attention import rope_frequencies
    rotary, theta, length = 64, 10000.0, 4096
    got, factor = rope_frequencies(rotary, theta, {"rope_type": "yarn", "factor": scale, "original_max_position_embeddings": length, **more})
    log = math.log(scale) if scale > 1 else 0.0                   # (contexts that do not grow want no factor)
    want = 0.1 * log + 1
    if more.get("mscale") and more.get("mscale_all_dim"):
        want = (0.1 * more["mscale"] * log + 1) / (0.1 * more["mscale_all_dim"] * log + 1)
    assert abs(factor - more.get("attention_factor", want)) < 1e-15
    edges = [rotary * math.log(length / (2 * math.pi * n)) / (2 * math.log(theta)) for n in (32, 1)]
    if more.get("truncate", True):
        edges = math.floor(edges[0]), math.ceil(edges[1])
    for i in range(rotary // 2):
        ramp = min(max((i - edges[0]) / (edges[1] - edges[0]), 0.0), 1.0)
        f = theta ** (-2 * i / rotary)
        assert abs(got[i].item() / (f / scale * ramp + f * (1 - ramp)) - 1) < 1e-12


@pytest.mark.parametrize("more", YARNS)
def test_yarn_is_that_of_transformers(more):
    test_rope_frequencies_are_those_of_transformers({"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096, **more})
