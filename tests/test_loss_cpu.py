"""What the losses of a ternary head refuse, without a GPU: the tensor-level checks, and the library's own in front of a launch.  And the oracle's gradients
against differences of its losses."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from ternaryllm_amd import TernaryLinear, _lib, ops, packing

from tests import losses


class Weight:
    """A DeviceWeight whose blob is on the CPU."""

    def __init__(self, K=64, N=100):
        packed = packing.PackedWeight.from_dense(torch.as_tensor(losses.head(K, N, torch.float32)[0]))
        self.header, self.blob = packed.header, torch.from_numpy(packed.blob)
        self.inners, self.columns, self.device = K, N, self.blob.device


class Back:
    def __init__(self, weight):
        self.header, self.blob, self.codes = weight.header, weight.blob, torch.zeros(16, dtype=torch.uint8)


def operands(rows=3):
    w = Weight()
    return w, torch.zeros((rows, 64), dtype=torch.float16), torch.zeros(rows, dtype=torch.int64), torch.zeros(100, dtype=torch.float16)


def test_operands_that_do_not_fit():
    w, x, t, s = operands()
    ids, logits = torch.zeros((3, 5), dtype=torch.int64), torch.zeros((3, 5))
    other = Back(Weight(64, 101))
    bad = [
        lambda: ops.cross_entropy(w, x[:, :63], t, s), lambda: ops.cross_entropy(w, x[0], t, s), lambda: ops.cross_entropy(w, x.bfloat16(), t, s),
        lambda: ops.cross_entropy(w, x, t[:2], s), lambda: ops.cross_entropy(w, x, t.int(), s), lambda: ops.cross_entropy(w, x, t[:, None], s),
        lambda: ops.cross_entropy(w, x, t, s[:99]), lambda: ops.cross_entropy(w, x, t, s.bfloat16()), lambda: ops.cross_entropy(w, x, t, s[None]),
        lambda: ops.cross_entropy(w, x, t, torch.zeros(200).half()[::2]), lambda: ops.cross_entropy(w, x, t, s, back=other),
        lambda: ops.cross_entropy(w, x.requires_grad_(), t, s), lambda: ops.distillation(w, x.detach(), ids[:2], logits, s),
        lambda: ops.distillation(w, x.detach(), ids, logits[:, :4], s), lambda: ops.distillation(w, x.detach(), ids.int(), logits, s),
        lambda: ops.distillation(w, x.detach(), ids, logits.bfloat16(), s), lambda: ops.distillation(w, x.detach(), ids[:, 0], logits[:, 0], s),
        lambda: ops.distillation(w, x.detach(), ids[:, :0], logits[:, :0], s), lambda: ops.distillation(w, x.detach(), ids, logits, s, temperature=0.0),
        lambda: ops.distillation(w, x.detach(), ids, logits, s, temperature=-1.0), lambda: ops.distillation(w, x.detach(), ids, logits, s, temperature=float("nan")),
        lambda: ops.distillation(w, x.detach(), ids.repeat(1, 300), logits.repeat(1, 300), s)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    x = x.detach()
    with pytest.raises(RuntimeError, match="gradient"):
        ops.distillation(w, x, ids, logits.requires_grad_(), s)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangents"):
        ops.cross_entropy(w, forward_ad.make_dual(x, torch.ones_like(x)), t, s)
    for call in (lambda: ops.cross_entropy(w, x, t, s), lambda: ops.distillation(w, x, ids, logits.detach(), s), lambda: ops.BackWeight(w)):
        with pytest.raises(RuntimeError, match="GPU"):           # taken, up to the GPU that is not there
            call()


def test_modules_refuse_rows_that_are_not_theirs():
    linear = TernaryLinear(64, 32, bias=False, reference_buffers=False)
    with pytest.raises(ValueError):
        linear.cross_entropy(torch.zeros((2, 63)), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        linear.cross_entropy(torch.zeros((2, 3, 64)), torch.zeros((2, 2), dtype=torch.int64))
    with pytest.raises(ValueError):
        linear.distillation(torch.zeros((2, 64)), torch.zeros((3, 4), dtype=torch.int64), torch.zeros((3, 4)))
    with pytest.raises(RuntimeError):
        linear.cross_entropy(torch.zeros((2, 64)), torch.zeros(2, dtype=torch.int64))


def target(**change):
    at = ctypes.c_void_p(256)
    t = dict(targets=at, ignore=-100, entries=None, shares=None, known=None, top=1, temperature=1.0)
    t.update(change)
    return _lib.LossTarget(**t)


def test_the_library_checks_before_it_launches():
    L, h, at = _lib.lib(), Weight().header, 256                  # (addresses that are never followed: every call is refused)
    size = ctypes.c_int64(0)
    teacher = dict(targets=None, entries=ctypes.c_void_p(256), shares=ctypes.c_void_p(256), known=ctypes.c_void_p(256), top=4)
    for t in (target(temperature=0.0), target(temperature=2.0), target(targets=None), target(**dict(teacher, targets=ctypes.c_void_p(256))),
              target(**dict(teacher, top=0)), target(**dict(teacher, top=1025)), target(**dict(teacher, shares=None)), target(**dict(teacher, temperature=float("inf")))):
        assert L.tl_head_loss_workspace(h, 10, _lib.TL_F16, t, 0, size) == -1
    good = target()
    assert L.tl_head_loss_workspace(h, -1, _lib.TL_F16, good, 0, size) == -1 and L.tl_head_loss_workspace(h, 10, 7, good, 0, size) == -3
    for M in (1, 48, 49, 5000):
        for code in (_lib.TL_F16, _lib.TL_F32):
            need = []
            for backward in (0, 1):
                assert L.tl_head_loss_workspace(h, M, code, good, backward, size) == 0 and size.value > 0
                need.append(size.value)
            forward = lambda **c: L.tl_head_loss(*dict(dict(h=h, b=at, x=at, t=code, l=64, m=M, s=at, k=_lib.TL_F32, w=good, o=at, e=at, ws=at, n=need[0], st=None), **c).values())
            assert forward(n=need[0] - 1) == -8 and forward(b=None) == -4 and forward(b=16) == -4 and forward(x=None) == -1 and forward(l=63) == -2
            assert forward(ws=None) == -4 and forward(ws=64) == -4 and forward(x=257) == -4 and forward(s=257) == -4 and forward(k=5) == -3 and forward(o=None) == -1
            assert forward(m=-1) == -2 or forward(m=-1) == -1
            back = lambda **c: L.tl_head_loss_backward(*dict(dict(h=h, b=at, c=at, x=at, t=code, l=64, m=M, s=at, k=_lib.TL_F32, w=good, e=at, g=at, d=at, dl=64,
                                                                  ds=at, ws=at, n=need[1], st=None), **c).values())
            assert back(n=need[1] - 1) == -8 and back(c=None) == -4 and back(c=8) == -4 and back(dl=63) == -2 and back(s=None) == -1 and back(e=None) == -1 and back(g=None) == -1
    # nothing to do
    assert L.tl_head_loss(h, at, None, _lib.TL_F16, 64, 0, None, 0, good, None, None, None, 0, None) == 0
    teach = lambda **c: L.tl_teacher_entries(*dict(dict(i=at, il=4, l=at, t=_lib.TL_F32, ll=4, m=3, top=4, n=100, h=1.0, e=at, s=at, k=at, st=None), **c).values())
    assert teach(il=3) == -2 and teach(ll=3) == -2 and teach(top=0) == -1 and teach(top=1025) == -1 and teach(h=0.0) == -1 and teach(t=9) == -3 and teach(i=None) == -1
    assert teach(n=0) == -2 and teach(m=-1) == -2 and teach(m=0) == 0
    assert L.tl_back_codes_make(h, at, None, None) == -4 and L.tl_back_codes_make(h, None, at, None) == -4
    assert L.tl_back_codes_size(h, size) == 0 and size.value == 1024 * 4      # 4 blocks of 16 columns, one unit of 256 rows
    old = _lib.LayoutHeader.from_buffer_copy(bytes(h))
    old.version, old.off_codes, old.code_units, old.code_planes = 5, 0, 0, 0   # (packed before the format had codes)
    assert L.tl_back_codes_size(old, size) == -5


def test_the_oracles_gradients_are_those_of_differences():
    w, s = losses.head(24, 40, torch.float32, 2)
    x, g = losses.rows(5, 24, torch.float32, 2), torch.rand(5, generator=torch.Generator().manual_seed(3))
    ids, logits = torch.randint(0, 40, (5, 4), generator=torch.Generator().manual_seed(4)), torch.randn((5, 4), generator=torch.Generator().manual_seed(5))
    logits[1] = float("-inf")
    wanted, counts = losses.teacher(ids, logits, 40, 2.0)
    ref = losses.Reference(x, w, s, wanted, counts, heat=2.0, grad=g)
    assert ref.loss[1] == 0 and (ref.dx[1] == 0).all()
    for i, (at, grad) in enumerate(((x.double(), ref.dx), (s.double(), ref.ds))):
        for index in [(0, 3), (2, 7), (4, 23)] if i == 0 else [(0,), (13,), (39,)]:
            total = []
            for sign in (1, -1):
                both = [x.double(), s.double()]
                both[i] = at.clone()
                both[i][index] += sign * 1e-5
                total.append(float((losses.Reference(both[0], w, both[1], wanted, counts, heat=2.0).loss * g.double()).sum()))
            assert abs((total[0] - total[1]) / 2e-5 - float(grad[index])) <= 1e-6 * (1 + abs(float(grad[index])))


@pytest.mark.parametrize("M,K,N", [(5, 72, 333), (60, 301, 333), (200, 64, 5003)])
def test_rows_of_all_bits_would_show_a_part_that_is_lost(M, K, N):
    """What the GPU's losses of fp32 rows are tried on: sums that are exact, and bounds that the oracle itself passes with none of its rows' bf16 parts left out."""
    w, x, s = losses.thin_head(K, N, 4, M), losses.long_rows(M, K, M), losses.long_scales(N, M)
    t, g = torch.randint(0, N, (M,), generator=torch.Generator().manual_seed(M)), torch.rand(M, generator=torch.Generator().manual_seed(1)) + 0.25
    ref = losses.Reference(x, w, s, *losses.targets(t, N), grad=g)
    assert torch.equal(ref.raw, ref.raw.float().double()) and float(ref.raw.abs().max()) < 16
    dx_bound, ds_bound = ref.gradient_bounds()
    for parts in (1, 2):
        less = losses.Reference(losses.leading_parts(x, parts), w, s, *losses.targets(t, N), grad=g)
        assert ((less.loss - ref.loss).abs() > 2 * ref.loss_bound()).any() and ((less.ds - ref.ds).abs() > 2 * ds_bound).any()


@pytest.mark.parametrize("temperature", [1e-7, 1e-20, 1e-39, 1e-45, 2e6, float("inf")])
def test_temperatures_whose_reciprocal_or_square_fp32_does_not_hold(temperature):
    w, x, _, s = operands()
    ids, logits = torch.zeros((3, 5), dtype=torch.int64), torch.zeros((3, 5))
    with pytest.raises(ValueError, match="temperature"):
        ops.distillation(w, x, ids, logits, s, temperature=temperature)
    at, size = ctypes.c_void_p(256), ctypes.c_int64(0)
    t = target(targets=None, entries=at, shares=at, known=at, top=4, temperature=temperature)
    assert _lib.lib().tl_head_loss_workspace(w.header, 10, _lib.TL_F16, t, 0, size) == -1
    assert _lib.lib().tl_teacher_entries(256, 4, 256, _lib.TL_F32, 4, 3, 4, 100, temperature, 256, 256, 256, None) == -1
