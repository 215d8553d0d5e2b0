"""Plain implementations, in float64 on the CPU, of the losses of a ternary head, and how far a kernel may be from them."""
import math

import torch

from tests.util import ternary_weight

U = 2.0 ** -24                  # half a step of fp32


def head(K, N, dtype, seed=0, sparsity=0.6, scaled=True):
    """A weight int32 [K, N] (numpy) and its columns' scales, or None."""
    w = ternary_weight(K, N, sparsity, seed)
    if not scaled:
        return w, None
    g = torch.Generator().manual_seed(seed + 1)
    return w, ((0.5 + torch.rand(N, generator=g)) / math.sqrt(max(1.0, 0.4 * K))).to(dtype)


def rows(M, K, dtype, seed=0):
    """Small integers: every sum of a product with ternary weights is exact in fp32, whatever its order."""
    return torch.randint(-8, 9, (M, K), generator=torch.Generator().manual_seed(seed + 2)).to(dtype)


def teacher(ids, logits, N, heat):
    """The distributions [rows, N] that a teacher's top logits stand for, and which rows have one."""
    there = (logits > -math.inf).any(-1) | logits.isnan().any(-1)
    t = torch.softmax(torch.where(there[:, None], logits.double(), 0.0) / heat, -1) * there[:, None]
    wanted = torch.zeros((ids.shape[0], N), dtype=torch.float64)
    for m in range(ids.shape[0]):
        for i in range(ids.shape[1]):
            if t[m, i] != 0:
                wanted[m, int(ids[m, i])] += t[m, i]
    return wanted, there


def targets(t, N, ignore=-100):
    wanted = torch.zeros((t.numel(), N), dtype=torch.float64)
    for m in range(t.numel()):
        if int(t[m]) != ignore:
            wanted[m, int(t[m])] = 1.0
    return wanted, t != ignore


class Reference:
    """Loss and gradients of sum(grad * loss), for `wanted` [rows, N] of the rows that count, and what bounds a kernel's distance from them."""

    def __init__(self, x, w, scale, wanted, counts, heat=1.0, grad=None):
        self.x, self.w = x.double(), torch.as_tensor(w).double()
        self.s = torch.ones(self.w.shape[1], dtype=torch.float64) if scale is None else scale.double()
        self.wanted, self.counts, self.heat, self.dtype = wanted, counts, heat, x.dtype
        self.raw = self.x @ self.w
        self.z = self.raw * self.s / heat
        logs = torch.log_softmax(self.z, -1)
        gap = wanted * -logs
        self.loss = torch.where(counts, heat * heat * (torch.special.xlogy(wanted, wanted) + gap).sum(-1), 0.0)
        self.grad = torch.ones(x.shape[0], dtype=torch.float64) if grad is None else grad.double()
        self.dz = torch.where(counts[:, None], (logs.exp() - wanted) * (heat * self.grad)[:, None], 0.0)
        self.dx = (self.dz * self.s) @ self.w.t()
        self.ds = (self.dz * self.raw).sum(0)
        self.far = self.z.abs().amax(-1)
        # A logit is rounded twice (scale, temperature); an exponential's argument once more, and itself by 2; sums of exponentials take at most 100 roundings
        # (8 and what is joined, then a tree); the logarithm 2 of its result, which is no more than the largest logit and log N.
        self.off = U * (8 * self.far + 120)
        self.probabilities = logs.exp()

    def loss_bound(self):
        gap = 2 * self.far + 20                      # of lse and a logit
        return self.heat ** 2 * (self.off + U * 24 * gap) + U * self.loss.abs()

    def gradient_bounds(self):
        half = torch.finfo(self.dtype).eps / 2
        g = (self.heat * self.grad).abs() * self.counts
        dz = self.probabilities * (self.off + U * 4)[:, None] + U * 4 * self.wanted
        size = (self.probabilities - self.wanted).abs() * self.s.abs()
        a = self.w.abs().t()
        # rounded to the rows' type, with a lower end; each of N additions may round what is there; the factor, and the result
        p = dz * self.s.abs() + (half + 3 * U) * size + 2.0 ** -39 * float(self.s.abs().max())
        dx = g[:, None] * ((p + U * (self.w.shape[1] + 8) * size) @ a) + half * self.dx.abs() + 2.0 ** -25
        ds = ((dz + U * (self.x.shape[0] + 4) * (self.probabilities - self.wanted).abs()) * g[:, None] * self.raw.abs()).sum(0)
        return dx, ds


def thin_head(K, N, entries, seed=0):
    """A weight int32 [K, N] (numpy) of `entries` weights in every column."""
    g = torch.Generator().manual_seed(seed)
    w = torch.zeros((K, N), dtype=torch.int32)
    for _ in range(entries):
        at = torch.randint(0, K, (1, N), generator=g)
        w.scatter_(0, at, torch.randint(0, 2, (1, N), generator=g, dtype=torch.int32) * 2 - 1)
    return w.numpy()


def long_rows(M, K, seed=0):
    """fp32 numbers of up to 22 bits below 4, which take all three of the bf16 parts that such rows are multiplied in: sums of four are exact in fp32 all the same."""
    return torch.randint(-(1 << 22) + 1, 1 << 22, (M, K), generator=torch.Generator().manual_seed(seed + 6)).float() * 2.0 ** -20


def long_scales(N, seed=0):
    """Column scales that make logits of up to a few tens of sums of those."""
    return torch.exp2(torch.rand(N, generator=torch.Generator().manual_seed(seed + 7)))


def leading_parts(x, parts):
    """fp32 rows with no more than their first `parts` bf16 parts."""
    bits = {1: 0xffff0000, 2: 0xffffff00}[parts] - (1 << 32)
    return (x.contiguous().view(torch.int32) & bits).view(torch.float32)
