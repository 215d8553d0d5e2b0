"""Plain implementations, in float64 on the CPU, of the operators of a paged cache, and batches to try them on."""
import math

import torch

LARGEST, LEAST_EXPONENT, MOST_EXPONENT = 448.0, -32, 8


def normed(x, weight, eps):
    x = x.double()
    return x if weight is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()


def rotated(x, positions, frequencies, interleaved, factor):
    """x [tokens, heads, head_dim] float64, pair by pair."""
    y = x.clone()
    for i in range(len(frequencies)):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + len(frequencies))
        angle = positions.double() * float(frequencies[i])
        c, s = (factor * angle.cos())[:, None], (factor * angle.sin())[:, None]
        y[..., lo] = x[..., lo] * c - x[..., hi] * s
        y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def rope_bound(x, partner_of, factor, dtype, y):
    """How far a result may be off: half a step of its type, and in fp32 the angle (3.2 steps of 2^-24, as turns rounded to 24 bits times 2 pi / 2), its
    sine and cosine (2), factor, product and sum (3), the norm's factor (10: 8 squares in a row and 6 sums, halved by the root, root and
    quotient) and two products -- 24 in all, of the two values of a pair."""
    half = torch.finfo(dtype).eps / 2
    return half * y.abs() + 24 * 2.0 ** -24 * factor * (x.abs() + partner_of.abs()) + 2.0 ** -25


def partners(x, pairs, interleaved):
    y = x.clone()
    for i in range(pairs):
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
        y[..., lo], y[..., hi] = x[..., hi], x[..., lo]
    return y


def exponents_of(x):
    """The least e from -32 to 8 with max|x| <= 448 * 2^e, over the last dimension; NaN left out."""
    most = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).abs().amax(-1)
    e = torch.full_like(most, LEAST_EXPONENT)
    for p in range(LEAST_EXPONENT, MOST_EXPONENT):
        e = torch.where(most > LARGEST * 2.0 ** p, p + 1.0, e)
    return e


def byte_values(x):
    """What rows of 8 bits stand for."""
    e = exponents_of(x)[..., None]
    bound = torch.where(e == MOST_EXPONENT, 240.0, LARGEST)
    y = torch.minimum(torch.maximum(x / 2.0 ** e, -bound), bound)
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * 2.0 ** e


class Sequences:
    """A batch of (new rows, length) on the CPU, their pages in any order among pages of nobody, rows in front of the first and behind the last."""

    def __init__(self, both, page_size, *, front=0, behind=0, spare=2, seed=0, widest=None):
        self.both, self.page_size, self.front = both, page_size, front
        count = [-(-length // page_size) for _, length in both]
        self.pages = sum(count) + spare
        order = torch.randperm(self.pages, generator=torch.Generator().manual_seed(seed)).tolist()
        columns = max([1, *count]) if widest is None else widest
        self.table = torch.full((len(both), columns), -7, dtype=torch.int32)      # (what is not to be read is no page)
        for b, n in enumerate(count):
            for j in range(n):
                self.table[b, j] = order.pop()
        self.starts = torch.tensor([front + sum(n for n, _ in both[:b]) for b in range(len(both) + 1)], dtype=torch.int32)
        self.lengths = torch.tensor([length for _, length in both], dtype=torch.int32)
        self.tokens = int(self.starts[-1]) + behind
        self.most = max([0, *(n for n, _ in both)])

    def batch(self, ops, device="cuda", most=None):
        return ops.PageBatch(self.table.to(device), self.starts.to(device), self.lengths.to(device), self.most if most is None else most)

    def rows(self):
        """(row, sequence, index, page, slot) of every row of a sequence that has a place."""
        for b, (n, length) in enumerate(self.both):
            for i in range(n):
                at = length - n + i
                if at >= 0:
                    yield int(self.starts[b]) + i, b, at, int(self.table[b, at // self.page_size]), at % self.page_size

    def held(self, b, pages):
        """Sequence b's rows [length, kv_heads, head_dim] out of pages [pages, kv_heads, page_size, head_dim]."""
        n = self.both[b][1]
        ids = [int(p) for p in self.table[b, :-(-n // self.page_size)]]
        return torch.cat([pages[i].transpose(0, 1) for i in ids])[:n] if n else pages.new_zeros((0, pages.shape[1], pages.shape[3]))


def values(codes, exponents):
    """Pages as float64."""
    return codes.double() if exponents is None else codes.double() * torch.pow(2.0, exponents.double() - 127)[..., None]


def attention(q, k_pages, v_pages, seqs, scale):
    """q [tokens, heads, head_dim], pages as float64: [tokens, heads, head_dim], NaN in rows of no sequence."""
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    group = q.shape[1] // k_pages.shape[1]
    for b, (n, length) in enumerate(seqs.both):
        k, v = (seqs.held(b, t).repeat_interleave(group, 1) for t in (k_pages, v_pages))
        for i in range(n):
            row, seen = int(seqs.starts[b]) + i, max(length - n + i + 1, 0)
            if seen == 0:
                out[row] = 0
                continue
            s = torch.einsum("hd,khd->hk", q[row].double(), k[:seen]) * scale
            out[row] = torch.einsum("hk,khd->hd", torch.softmax(s, -1), v[:seen])
    return out
