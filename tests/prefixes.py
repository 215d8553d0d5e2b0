"""Batches in which groups of sequences begin with the same tokens, on the CPU, to try the paged attention on."""
import torch

from tests import paged


class Shared(paged.Sequences):
    """groups: [(tokens that its sequences share, [(new rows, tokens behind the shared ones, the new ones among them), ...]), ...].  A group's sequences hold
    the shared tokens' whole pages in common, and each a copy of those that end inside a page."""

    def __init__(self, groups, page_size, **how):
        super().__init__([(n, shared + behind) for shared, rows in groups for n, behind in rows], page_size, **how)
        self.groups, self.firsts, self.shared = [0], [], []
        for shared, rows in groups:
            first = self.groups[-1]
            self.groups.append(first + len(rows))
            self.firsts += [first] * len(rows)
            self.shared += [shared] * len(rows)
        for b, (first, shared) in enumerate(zip(self.firsts, self.shared)):
            self.table[b, :shared // page_size] = self.table[first, :shared // page_size]

    def copied(self, *pages):
        """Pages with each group's shared tokens in its other sequences' copies as well."""
        for t in pages:
            if t is None:
                continue
            t = t.view(torch.uint8) if t.element_size() == 1 else t
            for b, (first, shared) in enumerate(zip(self.firsts, self.shared)):
                at, rest = shared // self.page_size, shared % self.page_size
                if rest and b != first:
                    t[int(self.table[b, at]), :, :rest] = t[int(self.table[first, at]), :, :rest]

    def prefix(self, ops, device="cuda", most=1 << 30):
        """(Said to be so long that they are read apart, however short they are.)"""
        return ops.PagePrefix(*(torch.tensor(t, dtype=torch.int32, device=device) for t in (self.groups, self.shared)), most)
