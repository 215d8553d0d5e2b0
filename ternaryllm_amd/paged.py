"""PagedCache: the keys and values of many sequences in pages of one pool, for serving sequences of different lengths in one pass
(`TernaryLlamaDecoder.extend`).  The reference keeps one contiguous cache for a batch (the `transformers` Cache that
ternaryLLM_GPU/TernaryLLM/TernaryAttn.py:96-98 updates); here a sequence holds the pages that its tokens need, and gives them back.
Sequences that go on from the same tokens (`fork`) hold the pages of those in common, and are attended together (`prefix`).

The pages are on the GPU and the kernels do the work (`ops.rope_to_pages`, `ops.paged_attention`, `ops.read_pages`); what a sequence
holds is kept on the host."""
import torch

from . import ops


_LEAST_SHARED = 64                               # tokens, for a group to be one


def _in_common(a, b):
    """How many of the first items of two lists are the same."""
    low, high = 0, min(len(a), len(b))
    while low < high:
        middle = (low + high + 1) // 2
        low, high = (middle, high) if a[low:middle] == b[low:middle] else (low, middle - 1)
    return low


class PagedCache:
    """`pages` pages of `page_size` tokens (a power of two, 16 to 1024) in each of `layers` layers, dtype float16 or float8_e4m3fn (half the
    memory and half the bytes of a decode step: 8 bits a value and a power of two for each row of a head)."""

    def __init__(self, layers, pages, kv_heads, head_dim, page_size=64, dtype=torch.float16, device="cuda"):
        if dtype not in (torch.float16, torch.float8_e4m3fn):
            raise ValueError(f"pages are float16 or float8_e4m3fn, not {dtype}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size={page_size} is not a power of two from 16 to 1024")
        if layers < 1 or pages < 1 or kv_heads < 1 or head_dim < 16 or head_dim % 16:
            raise ValueError("layers, pages and kv_heads must be positive, head_dim a multiple of 16")
        self.page_size, self.device = page_size, torch.device(device)
        self.layers, self.kv_heads, self.head_dim = layers, kv_heads, head_dim
        shape = (layers, 2, pages, kv_heads, page_size, head_dim)
        self._rows = torch.zeros(shape, dtype=torch.float16 if dtype == torch.float16 else torch.uint8, device=device)
        self._exponents = None if dtype == torch.float16 else torch.zeros(shape[:-1], dtype=torch.uint8, device=device)
        self.dtype = dtype
        self._free = list(range(pages - 1, -1, -1))
        self._holders = [0] * pages              # sequences that hold a page
        self._forks = 0                          # pages held more than once, counted each time
        self._sequences = {}                     # number -> (pages, length)
        self._next = 0

    @property
    def free_pages(self):
        return len(self._free)

    def layer(self, index):
        """The pages of one layer as the operators take them."""
        rows = self._rows[index].view(self.dtype)
        return ops.Pages(rows[0], rows[1], *(() if self._exponents is None else self._exponents[index]))

    def open(self):
        """A new sequence without tokens; returns its number."""
        self._sequences[self._next] = ([], 0)
        self._next += 1
        return self._next - 1

    def fork(self, sequence):
        """A new sequence that goes on from the tokens of another; returns its number.  The two hold the pages of those in common, and each gets a copy of the
        last one when it needs room there."""
        held, length = self._sequences[sequence]
        for p in held:
            self._holders[p] += 1
        self._forks += len(held)
        self._sequences[self._next] = (list(held), length)
        self._next += 1
        return self._next - 1

    def _give_back(self, pages):
        for p in reversed(pages):
            self._holders[p] -= 1
            if self._holders[p] == 0:
                self._free.append(p)
            else:
                self._forks -= 1

    def close(self, sequence):
        """Gives a sequence's pages back."""
        held, _ = self._sequences.pop(sequence)
        self._give_back(held)

    def length(self, sequence):
        return self._sequences[sequence][1]

    def truncate(self, sequence, length):
        """Forgets a sequence's tokens from `length` on (rejected ones, say) and gives back the pages that only they were in."""
        held, now = self._sequences[sequence]
        if not 0 <= length <= now:
            raise ValueError(f"a sequence of {now} tokens cannot be cut to {length}")
        keep = -(-length // self.page_size)
        self._give_back(held[keep:])
        self._sequences[sequence] = (held[:keep], length)

    def extend(self, chunks):
        """Makes room for new tokens, chunks = [(sequence, how many), ...], each sequence once, and returns the ops.PageBatch of a pass over
        them.  A page that tokens go into and that other sequences hold too is copied first, on the current stream.  Without pages enough RuntimeError is
        raised; nothing changes where anything is."""
        numbers = [s for s, _ in chunks]
        if not chunks or len(set(numbers)) < len(numbers) or any(n < 0 for _, n in chunks) or any(s not in self._sequences for s in numbers):
            raise ValueError("chunks are of open sequences, each named once, and not negative")
        more = [-(-(self._sequences[s][1] + n) // self.page_size) - len(self._sequences[s][0]) for s, n in chunks]
        copied, left_with = {}, {}               # sequence -> the page of which it needs a copy; page -> its holders but for those
        for s, n in chunks if self._forks else ():
            held, length = self._sequences[s]
            if n > 0 and length % self.page_size:
                p = held[length // self.page_size]
                if left_with.get(p, self._holders[p]) > 1:
                    copied[s] = p
                    left_with[p] = left_with.get(p, self._holders[p]) - 1
        needed = sum(more) + len(copied)
        if needed > len(self._free):
            raise RuntimeError(f"{needed} pages needed, {len(self._free)} free")
        after, left, copies = {}, len(self._free), []
        for (s, n), count in zip(chunks, more):
            held, length = self._sequences[s]
            if s in copied:
                at = length // self.page_size
                copies.append((copied[s], self._free[left - 1]))
                held, left = held[:at] + [self._free[left - 1]] + held[at + 1:], left - 1
            after[s] = (held + self._free[left - count:left][::-1], length + n)
            left -= count
        batch = self._batch(numbers, [n for _, n in chunks], after)
        if copies:
            old, new = torch.tensor(copies, device=self.device).unbind(1)
            for t in (self._rows, self._exponents):
                if t is not None:
                    t[:, :, new] = t[:, :, old]
        for p in self._free[left:]:
            self._holders[p] = 1
        for p in copied.values():
            self._holders[p] -= 1
            self._forks -= 1
        self._sequences.update(after)
        del self._free[left:]
        return batch

    def prefix(self, chunks):
        """The ops.PagePrefix of a pass over chunks (as extend was told of them), or None where no two neighbours among them have tokens in common that are worth
        it: sequences that begin with the same pages, side by side, are a group, as long as what all of them share is at least half of what the first two do."""
        if not self._forks or len(chunks) < 2:
            return None
        size = self.page_size
        groups, shared = [], [0] * len(chunks)
        held = [self._sequences[s][0] for s, _ in chunks]
        front = [(self._sequences[s][1] - n) // size for s, n in chunks]            # whole pages in front of a chunk's rows
        first = 0
        while first < len(chunks):
            common, last = front[first], first + 1
            while last < len(chunks) and common * size >= _LEAST_SHARED:
                both = min(common, front[last])
                if held[last][:both] != held[first][:both]:
                    both = _in_common(held[first][:both], held[last])
                if both * size < _LEAST_SHARED or (last > first + 1 and 2 * both < common):
                    break
                common, last = both, last + 1
            if last > first + 1:
                groups.append((first, last))
                shared[first:last] = [common * size] * (last - first)
            first = last
        if not groups:
            return None
        # (what stands between groups is a group by itself, of which nothing is shared)
        edges = sorted({0, len(chunks), *(e for g in groups for e in g)})
        both = torch.tensor(edges + shared, dtype=torch.int32).to(self.device)
        return ops.PagePrefix(both[:len(edges)], both[len(edges):], max(shared))

    def whole(self, sequences):
        """The ops.PageBatch whose rows are all tokens of these sequences (what ops.read_pages reads)."""
        return self._batch(sequences, [self._sequences[s][1] for s in sequences], self._sequences)

    def _batch(self, numbers, rows, sequences):
        held, lengths = zip(*(sequences[s] for s in numbers))
        columns = max(1, max(len(h) for h in held))
        starts = [0]
        for n in rows:
            starts.append(starts[-1] + n)
        # one copy to the device: the table, the starts, the lengths
        flat = [p for h in held for p in h + [0] * (columns - len(h))] + starts + list(lengths)
        both = torch.tensor(flat, dtype=torch.int32).to(self.device)
        table, starts, lengths = both.split((len(numbers) * columns, len(numbers) + 1, len(numbers)))
        return ops.PageBatch(table.view(len(numbers), columns), starts, lengths, max(rows))


__all__ = ["PagedCache"]
