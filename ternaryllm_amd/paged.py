"""PagedCache: the keys and values of many sequences in pages of one pool, for serving sequences of different lengths in one pass
(`TernaryLlamaDecoder.extend`).  The reference keeps one contiguous cache for a batch (the `transformers` Cache that
ternaryLLM_GPU/TernaryLLM/TernaryAttn.py:96-98 updates); here a sequence holds the pages that its tokens need, and gives them back.

The pages are on the GPU and the kernels do the work (`ops.rope_to_pages`, `ops.paged_attention`, `ops.read_pages`); what a sequence
holds is kept on the host."""
import torch

from . import ops


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

    def close(self, sequence):
        """Gives a sequence's pages back."""
        held, _ = self._sequences.pop(sequence)
        self._free.extend(reversed(held))

    def length(self, sequence):
        return self._sequences[sequence][1]

    def truncate(self, sequence, length):
        """Forgets a sequence's tokens from `length` on (rejected ones, say) and gives back the pages that only they were in."""
        held, now = self._sequences[sequence]
        if not 0 <= length <= now:
            raise ValueError(f"a sequence of {now} tokens cannot be cut to {length}")
        keep = -(-length // self.page_size)
        self._free.extend(reversed(held[keep:]))
        self._sequences[sequence] = (held[:keep], length)

    def extend(self, chunks):
        """Makes room for new tokens, chunks = [(sequence, how many), ...], each sequence once, and returns the ops.PageBatch of a pass over
        them.  Without pages enough RuntimeError is raised; nothing changes where anything is."""
        numbers = [s for s, _ in chunks]
        if not chunks or len(set(numbers)) < len(numbers) or any(n < 0 for _, n in chunks) or any(s not in self._sequences for s in numbers):
            raise ValueError("chunks are of open sequences, each named once, and not negative")
        more = [-(-(self._sequences[s][1] + n) // self.page_size) - len(self._sequences[s][0]) for s, n in chunks]
        if sum(more) > len(self._free):
            raise RuntimeError(f"{sum(more)} pages needed, {len(self._free)} free")
        after, left = {}, len(self._free)
        for (s, n), count in zip(chunks, more):
            held, length = self._sequences[s]
            after[s] = (held + self._free[left - count:left][::-1], length + n)
            left -= count
        batch = self._batch(numbers, [n for _, n in chunks], after)
        self._sequences.update(after)
        del self._free[left:]
        return batch

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
