"""A paged cache on the GPU for the tests of the operators that write and read one."""
import torch

DEV = "cuda"


class Paged:
    """`past[i]` tokens in the pages of sequence i and `new[i]` more in this step, pages dealt out of order.

    Places that hold no token of a sequence's past are NaN, pages that belong to nobody too."""

    def __init__(self, dtype, past, new, kv_heads, head_dim, page, prefix=0, heads_first=False, seed=0, spare=3, ragged=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.past, self.new, self.page, self.prefix = dtype, list(past), list(new), page, prefix
        batch = len(self.past)
        held = [-(-max(0, p + n) // page) for p, n in zip(self.past, self.new)]
        shared = -(-prefix // page)
        pages = shared + sum(held) + spare
        order = torch.randperm(pages, device=DEV, generator=g, dtype=torch.int32)
        width = max(held + [1])
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
        at = shared
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.prefix_table = order[:shared].clone()
        self.spare = order[at:].long()
        shape = (pages, kv_heads, page, head_dim) if heads_first else (pages, page, kv_heads, head_dim)

        def cache():
            c = torch.full(shape, float("nan"), device=DEV, dtype=dtype)
            return c.transpose(1, 2) if heads_first else c

        self.k, self.v = cache(), cache()
        self.lengths = torch.tensor(self.past, dtype=torch.int32, device=DEV)
        starts = [0]
        for n in self.new:
            starts.append(starts[-1] + n)
        self.starts, self.tokens = starts, starts[-1]
        ragged = any(n != 1 for n in self.new) if ragged is None else ragged
        self.offsets = torch.tensor(starts, dtype=torch.int32, device=DEV) if ragged else None

        def normal(n):
            return torch.randn(n, kv_heads, head_dim, device=DEV, generator=g).to(dtype)

        for c in (self.k, self.v):
            self.fill(c, self.prefix_table, 0, normal(prefix))
            for i, p in enumerate(self.past):
                self.fill(c, self.table[i], 0, normal(max(0, p)))

    def fill(self, cache, pages, first, rows):
        """Rows into places first, first + 1, ... of a list of pages."""
        if rows.shape[0]:
            place = torch.arange(first, first + rows.shape[0], device=DEV)
            cache[pages[place // self.page].long(), place % self.page] = rows

    def read(self, cache, pages, count):
        place = torch.arange(max(0, count), device=DEV)
        return cache[pages[place // self.page].long(), place % self.page]
