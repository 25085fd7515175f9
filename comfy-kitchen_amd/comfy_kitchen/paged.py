"""A key-value cache held in pages: which sequence owns which page, kept on the host; the rows
themselves are written, read and moved by `ck.paged_write` and `ck.paged_write_rope`, `ck.paged_attention` and
`ck.shared_attention`, `ck.paged_copy`.

A sequence is a list of page numbers and a length.  Pages are shared by counting: a fork owns its
parent's pages with it, and whoever first appends to a partly filled page that others own copies
its rows to a page of its own.  Nothing here waits for the GPU: a page that is given back may be
handed out at once, since the calls that still read it were queued on the stream before those
that write it again (use one stream for a cache, or order them as for any tensor).
"""
from __future__ import annotations

from collections.abc import Iterable, Sequence

import torch


class OutOfPages(RuntimeError):
    """The cache has fewer free pages than the call needs; the cache is as it was before."""


MOST_SPANS = 4096  # sequences and groups together that `ck.shared_attention` takes


class _Owner:
    __slots__ = ("length", "pages", "whole")

    def __init__(self, pages: list[int], length: int, whole: int | None = None):
        self.pages, self.length = pages, length
        self.whole = whole  # the pages before the first that was given back, or None: none was

    def held(self) -> int:
        """The pages that it begins with, up to the first that was given back."""
        return len(self.pages) if self.whole is None else self.whole


def _common(a: _Owner, b: _Owner) -> int:
    """With how many of the same pages both begin.  Two come to have a page at the same place by a fork, which gave them all
    that lie before it too, and these stay: so the first that differ are found by halving."""
    p, q = a.pages, b.pages
    same, most = 0, min(a.held(), b.held())
    if most and p[most - 1] == q[most - 1]:
        return most
    while same < most:
        middle = (same + most) // 2
        if p[middle] == q[middle]:
            same = middle + 1
        else:
            most = middle
    return same


class PagedKVCache:
    """K and V of `layers` layers, [layers, pages, page_size, kv_heads, head_dim], and their sequences.

    dtype: of the rows, f16 / bf16, or float8_e4m3fn, whose codes stand for value / k_scale and
    value / v_scale (floats; kept as one-element tensors on the device).
    head_dim: a multiple of 16; `attend` takes 64, 96, 128 and 256."""

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda",
                 k_scale: float | None = None, v_scale: float | None = None):
        if min(layers, pages, page_size, kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, page_size, kv_heads and head_dim must be positive")
        if dtype not in (torch.float16, torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"a cache holds float16, bfloat16 or float8_e4m3fn, not {dtype}")
        if dtype != torch.float8_e4m3fn and (k_scale is not None or v_scale is not None):
            raise ValueError(f"k_scale and v_scale are for a cache of float8_e4m3fn, not {dtype}")
        if head_dim % 16:
            raise ValueError(f"head_dim {head_dim} is not a multiple of 16, which `write` needs")
        if pages * page_size > 2 ** 31 - 1:
            raise ValueError(f"{pages} pages of {page_size} tokens: slots must fit 32 bits")
        shape = (layers, pages, page_size, kv_heads, head_dim)
        self.page_size = page_size
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.k_scale = None if k_scale is None else torch.tensor(float(k_scale), device=device)
        self.v_scale = None if v_scale is None else torch.tensor(float(v_scale), device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._owners = [0] * pages  # sequences that own a page
        self._sequences: dict[int, _Owner] = {}
        self._next = 0

    # ------------------------------------------------------------ bookkeeping
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __contains__(self, sequence: int) -> bool:
        return sequence in self._sequences

    def length(self, sequence: int) -> int:
        return self._sequences[sequence].length

    def pages(self, sequence: int) -> list[int]:
        """The sequence's page numbers in order; -1 for pages given back by `trim`."""
        return list(self._sequences[sequence].pages)

    def _next_free(self, count: int) -> list[int]:
        """The pages that `_take` of as many will take."""
        return self._free[:-count - 1:-1]

    def _take(self, count: int) -> list[int]:
        taken = [self._free.pop() for _ in range(count)]
        for page in taken:
            self._owners[page] = 1
        return taken

    def _drop(self, pages: Iterable[int]) -> None:
        for page in pages:
            if page >= 0:
                self._owners[page] -= 1
                if self._owners[page] == 0:
                    self._free.append(page)

    def _new(self, pages: list[int], length: int, whole: int | None = None) -> int:
        sequence, self._next = self._next, self._next + 1
        self._sequences[sequence] = _Owner(pages, length, whole)
        return sequence

    def _on_device(self, values, dtype=torch.int32) -> torch.Tensor:
        t = torch.tensor(values, dtype=dtype)
        if self.k.is_cuda and t.numel():
            t = t.pin_memory()
        return t.to(self.k.device, non_blocking=True)

    # ------------------------------------------------------------ sequences
    def add(self) -> int:
        """A new sequence of no tokens."""
        return self._new([], 0)

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens; nothing is copied until one of them is appended to."""
        owner = self._sequences[sequence]
        for page in owner.pages:
            if page >= 0:
                self._owners[page] += 1
        return self._new(list(owner.pages), owner.length, owner.whole)

    def free(self, sequence: int) -> None:
        """Forget a sequence; pages that no other owns can be handed out again."""
        self._drop(self._sequences.pop(sequence).pages)

    def append(self, sequences: Sequence[int], counts: Sequence[int] | int = 1) -> torch.Tensor:
        """Places for `counts` new tokens of each of the sequences (distinct): their slots, int32 on
        the device, sequence by sequence, for `write` in every layer."""
        counts = [counts] * len(sequences) if isinstance(counts, int) else list(counts)
        if len(set(sequences)) != len(sequences) or len(counts) != len(sequences) or min(counts, default=0) < 0:
            raise ValueError("append takes distinct sequences and a count of new tokens for each")
        size, need = self.page_size, 0
        shared = []  # whether the sequence's partly filled last page must be copied first
        claims: dict[int, int] = {}  # owners of such pages that leave them in this call
        for sequence, count in zip(sequences, counts):
            owner = self._sequences[sequence]
            copy = False
            if count and owner.length % size:
                page = owner.pages[-1]
                copy = self._owners[page] - claims.get(page, 0) > 1  # the last owner keeps it
                claims[page] = claims.get(page, 0) + copy
            shared.append(copy)
            need += -(-(owner.length + count) // size) - len(owner.pages) + copy
        if need > len(self._free):
            raise OutOfPages(f"append needs {need} pages, {len(self._free)} are free")
        # What the device is asked for may be refused, so it comes before any change here.
        fresh = iter(self._next_free(need))
        src, dst, slots, after = [], [], [], []
        for sequence, count, copy in zip(sequences, counts, shared):
            owner = self._sequences[sequence]
            first, fill = divmod(owner.length, size)
            pages = owner.pages[first:]  # those that the new tokens are in
            if copy:
                old, new = pages[0], next(fresh)
                src.extend(range(old * size, old * size + fill))
                dst.extend(range(new * size, new * size + fill))
                pages = [new]
            while len(pages) * size < fill + count:
                pages.append(next(fresh))
            after.append((owner, first, pages, owner.length + count, copy))
            for page in pages:
                begin, end = page * size + fill, page * size + min(size, fill + count)
                slots.extend(range(begin, end))
                fill, count = 0, count - (end - begin)
        placed = self._on_device(slots)
        if src:
            self._copy(src, dst)
        self._take(need)
        for owner, first, pages, end, copy in after:
            if copy:
                self._drop(owner.pages[first:])
            owner.pages[first:], owner.length = pages, end
        return placed

    def trim(self, sequence: int, window: int, sinks: int = 0) -> int:
        """Give back the pages that hold neither one of the last `window` tokens nor one of the first
        `sinks`, which attention with that window and sinks does not read: the pages' number."""
        owner, size = self._sequences[sequence], self.page_size
        if window < 1 or sinks < 0:
            raise ValueError("trim takes a window of at least one token and no negative sinks")
        first, last = -(-sinks // size), max(0, owner.length - window) // size
        gone = [i for i in range(first, last) if owner.pages[i] >= 0]
        self._drop(owner.pages[i] for i in gone)
        for i in gone:
            owner.pages[i] = -1
        if gone:
            owner.whole = min(gone[0], owner.held())
        return len(gone)

    def compact(self, sequence: int, keep: Sequence[int]) -> None:
        """Keep only the tokens at the ascending positions `keep`, moved together in fresh pages."""
        owner, size = self._sequences[sequence], self.page_size
        keep = keep.tolist() if isinstance(keep, torch.Tensor) else list(keep)
        if any(b <= a for a, b in zip(keep, keep[1:])) or (keep and not 0 <= keep[0] <= keep[-1] < owner.length):
            raise ValueError(f"compact takes ascending positions in 0..{owner.length - 1}")
        if any(owner.pages[t // size] < 0 for t in keep):
            raise ValueError("compact: a kept token's page was given back by trim")
        need = -(-len(keep) // size)
        if need > len(self._free):
            raise OutOfPages(f"compact needs {need} pages, {len(self._free)} are free")
        new = self._next_free(need)
        if keep:
            self._copy([owner.pages[t // size] * size + t % size for t in keep],
                       [new[i // size] * size + i % size for i in range(len(keep))])
        self._take(need)
        self._drop(owner.pages)
        owner.pages, owner.length, owner.whole = new, len(keep), None

    # ------------------------------------------------------------ device calls
    def _copy(self, src: list[int], dst: list[int]) -> None:
        import comfy_kitchen as ck

        ck.paged_copy(self.k, self.v, self._on_device(src), self._on_device(dst))

    def tables(self, sequences: Sequence[int]) -> tuple[torch.Tensor, torch.Tensor]:
        """(page_table, lengths) of the sequences for `attend`, int32 on the device."""
        owners = [self._sequences[s] for s in sequences]
        width = max((len(o.pages) for o in owners), default=0)
        rows = [o.pages + [-1] * (width - len(o.pages)) for o in owners]
        table = self._on_device(rows).reshape(len(owners), width)
        return table, self._on_device([o.length for o in owners])

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor) -> None:
        """Store [T, kv_heads, head_dim] keys and values of one layer in the slots of `append`."""
        import comfy_kitchen as ck

        ck.paged_write(key, value, self.k[layer], self.v[layer], slots, self.k_scale, self.v_scale)

    def write_rope(self, layer: int, q: torch.Tensor, key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                   rates: torch.Tensor, slots: torch.Tensor, interleaved: bool = True, magnitude: float = 1.0,
                   keep_key: bool = False) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
        """`write` of keys turned to their positions, and queries with them: `ck.paged_write_rope` on one layer."""
        import comfy_kitchen as ck

        return ck.paged_write_rope(q, key, value, positions, rates, self.k[layer], self.v[layer], slots, interleaved,
                                   magnitude, self.k_scale, self.v_scale, keep_key)

    def groups(self, sequences: Sequence[int], least_bytes: int | None = None) -> tuple[torch.Tensor, torch.Tensor] | None:
        """(groups, shared) of the sequences in this order for `attend`, int32 on the device: neighbours that begin with the
        same pages (forks of one sequence) are a group.  None where reading common rows once saves less than
        `least_bytes` of K and V a layer, and where there are more sequences and groups than `ck.shared_attention` takes
        (MOST_SPANS).
        By default that is 80 MB, from where on `ck.shared_attention` is the faster (4 sequences of 40 heads over 8: 22 us
        for 23 at 8192 common tokens of 16 bits, 96 MB; 16 for 15 at 2048, 36 for 83 at 32768), and 400 MB by the layers, for the
        host's time of this call, some 0.05 to 0.08 ms for 4 to 64 sequences, hardly more for many tokens."""
        owners = [self._sequences[s] for s in sequences]
        near = [_common(a, b) for a, b in zip(owners, owners[1:])]  # of each and the next
        row = 2 * self.k.shape[3] * self.k.shape[4] * self.k.element_size()
        least = max((80 << 20) + (400 << 20) / self.k.shape[0] if least_bytes is None else least_bytes, 1)
        if sum(near) * self.page_size * row < least:  # (more than any groups save)
            return None
        starts, shared = [], []
        first = 0  # pages that the group so far begins with
        for i, owner in enumerate(owners):
            same = min(first, near[i - 1]) if i else 0
            if same:
                members = i - starts[-1]
                after = near[i] if i + 1 < len(owners) else 0
                # it would cost the others more than it gains, or gains far more with those behind it
                if members * same < (members - 1) * first or (2 * same < after and members * same < after):
                    same = 0
            if same:
                first = same
            else:
                if starts:
                    shared.append(first)
                starts.append(i)
                first = owner.held()
        if starts:
            shared.append(first)
        starts.append(len(owners))
        tokens = [min(n * self.page_size, min(o.length for o in owners[a:b])) for n, a, b in zip(shared, starts, starts[1:])]
        saved = sum((b - a - 1) * n for n, a, b in zip(tokens, starts, starts[1:])) * row
        if saved < least:
            return None
        if len(owners) + len(tokens) > MOST_SPANS:  # neighbours that share nothing are then one group, of no common tokens
            alone = [b - a == 1 for a, b in zip(starts, starts[1:])]
            kept = [i for i in range(len(alone)) if not (i and alone[i] and alone[i - 1])]
            tokens = [0 if alone[i] else tokens[i] for i in kept]
            starts = [starts[i] for i in kept] + starts[-1:]
            if len(owners) + len(tokens) > MOST_SPANS:
                return None
        return self._on_device(starts), self._on_device(tokens)

    def attend(self, layer: int, q: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               scale: float | None = None, window: int = 0, sinks: int = 0,
               groups: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
        """`ck.paged_attention` of q [B, heads, head_dim] on one layer, or, with what `groups` gives, `ck.shared_attention`."""
        import comfy_kitchen as ck

        if groups is not None:
            if window:
                raise ValueError("attend takes groups or a window, not both")
            return ck.shared_attention(q, self.k[layer], self.v[layer], page_table, lengths, *groups, scale, self.k_scale,
                                       self.v_scale)
        return ck.paged_attention(q, self.k[layer], self.v[layer], page_table, lengths, scale, window, sinks,
                                  self.k_scale, self.v_scale)
