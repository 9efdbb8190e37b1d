"""Paged K/V cache: kept contexts, and the steps of new tokens that run over them.

The prefill (mica_b200.prefill) keeps nothing between requests. Here a context's K and V stay in
pages, so several questions about one document, or answers of several tokens, run only their own
rows (mica_b200.answers puts them together). The reference keeps whole-prefix states instead
(v0.5/serving/lib/fork.py, prefill_engine.py ForkGraphs).

    PagedCache            the pool [pages, layers, 2, KV, page, D] bf16 and its sequences: open, fork
                          (pages shared until written), reserve, commit, keep, free, compact
    Step                  the rows of one pass: which sequence they belong to and what they see
    append(...)           q/k norm + rotation, K and V written into their pages, q returned
    attention(...)        the step's rows over the cache: causal, or a tree by its mask
    copy_pages(...)       pool[dst] = pool[src]
    keep_tokens(...)      accepted rows of a step move together behind the context
    tree_mask(parents)    mask words of trees given by their parent lists

Errors follow fused_kernels: ValueError for arguments that fit no call, RuntimeError for what the
kernels do not serve (a CPU tensor, another dtype, another GPU). There is no CPU branch. What a
step's tables hold is on the device: a base, page number or position out of range touches nothing
and is recorded in the device error word (mica_device_error: bad_page), as is a cu that passes the
rows (those that are there are served) or runs backwards (attention is zero).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _native as N
from . import ops  # noqa: F401  (registers torch.ops.mica.*)
from .int8_kernels import _launched

PAGES = (16, 32, 64, 128)      # tokens a page may hold


class Step:
    """The rows of one pass over the cache, described by device tensors, taken as they are, whatever their strides
    (a captured graph serves new values in them):

      table int32 [B, P]   pages of each sequence      base int32 [B]   tokens already committed
      cu    int32 [B + 1]  rows cu[b] .. cu[b+1] belong to sequence b (cu[0] = 0; rows behind cu[B]
                           are padding)
      mask  int64 [N, W]   row sees node j of its own step when bit j % 64 of word j / 64 is set
                           (tree_mask); None: every row sees the rows before it and itself
      max_new              the most rows a sequence is expected to have (a hint for the kernel's
                           tile; the row count of the step when not given)

    Row i of sequence b sits at cache index base[b] + i and sees all of the committed tokens."""

    __slots__ = ('table', 'base', 'cu', 'mask', 'max_new', 'rows', 'lengths')

    def __init__(self, table, base, cu, max_new: Optional[int] = None, mask=None):
        if table.dim() != 2 or base.dim() != 1 or cu.dim() != 1 or not (
                table.shape[0] == base.shape[0] == cu.shape[0] - 1) or table.shape[1] < 1:
            raise ValueError(f'Step: table {tuple(table.shape)}, base {tuple(base.shape)}, cu {tuple(cu.shape)}')
        if not table.dtype == base.dtype == cu.dtype == torch.int32:
            raise ValueError(f'Step: int32 tensors, not {table.dtype}, {base.dtype}, {cu.dtype}')
        if mask is not None and (mask.dim() != 2 or mask.dtype != torch.int64 or mask.shape[1] < 1):
            raise ValueError(f'Step: mask is int64 [rows, words], not {mask.dtype} {tuple(mask.shape)}')
        if max_new is not None and max_new < 0:
            raise ValueError(f'Step: max_new {max_new}')
        self.table, self.base, self.cu, self.mask, self.max_new = table, base, cu, mask, max_new
        self.rows = None               # rows of each sequence and its committed tokens then, where the host
        self.lengths = None            # knows them (PagedCache.step)


def append(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, step: Step, heads: int, pos=None, eps: float = 1e-6):
    """Per-head RMSNorm of q and k, rotation by `pos` (int64 [N]; None: the cache index) and the write of K
    and V into the step's slots, in one pass over the QKV projection's output [N, (H + 2 KV) D] (q | k | v,
    unit column stride). Returns q [N, H D]; qkv is not changed. fp32, rounded to bf16 once
    (ops.qk_norm_rope keeps HF's rounding of every step). cos, sin bf16 [positions, D]. Sequences of a step
    have slots of their own: a page that two of them write is the caller's mistake (PagedCache copies it first)."""
    q = N.calls().append(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, step.table, step.base, step.cu, heads, pos, eps)
    _launched()
    return q


def attention(q, k_pages, v_pages, step: Step, heads: int, scale: Optional[float] = None):
    """Grouped-query attention of the step's rows (appended before) over the cache: q [N, H D] (unit column
    stride, any row stride) -> [N, H D] bf16. Every row sees its sequence's committed tokens and, of its own
    step, what step.mask says. A row that sees nothing, and a padding row, is zero."""
    out = N.calls().attention(q, k_pages, v_pages, step.table, step.base, step.cu, step.mask, heads, scale, step.max_new)
    _launched(2)
    return out


def copy_pages(pool, src: Sequence[int], dst: Sequence[int]) -> None:
    """pool[dst[i]] = pool[src[i]] for lists of page numbers, every layer of a page at once. No page may be
    written twice, or be both read and written. A captured graph keeps the lists."""
    N.calls().copy_pages(pool, src, dst)
    if len(src):
        _launched()


def keep_tokens(pool, step: Step, keep, n_keep):
    """Of the step's rows, sequence b keeps keep[b, :n_keep[b]] (int32 [B, A], increasing; int32 [B]): their K
    and V move to the slots behind its committed tokens, in all layers of the pool [pages, layers, 2, KV, page,
    D]. Returns the new base int32 [B]. A sequence whose list is out of order or range is left as it was."""
    new_base = N.calls().keep_tokens(pool, step.table, step.base, step.cu, keep, n_keep)
    _launched()
    return new_base


def tree_mask(parents: Sequence[Sequence[int]], device=None):
    """Mask words int64 [N, W] of trees, one parent list per sequence: parents[b][i] is the node above node i
    (before it in the list), -1 for a child of the context. A node sees its ancestors and itself."""
    most = max((len(p) for p in parents), default=0)
    words = max(1, -(-most // 64))
    rows = []
    for tree in parents:
        seen = []
        for i, p in enumerate(tree):
            if not -1 <= p < i:
                raise ValueError(f'tree_mask: node {i} hangs from {p}, which is not before it')
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
        for m in seen:
            w = [m >> 64 * k & (1 << 64) - 1 for k in range(words)]
            rows.append([x - (1 << 64) if x >> 63 else x for x in w])
    t = torch.tensor(rows, dtype=torch.int64).view(len(rows), words)
    return t if device is None else t.to(device)


class OutOfPages(RuntimeError):
    """The pool has too few free pages for a reservation; nothing was reserved."""


class PagedCache:
    """K and V of kept contexts: a pool of pages and the sequences that use them.

    Page numbers, lengths and shares are host state; the pool is written by append, copy_pages and
    keep_tokens on the current stream, so one cache is used from one stream at a time. A page that several
    sequences share is copied when one of them is about to write it."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, pages: int, page: int = 64, device='cuda'):
        if page not in PAGES or head_dim not in (64, 128) or layers < 1 or kv_heads < 1 or pages < 1:
            raise ValueError(f'PagedCache: {pages} pages of {page} tokens, {layers} layers, {kv_heads} heads of '
                             f'{head_dim} (page in {PAGES}, head_dim 64 or 128)')
        self.page = page
        self.pool = torch.zeros(pages, layers, 2, kv_heads, page, head_dim, dtype=torch.bfloat16, device=device)
        self._free = list(range(pages - 1, -1, -1))       # lowest page last: taken first
        self._shares = [0] * pages
        self._seqs: dict[int, list] = {}                   # id -> [pages, length]
        self._next = 0

    # ---- sequences ---------------------------------------------------------------------
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int):
        """K and V pages [pages, KV, page, D] of layer i (views of the pool)."""
        return self.pool[:, i, 0], self.pool[:, i, 1]

    def open(self) -> int:
        """A new empty sequence."""
        sid = self._next
        self._next += 1
        self._seqs[sid] = [[], 0]
        return sid

    def length(self, sid: int) -> int:
        return self._seqs[sid][1]

    def pages_of(self, sid: int) -> list:
        return list(self._seqs[sid][0])

    def fork(self, sid: int) -> int:
        """A new sequence with the same committed tokens: its pages are shared, none is copied yet."""
        pages, length = self._seqs[sid]
        used = pages[:-(-length // self.page)]
        for p in used:
            self._shares[p] += 1
        new = self.open()
        self._seqs[new] = [list(used), length]
        return new

    def free(self, sid: int) -> None:
        """Ends a sequence; pages that no other one shares return to the pool."""
        for p in self._seqs.pop(sid)[0]:
            self._release(p)

    def _release(self, p: int) -> None:
        self._shares[p] -= 1
        if self._shares[p] == 0:
            self._free.append(p)

    def _take(self) -> int:
        p = self._free.pop()
        self._shares[p] = 1
        return p

    def _fits(self, sequences, free: int) -> None:
        """Raises OutOfPages when room for n more tokens of each (pages, length, n) takes more than `free` pages."""
        need, own = 0, {}
        for pages, length, n in sequences:
            need += max(0, -(-(length + n) // self.page) - len(pages))
            if n and length % self.page and len(pages) > length // self.page:
                p = pages[length // self.page]
                own[p] = own.get(p, 0) + 1
        # of the sequences that write a shared page, all take a copy unless no other one holds it
        need += sum(k if self._shares[p] > k else k - 1 for p, k in own.items())
        if need > free:
            raise OutOfPages(f'{need} pages needed, {free} free')

    def fits_after(self, sids: Sequence[int], kept: Sequence[int], new: Sequence[int]) -> None:
        """Raises OutOfPages when `new` more tokens of each sequence would not fit once kept[b] reserved rows of it
        are committed, which gives the other rows' pages back. Nothing is changed."""
        free, after = len(self._free), []
        for sid, k, n in zip(sids, kept, new):
            pages, length = self._seqs[sid]
            held = pages[:-(-(length + k) // self.page)]
            free += len(pages) - len(held)
            after.append((held, length + k, n))
        self._fits(after, free)

    def reserve(self, sids: Sequence[int], new: Sequence[int]) -> None:
        """Room for `new` more tokens of each sequence: pages are added, and a partly filled page that others
        share is copied (one launch for all). Raises OutOfPages, with nothing changed, when the pool is full."""
        if len(set(sids)) != len(sids) or len(sids) != len(new) or any(n < 0 for n in new):
            raise ValueError(f'reserve: {list(new)} tokens of sequences {list(sids)}')
        self._fits([(*self._seqs[sid], n) for sid, n in zip(sids, new)], len(self._free))
        src, dst = [], []
        for sid, n in zip(sids, new):
            pages, length = self._seqs[sid]
            at = length // self.page
            if n and length % self.page and len(pages) > at and self._shares[pages[at]] > 1:
                p = self._take()
                src.append(pages[at])
                dst.append(p)
                self._release(pages[at])
                pages[at] = p
            while len(pages) * self.page < length + n:
                pages.append(self._take())
        if src:
            copy_pages(self.pool, src, dst)

    def step(self, sids: Sequence[int], new: Sequence[int], mask=None) -> Step:
        """Reserves room and describes a pass of new[b] rows of each sequence, in order. One pinned copy."""
        self.reserve(sids, new)
        b = len(sids)
        width = max([len(self._seqs[s][0]) for s in sids] + [1])
        flat = []
        for s in sids:
            pages = self._seqs[s][0]
            flat += pages + [0] * (width - len(pages))
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        meta = torch.tensor(flat + [self._seqs[s][1] for s in sids] + cu, dtype=torch.int32)
        meta = meta.pin_memory().to(self.pool.device, non_blocking=True)
        w = b * width
        s = Step(meta[:w].view(b, width), meta[w:w + b], meta[w + b:], max_new=max(new, default=0), mask=mask)
        s.rows, s.lengths = list(new), [self._seqs[i][1] for i in sids]
        return s

    def commit(self, sids: Sequence[int], new: Sequence[int]) -> None:
        """The first new[b] appended rows of each sequence become committed tokens."""
        if len(set(sids)) != len(sids) or len(sids) != len(new):
            raise ValueError(f'commit: {list(new)} tokens of sequences {list(sids)}')
        for sid, n in zip(sids, new):
            pages, length = self._seqs[sid]
            if n < 0 or length + n > len(pages) * self.page:
                raise ValueError(f'commit: {n} tokens of sequence {sid}, {len(pages) * self.page - length} reserved')
        for sid, n in zip(sids, new):
            self._seqs[sid][1] += n
            self._trim(sid)

    def keep(self, sids: Sequence[int], step: Step, keep: Sequence[Sequence[int]]) -> None:
        """Commits the rows keep[b] (increasing) of the step's tree: the accepted tokens of each sequence."""
        if len(set(sids)) != len(sids) or len(sids) != len(keep) or step.rows is None or len(sids) != len(step.rows):
            raise ValueError(f'keep: {len(keep)} lists for {len(sids)} sequences of a step of this cache')
        if step.lengths is not None and step.lengths != [self._seqs[sid][1] for sid in sids]:
            raise ValueError(f'keep: sequences {list(sids)} are not as they were when the step was described')
        for sid, rows, n in zip(sids, keep, step.rows):
            pages, length = self._seqs[sid]
            if any(a >= b for a, b in zip(rows, rows[1:])) or (rows and (rows[0] < 0 or rows[-1] >= n)) or (
                    length + n > len(pages) * self.page):
                raise ValueError(f'keep: rows {list(rows)} of {n} of sequence {sid}')
        most = max((len(r) for r in keep), default=0)
        if any(list(r) != list(range(len(r))) for r in keep):
            flat = [list(r) + [0] * (most - len(r)) for r in keep]
            meta = torch.tensor([x for r in flat for x in r] + [len(r) for r in keep], dtype=torch.int32)
            meta = meta.pin_memory().to(self.pool.device, non_blocking=True)
            cut = most * len(sids)
            keep_tokens(self.pool, step, meta[:cut].view(len(sids), most), meta[cut:])
        self.commit(sids, [len(r) for r in keep])

    def _trim(self, sid: int) -> None:
        """Returns the pages behind the committed tokens to the pool."""
        pages, length = self._seqs[sid]
        while len(pages) > -(-length // self.page):
            self._release(pages.pop())

    def compact(self) -> int:
        """Moves the used pages to the front of the pool, so that its end is free; returns the first page behind
        them. Steps described before are out of date."""
        used = [p for p, n in enumerate(self._shares) if n]
        last = len(used)
        holes = [p for p in range(last) if self._shares[p] == 0]
        moved = dict(zip([p for p in used if p >= last], holes))
        if moved:
            copy_pages(self.pool, list(moved), list(moved.values()))
            for p, q in moved.items():
                self._shares[q], self._shares[p] = self._shares[p], 0
            for entry in self._seqs.values():
                entry[0] = [moved.get(p, p) for p in entry[0]]
        self._free = [p for p in range(len(self._shares) - 1, -1, -1) if self._shares[p] == 0]
        return last
