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
and is recorded in the device error word (mica_device_error: bad_page).
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import ops
from .int8_kernels import _CAPS, _launched, _supported

PAGES = (16, 32, 64, 128)      # tokens a page may hold


def _served(dev):
    c = _CAPS.get(dev.index)            # what _supported found the first time
    return bool(c.supported) if c is not None else _supported(dev)


def _cuda(name, *ts):
    dev = ts[0].device
    if dev.type != 'cuda':
        raise RuntimeError(f'{name}: CUDA tensors only (this library has no CPU path)')
    for t in ts[1:]:
        if t is not None and t.device != dev:
            raise RuntimeError(f'{name}: tensors on {dev} and {t.device}')
    if not _served(dev):
        raise RuntimeError(f'{name}: {dev} is not a B200 (sm_100)')


def _no_grad(name, *ts):
    if torch.is_grad_enabled() and True in [t.requires_grad for t in ts]:
        raise RuntimeError(f'{name}: no backward pass (call it under torch.no_grad())')


class Step:
    """The rows of one pass over the cache, described by device tensors (a captured graph serves new
    values in them):

      table int32 [B, P]   pages of each sequence      base int32 [B]   tokens already committed
      cu    int32 [B + 1]  rows cu[b] .. cu[b+1] belong to sequence b (cu[0] = 0; rows behind cu[B]
                           are padding)
      mask  int64 [N, W]   row sees node j of its own step when bit j % 64 of word j / 64 is set
                           (tree_mask); None: every row sees the rows before it and itself
      max_new              the most rows a sequence is expected to have (a hint for the kernel's
                           tile; the row count of the step when not given)

    Row i of sequence b sits at cache index base[b] + i and sees all of the committed tokens."""

    __slots__ = ('table', 'base', 'cu', 'mask', 'max_new')

    def __init__(self, table, base, cu, max_new: Optional[int] = None, mask=None):
        if table.dim() != 2 or base.dim() != 1 or cu.dim() != 1 or not (
                table.shape[0] == base.shape[0] == cu.shape[0] - 1) or table.shape[1] < 1:
            raise ValueError(f'Step: table {tuple(table.shape)}, base {tuple(base.shape)}, cu {tuple(cu.shape)}')
        if not table.dtype == base.dtype == cu.dtype == torch.int32:
            raise ValueError(f'Step: int32 tensors, not {table.dtype}, {base.dtype}, {cu.dtype}')
        if not table.is_contiguous():
            table = table.contiguous()
        if not base.is_contiguous() or not cu.is_contiguous():
            base, cu = base.contiguous(), cu.contiguous()
        if mask is not None:
            if mask.dim() != 2 or mask.dtype != torch.int64 or mask.shape[1] < 1:
                raise ValueError(f'Step: mask is int64 [rows, words], not {mask.dtype} {tuple(mask.shape)}')
            if not mask.is_contiguous():
                mask = mask.contiguous()
        if max_new is not None and max_new < 0:
            raise ValueError(f'Step: max_new {max_new}')
        self.table, self.base, self.cu, self.mask, self.max_new = table, base, cu, mask, max_new


def _pages_ok(name, k, v):
    if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride():
        raise ValueError(f'{name}: K pages {tuple(k.shape)} and V pages {tuple(v.shape)}')
    pages, kv, page, d = k.shape
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise RuntimeError(f'{name}: pages of {k.dtype} are not served (bf16)')
    if page not in PAGES or d not in (64, 128) or k.stride()[1:] != (page * d, d, 1) or kv < 1 or pages < 1 or (
            k.stride(0) < kv * page * d):
        raise ValueError(f'{name}: pages {tuple(k.shape)} with strides {k.stride()} (a page is [KV, page, D] '
                         f'contiguous, page in {PAGES}, D 64 or 128)')
    return kv, d


def append(qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, step: Step, heads: int, pos=None, eps: float = 1e-6):
    """Per-head RMSNorm of q and k, rotation by `pos` (int64 [N]; None: the cache index) and the write of K
    and V into the step's slots, in one pass over the QKV projection's output [N, (H + 2 KV) D] (q | k | v,
    unit column stride). Returns q [N, H D]; qkv is not changed. fp32, rounded to bf16 once
    (ops.qk_norm_rope keeps HF's rounding of every step). cos, sin bf16 [positions, D]."""
    kv, d = _pages_ok('append', k_pages, v_pages)
    n = qkv.shape[0]
    if qkv.dim() != 2 or heads < 1 or qkv.shape[1] != (heads + 2 * kv) * d or qkv.stride(1) != 1:
        raise ValueError(f'append: qkv {tuple(qkv.shape)} for {heads} + 2 x {kv} heads of {d}')
    if q_norm.shape != (d,) or k_norm.shape != (d,) or cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != d:
        raise ValueError(f'append: norms {tuple(q_norm.shape)}, {tuple(k_norm.shape)}, tables {tuple(cos.shape)}, '
                         f'{tuple(sin.shape)} for heads of {d}')
    if not (qkv.dtype == q_norm.dtype == k_norm.dtype == cos.dtype == sin.dtype == torch.bfloat16):
        raise RuntimeError('append: bf16 tensors only')
    if pos is not None and (pos.dtype != torch.int64 or pos.shape != (n,)):
        raise ValueError(f'append: pos is int64 [{n}], not {pos.dtype} {tuple(pos.shape)}')
    if not cos.is_contiguous() or not sin.is_contiguous() or cos.shape[0] < 1:
        raise ValueError('append: cos and sin are contiguous [positions, D]')
    _cuda('append', qkv, q_norm, k_norm, cos, sin, k_pages, v_pages, step.table, step.base, step.cu, pos)
    _no_grad('append', qkv, q_norm, k_norm)
    if n > 1 and (qkv.stride(0) < qkv.shape[1] or qkv.stride(0) % 8) or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    if pos is not None and not pos.is_contiguous():
        pos = pos.contiguous()
    q = ops.cache_append_do(qkv, q_norm.contiguous(), k_norm.contiguous(), cos, sin, k_pages, v_pages, step.table,
                            step.base, step.cu, heads, pos, float(eps))
    _launched()
    return q


def attention(q, k_pages, v_pages, step: Step, heads: int, scale: Optional[float] = None):
    """Grouped-query attention of the step's rows (appended before) over the cache: q [N, H D] (unit column
    stride, any row stride) -> [N, H D] bf16. Every row sees its sequence's committed tokens and, of its own
    step, what step.mask says. A row that sees nothing, and a padding row, is zero."""
    kv, d = _pages_ok('attention', k_pages, v_pages)
    n = q.shape[0]
    if q.dim() != 2 or heads < 1 or heads % kv or heads // kv > 128 or q.shape[1] != heads * d or q.stride(1) != 1:
        raise ValueError(f'attention: q {tuple(q.shape)} for {heads} heads of {d} over {kv} K/V heads')
    if q.dtype != torch.bfloat16:
        raise RuntimeError(f'attention: {q.dtype} is not served (bf16)')
    mask = step.mask
    if mask is not None and mask.shape[0] != n:
        raise ValueError(f'attention: mask of {mask.shape[0]} rows for {n}')
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float('inf'):
        raise ValueError(f'attention: scale {scale}')
    _cuda('attention', q, k_pages, v_pages, step.table, step.base, step.cu, mask)
    _no_grad('attention', q, k_pages, v_pages)
    if n > 1 and (q.stride(0) < q.shape[1] or q.stride(0) % 8) or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = ops.cache_attention_do(q, k_pages, v_pages, step.table, step.base, step.cu, mask, heads, scale,
                                 n if step.max_new is None else min(step.max_new, n))
    _launched()
    return out


def _pool_ok(name, pool):
    if pool.dim() < 2 or pool.shape[0] < 1 or not pool[0].is_contiguous() or pool.stride(0) < pool[0].numel() or (
            pool.data_ptr() % 16 or pool.stride(0) * pool.element_size() % 16
            or pool[0].numel() * pool.element_size() % 16 or pool[0].numel() == 0):
        raise ValueError(f'{name}: pool {tuple(pool.shape)} with strides {pool.stride()} (each page contiguous, whole '
                         '16-byte pieces)')


def copy_pages(pool, src: Sequence[int], dst: Sequence[int]) -> None:
    """pool[dst[i]] = pool[src[i]] for lists of page numbers, every layer of a page at once. No page may be
    written twice, or be both read and written. A captured graph keeps the lists."""
    _pool_ok('copy_pages', pool)
    if len(src) != len(dst):
        raise ValueError(f'copy_pages: {len(src)} pages onto {len(dst)}')
    both = set(dst)
    if len(both) != len(dst) or not both.isdisjoint(src):
        raise ValueError('copy_pages: a page is written twice, or read and written')
    if len(src) and not (0 <= min(src) and max(src) < pool.shape[0] and 0 <= min(dst) and max(dst) < pool.shape[0]):
        raise ValueError(f'copy_pages: a page outside the pool of {pool.shape[0]}')
    _cuda('copy_pages', pool)
    if len(src):
        ops.cache_copy_do(pool, src, dst)
        _launched()


def keep_tokens(pool, step: Step, keep, n_keep):
    """Of the step's rows, sequence b keeps keep[b, :n_keep[b]] (int32 [B, A], increasing; int32 [B]): their K
    and V move to the slots behind its committed tokens, in all layers of the pool [pages, layers, 2, KV, page,
    D]. Returns the new base int32 [B]. A sequence whose list is out of order or range is left as it was."""
    if pool.dim() != 6 or pool.shape[2] != 2 or pool.dtype != torch.bfloat16 or pool.shape[4] not in PAGES or (
            pool.shape[5] not in (64, 128)):
        raise ValueError(f'keep_tokens: pool {pool.dtype} {tuple(pool.shape)}')
    _pool_ok('keep_tokens', pool)
    b = step.base.shape[0]
    if keep.dim() != 2 or keep.shape[0] != b or n_keep.shape != (b,) or not keep.dtype == n_keep.dtype == torch.int32:
        raise ValueError(f'keep_tokens: keep {keep.dtype} {tuple(keep.shape)}, n_keep {n_keep.dtype} '
                         f'{tuple(n_keep.shape)} for {b} sequences')
    _cuda('keep_tokens', pool, step.table, step.base, step.cu, keep, n_keep)
    if b == 0 or keep.shape[1] == 0:
        return step.base.clone()
    new_base = ops.cache_keep_do(pool, step.table, step.base, step.cu, keep.contiguous(), n_keep.contiguous())
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

    def reserve(self, sids: Sequence[int], new: Sequence[int]) -> None:
        """Room for `new` more tokens of each sequence: pages are added, and a partly filled page that others
        share is copied (one launch for all). Raises OutOfPages, with nothing changed, when the pool is full."""
        if len(set(sids)) != len(sids) or len(sids) != len(new) or any(n < 0 for n in new):
            raise ValueError(f'reserve: {list(new)} tokens of sequences {list(sids)}')
        need, own = 0, {}
        for sid, n in zip(sids, new):
            pages, length = self._seqs[sid]
            need += max(0, -(-(length + n) // self.page) - len(pages))
            if n and length % self.page and len(pages) > length // self.page:
                p = pages[length // self.page]
                own[p] = own.get(p, 0) + 1
        # of the sequences that write a shared page, all take a copy unless no other one holds it
        need += sum(k if self._shares[p] > k else k - 1 for p, k in own.items())
        if need > len(self._free):
            raise OutOfPages(f'{need} pages needed, {len(self._free)} free')
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
        return Step(meta[:w].view(b, width), meta[w:w + b], meta[w + b:], max_new=max(new, default=0), mask=mask)

    def commit(self, sids: Sequence[int], new: Sequence[int]) -> None:
        """The first new[b] appended rows of each sequence become committed tokens."""
        for sid, n in zip(sids, new):
            pages, length = self._seqs[sid]
            if n < 0 or length + n > len(pages) * self.page:
                raise ValueError(f'commit: {n} tokens of sequence {sid}, {len(pages) * self.page - length} reserved')
        for sid, n in zip(sids, new):
            self._seqs[sid][1] += n
            self._trim(sid)

    def keep(self, sids: Sequence[int], step: Step, keep: Sequence[Sequence[int]]) -> None:
        """Commits the rows keep[b] (increasing) of the step's tree: the accepted tokens of each sequence."""
        if len(sids) != len(keep) or len(sids) != step.base.shape[0]:
            raise ValueError(f'keep: {len(keep)} lists for {len(sids)} sequences')
        for sid, rows in zip(sids, keep):
            pages, length = self._seqs[sid]
            if any(a >= b for a, b in zip(rows, rows[1:])) or (rows and (
                    rows[0] < 0 or length + rows[-1] >= len(pages) * self.page)):
                raise ValueError(f'keep: rows {list(rows)} of sequence {sid}')
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
