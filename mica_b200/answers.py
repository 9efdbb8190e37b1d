"""Scores answers of several tokens over kept contexts, on the W8A8 decoder.

Prefill (mica_b200.prefill) answers one request with one pass and keeps nothing; its options are single
tokens. AnswerScorer keeps a context's K and V in a paged cache, so that

  * a document is read once and any number of questions fork from it (pages shared until written);
  * a set of answers runs as one tree: each distinct proper prefix of the answers is one row, which sees the
    context and its own prefix, and the log probability of an answer is the sum over its tokens;
  * the chosen answer becomes part of the context without running its tokens again: the accepted rows move
    together behind it.

The reference scores single label tokens after a whole prefill per request, and forks whole-prefix states
(v0.5/serving/lib/release_runtime.py:298-306, v0.5/serving/lib/fork.py).

    s = AnswerScorer(model, pages=2048)
    doc = s.open(document_ids)
    q = s.fork(doc); s.extend([q], [question_ids])
    r = s.score([q], [[[tok, tok], [tok], ...]])        # r[0].logprob: one value per answer
    best = s.answer([q], [answers])                     # scores, and keeps the best in the context
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch
import torch.nn.functional as F

from . import int8_kernels as K
from . import paged
from ._native import NORM_WEIGHT
from .logprobs import MAX_TOP, token_logprobs
from .prefill import Decoder, Prefill


@dataclass
class Scores:
    logprob: torch.Tensor          # fp32 [answers]: sum over the answer's tokens
    entropy: torch.Tensor          # fp32 scalar: of the first token's distribution, in nats
    top_logprob: torch.Tensor      # fp32 [top]: the first token's largest log probabilities
    top_id: torch.Tensor           # int64 [top]


def _in_vocabulary(name, least, most, vocab):
    if least < 0 or most >= vocab:
        raise ValueError(f'{name}: token {least if least < 0 else most} is not in the vocabulary of {vocab}')


class _Trie:
    """The answers of one context: its nodes are their distinct proper prefixes, parents first."""

    def __init__(self, answers, vocab):
        if not answers or any(len(a) == 0 for a in answers):
            raise ValueError('answers: at least one, none of them empty')
        _in_vocabulary('answers', min(min(a) for a in answers), max(max(a) for a in answers), vocab)
        self.parents, self.tokens, self.depth = [], [], []
        self.children = [{}]           # of the context, then of each node: token -> place among its row's tokens
        seen = {(): -1}
        self.paths = []                # per answer: (row, place) of each token; row 0 is the context's last
        self.nodes = []                # per answer: the nodes of its proper prefixes
        for a in answers:
            path, nodes, at = [], [], -1
            for i, tok in enumerate(a):
                kids = self.children[at + 1]
                path.append((at + 1, kids.setdefault(int(tok), len(kids))))
                if i + 1 < len(a):
                    key = tuple(int(x) for x in a[:i + 1])
                    if key not in seen:
                        seen[key] = len(self.parents)
                        self.parents.append(at)
                        self.tokens.append(int(tok))
                        self.depth.append(i)
                        self.children.append({})
                    at = seen[key]
                    nodes.append(at)
            self.paths.append(path)
            self.nodes.append(nodes)


class AnswerScorer(Prefill):
    """A Prefill that also keeps contexts. One scorer is used from one stream at a time, as its cache is."""

    def __init__(self, model: Decoder, pages: int, page: int = 64, option_ids=(0,), max_len: int = 32768,
                 chunk: int = 8192, **kw):
        """pages: pages of `page` tokens for all contexts together. chunk: the most tokens of one pass."""
        super().__init__(model, option_ids, max_len, **kw)
        c = self.cfg
        if chunk < 1:
            raise ValueError(f'chunk {chunk}')
        self.cache = paged.PagedCache(c.layers, c.kv_heads, c.head_dim, pages, page, model.device)
        self.head = model.lm_head if model.lm_head is not None else model.embed
        self.chunk = chunk
        self.vocab = min(self.head.shape[0], model.embed.shape[0])
        self._last = {}                # context -> its last row, final norm applied, bf16 [1, hidden]

    # ---- one pass ----------------------------------------------------------------------
    def _rows(self, ids, step: paged.Step, pos=None, rows=None):
        """The decoder over a step's rows: ids [N]; returns the rows (all, or `rows`) after the final norm."""
        cfg, m = self.cfg, self.m
        h = F.embedding(ids, m.embed)
        prev = None
        for li, lay in enumerate(m.layers):
            nq, h = self._normed(prev if prev is not None else h, lay.in_norm, h if prev is not None else None,
                                 lay.parts()[0][2], lay.distinct_attn_invs())
            qkv = self._qkv_cols(lay, nq, 0, lay.qkv_w.shape[0])
            k, v = self.cache.layer(li)
            q = paged.append(qkv, lay.q_norm, lay.k_norm, self.cos, self.sin, k, v, step, cfg.heads, pos=pos,
                             eps=cfg.eps)
            attn = paged.attention(q, k, v, step, cfg.heads, scale=self.scale)
            qa, sa = torch.ops.mica.act_quant(attn, lay.o_inv, K._round_code())
            o = self._gemm(qa, sa, lay.o_w, lay.o_s, lay.o_b)
            nm, h = self._normed(o, lay.post_norm, h, lay.mlp_in_inv(), lay.distinct_mlp_invs())
            prev = self._mlp(nm, lay)
        out = h + prev
        if rows is not None:
            out = out.index_select(0, rows)
        _, _, y, _ = torch.ops.mica.rmsnorm_quant(out, None, m.final_norm, None, cfg.eps, NORM_WEIGHT, K._round_code(),
                                                  True, False)
        return y

    def logits(self, rows):
        """fp32 logits [N, vocab] of rows after the final norm."""
        return torch.mm(rows, self.head.t(), out_dtype=torch.float32)

    def _tokens(self, flat):
        t = torch.tensor(flat, dtype=torch.long)
        return t.pin_memory().to(self.m.device, non_blocking=True)

    # ---- contexts ----------------------------------------------------------------------
    @torch.no_grad()
    def open(self, ids) -> int:
        """A new context of the tokens ids (1-D, at least one)."""
        sid = self.cache.open()
        try:
            self.extend([sid], [ids])
        except Exception:
            self.free(sid)
            raise
        return sid

    @torch.no_grad()
    def extend(self, sids: Sequence[int], ids: Sequence) -> None:
        """Appends tokens to contexts (1-D tensors or lists, at least one token each), `chunk` rows at a pass.
        Tokens outside the vocabulary are refused where they are on the host; ids on the device are not looked at."""
        if len(set(sids)) != len(sids) or len(sids) != len(ids):
            raise ValueError(f'extend: {len(ids)} token lists for contexts {list(sids)}')
        rest = [torch.as_tensor(t, dtype=torch.long).reshape(-1) for t in ids]
        for t in rest:
            if not t.is_cuda and t.numel():
                _in_vocabulary('extend', int(t.min()), int(t.max()), self.vocab)
        rest = [t.to(self.m.device) for t in rest]
        for sid, t in zip(sids, rest):
            if t.numel() == 0 or self.cache.length(sid) + t.numel() > self.max_len:
                raise ValueError(f'extend: {t.numel()} tokens on {self.cache.length(sid)} (1 .. {self.max_len})')
        self.cache.reserve(sids, [t.numel() for t in rest])          # all of it, or nothing is changed
        try:
            self._extend(sids, rest)
        except Exception:
            self.cache.commit(sids, [0] * len(sids))                  # what is still reserved goes back
            raise

    def _extend(self, sids, rest):
        at = [0] * len(rest)
        while True:
            todo, room = [], self.chunk
            for i, t in enumerate(rest):
                n = min(room, t.numel() - at[i])
                if n > 0:
                    todo.append((i, n))
                    room -= n
            if not todo:
                return
            who = [sids[i] for i, _ in todo]
            new = [n for _, n in todo]
            step = self.cache.step(who, new)
            row = torch.cat([rest[i][at[i]:at[i] + n] for i, n in todo])
            last = self._rows(row, step, rows=step.cu[1:].long() - 1)
            left = [rest[i].numel() - at[i] - n for i, n in todo]
            self.cache.commit(who, new)
            self.cache.reserve(who, left)
            for j, (i, n) in enumerate(todo):
                at[i] += n
                self._last[sids[i]] = last[j:j + 1]

    def fork(self, sid: int) -> int:
        """A context with the same tokens; its pages are shared until one of the two is extended."""
        new = self.cache.fork(sid)
        if sid in self._last:
            self._last[new] = self._last[sid]
        return new

    def free(self, sid: int) -> None:
        self.cache.free(sid)
        self._last.pop(sid, None)

    def length(self, sid: int) -> int:
        return self.cache.length(sid)

    # ---- answers -----------------------------------------------------------------------
    def _run(self, sids, answers, top):
        if len(set(sids)) != len(sids) or len(sids) != len(answers) or not sids:
            raise ValueError(f'answers: {len(answers)} sets for contexts {list(sids)}')
        if not 0 <= top <= min(MAX_TOP, self.vocab):
            raise ValueError(f'answers: top {top} of {self.vocab} tokens (at most {MAX_TOP})')
        tries = [_Trie(a, self.vocab) for a in answers]
        for sid in sids:
            if self.cache.length(sid) and sid not in self._last:
                raise ValueError(f'answers: context {sid} has no last row (its last pass failed): extend it')
        base = [self.cache.length(s) for s in sids]
        for b, t in zip(base, tries):
            if b + 1 + max(t.depth, default=-1) > self.max_len:
                raise ValueError(f'answers: they pass {self.max_len} positions')
        try:
            return self._run_tries(sids, answers, tries, base, top)
        except Exception:
            self.cache.commit(sids, [0] * len(sids))                  # the trees' pages go back
            raise

    def _run_tries(self, sids, answers, tries, base, top):
        new = [len(t.parents) for t in tries]
        step = None
        last = torch.cat([self._last[s] for s in sids])
        # rows: the contexts' last ones, then the trees' nodes
        start = [len(sids)]
        for n in new:
            start.append(start[-1] + n)
        if sum(new):
            mask = paged.tree_mask([t.parents for t in tries]).pin_memory().to(self.m.device, non_blocking=True)
            step = self.cache.step(sids, new, mask=mask)
            ids = self._tokens([x for t in tries for x in t.tokens] + [b + d for b, t in zip(base, tries) for d in t.depth])
            n = sum(new)
            last = torch.cat((last, self._rows(ids[:n], step, pos=ids[n:])))
        kids = [list(t.children[0]) for t in tries] + [list(c) for t in tries for c in t.children[1:]]
        most = max(len(k) for k in kids)
        given = self._tokens([x for k in kids for x in k + [-1] * (most - len(k))]).view(len(kids), most)
        lp, ent, top_lp, top_id = token_logprobs(self.logits(last), given, top)
        # an answer's value: the sum over its path; places behind its end point at a zero
        flat = torch.cat((lp.reshape(-1), lp.new_zeros(1)))
        longest = max(len(p) for t in tries for p in t.paths)
        at = []
        for i, t in enumerate(tries):
            for p in t.paths:
                place = [(i if r == 0 else start[i] + r - 1) * most + c for r, c in p]
                at += place + [lp.numel()] * (longest - len(place))
        total = flat[self._tokens(at)].view(-1, longest).sum(1)
        out, k = [], 0
        for i, a in enumerate(answers):
            out.append(Scores(total[k:k + len(a)], ent[i], top_lp[i], top_id[i]))
            k += len(a)
        return out, tries, step

    @torch.no_grad()
    def score(self, sids: Sequence[int], answers: Sequence[Sequence[Sequence[int]]], top: int = 0) -> list:
        """Log probability of each answer (a list of token ids, at least one) after its context: answers[b] are
        those of sids[b]. One pass for all of them; the contexts are not changed. Returns Scores per context."""
        out, _, _ = self._run(sids, answers, top)
        self.cache.commit(sids, [0] * len(sids))                  # the trees' pages go back
        return out

    @torch.no_grad()
    def answer(self, sids: Sequence[int], answers: Sequence[Sequence[Sequence[int]]]) -> list:
        """Scores the answers and appends the likeliest one (the first, if several are) to each context.
        Returns its index per context. Waits for the device. Where a chosen answer has no room (max_len, or
        the pages), no context is changed."""
        out, tries, step = self._run(sids, answers, 0)
        best = [int(i) for i in torch.stack([s.logprob.argmax() for s in out]).tolist()]
        nodes = [t.nodes[i] for t, i in zip(tries, best)]
        try:
            for sid, n in zip(sids, nodes):
                if self.cache.length(sid) + len(n) + 1 > self.max_len:
                    raise ValueError(f'answer: {len(n) + 1} tokens on {self.cache.length(sid)} (up to {self.max_len})')
            self.cache.fits_after(sids, [len(n) for n in nodes], [1] * len(sids))
        except Exception:
            self.cache.commit(sids, [0] * len(sids))              # the trees' pages go back
            raise
        if step is not None:
            for sid, n in zip(sids, nodes):
                if n:
                    del self._last[sid]                           # until the answer's last token has been run
            self.cache.keep(sids, step, nodes)
        self.extend(sids, [[a[i][-1]] for a, i in zip(answers, best)])
        return best
