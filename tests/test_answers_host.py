"""AnswerScorer's host side without a GPU: what it checks before it runs anything, and the state that a refusal
leaves. The decoder's pass, the readout and the moves in the pool are stood in for: row i of a pass is the
position it stands at, so that a context's last row says which token it is of."""
from types import SimpleNamespace

import pytest
import torch

VOCAB = 50


@pytest.fixture
def make(monkeypatch):
    from mica_b200 import answers, paged
    monkeypatch.setattr(torch.Tensor, 'pin_memory', lambda t: t)
    monkeypatch.setattr(paged, 'copy_pages', lambda pool, s, d: None)
    monkeypatch.setattr(paged, 'keep_tokens', lambda pool, step, keep, n: None)

    def logprobs(z, ids, top):
        """As the kernel: 0 for padding, NaN past the end, else -id / 10."""
        lp = torch.where(ids < 0, 0.0, torch.where(ids >= VOCAB, float('nan'), -0.1 * ids))
        n = z.shape[0]
        return lp, torch.zeros(n), torch.zeros(n, top), torch.zeros(n, top, dtype=torch.int64)

    monkeypatch.setattr(answers, 'token_logprobs', logprobs)

    def rows(self, ids, step, pos=None, rows=None):
        self.passes.append(ids.tolist())
        assert all(0 <= i < VOCAB for i in self.passes[-1])         # what the embedding can look up
        at = [int(b) + i for b, a, e in zip(step.base, step.cu, step.cu[1:]) for i in range(int(e - a))]
        out = torch.tensor(at, dtype=torch.float32)[:, None]
        return out if rows is None else out[rows]

    monkeypatch.setattr(answers.AnswerScorer, '_rows', rows)

    def build(pages=20, page=16, max_len=100, chunk=1000):
        s = answers.AnswerScorer.__new__(answers.AnswerScorer)
        s.m = SimpleNamespace(device='cpu', embed=torch.zeros(VOCAB, 1))
        s.head, s.vocab = torch.zeros(VOCAB, 1), VOCAB
        s.cache = paged.PagedCache(1, 1, 64, pages, page=page, device='cpu')
        s.max_len, s.chunk, s._last, s.passes = max_len, chunk, {}, []
        return s

    return build


def state(s):
    return {x: (s.length(x), s.cache.pages_of(x), s._last[x].tolist()) for x in s._last}, s.cache.free_pages


BAD = [-1, VOCAB, VOCAB + 7, -(1 << 40), 1 << 40]


@pytest.mark.parametrize('bad', BAD)
def test_answers_with_tokens_outside_the_vocabulary_are_refused(make, bad):
    s = make()
    sid = s.open([1, 2, 3])
    was, ran = state(s), len(s.passes)
    for answers in ([[3], [bad]], [[3, bad]], [[bad, 3]], [[3], [3, bad, 4]]):
        for call in (s.score, s.answer):
            with pytest.raises(ValueError, match='vocabulary'):
                call([sid], [answers])
    assert state(s) == was and len(s.passes) == ran


@pytest.mark.parametrize('bad', BAD)
def test_contexts_with_tokens_outside_the_vocabulary_are_refused(make, bad):
    s = make()
    sid = s.open([1, 2, 3])
    was, ran = state(s), len(s.passes)
    for ids in ([bad], (4, bad), torch.tensor([4, bad, 5])):
        with pytest.raises(ValueError, match='vocabulary'):
            s.extend([sid], [ids])
        with pytest.raises(ValueError, match='vocabulary'):
            s.open(ids)
    assert state(s) == was and len(s.passes) == ran
