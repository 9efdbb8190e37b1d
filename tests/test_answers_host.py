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
    monkeypatch.setattr(answers.AnswerScorer, 'logits', lambda self, rows: torch.zeros(rows.shape[0], VOCAB))

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


def test_an_answer_that_does_not_fit_changes_nothing(make):
    """The whole chosen answer has to fit, its last token too: in the positions, and in the pages."""
    s = make(max_len=20)
    sids = [s.open([9] * 17), s.open([9] * 5)]
    was = state(s)
    with pytest.raises(ValueError):
        s.answer(sids, [[[1, 2, 3, 4]], [[5]]])
    assert state(s) == was
    assert s.answer(sids, [[[1, 2, 3, 4], [0, 0, 0]], [[5]]]) == [1, 0]         # one that is not chosen may be longer
    assert [s.length(x) for x in sids] == [20, 6] and [s._last[x].tolist() for x in sids] == [[[19.0]], [[5.0]]]

    from mica_b200.paged import OutOfPages
    s = make(pages=2)
    sids = [s.open([9] * 13), s.open([9] * 3)]
    was = state(s)
    with pytest.raises(OutOfPages):
        s.answer(sids, [[[1, 2, 3, 4]], [[5, 6]]])
    assert state(s) == was
    assert s.answer(sids, [[[1, 2, 3]], [[5, 6]]]) == [0, 0] and [s.length(x) for x in sids] == [16, 5]


def test_an_answer_takes_the_pages_that_its_tree_gives_back(make):
    s = make(pages=4)
    sids = [s.open([9] * 16), s.open([9] * 15)]
    # the first tree takes two pages and keeps none but one; the second answer's last token needs one
    assert s.answer(sids, [[[1] * 20, [0, 0]], [[5, 6]]]) == [1, 0]
    assert [s.length(x) for x in sids] == [18, 17] and s.cache.free_pages == 0


def test_an_answer_of_one_token_to_a_fork_without_a_page_for_its_copy(make):
    from mica_b200.paged import OutOfPages
    s = make(pages=1)
    a = s.open([9] * 5)
    b = s.fork(a)
    was = state(s)
    with pytest.raises(OutOfPages):
        s.answer([b], [[[1]]])
    assert state(s) == was
    s.free(a)
    assert s.answer([b], [[[1]]]) == [0] and s.length(b) == 6


def test_a_context_that_lost_its_last_row_is_not_scored(make, monkeypatch):
    """An error of the last pass (no memory, say) leaves the kept tokens without a row to go on from."""
    s = make()
    sid = s.open([9] * 5)
    rows = type(s)._rows

    def fails(self, ids, step, pos=None, rows_=None, **kw):
        if len(ids) == 1:
            raise MemoryError
        return rows(self, ids, step, pos=pos, **kw)

    monkeypatch.setattr(type(s), '_rows', fails)
    with pytest.raises(MemoryError):
        s.answer([sid], [[[1, 2, 3]]])
    monkeypatch.setattr(type(s), '_rows', rows)
    assert s.length(sid) == 7
    for call in (s.score, s.answer):
        with pytest.raises(ValueError, match='last row'):
            call([sid], [[[1]]])
    s.extend([sid], [[3]])
    assert s.score([sid], [[[1]]])[0].logprob.shape == (1,) and s._last[sid].tolist() == [[7.0]]


def test_a_fork_needs_no_last_row(make):
    """A context that has no tokens yet, or lost its last row, forks as it is."""
    s = make()
    a = s.cache.open()
    b = s.fork(a)
    assert s.length(b) == 0
    s.extend([b], [[1, 2]])
    c = s.fork(b)
    assert s._last[c] is s._last[b] and s.length(a) == 0 and len(s.cache._seqs) == 3


@pytest.mark.parametrize('top', [-1, 33, VOCAB + 1])
def test_top_is_refused_before_anything_runs(make, top):
    s = make()
    sid = s.open([9] * 5)
    was, ran = state(s), len(s.passes)
    with pytest.raises(ValueError, match='top'):
        s.score([sid], [[[1, 2]]], top=top)
    assert state(s) == was and len(s.passes) == ran


def test_an_error_in_a_pass_gives_the_reserved_pages_back(make, monkeypatch):
    from mica_b200 import answers
    s = make(chunk=20)
    sids = [s.open([9] * 5), s.open([9] * 30)]
    was = state(s)

    def fails(*a, **kw):
        raise MemoryError

    with monkeypatch.context() as m:
        m.setattr(answers, 'token_logprobs', fails)
        for call in (s.score, s.answer):
            with pytest.raises(MemoryError):
                call(sids, [[[1, 2] * 20], [[3, 4]]])
            assert state(s) == was
    rows = type(s)._rows
    with monkeypatch.context() as m:
        m.setattr(type(s), '_rows', fails)
        with pytest.raises(MemoryError):
            s.extend(sids, [[1] * 40, [2] * 3])
        assert state(s) == was
        # the second pass of 20 rows: the first one's tokens stay, with their last row
        m.setattr(type(s), '_rows', lambda self, ids, *a, **kw: fails() if len(self.passes) > n else rows(self, ids, *a, **kw))
        n = len(s.passes)
        with pytest.raises(MemoryError):
            s.extend(sids, [[1] * 40, [2] * 3])
    assert s.length(sids[0]) == 25 and s._last[sids[0]].tolist() == [[24.0]] and s.length(sids[1]) == 30
    assert s.cache.free_pages == was[1] - 1
