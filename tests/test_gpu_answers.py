"""AnswerScorer: the paged-cache operators and the readout together, on a small random decoder, against the
prefill path run on every prefix by itself.

Both paths quantise every projection's input to int8 per token and differ in the last bit of some bf16 values
(attention's order of sums, q and k rounded once instead of after every step). By how much that moves a log
probability: a row's largest value is about 3 of its standard deviations d, so a code is 3 d / 127 = 0.024 d
wide; a bf16 half step of a value of size d is 2^-8 d = 0.004 d, so about one code in six (0.004 / 0.024) moves by
one, which is a noise of sqrt(1/6) * 0.024 d = 0.01 d at each of the 4 projections of 3 layers: sqrt(12) * 0.01 =
0.034 of the final hidden state. The logits' spread is 0.06 * sqrt(256) = 0.96, so a token's log probability is off
by 0.033 (one standard deviation), and TOL is four and a half of that. A token scored after a wrong prefix is off
by 0.96 * sqrt(2) = 1.4."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 0.15


@pytest.fixture(scope='module')
def model():
    from mica_b200.prefill import DecoderConfig, random_decoder
    cfg = DecoderConfig(hidden=256, inter=512, layers=3, heads=4, kv_heads=2, head_dim=128, vocab=5000)
    m = random_decoder(cfg, 'cuda', seed=3, std=0.06)
    return m


def scorer(model, **kw):
    from mica_b200.answers import AnswerScorer
    return AnswerScorer(model, **{**dict(pages=80, page=16, max_len=2048), **kw})


def plain(s, ids):
    """Log probabilities of the token after ids, by the prefill path."""
    h = s.hidden_last(torch.tensor(ids, device='cuda'))
    y = torch.ops.mica.rmsnorm_quant(h, None, s.m.final_norm, None, s.cfg.eps, 1, 0, True, False)[2]
    return torch.log_softmax(y.double() @ s.head.double().t(), 1)[0]


def tokens(n, seed):
    return torch.randint(0, 5000, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


ANSWERS = [[7, 8, 9], [7, 8], [7, 11, 12, 13], [4], [7, 8, 10], [300, 4], [4]]


def check(s, sid, context, answers, scores):
    for a, got in zip(answers, scores.logprob.tolist()):
        ref = sum(float(plain(s, context + a[:i])[a[i]]) for i in range(len(a)))
        assert abs(got - ref) < TOL * len(a), (a, got, ref)


@pytest.mark.parametrize('n', [1, 15, 64, 200, 700])
def test_answers_equal_the_prefixes_run_one_by_one(model, n):
    s = scorer(model)
    ctx = tokens(n, n)
    sid = s.open(ctx)
    r = s.score([sid], [ANSWERS], top=5)[0]
    check(s, sid, ctx, ANSWERS, r)
    p = plain(s, ctx)
    assert abs(float(r.entropy) + float((p * p.exp()).sum())) < TOL
    assert abs(float(r.top_logprob[0]) - float(p.max())) < TOL
    assert r.logprob[3] == r.logprob[6]
    s.free(sid)
    assert s.cache.free_pages == 80


def test_contexts_in_chunks_and_together(model):
    """A context read in passes of 37 rows, and three contexts extended and scored at once."""
    s, t = scorer(model), scorer(model, chunk=37)
    ctx = [tokens(150, 1), tokens(33, 2), tokens(1, 3)]
    a = [s.open(c) for c in ctx]
    b = [t.cache.open() for _ in ctx]
    t.extend(b, ctx)
    sets = [ANSWERS, [[5]], [[9, 9, 9, 9], [9, 9]]]
    ra, rb = s.score(a, sets), t.score(b, sets)
    for i, c in enumerate(ctx):
        check(s, a[i], c, sets[i], ra[i])
        assert (ra[i].logprob - rb[i].logprob).abs().max() < TOL * 4
    assert [s.length(x) for x in a] == [t.length(x) for x in b] == [150, 33, 1]


def test_forks_leave_their_document_as_it_was(model):
    s = scorer(model)
    doc = tokens(90, 5)
    d = s.open(doc)
    before = s.score([d], [ANSWERS])[0].logprob.clone()
    forks = [s.fork(d) for _ in range(3)]
    assert s.cache.free_pages == 80 - 6
    q = [tokens(20, 6), tokens(1, 7), tokens(40, 8)]
    s.extend(forks, q)
    for f, x in zip(forks, q):
        check(s, f, doc + x, ANSWERS, s.score([f], [ANSWERS])[0])
    assert torch.equal(s.score([d], [ANSWERS])[0].logprob, before)
    kept = s.score([forks[2]], [ANSWERS])[0].logprob.clone()
    for x in (d, forks[0], forks[1]):
        s.free(x)
    s.cache.compact()
    assert torch.equal(s.score([forks[2]], [ANSWERS])[0].logprob, kept)
    s.free(forks[2])
    assert s.cache.free_pages == 80


def test_the_chosen_answer_joins_the_context(model):
    s = scorer(model)
    ctx = [tokens(70, 9), tokens(16, 10)]
    sids = [s.open(c) for c in ctx]
    sets = [ANSWERS, [[1, 2, 3, 4, 5], [1, 2, 6], [8]]]
    ref = [r.logprob.clone() for r in s.score(sids, sets)]
    best = s.answer(sids, sets)
    assert best == [int(r.argmax()) for r in ref]
    for sid, c, a, i in zip(sids, ctx, sets, best):
        full = c + a[i]
        assert s.length(sid) == len(full)
        check(s, sid, full, ANSWERS, s.score([sid], [ANSWERS])[0])


def test_single_tokens_need_no_pass(model):
    """Answers of one token read the context's last row alone (no tree)."""
    s = scorer(model)
    ctx = tokens(40, 11)
    sid = s.open(ctx)
    from mica_b200.int8_kernels import STATS
    before = STATS['launch']
    r = s.score([sid], [[[i] for i in range(50)]])[0]
    assert STATS['launch'] - before == 1
    check(s, sid, ctx, [[0], [49]], type(r)(r.logprob[[0, 49]], None, None, None))
    assert s.answer([sid], [[[3]]]) == [0] and s.length(sid) == 41


def test_refusals_change_nothing(model):
    from mica_b200.paged import OutOfPages
    s = scorer(model, pages=6)
    sid = s.open(tokens(60, 1))
    before = s.score([sid], [[[5]]])[0].logprob.clone()
    with pytest.raises(OutOfPages):
        s.extend([sid], [tokens(60, 2)])
    with pytest.raises(OutOfPages):
        s.open(tokens(100, 2))
    for bad in ([], [[]], [[1], []]):
        with pytest.raises(ValueError):
            s.score([sid], [bad])
    with pytest.raises(ValueError):
        s.score([sid, sid], [[[1]], [[1]]])
    with pytest.raises(ValueError):
        s.extend([sid], [[]])
    with pytest.raises(ValueError):
        scorer(model, max_len=50).open(tokens(60, 1))
    assert s.length(sid) == 60 and torch.equal(s.score([sid], [[[5]]])[0].logprob, before)


def test_an_answer_without_room_leaves_its_contexts_as_they_were(model):
    from mica_b200.paged import OutOfPages
    for kw, ctx, wrong in ((dict(max_len=64), 61, ValueError), (dict(pages=5), 61, OutOfPages)):
        s = scorer(model, **kw)
        sids = [s.open(tokens(ctx, 1)), s.open(tokens(5, 2))]
        sets = [[[7, 8, 9, 10]], [[4, 5]]]
        before = [r.logprob.clone() for r in s.score(sids, sets)]
        with pytest.raises(wrong):
            s.answer(sids, sets)
        assert [s.length(x) for x in sids] == [ctx, 5] and s.cache.free_pages == s.cache.pool.shape[0] - 5
        again = [r.logprob for r in s.score(sids, sets)]
        assert all(torch.equal(a, b) for a, b in zip(before, again))


def test_ids_on_the_device_and_on_the_host_are_the_same_context(model):
    s = scorer(model)
    ctx = tokens(50, 3)
    made = [s.open(ctx), s.open(torch.tensor(ctx)), s.open(torch.tensor(ctx, device='cuda', dtype=torch.int32))]
    got = [r.logprob for r in s.score(made, [ANSWERS] * 3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
