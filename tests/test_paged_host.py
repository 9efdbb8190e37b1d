"""Refusals of the paged-cache and log-probability entry points and the cache's host state, without a GPU."""
import ctypes

import pytest
import torch

from mica_b200 import build


@pytest.fixture(scope='module')
def lib():
    build.build()
    from mica_b200 import _native as N
    return N.lib()


def append(lib, **kw):
    a = dict(qkv=16, ld=768, q_w=16, k_w=16, cos=16, sin=16, n_pos=8, pos=None, q_out=16, ldq=512, k=16, v=16,
             stride=2048, pages=4, page=16, table=16, ld_table=2, P=2, base=16, cu=16, B=1, N=4, H=8, KV=2, D=64,
             eps=1e-6, stream=None)
    a.update(kw)
    return lib.mica_cache_append(*a.values())


def attention(lib, **kw):
    a = dict(q=16, ldq=512, k=16, v=16, stride=2048, pages=4, page=16, table=16, ld_table=2, P=2, base=16, cu=16,
             mask=None, ld_mask=0, words=0, B=1, N=4, max_new=4, H=8, KV=2, D=64, scale=0.1, out=16, ldo=512, ws=16,
             ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return lib.mica_cache_attention(*a.values())


def test_append_refusals(lib):
    for name in ('qkv', 'q_w', 'k_w', 'cos', 'sin', 'q_out', 'k', 'v', 'table', 'base', 'cu'):
        assert append(lib, **{name: None}) == 1
    for bad in (dict(D=96), dict(page=48), dict(page=8), dict(P=0), dict(ld_table=1), dict(pages=0), dict(B=-1),
                dict(N=-1), dict(H=0), dict(KV=0), dict(n_pos=0), dict(ld=760), dict(ldq=504), dict(stride=2040)):
        assert append(lib, **bad) == 2, bad
    for bad in (dict(qkv=24), dict(ld=770), dict(q_out=8), dict(k=8), dict(v=8), dict(cos=8), dict(pos=4),
                dict(table=2), dict(cu=2), dict(base=2), dict(stride=2052)):
        assert append(lib, **bad) == 3, bad


def test_attention_refusals(lib):
    for name in ('q', 'k', 'v', 'table', 'base', 'cu', 'out'):
        assert attention(lib, **{name: None}) == 1
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf'))):
        assert attention(lib, **bad) == 1, bad
    for bad in (dict(D=80), dict(page=256), dict(H=7), dict(H=258, KV=2, ldq=1 << 20, ldo=1 << 20), dict(max_new=-1),
                dict(mask=16, words=0), dict(mask=16, words=2, ld_mask=1), dict(ldo=504), dict(P=0)):
        assert attention(lib, **bad) == 2, bad
    assert attention(lib, P=1 << 28, ld_table=1 << 28) == 6
    for bad in (dict(q=24), dict(out=24), dict(mask=20, words=1, ld_mask=1), dict(ws=8), dict(ldq=516)):
        assert attention(lib, **bad) == 3, bad


def test_copy_refusals(lib):
    ints = lambda *v: (ctypes.c_int * len(v))(*v)  # noqa: E731
    copy = lib.mica_cache_copy
    assert copy(None, 64, 64, 4, ints(0), ints(1), 1, None) == 1
    assert copy(16, 64, 64, 4, None, ints(1), 1, None) == 1
    assert copy(16, 64, 64, 4, ints(0), ints(1), -1, None) == 1
    assert copy(16, 48, 64, 4, ints(0), ints(1), 1, None) == 2
    assert copy(16, 64, 64, 0, ints(0), ints(1), 1, None) == 2
    assert copy(24, 64, 64, 4, ints(0), ints(1), 1, None) == 3
    assert copy(16, 72, 64, 4, ints(0), ints(1), 1, None) == 3
    for src, dst in (((0, 1), (2, 2)), ((0, 2), (2, 3)), ((0,), (0,)), ((4,), (0,)), ((0,), (4,)), ((-1,), (0,)),
                     ((0,), (-1,))):
        assert copy(16, 64, 64, 4, ints(*src), ints(*dst), len(src), None) == 1, (src, dst)


def test_keep_and_logprob_refusals(lib):
    def keep(**kw):
        a = dict(pool=16, stride=4096, slabs=2, pages=4, page=16, D=64, table=16, ld_table=2, P=2, base=16, cu=16, B=1,
                 keep=16, ld_keep=3, n_keep=16, A=3, new_base=32, stream=None)
        a.update(kw)
        return lib.mica_cache_keep(*a.values())
    for name in ('pool', 'table', 'base', 'cu', 'keep', 'n_keep', 'new_base'):
        assert keep(**{name: None}) == 1
    assert keep(new_base=16) == 1                      # in place of base
    for bad in (dict(slabs=0), dict(D=72), dict(A=-1), dict(ld_keep=2), dict(stride=4080), dict(page=24)):
        assert keep(**bad) == 2, bad
    assert keep(pool=24) == 3 and keep(keep=18) == 3

    def lp(**kw):
        a = dict(z=16, dtype=2, ld=100, N=2, V=100, ids=16, ld_ids=1, M=1, top=4, lp=16, ent=16, tl=16, ti=16,
                 stream=None)
        a.update(kw)
        return lib.mica_token_logprobs(*a.values())
    for bad in (dict(z=None), dict(ent=None), dict(dtype=3), dict(M=-1), dict(top=-1), dict(ids=None), dict(lp=None),
                dict(tl=None), dict(ti=None)):
        assert lp(**bad) == 1, bad
    for bad in (dict(N=-1), dict(V=0), dict(ld=99), dict(ld_ids=0), dict(top=33), dict(V=3, top=4)):
        assert lp(**bad) == 2, bad
    for bad in (dict(z=18), dict(ids=20), dict(ti=20), dict(lp=18)):
        assert lp(**bad) == 3, bad


def test_python_refusals():
    from mica_b200 import logprobs, paged
    i32 = {'dtype': torch.int32}
    table, base, cu = torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
    step = paged.Step(table, base, cu)
    with pytest.raises(ValueError):
        paged.Step(table, base, torch.zeros(2, **i32))
    with pytest.raises(ValueError):
        paged.Step(table.long(), base, cu)
    with pytest.raises(ValueError):
        paged.Step(table, base, cu, mask=torch.zeros(4, 1, **i32))
    with pytest.raises(ValueError):
        paged.Step(table, base, cu, max_new=-1)
    k = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    q = torch.zeros(4, 8 * 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='CUDA'):
        paged.attention(q, k, k, step, 8)
    with pytest.raises(ValueError):
        paged.attention(q, k, k, step, 7)
    with pytest.raises(ValueError):
        paged.attention(q, k[:, :, :, :32], k[:, :, :, :32], step, 8)
    with pytest.raises(ValueError):
        paged.attention(q, k.transpose(1, 2), k.transpose(1, 2), step, 8)
    with pytest.raises(ValueError):
        paged.attention(q, k, k, step, 8, scale=-1.0)
    with pytest.raises(ValueError):
        paged.attention(q, k, k, paged.Step(table, base, cu, mask=torch.zeros(3, 1, dtype=torch.int64)), 8)
    with pytest.raises(RuntimeError):
        paged.attention(q.float(), k, k, step, 8)
    w, t = torch.ones(64, dtype=torch.bfloat16), torch.ones(9, 64, dtype=torch.bfloat16)
    qkv = torch.zeros(4, 12 * 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='CUDA'):
        paged.append(qkv, w, w, t, t, k, k, step, 8)
    with pytest.raises(ValueError):
        paged.append(qkv, w, w, t, t, k, k, step, 7)
    with pytest.raises(ValueError):
        paged.append(qkv, w[:32], w, t, t, k, k, step, 8)
    with pytest.raises(ValueError):
        paged.append(qkv, w, w, t, t, k, k, step, 8, pos=torch.zeros(4, **i32))
    pool = torch.zeros(6, 2, 2, 2, 16, 64, dtype=torch.bfloat16)
    for src, dst in (([0], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([6], [0]), ([0], [6]), ([-1], [0]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            paged.copy_pages(pool, src, dst)
    with pytest.raises(RuntimeError, match='CUDA'):
        paged.copy_pages(pool, [0], [1])
    with pytest.raises(ValueError):
        paged.keep_tokens(pool, step, torch.zeros(1, 2, **i32), torch.zeros(2, **i32))
    with pytest.raises(ValueError):
        paged.keep_tokens(pool.float(), step, torch.zeros(2, 2, **i32), torch.zeros(2, **i32))
    z, ids = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match='CUDA'):
        logprobs.token_logprobs(z, ids)
    for bad in ((z, ids[:2], 0), (z, ids.int(), 0), (z, ids, 11), (z, ids, -1), (z[0], ids, 0), (z[:, :0], ids, 0)):
        with pytest.raises(ValueError):
            logprobs.token_logprobs(*bad)


def test_tree_mask_words():
    from mica_b200 import paged
    m = paged.tree_mask([[-1, 0, 0, 2], [], [-1] * 70])
    assert m.shape == (74, 2)
    assert m[:4, 0].tolist() == [1, 3, 5, 13]
    assert m[4 + 63].tolist() == [-(1 << 63), 0] and m[4 + 64].tolist() == [0, 1]
    with pytest.raises(ValueError):
        paged.tree_mask([[0]])
    assert paged.tree_mask([[]]).shape == (0, 1)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from mica_b200 import ops  # noqa: F401
    with FakeTensorMode():
        k = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16)
        i = torch.empty(2, 3, dtype=torch.int32)
        q = torch.empty(5, 8 * 64, dtype=torch.bfloat16)
        assert torch.ops.mica.cache_attention(q, k, k, i, i[:, 0], i[0], None, 8, 0.1, 5).shape == q.shape
        out = torch.ops.mica.token_logprobs(torch.empty(5, 100), torch.empty(5, 2, dtype=torch.int64), 3)
        assert [tuple(t.shape) for t in out] == [(5, 2), (5,), (5, 3), (5, 3)]


def test_cache_host_state(monkeypatch):
    """Pages, shares and lengths on the host (copies recorded, not run)."""
    from mica_b200 import paged
    copies = []
    monkeypatch.setattr(paged, 'copy_pages', lambda pool, s, d: copies.append((list(s), list(d))))
    c = paged.PagedCache(1, 1, 64, 10, page=16, device='cpu')
    a = c.open()
    c.reserve([a], [33])
    assert c.pages_of(a) == [0, 1, 2] and c.free_pages == 7
    c.commit([a], [20])
    assert c.pages_of(a) == [0, 1] and c.length(a) == 20 and c.free_pages == 8
    kids = [c.fork(a) for _ in range(3)]
    with pytest.raises(paged.OutOfPages):
        c.reserve(kids, [200, 1, 1])
    assert copies == [] and c.free_pages == 8 and c.pages_of(kids[0]) == [0, 1]
    c.reserve(kids[:2], [1, 1])                        # two writers of a page that two others keep: two copies
    assert copies == [([1, 1], [2, 3])] and c.free_pages == 6
    c.free(a)
    c.reserve([kids[2]], [1])                          # the last one left writes in place
    assert len(copies) == 1 and c.pages_of(kids[2]) == [0, 1]
    with pytest.raises(ValueError):
        c.commit([kids[2]], [13])
    step = paged.Step(*(torch.zeros(n, dtype=torch.int32) for n in ((1, 2), (1,), (2,))))
    with pytest.raises(ValueError):
        c.keep([kids[2]], step, [[0]])                 # not a step of the cache
    step.rows = [2]
    for rows in ([2], [1, 0], [0, 0], [-1]):
        with pytest.raises(ValueError):
            c.keep([kids[2]], step, [rows])
    with pytest.raises(ValueError):
        c.reserve([kids[2], kids[2]], [1, 1])
    for s in kids:
        c.free(s)
    assert c.free_pages == 10
    with pytest.raises(KeyError):
        c.free(a)
    for bad in (dict(page=24), dict(head_dim=80), dict(pages=0)):
        with pytest.raises(ValueError):
            paged.PagedCache(**{**dict(layers=1, kv_heads=1, head_dim=64, pages=2, device='cpu'), **bad})


def test_commit_and_keep_name_each_sequence_once(monkeypatch):
    """A sequence named twice would pass the check of its room twice, and lists of two lengths lose their ends."""
    from mica_b200 import paged
    monkeypatch.setattr(torch.Tensor, 'pin_memory', lambda t: t)
    c = paged.PagedCache(1, 1, 64, 10, page=16, device='cpu')
    a, b = c.open(), c.open()
    step = c.step([a, b], [10, 10])
    for sids, new in (([a, a], [10, 10]), ([a, b], [1]), ([a], [1, 1]), ([], [1])):
        with pytest.raises(ValueError):
            c.commit(sids, new)
    for sids, rows in (([a, a], [[0], [0]]), ([a], [[0]]), ([a, b], [[0]])):
        with pytest.raises(ValueError):
            c.keep(sids, step, rows)
    assert c.length(a) == c.length(b) == 0
    c.commit([a, b], [10, 3])
    assert c.length(a) == 10 and c.length(b) == 3


def test_a_step_keeps_the_tensors_it_is_given():
    """Whatever their strides: a captured graph reads new values where they are written."""
    from mica_b200 import paged
    i32 = {'dtype': torch.int32}
    table, base, cu = torch.zeros(2, 9, **i32), torch.zeros(4, **i32), torch.zeros(6, **i32)
    mask = torch.zeros(5, 3, dtype=torch.int64)
    step = paged.Step(table[:, ::3], base[::2], cu[::2], mask=mask.t())
    for t in (table, base, cu, mask):
        t += 1
    assert step.table.sum() == 6 and step.base.sum() == 2 and step.cu.sum() == 3 and step.mask.sum() == 15


def test_keep_serves_any_number_of_sequences(lib):
    """What is refused first is the pool's place, not the number of sequences."""
    assert lib.mica_cache_keep(24, 4096, 2, 4, 16, 64, 16, 2, 2, 16, 16, 70000, 16, 3, 16, 3, 32, None) == 3


def test_keep_refuses_a_step_whose_sequences_have_moved_on(monkeypatch):
    """The step's rows stand behind the tokens that were committed when it was described."""
    from mica_b200 import paged
    monkeypatch.setattr(torch.Tensor, 'pin_memory', lambda t: t)
    monkeypatch.setattr(paged, 'keep_tokens', lambda *a: None)
    c = paged.PagedCache(1, 1, 64, 10, page=16, device='cpu')
    a, b = c.open(), c.open()
    c.step([b], [2])
    c.commit([b], [2])
    step = c.step([a, b], [5, 5])
    with pytest.raises(ValueError):
        c.keep([b, a], step, [[0], [1]])               # the other way round
    c.keep([a, b], step, [[1, 3], [0]])
    assert c.length(a) == 2 and c.length(b) == 3
    with pytest.raises(ValueError):
        c.keep([a, b], step, [[0], [0]])               # once more
    assert c.length(a) == 2 and c.length(b) == 3


def test_a_scale_that_passes_fp32_in_base_two_is_refused(lib):
    assert attention(lib, scale=3e38) == 1 and attention(lib, scale=2e38, ws=8) == 3
