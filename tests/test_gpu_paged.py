"""The paged-cache operators against their definitions in 64 bits.

Tolerances, counted in half steps of bf16 (u = 2^-8, relative to the value). attention: the output is
rounded once (u |o|) and each weight p once before the product with V, so an output element is off by at
most u |o| + u sum_s p_s |v_s|, plus fp32 sums (2^-24 a step) and the exponential's 2^-21, far below u; the
test allows 1.1 of that bound. append: one rounding of an fp32 value, u |y| plus fp32 noise on the products
that may cancel (2^-20 of their sum). Copies and moves are bit-exact."""
import pytest
import torch

from paged_reference import Case, holes, norm_rope, tree

pytestmark = pytest.mark.gpu
U = 2.0 ** -8


def run_attention(c, scale=None, **kw):
    from mica_b200 import paged
    return paged.attention(c.q, c.k, c.v, c.step(**kw), c.heads, scale=scale)


def check_attention(c, o, scale=None):
    ref = c.attention(scale)
    was = c.keys
    c.keys = [(k, v.abs()) for k, v in was]
    size = c.attention(scale)                      # sum p |v|
    c.keys = was
    err = (o.double() - ref).abs()
    bound = 1.1 * U * (ref.abs() + size) + 1e-6
    assert torch.isfinite(o).all()
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, worst


SHAPES = [(32, 8, 128), (4, 4, 64), (6, 2, 128), (5, 1, 64), (28, 4, 128), (16, 1, 128)]


@pytest.mark.parametrize('heads,kv,dim', SHAPES)
@pytest.mark.parametrize('page', [16, 32, 64, 128])
def test_attention_next_token(heads, kv, dim, page):
    c = Case([0, 1, 15, 16, 127, 128, 129, 700], [1] * 8, heads, kv, dim, page, seed=page + heads)
    check_attention(c, run_attention(c, max_new=1))


@pytest.mark.parametrize('heads,kv,dim', SHAPES)
@pytest.mark.parametrize('mask', [None, tree, holes])
def test_attention_of_ragged_trees(heads, kv, dim, mask):
    c = Case([0, 300, 5, 129, 1000], [7, 1, 65, 130, 33], heads, kv, dim, 16, seed=heads + dim, mask=mask)
    check_attention(c, run_attention(c, max_new=130))


@pytest.mark.parametrize('new', [1, 31, 32, 33, 63, 64, 65, 128, 129, 200, 700])
def test_attention_row_counts(new):
    """One sequence, tree rows around the tile's edges; the hint may be wrong either way."""
    c = Case([333], [new], 8, 2, 128, 64, seed=new, mask=tree)
    o = run_attention(c)
    check_attention(c, o)
    check_attention(c, run_attention(c, max_new=1))
    check_attention(c, run_attention(c, max_new=new))


@pytest.mark.parametrize('ctx,new', [([20000], [1]), ([9001, 3, 0], [5, 64, 1]), ([4096] * 3, [17] * 3),
                                     ([0], [1500]), ([777], [1025])])
def test_attention_long_axes(ctx, new):
    c = Case(ctx, new, 8, 2, 128, 64, seed=len(ctx))
    check_attention(c, run_attention(c, max_new=max(new)))


@pytest.mark.parametrize('heads,new', [(1, 1), (5, 1), (5, 60), (4, 7)])
def test_attention_of_one_unit_in_many_parts(heads, new):
    """One K/V head and a long context: its one unit is cut into a part for each SM (and with few keys into
    some), which several threads join."""
    for ctx in (128 * 148 * 2 + 17, 128 * 20, 128 * 9, 128 * 5, 128 * 3 + 1):
        c = Case([ctx], [new], heads, 1, 128, 128, seed=ctx + new, mask=tree)
        o = run_attention(c, max_new=new)
        check_attention(c, o)
        assert torch.equal(o, run_attention(c, max_new=new))


@pytest.mark.parametrize('heads,kv,dim,new', [(8, 2, 128, 1), (8, 2, 64, 8), (16, 2, 128, 4), (16, 2, 64, 8), (5, 1, 128, 13),
                                              (6, 2, 128, 33), (64, 1, 64, 1), (8, 8, 64, 1), (8, 8, 128, 32)])
def test_attention_of_few_rows(heads, kv, dim, new):
    """Steps whose rows of a K/V head fill a quarter, a half or more of a row tile, whole units and divided ones,
    with rows that see nothing, or the keys of one part of a tile only."""
    for ctx in ([0, 5, 31, 32, 33, 64, 100, 127, 128, 129, 700], [9000], [40] * 70):
        n = [min(new, 1 + i % new) for i in range(len(ctx) - 1)] + [new]
        c = Case(ctx, n, heads, kv, dim, 64, seed=len(ctx) + new, mask=tree)
        o = run_attention(c, max_new=new)
        check_attention(c, o)
        assert torch.equal(o, run_attention(c, max_new=new))


@pytest.mark.parametrize('heads,new', [(4, 4), (4, 16), (4, 32)])
def test_few_rows_that_see_nothing_or_one_key(heads, new):
    made = []

    def blind(rng, t):
        made.append(torch.zeros(t, t, dtype=torch.bool))
        if len(made) == 2:
            made[1][:, t - 1] = True                                    # the second sequence's see its last node
        return made[-1]

    c = Case([0, 0], [new, new], heads, 1, 128, 32, seed=new, mask=blind)
    o = run_attention(c, max_new=new)
    check_attention(c, o)
    assert torch.equal(o[:new], torch.zeros_like(o[:new]))


@pytest.mark.parametrize('new', [1, 2, 8, 16, 33])
def test_infinities_of_committed_keys(new):
    """In tiles that every row sees and in the last, alone or two of a kind or of two kinds in a column, whatever
    part of the tile holds them."""
    inf = float('inf')
    c = Case([700, 40000], [new, new], 4, 1, 128, 32, seed=new, mask=tree)
    for b in range(2):
        for s, d, bad in ((100, 3, inf), (101, 4, -inf), (130, 5, inf), (190, 5, inf), (131, 6, inf), (250, 6, -inf),
                          (300, 64, float('nan')), (301, 65, inf), (699, 65, inf), (600, 66, inf), (699, 67, -inf),
                          (127, 127, -inf)):
            c.v[c.rows[b][s // 32], 0, s % 32, d] = bad
            c.keys[b][1][0, s, d] = bad
    o = run_attention(c, scale=0.01, max_new=new)                        # no weight is so small that it is zero
    ref = c.attention(0.01)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(o), torch.isnan(ref)) and torch.equal(o.double()[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()])
    assert (o.double() - ref)[fine].abs().max() < 0.05                  # 1.1 u (|o| + sum p |v|), |v| < 5.8


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_odd_values_in_a_causal_extension(bad):
    """Without a mask, rows do not see later rows' K and V: an odd value there changes nothing before its row."""
    c = Case([90, 0], [300, 200], 8, 2, 128, 32, seed=11)
    clean = run_attention(c)
    for b, at in ((0, 170), (1, 30)):
        s = c.ctx[b] + at
        c.v[c.rows[b][s // 32], :, s % 32] = bad
        c.k[c.rows[b][s // 32], :, s % 32] = bad
    o = run_attention(c)
    assert torch.equal(o[:170], clean[:170]) and torch.equal(o[300:330], clean[300:330])
    assert not torch.isfinite(o[170:300]).any(1).all() and not torch.isfinite(o[330:]).any(1).all()


def test_attention_many_sequences():
    ctx = [(i * 37) % 211 for i in range(500)]
    c = Case(ctx, [1 + i % 3 for i in range(500)], 4, 2, 64, 16, seed=2)
    check_attention(c, run_attention(c, max_new=3))


def test_attention_sequences_without_rows_and_padding_rows():
    """Sequences that have no rows in this step, rows behind the last sequence (zero), extra mask words."""
    c = Case([10, 500, 0, 40], [0, 3, 0, 70], 8, 2, 128, 32, seed=4, pad_rows=9, mask=tree, extra_words=2)
    o = run_attention(c)
    check_attention(c, o)
    assert float(o[-9:].float().abs().max()) == 0.0
    empty = Case([10, 5], [0, 0], 8, 2, 128, 32, seed=4, pad_rows=3)
    assert float(run_attention(empty).float().abs().max()) == 0.0


def test_attention_no_rows_and_no_sequences():
    from mica_b200 import paged
    c = Case([10], [0], 8, 2, 128, 32)
    assert run_attention(c).shape == (0, 8 * 128)
    i32 = {'dtype': torch.int32, 'device': 'cuda'}
    step = paged.Step(torch.zeros(0, 1, **i32), torch.zeros(0, **i32), torch.zeros(1, **i32))
    q = torch.ones(2, 8 * 128, dtype=torch.bfloat16, device='cuda')
    o = paged.attention(q, c.k, c.v, step, 8)
    assert float(o.float().abs().max()) == 0.0


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('ctx,new', [([70761, 30001], [13, 15]), ([40000], [60]), ([5000, 9000, 130], [33, 64, 40])])
def test_attention_adds_up_every_key_once(dim, ctx, new):
    """V says where its key stands: one column for each place of 16 keys in the tile (of the first 8 columns),
    one for each tile modulo the rest. Scores near zero make all weights alike, so a column is the share of its
    keys, off by the roundings of the weights (u each, at most) and of the output: a tile lost, read twice or
    changed under way, in one step of 16 keys even, is a change of a 60th of its column's own share or more."""
    c = Case(ctx, new, 8, 2, dim, 64, seed=dim, mask=tree)
    for b in range(len(ctx)):
        kk, vv = c.keys[b]
        s = torch.arange(vv.shape[1], device='cuda')
        vv.zero_()
        vv[:, s, s % 128 // 16] = 1
        vv[:, s, 8 + s // 128 % (dim - 8)] = 1
        for i in range(0, vv.shape[1], 64):
            m = min(64, vv.shape[1] - i)
            c.v[c.rows[b][i // 64], :, :m] = vv[:, i:i + m]
    ref = c.attention(1e-3)
    for _ in range(20):
        o = run_attention(c, scale=1e-3).double()
        assert ((o - ref).abs() <= 2.2 * U * ref + 1e-9).all(), float(((o - ref).abs() / (ref + 1e-9)).max())


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
@pytest.mark.parametrize('new', [20, 90])
def test_attention_odd_values_in_masked_nodes(bad, new):
    """A node's K and V that a row does not see change nothing in that row."""
    c = Case([50, 130], [new, new], 8, 2, 128, 32, seed=6, mask=tree)
    clean = run_attention(c)
    node = new - 4
    for b in range(2):
        kk, vv = c.keys[b]
        s = c.ctx[b] + node
        p, slot = c.rows[b][s // 32], s % 32
        vv[:, s] = bad
        c.v[p, :, slot] = bad
        kk[:, s] = bad
        c.k[p, :, slot] = bad
    o = run_attention(c)
    blind = torch.cat([~c.seen[b][:, node] for b in range(2)])
    assert blind.sum() > 0 and (~blind).sum() > 0
    assert torch.equal(o[blind.cuda()], clean[blind.cuda()])


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_attention_odd_values_that_are_seen(bad):
    """An infinite or NaN value in one element of a seen V reaches that element alone."""
    c = Case([70], [40], 4, 2, 128, 32, seed=8, mask=tree)
    clean = run_attention(c)
    s = 70 + 30
    c.v[c.rows[0][s // 32], 1, s % 32, 5] = bad
    c.keys[0][1][1, s, 5] = bad
    o = run_attention(c)
    ref = c.attention()
    assert torch.equal(torch.isnan(o), torch.isnan(ref)) and torch.equal(torch.isinf(o), torch.isinf(ref))
    fine = torch.isfinite(ref)
    assert (o.double() - ref)[fine].abs().max() < 0.05
    rows = ~c.seen[0][:, 30].cuda()
    assert torch.equal(o[rows], clean[rows])


@pytest.mark.parametrize('scale', [1e-4, 0.3, 3.0])
def test_attention_scales(scale):
    """Nearly even weights, and scores whose maximum moves by hundreds between tiles."""
    c = Case([600], [33], 8, 2, 128, 64, seed=12, mask=tree)
    check_attention(c, run_attention(c, scale=scale), scale)


def test_attention_growing_scores():
    """Keys whose scores rise along the axis: the running maximum moves in every tile."""
    c = Case([1000], [3], 4, 1, 128, 64, seed=3)
    kk, _ = c.keys[0]
    grow = torch.linspace(0.0, 6.0, kk.shape[1], device='cuda')[None, :, None]
    kk.copy_((grow * torch.sign(c.q[0, :128].float())[None, None]).bfloat16())
    for s in range(0, kk.shape[1], 64):
        m = min(64, kk.shape[1] - s)
        c.k[c.rows[0][s // 64], :, :m] = kk[:, s:s + m]
    check_attention(c, run_attention(c))


def test_attention_strided_rows_and_layer_of_a_pool():
    """q as columns of a wider buffer, pages as one layer of a pool of three."""
    c = Case([300, 40], [9, 70], 8, 2, 128, 64, seed=9, layers=3, layer=1, mask=tree)
    wide = torch.randn(c.n, 12 * 128 + 24, device='cuda').bfloat16()
    wide[:, 128:128 + 8 * 128] = c.q
    c.q = wide[:, 128:128 + 8 * 128]
    check_attention(c, run_attention(c))
    odd = torch.zeros(c.n, 8 * 128 + 3, dtype=torch.bfloat16, device='cuda')     # rows not 16-byte aligned
    odd[:, 3:] = c.q
    assert torch.equal(run_attention(c), _with_q(c, odd[:, 3:]))


def _with_q(c, q):
    was, c.q = c.q, q
    o = run_attention(c)
    c.q = was
    return o


def test_attention_same_bits_again_on_other_streams_and_in_graphs():
    """Repeated, on a side stream, two graphs replayed in turn and together with new lengths: the same bits."""
    c = Case([3000, 20, 700], [5, 16, 1], 32, 8, 128, 64, seed=5, mask=tree)
    o = run_attention(c)
    for _ in range(3):
        assert torch.equal(run_attention(c), o)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run_attention(c)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_attention(c))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], o) and torch.equal(outs[1], o)
    # the step's tensors changed in place: fewer committed tokens
    c.base.copy_(torch.tensor([100, 20, 64], dtype=torch.int32))
    eager = run_attention(c)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], eager) and not torch.equal(eager, o)


def test_attention_bad_pages_are_recorded_and_not_read():
    import ctypes

    from mica_b200 import _native as N
    st = torch.cuda.current_stream().cuda_stream
    code = ctypes.c_int(0)
    N.call('mica_device_error', ctypes.byref(code), st)
    for change in ('page', 'negative', 'base', 'negative_base'):
        c = Case([200, 30], [3, 4], 8, 2, 128, 64, seed=1)
        good = run_attention(c)
        if change == 'page':
            c.table[0, 1] = c.pool.shape[0]
        elif change == 'negative':
            c.table[0, 0] = -1
        elif change == 'base':
            c.base[0] = 100000
        else:
            c.base[0] = -5
        o = run_attention(c)
        N.call('mica_device_error', ctypes.byref(code), st)
        assert code.value == 9, change
        assert torch.equal(o[3:], good[3:])
        N.call('mica_device_error', ctypes.byref(code), st)
        assert code.value == 0


# ---- append -----------------------------------------------------------------------------
def tables(dim, n=5000):
    f = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device='cuda') / dim)
    a = torch.arange(n, dtype=torch.float64, device='cuda')[:, None] * torch.cat((f, f))
    return a.cos().bfloat16(), a.sin().bfloat16()


@pytest.mark.parametrize('heads,kv,dim', SHAPES)
@pytest.mark.parametrize('page', [16, 128])
@pytest.mark.parametrize('positions', [False, True])
def test_append(heads, kv, dim, page, positions):
    from mica_b200 import paged
    c = Case([0, 17, 700, 3], [1, 40, 0, 333], heads, kv, dim, page, seed=heads, layers=2, layer=1, pad_rows=2)
    g = torch.Generator(device='cuda').manual_seed(1)
    wide = (2 * torch.randn(c.n, (heads + 2 * kv) * dim + 8, generator=g, device='cuda')).bfloat16()
    qkv = wide[:, :(heads + 2 * kv) * dim]
    qkv[0, :dim] = 0
    qw, kw = (1 + 0.1 * torch.randn(2, dim, generator=g, device='cuda')).bfloat16()
    cos, sin = tables(dim)
    index = torch.cat([torch.arange(a, a + t) for a, t in zip(c.ctx, c.new)]).cuda()
    pos = torch.randint(0, 5000, (c.n,), generator=g, device='cuda') if positions else None
    c.pool.zero_()
    before, src = c.pool.clone(), wide.clone()
    q = paged.append(qkv, qw, kw, cos, sin, c.k, c.v, c.step(), heads, pos=pos)
    assert torch.equal(wide, src)
    p = pos[:index.numel()] if positions else index
    n = index.numel()
    x = qkv[:n].view(n, heads + 2 * kv, dim)
    ref = torch.cat((norm_rope(x[:, :heads], qw, cos[p], sin[p], 1e-6),
                     norm_rope(x[:, heads:heads + kv], kw, cos[p], sin[p], 1e-6)), 1)
    size = torch.cat((norm_rope(x[:, :heads], qw, cos[p], sin[p], 1e-6).abs().amax(-1, keepdim=True),
                      norm_rope(x[:, heads:heads + kv], kw, cos[p], sin[p], 1e-6).abs().amax(-1, keepdim=True)), 1)
    bound = U * ref.abs() + 2.0 ** -20 * 4 * size + 1e-12
    assert ((q[:n].view(n, heads, dim).double() - ref[:, :heads]).abs() <= bound[:, :heads]).all()
    assert float(q[n:].float().abs().max()) == 0.0
    b = torch.cat([torch.full((t,), i) for i, t in enumerate(c.new)]).cuda()
    page_of, slot = c.table.long()[b, index // page], index % page
    got = c.k[page_of, :, slot].double()
    assert ((got - ref[:, heads:]).abs() <= bound[:, heads:]).all()
    assert torch.equal(c.v[page_of, :, slot], x[:, heads + kv:])
    c.k[page_of, :, slot] = 0                      # nothing else was written
    c.v[page_of, :, slot] = 0
    assert torch.equal(c.pool, before)


@pytest.mark.parametrize('heads,kv,dim', [(32, 8, 128), (5, 1, 64), (16, 1, 128)])
def test_append_many_rows(heads, kv, dim):
    """A prompt of thousands of rows (the ring): ragged sequences, padding rows, one sequence without room."""
    from mica_b200 import paged
    ctx, new = [0, 300, 5, 64], [2000, 1, 900, 3000]
    c = Case(ctx, new, heads, kv, dim, 64, seed=heads, layers=2, layer=1, pad_rows=5)
    g = torch.Generator(device='cuda').manual_seed(1)
    qkv = (2 * torch.randn(c.n, (heads + 2 * kv) * dim, generator=g, device='cuda')).bfloat16()
    qw, kw = (1 + 0.1 * torch.randn(2, dim, generator=g, device='cuda')).bfloat16()
    cos, sin = tables(dim)
    c.pool.zero_()
    pos = torch.randint(0, 5000, (c.n,), generator=g, device='cuda')
    c.base[1] = 64 * c.table.shape[1]                     # its row has no slot
    q = paged.append(qkv, qw, kw, cos, sin, c.k, c.v, c.step(), heads, pos=pos)
    n = sum(new)
    x = qkv[:n].view(n, heads + 2 * kv, dim)
    ref = torch.cat((norm_rope(x[:, :heads], qw, cos[pos[:n]], sin[pos[:n]], 1e-6),
                     norm_rope(x[:, heads:heads + kv], kw, cos[pos[:n]], sin[pos[:n]], 1e-6)), 1)
    bound = U * ref.abs() + 2.0 ** -20 * 4 * ref.abs().amax(-1, keepdim=True) + 1e-12
    good = torch.ones(n, dtype=torch.bool, device='cuda')
    good[2000] = False
    assert ((q[:n].view(n, heads, dim).double() - ref[:, :heads]).abs() <= bound[:, :heads])[good].all()
    assert float(q[n:].float().abs().max()) == 0.0 and float(q[2000].float().abs().max()) == 0.0
    b = torch.cat([torch.full((t,), i) for i, t in enumerate(new)]).cuda()[good]
    index = torch.cat([torch.arange(a, a + t) for a, t in zip(ctx, new)]).cuda()[good]
    page_of, slot = c.table.long()[b, index // 64], index % 64
    assert ((c.k[page_of, :, slot].double() - ref[good][:, heads:]).abs() <= bound[good][:, heads:]).all()
    assert torch.equal(c.v[page_of, :, slot], x[good][:, heads + kv:])
    c.k[page_of, :, slot] = 0
    c.v[page_of, :, slot] = 0
    assert float(c.pool.float().abs().max()) == 0.0
    import ctypes

    from mica_b200 import _native as N
    code = ctypes.c_int(0)
    N.call('mica_device_error', ctypes.byref(code), torch.cuda.current_stream().cuda_stream)
    assert code.value == 9


def test_append_bad_indexes_write_nothing():
    import ctypes

    from mica_b200 import _native as N
    from mica_b200 import paged
    st = torch.cuda.current_stream().cuda_stream
    code = ctypes.c_int(0)
    cos, sin = tables(64, 100)
    one = torch.ones(64, dtype=torch.bfloat16, device='cuda')
    for change in ('page', 'negative', 'base', 'pos', 'table_end'):
        c = Case([5], [4], 4, 2, 64, 16, fill=0.0)
        c.pool.zero_()
        qkv = torch.ones(4, 8 * 64, dtype=torch.bfloat16, device='cuda')
        pos = torch.zeros(4, dtype=torch.int64, device='cuda')
        if change == 'page':
            c.table[0, 0] = 1000
        elif change == 'negative':
            c.table[0, 0] = -1
        elif change == 'base':
            c.base[0] = -1
        elif change == 'pos':
            pos += 100
        else:
            c.base[0] = 16 * c.table.shape[1]
        N.call('mica_device_error', ctypes.byref(code), st)
        q = paged.append(qkv, one, one, cos, sin, c.k, c.v, c.step(), 4, pos=pos)
        N.call('mica_device_error', ctypes.byref(code), st)
        assert code.value == 9, change
        assert float(c.pool.float().abs().max()) == 0.0 and float(q.float().abs().max()) == 0.0


# ---- pages --------------------------------------------------------------------------------
@pytest.mark.parametrize('shape', [(9, 3, 2, 2, 16, 64), (700, 1, 2, 1, 16, 64), (6, 36, 2, 8, 64, 128)])
@pytest.mark.parametrize('pairs', [1, 3, 'all'])
def test_copy_pages(shape, pairs):
    from mica_b200 import paged
    pool = torch.randn(shape, device='cuda').bfloat16()
    pool.view(torch.int16)[0, 0, 0, 0, 0, 0] = 0x7fff          # a NaN's bits travel as they are
    order = torch.randperm(shape[0], generator=torch.Generator().manual_seed(1)).tolist()
    n = shape[0] // 2 if pairs == 'all' else pairs
    src, dst = order[:n], order[n:2 * n]
    ref = pool.clone()
    ref[dst] = ref[src]
    paged.copy_pages(pool, src, dst)
    assert torch.equal(pool.view(torch.int16), ref.view(torch.int16))
    two = order[:1] * 2, order[1:3]                             # one page into two
    ref[two[1]] = ref[two[0]]
    paged.copy_pages(pool, *two)
    assert torch.equal(pool.view(torch.int16), ref.view(torch.int16))


def test_copy_pages_of_a_wider_buffer_and_fp32():
    from mica_b200 import paged
    wide = torch.randn(8, 100, device='cuda')
    pool = wide[:, :84]
    ref = wide.clone()
    ref[3, :84] = ref[5, :84]
    paged.copy_pages(pool, [5], [3])
    assert torch.equal(wide, ref)


@pytest.mark.parametrize('layers,kv,dim,page', [(1, 1, 64, 16), (3, 2, 128, 32), (36, 8, 128, 64), (2, 5, 64, 128)])
def test_keep_tokens(layers, kv, dim, page):
    from mica_b200 import paged
    ctx, new = [0, 3, 130, 40, 7, 16], [64, 16, 200, 1, 30, 0]
    c = Case(ctx, new, kv, kv, dim, page, seed=layers, layers=layers)
    c.pool.normal_()
    keep = [[0, 1, 5, 9, 10, 63], [3], list(range(1, 200, 2)), [0], [], []]
    most = max(len(k) for k in keep)
    kt = torch.tensor([k + [-3] * (most - len(k)) for k in keep], dtype=torch.int32, device='cuda')
    nk = torch.tensor([len(k) for k in keep], dtype=torch.int32, device='cuda')
    ref, was = c.pool.clone(), c.pool.clone()
    for b, rows in enumerate(keep):
        for j, i in enumerate(rows):
            s, d = ctx[b] + i, ctx[b] + j
            ref[c.rows[b][d // page], :, :, :, d % page] = was[c.rows[b][s // page], :, :, :, s % page]
    base = paged.keep_tokens(c.pool, c.step(), kt, nk)
    assert base.tolist() == [a + len(k) for a, k in zip(ctx, keep)]
    assert torch.equal(c.pool, ref)


def test_keep_tokens_bad_lists_change_nothing():
    import ctypes

    from mica_b200 import _native as N
    from mica_b200 import paged
    st = torch.cuda.current_stream().cuda_stream
    code = ctypes.c_int(0)
    good = [1, 3, 4]
    for bad, n in (([3, 1, 4], 3), ([1, 1, 2], 3), ([-1, 2, 3], 3), ([1, 2, 8], 3), ([0, 1, 2], 4), ([0, 1, 2], -1)):
        c = Case([5, 20], [8, 8], 2, 2, 64, 16, layers=2)
        c.pool.normal_()
        ref = c.pool.clone()
        for j, i in enumerate(good):
            s, d = 20 + i, 20 + j
            was = ref[c.rows[1][s // 16], :, :, :, s % 16].clone()
            ref[c.rows[1][d // 16], :, :, :, d % 16] = was
        N.call('mica_device_error', ctypes.byref(code), st)
        base = paged.keep_tokens(c.pool, c.step(), torch.tensor([bad, good], dtype=torch.int32, device='cuda'),
                                 torch.tensor([n, 3], dtype=torch.int32, device='cuda'))
        N.call('mica_device_error', ctypes.byref(code), st)
        assert code.value == 9 and base.tolist() == [5, 23]
        assert torch.equal(c.pool, ref)


# ---- the cache object -----------------------------------------------------------------------
def test_cache_forks_share_pages_until_one_writes():
    from mica_b200 import paged
    cache = paged.PagedCache(2, 2, 64, 12, page=16)
    a = cache.open()
    cache.step([a], [40])
    cache.pool.normal_()
    cache.commit([a], [40])
    b, c = cache.fork(a), cache.fork(a)
    assert cache.free_pages == 9 and cache.pages_of(b) == cache.pages_of(a)
    tail = cache.pages_of(a)[2]
    cache.step([a, b, c], [1, 20, 1])              # two copies, the last writer keeps the page; b takes two more
    assert cache.free_pages == 12 - 3 - 2 - 1
    tails = [cache.pages_of(s)[2] for s in (a, b, c)]
    assert len(set(tails)) == 3 and tail in tails
    for t in tails:
        assert torch.equal(cache.pool[t], cache.pool[tail])
    cache.commit([b], [2])
    assert len(cache.pages_of(b)) == 3
    cache.free(a)
    cache.free(c)
    content = torch.cat([cache.pool[p] for p in cache.pages_of(b)])
    assert cache.compact() == 3
    assert sorted(cache.pages_of(b)) == [0, 1, 2]
    assert torch.equal(torch.cat([cache.pool[p] for p in cache.pages_of(b)]), content)
    cache.free(b)
    assert cache.free_pages == 12


# ---- a run of them together --------------------------------------------------------------------
def test_a_tree_step_then_keep_equals_the_kept_tokens_appended_alone():
    """Append a tree, attend, keep one path: the cache and the next token's attention are those of the path
    appended without the other branches (same positions)."""
    from mica_b200 import paged
    heads, kv, dim = 8, 2, 128
    g = torch.Generator(device='cuda').manual_seed(2)
    cos, sin = tables(dim)
    w = (1 + 0.1 * torch.randn(2, dim, generator=g, device='cuda')).bfloat16()
    cache = paged.PagedCache(1, kv, dim, 20, page=32)
    k, v = cache.layer(0)
    rows = torch.randn(100 + 7 + 1, (heads + 2 * kv) * dim, generator=g, device='cuda').bfloat16()

    def go(sid, x, mask=None, pos=None):
        step = cache.step([sid], [x.shape[0]], mask=mask)
        q = paged.append(x, w[0], w[1], cos, sin, k, v, step, heads, pos=pos)
        return step, paged.attention(q, k, v, step, heads)

    a = cache.open()
    go(a, rows[:100])
    cache.commit([a], [100])
    b = cache.fork(a)
    parents = [[-1, 0, 0, 1, 2, 4, 3]]
    depth = [0, 1, 1, 2, 2, 3, 3]
    pos = torch.tensor([100 + d for d in depth], device='cuda')
    path = [0, 2, 4, 5]
    step, o = go(a, rows[100:107], paged.tree_mask(parents, 'cuda'), pos)
    cache.keep([a], step, [path])
    _, ob = go(b, rows[[100 + i for i in path]])
    cache.commit([b], [4])
    # one summation order differs: equal to within the rounding of the weights and outputs
    assert (o[path].float() - ob.float()).abs().max() <= 2 * U * 4
    assert cache.length(a) == cache.length(b) == 104
    ka, kb = (torch.cat([cache.pool[p, 0] for p in cache.pages_of(s)], 2)[:, :, :104] for s in (a, b))
    assert torch.equal(ka, kb)
    _, na = go(a, rows[107:])
    _, nb = go(b, rows[107:])
    assert torch.equal(na, nb)


def test_registered_ops_are_the_same_calls():
    from mica_b200 import logprobs
    c = Case([100, 7], [5, 9], 8, 2, 128, 32, seed=1, mask=tree)
    o = torch.ops.mica.cache_attention(c.q, c.k, c.v, c.table, c.base, c.cu, c.mask, 8, None, None)
    assert torch.equal(o, run_attention(c))
    z, ids = torch.randn(4, 999, device='cuda'), torch.zeros(4, 2, dtype=torch.int64, device='cuda')
    for a, b in zip(torch.ops.mica.token_logprobs(z, ids, 3), logprobs.token_logprobs(z, ids, 3)):
        assert torch.equal(a, b)
    pool = torch.randn(4, 8, device='cuda')
    ref = pool.clone()
    ref[1] = ref[3]
    torch.ops.mica.cache_copy(pool, [3], [1])
    assert torch.equal(pool, ref)


def test_gradients_are_refused():
    from mica_b200 import logprobs, paged
    c = Case([10], [2], 8, 2, 128, 32)
    c.q.requires_grad_(True)
    with pytest.raises(RuntimeError, match='no backward'):
        run_attention(c)
    with torch.no_grad():
        run_attention(c)
    z = torch.randn(2, 50, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='no backward'):
        logprobs.token_logprobs(z, torch.zeros(2, dtype=torch.int64, device='cuda'))
    with pytest.raises(RuntimeError, match='tensors on'):
        paged.attention(c.q.detach(), c.k.cpu(), c.v.cpu(), c.step(), 8)


def test_two_steps_of_one_cache_at_once():
    """Two attentions on two streams over the same pages: each has its own workspace."""
    c = Case([9000, 40], [3, 64], 32, 8, 128, 64, seed=7, mask=tree)
    d = Case([9000, 40], [3, 64], 32, 8, 128, 64, seed=7, mask=tree)
    d.k, d.v, d.q = c.k, c.v, c.q.flip(0).contiguous()
    ref = run_attention(c), run_attention(d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        a = run_attention(c)
        with torch.cuda.stream(side):
            b = run_attention(d)
        torch.cuda.synchronize()
        assert torch.equal(a, ref[0]) and torch.equal(b, ref[1])


def test_strided_norm_weights_and_positions():
    from mica_b200 import paged
    c = Case([3], [5], 4, 2, 64, 16)
    qkv = torch.randn(5, 8 * 64, device='cuda').bfloat16()
    w = torch.randn(128, device='cuda').bfloat16()
    cos, sin = tables(64)
    pos = torch.arange(10, device='cuda')
    a = paged.append(qkv, w[::2], w[1::2], cos, sin, c.k, c.v, c.step(), 4, pos=pos[::2])
    k = c.k.clone()
    b = paged.append(qkv, w[::2].clone(), w[1::2].clone(), cos, sin, c.k, c.v, c.step(), 4, pos=pos[::2].clone())
    assert torch.equal(a, b) and torch.equal(k.view(torch.int16), c.k.view(torch.int16))


def test_long_causal_extension_of_many_row_blocks():
    """Thousands of new rows over a context: row blocks of different lengths, cut anywhere in the line."""
    c = Case([100, 900], [1300, 700], 4, 1, 64, 128, seed=31)
    check_attention(c, run_attention(c, max_new=1300))


@pytest.mark.parametrize('heads,kv,dim,most', [(4, 4, 128, 130), (32, 4, 128, 40), (16, 4, 64, 70)])
@pytest.mark.parametrize('mask', [None, tree])
def test_two_tile_units_before_many_that_fill_one(heads, kv, dim, most, mask):
    """With two row tiles, units whose nodes fill one are passed over by row tile 1's warps, which may still be
    writing the rows of a two-tile unit some units back: each CTA has about 20 units, every 19th of two tiles."""
    new = [most if i % 19 == 0 else 1 + i % 3 for i in range(600)]
    c = Case([(i * 37) % 120 for i in range(600)], new, heads, kv, dim, 64, seed=heads, mask=mask)
    o = run_attention(c, max_new=most)
    check_attention(c, o)
    for _ in range(20):
        assert torch.equal(run_attention(c, max_new=most), o)


def test_strided_steps_and_their_new_values_in_a_graph():
    """Every second word of wider tables: the same bits, and a replayed graph reads what is written there."""
    from mica_b200 import paged
    heads, kv, dim = 8, 2, 64
    c = Case([100, 37, 5], [9, 1, 4], heads, kv, dim, 16, seed=2, mask=tree)
    i32 = {'dtype': torch.int32, 'device': 'cuda'}

    def spread(t):
        w = torch.full([2 * n for n in t.shape], -9, dtype=t.dtype, device='cuda')
        w[tuple(slice(None, None, 2) for _ in t.shape)] = t
        return w

    wide = [spread(t) for t in (c.table, c.base, c.cu, c.mask)]
    table, base, cu, mask = wide[0][::2, ::2], wide[1][::2], wide[2][::2], wide[3][::2, ::2]
    step = paged.Step(table, base, cu, mask=mask)
    o = run_attention(c)
    assert torch.equal(paged.attention(c.q, c.k, c.v, step, heads), o)
    cos, sin = tables(dim, 300)
    one = torch.ones(dim, dtype=torch.bfloat16, device='cuda')
    qkv = torch.randn(c.n, (heads + 2 * kv) * dim, device='cuda').bfloat16()
    keep, n = torch.tensor([[1, 3], [0, 0], [1, 2]], **i32), torch.tensor([2, 1, 2], **i32)

    def run(step, pool):
        k, v = pool[:, 0, 0], pool[:, 0, 1]
        q = paged.append(qkv, one, one, cos, sin, k, v, step, heads)
        a = paged.attention(q, k, v, step, heads)
        return a, paged.keep_tokens(pool, step, keep, n)

    pool, again = c.pool.clone(), c.pool.clone()
    for _ in range(2):
        ref = run(c.step(), pool)
        got = run(step, again)
        assert torch.equal(ref[0], got[0]) and torch.equal(ref[1], got[1])
        assert torch.equal(pool.view(torch.int16), again.view(torch.int16))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run(step, again)
    rows = c.table.flip(0).contiguous()                     # other pages, other lengths
    for t, new in ((c.table, rows), (c.base, torch.tensor([3, 20, 60], **i32)), (c.cu, torch.tensor([0, 4, 6, 14], **i32))):
        t.copy_(new)
    table.copy_(c.table)
    base.copy_(c.base)
    cu.copy_(c.cu)
    keep.copy_(torch.tensor([[1, 2], [0, 1], [4, 7]], **i32))
    c.table[c.table < 0] = 0
    table.copy_(c.table)
    pool.copy_(again)
    g.replay()
    ref = run(c.step(), pool)
    assert torch.equal(ref[0], out[0]) and torch.equal(ref[1], out[1])
    assert torch.equal(pool.view(torch.int16), again.view(torch.int16))


def _error():
    import ctypes

    from mica_b200 import _native as N
    code = ctypes.c_int(0)
    N.call('mica_device_error', ctypes.byref(code), torch.cuda.current_stream().cuda_stream)
    return code.value


@pytest.mark.parametrize('pad', [0, 3000])            # append: a warp a row, and the ring
@pytest.mark.parametrize('seqs', [3, 40, 700])        # the three ways to find a place in the line
def test_row_offsets_out_of_range_are_recorded(seqs, pad):
    """cu behind the rows: those that are there are served, by append and attention alike. cu that runs backwards
    or starts below zero: zeros. Every row is written either way."""
    from mica_b200 import paged
    heads, kv, dim = 4, 2, 64
    new = [2 + i % 3 for i in range(seqs - 1)] + [6 + pad]
    c = Case([(i * 7) % 40 for i in range(seqs)], new, heads, kv, dim, 16, seed=seqs)
    cos, sin = tables(dim, 5000)
    one = torch.ones(dim, dtype=torch.bfloat16, device='cuda')
    qkv = torch.randn(c.n, (heads + 2 * kv) * dim, device='cuda').bfloat16()
    good, was = c.cu.clone(), c.pool.clone()

    def near(a, b):
        """The line is cut elsewhere: two results, each within u (|o| + sum p |v|) of the exact one, |v| < 5.6."""
        return bool((a.float() - b.float()).abs().max() <= 2 * U * 2 * 5.6)

    def run(n):
        pool = was.clone()
        k, v = pool[:, 0, 0], pool[:, 0, 1]
        odd = [torch.full_like(c.q[:n], float('nan')) for _ in range(2)]
        del odd                                         # what the outputs' memory may hold
        step = paged.Step(c.table, c.base, c.cu)
        q = paged.append(qkv[:n], one, one, cos, sin, k, v, step, heads)
        first = _error()
        return q, paged.attention(q, k, v, step, heads), first, _error()

    _error()
    q, o, e1, e2 = run(c.n)
    assert (e1, e2) == (0, 0) and torch.isfinite(o).all()
    n = c.n - 4                                         # the last sequence passes the rows
    c.cu[-1] += 1000
    qs, os_, e1, e2 = run(n)
    assert (e1, e2) == (9, 9) and torch.equal(qs, q[:n]) and near(os_, o[:n])
    c.cu.copy_(good)
    c.cu[1] = c.cu[2] + 1                               # runs backwards
    qs, os_, e1, e2 = run(c.n)
    assert (e1, e2) == (9, 9) and float(os_.float().abs().max()) == 0.0 and torch.isfinite(qs).all()
    c.cu.copy_(good)
    c.cu[0] = -1
    qs, os_, e1, e2 = run(c.n)
    assert (e1, e2) == (9, 9) and float(os_.float().abs().max()) == 0.0
    c.cu.copy_(good)
    c.cu[0] = 1                                         # a row before the first sequence is padding
    qs, os_, e1, e2 = run(c.n)
    assert (e1, e2) == (0, 0) and float(qs[0].float().abs().max()) == 0.0 and float(os_[0].float().abs().max()) == 0.0
    assert near(os_[new[0]:], o[new[0]:])


def test_keep_tokens_of_more_sequences_than_a_grid_has_rows():
    """65541 sequences of one page each, most of which keep nothing or what they have."""
    from mica_b200 import paged
    n = 65541
    i32 = {'dtype': torch.int32, 'device': 'cuda'}
    pool = torch.randn(n, 1, 2, 1, 16, 64, device='cuda').bfloat16()
    table = torch.arange(n - 1, -1, -1, **i32)[:, None]
    base, cu = torch.full((n,), 3, **i32), 5 * torch.arange(n + 1, **i32)
    keep = torch.tensor([[0, 2, 4]], **i32).repeat(n, 1)
    count = torch.zeros(n, **i32)
    some = torch.tensor([0, 1, 5, 6, 65534, 65535, 65536, 65540], device='cuda')
    count[some] = 3
    keep[6] = torch.tensor([0, 1, 2], **i32)
    keep[65536] = torch.tensor([0, 4, 2], **i32)                    # out of order: left as it was
    ref = pool.clone()
    for b in some.tolist():
        p = n - 1 - b
        if b != 65536:
            for j, i in enumerate(keep[b].tolist()):
                ref[p, ..., 3 + j, :] = pool[p, ..., 3 + i, :]
    step = paged.Step(table, base, cu)
    _error()
    new = paged.keep_tokens(pool, step, keep, count)
    assert _error() == 9 and torch.equal(pool, ref)
    count[65536] = 0
    assert torch.equal(new, base + count)


@pytest.mark.parametrize('heads,new', [(4, 1), (4, 8), (4, 33), (4, 80)])
@pytest.mark.parametrize('power', [10, 24, 29, 31, 33, 40, 64, 100, 120])
@pytest.mark.parametrize('sign', [1, -1])
def test_attention_of_scores_of_any_size(heads, new, power, sign):
    """Scores k 2^power / 11.3, exact in fp32: all alike, a few largest ones, growing along the axis, one key of
    each size, in one tile, several, and parts that several CTAs hold. A step of one score is a factor of 2^90 at
    the least (power 10), so a row is the mean of the values at its largest score."""
    c = Case([0, 100, 300, 700, 20000], [new] * 5, heads, 1, 128, 64, seed=new, mask=tree)
    c.q.zero_()
    c.q[:, ::128] = sign * 2.0 ** (power // 2)
    for b, (kk, vv) in enumerate(c.keys):
        s = torch.arange(kk.shape[1], device='cuda')
        kk.zero_()
        kk[:, s, 0] = (torch.full_like(s, 3), 1 + s % 3, 1 + s // 64, 1 + s % 101, 1 + s // 1024)[b].bfloat16() * \
            2.0 ** (power - power // 2)
        for i in range(0, kk.shape[1], 64):
            m = min(64, kk.shape[1] - i)
            c.k[c.rows[b][i // 64], :, :m] = kk[:, i:i + m]
    o = run_attention(c, max_new=new)
    check_attention(c, o)
    assert torch.equal(o, run_attention(c, max_new=new))


@pytest.mark.parametrize('scale', [1e-38, 1e-30, 1e30])
def test_attention_scales_at_the_ends(scale):
    c = Case([300, 20000], [5, 40], 4, 1, 128, 64, seed=1, mask=tree)
    if scale > 1:                                           # powers of two, exact: one largest score
        c.q.zero_()
        c.q[:, ::128] = 1
        for b, (kk, _) in enumerate(c.keys):
            kk.zero_()
            kk[:, :, 0] = (torch.arange(kk.shape[1], device='cuda') % 128).bfloat16()
            for i in range(0, kk.shape[1], 64):
                m = min(64, kk.shape[1] - i)
                c.k[c.rows[b][i // 64], :, :m] = kk[:, i:i + m]
    check_attention(c, run_attention(c, scale=scale), scale)


@pytest.mark.parametrize('heads,kv,dim', [(32, 8, 128), (24, 8, 64)])
@pytest.mark.parametrize('more', [-1, 0, 1])
def test_append_around_the_ring(heads, kv, dim, more):
    """Row counts where a warp a row gives way to the ring."""
    from mica_b200 import paged
    n = 7 * torch.cuda.get_device_properties(0).multi_processor_count + more
    c = Case([9, 0], [n - 400, 400], heads, kv, dim, 64, seed=heads)
    g = torch.Generator(device='cuda').manual_seed(1)
    qkv = (2 * torch.randn(n, (heads + 2 * kv) * dim, generator=g, device='cuda')).bfloat16()
    qw, kw = (1 + 0.1 * torch.randn(2, dim, generator=g, device='cuda')).bfloat16()
    cos, sin = tables(dim)
    q = paged.append(qkv, qw, kw, cos, sin, c.k, c.v, c.step(), heads)
    index = torch.cat([torch.arange(9, 9 + n - 400), torch.arange(400)]).cuda()
    x = qkv.view(n, heads + 2 * kv, dim)
    ref = torch.cat((norm_rope(x[:, :heads], qw, cos[index], sin[index], 1e-6),
                     norm_rope(x[:, heads:heads + kv], kw, cos[index], sin[index], 1e-6)), 1)
    bound = U * ref.abs() + 2.0 ** -20 * 4 * ref.abs().amax(-1, keepdim=True) + 1e-12
    assert ((q.view(n, heads, dim).double() - ref[:, :heads]).abs() <= bound[:, :heads]).all()
    b = torch.cat([torch.full((t,), i) for i, t in enumerate(c.new)]).cuda()
    page_of, slot = c.table.long()[b, index // 64], index % 64
    assert ((c.k[page_of, :, slot].double() - ref[:, heads:]).abs() <= bound[:, heads:]).all()
    assert torch.equal(c.v[page_of, :, slot], x[:, heads + kv:])


def test_tangents_and_pages_that_need_gradients_are_refused():
    from torch.autograd import forward_ad as fw

    from mica_b200 import logprobs, paged
    c = Case([10], [2], 8, 2, 64, 32)
    i32 = {'dtype': torch.int32, 'device': 'cuda'}
    qkv = torch.randn(2, 12 * 64, device='cuda').bfloat16()
    cos, sin = tables(64, 100)
    one = torch.ones(64, dtype=torch.bfloat16, device='cuda')
    keep, n = torch.zeros(1, 1, **i32), torch.ones(1, **i32)
    with fw.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match='forward-mode'):
            paged.attention(fw.make_dual(c.q, c.q), c.k, c.v, c.step(), 8)
        with pytest.raises(RuntimeError, match='forward-mode'):
            paged.append(fw.make_dual(qkv, qkv), one, one, cos, sin, c.k, c.v, c.step(), 8)
        z = torch.randn(2, 50, device='cuda')
        with pytest.raises(RuntimeError, match='forward-mode'):
            logprobs.token_logprobs(fw.make_dual(z, z), torch.zeros(2, dtype=torch.int64, device='cuda'))
        paged.attention(c.q, c.k, c.v, c.step(), 8)
    pool = torch.zeros(4, 1, 2, 2, 32, 64, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    step = paged.Step(c.table.clamp(0, 3), c.base, c.cu)
    for call in (lambda: paged.copy_pages(pool, [0], [1]), lambda: paged.keep_tokens(pool, step, keep, n),
                 lambda: paged.append(qkv, one, one, cos, sin, pool[:, 0, 0], pool[:, 0, 1], step, 8)):
        with pytest.raises(RuntimeError, match='no backward'):
            call()
        with torch.no_grad():
            call()
