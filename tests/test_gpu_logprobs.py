"""token_logprobs against its definition in 64 bits. Tolerance: the result is a difference of fp32 values of
size |z - m| + log S, each rounded once (2^-24), and a sum of at most V exponentials with a relative error of
2^-20 (fp32 sums in a fixed order, the exponential's error among it): absolute error at most
2^-23 (|logprob| + |z - m| + log S) + 2^-20. Entropy adds terms (m - z) e^(z-m) / S, relative 2^-20 each."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(z, ids, top):
    z = z.double()
    full = torch.log_softmax(z, 1)
    dead = (z == float('-inf')).all(1)
    full[dead] = float('-inf')
    ent = -torch.where(full > float('-inf'), full * full.exp(), 0.0).sum(1)
    lp = full.gather(1, ids.clamp(0, z.shape[1] - 1))
    lp = torch.where(ids < 0, 0.0, torch.where(ids >= z.shape[1], float('nan'), lp))
    order = torch.sort(torch.where(z.isnan(), float('inf'), z), dim=1, descending=True, stable=True).indices
    return lp, ent, full.gather(1, order[:, :top]), order[:, :top]


def check(z, ids, top):
    from mica_b200 import logprobs
    lp, ent, tl, ti = logprobs.token_logprobs(z, ids, top)
    two = ids[:, None] if ids.dim() == 1 else ids
    rl, re, rt, ri = reference(z, two, top)
    assert lp.shape == ids.shape and ent.shape == (z.shape[0],) and tl.shape == ti.shape == (z.shape[0], top)
    spread = 60.0
    for got, ref in ((lp.view(rl.shape), rl), (ent, re), (tl, rt)):
        fin = torch.isfinite(ref)
        assert torch.equal(fin, torch.isfinite(got)) and torch.equal(ref.isnan(), got.isnan())
        assert torch.equal(ref[~fin & ~ref.isnan()], got.double()[~fin & ~ref.isnan()])
        err = (got.double() - ref)[fin].abs()
        assert (err <= 2.0 ** -23 * (ref[fin].abs() + spread) + 2.0 ** -20 * (1 + ref[fin].abs())).all(), float(err.max())
    assert torch.equal(ti, ri)
    return lp, ent, tl, ti


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('n,v', [(1, 1), (1, 7), (3, 31), (2, 32), (5, 1000), (2, 4097), (1, 151936), (6, 151936),
                                 (40, 20001), (300, 5003), (700, 129)])
@pytest.mark.parametrize('top', [0, 1, 8, 32])
def test_rows_of_any_size(dtype, n, v, top):
    g = torch.Generator(device='cuda').manual_seed(n * 31 + v)
    z = (3 * torch.randn(n, v, generator=g, device='cuda')).to(dtype)
    ids = torch.randint(0, v, (n, 3), generator=g, device='cuda')
    check(z, ids, min(top, v))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_ties_go_to_the_lowest_id(dtype):
    z = torch.zeros(4, 5000, dtype=dtype, device='cuda')
    z[1, 4000:] = 1
    z[2, ::7] = 2.5
    z[3] = torch.arange(5000, device='cuda') % 3
    z[0, 1::2] = -0.0
    ids = torch.tensor([0, 4999, 7, 2], device='cuda')
    lp, ent, tl, ti = check(z, ids, 32)
    assert ti[0].tolist() == list(range(32)) and ti[1].tolist() == list(range(4000, 4032))
    assert ti[2].tolist() == [7 * i for i in range(32)]


@pytest.mark.parametrize('order', ['rising', 'falling'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_sorted_rows(order, dtype):
    """Rows in which every value is larger than all before it (and the reverse)."""
    z = torch.linspace(-20, 20, 50001, device='cuda')[None].repeat(3, 1)
    z = (z if order == 'rising' else z.flip(1)).to(dtype).contiguous()
    check(z, torch.tensor([[0, 50000], [25000, 1], [2, 3]], device='cuda'), 20)


def test_tokens_that_are_not_allowed():
    """-inf logits: single ones, all but one, all; and entropies of zero."""
    g = torch.Generator(device='cuda').manual_seed(0)
    z = torch.randn(6, 3001, generator=g, device='cuda')
    z[0, :3000] = float('-inf')
    z[1] = float('-inf')
    z[2, ::2] = float('-inf')
    z[3, 1:] = float('-inf')
    z[4, 0] = float('-inf')
    z[5, 17] = 1000.0
    ids = torch.tensor([[3000, 0], [0, 1], [0, 1], [0, 5], [0, 1], [17, 3]], device='cuda')
    lp, ent, tl, ti = check(z, ids, 8)
    assert ent[0] == 0 and ent[1] == 0 and ent[3] == 0
    assert lp[1].tolist() == [float('-inf')] * 2 and ti[1].tolist() == list(range(8))
    assert ti[0].tolist() == [3000, 0, 1, 2, 3, 4, 5, 6]


def test_nan_and_infinite_logits():
    from mica_b200 import logprobs
    z = torch.randn(3, 2000, device='cuda')
    z[0, 1500] = float('nan')
    z[0, 300] = float('nan')
    z[1, 5] = float('inf')
    lp, ent, tl, ti = logprobs.token_logprobs(z, torch.zeros(3, dtype=torch.int64, device='cuda'), 4)
    assert lp[0].isnan() and ent[0].isnan() and tl[0].isnan().all() and ti[0, :2].tolist() == [300, 1500]
    assert ti[1, 0] == 5 and lp[1].isnan() and ent[1].isnan() and tl[1].isnan().all()
    assert torch.isfinite(lp[2]) and torch.isfinite(tl[2]).all()


def test_ids_that_are_padding_or_out_of_range():
    from mica_b200 import logprobs
    z = torch.randn(2, 100, device='cuda')
    ids = torch.tensor([[-1, 99, 100], [-(2 ** 62), 0, 2 ** 62]], device='cuda')
    lp = logprobs.token_logprobs(z, ids)[0]
    ref = torch.log_softmax(z.double(), 1)
    assert lp[0, 0] == 0 and lp[1, 0] == 0 and lp[0, 2].isnan() and lp[1, 2].isnan()
    assert abs(float(lp[0, 1] - ref[0, 99])) < 1e-5 and abs(float(lp[1, 1] - ref[1, 0])) < 1e-5
    assert logprobs.token_logprobs(z, ids[:, :0])[0].shape == (2, 0)
    assert logprobs.token_logprobs(z[:0], ids[:0], 3)[3].shape == (0, 3)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_rows(dtype):
    """Columns of a wider buffer, at every offset within 16 bytes; transposed and expanded logits."""
    g = torch.Generator(device='cuda').manual_seed(0)
    wide = torch.randn(7, 5011, generator=g, device='cuda').to(dtype)
    ids = torch.randint(0, 4000, (7, 2), generator=g, device='cuda')
    for off in range(9):
        check(wide[:, off:off + 4001], ids, 5)
    check(wide[:4000].t()[:, :].contiguous().t()[:, :4001], ids, 5)
    check(wide[:1, :4001].expand(7, -1), ids, 5)
    check(wide[:, :4001], ids.t().contiguous().t(), 5)


def test_same_bits_again_on_other_streams_and_in_graphs():
    from mica_b200 import logprobs
    z = torch.randn(9, 60000, device='cuda').bfloat16()
    ids = torch.randint(0, 60000, (9, 2), device='cuda')
    ref = logprobs.token_logprobs(z, ids, 20)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            logprobs.token_logprobs(z, ids, 20)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(logprobs.token_logprobs(z, ids, 20))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, ref))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('big', [1000.0, 30000.0, 100000.0])
def test_a_dominating_logit_at_either_end(dtype, big):
    """The elements before and behind a row's 16-byte vectors weigh as they would inside one: log probability and
    entropy near zero for a logit far above the rest, at every offset within 16 bytes."""
    if dtype == torch.float16 and big > 65504:
        return
    wide = torch.randn(4, 5011, device='cuda').to(dtype)
    for off in range(17):
        z = wide[:, off:off + 4001].clone().new_zeros(4, 5011)[:, off:off + 4001]
        z.copy_(wide[:, off:off + 4001])
        z[0, 0] = z[1, 4000] = z[2, 1] = z[3, 3998] = big
        z[0, 4000] = big                              # and shared with the other end
        ids = torch.tensor([[0, 4000], [4000, 0], [1, 0], [3998, 2]], device='cuda')
        lp, ent, _, _ = check(z, ids, 2)
        assert lp[1, 0].abs() < 1e-5 and ent[1] < 1e-5 and abs(float(lp[0, 0]) + 0.6931472) < 1e-5


def check_wide(z, ids, top):
    """Logits of any finite size: the exact values are within fp32's range or infinite; each is a difference
    z - m of two fp32 values, rounded once (2^-24 of it), minus log S, and rounded again."""
    from mica_b200 import logprobs
    lp, ent, tl, ti = logprobs.token_logprobs(z, ids, top)
    rl, re, rt, ri = reference(z, ids, top)
    for got, ref in ((lp, rl), (ent, re), (tl, rt)):
        r32 = ref.float()
        fin = torch.isfinite(r32)
        assert torch.equal(fin, torch.isfinite(got)) and torch.equal(r32[~fin], got[~fin])
        err = (got.double() - ref)[fin].abs()
        assert (err <= 2.0 ** -22 * ref[fin].abs() + 2.0 ** -23 * 60 + 2.0 ** -20 * (1 + ref[fin].abs().clamp(max=60))).all(), float(err.max())
    assert torch.equal(ti, ri)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('n', [1, 5, 400])            # rows in parts, and one after another
@pytest.mark.parametrize('big', [1e5, 1e6, 5e6, 9e6, 2e7, 1e8, 5e9, 1e10, 1e12, 1e15, 1e20, 1e30, 3e38])
def test_rows_of_large_logits(dtype, n, big):
    """Maxima of any size and sign, alone, in numbers, and as a step of ordinary logits."""
    g = torch.Generator(device='cuda').manual_seed(n)
    z = torch.randn(5 * n, 3003, generator=g, device='cuda')
    z[0::5, 17] = big
    z[1::5, 100:2900] = big
    z[2::5] = -big                                    # all alike
    z[3::5] = -big
    z[3::5, 3000] = -big / 2
    z[4::5] *= big / 5                                # spread over the whole size
    ids = torch.tensor([[17, 3000, 2, 3002]], device='cuda').repeat(5 * n, 1)
    check_wide(z.to(dtype), ids, 6)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_finite_masks_in_ordinary_rows(dtype):
    """Tokens banned by the type's lowest value, or by any large one, among ordinary logits: their log
    probabilities are finite, the others' as without them; few and most of the row."""
    for mask in (torch.finfo(dtype).min, -2.5e38, -1e30, -1e12, -1e9, -7e7, -6e7, -1e7, -1e4):
        for n in (1, 5, 400):
            g = torch.Generator(device='cuda').manual_seed(n)
            z = torch.randn(2 * n, 3003, generator=g, device='cuda')
            z[0::2, 5:50] = mask
            z[1::2, 7:] = mask
            ids = torch.tensor([[6, 3000, 2, 20]], device='cuda').repeat(2 * n, 1)
            check_wide(z.to(dtype), ids, 10)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_one_allowed_token_anywhere(dtype):
    """Its log probability and the entropy are zero to the bit, in a vector or before and behind them."""
    z = torch.full((64, 3001), float('-inf'), dtype=dtype, device='cuda')
    at = torch.tensor([0, 1, 2, 3, 7, 8, 1500, 1501, 2990, 2997, 2998, 2999, 3000] * 5, device='cuda')[:64]
    row = torch.arange(64, device='cuda')
    z[row, at] = torch.linspace(-700, 900, 64, device='cuda').to(dtype)
    lp, ent, tl, ti = check(z, at, 3)
    assert (lp == 0).all() and (ent == 0).all() and (tl[:, 0] == 0).all() and torch.equal(ti[:, 0], at)
