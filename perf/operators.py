"""Cases of the operators that score several-token answers over a kept context: K/V written into a
paged cache, attention of a tree of new tokens over it, pages copied and accepted tokens moved, and
the log probabilities of given tokens.

`own` false: the operators in elementary torch operations (fp32, rounded once); true: the calls a
user makes (mica_b200.paged, mica_b200.logprobs). Sequences of a case have lengths drawn from the
case's own "mix" number, so the work of a case does not depend on the input seed.
"""
import math
import random

import torch

own = False


def _calls():
    """The framework's entry points (imported only where `own` is true)."""
    from mica_b200 import logprobs, paged
    return paged, logprobs


DT = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-6
TABLE = 32768         # rows of the rotation tables


# ---- cases ----------------------------------------------------------------------------
def listed():
    att = {'op': 'attention', 'heads': 32, 'kv': 8, 'dim': 128, 'page': 64, 'causal': False}
    app = {'op': 'append', 'heads': 32, 'kv': 8, 'dim': 128, 'page': 64}
    pages = {'layers': 36, 'kv': 8, 'dim': 128, 'page': 64}
    return [
        # one next token of each of a few short conversations: latency counts
        {**att, 'name': 'attention_next_token', 'seqs': 4, 'ctx_lo': 50, 'ctx_hi': 700, 'new_lo': 1, 'new_hi': 1,
         'causal': True, 'mix': 1},
        # answers of a few tokens over ragged contexts, a tree per question, one page size down
        {**att, 'name': 'attention_answer_trees', 'page': 16, 'seqs': 16, 'ctx_lo': 1000, 'ctx_hi': 9000, 'new_lo': 17,
         'new_hi': 64, 'mix': 2},
        # a few tokens over very long documents: the cache is read once, the axis is split
        {**att, 'name': 'attention_long_documents', 'seqs': 2, 'ctx_lo': 60001, 'ctx_hi': 120000, 'new_lo': 8,
         'new_hi': 16, 'mix': 3},
        # the whole label set (255 answers of up to three tokens) as one tree over a long document
        {**att, 'name': 'attention_label_set', 'seqs': 1, 'ctx_lo': 20000, 'ctx_hi': 20000, 'new_lo': 700,
         'new_hi': 700, 'mix': 4},
        # one token each of eight sequences / a prompt of 8000 tokens in two sequences
        {**app, 'name': 'append_next_token', 'seqs': 8, 'ctx_lo': 50, 'ctx_hi': 700, 'new_lo': 1, 'new_hi': 1, 'mix': 5},
        {**app, 'name': 'append_prompt', 'seqs': 2, 'ctx_lo': 1, 'ctx_hi': 300, 'new_lo': 3001, 'new_hi': 5000, 'mix': 6},
        # a fork's partly filled last page in all layers / pages moved together
        {**pages, 'op': 'copy', 'name': 'copy_fork_tails', 'pool': 40, 'pairs': 3},
        {**pages, 'op': 'copy', 'name': 'copy_move_pages', 'pool': 150, 'pairs': 61},
        # the accepted tokens of one tree / of many trees move together behind the context
        {**pages, 'op': 'keep', 'name': 'keep_one_answer', 'seqs': 1, 'ctx_lo': 100, 'ctx_hi': 100, 'new_lo': 16,
         'new_hi': 16, 'keep': 5, 'mix': 7},
        {**pages, 'op': 'keep', 'name': 'keep_many_answers', 'seqs': 48, 'ctx_lo': 3, 'ctx_hi': 70, 'new_lo': 33,
         'new_hi': 64, 'keep': 24, 'mix': 8},
        # the readout of a few last positions, and of a long text with a bf16 head
        {'op': 'logprobs', 'name': 'logprobs_few_rows', 'rows': 6, 'vocab': 151936, 'type': 'fp32', 'given': 1, 'top': 8,
         'banned': 0.0},
        {'op': 'logprobs', 'name': 'logprobs_long_text', 'rows': 1025, 'vocab': 151936, 'type': 'bf16', 'given': 3,
         'top': 20, 'banned': 0.01},
    ]


SHAPES = ((32, 8, 128), (16, 2, 64), (6, 2, 128), (5, 1, 128), (28, 4, 128), (32, 32, 64), (24, 8, 64), (16, 16, 128))
PAGES = (16, 32, 64, 128)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('attention', 'attention', 'attention', 'append', 'copy', 'keep', 'logprobs', 'logprobs'))
    mix = rng.randrange(1 << 30)
    heads, kv, dim = rng.choice(SHAPES)
    page = rng.choice(PAGES)
    if op == 'attention':
        new = _log(rng, 1, 700)
        case = {'op': op, 'heads': heads, 'kv': kv, 'dim': dim, 'page': page, 'causal': rng.random() < 0.4,
                'seqs': _log(rng, 1, 64), 'ctx_lo': rng.choice((0, 1, 100)), 'ctx_hi': _log(rng, 100, 100000),
                'new_lo': rng.choice((1, new)), 'new_hi': new, 'mix': mix}
        most = work(listed()[3]), work(listed()[2])
        while work(case)['flops'] > most[0]['flops'] or work(case)['bytes'] > most[1]['bytes']:
            case['ctx_hi'] = max(case['ctx_lo'] + 1, case['ctx_hi'] * 2 // 3)
            case['seqs'] = max(1, case['seqs'] * 2 // 3)
        return case
    if op == 'append':
        new = _log(rng, 1, 5000)
        return {'op': op, 'heads': heads, 'kv': kv, 'dim': dim, 'page': page,
                'seqs': max(1, min(_log(rng, 1, 64), 8000 // new)), 'ctx_lo': 0,
                'ctx_hi': _log(rng, 1, 5000), 'new_lo': rng.choice((1, new)), 'new_hi': new, 'mix': mix}
    layers = rng.choice((1, 4, 12, 36))
    if op == 'copy':
        pairs = _log(rng, 1, 61)
        return {'op': op, 'layers': layers, 'kv': min(kv, 8), 'dim': dim, 'page': min(page, 64),
                'pool': 2 * pairs + rng.randint(0, 20), 'pairs': pairs}
    if op == 'keep':
        new = _log(rng, 2, 64)
        return {'op': op, 'layers': layers, 'kv': min(kv, 8), 'dim': dim, 'page': min(page, 64),
                'seqs': _log(rng, 1, 48), 'ctx_lo': 0, 'ctx_hi': _log(rng, 1, 100),
                'new_lo': rng.choice((2, new)), 'new_hi': new,
                'keep': rng.randint(1, max(1, min(24, new // 2))), 'mix': mix}
    rows = _log(rng, 1, 1025)
    return {'op': op, 'rows': rows, 'vocab': min(_log(rng, 1000, 260000), 151936 * 1025 // rows),
            'type': rng.choice(('fp32', 'bf16', 'fp16')) if rows < 500 else 'bf16', 'given': rng.randint(1, 4),
            'top': rng.choice((0, 1, 5, 8, 20)), 'banned': rng.choice((0.0, 0.01, 0.5))}


def _lengths(case):
    """Committed and new tokens of each sequence: two lists."""
    rng = random.Random(case['mix'])
    lo, hi = case['ctx_lo'], max(case['ctx_lo'], case['ctx_hi'])
    ctx = [max(lo, min(hi, _log(rng, max(lo, 1), max(hi, 1)))) for _ in range(case['seqs'])]
    new = [rng.randint(case['new_lo'], case['new_hi']) for _ in range(case['seqs'])]
    return ctx, new


def _parents(case, new):
    """A tree for each sequence: parent of each node (-1: the context). Most nodes hang from one of the
    last few before them, as answers written depth first do; some start a branch at the context."""
    rng = random.Random(case['mix'] + 1)
    return [[-1 if i == 0 or rng.random() < 0.08 else i - 1 - min(i - 1, int(rng.expovariate(0.7))) for i in range(t)]
            for t in new]


def _kept(case, new):
    """Accepted nodes of each sequence: the first few, then nodes of a later branch. A node that moves
    comes from behind the places that are written, so a second pass finds the same nodes there."""
    rng = random.Random(case['mix'] + 2)
    kept = []
    for t in new:
        n = rng.randint(1, min(case['keep'], t))
        later = list(range(n, t))
        take = sorted(rng.sample(later, min(n - rng.randint(0, n // 2), len(later))))
        kept.append(list(range(n - len(take))) + take)
    return kept


# ---- inputs ---------------------------------------------------------------------------
def prepare(case, seed):
    op = case['op']
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        x = torch.empty(shape, dtype=dtype, device='cuda')
        return x.normal_(0, std, generator=g)

    s = {'case': dict(case)}
    if op == 'logprobs':
        z = normal(case['rows'], case['vocab'], std=3.0, dtype=DT[case['type']])
        if case['banned']:
            z.masked_fill_(torch.rand(z.shape, generator=g, device='cuda') < case['banned'], float('-inf'))
        s['logits'] = z
        s['ids'] = torch.randint(0, case['vocab'], (case['rows'], case['given']), generator=g, device='cuda')
        return s
    if op == 'copy':
        s['pool'] = normal(case['pool'], case['layers'], 2, case['kv'], case['page'], case['dim'])
        order = list(range(case['pool']))
        random.Random(seed).shuffle(order)
        s['src'], s['dst'] = order[:case['pairs']], order[case['pairs']:2 * case['pairs']]
        return s
    # a step over sequences: pages in random order in a pool with a few pages to spare
    ctx, new = _lengths(case)
    page, kv, dim, layers = case['page'], case['kv'], case['dim'], case.get('layers', 1)
    need = [-(-(c + t) // page) for c, t in zip(ctx, new)]
    total = sum(need) + 3
    order = list(range(total))
    random.Random(seed).shuffle(order)
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [0] * (max(need) - n))
        at += n
    s['pool'] = normal(total, layers, 2, kv, page, dim)
    s['table'] = torch.tensor(rows, dtype=torch.int32, device='cuda')
    s['base'] = torch.tensor(ctx, dtype=torch.int32, device='cuda')
    cu = [0]
    for t in new:
        cu.append(cu[-1] + t)
    s['cu'] = torch.tensor(cu, dtype=torch.int32, device='cuda')
    s['max_new'], s['max_keys'] = max(new), max(c + t for c, t in zip(ctx, new))
    if op == 'keep':
        kept = _kept(case, new)
        most = max(len(k) for k in kept)
        s['keep'] = torch.tensor([k + [0] * (most - len(k)) for k in kept], dtype=torch.int32, device='cuda')
        s['n_keep'] = torch.tensor([len(k) for k in kept], dtype=torch.int32, device='cuda')
        return s
    s['k'], s['v'] = s['pool'][:, 0, 0], s['pool'][:, 0, 1]
    n, heads = cu[-1], case['heads']
    if op == 'attention':
        s['q'] = normal(n, heads * dim, std=1.5)
        s['scale'] = dim ** -0.5
        s['mask'] = None
        if not case['causal']:
            words = -(-max(new) // 64)
            bits = []
            for parent in _parents(case, new):
                seen = []
                for i, p in enumerate(parent):
                    seen.append((seen[p] if p >= 0 else 0) | 1 << i)
                bits += [[_signed(m >> 64 * w & (1 << 64) - 1) for w in range(words)] for m in seen]
            s['mask'] = torch.tensor(bits, dtype=torch.int64, device='cuda')
        return s
    s['qkv'] = normal(n, (heads + 2 * kv) * dim, std=2.0)
    s['q_w'], s['k_w'] = ((1 + 0.1 * normal(dim, dtype=torch.float32)).bfloat16() for _ in range(2))
    freq = 1e6 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device='cuda') / dim)
    angle = torch.arange(TABLE, dtype=torch.float64, device='cuda')[:, None] * torch.cat((freq, freq))
    s['cos'], s['sin'] = angle.cos().bfloat16(), angle.sin().bfloat16()
    # depth of each token in its tree: the position it is rotated by
    pos = []
    for c, parent in zip(ctx, _parents(case, new)):
        depth = []
        for p in parent:
            depth.append(depth[p] + 1 if p >= 0 else c)
        pos += depth
    s['pos'] = torch.tensor(pos, dtype=torch.int64, device='cuda')
    return s


def _signed(m):
    return m - (1 << 64) if m >> 63 else m


# ---- one pass -------------------------------------------------------------------------
def run(s):
    case = s['case']
    op = case['op']
    if own:
        paged, logprobs = _calls()
        if op == 'logprobs':
            lp, ent, top_lp, top_id = logprobs.token_logprobs(s['logits'], s['ids'], top=case['top'])
            return {'logprob': lp, 'entropy': ent, 'top_logprob': top_lp, 'top_id': top_id}
        if op == 'copy':
            paged.copy_pages(s['pool'], s['src'], s['dst'])
            return {'pool': s['pool']}
        step = paged.Step(s['table'], s['base'], s['cu'], max_new=s['max_new'], mask=s.get('mask'))
        if op == 'keep':
            return {'pool': s['pool'], 'base': paged.keep_tokens(s['pool'], step, s['keep'], s['n_keep'])}
        if op == 'append':
            q = paged.append(s['qkv'], s['q_w'], s['k_w'], s['cos'], s['sin'], s['k'], s['v'], step, case['heads'],
                             pos=s['pos'], eps=EPS)
            return {'q': q, 'k': s['k'], 'v': s['v']}
        return {'out': paged.attention(s['q'], s['k'], s['v'], step, case['heads'], scale=s['scale'])}
    if op == 'logprobs':
        return _plain_logprobs(s['logits'], s['ids'], case['top'])
    if op == 'copy':
        src, dst = (torch.tensor(x, device='cuda') for x in (s['src'], s['dst']))
        s['pool'][dst] = s['pool'][src]
        return {'pool': s['pool']}
    if op == 'keep':
        return _plain_keep(s, case)
    if op == 'append':
        return _plain_append(s, case)
    return _plain_attention(s, case)


def _plain_logprobs(logits, ids, top):
    z = logits.float()
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    lse = total.log()
    weight = torch.where(e > 0, (m - z) * e, 0.0).sum(1, keepdim=True, dtype=torch.float64)
    out = {'logprob': (z.gather(1, ids) - m - lse).float(), 'entropy': (lse + weight / total)[:, 0].float()}
    del e
    best, at = z.sort(dim=1, descending=True, stable=True)     # stable: ties keep the lowest id first
    return {**out, 'top_logprob': (best[:, :top] - m - lse).float(), 'top_id': at[:, :top].contiguous()}


def _slots(table, index, page):
    """Page and slot of cache index `index` [B, n] of each sequence."""
    return table.long().gather(1, index // page), index % page


def _plain_keep(s, case):
    pool, page = s['pool'], case['page']
    j = torch.arange(s['keep'].shape[1], device='cuda')
    live = j < s['n_keep'][:, None]
    # places that are not kept are written with themselves
    to = s['base'].long()[:, None] + j
    to = torch.minimum(to, (s['base'] + (s['cu'][1:] - s['cu'][:-1])).long()[:, None] - 1)
    again = torch.where(live, s['keep'].long(), to - s['base'].long()[:, None])
    sp, ss = _slots(s['table'], s['base'].long()[:, None] + again, page)
    dp, ds = _slots(s['table'], to, page)
    pool[dp.flatten(), :, :, :, ds.flatten()] = pool[sp.flatten(), :, :, :, ss.flatten()]
    return {'pool': pool, 'base': s['base'] + s['n_keep']}


def _sequence_of(s, n):
    row = torch.arange(n, device='cuda')
    b = torch.searchsorted(s['cu'][1:].long(), row, right=True)
    return b, row - s['cu'].long()[b]


def _plain_append(s, case):
    heads, kv, dim, page = case['heads'], case['kv'], case['dim'], case['page']
    n = s['qkv'].shape[0]
    x = s['qkv'].float().view(n, heads + 2 * kv, dim)
    qk = x[:, :heads + kv]
    y = qk * (qk.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = y * torch.cat((s['q_w'].float().expand(heads, dim), s['k_w'].float().expand(kv, dim)))
    turned = torch.cat((-y[..., dim // 2:], y[..., :dim // 2]), -1)
    y = (y * s['cos'].float()[s['pos']][:, None] + turned * s['sin'].float()[s['pos']][:, None]).bfloat16()
    b, i = _sequence_of(s, n)
    index = s['base'].long()[b] + i
    at, slot = s['table'].long()[b, index // page], index % page
    s['k'][at, :, slot] = y[:, heads:]
    s['v'][at, :, slot] = x[:, heads + kv:].bfloat16()
    return {'q': y[:, :heads].reshape(n, heads * dim), 'k': s['k'], 'v': s['v']}


def _visible(s, t_max, keys):
    """[B, T, S]: which keys each row of each sequence sees."""
    base, new = s['base'].long(), (s['cu'][1:] - s['cu'][:-1]).long()
    node = torch.arange(t_max, device='cuda')
    key = torch.arange(keys, device='cuda')
    j = key - base[:, None]                                             # [B, S] node of each key
    if s['mask'] is None:
        seen = j[:, None] <= node[:, None]
    else:
        rows = (s['cu'][:-1].long()[:, None] + node).clamp(max=s['mask'].shape[0] - 1)
        bits = (s['mask'][rows][..., None] >> torch.arange(64, device='cuda') & 1).bool().flatten(2)     # [B, T, W*64]
        seen = bits.gather(2, j.clamp(0, bits.shape[2] - 1)[:, None].expand(-1, t_max, -1))
    return (j < 0)[:, None] | seen & (j >= 0)[:, None] & (j < new[:, None])[:, None]


def _plain_attention(s, case):
    heads, kv, dim, page = case['heads'], case['kv'], case['dim'], case['page']
    t, keys, seqs = s['max_new'], s['max_keys'], case['seqs']
    rows = s['cu'][:-1].long()[:, None] + torch.arange(t, device='cuda')                  # [B, T]
    live = rows < s['cu'][1:, None]
    q = s['q'][rows.clamp(max=s['q'].shape[0] - 1)].float().view(seqs, t, kv, heads // kv, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kv, -1, dim)
    at, slot = _slots(s['table'], torch.arange(keys, device='cuda').expand(seqs, -1), page)
    k = s['k'][at, :, slot].float()                                                      # [B, S, KV, D]
    p = (q * s['scale']) @ k.permute(0, 2, 3, 1)                                          # [B, KV, T*G, S]
    del k
    seen = _visible(s, t, keys)[:, None, :, None].expand(-1, kv, -1, heads // kv, -1).reshape(p.shape)
    p.masked_fill_(~seen, float('-inf'))
    m = p.amax(-1, keepdim=True)
    p.sub_(torch.where(m > float('-inf'), m, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    v = s['v'][at, :, slot].float()
    o = (p @ v.transpose(1, 2)) / torch.where(total > 0, total, 1.0)
    o = o.view(seqs, kv, t, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(seqs, t, heads * dim).bfloat16()
    out = torch.empty_like(s['q'])
    # rows past a sequence's own go nowhere: they repeat that sequence's first row
    first = rows[:, :1].expand(-1, t)
    keep = torch.where(live, rows, first)
    out[keep.flatten()] = torch.where(live[..., None], o, o[:, :1]).flatten(0, 1)
    return {'out': out}


# ---- what a pass cannot do without ------------------------------------------------------
def work(case):
    op = case['op']
    if op == 'logprobs':
        size = 4 if case['type'] == 'fp32' else 2
        n = case['rows'] * case['vocab']
        return {'bytes': n * size + case['rows'] * (4 + 12 * case['given'] + 12 * case['top']), 'flops': 6 * n}
    if op == 'copy':
        one = case['layers'] * 2 * case['kv'] * case['page'] * case['dim'] * 2
        return {'bytes': 2 * case['pairs'] * one, 'flops': 0}
    ctx, new = _lengths(case)
    if op == 'keep':
        moved = sum(sum(i != j for j, i in enumerate(k)) for k in _kept(case, new))
        return {'bytes': 2 * moved * case['layers'] * 2 * case['kv'] * case['dim'] * 2 + 12 * case['seqs'], 'flops': 0}
    heads, kv, dim, n = case['heads'], case['kv'], case['dim'], sum(new)
    if op == 'append':
        return {'bytes': n * ((heads + 2 * kv) * dim * 4 + dim * 4 + 8), 'flops': n * (heads + kv) * dim * 10}
    if case['causal']:
        seen = sum(c * t + t * (t + 1) // 2 for c, t in zip(ctx, new))
    else:
        seen = 0
        for c, parent in zip(ctx, _parents(case, new)):
            depth = []
            for p in parent:
                depth.append((depth[p] if p >= 0 else 0) + 1)
            seen += c * len(parent) + sum(depth)
    return {'bytes': sum(c + t for c, t in zip(ctx, new)) * kv * dim * 4 + n * heads * dim * 4,
            'flops': 4 * heads * dim * seen}


# ---- the definitions in 64 bits ---------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'logprobs':
        lp, ent, best = [], [], []
        for z, ids in zip(s['logits'].split(64), s['ids'].split(64)):
            full = torch.log_softmax(z.double(), 1)
            lp.append(full.gather(1, ids))
            ent.append(-torch.where(full > float('-inf'), full * full.exp(), 0.0).sum(1))
            best.append(full.topk(case['top'], 1).values)
        return {'logprob': torch.cat(lp), 'entropy': torch.cat(ent), 'top_logprob': torch.cat(best), 'top_id': None}
    if op == 'copy':
        pool = s['pool'].double()
        for a, b in zip(s['src'], s['dst']):
            pool[b] = s['pool'][a].double()
        return {'pool': pool}
    ctx, new = _lengths(case)
    page = case['page']
    table = s['table'].tolist()
    if op == 'keep':
        pool = s['pool'].double()
        for b, nodes in enumerate(_kept(case, new)):
            for j, i in enumerate(nodes):
                src, dst = ctx[b] + i, ctx[b] + j
                moved = s['pool'][table[b][src // page], :, :, :, src % page]
                pool[table[b][dst // page], :, :, :, dst % page] = moved.double()
        return {'pool': pool, 'base': s['base'] + s['n_keep']}
    heads, kv, dim = case['heads'], case['kv'], case['dim']
    at = 0
    if op == 'append':
        k, v, qs = s['k'].double(), s['v'].double(), []
        half = dim // 2
        for b, (c, t) in enumerate(zip(ctx, new)):
            x = s['qkv'][at:at + t].double().view(t, heads + 2 * kv, dim)
            pos = s['pos'][at:at + t]
            cos, sin = s['cos'][pos].double()[:, None], s['sin'][pos].double()[:, None]

            def turn(h, w):
                h = h / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
                a, z = h[..., :half], h[..., half:]
                return torch.cat((a * cos[..., :half] - z * sin[..., :half], z * cos[..., half:] + a * sin[..., half:]), -1)

            qs.append(turn(x[:, :heads], s['q_w']).reshape(t, heads * dim))
            index = torch.arange(c, c + t, device='cuda')
            where, slot = s['table'][b].long()[index // page], index % page
            k[where, :, slot] = turn(x[:, heads:heads + kv], s['k_w'])
            v[where, :, slot] = x[:, heads + kv:]
            at += t
        return {'q': torch.cat(qs), 'k': k, 'v': v}
    outs = []
    trees = _parents(case, new)
    for b, (c, t) in enumerate(zip(ctx, new)):
        pages = s['table'][b, :-(-(c + t) // page)].long()
        k, v = (x[pages].double().transpose(1, 2).reshape(-1, kv, dim)[:c + t] for x in (s['k'], s['v']))
        seen = torch.zeros(t, c + t, dtype=torch.bool)
        for i in range(t):
            if case['causal']:
                seen[i, :c + i + 1] = True
            else:
                p = trees[b][i]
                seen[i] = seen[p] if p >= 0 else torch.arange(c + t) < c
                seen[i, c + i] = True
        seen = seen.cuda()
        q = s['q'][at:at + t].double().view(t, heads, dim)
        o = []
        for h in range(heads):
            z = (q[:, h] @ k[:, h * kv // heads].T) * s['scale']
            o.append(z.masked_fill(~seen, float('-inf')).softmax(-1) @ v[:, h * kv // heads])
        outs.append(torch.stack(o, 1).reshape(t, heads * dim))
        at += t
    return {'out': torch.cat(outs)}
