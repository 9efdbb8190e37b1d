"""Plain 64-bit forms of the paged-cache operators, and random steps, for the tests."""
import random

import torch


class Case:
    """A random step: sequences with ctx[b] committed tokens and new[b] rows, pages in random order in a
    pool whose unused slots hold `fill`."""

    def __init__(self, ctx, new, heads, kv, dim, page, seed=0, layers=1, layer=0, fill=float('nan'), pad_rows=0,
                 mask=None, device='cuda', spare=2, extra_words=0):
        g = torch.Generator(device=device).manual_seed(seed)
        rng = random.Random(seed)
        self.ctx, self.new, self.heads, self.kv, self.dim, self.page = ctx, new, heads, kv, dim, page
        need = [-(-(c + t) // page) for c, t in zip(ctx, new)]
        total = sum(need) + spare
        order = list(range(total))
        rng.shuffle(order)
        self.pool = torch.full((total, layers, 2, kv, page, dim), fill, dtype=torch.bfloat16, device=device)
        self.k, self.v = self.pool[:, layer, 0], self.pool[:, layer, 1]
        rows, at = [], 0
        width = max(need + [1])
        for n in need:
            rows.append(order[at:at + n] + [-7] * (width - n))       # never read
            at += n
        self.rows = rows
        self.n = sum(new) + pad_rows
        cu = [0]
        for t in new:
            cu.append(cu[-1] + t)
        i32 = {'dtype': torch.int32, 'device': device}
        self.table = torch.tensor(rows, **i32).view(len(ctx), width)
        self.base, self.cu = torch.tensor(ctx, **i32), torch.tensor(cu, **i32)
        self.keys = []            # per sequence: K, V [KV, keys, D]
        for b, (c, t) in enumerate(zip(ctx, new)):
            kk, vv = (torch.randn(kv, c + t, dim, generator=g, device=device).bfloat16() for _ in range(2))
            for s in range(0, c + t, page):
                p = rows[b][s // page]
                m = min(page, c + t - s)
                self.k[p, :, :m] = kk[:, s:s + m]
                self.v[p, :, :m] = vv[:, s:s + m]
            self.keys.append((kk, vv))
        self.q = (1.5 * torch.randn(self.n, heads * dim, generator=g, device=device)).bfloat16()
        self.seen = None          # per sequence [T, T] bool, or None: causal
        self.mask = None
        if mask is not None:
            self.seen = [mask(rng, t) for t in new]
            words = max([1] + [-(-t // 64) for t in new]) + extra_words
            bits = []
            for m in self.seen:
                for r in m.tolist():
                    v = sum(1 << j for j, x in enumerate(r) if x)
                    w = [v >> 64 * k & (1 << 64) - 1 for k in range(words)]
                    bits.append([x - (1 << 64) if x >> 63 else x for x in w])
            bits += [[-1] * words] * pad_rows
            self.mask = torch.tensor(bits, dtype=torch.int64, device=device).view(self.n, words)

    def step(self, **kw):
        from mica_b200 import paged
        return paged.Step(self.table, self.base, self.cu, mask=self.mask, **kw)

    def attention(self, scale=None):
        """The definition in 64 bits, [N, H D]; padding rows zero."""
        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.zeros(self.n, self.heads, self.dim, dtype=torch.float64, device=self.q.device)
        at = 0
        for b, (c, t) in enumerate(zip(self.ctx, self.new)):
            k, v = (x.double().repeat_interleave(self.heads // self.kv, 0) for x in self.keys[b])
            q = self.q[at:at + t].double().view(t, self.heads, self.dim).transpose(0, 1)
            own = torch.ones(t, t, dtype=torch.bool).tril() if self.seen is None else self.seen[b]
            seen = torch.cat((torch.ones(t, c, dtype=torch.bool), own), 1).to(q.device)
            z = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, float('-inf'))
            m = z.amax(-1, keepdim=True) if c + t else z.new_zeros(self.heads, t, 1)
            p = torch.exp(z - torch.where(m == float('-inf'), 0.0, m))
            p = torch.where(seen, p, 0.0)
            den = p.sum(-1, keepdim=True)
            p = p / torch.where(den == 0, 1.0, den)
            # a key that a row does not see adds nothing to it, whatever its value holds
            o = torch.where(torch.isfinite(v), v, 0.0)
            o = p @ o
            if not bool(torch.isfinite(v).all()):
                for s in (~torch.isfinite(v)).any(0).any(-1).nonzero().flatten().tolist():
                    odd = torch.where(torch.isfinite(v[:, s]), 0.0, v[:, s])
                    o += torch.where(seen[:, s][None, :, None], p[:, :, s:s + 1] * odd[:, None], 0.0)
            out[at:at + t] = o.transpose(0, 1)
            at += t
        return out.view(self.n, -1)


def tree(rng, t):
    """Ancestors and itself of a random tree."""
    m = torch.zeros(t, t, dtype=torch.bool)
    for i in range(t):
        p = rng.randint(-1, i - 1) if rng.random() < 0.3 else i - 1
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def holes(rng, t):
    """A mask with rows that see nothing, rows that see only later nodes, and random ones."""
    m = torch.tensor([[rng.random() < 0.4 for _ in range(t)] for _ in range(t)], dtype=torch.bool).view(t, t)
    for i in range(0, t, 3):
        m[i] = False
    return m


def norm_rope(x, w, cos, sin, eps):
    """[N, heads, D] in 64 bits."""
    x = x.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = x.shape[-1] // 2
    turned = torch.cat((-y[..., half:], y[..., :half]), -1)
    return y * cos.double()[:, None] + turned * sin.double()[:, None]
