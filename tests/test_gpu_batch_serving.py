"""The operators over several requests, together: packed prompts rotated, appended
and attended, then decode and verify steps of requests of different lengths, tokens
drawn from the logits, against a float64 restatement that keeps every key and value
and re-reads nothing from the GPU.

Half-precision caches and weights bound what agrees: an output of one layer is off by
about 2^-10 of its size (k and v rounded to fp16, weights to fp16), so the second
layer's q by as much; 0.02 of the largest output is a margin of ten over the sum."""
import math

import numpy as np
import pytest
import torch

from conftest import case_banner
from speculative_decode_engine_amd import (KVCache, batch_append, batch_attention, prompt_attention,
                                           sample)

pytestmark = pytest.mark.gpu

F16 = torch.float16


class Model:
    """Attention sublayers with seeded projections, and an output head."""

    def __init__(self, seed, layers, nh, nkv, dph, vocab):
        g = np.random.default_rng(seed)
        self.layers, self.nh, self.nkv, self.dph, self.vocab = layers, nh, nkv, dph, vocab
        d = nh * dph
        self.d, self.width = d, d + 2 * nkv * dph
        self.emb = torch.from_numpy(g.standard_normal((vocab, d))).half()
        self.qkv = [torch.from_numpy(g.standard_normal((d, self.width)) / math.sqrt(d)).half()
                    for _ in range(layers)]
        self.head = torch.from_numpy(g.standard_normal((d, vocab)) * 3 / math.sqrt(d)).half()


def rotate_f64(x, pos, heads, dph, theta=10000.0):
    x = x.view(len(pos), heads, 2, dph // 2)
    a = torch.tensor(pos, dtype=torch.float64)[:, None] * theta ** (
        -2 * torch.arange(dph // 2, dtype=torch.float64) / dph)
    c, s = a.cos()[:, None], a.sin()[:, None]
    return torch.stack((x[:, :, 0] * c - x[:, :, 1] * s, x[:, :, 1] * c + x[:, :, 0] * s),
                       2).reshape(len(pos), heads * dph)


class Reference:
    """One request in float64: forward(tokens) appends them and gives the last
    layer's rows."""

    def __init__(self, model):
        self.m, self.n = model, 0
        self.k = [torch.zeros(0, model.nkv * model.dph, dtype=torch.float64)
                  for _ in range(model.layers)]
        self.v = [x.clone() for x in self.k]

    def forward(self, tokens):
        m = self.m
        x = m.emb[tokens].double()
        pos = list(range(self.n, self.n + len(tokens)))
        for l in range(m.layers):
            q, k, v = (x @ m.qkv[l].double()).split([m.d, m.nkv * m.dph, m.nkv * m.dph], 1)
            q, k = rotate_f64(q, pos, m.nh, m.dph), rotate_f64(k, pos, m.nkv, m.dph)
            self.k[l], self.v[l] = torch.cat((self.k[l], k)), torch.cat((self.v[l], v))
            out = torch.zeros(len(tokens), m.d, dtype=torch.float64)
            hidden = torch.arange(self.n + len(tokens))[None] > torch.tensor(pos)[:, None]
            for h in range(m.nh):
                g, s = h // (m.nh // m.nkv), slice(h * m.dph, (h + 1) * m.dph)
                c = slice(g * m.dph, (g + 1) * m.dph)
                w = q[:, s] @ self.k[l][:, c].t() / math.sqrt(m.dph)
                out[:, s] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ self.v[l][:, c]
            x = x + out
        self.n += len(tokens)
        return x

    def rewind(self, n):
        self.n = n
        self.k, self.v = [x[:n] for x in self.k], [x[:n] for x in self.v]


@pytest.mark.parametrize("nh,nkv,dph,bs", [(8, 2, 64, 16), (4, 4, 96, 8), (4, 1, 128, 32)])
def test_serving(gpu, nh, nkv, dph, bs):
    m = Model(nh + dph, 2, nh, nkv, dph, 401)
    rng = np.random.default_rng(5)
    lens = [37, 1, 120, 64]
    B, blocks = len(lens), 16 * 32 // bs
    # the pool and layout of a KVCache; its single sequence's tables are not used
    cache = KVCache(1, nkv * dph, m.layers * B * blocks, block_size=bs)
    pool = cache.pool_blocks_view()
    tables = torch.from_numpy(rng.permutation(m.layers * B * blocks).reshape(
        m.layers, B, blocks).astype(np.int32)).cuda()
    refs = [Reference(m) for _ in range(B)]
    emb, qkv = m.emb.cuda(), [w.cuda() for w in m.qkv]
    ints = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    d, kvd = m.d, nkv * dph
    case_banner("serving", nh, nkv, dph, bs)

    def near(got, want):
        want = torch.cat(want)
        assert (got.cpu().double() - want).abs().max() <= 0.02 * want.abs().max()

    # packed prompts, two padding rows behind them
    prompts = [torch.from_numpy(rng.integers(0, m.vocab, n)) for n in lens]
    starts = ints([0] + list(np.cumsum(lens)))
    pad = torch.zeros(2, dtype=torch.long)
    x = emb[torch.cat(prompts + [pad]).cuda()].float()
    seq = ints([b for b, n in enumerate(lens) for _ in range(n)] + [-1, -1])
    pos = ints([i for n in lens for i in range(n)] + [0, 0])
    for l in range(m.layers):
        rows = x.half() @ qkv[l]
        q, k, v = rows.split([d, kvd, kvd], 1)
        batch_append(pool, tables[l], seq, pos, k, v, nh, nkv, dph, q=q, q_out=q, k_out=k)
        x = x + prompt_attention(q, k, v, starts, nh, nkv, dph).float()
    near(x[:sum(lens)], [r.forward(p) for r, p in zip(refs, prompts)])

    # decode and verify steps: m new tokens of each request, then a rewind of some
    now = list(lens)
    for step, new in enumerate([1, 1, 4, 1, 3]):
        toks = torch.from_numpy(rng.integers(0, m.vocab, (B, new)))
        x = emb[toks.flatten().cuda()].float()
        seq = ints([b for b in range(B) for _ in range(new)])
        pos = ints([n + i for n in now for i in range(new)])
        n_dev = ints([n + new for n in now])
        for l in range(m.layers):
            q, k, v = (x.half() @ qkv[l]).float().split([d, kvd, kvd], 1)
            q = batch_append(pool, tables[l], seq, pos, k, v, nh, nkv, dph, q=q)
            x = x + batch_attention(q, pool, tables[l], n_dev, nh, nkv, dph, n_queries=new)
        want = [r.forward(t) for r, t in zip(refs, toks)]
        near(x, want)
        now = [n + new for n in now]
        # what is drawn is drawn from these logits
        logits = (x.half() @ m.head.cuda()).float()
        u = torch.from_numpy(rng.random(len(logits), dtype=np.float32)).cuda()
        k_row = ints([0 if i % 2 else 20 for i in range(len(logits))])
        tokens, probs = sample(logits, u, top_k=k_row)
        w = torch.softmax(logits.double(), 1)
        for i in range(len(logits)):
            wi = w[i].clone()
            if i % 2 == 0:
                wi[torch.argsort(-logits[i].double(), stable=True)[20:]] = 0
            wi /= wi.sum()
            c = wi.cumsum(0)
            t = int((c > float(u[i])).nonzero()[0])
            assert int(tokens[i]) == t
            assert abs(float(probs[i]) - float(wi[t])) <= 1e-6
        if new > 1:  # rejected drafts: the lengths alone go back
            keep = [int(rng.integers(1, new + 1)) for _ in range(B)]
            now = [n - new + kp for n, kp in zip(now, keep)]
            for r, n in zip(refs, now):
                r.rewind(n)
    torch.cuda.synchronize()
    cache.free()
