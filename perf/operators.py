"""The operators of a step over several requests, as cases whose speed is measured.

A server that holds many requests in one paged KV pool runs, per layer and step:
the new tokens' keys rotated and appended with their values (`append`), then the
attention of each request's newest tokens over its own cached positions
(`decode`); new prompts, packed one behind the other, attend within themselves
(`prompt`); and at the step's end a token is drawn from each row of logits under
that request's temperature, top-k, top-p and min-p (`sample`).

Shapes are those of the package's workload configurations (tiny, TinyLlama-1.1B,
Llama-3-8B, Qwen2.5-7B), the head sizes its tests use, and its vocabularies; `draw`
spreads over the ranges between and around them.  Every input is made on the GPU
from the seed alone: q, k, v and cached rows N(0, 1), fragmented block tables,
logits N(0, 3) with a few tokens well above the rest.

`run` computes an operator in its plain form, elementary torch operations in 32
bits (64 for angles and for the sampler's sums, whose result is a whole number),
or, with `own`, by the package's entry point.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token of each of 8 requests, TinyLlama-1.1B-shaped: the smallest append
        dict(name="append_8x1", kind="append", nh=32, nkv=4, dph=64, bs=16, seqs=8, m=1, ctx=2048,
             pad=0, type="f32", fused=False, keep_k=False, theta=10000.0, scaling=0, factor=1.0),
        # packed prompts of 7 requests, Llama-3-8B-shaped half-precision rows out of one
        # fused projection; the rotated k is kept for the prompts' own attention
        dict(name="append_prompts_8191", kind="append", nh=32, nkv=8, dph=128, bs=16, seqs=7,
             m=1170, ctx=0, pad=1, type="f16", fused=True, keep_k=True, theta=500000.0, scaling=0,
             factor=1.0),
        # 4 requests of the 4-layer dummy model at up to 128 tokens: the smallest attention
        dict(name="decode_tiny_4", kind="decode", nh=4, nkv=2, dph=64, bs=16, seqs=4, m=1, ctx=128,
             type="f32"),
        # 16 requests of different lengths up to 4K, Llama-3-8B-shaped
        dict(name="decode_16x4k", kind="decode", nh=32, nkv=8, dph=128, bs=16, seqs=16, m=1,
             ctx=4096, type="f32"),
        # a speculative verify step of 3 requests up to 32K (k = 4 drafts each), Qwen2.5-7B-shaped
        dict(name="decode_verify_3x32k", kind="decode", nh=28, nkv=4, dph=128, bs=32, seqs=3, m=5,
             ctx=32768, type="f32"),
        # a full server: 96 requests up to 8K, bf16 activations
        dict(name="decode_96x8k", kind="decode", nh=32, nkv=8, dph=128, bs=16, seqs=96, m=1,
             ctx=8192, type="bf16"),
        # five short prompts, TinyLlama-shaped, with rows behind the last one
        dict(name="prompt_5x60", kind="prompt", nh=32, nkv=4, dph=64, seqs=5, total=301, tail=19,
             type="f16", fused=True),
        # six prompts of different lengths, Llama-3-8B-shaped
        dict(name="prompt_6_4093", kind="prompt", nh=32, nkv=8, dph=128, seqs=6, total=4093, tail=0,
             type="bf16", fused=True),
        # one long prompt
        dict(name="prompt_1_8192", kind="prompt", nh=32, nkv=8, dph=128, seqs=1, total=8192, tail=0,
             type="f16", fused=False),
        # one request's next token, TinyLlama's vocabulary
        dict(name="sample_1x32000", kind="sample", rows=1, vocab=32000, type="f32", mode="top_kp"),
        # a batch whose requests ask for different filters, Llama-3's vocabulary
        dict(name="sample_24x128256", kind="sample", rows=24, vocab=128256, type="f32",
             mode="mixed"),
        # a full server's rows of half-precision logits, nucleus sampling
        dict(name="sample_192x128256", kind="sample", rows=192, vocab=128256, type="bf16",
             mode="top_p"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(4, 2, 64), (32, 4, 64), (32, 8, 128), (28, 4, 128), (8, 8, 128), (16, 2, 128), (8, 2, 96),
         (32, 32, 80), (16, 8, 256), (12, 4, 48), (8, 1, 112), (16, 2, 160), (8, 8, 32)]


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "prompt", "sample"])
    nh, nkv, dph = rng.choice(HEADS)
    bs = rng.choice([8, 16, 16, 32, 64, 12, 20])
    if kind == "append":
        m = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 2000)])
        return dict(kind=kind, nh=nh, nkv=nkv, dph=dph, bs=bs, seqs=_log(rng, 1, max(1, 8000 // m)),
                    m=m, ctx=_log(rng, 1, 30000), pad=rng.choice([0, 0, 3]),
                    type=rng.choice(["f32", "f16", "bf16"]), fused=rng.random() < 0.5,
                    keep_k=rng.random() < 0.3, theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                    scaling=rng.choice([0, 0, 1, 2]), factor=rng.choice([2.0, 4.0]))
    if kind == "decode":
        m = rng.choice([1, 1, 1, rng.randint(2, 9)])
        seqs = _log(rng, 1, 128)
        most = min(32768, (96 * 8192 * 1024) // (2 * seqs * nkv * dph))
        return dict(kind=kind, nh=nh, nkv=nkv, dph=dph, bs=bs, seqs=seqs, m=m,
                    ctx=max(m, _log(rng, 4, max(5, most))),
                    type=rng.choice(["f32", "f32", "f16", "bf16"]))
    if kind == "prompt":
        total = _log(rng, 17, 6000)
        return dict(kind=kind, nh=nh, nkv=nkv, dph=dph, seqs=min(total, _log(rng, 1, 40)),
                    total=total, tail=rng.choice([0, 0, rng.randint(1, 70)]),
                    type=rng.choice(["f16", "bf16"]), fused=rng.random() < 0.5)
    rows = _log(rng, 1, 192)
    return dict(kind="sample", rows=rows, vocab=_log(rng, 509, 152064 if rows <= 96 else 76000),
                type=rng.choice(["f32", "f32", "f16", "bf16"]),
                mode=rng.choice(["mixed", "top_kp", "top_p", "min_p", "none"]))


# ---- inputs ---------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _lengths(n, most):
    """n lengths up to `most` (the first), spread evenly over 1 .. most."""
    return [max(1, most - int(most * ((b * 0.6180339887) % 1.0))) for b in range(n)]


def _splits(n, total):
    """n lengths that add up to `total`, different and uneven."""
    w = [1.0 + 3.0 * ((b * 0.6180339887) % 1.0) for b in range(n)]
    ends = [int(round(total * sum(w[:b + 1]) / sum(w))) for b in range(n)]
    return [e - s for s, e in zip([0] + ends[:-1], ends)]


def _append_lengths(c):
    """(tokens each request has, new tokens it gets)."""
    had = [0] * c["seqs"] if c["ctx"] == 0 else [x - 1 for x in _lengths(c["seqs"], c["ctx"])]
    return had, [c["m"]] * c["seqs"]


def _pool(c, g, lengths, fill):
    """The pool float16 [blocks][2][bs][kv_dim] and fragmented tables int32 [seqs][n]."""
    need = [-(-x // c["bs"]) for x in lengths]
    n, blocks = max(need), sum(need)
    kvd = c["nkv"] * c["dph"]
    shape = (blocks + blocks // 8 + 1, 2, c["bs"], kvd)
    pool = _randn(g, *shape, dtype=torch.float16) if fill else torch.zeros(
        shape, dtype=torch.float16, device=DEV)
    perm = torch.randperm(shape[0], generator=g, device=DEV)[:blocks].to(torch.int32)
    tables = torch.zeros(c["seqs"], n, dtype=torch.int32, device=DEV)
    at = 0
    for b, x in enumerate(need):
        tables[b, :x] = perm[at:at + x]
        at += x
    return pool, tables


def _rows(c, g, n, t):
    """q, k, v rows of n tokens; views into one fused projection's rows where `fused`."""
    dq, dk = c["nh"] * c["dph"], c["nkv"] * c["dph"]
    if c["fused"]:
        x = _randn(g, n, dq + 2 * dk, dtype=t)
        return x[:, :dq], x[:, dq:dq + dk], x[:, dq + dk:]
    return _randn(g, n, dq, dtype=t), _randn(g, n, dk, dtype=t), _randn(g, n, dk, dtype=t)


MODES = {  # temperature, top_k (0: off), top_p (1: off), min_p (0: off)
    "top_kp": [(0.8, 50, 0.9, 0.0)],
    "top_p": [(0.7, 0, 0.9, 0.0), (1.0, 0, 0.95, 0.0)],
    "min_p": [(1.2, 0, 1.0, 0.05), (1.0, 200, 1.0, 0.02)],
    "none": [(1.0, 0, 1.0, 0.0), (0.6, 0, 1.0, 0.0)],
    "mixed": [(0.8, 50, 0.9, 0.0), (1.0, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 0.0),
              (1.3, 0, 0.98, 0.05), (0.6, 1000, 1.0, 0.0), (1.0, 1, 0.5, 0.0)],
}


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"c": c}
    if c["kind"] == "append":
        had, new = _append_lengths(c)
        s["pool"], s["tables"] = _pool(c, g, [h + n for h, n in zip(had, new)], fill=False)
        seq = [b for b, n in enumerate(new) for _ in range(n)] + [-1] * c["pad"]
        pos = [had[b] + i for b, n in enumerate(new) for i in range(n)] + [0] * c["pad"]
        s["seq"] = torch.tensor(seq, dtype=torch.int32).to(DEV)
        s["pos"] = torch.tensor(pos, dtype=torch.int32).to(DEV)
        s["q"], s["k"], s["v"] = _rows(c, g, len(seq), TYPES[c["type"]])
        s["q_out"] = torch.zeros(len(seq), c["nh"] * c["dph"], dtype=s["q"].dtype, device=DEV)
        s["k_out"] = torch.zeros(len(seq), c["nkv"] * c["dph"], dtype=s["q"].dtype,
                                 device=DEV) if c["keep_k"] else None
    elif c["kind"] == "decode":
        lengths = _lengths(c["seqs"], c["ctx"])
        s["pool"], s["tables"] = _pool(c, g, lengths, fill=True)
        s["lens"] = torch.tensor(lengths, dtype=torch.int32).to(DEV)
        s["q"] = _randn(g, c["seqs"] * c["m"], c["nh"] * c["dph"], dtype=TYPES[c["type"]])
    elif c["kind"] == "prompt":
        ends = [0]
        for n in _splits(c["seqs"], c["total"]):
            ends.append(ends[-1] + n)
        s["starts"] = torch.tensor(ends, dtype=torch.int32).to(DEV)
        s["q"], s["k"], s["v"] = _rows(c, g, c["total"] + c["tail"], TYPES[c["type"]])
        s["out"] = torch.zeros(c["total"] + c["tail"], c["nh"] * c["dph"], dtype=s["q"].dtype,
                               device=DEV)
    else:
        M, V = c["rows"], c["vocab"]
        x = 3.0 * _randn(g, M, V)
        few = torch.randint(0, V, (M, 12), generator=g, device=DEV)
        x.scatter_add_(1, few, 4.0 + 3.0 * _randn(g, M, 12))
        s["logits"] = x.to(TYPES[c["type"]])
        s["u"] = torch.rand(M, generator=g, device=DEV)
        modes = MODES[c["mode"]]
        rows = [modes[i % len(modes)] for i in range(M)]
        for j, (name, t) in enumerate((("temperature", torch.float32), ("top_k", torch.int32),
                                       ("top_p", torch.float32), ("min_p", torch.float32))):
            s[name] = torch.tensor([r[j] for r in rows], dtype=t).to(DEV)
    return s


# ---- one pass -------------------------------------------------------------------

def run(s):
    return (_own if own else _plain)[s["c"]["kind"]](s)


def _own_append(s):
    from speculative_decode_engine_amd import batch_append
    c = s["c"]
    batch_append(s["pool"], s["tables"], s["seq"], s["pos"], s["k"], s["v"], c["nh"], c["nkv"],
                 c["dph"], theta=c["theta"], scaling_type=c["scaling"], scaling_factor=c["factor"],
                 q=s["q"], q_out=s["q_out"], k_out=s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"], "pool": s["pool"]}


def _own_decode(s):
    from speculative_decode_engine_amd import batch_attention
    c = s["c"]
    return batch_attention(s["q"], s["pool"], s["tables"], s["lens"], c["nh"], c["nkv"], c["dph"],
                           n_queries=c["m"], max_len=c["ctx"])


def _own_prompt(s):
    from speculative_decode_engine_amd import prompt_attention
    c = s["c"]
    return prompt_attention(s["q"], s["k"], s["v"], s["starts"], c["nh"], c["nkv"], c["dph"],
                            out=s["out"])


def _own_sample(s):
    from speculative_decode_engine_amd import sample
    return sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])


_own = {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt, "sample": _own_sample}


def _angles(c, pos):
    """cos and sin of each position and rotation pair: angles in 64 bits (a far position times a
    frequency keeps no fraction in 32), rotate-half pairs (j, j + dph/2)."""
    theta, divisor = float(c["theta"]), 1.0
    if c["scaling"] == 2:
        theta *= c["factor"] ** (c["dph"] / (c["dph"] - 2.0))
    elif c["scaling"] in (1, 3):
        divisor = c["factor"]
    j = torch.arange(c["dph"] // 2, device=DEV, dtype=torch.float64)
    a = (pos.double() / divisor)[:, None] * torch.pow(theta, -2.0 * j / c["dph"])
    return a.cos().float(), a.sin().float()


def _rotate(x, cos, sin, heads, dph):
    x = x.float().reshape(x.shape[0], heads, 2, dph // 2)
    a, b, cos, sin = x[:, :, 0], x[:, :, 1], cos[:, None], sin[:, None]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), 2).reshape(x.shape[0], heads * dph)


def _plain_append(s):
    c, pool = s["c"], s["pool"]
    seq, pos = s["seq"].long(), s["pos"].long()
    n = seq.numel() - c["pad"]  # (padding rows stand last)
    seq, pos = seq[:n], pos[:n]
    cos, sin = _angles(c, pos)
    s["q_out"][:n] = _rotate(s["q"][:n], cos, sin, c["nh"], c["dph"]).to(s["q"].dtype)
    k = _rotate(s["k"][:n], cos, sin, c["nkv"], c["dph"])
    block, slot = s["tables"][seq, pos // c["bs"]].long(), pos % c["bs"]
    pool[block, 0, slot] = k.half()
    pool[block, 1, slot] = s["v"][:n].half()
    if s["k_out"] is not None:
        s["k_out"][:n] = k.to(s["k"].dtype)
    return {"q": s["q_out"], "k": s["k_out"], "pool": pool}


def _plain_decode(s):
    c = s["c"]
    B, m, nh, nkv, dph, L = c["seqs"], c["m"], c["nh"], c["nkv"], c["dph"], c["ctx"]
    G = nh // nkv
    pos = torch.arange(L, device=DEV)
    block, slot = s["tables"][:, pos // c["bs"]].long(), (pos % c["bs"])[None]
    kt = s["pool"][block, 0, slot].view(B, L, nkv, dph).permute(0, 2, 3, 1).float().contiguous()
    q = s["q"].float().view(B, m, nkv, G, dph).transpose(1, 2).reshape(B, nkv, m * G, dph)
    x = (q @ kt).view(B, nkv, m, G, L) * dph ** -0.5
    del kt
    # query i of a request sees all but the last m - 1 - i of its positions
    ends = s["lens"][:, None] - (m - 1 - torch.arange(m, device=DEV))[None]
    seen = (pos < ends[..., None])[:, None, :, None]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(B, nkv, m * G, L)
    v = s["pool"][block, 1, slot].view(B, L, nkv, dph).transpose(1, 2).float().contiguous()
    out = (p @ v).view(B, nkv, m, G, dph).transpose(1, 2)
    return out.reshape(B * m, nh * dph).to(s["q"].dtype)


def _plain_prompt(s):
    c = s["c"]
    nh, nkv, dph, T = c["nh"], c["nkv"], c["dph"], c["total"]
    q = s["q"][:T].float().view(T, nh, dph).transpose(0, 1).contiguous()
    k = s["k"][:T].float().view(T, nkv, dph).permute(1, 2, 0)
    v = s["v"][:T].float().view(T, nkv, dph).transpose(0, 1)
    row = torch.arange(T, device=DEV)
    part = torch.searchsorted(s["starts"][1:], row, right=True)
    seen = (part[:, None] == part[None]) & (row[:, None] >= row[None])
    x = q @ k.repeat_interleave(nh // nkv, 0).contiguous()
    x = torch.where(seen, x * dph ** -0.5, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    del x
    p /= p.sum(-1, keepdim=True)
    out = p @ v.repeat_interleave(nh // nkv, 0).contiguous()
    s["out"][:T] = out.transpose(0, 1).reshape(T, nh * dph).to(s["out"].dtype)
    return s["out"]


def _plain_sample(s):
    """In 64 bits: which token is drawn hangs on sums next to a border.  top_k, then top_p of what
    that leaves, then min_p; ties by index; the token where the sum in index order passes u."""
    V = s["logits"].shape[1]
    x = s["logits"].double()
    hot = s["temperature"] >= 1e-6
    t = torch.where(hot, s["temperature"], 1.0).double()[:, None]
    x, order = x.sort(dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / t)
    rank = torch.arange(V, device=DEV)[None]
    k = torch.where(hot, torch.where(s["top_k"] > 0, s["top_k"], V), 1)[:, None]
    w = torch.where(rank < k, w, 0.0)
    sums = w.cumsum(1)
    before = torch.cat((torch.zeros_like(sums[:, :1]), sums[:, :-1]), 1)
    p = torch.where(s["top_p"] < 1, s["top_p"].double(), 2.0)[:, None]
    w = torch.where((before < p * sums[:, -1:]) | (rank == 0), w, 0.0)
    w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    sums = w.cumsum(1)
    total = sums[:, -1:]
    passed = sums > s["u"].double()[:, None] * total
    token = torch.where(passed, rank, V).amin(1)
    prob = (w.gather(1, token[:, None].clamp(max=V - 1)) / total)[:, 0]
    return token.int(), prob.float()


_plain = {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt,
          "sample": _plain_sample}


# ---- the same in 64 bits, from the definitions ------------------------------------

def exact(case, seed):
    return {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt,
            "sample": _exact_sample}[case["kind"]](prepare(case, seed))


def _exact_append(s):
    c, d = s["c"], s["c"]["dph"]
    half = d // 2
    theta = c["theta"] * (c["factor"] ** (d / (d - 2)) if c["scaling"] == 2 else 1)
    scale = c["factor"] if c["scaling"] in (1, 3) else 1.0
    freq = torch.tensor([theta ** (-2 * j / d) / scale for j in range(half)],
                        dtype=torch.float64).to(DEV)
    # the rotation as a product of complex numbers
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                       s["pos"].double().view(-1, 1, 1) * freq)

    def rotated(x, heads):
        x = x.double().reshape(-1, heads, d)
        z = torch.complex(x[..., :half], x[..., half:]) * turn
        return torch.cat((z.real, z.imag), -1).reshape(-1, heads * d)

    live = s["seq"] >= 0
    q = rotated(s["q"], c["nh"]) * live[:, None]
    k = rotated(s["k"], c["nkv"]) * live[:, None]
    pool = s["pool"].double()
    flat = pool.view(-1, pool.shape[-1])
    seq, pos = s["seq"][live].long(), s["pos"][live].long()
    at = s["tables"][seq].long().gather(1, (pos // c["bs"])[:, None])[:, 0] * 2 * c["bs"]
    at += pos % c["bs"]
    flat[at] = k[live]
    flat[at + c["bs"]] = s["v"][live].double()
    return {"q": q, "k": k if c["keep_k"] else None, "pool": pool}


def _exact_decode(s):
    c = s["c"]
    G, d, bs = c["nh"] // c["nkv"], c["dph"], c["bs"]
    rows = []
    for b, n in enumerate(s["lens"].tolist()):
        kv = s["pool"][s["tables"][b, :-(-n // bs)].long()].double()
        kv = kv.transpose(0, 1).reshape(2, -1, c["nkv"], d)[:, :n].permute(0, 2, 1, 3).contiguous()
        kt = kv[0].transpose(1, 2).contiguous()
        for i in range(c["m"]):
            q = s["q"][b * c["m"] + i].double().view(c["nkv"], G, d)
            end = max(0, n - (c["m"] - 1 - i))
            if end == 0:
                rows.append(torch.zeros(c["nh"] * d, dtype=torch.float64, device=DEV))
                continue
            p = torch.softmax(torch.bmm(q, kt)[:, :, :end] / math.sqrt(d), -1)
            rows.append(torch.bmm(p, kv[1, :, :end]).reshape(-1))
    return torch.stack(rows)


def _exact_prompt(s):
    c = s["c"]
    G, d = c["nh"] // c["nkv"], c["dph"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    ends = s["starts"].tolist()
    for a, b in zip(ends[:-1], ends[1:]):
        n = b - a
        hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
        for h in range(c["nh"]):
            g = h // G
            q = s["q"][a:b, h * d:(h + 1) * d].double()
            k = s["k"][a:b, g * d:(g + 1) * d].double()
            x = torch.mm(q, k.t().contiguous()).div_(math.sqrt(d)).masked_fill_(hidden, -math.inf)
            out[a:b, h * d:(h + 1) * d] = torch.mm(torch.softmax(x, -1),
                                                   s["v"][a:b, g * d:(g + 1) * d].double())
    return out


def _exact_sample(s):
    tokens, probs = [], []
    for i in range(s["logits"].shape[0]):
        x = s["logits"][i].double()
        T, k = float(s["temperature"][i]), int(s["top_k"][i])
        if T < 1e-6:
            tokens.append(int((x == x.max()).nonzero()[0]))
            probs.append(1.0)
            continue
        w = ((x - x.max()) / T).exp()
        order = torch.argsort(-x, stable=True)
        order = order[:k] if k > 0 else order
        p = w[order]
        if float(s["top_p"][i]) < 1:
            share = p.cumsum(0)
            n = 1 + int((share < float(s["top_p"][i]) * share[-1]).sum())
            order, p = order[:n], p[:n]
        order = order[p >= float(s["min_p"][i])].sort().values
        share = w[order].cumsum(0)
        n = int((share <= float(s["u"][i]) * share[-1]).sum())
        tokens.append(int(order[n]))
        probs.append(float(w[order[n]] / share[-1]))
    return (torch.tensor(tokens, dtype=torch.int32),
            torch.tensor(probs, dtype=torch.float64).to(DEV))


# ---- what one pass cannot do without ----------------------------------------------

def work(case):
    c, size = case, {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * size + 28 * c["rows"], "flops": 4 * n}
    dq, dk = c["nh"] * c["dph"], c["nkv"] * c["dph"]
    if c["kind"] == "append":
        n = sum(_append_lengths(c)[1])
        rows = 2 * dq * size + 2 * dk * size + 2 * dk * 2 + (dk * size if c["keep_k"] else 0)
        return {"bytes": n * (rows + 12), "flops": 3 * n * (dq + dk)}
    if c["kind"] == "decode":
        lengths = _lengths(c["seqs"], c["ctx"])
        keys = sum(max(0, n - c["m"] + 1 + i) for n in lengths for i in range(c["m"]))
        return {"bytes": sum(lengths) * 4 * dk + sum(-(-n // c["bs"]) * 4 for n in lengths)
                + c["seqs"] * (4 + 2 * c["m"] * dq * size), "flops": 4 * keys * dq}
    keys = sum(n * (n + 1) // 2 for n in _splits(c["seqs"], c["total"]))
    return {"bytes": c["total"] * 2 * (dq + dk) * size, "flops": 4 * keys * dq}
