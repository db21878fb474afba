"""batch_append and batch_attention against plain float64 restatements, over head
layouts, types, strides, page sizes, lengths from none to several partitions,
masked places that hold NaN and infinities, padding and bad pages.

Tolerances.  A stored value is off by at most half a step of its type (float32
2^-24, float16 2^-11, bfloat16 2^-8 of the value).  Attention: logits are products
of 22-bit halves summed in fp32, |logit| <= ~40 here, so a weight is off by at
most ~40 * 2^-22 + 2^-22 (exp2, the split) < 2^-16 of itself, and with the sums
an output by no more than 2^-16 of the largest |v| it averages (below 6 for
N(0, 1)): 1e-4 absolute, then the output's rounding.  Rotation: angles within
2^-32 turns + fp32 sin/cos (2^-22) times |x| < 6: 2e-6, then the rounding."""
import math

import numpy as np
import pytest
import torch

from conftest import case_banner
from speculative_decode_engine_amd import SDEError, batch_append, batch_attention
from speculative_decode_engine_amd import batch_attention_workspace_size

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def make_pool(rng, lens, bs, kvd, extra=3, dev="cuda", fill="normal"):
    """Pool and tables for these lengths; stale and unmapped places hold NaN."""
    need = [-(-max(n, 0) // bs) for n in lens]
    width = max(max(need), 1) + 1
    total = sum(need) + extra
    pool = np.full((total, 2, bs, kvd), np.nan, np.float16)
    perm = rng.permutation(total)
    tables = np.full((len(lens), width), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        tables[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
        for p in range(max(n, 0)):
            pool[tables[b, p // bs], :, p % bs] = rng.standard_normal((2, kvd))
    return torch.from_numpy(pool).to(dev), torch.from_numpy(tables).to(dev)


def attention_f64(q, pool, tables, lens, nh, nkv, dph, m):
    pool, tables, q = pool.cpu().double(), tables.cpu(), q.cpu().double()
    bs, G = pool.shape[2], nh // nkv
    out = torch.zeros(len(lens) * m, nh * dph, dtype=torch.float64)
    for b, n in enumerate(lens):
        for i in range(m):
            end = n - m + 1 + i
            pos = [p for p in range(max(end, 0)) if 0 <= int(tables[b, p // bs]) < pool.shape[0]]
            if not pos:
                continue
            rows = torch.stack([pool[int(tables[b, p // bs]), :, p % bs] for p in pos])
            k = rows[:, 0].reshape(-1, nkv, dph)
            v = rows[:, 1].reshape(-1, nkv, dph)
            for h in range(nh):
                x = k[:, h // G] @ q[b * m + i, h * dph:(h + 1) * dph] / math.sqrt(dph)
                out[b * m + i, h * dph:(h + 1) * dph] = torch.softmax(x, 0) @ v[:, h // G]
    return out


def check(got, want, dtype, absolute):
    got, want = got.cpu().double(), want.double()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - absolute - HALF_STEP[dtype] * want.abs()
    assert off.max() <= 0, f"over by {off.max():.3g}, at {np.unravel_index(off.argmax(), off.shape)}"


SHAPES = [(4, 2, 64, 16), (32, 4, 64, 16), (8, 8, 128, 32), (28, 4, 128, 8), (8, 2, 96, 12),
          (4, 4, 80, 1), (6, 1, 256, 20), (2, 2, 32, 64), (12, 4, 48, 5), (8, 1, 112, 16),
          (4, 2, 160, 16), (2, 1, 8, 16), (4, 1, 200, 16)]


@pytest.mark.parametrize("nh,nkv,dph,bs", SHAPES)
@pytest.mark.parametrize("m,dtype", [(1, F32), (3, F16), (5, BF16)])
def test_attention_shapes(gpu, nh, nkv, dph, bs, m, dtype):
    rng = np.random.default_rng(nh * 1000 + dph + m)
    lens = [0, 1, m, bs, bs + 1, 31, 32, 33, 130, 300]
    case_banner("batch_attention", nh, nkv, dph, bs, m, dtype)
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    q = torch.from_numpy(rng.standard_normal((len(lens) * m, nh * dph))).to(dtype).cuda()
    got = batch_attention(q, pool, tables, torch.tensor(lens, dtype=torch.int32).cuda(), nh, nkv,
                          dph, n_queries=m)
    assert got.dtype == dtype
    check(got, attention_f64(q, pool, tables, lens, nh, nkv, dph, m), dtype, 1e-4)


@pytest.mark.parametrize("nh,nkv,dph,bs,lens,m", [
    (8, 2, 128, 16, [4000, 17], 1), (4, 1, 64, 16, [2500], 9), (14, 2, 128, 32, [1500, 0, 700], 9),
    (2, 1, 96, 1, [1100], 2), (4, 1, 256, 16, [900, 1030], 4)])
def test_attention_partitions(gpu, nh, nkv, dph, bs, lens, m):
    """Lengths over several partitions, and row groups of more than 16 rows."""
    rng = np.random.default_rng(7)
    case_banner("batch_attention partitions", nh, nkv, dph, bs, lens, m)
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    assert batch_attention_workspace_size(len(lens), nh, nkv, dph, m, max(lens), bs) > 0
    q = torch.from_numpy(rng.standard_normal((len(lens) * m, nh * dph))).float().cuda()
    got = batch_attention(q, pool, tables, torch.tensor(lens, dtype=torch.int32).cuda(), nh, nkv,
                          dph, n_queries=m, max_len=max(lens))
    check(got, attention_f64(q, pool, tables, lens, nh, nkv, dph, m), F32, 1e-4)


@pytest.mark.parametrize("nh,nkv,dph,bs,lens,m,parts", [
    (8, 4, 72, 16, [1500, 0, 513, 512] + [40] * 66, 1, 3), (8, 4, 256, 16, [2000, 1, 0, 257, 1999], 1, 8),
    (8, 4, 80, 16, [2300, 256, 0, 2], 2, 9), (28, 4, 128, 16, [9000, 3, 4700, 5], 5, 36),
    (8, 2, 64, 16, [20000, 6], 1, 79)])
def test_attention_joins(gpu, nh, nkv, dph, bs, lens, m, parts):
    """Few and many partitions of a row, of which a short request fills one or none.
    Joining adds a rounding of fp32 per partition, far below the tolerance of a
    row of one."""
    rng = np.random.default_rng(17)
    case_banner("batch_attention joins", nh, nkv, dph, bs, m, parts)
    size = batch_attention_workspace_size(len(lens), nh, nkv, dph, m, max(lens), bs)
    assert size == len(lens) * nh * m * parts * (dph + 2) * 4
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    q = torch.from_numpy(rng.standard_normal((len(lens) * m, nh * dph))).float().cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    got = batch_attention(q, pool, tables, n, nh, nkv, dph, n_queries=m, max_len=max(lens))
    check(got, attention_f64(q, pool, tables, lens, nh, nkv, dph, m), F32, 1e-4)
    again = batch_attention(q, pool, tables, n, nh, nkv, dph, n_queries=m, max_len=max(lens))
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_nonfinite_where_hidden(gpu, dtype):
    """NaN and infinities of a window's later tokens do not reach the earlier
    queries; a finite query sees what it should."""
    rng = np.random.default_rng(3)
    nh, nkv, dph, bs, m, lens = 8, 2, 64, 16, 6, [6, 40, 77]
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    q = torch.from_numpy(rng.standard_normal((len(lens) * m, nh * dph))).to(dtype).cuda()
    clean = attention_f64(q, pool, tables, lens, nh, nkv, dph, m)
    for b, n in enumerate(lens):  # positions seen by queries 4 and 5 alone, and by 5
        for p, x in ((n - 2, float("inf")), (n - 1, float("nan"))):
            pool[int(tables[b, p // bs]), :, p % bs] = x
    case_banner("batch_attention nonfinite", dtype)
    got = batch_attention(q, pool, tables, torch.tensor(lens, dtype=torch.int32).cuda(), nh, nkv,
                          dph, n_queries=m).view(len(lens), m, -1)
    want = clean.view(len(lens), m, -1)
    check(got[:, :4], want[:, :4], dtype, 1e-4)
    assert not torch.isfinite(got[:, 4:].float()).any()


def test_attention_bad_pages_and_lengths(gpu):
    """Pages outside the pool are left out; lengths are clamped."""
    rng = np.random.default_rng(4)
    nh, nkv, dph, bs = 8, 2, 128, 16
    lens = [100, 50, 200, 40]
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    tables[0, 2], tables[0, 6] = -5, pool.shape[0]
    tables[1, :] = 1 << 30
    q = torch.from_numpy(rng.standard_normal((4, nh * dph))).float().cuda()
    given = torch.tensor([100, 50, 1000, -3], dtype=torch.int32).cuda()
    case_banner("batch_attention bad pages")
    got = batch_attention(q, pool, tables, given, nh, nkv, dph, max_len=200)
    want = attention_f64(q, pool, tables, [100, 50, 200, 0], nh, nkv, dph, 1)
    check(got, want, F32, 1e-4)
    assert (got[1] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_strides_and_extremes(gpu, dtype):
    """Rows out of a wider buffer, at odd offsets; large and tiny q; tied logits."""
    rng = np.random.default_rng(5)
    nh, nkv, dph, bs, lens = 4, 2, 64, 16, [70, 300, 1]
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    wide = torch.zeros(3, 5 * nh * dph + 3, dtype=dtype, device="cuda")
    for off in (0, 1, 8):
        q = wide[:, off:off + nh * dph]
        q.copy_(torch.from_numpy(rng.standard_normal((3, nh * dph))))
        q[0] *= 3e4 / 6
        q[1] = 0.0
        out = torch.full((3, nh * dph + 5), 7.0, dtype=dtype, device="cuda")[:, 1:1 + nh * dph]
        case_banner("batch_attention strides", dtype, off)
        batch_attention(q, pool, tables, torch.tensor(lens, dtype=torch.int32).cuda(), nh, nkv, dph,
                        out=out)
        want = attention_f64(q, pool, tables, lens, nh, nkv, dph, 1)
        check(out[1:], want[1:], dtype, 1e-4)
        # row 0: logits are below |q| |k| / 8, off by 2^-21 of that, d; a weight
        # by a factor e^d, an output by less than 2 (e^d - 1) max |v|
        real = pool[tables[0, :lens[0] // bs].long()].float().view(-1, 2, bs, nkv, dph)
        top = q[0].float().view(nh, dph).norm(dim=1).max() * real[:, 0].norm(dim=-1).max() / 8
        limit = 2 * math.expm1(float(top) * 2.0 ** -21) * 6
        assert limit < 1
        check(out[:1], want[:1], dtype, limit)
        base = out._base
        assert (base[:, 0] == 7).all() and (base[:, 1 + nh * dph:] == 7).all()


def test_attention_same_results_each_time(gpu):
    """No answer depends on scheduling, on a call before, or on the stream."""
    rng = np.random.default_rng(6)
    nh, nkv, dph, bs, lens = 8, 2, 128, 16, [3000, 5, 700]
    pool, tables = make_pool(rng, lens, bs, nkv * dph)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    q = torch.from_numpy(rng.standard_normal((3, nh * dph))).float().cuda()
    case_banner("batch_attention repeated")
    first = batch_attention(q, pool, tables, n, nh, nkv, dph, max_len=3000)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = batch_attention(q, pool, tables, n, nh, nkv, dph, max_len=3000, stream=side)
    for _ in range(3):
        assert torch.equal(first, batch_attention(q, pool, tables, n, nh, nkv, dph, max_len=3000))
    torch.cuda.synchronize()
    assert torch.equal(first, other)


def rotate_f64(x, pos, heads, dph, theta, scaling, factor):
    x = x.cpu().double().view(len(pos), heads, 2, dph // 2)
    if scaling == 2 and factor > 1:
        theta = theta * factor ** (dph / (dph - 2))
    div = factor if scaling in (1, 3) and factor > 1 else 1.0
    j = torch.arange(dph // 2, dtype=torch.float64)
    a = torch.tensor([float(p) for p in pos], dtype=torch.float64)[:, None] / div \
        * theta ** (-2 * j / dph)
    c, s = a.cos()[:, None], a.sin()[:, None]
    return torch.stack((x[:, :, 0] * c - x[:, :, 1] * s, x[:, :, 1] * c + x[:, :, 0] * s),
                       2).reshape(len(pos), heads * dph)


@pytest.mark.parametrize("nh,nkv,dph,bs", SHAPES + [(3, 1, 10, 7), (2, 1, 512, 16)])
@pytest.mark.parametrize("dtype,scaling,offset", [(F32, 0, 0), (F16, 1, 8), (BF16, 2, 3)])
def test_append(gpu, nh, nkv, dph, bs, dtype, scaling, offset):
    """Ragged tokens of several requests in no order, padding rows and bad pages
    left as they were, k_out, rows out of a wider buffer."""
    rng = np.random.default_rng(dph + nh)
    kvd, theta, factor = nkv * dph, 500000.0, 4.0
    width = 1000 // bs + 1
    tables = torch.from_numpy(rng.permutation(6 * width).reshape(6, width).astype(np.int32))
    places = [(s, p) for s in range(6) for p in (0, 1, bs - 1, bs, 517, 999) if p < width * bs]
    places = sorted(set(places))
    order = rng.permutation(len(places))
    seq = [places[i][0] for i in order] + [-1, 6, 2, 3, 4]
    pos = [places[i][1] for i in order] + [5, 5, -1, width * bs, 40]
    tables[4, 40 // bs] = -1  # (its other tokens' block, where bs makes it theirs)
    keep = [t for t in range(len(seq)) if 0 <= seq[t] < 6 and 0 <= pos[t] < width * bs
            and not (seq[t] == 4 and pos[t] // bs == 40 // bs)]
    T = len(seq)
    wide = torch.from_numpy(rng.standard_normal((T, offset + (nh + 2 * nkv) * dph + 5))).to(dtype)
    wide = wide.cuda()
    q, k, v = wide[:, offset:].split([nh * dph, kvd, kvd, wide.shape[1] - offset
                                      - (nh + 2 * nkv) * dph], 1)[:3]
    pool = torch.full((6 * width, 2, bs, kvd), 0.25, dtype=F16, device="cuda")
    q_out = torch.full((T, nh * dph), 0.5, dtype=dtype, device="cuda")
    k_out = torch.full((T, kvd), 0.5, dtype=dtype, device="cuda")
    case_banner("batch_append", nh, nkv, dph, bs, dtype, scaling, offset)
    batch_append(pool, tables.cuda(), torch.tensor(seq, dtype=torch.int32).cuda(),
                 torch.tensor(pos, dtype=torch.int32).cuda(), k, v, nh, nkv, dph, theta=theta,
                 scaling_type=scaling, scaling_factor=factor, q=q, q_out=q_out, k_out=k_out)
    qw = rotate_f64(q, [max(p, 0) for p in pos], nh, dph, theta, scaling, factor)
    kw = rotate_f64(k, [max(p, 0) for p in pos], nkv, dph, theta, scaling, factor)
    drop = [t for t in range(T) if t not in keep]
    assert (q_out[drop] == 0.5).all() and (k_out[drop] == 0.5).all()
    check(q_out[keep], qw[keep], dtype, 2e-6 + 1e-7)
    check(k_out[keep], kw[keep], dtype, 2e-6 + 1e-7)
    want = torch.full(pool.shape, 0.25, dtype=torch.float64)
    wrote = torch.zeros(pool.shape[:3], dtype=torch.bool)
    for t in keep:
        page, slot = int(tables[seq[t], pos[t] // bs]), pos[t] % bs
        want[page, 0, slot] = kw[t]
        want[page, 1, slot] = v[t].cpu().double()
        wrote[page, :, slot] = True
    check(pool, want, F16, 2e-6 + 1e-7)
    assert (pool.cpu()[~wrote] == 0.25).all()


def test_append_far_positions_and_in_place(gpu):
    """Angles hold at positions far out; q rotated where it lies."""
    rng = np.random.default_rng(1)
    nh, nkv, dph, bs = 4, 2, 128, 64
    pos = [0, 1, 65535, 1000003, 2 ** 24 + 1, 99_999_999]
    # one pool block serves every position of the long tables
    tables = torch.zeros(6, (max(pos) // bs) + 1, dtype=torch.int32, device="cuda")
    tables += torch.arange(6, dtype=torch.int32, device="cuda")[:, None]
    pool = torch.zeros(6, 2, bs, nkv * dph, dtype=F16, device="cuda")
    k = torch.from_numpy(rng.standard_normal((6, nkv * dph))).float().cuda()
    q = torch.from_numpy(rng.standard_normal((6, nh * dph))).float().cuda()
    want = rotate_f64(q, pos, nh, dph, 10000.0, 0, 1.0)
    case_banner("batch_append far")
    got = batch_append(pool, tables, torch.arange(6, dtype=torch.int32, device="cuda"),
                       torch.tensor(pos, dtype=torch.int32, device="cuda"), k, k, nh, nkv, dph,
                       q=q, q_out=q)
    assert got is q
    # float64's own product is off by pos * 2^-53 radians: 1.1e-8 * |x| here
    check(q, want, F32, 2e-6 + 1e-7)


def test_append_without_rotation_and_empty(gpu):
    rng = np.random.default_rng(2)
    pool = torch.zeros(8, 2, 16, 128, dtype=F16, device="cuda")
    tables = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    k = torch.from_numpy(rng.standard_normal((3, 128))).float().cuda()
    k[0, 0], k[1, 1] = float("inf"), float("nan")
    seq = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([9, 63, 16], dtype=torch.int32, device="cuda")
    case_banner("batch_append no rotation")
    batch_append(pool, tables, seq, pos, k, 2 * k, 2, 2, 64, rotate=False)
    for t, (page, slot) in enumerate([(4, 9), (3, 15), (5, 0)]):
        assert torch.equal(pool[page, 0, slot].nan_to_num(1), k[t].half().nan_to_num(1))
        assert torch.equal(pool[page, 1, slot].nan_to_num(1), (2 * k[t]).half().nan_to_num(1))
    before = pool.clone()
    batch_append(pool, tables, seq[:0], pos[:0], k[:0], k[:0], 2, 2, 64)
    q = torch.zeros(0, 128, device="cuda")
    assert batch_attention(q, pool, tables[:0], seq[:0], 2, 2, 64).shape == (0, 128)
    assert torch.equal(before.view(torch.int16), pool.view(torch.int16))


def test_attention_past_32_bits(gpu):
    """A pool of 2^32 elements and more: pages on both sides, and the last."""
    rng = np.random.default_rng(8)
    nh, nkv, dph, bs = 8, 8, 128, 64
    blocks = (1 << 32) // (2 * bs * nkv * dph) + 40
    pool = torch.zeros(blocks, 2, bs, nkv * dph, dtype=F16, device="cuda")
    lens = [100, 130]
    tables = torch.tensor([[blocks - 1, 0, 5], [blocks - 2, 3, blocks - 30]], dtype=torch.int32)
    used = sorted(set(tables.flatten().tolist()))
    for b in used:
        pool[b] = torch.from_numpy(rng.standard_normal((2, bs, nkv * dph))).half().cuda()
    packed = pool[used].clone()
    new = torch.tensor([[used.index(int(x)) for x in row] for row in tables], dtype=torch.int32)
    q = torch.from_numpy(rng.standard_normal((2, nh * dph))).float().cuda()
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    case_banner("batch_attention 64-bit offsets", blocks)
    got = batch_attention(q, pool, tables.cuda(), n, nh, nkv, dph)
    check(got, attention_f64(q, packed, new, lens, nh, nkv, dph, 1), F32, 1e-4)
    k = torch.from_numpy(rng.standard_normal((1, nkv * dph))).float().cuda()
    batch_append(pool, tables.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"),
                 torch.full((1,), 7, dtype=torch.int32, device="cuda"), k, k, nh, nkv, dph,
                 rotate=False)
    assert torch.equal(pool[blocks - 1, 0, 7], k[0].half())
    assert torch.equal(pool[blocks - 1, 1, 7], k[0].half())


def test_step_captured_and_replayed(gpu):
    """Append and attention in one graph, replayed with other tokens and lengths
    and with eager work between, against the eager results."""
    rng = np.random.default_rng(9)
    nh, nkv, dph, bs, B = 8, 2, 64, 16, 3
    tables = torch.from_numpy(rng.permutation(3 * 80).reshape(3, 80).astype(np.int32)).cuda()
    pool = torch.from_numpy(rng.standard_normal((240, 2, bs, nkv * dph))).half().cuda()
    seq = torch.arange(B, dtype=torch.int32, device="cuda")
    pos = torch.tensor([5, 900, 1200], dtype=torch.int32, device="cuda")
    lens = pos + 1
    q, k, v = (torch.zeros(B, w, device="cuda") for w in (nh * dph, nkv * dph, nkv * dph))
    qr, out = torch.zeros_like(q), torch.zeros_like(q)

    def step():
        batch_append(pool, tables, seq, pos, k, v, nh, nkv, dph, q=q, q_out=qr)
        batch_attention(qr, pool, tables, lens, nh, nkv, dph, out=out)

    case_banner("batch step capture")
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape)))
        k.copy_(torch.from_numpy(rng.standard_normal(k.shape)))
        v.copy_(torch.from_numpy(rng.standard_normal(v.shape)))
        pos.copy_(torch.from_numpy(rng.integers(0, 1280, B).astype(np.int32)))
        lens.copy_(pos + 1)
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        replayed, cached = out.clone(), pool.clone()
        pool.copy_(before)
        out.zero_()
        step()
        assert torch.equal(replayed, out) and torch.equal(cached, pool)


def test_refusals(gpu):
    pool = torch.zeros(8, 2, 16, 128, dtype=F16, device="cuda")
    tables = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    lens = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 128, device="cuda")
    ok = dict(nh=2, nkv=2, dph=64)
    batch_attention(q, pool, tables, lens, **ok)
    for bad, error in [
            (dict(q=q.double()), TypeError), (dict(q=q.cpu()), TypeError),
            (dict(q=q[:, ::2].expand(2, 64)), ValueError), (dict(q=q[:1]), ValueError),
            (dict(lens=lens.long()), TypeError), (dict(lens=lens.cpu()), TypeError),
            (dict(tables=tables.long()), TypeError), (dict(tables=tables.t()), ValueError),
            (dict(pool=pool[:, :, ::2]), ValueError), (dict(pool=pool.float()), TypeError),
            (dict(out=torch.zeros(2, 64, device="cuda")), ValueError),
            (dict(out=q.half()), TypeError), (dict(max_len=65), SDEError),
            (dict(max_len=-1), SDEError), (dict(nh=3), (ValueError, SDEError)),
            (dict(n_queries=0), (ValueError, SDEError)),
            (dict(workspace=torch.zeros(4, device="cpu")), ValueError)]:
        args = dict(q=q, pool=pool, tables=tables, lens=lens, **ok)
        args.update(bad)
        with pytest.raises(error):
            batch_attention(**args)
    seq = torch.zeros(2, dtype=torch.int32, device="cuda")
    k = torch.zeros(2, 128, device="cuda")
    batch_append(pool, tables, seq, seq, k, k, **ok)
    for bad, error in [
            (dict(k=k.double()), TypeError), (dict(v=k.half()), TypeError),
            (dict(v=k[:1]), ValueError), (dict(pos=seq[:1]), ValueError),
            (dict(q_out=q), ValueError), (dict(q=q.half()), TypeError),
            (dict(k_out=k.half()), TypeError), (dict(scaling_type=9), SDEError),
            (dict(theta=float("nan")), SDEError), (dict(nkv=1), ValueError)]:
        args = dict(pool=pool, tables=tables, seq=seq, pos=seq, k=k, v=k, **ok)
        args.update(bad)
        with pytest.raises(error):
            batch_append(**args)
    torch.cuda.synchronize()


def test_workspace_too_small(gpu):
    pool = torch.zeros(600, 2, 16, 64, dtype=F16, device="cuda")
    tables = torch.arange(600, dtype=torch.int32, device="cuda").view(1, 600)
    lens = torch.tensor([9000], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, 64, device="cuda")
    need = batch_attention_workspace_size(1, 1, 1, 64, 1, 9600, 16)
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    batch_attention(q, pool, tables, lens, 1, 1, 64, workspace=ws)
    with pytest.raises(SDEError) as e:
        batch_attention(q, pool, tables, lens, 1, 1, 64, workspace=ws[:-16])
    assert e.value.status == 5
