"""sample against a plain float64 restatement (a full sort per row): the same
token for every row, over types, vocabulary sizes, filters, ties, masked and
non-finite logits, and rows that keep from one token to all.

Tolerances: tokens are whole numbers and equal.  A cumulative weight here and
there differs by ~1e-13 of the total, and rows are drawn from u with 24 bits, so a
row lies that near a border with a chance of ~ kept * 1e-13: none among these.  The
probability is one float32 rounding of a value off by ~1e-13: 2^-24 of it, 2^-23
allowed."""
import numpy as np
import pytest
import torch

from conftest import case_banner
from speculative_decode_engine_amd import SDEError, sample, sample_workspace_size

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def reference_row(x, u, T=1.0, k=0, p=1.0, min_p=0.0):
    """x float64 [V] (the stored values); (token, probability, tokens kept)."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, 0.0, 0
    if not T >= np.float32(1e-6):
        return int(np.argmax(x)), 1.0, 1
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / float(T))))
    order = np.argsort(-x, kind="stable")
    if 0 < k < len(x):
        order = order[:k]
    if p < 1:
        c = np.cumsum(w[order])
        before = np.concatenate([[0.0], c[:-1]])
        order = order[(before < float(p) * c[-1]) | (np.arange(len(order)) == 0)]
    if min_p > 0:
        order = order[w[order] >= min(float(min_p), 1.0)]
    kept = np.sort(order[w[order] > 0])
    c = np.cumsum(w[kept])
    hit = np.nonzero(c > float(u) * c[-1])[0]
    i = int(hit[0]) if len(hit) else len(kept) - 1
    return int(kept[i]), float(w[kept[i]] / c[-1]), len(kept)


def run(logits, u, T=None, k=None, p=None, min_p=None):
    def dev(v, dt):
        return None if v is None else torch.tensor(np.asarray(v), dtype=dt).cuda()
    tokens, probs = sample(logits, dev(u, F32), dev(T, F32), dev(k, torch.int32), dev(p, F32),
                           dev(min_p, F32))
    assert tokens.dtype == torch.int32 and probs.dtype == F32
    x = logits.double().cpu().numpy()
    f = lambda v, i, d: d if v is None else np.float32(v[i])  # noqa: E731
    kept = []
    for i in range(len(x)):
        t, q, n = reference_row(x[i], np.float32(u[i]), f(T, i, 1.0), 0 if k is None else k[i],
                                f(p, i, 1.0), f(min_p, i, 0.0))
        assert int(tokens[i]) == t, f"row {i}: {int(tokens[i])}, not {t} ({n} kept)"
        assert abs(float(probs[i]) - q) <= 2.0 ** -23 * q
        kept.append(n)
    return kept


def make_logits(rng, rows, V, dtype, spread=3.0):
    x = rng.standard_normal((rows, V)) * spread
    for _ in range(min(V, 6)):
        x[np.arange(rows), rng.integers(0, V, rows)] += 4 + 3 * rng.standard_normal(rows)
    return torch.from_numpy(x).to(dtype).cuda()


FILTERS = [dict(), dict(T=0.7), dict(k=50, p=0.9, T=0.8), dict(k=1), dict(k=7, T=1.5),
           dict(p=0.95), dict(p=0.5, T=1.3), dict(p=0.0), dict(min_p=0.05), dict(k=600, p=0.97),
           dict(k=5000), dict(p=0.999, T=2.5), dict(min_p=0.001, p=0.99, T=2.0), dict(T=0.0),
           dict(min_p=1.0), dict(k=300, min_p=0.02, p=0.9)]


@pytest.mark.parametrize("V", [1, 2, 5, 63, 509, 1024, 4099, 32000, 50257, 128256])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_filters(gpu, V, dtype):
    """Every filter in one call, a row each, twice over other logits."""
    rng = np.random.default_rng(V)
    n = len(FILTERS)
    col = lambda name, d: [f.get(name, d) for f in FILTERS]  # noqa: E731
    for spread in (3.0, 0.3):
        x = make_logits(rng, n, V, dtype, spread)
        case_banner("sample", V, dtype, spread)
        kept = run(x, rng.random(n, dtype=np.float32), col("T", 1.0), col("k", 0), col("p", 1.0),
                   col("min_p", 0.0))
        assert V < 4000 or spread > 1 or max(kept) > 2000  # (flat rows keep many)


def test_u_over_its_range(gpu):
    rng = np.random.default_rng(0)
    us = [0.0, 2.0 ** -24, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0, 2.0, -1.0]
    x = make_logits(rng, 1, 3001, F32).expand(len(us), 3001).contiguous()
    case_banner("sample u")
    for kw in (dict(), dict(k=[40] * len(us)), dict(p=[0.8] * len(us)), dict(p=[0.9999] * len(us))):
        run(x, us, **kw)


@pytest.mark.parametrize("V", [700, 20000])
def test_ties(gpu, V):
    """Equal logits: kept by rising index, and cut exactly."""
    rng = np.random.default_rng(V)
    x = np.zeros((6, V))
    x[1] = rng.integers(-2, 3, V)           # five values
    x[2] = rng.integers(-40, 3, V) * 0.25
    x[3, ::2] = -np.inf
    x[4, V // 2:] = 1.0
    x[5] = -3.4028234663852886e38           # all masked by the type's lowest value
    x = torch.from_numpy(x).float().cuda()
    for kw in (dict(), dict(p=[0.5] * 6), dict(k=[V // 3] * 6), dict(k=[600] * 6, p=[0.25] * 6),
               dict(k=[3] * 6), dict(p=[0.999] * 6, min_p=[0.5] * 6), dict(T=[0.0] * 6)):
        for _ in range(3):
            case_banner("sample ties", V, kw)
            run(x, rng.random(6, dtype=np.float32), **kw)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_masked_and_nonfinite(gpu, dtype):
    rng = np.random.default_rng(1)
    V = 5003
    x = rng.standard_normal((8, V)) * 3
    lowest = float(torch.finfo(dtype).min)
    x[0] = -np.inf                          # nothing to draw
    x[1] = np.nan
    x[2, rng.permutation(V)[:V - 3]] = -np.inf
    x[3, rng.permutation(V)[:V // 2]] = np.nan
    x[4, [17, 4000]] = np.inf
    x[5, 1:] = lowest
    x[6, rng.permutation(V)[:V - 30]] = lowest
    x[7, 5] = -np.inf
    x = torch.from_numpy(x).to(dtype).cuda()
    for kw in (dict(), dict(k=[20] * 8), dict(p=[0.9] * 8), dict(T=[0.0] * 8), dict(k=[4000] * 8),
               dict(min_p=[0.1] * 8, T=[3.0] * 8), dict(T=[float("inf")] * 8),
               dict(T=[float("nan")] * 8), dict(p=[float("nan")] * 8, min_p=[float("nan")] * 8)):
        for _ in range(2):
            case_banner("sample nonfinite", dtype, kw)
            run(x, rng.random(8, dtype=np.float32), **kw)


def test_extreme_temperatures_and_values(gpu):
    rng = np.random.default_rng(2)
    x = make_logits(rng, 5, 3001, F32)
    x[1] *= 1e30
    x[2] *= 1e-30
    x[3, 0] = 3e38
    x[3, 1:] = -3e38
    x[4, 2:] -= 200.0
    for T in (1e-6, 1e-3, 50.0, 1e6, 1e38):
        case_banner("sample temperature", T)
        run(x, rng.random(5, dtype=np.float32), T=[T] * 5)
        run(x, rng.random(5, dtype=np.float32), T=[T] * 5, p=[0.7] * 5)
        run(x, rng.random(5, dtype=np.float32), T=[T] * 5, k=[33] * 5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_a_wider_buffer(gpu, dtype):
    """Strides and alignments: nothing outside a row is looked at."""
    rng = np.random.default_rng(3)
    for V, off in ((1001, 1), (998, 3), (1024, 8), (77, 5)):
        wide = torch.full((5, V + 20), 1e4, dtype=dtype, device="cuda")
        x = wide[:, off:off + V]
        x.copy_(make_logits(rng, 5, V, dtype))
        case_banner("sample strides", V, off, dtype)
        run(x, rng.random(5, dtype=np.float32), T=[0.9] * 5, k=[0, 40, 0, 0, 1],
            p=[0.9, 0.9, 1.0, 0.99, 1.0])


def test_many_rows_and_few(gpu):
    rng = np.random.default_rng(4)
    for rows, V in ((1, 152064), (300, 1000), (3, 128256), (0, 100)):
        x = make_logits(rng, rows, V, F32) if rows else torch.zeros(0, V, device="cuda")
        case_banner("sample rows", rows, V)
        if rows:
            run(x, rng.random(rows, dtype=np.float32), T=[0.8] * rows, k=[50] * rows,
                p=[0.9] * rows)
            run(x, rng.random(rows, dtype=np.float32), p=[0.92] * rows)
            run(x, rng.random(rows, dtype=np.float32))
        else:
            t, q = sample(x, torch.zeros(0, device="cuda"))
            assert t.shape == (0,) and q.shape == (0,)


def test_distribution(gpu):
    """One row under many u: the shares of the tokens are the probabilities.
    u goes over an even grid, so a token's count is off by at most one."""
    rng = np.random.default_rng(5)
    N, V = 4096, 40
    x = make_logits(rng, 1, V, F32)
    u = (torch.arange(N, device="cuda") / N).float()
    tokens, probs = sample(x.expand(N, V).contiguous(), u)
    share = torch.softmax(x[0].double(), 0).cpu()
    counts = torch.bincount(tokens.cpu().long(), minlength=V)
    assert ((counts - N * share).abs() <= 1.0 + 1e-6).all()


def test_captured_and_replayed(gpu):
    rng = np.random.default_rng(6)
    rows, V = 9, 32000
    x = make_logits(rng, rows, V, F32)
    u = torch.rand(rows, device="cuda")
    k = torch.tensor([0, 50, 0] * 3, dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 0.9, 1.0] * 3, device="cuda")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    probs = torch.zeros(rows, device="cuda")
    case_banner("sample capture")
    sample(x, u, None, k, p, None, tokens, probs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample(x, u, None, k, p, None, tokens, probs)
    for _ in range(4):
        x.copy_(make_logits(rng, rows, V, F32))
        u.copy_(torch.rand(rows, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = tokens.clone(), probs.clone()
        again = sample(x, u, None, k, p)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_refusals(gpu):
    x = torch.zeros(3, 50, device="cuda")
    u = torch.zeros(3, device="cuda")
    sample(x, u)
    for bad, error in [
            (dict(logits=x.double()), TypeError), (dict(logits=x.cpu()), TypeError),
            (dict(logits=x[0]), TypeError), (dict(logits=x.t()), ValueError),
            (dict(u=u.double()), TypeError), (dict(u=u[:2]), ValueError),
            (dict(u=None), TypeError), (dict(top_k=u), TypeError),
            (dict(top_p=u.int()), TypeError), (dict(min_p=u.cpu()), TypeError),
            (dict(temperature=u[:1]), ValueError), (dict(tokens=u), TypeError),
            (dict(probs=u[::2]), ValueError),
            (dict(workspace=torch.zeros(9)), ValueError),
            (dict(logits=torch.zeros(3, 0, device="cuda")), (ValueError, SDEError))]:
        args = dict(logits=x, u=u)
        args.update(bad)
        with pytest.raises(error):
            sample(**args)
    y = torch.zeros(2, 40000, device="cuda")
    need = sample_workspace_size(2, 40000)
    assert need > 0 and sample_workspace_size(2, 50) == 0
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    sample(y, u[:2], workspace=ws)
    with pytest.raises(SDEError) as e:
        sample(y, u[:2], workspace=ws[:-16])
    assert e.value.status == 5
