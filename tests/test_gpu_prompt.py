"""prompt_attention against a plain float64 restatement: head layouts, types,
packed sequences of no token to several tiles, strides, rows behind the last
sequence, non-finite keys and values where they are hidden.

Tolerance: a weight is rounded once to the inputs' type, half a step of it
(float16 2^-11, bfloat16 2^-8), so an output is off by that times sum p |v|; fp32
logits below ~40 add 2^-17 of it, sums less: 2^-16 sum p |v| in all; then the
output's own rounding, half a step of the value."""
import math

import numpy as np
import pytest
import torch

from conftest import case_banner
from speculative_decode_engine_amd import SDEError, prompt_attention

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def reference(q, k, v, starts, nh, nkv, dph):
    """(out, sum p |v|) in float64; rows of no sequence are 0."""
    q, k, v = q.double(), k.double(), v.double()
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        if n <= 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(nh):
            g = h // (nh // nkv)
            c, d = slice(h * dph, (h + 1) * dph), slice(g * dph, (g + 1) * dph)
            x = torch.mm(q[a:b, c], k[a:b, d].t().contiguous()) / math.sqrt(dph)
            p = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
            out[a:b, c] = torch.mm(p, v[a:b, d])
            mag[a:b, c] = torch.mm(p, v[a:b, d].abs())
    return out, mag


def check(got, want, mag, dtype):
    h = HALF_STEP[dtype]
    assert torch.isfinite(got.float()).all()
    over = (got.double() - want).abs() - (h + 2.0 ** -16) * mag - h * want.abs() - 1e-6
    assert over.max() <= 0, f"over by {float(over.max()):.3g}"


def make(rng, T, nh, nkv, dph, dtype, fused=False):
    dq, dk = nh * dph, nkv * dph
    if fused:
        x = torch.from_numpy(rng.standard_normal((T, dq + 2 * dk))).to(dtype).cuda()
        return x[:, :dq], x[:, dq:dq + dk], x[:, dq + dk:]
    return [torch.from_numpy(rng.standard_normal((T, w))).to(dtype).cuda() for w in (dq, dk, dk)]


def ends(lens):
    return [0] + list(np.cumsum(lens))


SHAPES = [(4, 2, 64), (32, 4, 64), (8, 8, 128), (28, 4, 128), (8, 2, 96), (4, 4, 80), (6, 1, 256),
          (2, 2, 32), (12, 4, 48), (8, 1, 112), (4, 2, 160), (2, 1, 8), (4, 1, 200), (3, 3, 192)]


@pytest.mark.parametrize("nh,nkv,dph", SHAPES)
@pytest.mark.parametrize("dtype,fused", [(F16, True), (BF16, False)])
def test_shapes(gpu, nh, nkv, dph, dtype, fused):
    rng = np.random.default_rng(nh + dph)
    lens = [1, 0, 2, 31, 33, 64, 0, 65, 127, 128, 129, 300, 5]
    starts, tail = ends(lens), 7
    T = starts[-1] + tail
    q, k, v = make(rng, T, nh, nkv, dph, dtype, fused)
    out = torch.full((T, nh * dph), 0.5, dtype=dtype, device="cuda")
    case_banner("prompt_attention", nh, nkv, dph, dtype)
    prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32).cuda(), nh, nkv, dph, out=out)
    want, mag = reference(q, k, v, starts, nh, nkv, dph)
    check(out[:-tail], want[:-tail], mag[:-tail], dtype)
    assert (out[-tail:] == 0.5).all()


@pytest.mark.parametrize("lens", [[1], [2000], [700, 1300], [3] * 200, [1] * 300 + [500],
                                  [0, 0, 0], [0] * 100 + [40] + [0] * 30])
def test_lengths(gpu, lens):
    """Single tokens, long prompts, more sequences than a wave has lanes."""
    rng = np.random.default_rng(len(lens))
    nh, nkv, dph = 8, 2, 64
    starts = ends(lens)
    T = max(starts[-1], 1)
    q, k, v = make(rng, T, nh, nkv, dph, F16)
    case_banner("prompt_attention lengths", lens[:3], len(lens))
    out = prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32).cuda(), nh, nkv, dph)
    want, mag = reference(q, k, v, starts, nh, nkv, dph)
    check(out, want, mag, F16)


@pytest.mark.parametrize("nh,nkv,dph,lens,dtype", [
    (64, 8, 64, [1030, 1070], F16), (64, 2, 56, [2100], BF16), (32, 8, 128, [2101, 2099], BF16),
    (32, 8, 128, [4111], F16), (32, 32, 120, [1, 4201, 0], F16)])
def test_long_prompts(gpu, nh, nkv, dph, lens, dtype):
    """Enough rows of long prompts for workgroups of 256."""
    rng = np.random.default_rng(nh + dph)
    starts, tail = ends(lens), 3
    g = torch.Generator(device="cuda").manual_seed(nh + dph)
    T = starts[-1] + tail
    q, k, v = (torch.randn(T, w, generator=g, device="cuda").to(dtype)
               for w in (nh * dph, nkv * dph, nkv * dph))
    out = torch.full((T, nh * dph), 0.5, dtype=dtype, device="cuda")
    case_banner("prompt_attention long", nh, nkv, dph, lens, dtype)
    st = torch.tensor(starts, dtype=torch.int32).cuda()
    prompt_attention(q, k, v, st, nh, nkv, dph, out=out)
    want, mag = reference(q, k, v, starts, nh, nkv, dph)
    check(out[:-tail], want[:-tail], mag[:-tail], dtype)
    assert (out[-tail:] == 0.5).all()
    # a key and a value that are not finite, at the longest one's middle
    b = int(np.argmax(lens))
    at = starts[b] + lens[b] // 2 + int(rng.integers(0, 64))
    k[at, :dph] = float("nan")
    v[at, -1] = float("inf")
    prompt_attention(q, k, v, st, nh, nkv, dph, out=out)
    rest = [i for i in range(starts[-1]) if not at <= i < starts[b + 1]]
    check(out[rest], want[rest], mag[rest], dtype)
    later = out[at:starts[b + 1]].float().view(-1, nh, dph)
    assert torch.isnan(later[:, :nh // nkv]).all()
    assert not torch.isfinite(later[:, nh - nh // nkv:, -1]).any()


def test_starts_out_of_order_or_range(gpu):
    """Rows before the first start stay; starts beyond the rows count as their
    end; a falling start leaves its rows out; nothing else is touched."""
    rng = np.random.default_rng(1)
    nh, nkv, dph, T = 4, 2, 64, 200
    q, k, v = make(rng, T, nh, nkv, dph, F16)
    case_banner("prompt_attention starts")
    for given, seqs in (([20, 90, 150], [(20, 90), (90, 150)]), ([-5, 60, 900], [(0, 60), (60, 200)]),
                        ([250, 300], []), ([0, 0], [])):
        out = torch.full((T, nh * dph), 0.5, dtype=F16, device="cuda")
        prompt_attention(q, k, v, torch.tensor(given, dtype=torch.int32).cuda(), nh, nkv, dph,
                         out=out)
        left = torch.ones(T, dtype=torch.bool)
        for a, b in seqs:
            want, mag = reference(q[a:b], k[a:b], v[a:b], [0, b - a], nh, nkv, dph)
            check(out[a:b], want, mag, F16)
            left[a:b] = False
        assert (out[left] == 0.5).all()
    out = torch.full((T, nh * dph), 0.5, dtype=F16, device="cuda")
    prompt_attention(q, k, v, torch.tensor([150, 40, 90], dtype=torch.int32).cuda(), nh, nkv, dph,
                     out=out)
    assert (out[:40] == 0.5).all() and (out[90:] == 0.5).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nonfinite_where_hidden(gpu, dtype):
    """NaN and infinities in k and v reach the queries that see them alone."""
    rng = np.random.default_rng(2)
    nh, nkv, dph, lens = 8, 2, 128, [40, 200, 9]
    starts = ends(lens)
    q, k, v = make(rng, starts[-1] + 3, nh, nkv, dph, dtype)
    want, mag = reference(q, k, v, starts, nh, nkv, dph)
    marks = {0: 37, 1: 150, 2: 8}  # sequence: the first key that is not finite
    for b, at in marks.items():
        k[starts[b] + at, :dph] = float("nan")
        v[starts[b] + at, dph + 5] = float("inf")
        v[starts[b] + at, 7] = float("nan")
    k[starts[-1]:] = float("nan")
    v[starts[-1]:] = float("inf")
    case_banner("prompt_attention nonfinite", dtype)
    out = prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32).cuda(), nh, nkv, dph)
    for b, at in marks.items():
        lo, hi, mid = starts[b], starts[b + 1], starts[b] + at
        check(out[lo:mid], want[lo:mid], mag[lo:mid], dtype)
        later = out[mid:hi].view(-1, nh, dph)
        assert torch.isnan(later[:, :4]).all()            # NaN logits: KV head 0
        assert not torch.isfinite(later[:, 4:, 5]).any()  # an infinite value: head 1, feature 5
        rest = torch.ones(nh, dph, dtype=torch.bool)
        rest[:4] = False
        rest[:, 5] = False
        cols = rest.flatten().nonzero().flatten().cuda()
        check(out[mid:hi][:, cols], want[mid:hi][:, cols], mag[mid:hi][:, cols], dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_large_logits_and_ties(gpu, dtype):
    rng = np.random.default_rng(3)
    nh, nkv, dph, n = 4, 1, 64, 333
    q, k, v = make(rng, n, nh, nkv, dph, dtype)
    q[100:] *= 30  # logits of some 30 nats apart
    q[:50] = 0     # all tied
    k[200] = 0
    starts = [0, n]
    case_banner("prompt_attention large", dtype)
    out = prompt_attention(q, k, v, torch.tensor(starts, dtype=torch.int32).cuda(), nh, nkv, dph)
    want, mag = reference(q, k, v, starts, nh, nkv, dph)
    # logits up to ~150 in fp32: off by 2^-16, so weights by 2^-15
    h = HALF_STEP[dtype]
    over = (out.double() - want).abs() - (h + 2.0 ** -14) * mag - h * want.abs() - 1e-6
    assert over.max() <= 0


def test_repeated_and_captured(gpu):
    rng = np.random.default_rng(4)
    nh, nkv, dph = 8, 2, 64
    starts = torch.tensor([0, 70, 400], dtype=torch.int32, device="cuda")
    q, k, v = make(rng, 400, nh, nkv, dph, F16)
    out = torch.zeros(400, nh * dph, dtype=F16, device="cuda")
    case_banner("prompt_attention capture")
    prompt_attention(q, k, v, starts, nh, nkv, dph, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = torch.zeros_like(out)
    side.wait_stream(torch.cuda.current_stream())
    prompt_attention(q, k, v, starts, nh, nkv, dph, out=other, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(out, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt_attention(q, k, v, starts, nh, nkv, dph, out=out)
    for cut in (1, 200, 399, 33):
        starts[1] = cut
        q.copy_(torch.from_numpy(rng.standard_normal(q.shape)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, prompt_attention(q, k, v, starts, nh, nkv, dph))


def test_refusals(gpu):
    q = torch.zeros(10, 128, dtype=F16, device="cuda")
    starts = torch.tensor([0, 10], dtype=torch.int32, device="cuda")
    ok = dict(q=q, k=q, v=q, starts=starts, nh=2, nkv=2, dph=64)
    prompt_attention(**ok)
    wide = torch.zeros(10, 140, dtype=F16, device="cuda")
    for bad, error in [
            (dict(q=q.float()), TypeError), (dict(q=q.cpu()), TypeError),
            (dict(k=q.bfloat16()), TypeError), (dict(v=q[:5]), ValueError),
            (dict(starts=starts.long()), TypeError), (dict(starts=starts[:0]), ValueError),
            (dict(starts=starts.view(1, 2)), ValueError), (dict(out=q.float()), TypeError),
            (dict(out=torch.zeros(9, 128, dtype=F16, device="cuda")), ValueError),
            (dict(q=wide[:, 1:129]), SDEError), (dict(k=wide[:, :128]), SDEError),
            (dict(nh=3), (ValueError, SDEError)), (dict(nkv=1), ValueError)]:
        args = dict(ok)
        args.update(bad)
        with pytest.raises(error):
            prompt_attention(**args)
    x = torch.zeros(4, 264, dtype=F16, device="cuda")
    with pytest.raises(SDEError):
        prompt_attention(x, x, x, starts, 1, 1, 264)
    with pytest.raises(SDEError):
        y = torch.zeros(4, 128, dtype=F16, device="cuda")
        prompt_attention(y, y, y, starts, 32, 32, 4)
    e = torch.zeros(0, 128, dtype=F16, device="cuda")
    assert prompt_attention(e, e, e, starts, 2, 2, 64).shape == (0, 128)
