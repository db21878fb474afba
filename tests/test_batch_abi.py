"""CPU checks of the calls over several requests (no kernel launches): sizes from
host arithmetic, and bad arguments rejected with the documented status before any
device work.  Pointers are addresses that are never followed."""
import ctypes

import pytest

from speculative_decode_engine_amd import _native as N

P = 1 << 20  # an aligned address, never read


@pytest.fixture(scope="module")
def lib():
    return N.load()


def pool(**kw):
    a = dict(pool=P, tables=P, pool_blocks=64, block_size=16, kv_dim=128, n_seqs=2, max_blocks=8,
             table_stride=8)
    a.update(kw)
    return N.BatchPool(*[a[f] for f, _ in N.BatchPool._fields_])


def append(lib, d=None, rope=None, **kw):
    a = dict(seq=P, pos=P, n=3, dtype=N.SDE_F32, k=P, ks=128, v=P, vs=128, ko=None, kos=0, q=None,
             qs=0, qo=None, qos=0, nh=4, nkv=2, dph=64)
    a.update(kw)
    return lib.sde_batch_append(ctypes.byref(d or pool()), a["seq"], a["pos"], a["n"], a["dtype"],
                                a["k"], a["ks"], a["v"], a["vs"], a["ko"], a["kos"], a["q"],
                                a["qs"], a["qo"], a["qos"], a["nh"], a["nkv"], a["dph"],
                                ctypes.byref(rope) if rope else None, None)


def attention(lib, d=None, **kw):
    a = dict(lens=P, m=1, max_len=128, dtype=N.SDE_F32, q=P, qs=256, out=P, os=256, nh=4, nkv=2,
             dph=64, ws=None, size=0)
    a.update(kw)
    return lib.sde_batch_attention(ctypes.byref(d or pool()), a["lens"], a["m"], a["max_len"],
                                   a["dtype"], a["q"], a["qs"], a["out"], a["os"], a["nh"],
                                   a["nkv"], a["dph"], a["ws"], a["size"], None)


def prompt(lib, **kw):
    a = dict(starts=P, n_seqs=2, n=10, dtype=N.SDE_F16, q=P, qs=256, k=P, ks=128, v=P, vs=128,
             out=P, os=256, nh=4, nkv=2, dph=64)
    a.update(kw)
    return lib.sde_prompt_attention(a["starts"], a["n_seqs"], a["n"], a["dtype"], a["q"], a["qs"],
                                    a["k"], a["ks"], a["v"], a["vs"], a["out"], a["os"], a["nh"],
                                    a["nkv"], a["dph"], None)


def sample(lib, **kw):
    a = dict(logits=P, stride=100, dtype=N.SDE_F32, rows=2, vocab=100, u=P, t=None, k=None, p=None,
             m=None, tokens=P, probs=None, ws=None, size=0)
    a.update(kw)
    return lib.sde_sample(a["logits"], a["stride"], a["dtype"], a["rows"], a["vocab"], a["u"],
                          a["t"], a["k"], a["p"], a["m"], a["tokens"], a["probs"], a["ws"],
                          a["size"], None)


INVALID, CAPACITY, UNSUPPORTED, WORKSPACE = (N.SDE_ERR_INVALID_ARGUMENT, N.SDE_ERR_CAPACITY,
                                             N.SDE_ERR_UNSUPPORTED, N.SDE_ERR_WORKSPACE)

BAD_POOLS = [
    (dict(pool=None), INVALID), (dict(tables=None), INVALID), (dict(pool_blocks=0), INVALID),
    (dict(block_size=0), INVALID), (dict(n_seqs=-1), INVALID), (dict(max_blocks=0), INVALID),
    (dict(table_stride=7), INVALID), (dict(block_size=1025), UNSUPPORTED),
    (dict(max_blocks=1 << 28, table_stride=1 << 28), UNSUPPORTED),
    (dict(pool_blocks=1 << 28), UNSUPPORTED)]


@pytest.mark.parametrize("bad,status", BAD_POOLS)
def test_bad_pools(lib, bad, status):
    assert append(lib, pool(**bad)) == status
    assert attention(lib, pool(**bad)) == status


@pytest.mark.parametrize("bad,status", [
    (dict(seq=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(n=-1), INVALID), (dict(dtype=3), INVALID), (dict(nkv=3), INVALID),
    (dict(ks=127), INVALID), (dict(vs=0), INVALID), (dict(ko=P, kos=64), INVALID),
    (dict(q=P, qs=256), INVALID), (dict(q=P, qs=255, qo=P, qos=256), INVALID),
    (dict(q=P, qs=256, qo=P, qos=256, nh=0), INVALID), (dict(k=P + 2), INVALID),
    (dict(n=(1 << 23) + 1), UNSUPPORTED)])
def test_bad_appends(lib, bad, status):
    assert append(lib, **bad) == status


def test_bad_append_heads_and_rotation(lib):
    assert append(lib, pool(kv_dim=126), nkv=2, dph=63, ks=126, vs=126) == UNSUPPORTED
    assert append(lib, pool(kv_dim=1028), nkv=2, dph=514, ks=1028, vs=1028) == UNSUPPORTED
    for rope in (N.RopeConfig(1e4, -1, 1.0), N.RopeConfig(1e4, 4, 1.0),
                 N.RopeConfig(float("nan"), 0, 1.0), N.RopeConfig(1e4, 1, float("inf"))):
        assert append(lib, rope=rope) == INVALID


def test_nothing_to_do(lib):
    assert append(lib, n=0, seq=None, pos=None, k=None, v=None) == N.SDE_OK
    assert append(lib, pool(n_seqs=0, tables=None)) == N.SDE_OK
    assert attention(lib, pool(n_seqs=0, tables=None), lens=None, q=None, out=None) == N.SDE_OK
    assert prompt(lib, n_seqs=0) == N.SDE_OK and prompt(lib, n=0, q=None) == N.SDE_OK
    assert sample(lib, rows=0, logits=None, u=None, tokens=None) == N.SDE_OK


@pytest.mark.parametrize("bad,status", [
    (dict(lens=None), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID),
    (dict(m=0), INVALID), (dict(m=65), UNSUPPORTED), (dict(max_len=-1), INVALID),
    (dict(max_len=129), CAPACITY), (dict(dtype=-1), INVALID), (dict(nh=3), INVALID),
    (dict(nkv=1), INVALID), (dict(qs=255), INVALID), (dict(os=0), INVALID),
    (dict(q=P + 2), INVALID), (dict(out=P + 1, dtype=N.SDE_F16), INVALID)])
def test_bad_attention(lib, bad, status):
    assert attention(lib, **bad) == status


def test_bad_attention_heads_and_pool(lib):
    assert attention(lib, pool(kv_dim=264), nkv=1, nh=1, dph=264, qs=264, os=264) == UNSUPPORTED
    assert attention(lib, pool(kv_dim=120), nkv=2, dph=60) == UNSUPPORTED
    assert attention(lib, pool(pool=P + 8)) == UNSUPPORTED


def test_attention_workspace(lib):
    size = lib.sde_batch_attention_workspace_size
    assert size(2, 4, 2, 64, 1, 128, 16) == 0          # one partition
    need = size(2, 4, 2, 64, 1, 8192, 16)
    assert need > 0 and need % 8 == 0
    d = pool(max_blocks=512, table_stride=512)
    assert attention(lib, d, max_len=8192) == WORKSPACE
    assert attention(lib, d, max_len=8192, ws=P, size=need - 1) == WORKSPACE
    assert attention(lib, d, max_len=8192, ws=P + 8, size=need) == WORKSPACE
    # pages of one token: partitions no longer than the table entries in LDS
    assert size(64, 4, 4, 64, 1, 5000, 1) > 0
    for bad in ((-1, 4, 2, 64, 1, 128, 16), (2, 3, 2, 64, 1, 128, 16), (2, 4, 2, 63, 1, 128, 16),
                (2, 4, 2, 64, 0, 128, 16), (2, 4, 2, 64, 65, 128, 16), (2, 4, 2, 64, 1, -1, 16),
                (2, 4, 2, 64, 1, 128, 0)):
        assert size(*bad) == 0


@pytest.mark.parametrize("bad,status", [
    (dict(starts=None), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID),
    (dict(n_seqs=-1), INVALID), (dict(n=-1), INVALID), (dict(nh=3), INVALID),
    (dict(dtype=7), INVALID), (dict(dtype=N.SDE_F32), UNSUPPORTED), (dict(ks=127), INVALID),
    (dict(os=255), INVALID), (dict(q=P + 8), UNSUPPORTED), (dict(vs=132), UNSUPPORTED),
    (dict(ks=(1 << 24) + 8), UNSUPPORTED), (dict(dph=60), UNSUPPORTED),
    (dict(dph=264, nh=1, nkv=1, qs=264, ks=264, vs=264, os=264), UNSUPPORTED)])
def test_bad_prompts(lib, bad, status):
    assert prompt(lib, **bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(logits=None), INVALID), (dict(u=None), INVALID), (dict(tokens=None), INVALID),
    (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(dtype=4), INVALID),
    (dict(stride=99), INVALID), (dict(logits=P + 2), INVALID),
    (dict(vocab=(1 << 24) + 1, stride=1 << 25), UNSUPPORTED),
    (dict(rows=(1 << 21) + 1), UNSUPPORTED)])
def test_bad_samples(lib, bad, status):
    assert sample(lib, **bad) == status


def test_sample_workspace(lib):
    size = lib.sde_sample_workspace_size
    assert size(4, 32000) == 0 and size(0, 128256) == 0 and size(1, 1 << 25) == 0
    need = size(4, 128256)
    assert need > 0
    args = dict(rows=4, vocab=128256, stride=128256)
    assert sample(lib, **args) == WORKSPACE
    assert sample(lib, ws=P, size=need - 1, **args) == WORKSPACE
    assert sample(lib, ws=P + 4, size=need, **args) == WORKSPACE
