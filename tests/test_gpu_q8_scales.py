"""Attention over 8-bit caches whose blocks have very different scales: values of 0 beside large ones, keys of 0, magnitudes from the
smallest to the largest f16.  The 64-bit form and its tolerances are those of tests/q8case.py; codes times scales are exact there."""
import numpy as np
import pytest
import torch

from tests import q8case as Q
from tests.kvcase import guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from oxide_infer_b200 import KvPath
    return KvPath(0, max_batch=64, max_seq_len=8192, max_prefill_rows=1024)


def _fill(c, k, v):
    """Quantises k, v [tokens of all sequences, one after the other][4][128] into the cache's blocks."""
    at = 0
    for i, n in enumerate(c.lens):
        for b0 in range(0, n, c.bs):
            m = min(c.bs, n - b0)
            blk = int(c.tables[i, b0 // c.bs])
            for x, p, s in ((k, c.kp, c.ks), (v, c.vp, c.vs)):
                pad = np.zeros((1, c.bs, Q.NKV, Q.HD), np.float32)
                pad[0, :m] = x[at + b0:at + b0 + m]
                codes, scale = Q.quantise_blocks(pad, c.fmt)
                p[blk, :m] = codes[0, :m].cuda()
                s[blk] = scale[0].cuda()
        at += n


def _both(kv, c, q, gate, lens, window=0, sinks=0):
    """The same rows as a decode batch and as a prefill wave (a row per sequence)."""
    outs = []
    for decode in (True, False):
        ctx = guarded(np.full((len(lens), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
        if decode:
            kv.decode_attn_q8(ctx, q, gate, c.layout(), Q.i32(lens), window=window, sinks=sinks)
        else:
            kv.prefill_attn_q8(ctx, q, gate, c.layout(), Q.i32(np.arange(len(lens))), Q.i32(lens), window=window, sinks=sinks)
        outs.append(ctx)
    assert kv.device_status() == 0
    return outs


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("large", [3e4, 1.0, 1e-7])
def test_many_zero_values_beside_a_token_that_holds_most_of_the_weight(kv, fmt, bs, large):
    """All values are 0 but for one token's, whose key scores `ahead` higher: the others' weights are small one by one and count
    together - 4,095 of them at e^-5 ... e^-17 of the token's."""
    aheads, n = [5.0, 9.0, 12.0, 13.0, 14.0, 17.0], 4096
    lens = [n] * len(aheads)
    rng = np.random.default_rng(100)
    c = Q.Q8Cache(lens, fmt, bs, seed=101)
    u = rng.choice([-1.0, 1.0], Q.HD).astype(np.float32)
    k = np.zeros((n * len(aheads), Q.NKV, Q.HD), np.float32)
    v = np.zeros_like(k)
    for i, ahead in enumerate(aheads):
        b0 = n * i + bs * (37 % (n // bs))
        k[b0] = u * (ahead * np.sqrt(Q.HD) / Q.HD)
        v[b0] = rng.uniform(-large, large, (Q.NKV, Q.HD))
    _fill(c, k, v)
    q = torch.from_numpy(np.broadcast_to(u, (len(aheads), Q.NQ, Q.HD)).astype(np.float16).copy()).cuda()
    for ctx in _both(kv, c, q, None, lens):
        Q.check_rows(ctx, q, None, [(i, i, np.arange(n)) for i in range(len(aheads))], c.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (400, 33), (100, 0)])
def test_scales_of_every_magnitude_next_to_one_another(kv, fmt, window, sinks):
    """Values from 0 and the smallest f16 to 3e4, keys from 0 to 8, block by block, lengths around key ranges and tiles."""
    lens = [1, 16, 17, 64, 65, 255, 300, 700, 1500, 3000]
    rng = np.random.default_rng(102)
    c = Q.Q8Cache(lens, fmt, 16, seed=103)
    total = sum(lens)
    k = rng.standard_normal((total, Q.NKV, Q.HD)).astype(np.float32)
    v = rng.standard_normal((total, Q.NKV, Q.HD)).astype(np.float32)
    at = 0
    for n in lens:
        for b0 in range(0, n, 16):
            rows = slice(at + b0, at + min(n, b0 + 16))
            k[rows] *= rng.choice([0.0, 0.01, 0.3, 1.0, 2.0], (1, Q.NKV, 1))
            v[rows] *= rng.choice([0.0, 6e-8, 1e-4, 1.0, 50.0, 7e3], (1, Q.NKV, 1))
        at += n
    _fill(c, np.clip(k, -8, 8), np.clip(v, -3e4, 3e4))
    q, g = Q.activations(len(lens), 104)
    for gate in (g, None):
        for ctx in _both(kv, c, q, gate, lens, window, sinks):
            Q.check_rows(ctx, q, gate, [(i, i, Q.visible(n, window, sinks)) for i, n in enumerate(lens)], c.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("vscale,kscale", [(1e-4, 1.0), (2e3, 4.0), (0.0, 1.0), (1.0, 0.0)])
def test_prefill_attention_of_small_and_large_values(kv, fmt, vscale, kscale):
    c = Q.Q8Cache([700, 90], fmt, 32, seed=105, vscale=vscale, kscale=kscale)
    row_seq, pos = Q.wave([(0, 600, 90), (1, 10, 70)])
    q, g = Q.activations(len(pos), 106)
    ctx = guarded(np.full((len(pos), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    kv.prefill_attn_q8(ctx, q, g, c.layout(), Q.i32(row_seq), Q.i32(pos + 1))
    Q.check_rows(ctx, q, g, [(r, row_seq[r], np.arange(pos[r] + 1)) for r in range(0, len(pos), 5)], c.values)
    assert kv.device_status() == 0
