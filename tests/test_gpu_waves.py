"""Waves as large as a handle takes: prefill attention in which a CTA works through two to four items (more than 37 blocks of 64 rows:
the plan's order, claims, rings and scale tables that go on from item to item), and quantising appends of more than 1,184 rows (two
of the three ways in which a window's heads are shared out).  Against the 64-bit forms of tests/q8case.py."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import q8case as Q
from tests.test_gpu_q8 import Append
from tests.test_gpu_sinks import F16Cache
from tests.kvcase import guarded

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def kv():
    from oxide_infer_b200 import KvPath
    return KvPath(0, max_batch=64, max_seq_len=8192, max_prefill_rows=8192)


# chunks: (sequence, first position, rows)
WAVES = {
    "two items a CTA": [(i, 61 * i, 128) for i in range(32)],                                              # 4,096 rows, 256 items
    "ragged": [(i, (317 * i) % 1900, 60 + (41 * i) % 130) for i in range(21)],                             # 2,500 rows or so
    "short and long": [(i, 0 if i % 3 else 1500 + 40 * i, 1 + (97 * i) % 150) for i in range(40)],
    "four items a CTA": [(i, 23 * i, 160) for i in range(51)],                                             # 8,160 rows, 512 items
}


def _sample(pos):
    """Rows at both ends, at the ends of blocks and of query tiles, and some in between."""
    n = len(pos)
    return sorted({r for r in (*range(3), 31, 32, 63, 64, 65, n - 65, n - 64, n - 2, n - 1, *range(0, n, n // 48 + 1)) if r < n})


def _run(kv, call, n, seed):
    q, g = Q.activations(n, seed)
    outs = []
    for _ in range(2):
        ctx = guarded(np.full((n, Q.NQ, Q.HD), 7.0, np.float16), "ctx")
        call(ctx, q, g)
        outs.append(ctx)
    assert kv.device_status() == 0
    assert torch.equal(outs[0].view(torch.int16), outs[1].view(torch.int16))  # which CTA takes an item does not matter
    return outs[0], q, g


@pytest.mark.parametrize("fmt,bs", [("int8", 16), ("e4m3", 64)])
@pytest.mark.parametrize("name", list(WAVES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1024, 4), (256, 70), (40, 0)])
def test_8_bit_prefill(kv, fmt, bs, name, window, sinks):
    chunks = WAVES[name]
    c = Q.Q8Cache([p + n for _, p, n in chunks], fmt, bs, seed=110, spare=0)
    row_seq, pos = Q.wave(chunks)
    rs, lens, lay = Q.i32(row_seq), Q.i32(pos + 1), c.layout()
    ctx, q, g = _run(kv, lambda o, q, g: kv.prefill_attn_q8(o, q, g, lay, rs, lens, window=window, sinks=sinks), len(pos), 111)
    Q.check_rows(ctx, q, g, [(r, row_seq[r], Q.visible(pos[r] + 1, window, sinks)) for r in _sample(pos)], c.values)


@pytest.mark.parametrize("bs", [0, 16, 128])
@pytest.mark.parametrize("name", list(WAVES))
@pytest.mark.parametrize("window,sinks", [(1024, 4), (256, 70), (40, 1)])
def test_prefill_with_sinks(kv, bs, name, window, sinks):
    chunks = WAVES[name]
    c = F16Cache([p + n for _, p, n in chunks], bs, seed=112)
    row_seq, pos = Q.wave(chunks)
    ctx, q, g = _run(kv, lambda o, q, g: c.prefill(kv, o, q, g, row_seq, pos + 1, window, sinks), len(pos), 113)
    Q.check_rows(ctx, q, g, [(r, row_seq[r], Q.visible(pos[r] + 1, window, sinks)) for r in _sample(pos)], c.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_rows_without_keys_in_a_wave_of_many_items(kv, fmt):
    """Rows of length 0 and blocks without any key: left as they are, and the items behind them are right."""
    chunks = WAVES["two items a CTA"]
    c = Q.Q8Cache([p + n for _, p, n in chunks], fmt, 32, seed=114, spare=0)
    row_seq, pos = Q.wave(chunks)
    lens = pos + 1
    lens[np.arange(len(lens)) % 7 == 3] = 0
    lens[640:1100] = 0
    rs, ln, lay = Q.i32(row_seq), Q.i32(lens), c.layout()
    q, g = Q.activations(len(pos), 115)
    ctx = guarded(np.full((len(pos), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    kv.prefill_attn_q8(ctx, q, g, lay, rs, ln)
    assert kv.device_status() == 2
    assert bool((ctx[torch.from_numpy(lens == 0).cuda()] == 7.0).all())
    Q.check_rows(ctx, q, g, [(r, row_seq[r], np.arange(lens[r])) for r in _sample(pos) if lens[r]], c.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("scale", [0.2, 4.0])
def test_append_of_many_rows(kv, fmt, bs, scale):
    """Runs that cross windows of 16 rows and blocks, single rows between them, scales that grow (4.0): 1,185 to 3,000 rows."""
    chunks = [(0, 5, 400), (1, bs - 1, 1), (2, 0, 130), (3, 3 * bs + 1, 300), (4, 9, 2), (5, 2 * bs - 3, 257), (6, 1, 33), (7, bs, bs),
              (8, 77, 15), (9, 6, 48)]
    chunks += [(10 + i, (13 * i) % 50, 1 + (29 * i) % 90) for i in range(30 if bs in (16, 64) else 2)]
    c = Q.Q8Cache([p + n for _, p, n in chunks], fmt, bs, seed=116)
    a = Append(c, *Q.wave(chunks), seed=117, scale=scale)
    assert len(a.pos) > 1184
    a.run(kv, in_place=scale < 1)


@pytest.mark.parametrize("bs", [16, 64])
def test_append_of_many_rows_refuses_what_it_cannot_place(kv, bs):
    """The refusals of a small append in a large one: a row beyond the table, a block that the pool does not have, two runs in a block."""
    chunks = [(i, 3 * i + 1, 100) for i in range(14)]
    c = Q.Q8Cache([p + n + 40 for _, p, n in chunks], "int8", bs, seed=118)
    row_seq, pos = Q.wave(chunks)
    row_seq, pos = np.append(row_seq, [0, 14]), np.append(pos, [pos[99], 0])  # sequence 0's last token again, and a row that the table lacks
    a = Append(c, row_seq, pos, seed=119)
    blk = lambda r: pos[r] // bs  # noqa: E731
    clash = [r for r in range(100) if blk(r) == blk(99)] + [1400]
    c.dtables[5, blk(500)] = c.nblocks
    missing = [500 + i for i in range(100) if blk(500 + i) == blk(500)]
    a.run(kv, status=2 | 16 | 64, skip_q=(1401,), skip_kv=(*clash, *missing, 1401))
    assert bool((a.q_out[1401] == 7.0).all())


@pytest.mark.parametrize("window,sinks", [(300, 5), (64, 64)])
def test_a_wave_of_more_blocks_than_the_small_plan_takes(window, sinks):
    """More than 65,536 rows: the plan that sorts the blocks by counting."""
    from oxide_infer_b200 import KvPath
    kv = KvPath(0, max_batch=4, max_seq_len=8192, max_prefill_rows=66000)
    chunks = [(i, 100 * i, 2000) for i in range(33)]
    row_seq, pos = Q.wave(chunks)
    rows = [(r, row_seq[r], Q.visible(pos[r] + 1, window, sinks)) for r in _sample(pos)]
    lens = [p + n for _, p, n in chunks]
    c = Q.Q8Cache(lens, "int8", 64, seed=120, spare=0)
    rs, ln, lay = Q.i32(row_seq), Q.i32(pos + 1), c.layout()
    ctx, q, g = _run(kv, lambda o, q, g: kv.prefill_attn_q8(o, q, g, lay, rs, ln, window=window, sinks=sinks), len(pos), 121)
    Q.check_rows(ctx, q, g, rows, c.values)
    c = F16Cache(lens, 64, seed=122)
    ctx, q, g = _run(kv, lambda o, q, g: c.prefill(kv, o, q, g, row_seq, pos + 1, window, sinks), len(pos), 123)
    Q.check_rows(ctx, q, g, rows, c.values)


def test_waves_and_scales_are_clean_under_the_bounds_build():
    if os.environ.get("OXI_KV_LIB"):
        pytest.skip("already running against a substituted library")
    from oxide_infer_b200 import build
    env = dict(os.environ, OXI_KV_LIB=build.build(bounds=True))
    subset = "append or ragged or keys or magnitude or zero"
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-k", subset, "tests/test_gpu_waves.py",
                        "tests/test_gpu_q8_scales.py"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0 and " passed" in r.stdout and "failed" not in r.stdout, (r.stdout + r.stderr)[-3000:]
