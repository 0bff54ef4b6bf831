"""Small prefill waves with sinks or over the 8-bit cache whose blocks of 64 rows hold rows of many sequences: CTAs share a block by
its runs.  Against the 64-bit form of tests/q8case.py, and against the same rows in calls of their own."""
import numpy as np
import pytest
import torch

from tests import q8case as Q
from tests.test_gpu_sinks import F16Cache
from tests.kvcase import guarded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from oxide_infer_b200 import KvPath
    return KvPath(0, max_batch=64, max_seq_len=4096, max_prefill_rows=2048)


def _waves():
    alternating = [(i % 2, 300 + 7 * i, 1) for i in range(64)]
    return {
        "a row each of 64 sequences": [(i, 100 + 13 * i, 1) for i in range(64)],
        "a row each of 300 calls": [(i % 64, 50 + 5 * i, 1) for i in range(300)],
        "two sequences alternating": alternating,
        "runs of three": [(i, 200 + 9 * i, 3) for i in range(50)],
        "one run and many": [(0, 700, 61), *[(1 + i, 20 * i, 2) for i in range(40)], (50, 90, 77)],
        "one row": [(3, 999, 1)],
    }


def _cache(form, lens, seed):
    if form in ("int8", "e4m3"):
        return Q.Q8Cache(lens, form, 16, seed=seed, spare=0)
    return F16Cache(lens, 0 if form == "pointers" else 32, seed=seed)


def _call(kv, c, ctx, q, g, row_seq, lens, window, sinks):
    if isinstance(c, Q.Q8Cache):
        kv.prefill_attn_q8(ctx, q, g, c.layout(), Q.i32(row_seq), Q.i32(lens), window=window, sinks=sinks)
    else:
        c.prefill(kv, ctx, q, g, row_seq, lens, window, sinks)


@pytest.mark.parametrize("form", ["int8", "e4m3", "pointers", "paged"])
@pytest.mark.parametrize("name", list(_waves()))
@pytest.mark.parametrize("window,sinks", [(64, 4), (256, 4), (100, 70), (1, 1), (700, 9)])
def test_blocks_of_many_runs(kv, form, name, window, sinks):
    chunks = _waves()[name]
    nseq = 1 + max(s for s, _, _ in chunks)
    lens = [max([p + n for s, p, n in chunks if s == i], default=1) for i in range(nseq)]
    c = _cache(form, lens, 130)
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), 131)
    ctx = guarded(np.full((len(pos), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    _call(kv, c, ctx, q, g, row_seq, pos + 1, window, sinks)
    assert kv.device_status() == 0
    step = 1 + len(pos) // 70
    Q.check_rows(ctx, q, g, [(r, row_seq[r], Q.visible(pos[r] + 1, window, sinks)) for r in range(0, len(pos), step)], c.values)


@pytest.mark.parametrize("form", ["int8", "e4m3", "pointers", "paged"])
def test_a_run_has_the_bytes_of_a_call_of_its_own(kv, form):
    """Runs inside one block, among rows that are skipped, in waves of different size (so in other shares)."""
    chunks = [(i, 40 * i + 11, 1 + (7 * i) % 12) for i in range(24)]
    c = _cache(form, [p + n for _, p, n in chunks], 132)
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), 133)
    lens = pos + 1
    skipped = [r for r in (5, 6, 70) if r < len(pos)]
    lens[skipped] = 0
    window, sinks = 90, 5
    whole = guarded(np.full((len(pos), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    _call(kv, c, whole, q, g, row_seq, lens, window, sinks)
    assert kv.device_status() == 2
    assert bool((whole[skipped] == 7.0).all())
    at = 0
    for s, _, n in chunks:
        rows = slice(at, at + n)
        at += n
        if rows.start // 64 != (rows.stop - 1) // 64 or any(r in skipped for r in range(rows.start, rows.stop)):
            continue  # a run that a block border cuts in two is two runs
        own = guarded(np.full((n, Q.NQ, Q.HD), 7.0, np.float16), "ctx")
        _call(kv, c, own, q[rows].contiguous(), g[rows].contiguous(), row_seq[rows], lens[rows], window, sinks)
        assert torch.equal(own.view(torch.int16), whole[rows].view(torch.int16)), s
    assert kv.device_status() == 0


@pytest.mark.parametrize("form", ["int8", "pointers"])
def test_rows_of_many_sequences_are_not_worked_off_one_after_the_other(kv, form):
    """64 rows of 64 sequences against 64 rows of one, window 64: a CTA has two runs of two to three tiles and one run of three.  One CTA
    for all 64 runs took 16 times as long."""
    c = _cache(form, [1564] * 64, 134)
    q, g = Q.activations(64, 135)
    ctx = torch.zeros_like(q)

    def us(row_seq):
        pos = 1500 + np.arange(64)
        if isinstance(c, Q.Q8Cache):
            args = c.layout(), Q.i32(row_seq), Q.i32(pos + 1)
            call = lambda: kv.prefill_attn_q8(ctx, q, g, *args, window=64, sinks=4)  # noqa: E731
        else:
            rs = torch.as_tensor(row_seq, device="cuda")
            args = c.k_ptrs[rs].contiguous(), c.v_ptrs[rs].contiguous(), Q.i32(pos + 1)
            call = lambda: kv.prefill_attn_sinks(ctx, q, g, *args, 64, 4)  # noqa: E731
        times = []
        for _ in range(12):
            t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(300_000)  # the calls are enqueued by the time it ends
            t0.record()
            for _ in range(10):
                call()
            t1.record()
            torch.cuda.synchronize()
            times.append(t0.elapsed_time(t1))
        return sorted(times)[len(times) // 2] * 100

    one, many = us(np.zeros(64, np.int64)), us(np.arange(64))
    assert kv.device_status() == 0
    assert many <= 4.0 * one, (many, one)
