"""The 8-bit paged cache through the C ABI: append, decode attention and prefill attention against plain 64-bit
forms (tests/q8case.py derives the tolerances), refusals, and a prompt followed by generated tokens."""
import numpy as np
import pytest
import torch

from tests import q8case as Q
from tests.kvcase import guarded

pytestmark = pytest.mark.gpu

BAD_SEQ_LEN, BAD_BLOCK, CONFLICT, NONFINITE = 2, 16, 64, 128
MAX_SEQ = 8192


@pytest.fixture(scope="module")
def kv():
    from oxide_infer_b200 import KvPath
    return KvPath(0, max_batch=64, max_seq_len=MAX_SEQ, max_prefill_rows=1024)


# ---------------------------------------------------------------------------------------------- append
class Append:
    """Inputs of one append call, its 64-bit form and its check."""

    def __init__(self, cache, row_seq, pos, seed, scale=1.0):
        rng = np.random.default_rng(seed)
        n = len(pos)
        self.cache, self.row_seq, self.pos = cache, np.asarray(row_seq), np.asarray(pos)
        f16 = lambda *s: rng.standard_normal(s, dtype=np.float32).astype(np.float16)  # noqa: E731
        self.q, self.k = f16(n, Q.NQ, Q.HD), f16(n, Q.NKV, Q.HD)
        self.v = (f16(n, Q.NKV, Q.HD).astype(np.float32) * scale).astype(np.float16)
        self.wq, self.wk = ((1 + 0.1 * rng.standard_normal(Q.HD)).astype(np.float16) for _ in range(2))
        ang = rng.uniform(0, 6.28, (int(self.pos.max()) + 1, Q.HD)).astype(np.float32)
        self.cos, self.sin = np.cos(ang).astype(np.float16), np.sin(ang).astype(np.float16)

    def call(self, kv, with_seq=True, in_place=False):
        d = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        q = guarded(self.q, "q")
        self.q_out = q if in_place else guarded(np.full_like(self.q, 7.0), "q_out")
        kv.append_q8(self.q_out, q, d(self.k), d(self.v), d(self.wq), d(self.wk), d(self.cos), d(self.sin), Q.i32(self.pos),
                     self.cache.layout(), row_seq=Q.i32(self.row_seq) if with_seq else None)
        torch.cuda.synchronize()

    def check(self, skip_q=(), skip_kv=()):
        c, fmt, bs = self.cache, self.cache.fmt, self.cache.bs
        live = np.array([r for r in range(len(self.pos)) if r not in skip_q])
        at = self.pos[live]
        q64 = Q.norm_rope64(self.q[live], self.wq, self.cos[at], self.sin[at])
        # one rounding to f16, and f32 arithmetic: 20 roundings in the norm, 3 in the rotation, amplified by the
        # cancellation of the rotation's two terms (each at most max|y|)
        err = np.abs(self.q_out.cpu().numpy()[live].astype(np.float64) - q64)
        assert np.all(err <= 2.0 ** -11 * np.abs(q64) + 2.0 ** -18 * np.abs(q64).max(-1, keepdims=True))
        for name, x in (("k", None), ("v", self.v.astype(np.float64))):
            if x is None:
                ok = self.pos < len(self.cos)
                p = np.where(ok, self.pos, 0)
                x = Q.norm_rope64(self.k, self.wk, self.cos[p], self.sin[p])
            x = np.where(np.isnan(x), 0, np.clip(x, -65504, 65504))
            old_c, old_s = self.before[name]
            new_c, new_s = self._state(name)
            want_c, want_s = old_c.copy(), old_s.copy()  # what is not written stays
            tol_c = np.zeros_like(old_c)
            r = 0
            while r < len(self.pos):
                e = r + 1
                while e < len(self.pos) and self.row_seq[e] == self.row_seq[r] and self.pos[e] == self.pos[e - 1] + 1 and self.pos[e] % bs and e not in skip_kv:
                    e += 1
                if r in skip_kv:
                    r += 1
                    continue
                b, first, n = c.tables[self.row_seq[r], self.pos[r] // bs], self.pos[r] % bs, e - r
                need = Q.scale64(np.abs(x[r:e]).max(axis=(0, 2)), fmt)
                s = np.maximum(need, old_s[b]) if first else need
                got = new_s[b].astype(np.float64)
                assert np.all(np.abs(got - s) <= 2.0 ** -18 * s), (name, got, s)
                div = np.where(got > 0, got, 1.0)[None, :, None]
                want_s[b] = new_s[b]
                if first:
                    grown = (got > old_s[b])[None, :, None]
                    again = old_c[b, :first] * (old_s[b][None, :, None] / div)
                    want_c[b, :first] = np.where(grown, again, old_c[b, :first])
                    tol_c[b, :first] = np.where(grown, self._half_step(again, fmt), 0)
                y = x[r:e] / div
                want_c[b, first:first + n] = y
                tol_c[b, first:first + n] = self._half_step(y, fmt)
                r = e
            same = (old_c == new_c) | (np.isnan(old_c) & np.isnan(new_c))
            fixed = tol_c == 0
            assert np.all(same[fixed] | (np.abs(want_c - new_c)[fixed] == 0)), name
            assert np.all(np.abs(want_c - new_c)[~fixed] <= tol_c[~fixed]), name
            assert np.array_equal(want_s, new_s, equal_nan=True), name

    @staticmethod
    def _half_step(y, fmt):
        # half a step of the format (values of up to QMAX), and the f32 value that is rounded is off by up to 2^-18
        slack = 2.0 ** -18 * np.abs(y).max() if y.size else 0
        if fmt == "int8":
            return 0.5 + slack + 0 * y
        e = np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6)))
        return np.exp2(e - 4) * (1 + 2.0 ** -6) + slack

    def _state(self, name):
        p, s = (self.cache.kp, self.cache.ks) if name == "k" else (self.cache.vp, self.cache.vs)
        return p.double().cpu().numpy(), s.cpu().numpy().astype(np.float64)

    def run(self, kv, status=0, skip_q=(), skip_kv=(), **kw):
        self.before = {n: self._state(n) for n in "kv"}
        self.call(kv, **kw)
        assert kv.device_status() == status
        self.check(skip_q, skip_kv)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 64, 256])
@pytest.mark.parametrize("scale", [0.1, 6.0])
def test_append_of_one_token_per_sequence(kv, fmt, bs, scale):
    """Slots at both ends of a block, a first token, scales that grow (6.0) and that mostly do not (0.1)."""
    pos = [0, 1, bs - 1, bs, bs + 1, 2 * bs - 1, 5 * bs + 3, 700]
    c = Q.Q8Cache(pos, fmt, bs, seed=1)
    Append(c, range(len(pos)), pos, seed=2, scale=scale).run(kv, with_seq=False)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 32, 128, 256])
def test_append_of_a_wave(kv, fmt, bs):
    """Runs that start and end inside blocks, one row, several blocks, the same sequence in neighbouring blocks."""
    chunks = [(0, 0, 1), (1, 5, 130), (2, bs - 1, 2), (3, 2 * bs, bs), (4, 3, 300), (5, 40, 17)]
    c = Q.Q8Cache([p + n for _, p, n in chunks], fmt, bs, seed=3)
    Append(c, *Q.wave(chunks), seed=4, scale=2.0).run(kv, in_place=True)


def test_append_with_gaps_between_blocks_and_scales(kv):
    chunks = [(0, 7, 40), (1, 0, 33)]
    c = Q.Q8Cache([47, 33], "int8", 16, seed=5, gap=48, scale_gap=4)
    Append(c, *Q.wave(chunks), seed=6).run(kv)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_of_zeros_and_of_values_without_a_code(kv, fmt):
    c = Q.Q8Cache([16, 20, 0, 0], fmt, 16, seed=7)
    a = Append(c, range(4), [16, 20, 0, 0], seed=8)
    a.k[0], a.v[0] = 0, 0          # a fresh block of zeros: scale 0
    a.v[1, 2, 5], a.v[1, 2, 6] = np.inf, -np.inf
    a.v[2, 0, 0] = np.nan
    a.v[3] = 6e-8                  # the smallest f16
    a.run(kv, status=NONFINITE, with_seq=False)
    assert float(c.ks[c.tables[0, 1]].abs().max()) == 0.0


def test_append_refuses_rows_that_it_cannot_place(kv):
    c = Q.Q8Cache([10, 10, 10, 40], "int8", 16, seed=9)
    far = 16 * c.max_blocks  # the table has no such column
    c.dtables[1, 0] = c.nblocks  # no such block
    row_seq, pos = [0, 1, 2, 3], [10, 10, far, 40]
    a = Append(c, row_seq, pos, seed=10)
    a.run(kv, status=BAD_SEQ_LEN | BAD_BLOCK, skip_q=(2,), skip_kv=(1, 2))
    assert bool((a.q_out[2] == 7.0).all())


def test_rows_of_a_sequence_that_the_table_does_not_have(kv):
    """row_seq beyond the table's rows: nothing of such a row is read or written, its neighbours are right."""
    c = Q.Q8Cache([30, 30], "int8", 16, seed=16)
    a = Append(c, [0, 0, 1, 1, 1], [28, 29, 28, 29, 30], seed=17)
    for bad in (2, 2 ** 31, 2 ** 32 - 1):
        a.row_seq = np.array([0, bad, bad, 1, 1])
        a.run(kv, status=BAD_SEQ_LEN, skip_q=(1, 2), skip_kv=(1, 2))
        assert bool((a.q_out[1:3] == 7.0).all())
        q, g = Q.activations(5, 18)
        ctx = guarded(np.full((5, Q.NQ, Q.HD), 7.0, np.float16), "ctx")
        kv.prefill_attn_q8(ctx, q, g, c.layout(), Q.i32(a.row_seq), Q.i32([29, 30, 29, 30, 31]))
        assert kv.device_status() == BAD_SEQ_LEN
        assert bool((ctx[1:3] == 7.0).all())
        Q.check_rows(ctx, q, g, [(0, 0, np.arange(29)), (3, 1, np.arange(30)), (4, 1, np.arange(31))], c.values)


def test_append_refuses_two_runs_in_one_block(kv):
    """Rows 0-1 and 4-5 are two runs of sequence 0 in its first block; row 2-3 (sequence 1) and 6 (the next block) are fine."""
    c = Q.Q8Cache([30, 30], "e4m3", 16, seed=11)
    a = Append(c, [0, 0, 1, 1, 0, 0, 0], [3, 4, 3, 4, 7, 8, 16], seed=12)
    a.run(kv, status=CONFLICT, skip_kv=(0, 1, 4, 5))
    b = Append(c, [0, 0], [20, 20], seed=13)  # the same token twice
    b.run(kv, status=CONFLICT, skip_kv=(0, 1))


def test_append_again_at_the_same_place_changes_nothing(kv):
    c = Q.Q8Cache([21, 9], "int8", 16, seed=14)
    a = Append(c, [0, 1], [21, 9], seed=15)
    a.run(kv)
    first = [t.clone() for t in (c.kp, c.vp, c.ks, c.vs)]
    a.call(kv)
    assert all(torch.equal(x.reshape(-1), y.reshape(-1)) or torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))
               for x, y in zip(first, (c.kp, c.vp, c.ks, c.vs)))


# ---------------------------------------------------------------------------------------------- decode attention
LENS = [1, 2, 15, 16, 17, 31, 63, 64, 65, 128, 255, 256, 257, 511, 513, 1000, 2049, 4096]
VIEWS = [(0, 0), (0, 9), (1, 0), (1, 1), (7, 3), (64, 64), (100, 4), (300, 70), (256, 5), (1000, 16), (8000, 4)]


def _decode(kv, c, lens, window, sinks, seed=20, gate=True, **kw):
    q, g = Q.activations(len(lens), seed)
    ctx = guarded(np.full((len(lens), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    kv.decode_attn_q8(ctx, q, g if gate else None, c.layout(), Q.i32(lens), window=window, sinks=sinks, **kw)
    torch.cuda.synchronize()
    return ctx, q, g if gate else None


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bs", [16, 64, 256])
@pytest.mark.parametrize("window,sinks", VIEWS)
def test_decode_attention(kv, fmt, bs, window, sinks):
    c = Q.Q8Cache(LENS, fmt, bs, seed=21)
    ctx, q, g = _decode(kv, c, LENS, window, sinks)
    assert kv.device_status() == 0
    Q.check_rows(ctx, q, g, [(i, i, Q.visible(n, window, sinks)) for i, n in enumerate(LENS)], c.values)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_decode_attention_of_small_and_large_values(kv, fmt):
    """Value scales from 1e-4 to 3e4 next to one another, peaked scores, no gate."""
    lens = [300, 77]
    for vscale, kscale in ((1e-4, 1.0), (2e3, 4.0)):
        c = Q.Q8Cache(lens, fmt, 16, seed=22, vscale=vscale, kscale=kscale)
        ctx, q, g = _decode(kv, c, lens, 0, 0, gate=False)
        Q.check_rows(ctx, q, g, [(i, i, Q.visible(n, 0, 0)) for i, n in enumerate(lens)], c.values)


def test_decode_attention_ignores_what_is_not_visible(kv):
    """Codes and scales outside the window, behind the last token and in other blocks: any bytes, the same result."""
    lens, window, sinks, bs = [500, 90], 50, 20, 16
    a = Q.Q8Cache(lens, "e4m3", bs, seed=23)
    base, q, g = _decode(kv, a, lens, window, sinks)
    for i, n in enumerate(lens):
        t = np.setdiff1d(np.arange(n), Q.visible(n, window, sinks))
        whole = [b for b in range(n // bs) if set(range(b * bs, (b + 1) * bs)) <= set(t)]
        tt = torch.from_numpy(t).cuda()
        blk = a.dtables[i].long()[tt // bs]
        for p in (a.kp, a.vp):
            p.view(torch.uint8)[blk, tt % bs] = 0x7f
        for s in (a.ks, a.vs):
            s[a.dtables[i].long()[torch.tensor(whole, dtype=torch.long, device="cuda")]] = float("nan")
    again, _, _ = _decode(kv, a, lens, window, sinks)
    assert torch.equal(base.view(torch.int16), again.view(torch.int16))


def test_decode_attention_with_gaps_and_offsets_behind_32_bits(kv):
    """Blocks 600 KB apart: the last of 8,000 begin 4.8 GB behind the pool's start."""
    nb, pitch, bs, n = 8000, 600 * 1024, 16, 100
    rng = np.random.default_rng(24)
    tables = torch.from_numpy((nb - 1 - rng.permutation(16)[:8]).astype(np.int32)[None].copy()).cuda()
    pools = [torch.zeros(nb * pitch, dtype=torch.int8, device="cuda").as_strided((nb, bs, 4, 128), (pitch, 512, 128, 1)) for _ in range(2)]
    scales = [torch.zeros(nb, 4, device="cuda") for _ in range(2)]
    for p, s in zip(pools, scales):
        codes, sc = Q.quantise_blocks(rng.standard_normal((8, bs, 4, 128), dtype=np.float32), "int8")
        p[tables[0].long()] = codes.cuda()
        s[tables[0].long()] = sc.cuda()
    from oxide_infer_b200 import PagedQ8Layout
    q, g = Q.activations(1, 25)
    ctx = torch.zeros(1, 16, 128, dtype=torch.float16, device="cuda")
    kv.decode_attn_q8(ctx, q, g, PagedQ8Layout.of(*pools, *scales, tables), Q.i32([n]))
    t = torch.arange(n, device="cuda")
    b = tables[0].long()[t // bs]
    def values(seq, tokens):
        t = torch.as_tensor(tokens, device="cuda")
        b = tables[0].long()[t // bs]
        return tuple(p[b, t % bs].double() * sc.double()[b][..., None] for p, sc in zip(pools, scales))
    Q.check_rows(ctx, q, g, [(0, 0, np.arange(n))], values)
    # a chunk of 20 rows appended behind them, and its attention
    lay, m = PagedQ8Layout.of(*pools, *scales, tables), 20
    half = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float16)).cuda()  # noqa: E731
    q, k, v, gate, w = half(m, 16, 128), half(m, 4, 128), half(m, 4, 128), half(m, 16), torch.ones(128, dtype=torch.float16, device="cuda")
    cos, sin = torch.ones(128, 128, dtype=torch.float16, device="cuda"), torch.zeros(128, 128, dtype=torch.float16, device="cuda")
    pos, rs, ctx = Q.i32(np.arange(n, n + m)), Q.i32(np.zeros(m)), torch.zeros(m, 16, 128, dtype=torch.float16, device="cuda")
    kv.append_q8(q, q, k, v, w, w, cos, sin, pos, lay, row_seq=rs)
    got = values(0, np.arange(n, n + m))[1]
    assert float((got - v.double()).abs().max()) <= float(v.double().abs().max()) / 250
    kv.prefill_attn_q8(ctx, q, gate, lay, rs, pos + 1)
    Q.check_rows(ctx, q, gate, [(r, 0, np.arange(n + r + 1)) for r in range(m)], values)
    assert kv.device_status() == 0


def test_decode_attention_skips_rows_without_a_valid_length(kv):
    lens = [100, 0, 50, MAX_SEQ + 1, 33]
    c = Q.Q8Cache([100, 1, 50, 1, 33], "int8", 16, seed=26)
    ctx, q, g = _decode(kv, c, lens, 0, 0)
    assert kv.device_status() == BAD_SEQ_LEN
    assert bool((ctx[1] == 7.0).all()) and bool((ctx[3] == 7.0).all())
    Q.check_rows(ctx, q, g, [(i, i, np.arange(lens[i])) for i in (0, 2, 4)], c.values)
    lens[1], lens[3] = 16 * c.max_blocks + 1, 5  # beyond the table's columns
    ctx, q, g = _decode(kv, c, lens, 0, 0)
    assert kv.device_status() == BAD_SEQ_LEN and bool((ctx[1] == 7.0).all())


def test_decode_attention_reports_a_bad_block(kv):
    c = Q.Q8Cache([100, 40], "int8", 16, seed=27)
    want, q, g = _decode(kv, c, [100, 40], 0, 0)
    c.ks.nan_to_num_(0.0)
    c.vs.nan_to_num_(0.0)
    c.dtables[1, 1] = 2 ** 31 - 1
    got, _, _ = _decode(kv, c, [100, 40], 0, 0)
    assert kv.device_status() == BAD_BLOCK
    assert torch.equal(want[0].view(torch.int16), got[0].view(torch.int16))


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 9)])
def test_decode_attention_of_a_row_does_not_depend_on_the_batch(kv, window, sinks):
    from oxide_infer_b200 import KvPath
    lens = [3000, 5, 777, 1024, 6001, 64]
    c = Q.Q8Cache(lens, "e4m3", 32, seed=28)
    full, q, g = _decode(kv, c, lens, window, sinks)
    again, _, _ = _decode(kv, c, lens, window, sinks)
    assert torch.equal(full.view(torch.int16), again.view(torch.int16))
    other = KvPath(0, max_batch=2, max_seq_len=20000, max_prefill_rows=0)
    for i, n in enumerate(lens):
        ctx = torch.zeros(1, 16, 128, dtype=torch.float16, device="cuda")
        lay = c.layout()
        lay.block_tables, lay.table_rows = c.dtables[i:i + 1].data_ptr(), 1
        other.decode_attn_q8(ctx, q[i:i + 1].contiguous(), g[i:i + 1].contiguous(), lay, Q.i32([n]), window=window, sinks=sinks)
        assert torch.equal(ctx[0].view(torch.int16), full[i].view(torch.int16)), n
    assert kv.device_status() == 0 and other.device_status() == 0


def test_decode_attention_of_a_full_and_of_a_long_batch():
    from oxide_infer_b200 import KvPath
    kv = KvPath(0, max_batch=1024, max_seq_len=70000, max_prefill_rows=0)
    rng = np.random.default_rng(29)
    lens = [int(n) for n in rng.integers(1, 90, 1024)]
    c = Q.Q8Cache(lens, "int8", 16, seed=30)
    ctx, q, g = _decode(kv, c, lens, 40, 3)
    Q.check_rows(ctx, q, g, [(i, i, Q.visible(lens[i], 40, 3)) for i in range(0, 1024, 41)], c.values)
    lens = [66000, 40001, 3]
    c = Q.Q8Cache(lens, "int8", 64, seed=31)
    ctx, q, g = _decode(kv, c, lens, 0, 0)
    Q.check_rows(ctx, q, g, [(i, i, np.arange(n)) for i, n in enumerate(lens)], c.values)
    assert kv.device_status() == 0


# ---------------------------------------------------------------------------------------------- prefill attention
WAVES = {
    "one row": [(0, 0, 1)],
    "a row behind a prefix": [(0, 777, 1)],
    "ragged": [(0, 0, 96), (1, 400, 128), (2, 17, 3), (3, 64, 64), (4, 1000, 33)],
    "many short": [(i, 11 * i, 1 + i % 5) for i in range(40)],
    "long prefix": [(0, 4000, 128)],
}


def _prefill(kv, c, chunks, window, sinks, seed=40, gate=True):
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), seed)
    ctx = guarded(np.full((len(pos), Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    kv.prefill_attn_q8(ctx, q, g if gate else None, c.layout(), Q.i32(row_seq), Q.i32(pos + 1), window=window, sinks=sinks)
    torch.cuda.synchronize()
    return ctx, q, g if gate else None, row_seq, pos


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("name", list(WAVES))
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (100, 4), (64, 70), (500, 200), (3000, 64)])
def test_prefill_attention(kv, fmt, name, window, sinks):
    chunks = WAVES[name]
    c = Q.Q8Cache([p + n for _, p, n in chunks], fmt, 16 if fmt == "int8" else 64, seed=41, spare=0)
    ctx, q, g, row_seq, pos = _prefill(kv, c, chunks, window, sinks)
    assert kv.device_status() == 0
    Q.check_rows(ctx, q, g, [(r, s, Q.visible(p + 1, window, sinks)) for r, (s, p) in enumerate(zip(row_seq, pos)) if r % 3 == 0 or r < 9 or r > len(pos) - 9],
                 c.values)


def test_prefill_attention_of_a_wave_that_fills_the_gpu(kv):
    chunks = [(i, 130 * i, 128) for i in range(8)]
    c = Q.Q8Cache([p + n for _, p, n in chunks], "int8", 32, seed=42, spare=0)
    ctx, q, g, row_seq, pos = _prefill(kv, c, chunks, 0, 0, gate=False)
    Q.check_rows(ctx, q, g, [(r, row_seq[r], np.arange(pos[r] + 1)) for r in range(0, 1024, 13)], c.values)
    again = _prefill(kv, c, chunks, 0, 0, gate=False)[0]
    assert torch.equal(ctx.view(torch.int16), again.view(torch.int16)) and kv.device_status() == 0


def test_prefill_attention_ignores_later_tokens_and_idle_blocks(kv):
    """Rows of a chunk in the middle of a longer cache: the tokens behind their positions may be anything finite, blocks
    that no row reads anything at all."""
    c = Q.Q8Cache([600], "e4m3", 16, seed=43)
    chunk = [(0, 200, 70)]
    base, *_ = _prefill(kv, c, chunk, 64, 5)
    t = torch.arange(288, 600, device="cuda")
    blk = c.dtables[0].long()[t // 16]
    for p in (c.kp, c.vp):
        p.view(torch.uint8)[blk, t % 16] = 0x7f
    for s in (c.ks, c.vs):
        s[c.dtables[0].long()[torch.arange(18, 37, device="cuda")]] = float("nan")
    again, *_ = _prefill(kv, c, chunk, 64, 5)
    assert torch.equal(base.view(torch.int16), again.view(torch.int16)) and kv.device_status() == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 1e38, 0.0])
def test_prefill_attention_ignores_keys_between_sinks_and_windows(kv, fmt, bad):
    """Tokens that no row of the wave sees: any codes; blocks without a visible token: any scales."""
    c = Q.Q8Cache([700, 300], fmt, 16, seed=46)
    chunks, window, sinks = [(0, 600, 90), (1, 250, 40)], 70, 21
    base, *_ = _prefill(kv, c, chunks, window, sinks)
    for s, p, n in chunks:
        t = np.arange(sinks, p + 1 - window)
        tt = torch.from_numpy(t).cuda()
        blk = c.dtables[s].long()[tt // 16]
        for x in (c.kp, c.vp):
            x.view(torch.uint8)[blk, tt % 16] = 0x7f if fmt == "e4m3" else 0x80
        hidden = [b for b in range(2, (p + 1 - window) // 16)]
        for x in (c.ks, c.vs):
            x[c.dtables[s].long()[torch.tensor(hidden, device="cuda")]] = bad
    again, *_ = _prefill(kv, c, chunks, window, sinks)
    assert torch.equal(base.view(torch.int16), again.view(torch.int16)) and kv.device_status() == 0


@pytest.mark.parametrize("fmt,bs", [("int8", 16), ("e4m3", 32), ("int8", 64)])
@pytest.mark.parametrize("window,sinks", [(70, 4), (40, 40), (300, 90), (100, 0)])
def test_blocks_between_sinks_and_window_may_be_given_back(kv, fmt, bs, window, sinks):
    """Table entries of blocks without a visible token hold an id that the pool does not have: same bytes, no status."""
    c = Q.Q8Cache([700, 2000], fmt, bs, seed=47)
    chunks = [(0, 620, 60), (1, 1900, 100)]
    q, g = Q.activations(2, 48)

    def both():
        b = guarded(np.full((2, Q.NQ, Q.HD), 7.0, np.float16), "ctx")
        kv.decode_attn_q8(b, q, g, c.layout(), Q.i32([680, 2000]), window, sinks)
        return _prefill(kv, c, chunks, window, sinks)[0], b

    want = both()
    for s, p, _ in chunks:
        c.dtables[s, -(-sinks // bs):(p + 1 - window) // bs] = -1
    got = both()
    assert kv.device_status() == 0
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(want, got))


def test_prefill_attention_skips_rows_and_reports_blocks(kv):
    c = Q.Q8Cache([100, 40], "int8", 16, seed=44)
    row_seq, lens = [0, 0, 1, 1, 0], [5, 0, 40, 16 * c.max_blocks + 1, 100]
    q, g = Q.activations(5, 45)
    ctx = guarded(np.full((5, Q.NQ, Q.HD), 7.0, np.float16), "ctx")
    kv.prefill_attn_q8(ctx, q, g, c.layout(), Q.i32(row_seq), Q.i32(lens))
    assert kv.device_status() == BAD_SEQ_LEN
    assert bool((ctx[1] == 7.0).all()) and bool((ctx[3] == 7.0).all())
    Q.check_rows(ctx, q, g, [(r, row_seq[r], np.arange(lens[r])) for r in (0, 2, 4)], c.values)


# ---------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 4)])
def test_a_prompt_and_generated_tokens(kv, fmt, window, sinks):
    """Two prompts of 150 and 37 tokens arrive in waves (append, attention), then twelve tokens are generated; the decode
    steps run from one captured graph whose tables advance on the device.  Every context is checked against the cache as
    it stands, the cache against the keys and values that went in."""
    c = Q.Q8Cache([0, 0], fmt, 16, seed=50, spare=180)
    lay = c.layout()
    rng = np.random.default_rng(51)
    half = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float16)).cuda()  # noqa: E731
    wq, wk = half(128) * 0.1 + 1, half(128) * 0.1 + 1
    ang = torch.rand(256, 128, device="cuda") * 6.28
    cos, sin = ang.cos().half(), ang.sin().half()
    lens, sent = [0, 0], [[], []]  # sent: the values of V
    def wave_of(chunks):
        row_seq, pos = Q.wave(chunks)
        n = len(pos)
        q, k, v, g = half(n, 16, 128), half(n, 4, 128), half(n, 4, 128), half(n, 16)
        qn, ctx = torch.zeros_like(q), torch.zeros_like(q)
        rs, p = Q.i32(row_seq), Q.i32(pos)
        kv.append_q8(qn, q, k, v, wq, wk, cos, sin, p, lay, row_seq=rs)
        kv.prefill_attn_q8(ctx, qn, g, lay, rs, p + 1, window=window, sinks=sinks)
        Q.check_rows(ctx, qn, g, [(r, s, Q.visible(t + 1, window, sinks)) for r, (s, t) in enumerate(zip(row_seq, pos))], c.values)
        for r, s in enumerate(row_seq):
            sent[s].append(v[r])
            lens[s] += 1
    wave_of([(0, 0, 128), (1, 0, 37)])
    wave_of([(0, 128, 22)])
    q, k, v, g = half(2, 16, 128), half(2, 4, 128), half(2, 4, 128), half(2, 16)
    qn, ctx = torch.zeros_like(q), torch.zeros_like(q)
    pos, sl = Q.i32(lens), Q.i32([n + 1 for n in lens])
    def step():
        kv.append_q8(qn, q, k, v, wq, wk, cos, sin, pos, lay)
        kv.decode_attn_q8(ctx, qn, g, lay, sl, window=window, sinks=sinks)
        kv.advance_step(pos, sl)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for _ in range(12):
            for t, s in ((q, (2, 16, 128)), (k, (2, 4, 128)), (v, (2, 4, 128)), (g, (2, 16))):
                t.copy_(half(*s))
            graph.replay()
            stream.synchronize()
            for i in range(2):
                sent[i].append(v[i].clone())
                lens[i] += 1
            Q.check_rows(ctx, qn, g, [(i, i, Q.visible(lens[i], window, sinks)) for i in range(2)], c.values)
    torch.cuda.current_stream().wait_stream(stream)
    assert kv.device_status() == 0
    for i in range(2):  # V was stored to within its format: int8 half a step of each of a block's scales, at most 16 of them
        _, vals = c.values(i, np.arange(lens[i]))
        true = torch.stack(sent[i]).double()
        amax = true.abs().max()
        assert float((vals - true).abs().max()) <= (16 * amax / 254 if fmt == "int8" else float(amax) * 2.0 ** -4 * 1.1)


def test_calls_on_another_stream(kv):
    """The calls run on torch's current stream: ordered behind work of that stream that the default stream does not see."""
    lens = [700, 33]
    c = Q.Q8Cache(lens, "int8", 16, seed=52)
    want, q, g = _decode(kv, c, lens, 0, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(q)
        torch.cuda._sleep(20_000_000)
        late.copy_(q)
        ctx = torch.zeros_like(want)
        kv.decode_attn_q8(ctx, late, g, c.layout(), Q.i32(lens))
    s.synchronize()
    assert torch.equal(ctx.view(torch.int16), want.view(torch.int16))


def test_refusals(kv):
    from oxide_infer_b200 import OxiError
    c = Q.Q8Cache([20], "int8", 16, seed=53)
    q, g = Q.activations(1, 54)
    ctx, sl = torch.zeros_like(q), Q.i32([20])

    def code(fn):
        with pytest.raises(OxiError) as e:
            fn()
        return e.value.code

    def broken(**kw):
        lay = c.layout()
        for k, v in kw.items():
            setattr(lay, k, v)
        return lay

    dec = lambda lay, **kw: kv.decode_attn_q8(ctx, q, g, lay, sl, **kw)  # noqa: E731
    for kw in (dict(k_pool=None), dict(v_scales=None), dict(block_tables=None)):
        assert code(lambda: dec(broken(**kw))) == -1
    for kw in (dict(table_rows=0), dict(block_size=8), dict(block_size=24), dict(block_size=512), dict(max_blocks=0), dict(num_blocks=0),
               dict(block_stride_bytes=16 * 512 - 16), dict(block_stride_bytes=16 * 512 + 8), dict(scale_stride=2),
               dict(scale_stride=6), dict(format=2), dict(k_pool=c.kp.data_ptr() + 8), dict(k_scales=c.ks.data_ptr() + 4)):
        assert code(lambda: dec(broken(**kw))) == -3, kw
    assert code(lambda: dec(c.layout(), batch=0)) == -2
    assert code(lambda: dec(c.layout(), batch=65)) == -2
    assert code(lambda: dec(c.layout(), batch=2)) == -2  # the table has one row
    assert code(lambda: kv.prefill_attn_q8(ctx, q, g, c.layout(), None, sl)) == -1
    assert code(lambda: kv.prefill_attn_q8(ctx, q, g, c.layout(), sl, sl, rows=1025)) == -2
    k = torch.zeros(1, 4, 128, dtype=torch.float16, device="cuda")
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    app = lambda **kw: kv.append_q8(ctx, q, k, k, w, w, w, w, sl, c.layout(), **kw)  # noqa: E731
    assert code(lambda: app(eps=-1.0)) == -3
    assert code(lambda: app(eps=float("nan"))) == -3
    assert code(lambda: app(rows=1025)) == -2
    assert code(lambda: app(rows=2)) == -2
    odd = torch.zeros(2 * 16 * 128, dtype=torch.float16, device="cuda")[1:1 + 16 * 128].view(1, 16, 128)
    assert code(lambda: kv.decode_attn_q8(ctx, odd, g, c.layout(), sl)) == -3
    assert kv.device_status() == 0
