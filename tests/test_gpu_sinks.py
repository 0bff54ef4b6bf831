"""Sliding-window attention with sinks over the f16 caches (pointer tables and paged) against a plain 64-bit form
(tests/q8case.py derives the tolerances)."""
import numpy as np
import pytest
import torch

from tests import q8case as Q
from tests.kvcase import dev_ptr_table, guarded

pytestmark = pytest.mark.gpu

BAD_SEQ_LEN, BAD_BLOCK, MISALIGNED = 2, 16, 1
MAX_SEQ = 8192


@pytest.fixture(scope="module")
def kv():
    from oxide_infer_b200 import KvPath
    return KvPath(0, max_batch=64, max_seq_len=MAX_SEQ, max_prefill_rows=1024)


class F16Cache:
    """Pointer tables (bs 0) or scattered blocks of bs tokens.  Rows behind a sequence's tokens hold NaN."""

    def __init__(self, lens, bs, seed, spare=1):
        rng = np.random.default_rng(seed)
        f16 = lambda n: rng.standard_normal((int(n), 4, 128), dtype=np.float32).astype(np.float16)  # noqa: E731
        nan = np.full((spare, 4, 128), np.nan, np.float16)
        self.lens, self.bs = list(lens), bs
        k, v = [np.concatenate([f16(n), nan]) for n in lens], [np.concatenate([f16(n), nan]) for n in lens]
        if not bs:
            self.k, self.v = [guarded(a, "k") for a in k], [guarded(a, "v") for a in v]
            self.k_ptrs, self.v_ptrs = dev_ptr_table(self.k), dev_ptr_table(self.v)
            return
        need = [-(-len(a) // bs) for a in k]
        self.nblocks = sum(need) + 1
        perm = rng.permutation(self.nblocks).astype(np.int32)
        self.max_blocks = max(need) + 1
        self.tables = np.full((len(lens), self.max_blocks), perm[-1], np.int32)
        pools = np.full((2, self.nblocks, bs, 4, 128), np.nan, np.float16)
        o = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = perm[o:o + n]
            o += n
            for j in range(n):
                for p, a in zip(pools, (k[i], v[i])):
                    part = a[j * bs:(j + 1) * bs]
                    p[self.tables[i, j], :len(part)] = part
        self.kp, self.vp = guarded(pools[0], "k_pool"), guarded(pools[1], "v_pool")
        self.dtables = torch.from_numpy(self.tables).cuda()

    def layout(self):
        from oxide_infer_b200 import PagedLayout
        return PagedLayout.of(self.kp, self.vp, self.dtables, self.bs)

    def values(self, seq, tokens):
        t = torch.as_tensor(tokens, device="cuda")
        if not self.bs:
            return self.k[seq][t].double(), self.v[seq][t].double()
        b = self.dtables[seq].long()[t // self.bs]
        return self.kp[b, t % self.bs].double(), self.vp[b, t % self.bs].double()

    def poison(self, seq, tokens):
        t = torch.as_tensor(tokens, device="cuda")
        if not self.bs:
            self.k[seq][t], self.v[seq][t] = float("nan"), float("inf")
            return
        b = self.dtables[seq].long()[t // self.bs]
        self.kp[b, t % self.bs], self.vp[b, t % self.bs] = float("nan"), float("inf")

    def decode(self, kv, ctx, q, g, lens, window, sinks, **kw):
        if self.bs:
            kv.decode_attn_paged_sinks(ctx, q, g, self.layout(), Q.i32(lens), window, sinks, **kw)
        else:
            kv.decode_attn_sinks(ctx, q, g, self.k_ptrs, self.v_ptrs, Q.i32(lens), window, sinks, **kw)

    def prefill(self, kv, ctx, q, g, row_seq, lens, window, sinks, **kw):
        rs = torch.as_tensor(np.asarray(row_seq), device="cuda").long()
        if self.bs:
            kv.prefill_attn_paged_sinks(ctx, q, g, self.layout(), Q.i32(row_seq), Q.i32(lens), window, sinks, **kw)
        else:
            kv.prefill_attn_sinks(ctx, q, g, self.k_ptrs[rs].contiguous(), self.v_ptrs[rs].contiguous(), Q.i32(lens), window, sinks, **kw)


LENS = [1, 2, 5, 16, 17, 63, 64, 65, 70, 130, 256, 257, 300, 511, 777, 1025, 2049, 4100]
VIEWS = [(1, 1), (1, 4), (7, 3), (64, 64), (100, 4), (63, 2), (255, 1), (256, 5), (300, 70), (300, 64), (1000, 300), (8000, 4), (50, 100000)]


def _ctx(n):
    return guarded(np.full((n, Q.NQ, Q.HD), 7.0, np.float16), "ctx")


@pytest.mark.parametrize("bs", [0, 16, 128])
@pytest.mark.parametrize("window,sinks", VIEWS)
def test_decode(kv, bs, window, sinks):
    c = F16Cache(LENS, bs, seed=60)
    q, g = Q.activations(len(LENS), 61)
    ctx = _ctx(len(LENS))
    c.decode(kv, ctx, q, g, LENS, window, sinks)
    assert kv.device_status() == 0
    Q.check_rows(ctx, q, g, [(i, i, Q.visible(n, window, sinks)) for i, n in enumerate(LENS)], c.values)


@pytest.mark.parametrize("bs", [0, 32])
def test_decode_without_window_or_sinks_is_the_plain_entry_point(kv, bs):
    c = F16Cache(LENS, bs, seed=62)
    q, g = Q.activations(len(LENS), 63)
    for window, sinks in ((0, 4), (100, 0), (0, 0)):
        a, b = _ctx(len(LENS)), _ctx(len(LENS))
        c.decode(kv, a, q, g, LENS, window, sinks)
        if bs:
            kv.decode_attn_paged(b, q, g, c.layout(), Q.i32(LENS), window)
        else:
            kv.decode_attn(b, q, g, c.k_ptrs, c.v_ptrs, Q.i32(LENS), window)
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("bs", [0, 16])
def test_decode_ignores_what_is_not_visible(kv, bs):
    lens, window, sinks = [500, 90, 40], 50, 13
    c = F16Cache(lens, bs, seed=64)
    q, g = Q.activations(3, 65)
    a, b = _ctx(3), _ctx(3)
    c.decode(kv, a, q, g, lens, window, sinks)
    for i, n in enumerate(lens):
        c.poison(i, np.setdiff1d(np.arange(n), Q.visible(n, window, sinks)))
    c.decode(kv, b, q, g, lens, window, sinks)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and kv.device_status() == 0


def test_decode_rows_do_not_depend_on_the_batch_and_bad_rows_are_skipped(kv):
    lens = [3000, 0, 777, MAX_SEQ + 1, 5000, 64]
    c = F16Cache([3000, 1, 777, 1, 5000, 64], 0, seed=66)
    q, g = Q.activations(6, 67)
    ctx = _ctx(6)
    c.k_ptrs[5] += 8
    c.decode(kv, ctx, q, None, lens, 600, 9)
    assert kv.device_status() == BAD_SEQ_LEN | MISALIGNED
    for i in (1, 3, 5):
        assert bool((ctx[i] == 7.0).all())
    Q.check_rows(ctx, q, None, [(i, i, Q.visible(lens[i], 600, 9)) for i in (0, 2, 4)], c.values)
    for i in (0, 2, 4):
        one = _ctx(1)
        kv.decode_attn_sinks(one, q[i:i + 1].contiguous(), None, c.k_ptrs[i:i + 1].contiguous(), c.v_ptrs[i:i + 1].contiguous(), Q.i32([lens[i]]), 600, 9)
        assert torch.equal(one[0].view(torch.int16), ctx[i].view(torch.int16))


def test_paged_decode_reports_bad_tables(kv):
    c = F16Cache([100, 40, 30], 16, seed=68)
    q, g = Q.activations(3, 69)
    a, b = _ctx(3), _ctx(3)
    c.decode(kv, a, q, g, [100, 40, 30], 20, 4)
    c.dtables[1, 0] = c.nblocks
    c.decode(kv, b, q, g, [100, 40, 16 * c.max_blocks + 1], 20, 4)
    assert kv.device_status() == BAD_SEQ_LEN | BAD_BLOCK
    assert torch.equal(a[0].view(torch.int16), b[0].view(torch.int16)) and bool((b[2] == 7.0).all())


@pytest.mark.parametrize("bs", [0, 16, 256])
@pytest.mark.parametrize("window,sinks", [(1, 1), (100, 4), (64, 70), (300, 33), (8000, 4)])
def test_fused_step_is_append_then_decode(kv, bs, window, sinks):
    lens = [0, 1, 3, 15, 16, 17, 63, 64, 100, 104, 255, 257, 700, 3001]
    n = len(lens)
    gen = torch.Generator(device="cuda").manual_seed(80)
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()  # noqa: E731
    q, k, v, g = half(n, 16, 128), half(n, 4, 128), half(n, 4, 128), half(n, 16)
    w = (1 + 0.1 * torch.randn(128, generator=gen, device="cuda")).half()
    ang = torch.rand(max(lens) + 1, 128, generator=gen, device="cuda") * 6.28
    cos, sin = ang.cos().half(), ang.sin().half()
    pos, sl = Q.i32(lens), Q.i32([x + 1 for x in lens])
    outs = []
    for fused in (False, True):
        c = F16Cache(lens, bs, seed=81)
        qq, ctx = q.clone(), _ctx(n)
        if bs and fused:
            kv.append_decode_paged_sinks(ctx, qq, k, v, g, w, w, cos, sin, sl, c.layout(), window, sinks)
        elif fused:
            kv.append_decode_sinks(ctx, qq, k, v, g, w, w, cos, sin, pos, sl, c.k_ptrs, c.v_ptrs, window, sinks)
        else:
            if bs:
                kv.append_paged(qq, k, v, w, w, cos, sin, pos, c.layout())
            else:
                kv.append(qq, k, v, w, w, cos, sin, pos, c.k_ptrs, c.v_ptrs)
            c.decode(kv, ctx, qq, g, [x + 1 for x in lens], window, sinks)
            Q.check_rows(ctx, qq, g, [(i, i, Q.visible(x + 1, window, sinks)) for i, x in enumerate(lens)], c.values)
        outs.append((ctx, torch.stack([torch.stack(c.values(i, [x])) for i, x in enumerate(lens)])))
        if fused:
            assert torch.equal(qq, q)  # read as the raw q
    assert kv.device_status() == 0
    assert torch.equal(outs[0][0].view(torch.int16), outs[1][0].view(torch.int16)) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (100, 4), (8, 4), (400, 20)])
@pytest.mark.parametrize("tail", [0, 1, 2, 3])
def test_fused_step_does_not_write_a_token_that_has_no_block(kv, window, sinks, tail):
    """The appended token's table entry is not a block of the pool: its key and value are not stored (block 0 belongs to another
    sequence here, whose result stays), and the context is that of append and decode attention one after the other."""
    lens = [16 + tail, 600, 560 + tail, 43]
    n = len(lens)
    gen = torch.Generator(device="cuda").manual_seed(92)
    half = lambda *s: torch.randn(*s, generator=gen, device="cuda").half()  # noqa: E731
    q, k, v, g = half(n, 16, 128), half(n, 4, 128), half(n, 4, 128), half(n, 16)
    w = (1 + 0.1 * torch.randn(128, generator=gen, device="cuda")).half()
    ang = torch.rand(max(lens) + 1, 128, generator=gen, device="cuda") * 6.28
    cos, sin = ang.cos().half(), ang.sin().half()
    pos, sl = Q.i32(lens), Q.i32([x + 1 for x in lens])
    outs = []
    for fused in (False, True):
        c = F16Cache(lens, 16, seed=93)
        c.kp.nan_to_num_(0.5)  # what is read in place of the missing block is finite
        c.vp.nan_to_num_(0.5)
        c.dtables[1, 0], c.dtables[0, 0], c.dtables[2, 3] = 0, 1, 2  # block 0 holds tokens that row 1 sees
        for i, entry in ((0, c.nblocks), (2, -1)):
            c.dtables[i, lens[i] // 16] = entry
        before = [p.clone() for p in (c.kp, c.vp)]
        qq, ctx = q.clone(), _ctx(n)
        if fused:
            kv.append_decode_paged_sinks(ctx, qq, k, v, g, w, w, cos, sin, sl, c.layout(), window, sinks)
        else:
            kv.append_paged(qq, k, v, w, w, cos, sin, pos, c.layout())
            c.decode(kv, ctx, qq, g, [x + 1 for x in lens], window, sinks)
        assert kv.device_status() == BAD_BLOCK
        for p, old, new in ((c.kp, before[0], None), (c.vp, before[1], v)):
            for i in (1, 3):  # the rows whose token has a block; everything else stays
                b = int(c.dtables[i, lens[i] // 16])
                if new is not None:
                    assert torch.equal(p[b, lens[i] % 16], new[i])
                old[b, lens[i] % 16] = p[b, lens[i] % 16]
            assert torch.equal(p, old)
        outs.append((ctx, c.kp, c.vp))
    assert all(torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16)) for a, b in zip(*outs))


WAVES = {
    "one row": [(0, 0, 1)],
    "a row behind a prefix": [(0, 900, 1)],
    "ragged": [(0, 0, 96), (1, 400, 128), (2, 17, 3), (3, 64, 64), (4, 1000, 33)],
    "many short": [(i, 29 * i, 1 + i % 5) for i in range(40)],
    "long prefix": [(0, 4000, 128)],
    "a full wave": [(i, 150 * i, 128) for i in range(8)],
}


@pytest.mark.parametrize("bs", [0, 16, 64])
@pytest.mark.parametrize("name", list(WAVES))
@pytest.mark.parametrize("window,sinks", [(1, 1), (100, 4), (64, 70), (500, 200), (3000, 64), (130, 5000)])
def test_prefill(kv, bs, name, window, sinks):
    chunks = WAVES[name]
    c = F16Cache([p + n for _, p, n in chunks], bs, seed=70)
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), 71)
    ctx = _ctx(len(pos))
    c.prefill(kv, ctx, q, g, row_seq, pos + 1, window, sinks)
    assert kv.device_status() == 0
    step = 1 + len(pos) // 60
    Q.check_rows(ctx, q, g, [(r, row_seq[r], Q.visible(pos[r] + 1, window, sinks)) for r in range(0, len(pos), step)], c.values)


@pytest.mark.parametrize("bs", [0, 32])
def test_prefill_without_window_or_sinks_is_the_plain_entry_point(kv, bs):
    c = F16Cache([200, 300], bs, seed=72)
    row_seq, pos = Q.wave([(0, 100, 100), (1, 172, 128)])
    q, g = Q.activations(len(pos), 73)
    rs = torch.as_tensor(row_seq, device="cuda")
    for window, sinks in ((0, 4), (100, 0)):
        a, b = _ctx(len(pos)), _ctx(len(pos))
        c.prefill(kv, a, q, g, row_seq, pos + 1, window, sinks)
        if bs:
            kv.prefill_attn_paged(b, q, g, c.layout(), Q.i32(row_seq), Q.i32(pos + 1), window)
        else:
            kv.prefill_attn(b, q, g, c.k_ptrs[rs].contiguous(), c.v_ptrs[rs].contiguous(), Q.i32(pos + 1), window)
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("bs", [0, 16])
@pytest.mark.parametrize("window,sinks", [(70, 21), (70, 64), (20, 130)])
def test_prefill_ignores_what_no_row_sees(kv, bs, window, sinks):
    c = F16Cache([700, 300], bs, seed=79)
    chunks = [(0, 600, 90), (1, 250, 40)]
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), 82)
    a, b = _ctx(len(pos)), _ctx(len(pos))
    c.prefill(kv, a, q, g, row_seq, pos + 1, window, sinks)
    for s, p, n in chunks:
        c.poison(s, np.arange(sinks, p + 1 - window))
        c.poison(s, np.arange(p + n, c.lens[s]))
    c.prefill(kv, b, q, g, row_seq, pos + 1, window, sinks)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and kv.device_status() == 0


@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("window,sinks", [(70, 4), (40, 40), (300, 90)])
def test_blocks_between_sinks_and_window_may_be_given_back(kv, bs, window, sinks):
    """Table entries of blocks without a visible token hold an id that the pool does not have: same bytes, no status."""
    c = F16Cache([700, 2000], bs, seed=90)
    chunks = [(0, 620, 60), (1, 1900, 100)]
    row_seq, pos = Q.wave(chunks)
    q, g = Q.activations(len(pos), 91)
    last = np.array([680, 2000])

    def both():
        a, b = _ctx(len(pos)), _ctx(2)
        c.prefill(kv, a, q, g, row_seq, pos + 1, window, sinks)
        c.decode(kv, b, q[:2], g[:2], last, window, sinks)
        return a, b

    want = both()
    for s, p, _ in chunks:
        c.dtables[s, -(-sinks // bs):(p + 1 - window) // bs] = -1
    got = both()
    assert kv.device_status() == 0
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip(want, got))


def test_prefill_skips_rows(kv):
    c = F16Cache([100, 40], 16, seed=74)
    row_seq, lens = [0, 0, 1, 1, 0], [5, 0, 40, 16 * c.max_blocks + 1, 100]
    q, g = Q.activations(5, 75)
    ctx = _ctx(5)
    c.prefill(kv, ctx, q, g, row_seq, lens, 30, 6)
    assert kv.device_status() == BAD_SEQ_LEN
    assert bool((ctx[1] == 7.0).all()) and bool((ctx[3] == 7.0).all())
    Q.check_rows(ctx, q, g, [(r, row_seq[r], Q.visible(lens[r], 30, 6)) for r in (0, 2, 4)], c.values)


def test_a_prompt_and_generated_tokens(kv):
    """Append and attention of the f16 path with a window and sinks: a prompt in one wave, then tokens one at a time."""
    window, sinks, total = 40, 4, 170
    cap = torch.zeros(2, total + 8, 4, 128, dtype=torch.float16, device="cuda")
    k_ptr, v_ptr = cap[0].data_ptr(), cap[1].data_ptr()
    g = torch.Generator(device="cuda").manual_seed(76)
    half = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    ang = torch.rand(total + 8, 128, device="cuda") * 6.28
    cos, sin = ang.cos().half(), ang.sin().half()
    n0 = 150
    q, k, v, gate = half(n0, 16, 128), half(n0, 4, 128), half(n0, 4, 128), half(n0, 16)
    kp = torch.full((n0,), k_ptr, dtype=torch.int64, device="cuda")
    vp = torch.full((n0,), v_ptr, dtype=torch.int64, device="cuda")
    pos = Q.i32(np.arange(n0))
    ctx = torch.zeros_like(q)
    values = lambda s, t: tuple(cap[i][torch.as_tensor(t, device="cuda")].double() for i in range(2))  # noqa: E731
    kv.append(q, k, v, w, w, cos, sin, pos, kp, vp)
    kv.prefill_attn_sinks(ctx, q, gate, kp, vp, pos + 1, window, sinks)
    Q.check_rows(ctx, q, gate, [(r, 0, Q.visible(r + 1, window, sinks)) for r in range(n0)], values)
    for p in range(n0, total):
        q, k, v, gate, ctx = half(1, 16, 128), half(1, 4, 128), half(1, 4, 128), half(1, 16), torch.zeros(1, 16, 128, dtype=torch.float16, device="cuda")
        kv.append(q, k, v, w, w, cos, sin, Q.i32([p]), kp[:1], vp[:1])
        kv.decode_attn_sinks(ctx, q, gate, kp[:1], vp[:1], Q.i32([p + 1]), window, sinks)
        Q.check_rows(ctx, q, gate, [(0, 0, Q.visible(p + 1, window, sinks))], values)
    assert kv.device_status() == 0


def test_refusals(kv):
    from oxide_infer_b200 import OxiError
    c, cp = F16Cache([20], 0, seed=77), F16Cache([20], 16, seed=77)
    q, g = Q.activations(1, 78)
    ctx = torch.zeros_like(q)

    def code(fn):
        with pytest.raises(OxiError) as e:
            fn()
        return e.value.code

    assert code(lambda: c.decode(kv, None, q, g, [20], 5, 2)) == -1
    assert code(lambda: cp.decode(kv, ctx, None, g, [20], 5, 2, batch=1)) == -1
    for x in (c, cp):
        assert code(lambda: x.decode(kv, ctx, q, g, [20], 5, 2, batch=65)) == -2
        assert code(lambda: x.prefill(kv, ctx, q, g, [0], [20], 5, 2, rows=1025)) == -2
        assert code(lambda: x.prefill(kv, ctx, q, g, [0], [20], 5, 2, rows=0)) == -2
    lay = cp.layout()
    lay.block_size = 24
    assert code(lambda: kv.decode_attn_paged_sinks(ctx, q, g, lay, Q.i32([20]), 5, 2)) == -3
