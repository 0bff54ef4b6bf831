"""Plain 64-bit forms of the 8-bit cache operators and of windowed attention with sinks, seeded inputs for their
tests, and the tolerances that the arithmetic allows.

Tolerance of an attention output (attention_bound): o = sum p v / sum p * g, rounded to f16 once.
  rounding of the result                      2^-11 |o|
  weights rounded to f16 for the product      2^-11 of each term of the numerator: 2^-11 A, A = sum p |v| / sum p * g
  weights below f16's normal range            2^-25 each, relative to a largest weight of at least 1: n 2^-25 max|v| g
  scores: 128 products added in f32           each addition within 2^-22 (twice a rounding, and the tensor core's
                                              truncation): dx <= 130 * 2^-22 * max_t sum_i |q_i k_ti| / sqrt(128); a weight
                                              is off by the factor e^dx, in numerator and denominator: 2 dx A
  exp2, reciprocal, sigmoid, f32 sums         2^-18 A: approximate instructions 2^-22, sums of slices 2^-22 a step
Keys dequantised by the reference form are exact products in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import torch

from tests.kvcase import guarded

NQ, NKV, GRP, HD = 16, 4, 4, 128
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}


def visible(length, window, sinks):
    """Tokens that a row of the given length sees, ascending."""
    start = length - window if window and length > window else 0
    return np.concatenate([np.arange(min(sinks, start)), np.arange(start, length)]).astype(np.int64)


def scale64(amax, fmt):
    if fmt == "int8":
        return amax / 127.0
    return np.where(amax > 0, np.exp2(np.ceil(np.log2(np.where(amax > 0, amax, 1.0) / 448.0))), 0.0)


def quantise_blocks(x, fmt):
    """Codes (torch, cpu) and scales (float32) of x [blocks][bs][4][128]."""
    s = scale64(np.abs(x).max(axis=(1, 3)), fmt).astype(np.float32)
    y = torch.from_numpy(x / np.where(s > 0, s, 1)[:, None, :, None]).float()
    codes = torch.round(y).clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, torch.from_numpy(s)


def norm_rope64(x, w, cos, sin, eps=1e-5):
    """x [rows][heads][128], cos / sin [rows][128]"""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    half = np.concatenate([-y[..., 64:], y[..., :64]], -1)
    return y * cos[:, None].astype(np.float64) + half * sin[:, None].astype(np.float64)


class Q8Cache:
    """An 8-bit paged cache on the GPU: `lens` tokens per sequence in scattered blocks, with guard bands.  Slots and blocks
    that no sequence uses hold the worst bytes of the format; extra strides put gaps between the blocks."""

    def __init__(self, lens, fmt, bs, seed=0, spare=1, gap=0, scale_gap=0, vscale=1.0, kscale=1.0):
        rng = np.random.default_rng(seed)
        self.lens, self.fmt, self.bs = list(lens), fmt, bs
        need = [max(1, -(-(int(n) + spare) // bs)) for n in lens]
        self.nblocks = sum(need) + 2
        perm = rng.permutation(self.nblocks).astype(np.int32)
        self.max_blocks = max(need) + 1
        self.tables = np.full((len(lens), self.max_blocks), self.nblocks - 1, np.int32)
        o = 0
        for i, k in enumerate(need):
            self.tables[i, :k] = perm[o:o + k]
            o += k
        mags = np.exp(0.7 * rng.standard_normal((2, self.nblocks, 1, 1, 1))).astype(np.float32)
        used = np.zeros((self.nblocks, bs), bool)
        for i, n in enumerate(lens):
            for t in range(0, int(n), bs):
                used[self.tables[i, t // bs], :min(bs, int(n) - t)] = True
        k = rng.standard_normal((self.nblocks, bs, NKV, HD), dtype=np.float32) * kscale
        v = rng.standard_normal((self.nblocks, bs, NKV, HD), dtype=np.float32) * mags[1] * vscale
        (kc, ks), (vc, vs) = quantise_blocks(np.where(used[:, :, None, None], k, 0), fmt), quantise_blocks(np.where(used[:, :, None, None], v, 0), fmt)
        worst = 0x7f if fmt == "e4m3" else 0x80  # NaN; -128, which no token has
        for c in (kc, vc):
            c.view(torch.uint8)[torch.from_numpy(~used)] = worst
        idle = torch.from_numpy(~used.any(1))
        ks[idle], vs[idle] = float("nan"), float("nan")
        self.used = used
        pitch, spitch = bs * NKV * HD + gap, NKV + scale_gap
        self.kp, self.vp = self._strided(kc, pitch, "k_pool"), self._strided(vc, pitch, "v_pool")
        self.ks, self.vs = self._scales(ks, spitch, "k_scales"), self._scales(vs, spitch, "v_scales")
        self.dtables = torch.from_numpy(self.tables).cuda()

    def _strided(self, codes, pitch, label):
        flat = torch.full((self.nblocks, pitch), 0x5a, dtype=torch.uint8)
        flat[:, :self.bs * NKV * HD] = codes.view(torch.uint8).reshape(self.nblocks, -1)
        d = guarded(flat, label)
        return d[:, :self.bs * NKV * HD].view(CODE[self.fmt]).unflatten(1, (self.bs, NKV, HD))

    def _scales(self, s, pitch, label):
        flat = torch.zeros(self.nblocks, pitch)
        flat[:, :NKV] = s
        return guarded(flat, label)[:, :NKV]

    def layout(self):
        from oxide_infer_b200 import PagedQ8Layout
        return PagedQ8Layout.of(self.kp, self.vp, self.ks, self.vs, self.dtables)

    def values(self, seq, tokens):
        """k, v [len(tokens)][4][128] in float64 (cuda)"""
        t = torch.as_tensor(tokens, device="cuda")
        b = self.dtables[seq].long()[t // self.bs]
        return tuple(p[b, t % self.bs].double() * s.double()[b][..., None] for p, s in ((self.kp, self.ks), (self.vp, self.vs)))


def attention64(q, gate, k, v):
    """One row: q [16][128], gate [16] or None, k / v [n][4][128] float64; returns the result and its tolerance."""
    q = q.double().view(NKV, GRP, HD)
    kk, vv = k.permute(1, 2, 0), v.permute(1, 0, 2)  # [4][128][n], [4][n][128]
    x = q @ kk / math.sqrt(HD)
    dx = (q.abs() @ kk.abs()).amax(-1) / math.sqrt(HD) * 130 * 2.0 ** -22  # [4][4]
    p = torch.softmax(x, -1)
    o, a = p @ vv, p @ vv.abs()
    g = torch.ones(NQ, device=q.device, dtype=torch.float64) if gate is None else torch.sigmoid(gate.double())
    g = g.view(NKV, GRP, 1)
    o, a = o * g, a * g
    small = k.shape[0] * 2.0 ** -25 * vv.abs().amax(dim=(1, 2)).view(NKV, 1, 1) * g
    tol = 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -18 + 2 * dx[..., None]) * a + small + 2.0 ** -25
    return o.reshape(NQ, HD), tol.reshape(NQ, HD)


def check_rows(ctx, q, gate, rows, kv_of):
    """rows: (row, seq, tokens); kv_of(seq, tokens) -> k, v in float64."""
    worst = 0.0
    for r, seq, tokens in rows:
        k, v = kv_of(seq, tokens)
        o, tol = attention64(q[r], None if gate is None else gate[r], k, v)
        err = (ctx[r].double() - o).abs()
        assert bool(torch.isfinite(ctx[r]).all()), (r, seq, len(tokens))
        over = float((err / tol).max())
        worst = max(worst, over)
        assert over <= 1.0, (r, seq, len(tokens), over)
    return worst


def activations(rows, seed, scale=1.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(rows, NQ, HD, generator=g, device="cuda") * scale).half()
    gate = torch.randn(rows, NQ, generator=g, device="cuda").half()
    return q, gate


def i32(a):
    return torch.as_tensor(np.asarray(a, dtype=np.int64).astype(np.uint32).view(np.int32), device="cuda")


def wave(chunks):
    """chunks: (seq, first position, rows) -> row_seq, pos"""
    return (np.concatenate([np.full(n, s) for s, _, n in chunks]).astype(np.int64),
            np.concatenate([np.arange(p, p + n) for _, p, n in chunks]).astype(np.int64))
