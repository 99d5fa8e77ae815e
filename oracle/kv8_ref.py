"""The 8-bit paged KV cache restated on the CPU in 64 bits, from the statement of its
format in include/acorn_hip.h: a table of the 256 e4m3 numbers, quantisation as the
nearest of them (ties to the even code), tile offsets one by one, attention over the
values the bytes stand for. No counterpart in the reference: parity unpinned."""
import math

import numpy as np
import torch


def _e4m3_table() -> np.ndarray:
    out = np.empty(256)
    for b in range(256):
        ex, man = b >> 3 & 15, b & 7
        x = (8 + man) * 2.0 ** (ex - 10) if ex else man * 2.0 ** -9
        out[b] = math.nan if ex == 15 and man == 7 else (-x if b & 128 else x)
    return out


E4M3 = _e4m3_table()
_POS = E4M3[:127]                       # 0 .. 448, rising


def scale_exp(amax: float) -> int:
    """The least e >= -126 with amax <= 448 * 2^e."""
    e = -126
    if amax > 0:
        e = max(e, math.frexp(amax)[1] - 10)
    while amax > math.ldexp(448.0, e):
        e += 1
    return e


def quantise_row(x: np.ndarray, fp16: bool) -> tuple[np.ndarray, int, bool]:
    """(bytes, code, whether the row is finite) of x [D] in 64 bits."""
    if not np.isfinite(x).all():
        return np.zeros(len(x), np.uint8), 255, False
    # (what is held has to be finite when it is read: in fp16 2^16, else 2^128 is not)
    top = 61440.0 if fp16 else math.ldexp(240.0, 120)
    x = np.clip(x, -top, top)
    e = scale_exp(float(np.abs(x).max()))
    y = np.abs(x) * 2.0 ** -e if e > -1000 else x
    hi = np.clip(np.searchsorted(_POS, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POS[hi] - y, y - _POS[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(y == _POS[hi], hi, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), e + 127, True


def k_byte(t: int, d: int, D: int) -> int:
    return d // 16 * 256 + t * 16 + d % 16


def v_byte(t: int, d: int, D: int) -> int:
    E = D // 16
    TP = 16 // E
    return t % 4 // TP * 1024 + (16 * (t // 4) + d // E) * 16 + t % TP * E + d % E


class Pool:
    """One layer's pages as numpy bytes."""

    def __init__(self, num_blocks, KV, D, P):
        self.NB, self.KV, self.D, self.P = num_blocks, KV, D, P
        self.k = np.zeros((num_blocks, KV, P // 16, 16 * D), np.uint8)
        self.v = np.zeros_like(self.k)
        self.scales = np.zeros((num_blocks, KV, P // 16, 32), np.uint8)
        t = np.arange(16)[:, None]
        d = np.arange(D)[None]
        self.kp = np.vectorize(lambda a, b: k_byte(a, b, D))(t, d)       # [16, D]
        self.vp = np.vectorize(lambda a, b: v_byte(a, b, D))(t, d)
        for p in (self.kp, self.vp):
            assert sorted(p.reshape(-1)) == list(range(16 * D))

    @classmethod
    def of(cls, kv, P):
        """The pool that a KV8Pages holds."""
        k = kv.k.cpu().numpy()
        p = cls(k.shape[0], k.shape[1], k.shape[3] // 16, P)
        p.k, p.v, p.scales = k, kv.v.cpu().numpy(), kv.scales.cpu().numpy()
        return p

    def put(self, k, v, pages, slots, fp16=False):
        """Rows k, v [R, KV, D] at (pages[i], slots[i]); targets outside are skipped."""
        k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
        for i, (b, s) in enumerate(zip(pages.tolist(), slots.tolist())):
            if not (0 <= b < self.NB and 0 <= s < self.P):
                continue
            g, t = s // 16, s % 16
            for h in range(self.KV):
                kb, kc, kok = quantise_row(k[i, h], fp16)
                vb, vc, vok = quantise_row(v[i, h], fp16)
                if not (kok and vok):
                    kb, vb, kc, vc = kb * 0, vb * 0, 255, 255
                self.k[b, h, g, self.kp[t]] = kb
                self.v[b, h, g, self.vp[t]] = vb
                self.scales[b, h, g, t] = kc
                self.scales[b, h, g, 16 + t] = vc

    def values(self, table, tokens):
        """k, v [len(tokens), KV, D] in 64 bits of the tokens of a block table."""
        out = []
        tok = np.asarray(list(tokens), dtype=np.int64)
        tab = np.asarray(table)
        b, g, t = tab[tok // self.P], tok % self.P // 16, tok % 16
        for tiles, place, first in ((self.k, self.kp, 0), (self.v, self.vp, 16)):
            x = E4M3[tiles[b[:, None, None], np.arange(self.KV)[None, :, None], g[:, None, None],
                           place[t][:, None, :]]]
            c = self.scales[b[:, None], np.arange(self.KV)[None], g[:, None], (t + first)[:, None]]
            s = np.where(c == 255, math.nan, 2.0 ** (c.astype(np.float64) - 127))
            out.append(torch.from_numpy(x * s[..., None]))
        return out


def attend(q, k, v):
    """q [H, D], k, v [L, KV, D] in 64 bits -> (out [H, D], the weighted mean of |v| [H, D], the
    largest sum of |q k| of a score): the mean and the sum bound what roundings can change."""
    H, D = q.shape
    rep = H // k.shape[1]
    kf = k.repeat_interleave(rep, 1)
    s = torch.einsum("hd,lhd->hl", q.double(), kf) * D ** -0.5
    big = (torch.einsum("hd,lhd->hl", q.double().abs(), kf.abs()) * D ** -0.5).amax() if len(k) else 0
    p = torch.softmax(s, -1)
    vf = v.repeat_interleave(rep, 1)
    return torch.einsum("hl,lhd->hd", p, vf), torch.einsum("hl,lhd->hd", p, vf.abs()), float(big)


def tolerance(out, mean_abs, big, dtype, L, terms=1):
    """Elementwise bound on |kernel - out|. A score is a sum of D products in 32 bits, its factor
    and the exponential (together under 2^-16 of the sum of magnitudes `big`, plus 2^-20); the
    result is rounded once (u). The weights p: with terms=1 (prompt rows) they are rounded to the
    type (u each, and their sum with them: 2 u of the mean of |v|), and fp16 weights, held
    times 2^7, have no steps finer than 2^-24 (of a largest weight of 1 or more, L of them);
    with terms=2 (decode, windows) they are two bf16 terms: p cut to 8 bits leaves under 2^-7
    of it, rounded to 8 bits itself, half a step of which is 2^-16 of p at most."""
    u = torch.finfo(dtype).eps / 2
    e = (u if terms == 1 else 2.0 ** -16) + big * 2.0 ** -16 + 2.0 ** -20
    sub = 2.0 ** -32 * L if dtype == torch.float16 and terms == 1 else 0.0
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return 2 * (e + sub) * mean_abs + u * out.abs() * (1 + 2 ** -6) + tiny
