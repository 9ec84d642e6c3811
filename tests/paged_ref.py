"""Plain numpy forms of the paged 4-bit cache, written from its definition:
bytes by address, quantization in the f32 steps that define it, attention in 64
bits.  Test infrastructure only."""
import numpy as np


def groups(hd, vd):
    d = max(hd, vd)
    return 2 if d <= 64 else 4 if d <= 128 else 8


def bf16_round(x):
    """f32 values rounded to bf16 (nearest even), as f32."""
    b = np.asarray(x, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32))


def quantize(x):
    """[.., 32] f32 -> codes 0..15 and f16 scales."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top, low = x.max(-1), x.min(-1)
        e = np.where(top >= -low, top, low).astype(np.float32) * np.float32(-0.125)
        d = (np.clip(e, np.float32(-8188), np.float32(8188)) + np.float32(0)).astype(np.float16)  # no -0
        df = d.astype(np.float32)
        r = np.where(df == 0, np.float32(0), np.float32(1) / df).astype(np.float32)
        c = np.clip(np.rint((x * r[..., None]).astype(np.float32)), -8, 7)
    return (np.nan_to_num(c, nan=-8.0) + 8).astype(np.uint8), d  # a NaN group: codes 0


class Pool:
    """A host pool: k and v byte arrays, addressed byte by byte."""

    def __init__(self, n_pages, ps, n_kv, hd, vd=None, fill=0xFF):
        self.n_pages, self.ps, self.n_kv, self.hd, self.vd = n_pages, ps, n_kv, hd, vd or hd
        self.G = groups(hd, self.vd)
        self.block = ps * 18 * self.G
        # 0xFFFF is a NaN scale: bytes nobody wrote poison whoever reads them
        self.k = np.full(n_pages * n_kv * self.block, fill, np.uint8)
        self.v = self.k.copy()

    def _at(self, page, head):
        return (page * self.n_kv + head) * self.block

    def store(self, which, page, off, rows):
        """rows [n_kv][dim] f32 at token `off` of `page`."""
        buf, G = (self.k if which == "k" else self.v), self.G
        dim = rows.shape[1]
        x = np.zeros((self.n_kv, 32 * G), np.float32)
        x[:, :dim] = rows
        codes, d = quantize(x.reshape(self.n_kv, G, 32))
        for h in range(self.n_kv):
            at = self._at(page, h)
            for g in range(G):
                c = codes[h, g].astype(np.uint8)
                if which == "k":
                    for kc in range(4):
                        for b in range(4):
                            buf[at + off * 16 * G + (kc * G + g) * 4 + b] = c[8 * kc + 2 * b] | c[8 * kc + 2 * b + 1] << 4
                else:
                    for i in range(16):
                        buf[at + ((off // 4 * 16 + i) * 4 + off % 4) * G + g] = c[i] | c[16 + i] << 4
                s = at + self.ps * 16 * G + (off * G + g) * 2
                buf[s:s + 2] = np.frombuffer(d[h, g].tobytes(), np.uint8)

    def load(self, which, page, off):
        """[n_kv][dim] values (f64, exact)."""
        buf, G = (self.k if which == "k" else self.v), self.G
        out = np.zeros((self.n_kv, 32 * G))
        for h in range(self.n_kv):
            at = self._at(page, h)
            for g in range(G):
                s = at + self.ps * 16 * G + (off * G + g) * 2
                d = float(buf[s:s + 2].view(np.float16)[0])
                c = np.zeros(32)
                if which == "k":
                    b = np.concatenate([buf[at + off * 16 * G + (kc * G + g) * 4:][:4] for kc in range(4)])
                    c[0::2], c[1::2] = b & 15, b >> 4
                else:
                    first = at + (off // 4 * 16 * 4 + off % 4) * G + g
                    b = buf[first:first + 64 * G:4 * G][:16]
                    c[:16], c[16:] = b & 15, b >> 4
                out[h, 32 * g:32 * g + 32] = d * (c - 8)
        return out[:, :self.hd if which == "k" else self.vd]


def rotate(x, cos, sin, neox):
    """[heads][dim] f32 by one position's cos / sin [rot / 2]: products rounded to
    f32 before they are added."""
    x = np.asarray(x, np.float32)
    out = x.copy()
    n = cos.shape[0]
    a, b = (x[:, :n], x[:, n:2 * n]) if neox else (x[:, 0:2 * n:2], x[:, 1:2 * n:2])
    u = (a * cos).astype(np.float32) - (b * sin).astype(np.float32)
    w = (a * sin).astype(np.float32) + (b * cos).astype(np.float32)
    if neox:
        out[:, :n], out[:, n:2 * n] = u, w
    else:
        out[:, 0:2 * n:2], out[:, 1:2 * n:2] = u, w
    return out


def attention(pool, table, kv_lens, q_starts, q, scale, window=0, sinks=None):
    """64-bit attention of q [rows][heads][hd].  Returns out, and per (row, head)
    the bounds that a tolerance is made of: sum p |v| / sum p per channel, and of
    scale times the row's keys at their largest 2 max |q| sum |k| + hd sum |q k|, and
    sum |q k|."""
    rows, heads, hd = q.shape
    mul = heads // pool.n_kv
    out = np.full((rows, heads, pool.vd), np.nan)
    spread = np.zeros((rows, heads, pool.vd))
    size = np.zeros((2, rows, heads))
    cached = {}
    for s in range(len(kv_lens)):
        a, b = q_starts[s], q_starts[s + 1]
        for r in range(a, b):
            pos = kv_lens[s] - (b - r)
            keys = []
            for t in range(max(0, pos - window + 1) if window else 0, pos + 1):
                if t // pool.ps >= table.shape[1]:
                    continue
                page = table[s, t // pool.ps]
                if 0 <= page < pool.n_pages:
                    keys.append((page, t % pool.ps))
            if not keys:
                out[r] = 0.0
                continue
            for key in keys:
                if key not in cached:
                    cached[key] = (pool.load("k", *key), pool.load("v", *key))
            k = np.stack([cached[key][0] for key in keys])
            v = np.stack([cached[key][1] for key in keys])
            for h in range(heads):
                x = q[r, h].astype(np.float64)
                w = scale * (k[:, h // mul] @ x)
                top = w.max() if sinks is None else max(w.max(), float(sinks[h]))
                p = np.exp(w - top)
                total = p.sum() + (0.0 if sinks is None else np.exp(float(sinks[h]) - top))
                out[r, h] = p @ v[:, h // mul] / total
                spread[r, h] = p @ np.abs(v[:, h // mul]) / total
                ka = np.abs(k[:, h // mul])
                size[1, r, h] = abs(scale) * (ka @ np.abs(x)).max()
                size[0, r, h] = abs(scale) * 2 * np.abs(x).max() * ka.sum(1).max() + hd * size[1, r, h]
    return out, spread, size


def tolerance(out, spread, size, dtype):
    """How far a computed value may be from the 64-bit one.

    Scores: a query is held to 2^-24 of its row's largest value, codes and scales
    are exact, and at most hd + 8 f32 additions and multiplications round by 2^-24
    each of partial sums no larger than sum |q k|: together under 2^-23 size[0].  In
    a long chunk's bf16 rows a key is one half besides: 2^-12 size[1].  A score off
    by x changes p by a factor within exp(+-x), in the numerator and in the sum: 2 x
    (1.1 for the second order; x < 0.05).  exp2 itself and the running rescales:
    2^-19.  p d, or p and d (c - 8), are two halves each for f32 rows, less the
    product of the small ones: 2^-20 of each term; one half each for bf16 rows:
    2^-11.  The f32 sums over the cached rows: 2^-17.  bf16 outputs round by 2^-8 of
    themselves."""
    x = 2.0 ** -23 * size[0] + (2.0 ** -12 * size[1] if dtype == "bf16" else 0.0)
    assert x.max(initial=0.0) < 0.05
    rel = 2.2 * x + 2.0 ** -19 + 2.0 ** -17 + (2.0 ** -20 if dtype == "f32" else 2.0 ** -11)
    tol = spread * rel[..., None] + 1e-30
    return tol + (2.0 ** -8 * (np.abs(out) + tol) if dtype == "bf16" else 0.0)
