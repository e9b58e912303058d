"""Plain 64-bit forms of the rotary, norm-with-rotation and attention operators, their gradients, and bounds of what
the kernels' roundings can do to each result.

Arrays are [batch, tokens, heads, size] (the memory order of the device's [size, heads, tokens] x batch).  A sequence is
(sample, first query, queries, first key, keys).

The bounds count roundings to first order: U = 2^-24 per fp32 operation, H = half a step of the storage type per value
rounded to it (each probability, each dS, each result), a dot product of n terms n U of the sum of the absolute
products.  They hold element by element and are multiplied by SLACK for the second order.
"""
import numpy as np

U = 2.0 ** -24
HALF = {"f32": U, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# absolute rounding below the normal range (fp16's subnormal numbers; the others' are too small to matter)
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}
SLACK = 1.05


def places(bs, tq, tk, q_lens=None, k_lens=None, packed=False):
    if q_lens is None:
        return [(b, 0, tq, 0, tk) for b in range(bs)]
    out, aq, ak = [], 0, 0
    for i, (n, m) in enumerate(zip(q_lens, q_lens if k_lens is None else k_lens)):
        out.append((0, aq, n, ak, m) if packed else (i, 0, n, 0, m))
        aq, ak = aq + n, ak + m
    return out


# ---- attention ----------------------------------------------------------------


class Attention:
    """y, stats, gq, gk, gv and a bound for the error of each (tol_y, ...), for results stored as `storage`."""

    def __init__(self, q, k, v, seqs, causal, scale, storage, gy=None):
        q, k, v = (x.astype(np.float64) for x in (q, k, v))
        d, g = q.shape[3], q.shape[2] // k.shape[2]
        h = HALF[storage]
        wide = storage == "f32"
        self.y, self.tol_y = np.zeros_like(q), np.zeros_like(q)
        self.stats = np.full(q.shape[:3], -np.inf)
        self.tol_stats = np.zeros(q.shape[:3])
        if gy is not None:
            gy = gy.astype(np.float64)
            self.gq, self.gk, self.gv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
            self.tol_gq, self.tol_gk, self.tol_gv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
        for b, aq, n, ak, m in seqs:
            if n == 0 or m == 0:
                continue
            i, j = np.arange(n)[:, None], np.arange(m)[None, :]
            seen = (j <= i + m - n) if causal else np.ones((n, m), dtype=bool)
            some = seen.any(1)
            for hq in range(q.shape[2]):
                at_q, at_k = (b, slice(aq, aq + n), hq), (b, slice(ak, ak + m), hq // g)
                # what is masked may hold anything
                Q, K, V = q[at_q], k[at_k], v[at_k]
                with np.errstate(all="ignore"):
                    s = scale * (Q @ K.T)
                    size = scale * (np.abs(Q) @ np.abs(K).T)
                s = np.where(seen, s, -np.inf)
                top = np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None]
                e = np.exp(s - top)
                total = e.sum(1)
                P = e / np.where(some, total, 1.0)[:, None]
                self.stats[at_q] = np.where(some, top[:, 0] + np.log(np.where(some, total, 1.0)), -np.inf)
                size = np.where(seen, size, 0.0)
                # the score's products and sum, its scaling, the exponent's subtraction and the exponential itself
                ds = (d + 4) * U * size.max(1, initial=0.0) + 4 * U * np.abs(np.where(seen, s, 0)).max(1, initial=0.0) + 8 * U
                self.tol_stats[at_q] = np.where(some, 2 * ds + m * U + 4 * U * np.abs(np.where(some, self.stats[at_q], 0)) + 4 * U, 0)
                dP = 2 * ds + (m + 8) * U + (0 if wide else h)   # relative, of a normalised probability
                low = np.where(some, 1.0, 0.0)[:, None] * (TINY[storage] if not wide else 0.0)
                absV = np.abs(V)
                y = P @ V
                self.y[at_q] = y
                tol_y = (dP[:, None] + (m + 4) * U) * (P @ absV) + low * absV.sum(0) + h * np.abs(y) + TINY[storage]
                self.tol_y[at_q] = SLACK * np.where(some[:, None], tol_y, 0)
                if gy is None:
                    continue
                G = gy[at_q]
                absG = np.abs(G)
                gv = P.T @ G
                self.gv[at_k] += gv
                # P is computed anew from stats here: once more the score's error and that of stats
                dP = dP + ds + self.tol_stats[at_q] * some
                self.tol_gv[at_k] += (P * (dP + (n * g + 4) * U)[:, None]).T @ absG + (low * np.ones_like(P)).T @ absG
                dp, delta = G @ V.T, (G * y).sum(1)[:, None]
                dS = P * (dp - delta)
                at_dp = (d + 4) * U * (absG @ absV.T) + (absG * (tol_y + (d + 4) * U * np.abs(y))).sum(1)[:, None]
                # the difference, times P, rounded (16-bit storage rounds P once and dS once; fp32 neither)
                at_dS = P * (np.abs(dp - delta) * (dP + 4 * U)[:, None] + at_dp) + h * np.abs(dS) + low
                self.gq[at_q] = scale * (dS @ K)
                self.tol_gq[at_q] = scale * ((at_dS + (m + 4) * U * np.abs(dS)) @ np.abs(K))
                self.gk[at_k] += scale * (dS.T @ Q)
                self.tol_gk[at_k] += scale * ((at_dS + (n * g + 4) * U * np.abs(dS)).T @ np.abs(Q))
        if gy is not None:
            for name in ("q", "k", "v"):
                r, t = getattr(self, "g" + name), getattr(self, "tol_g" + name)
                setattr(self, "tol_g" + name, SLACK * (t + h * np.abs(r) + TINY[storage]))


# ---- rotary positions -----------------------------------------------------------


def positions(shape, seqs, first):
    """Positions [batch, tokens], and which tokens belong to a sequence."""
    at, used = np.zeros(shape[:2], dtype=np.int64), np.zeros(shape[:2], dtype=bool)
    for b, a, n, _, m in seqs:
        at[b, a:a + n] = first + (m - n) + np.arange(n)
        used[b, a:a + n] = True
    return at, used


def turned(x, at, freqs, interleaved, amplitude, sign=1):
    """x rotated; with the sum of the absolute parts of each element (for bounds)."""
    p = len(freqs)
    angle = at[:, :, None, None].astype(np.float64) * np.asarray(freqs, dtype=np.float64)
    c, s = amplitude * np.cos(angle), sign * amplitude * np.sin(angle)
    y, size = x.copy(), np.abs(x)
    i0 = slice(0, 2 * p, 2) if interleaved else slice(0, p)
    i1 = slice(1, 2 * p, 2) if interleaved else slice(p, 2 * p)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = abs(amplitude) * (np.abs(a) + np.abs(b))
    return y, size


# cosine and sine: half a step, the reduced angle (half a step of pi / 4), the series and the amplitude; product and sum
TURN = 8 * U


class Rotary:
    """y, and with gy the gradients gx and gw, for one of queries and keys; w None: no norm."""

    def __init__(self, x, seqs, freqs, storage, interleaved=False, first=0, amplitude=1.0, w=None, eps=0.0, gy=None):
        h = HALF[storage]
        x = x.astype(np.float64)
        d = x.shape[3]
        at, used = positions(x.shape, seqs, first)
        mask = used[:, :, None, None]
        norm = w is not None
        if norm:
            w = w.astype(np.float64)
            r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
            n, rel = x * r * w, (d / 2 + 8) * U   # half of the sum's relative error, the root, the division, two products
        else:
            n, rel = x, 0.0
        y, size = turned(n, at, freqs, interleaved, amplitude)
        self.y = np.where(mask, y, 0)
        self.tol_y = SLACK * np.where(mask, size * (TURN + rel) + h * np.abs(y) + TINY[storage], 0)
        if gy is None:
            return
        g, gsize = turned(np.where(mask, gy.astype(np.float64), 0), at, freqs, interleaved, amplitude, -1)
        if not norm:
            self.gx, self.tol_gx = g, SLACK * (gsize * TURN + h * np.abs(g) + TINY[storage])
            return
        mean, mean_size = (g * w * x).mean(-1, keepdims=True), (gsize * np.abs(w * x)).mean(-1, keepdims=True)
        self.gx = np.where(mask, r * (g * w - x * r * r * mean), 0)
        size = r * (gsize * np.abs(w) + np.abs(x) * r * r * mean_size)
        self.tol_gx = SLACK * np.where(mask, size * (TURN + (2.5 * d + 24) * U) + h * np.abs(self.gx) + TINY[storage], 0)
        rows = np.where(mask, g * x * r, 0)
        count = x.shape[0] * x.shape[1] * x.shape[2]
        self.gw = rows.sum((0, 1, 2))
        size = np.where(mask, gsize * np.abs(x) * r, 0).sum((0, 1, 2))
        self.tol_gw = SLACK * (size * (TURN + (d / 2 + 8 + count) * U) + h * np.abs(self.gw) + TINY[storage])
