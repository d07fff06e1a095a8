"""The 8-bit K/V cache's definition in numpy (include/qwen_hip_kv8.h), token by token in 64 bits."""

from __future__ import annotations

import numpy as np


def place(which: str, dim: int) -> np.ndarray:
    """[64, dim] byte offsets of token t, dimension d within a block."""
    at = np.empty((64, dim), np.int64)
    for t in range(64):
        for d in range(dim):
            at[t, d] = (d // 64 * 64 + t) * 64 + d % 64 if which == "k" else d * 64 + 16 * (t // 4 % 4) + 4 * (t // 16) + t % 4
    return at


def need(x: np.ndarray) -> float:
    if not np.all(np.isfinite(x)):
        return float("nan")
    s = 2.0 ** -126
    while np.max(np.abs(x), initial=0.0) > 127 * s:
        s *= 2
    return s


class Cache:
    """Codes [sequences, blocks, kv, 64, dim] and scales [sequences, blocks, kv], K and V."""

    def __init__(self, code: dict, scale: dict):
        self.code = {n: c.astype(np.int64) for n, c in code.items()}
        self.scale = {n: s.astype(np.float64) for n, s in scale.items()}
        self.tokens = code["k"].shape[1] * 64

    @classmethod
    def of(cls, cache, layer: int = 0):
        """What a Kv8Cache holds."""
        code, scale = {}, {}
        for n in "kv":
            raw = getattr(cache, n)[layer].cpu().numpy()
            code[n] = raw[..., place(n, cache.head_dim)]
            scale[n] = getattr(cache, n + "_scale")[layer].cpu().numpy()
        return cls(code, scale)

    def store(self, k: np.ndarray, v: np.ndarray, positions) -> None:
        for n, x in (("k", k), ("v", v)):
            for b, pos in enumerate(positions):
                rows = min(x.shape[1], self.tokens - pos)
                if pos < 0 or rows <= 0:
                    continue
                for h in range(x.shape[2]):
                    for j in range(pos // 64, (pos + rows - 1) // 64 + 1):
                        lo, hi = max(pos, 64 * j), min(pos + rows, 64 * j + 64)
                        new = x[b, lo - pos:hi - pos, h].astype(np.float64)
                        s, old = need(new), self.scale[n][b, j, h]
                        if lo > 64 * j:
                            s = float("nan") if np.isnan(s) or np.isnan(old) else max(s, old)
                        c = self.code[n][b, j, h]
                        if np.isnan(s):
                            c[lo - 64 * j:hi - 64 * j] = 0
                        else:
                            c[:lo - 64 * j] = np.rint(c[:lo - 64 * j] * (old / s)) if lo > 64 * j else 0
                            c[lo - 64 * j:hi - 64 * j] = np.rint(new / s)
                        self.scale[n][b, j, h] = s

    def values(self, n: str, b: int) -> np.ndarray:
        """[tokens, kv, dim]"""
        v = self.code[n][b] * self.scale[n][b][:, :, None, None]
        return v.transpose(0, 2, 1, 3).reshape(self.tokens, v.shape[1], v.shape[3])

    def attend(self, q: np.ndarray, positions, scale: float):
        """(out, slack, floor, reach): slack[b, i, h, d] = sum_j p_j |v_jd|, floor = sum_j |v_jd| times the largest p,
        reach[b, i, h] = max_j scale sum_d |q_d k_jd|."""
        out, slack, floor, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3])
        group = q.shape[2] // self.code["k"].shape[2]
        for b, pos in enumerate(positions):
            k, v = self.values("k", b), self.values("v", b)
            for i in range(q.shape[1] if pos >= 0 else 0):
                n = min(pos + i + 1, self.tokens)
                for h in range(q.shape[2]):
                    kk, vv = k[:n, h // group], v[:n, h // group]
                    z = scale * (kk @ q[b, i, h].astype(np.float64))
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    out[b, i, h], slack[b, i, h], floor[b, i, h] = p @ vv, p @ np.abs(vv), p.max() * np.abs(vv).sum(0)
                    reach[b, i, h] = abs(scale) * (np.abs(kk) @ np.abs(q[b, i, h].astype(np.float64))).max()
        return out, slack, floor, reach


def tolerance(dtype: str, dim: int, slack: np.ndarray, floor: np.ndarray, reach: np.ndarray, out: np.ndarray) -> np.ndarray:
    """Largest error of the attention.  A score is a sum of dim exact products in fp32, at most dim + 4 roundings of
    2^-24 relative to sum |q k| (reach), of a query known to 2^-22 of its largest element (two fp16 terms; one
    holds a bf16 query); four further fp32 roundings of the scaled score and exp2's ulp.  A probability enters
    with a relative error of 2^-22 (two terms) or 2^-11 (one) as long as fp16 holds it as a normal number; the
    largest probability enters as 2^15, or, in tiles of many rows, as 2^11 to 2^15 times the block's V scale over
    the accumulator's unit (2^-6 to 1); fp16's last place is never below 2^-24, so the rounding of a far smaller
    one is at most 2^-25 / 2^11 = 2^-36 of the largest (floor, in units of up to 2^6 |v|).  An error e of every probability moves the output
    by at most 2 e sum p |v|; the sums over the keys are fp32.  bf16 results are rounded by 2^-8 at most."""
    score = reach * ((dim + 8) * 2.0 ** -24 + 2.0 ** -21)
    p = score + (2.0 ** -20 if dtype == "f32" else 2.0 ** -11)
    return 2 * p[..., None] * slack + 2.0 ** -30 * floor + (2.0 ** -22 if dtype == "f32" else 2.0 ** -8) * np.abs(out) + 1e-30
