"""Rotary positions and the paged 8-bit cache in 64 bits, one token and one page
at a time, from their definitions: what the GPU tests compare with."""
import numpy as np

MOST = {"i8": 127.0, "e4m3": 448.0}


def grid(fmt):
    """The value of every byte (NaN: no number)."""
    b = np.arange(256)
    if fmt == "i8":
        return b.astype(np.uint8).view(np.int8).astype(np.float64)
    e, f = (b >> 3) & 15, b & 7
    x = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    x[(b & 127) == 127] = np.nan
    return np.where(b >= 128, -x, x)


def code(x, fmt):
    """Bytes of values in units of their scale: nearest, ties to even,
    saturating, NaN as 0."""
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=MOST[fmt], neginf=-MOST[fmt])
    x = np.clip(x, -MOST[fmt], MOST[fmt])
    if fmt == "i8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    g = grid(fmt)[:127]
    a = np.abs(x)
    hi = np.minimum(np.searchsorted(g, a), 126)
    lo = np.maximum(hi - 1, 0)
    up, down = g[hi] - a, a - g[lo]
    n = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (n | np.where(x < 0, 128, 0)).astype(np.uint8)


def rotate(x, cs, half):
    """x [..., dim] by one table row cs [rot/2, 2]."""
    x = np.asarray(x, np.float64)
    c, s = cs[:, 0].astype(np.float64), cs[:, 1].astype(np.float64)
    rot, y = 2 * len(cs), x.copy()
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


class Cache:
    """k [pages, heads, tokens, dim], v [pages, heads, dim, tokens] bytes."""

    def __init__(self, k, v, ks, vs, table, fmt):
        self.k, self.v, self.ks, self.vs, self.table, self.fmt = k, v, ks, vs, table, fmt
        self.page, self.heads, self.dim = k.shape[2], k.shape[1], k.shape[3]

    def _block(self, which, pid, h):
        return self.k[pid, h] if which == "k" else self.v[pid, h].T  # [tokens, dim] view

    def append(self, b, start, k, v):
        """k, v [new, heads, dim] in 64 bits at positions start .. of sequence b."""
        j, n = start, start + len(k)
        while j < n:
            slot, off = divmod(j, self.page)
            m = min(self.page - off, n - j)
            pid = self.table[b, slot] if slot < self.table.shape[1] else -1
            if 0 <= pid < len(self.k):
                for which, x, scale in (("k", k, self.ks), ("v", v, self.vs)):
                    for h in range(self.heads):
                        y = x[j - start: j - start + m, h]
                        old = scale[pid, h] if off else np.float32(0)
                        top = np.abs(y[np.isfinite(y)]).max(initial=0.0)
                        now = np.fmax(old, np.float32(top / MOST[self.fmt]))  # a NaN scale counts as none
                        blk = self._block(which, pid, h)
                        if off and now > old:
                            held = grid(self.fmt)[blk[:off]]
                            blk[:off] = code(held * np.float64(old) / np.float64(now), self.fmt)
                        blk[off: off + m] = code(y / np.float64(now), self.fmt) if now > 0 else 0
                        scale[pid, h] = now
            j += m

    def read(self, b, h, n):
        """(k, v, present) of the first n positions, [n, dim] in 64 bits."""
        k, v, there = np.zeros((n, self.dim)), np.zeros((n, self.dim)), np.zeros(n, bool)
        for slot in range(-(-n // self.page)):
            pid = self.table[b, slot] if slot < self.table.shape[1] else -1
            if not 0 <= pid < len(self.k):
                continue
            a, z = slot * self.page, min(n, (slot + 1) * self.page)
            k[a:z] = grid(self.fmt)[self._block("k", pid, h)[: z - a]] * np.float64(self.ks[pid, h])
            v[a:z] = grid(self.fmt)[self._block("v", pid, h)[: z - a]] * np.float64(self.vs[pid, h])
            there[a:z] = True
        return k, v, there

    def attend(self, q, lens, new, scale, softcap=0.0, window=0):
        """q [rows, q heads, dim] -> (out, bound of an f32 evaluation), both
        [rows, q heads, dim].

        The bound: the score is a sum of dim products of a q held in 22 bits
        (relative 2^-22) and an exact k, added in f32 (dim additions at most):
        |ds| <= (dim + 8) 2^-24 scale sum|q||k|; a softcap's tanh adds 2^-20 of
        the cap. In the exponent it meets roundings of numbers as large as the
        distance to the maximum and the logarithms of V's scales (32 at most):
        2^-23 (|s| + |max - s| + 32). w is held in 22 bits and the base-2
        exponential is good to 2^-22. Each p_j is off by e_j relative, which
        moves the mean by sum p_j e_j (|v_j| + |out|); the sums of products are
        added in chains of at most 32 + n/32 numbers and a join of at most 64.
        """
        out = np.zeros(q.shape)
        tol = np.zeros(q.shape)
        group, eps, t = q.shape[1] // self.heads, 2.0 ** -24, 0
        for b, (n, m) in enumerate(zip(lens, new)):
            for h in range(self.heads):
                k, v, there = self.read(b, h, n)
                for i in range(m):
                    pos = n - m + i
                    j = np.arange(n)
                    see = there & (j <= pos)
                    if window:
                        see &= j > pos - window
                    if not see.any():
                        continue
                    for g in range(group):
                        x = q[t + i, h * group + g].astype(np.float64)
                        s = scale * (k[see] @ x)
                        ds = (self.dim + 8) * eps * scale * (np.abs(k[see]) @ np.abs(x))
                        if softcap:
                            s = softcap * np.tanh(s / softcap)
                            ds = ds + 16 * eps * softcap
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        o = p @ v[see]
                        e = ds + ds.max() + 2 * eps * (np.abs(s) + 2 * (s.max() - s) + 34) + 8 * eps
                        out[t + i, h * group + g] = o
                        chain = (96 + n / 32) * eps
                        tol[t + i, h * group + g] = ((p * (e + chain)) @ np.abs(v[see])
                                                     + (p @ (e + chain)) * np.abs(o) + eps * np.abs(o))
            t += m
        return out, tol
