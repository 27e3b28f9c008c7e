"""Attention over the paged cache in 64 bits where a row sees its window and the first
tokens: what the GPU tests compare with, and the bound of an f32 evaluation."""
import numpy as np


def attend(cache, q, lens, new, scale, softcap=0.0, window=0, sinks=0, pos_of=None):
    """q [rows, q heads, dim] -> (out, bound), both [rows, q heads, dim]; cache: a
    kv_reference.Cache. A row at position pos sees j <= pos with j > pos - window (window
    0: any) or j < sinks.

    The bound is that of kv_reference.Cache.attend, from the same steps: scores of dim
    products of a q held in 22 bits and an exact k ((dim + 8) 2^-24 of their size, with a
    softcap's tanh 2^-20 of the cap more), exponents rounded in f32 among numbers as
    large as the distance to the maximum and V's scales' logarithms, weights of 22 bits;
    each e_j moves the mean by p_j e_j (|v_j| + |out|); sums in chains of at most
    32 + n/32 numbers and a join of at most 64. A weight is p_j times its page's scale, as
    two f16 numbers with the largest at 2^14 to 2^15: the second one's steps end at 2^-24,
    half of which is 2^-39 of 2^14 and so at most 2^-38 of the largest. Below 2^-17 of the
    largest that is more than 2^-22 of the weight: every weight may be off by 2^-38 of the
    largest, each times its token's 8-bit value."""
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    group, eps, t = q.shape[1] // cache.heads, 2.0 ** -24, 0
    for b, (n, m) in enumerate(zip(lens, new)):
        pos = n - m + np.arange(m)
        j = np.arange(n)
        for h in range(cache.heads if m else 0):
            k, v, there = cache.read(b, h, n)
            see = there & (j <= pos[:, None])
            if window:
                see &= (j > pos[:, None] - window) | (j < sinks)
            some = see.any(1)
            vs = np.zeros(n)  # the scale of each token's page, and its 8-bit values
            for j0 in range(0, n, cache.page):
                slot = j0 // cache.page
                pid = cache.table[b, slot] if slot < cache.table.shape[1] else -1
                if 0 <= pid < len(cache.k):
                    vs[j0:j0 + cache.page] = cache.vs[pid, h]
            units = np.abs(v) / np.where(vs > 0, vs, 1.0)[:, None]
            for g in range(group):
                x = q[t:t + m, h * group + g].astype(np.float64)
                s = scale * (x @ k.T)
                ds = (cache.dim + 8) * eps * scale * (np.abs(x) @ np.abs(k).T)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                    ds = ds + 16 * eps * softcap
                s, ds = np.where(see, s, -np.inf), np.where(see, ds, 0.0)
                top = np.where(some, s.max(1, initial=-np.inf), 0.0)[:, None]
                p = np.exp(s - top)
                p /= np.where(some, p.sum(1), 1.0)[:, None]
                o = p @ v
                size = np.where(see, s, 0.0)
                e = ds + ds.max(1, initial=0.0)[:, None] + 8 * eps \
                    + 2 * eps * (np.abs(size) + 2 * np.where(see, top - size, 0.0) + 34)
                e += (96 + n / 32) * eps
                w = p * vs
                least = 2.0 ** -38 * w.max(1, initial=0.0)[:, None] * (see.astype(np.float64) @ units)
                out[t:t + m, h * group + g] = o
                tol[t:t + m, h * group + g] = ((p * e) @ np.abs(v) + (p * e).sum(1)[:, None] * np.abs(o)
                                               + eps * np.abs(o) + least)
        t += m
    return out, tol
