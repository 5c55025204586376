"""Plain float64 forms of the 8-bit serving operators (numpy, one sequence and one block at a time)."""
import math

import numpy as np


def quantize_rows(y):
    """(q, scale) of the rows of y (float64): scale = float32(max|y| / 127), q = y / scale to nearest even."""
    q = np.zeros(y.shape, np.int8)
    scale = np.zeros(y.shape[0], np.float32)
    for r in range(y.shape[0]):
        if not np.all(np.isfinite(y[r])):
            scale[r] = np.nan
            continue
        top = np.abs(y[r]).max()
        if top < 2.0 ** -100:
            continue
        scale[r] = np.float32(top / 127)
        q[r] = np.clip(np.rint(y[r] / np.float64(scale[r])), -127, 127)
    return q, scale


def rmsnorm(x, gamma, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(axis=1, keepdims=True) + np.float64(np.float32(eps))) * gamma.astype(np.float64)


def rotate(x, cos, sin):
    """x [heads, dim], cos and sin [dim], float64."""
    half = x.shape[-1] // 2
    turned = np.concatenate([-x[..., half:], x[..., :half]], axis=-1)
    return x * cos + turned * sin


def exponent_for(top):
    if top == 0:
        return -126
    f, x = math.frexp(top)
    return max(-126, min(127, x - 7 if f <= 127 / 128 else x - 6))


def append_block(held, scale, slot, x):
    """held int8 [size, dim] and scale of one block, x float64 [new, dim] from `slot` on: (held, scale)."""
    held = held.copy()
    new = x.shape[0]
    if not np.all(np.isfinite(x)) or (slot > 0 and np.isnan(scale)):
        held[slot:slot + new] = 0
        return held, np.float32(np.nan)
    e = exponent_for(np.abs(x).max())
    if slot > 0:
        before = math.frexp(float(scale))[1] - 1
        if e > before:
            held[:slot] = np.rint(held[:slot].astype(np.float64) * 2.0 ** (before - e))
        e = max(e, before)
    held[slot:slot + new] = np.clip(np.rint(np.ldexp(x, -e)), -127, 127)
    return held, np.float32(2.0 ** e)


class Cache:
    """k [pages, heads, size, dim], v [pages, heads, dim, size] int8; scales float32 [pages, heads]."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = (a.copy() for a in (k, v, k_scale, v_scale))
        self.size = k.shape[2]

    def append(self, table, position, k, v, cos=None, sin=None):
        """k, v float64 [new, heads, dim] of one sequence, the first at `position`."""
        if cos is not None and k.shape[0]:
            k = np.stack([rotate(k[i], cos[position + i], sin[position + i]) for i in range(k.shape[0])])
        at = 0
        while at < k.shape[0]:
            page, slot = table[(position + at) // self.size], (position + at) % self.size
            take = min(self.size - slot, k.shape[0] - at)
            for h in range(k.shape[1]):
                self.k[page, h], self.k_scale[page, h] = append_block(self.k[page, h], self.k_scale[page, h], slot,
                                                                      k[at:at + take, h])
                vt, self.v_scale[page, h] = append_block(self.v[page, h].T, self.v_scale[page, h], slot,
                                                         v[at:at + take, h])
                self.v[page, h] = vt.T
            at += take

    def tokens(self, table, length, head):
        """(k, v) float64 [length, dim] of one head of a sequence; a page outside the cache: None."""
        ks, vs = [], []
        for p in range(-(-length // self.size)):
            page = table[p]
            if page < 0 or page >= self.k.shape[0]:
                return None
            ks.append(self.k[page, head].astype(np.float64) * np.float64(self.k_scale[page, head]))
            vs.append(self.v[page, head].T.astype(np.float64) * np.float64(self.v_scale[page, head]))
        if not ks:
            return np.zeros((0, self.k.shape[3])), np.zeros((0, self.k.shape[3]))
        return np.concatenate(ks)[:length], np.concatenate(vs)[:length]


def attend(q, k, v, length, scale):
    """(out, bound) of one sequence and head: q [new, dim], k and v [length, dim], float64; query i sees the
    tokens up to length - new + i. bound[i]: sum_d |q_d| max_t |k_td| * scale, what a relative error of the
    products costs a score at most."""
    new, dim = q.shape
    out, bound = np.zeros((new, dim)), np.zeros(new)
    for i in range(new):
        sees = length - new + i + 1
        if sees <= 0:
            continue
        s = k[:sees] @ q[i] * scale
        bound[i] = (np.abs(k[:sees]) @ np.abs(q[i])).max() * scale
        if np.any(np.isnan(s)) or np.any(np.isnan(v[:sees])):
            out[i] = np.nan
            continue
        p = np.exp(s - s.max())
        out[i] = p @ v[:sees] / p.sum()
    return out, bound
