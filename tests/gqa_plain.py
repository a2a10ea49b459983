"""Grouped-query attention in 64 bits, row by row, and the 8-bit cache's rule: what the GPU tests of the 8-bit cache and of drafted trees compare with."""
import numpy as np

from oracle import binding as orc

D = 128


def bf16(x):
    """float32 -> the nearest bf16, as float32."""
    return orc.f32_from_bf16(orc.bf16_from_f32(np.ascontiguousarray(x, np.float32)))


def quantise(x):
    """float32 [..., 128] -> (codes int8, scale float32) by the cache's rule, every operation in float32."""
    x = np.asarray(x, np.float32)
    a = np.abs(x).max(-1)
    with np.errstate(all="ignore"):
        some = np.isfinite(a) & (a >= np.float32(1e-36))
        inv = np.where(some, np.float32(127) / np.where(some, a, 1), 0).astype(np.float32)
        codes = np.rint(np.where(some[..., None], x, 0).astype(np.float32) * inv[..., None]).astype(np.int8)
        scale = np.where(some, a / np.float32(127), np.where(np.isfinite(a), 0, np.nan)).astype(np.float32)
    return codes, scale


def held(x, int8):
    """What a cache holds of float32 rows, as float32."""
    if not int8:
        return bf16(x)
    c, s = quantise(x)
    return (c.astype(np.float32) * s[..., None]).astype(np.float32)


def ancestors(parents, nodes, S):
    """[S][S]: does node i see node j?"""
    see = np.zeros((S, S), bool)
    for i in range(nodes):
        j = i
        while j >= 0:
            see[i, j] = True
            j = parents[j]
    return see


def causal(S):
    return np.tril(np.ones((S, S), bool))


def attend(K, V, q, n, see, scale, q_rounding=0.0):
    """K, V [n + m, Hkv, D] as held, q [S, H, D], see [S][m]: query i sees the first n rows and, of the others, see[i].  Returns (out, bound) [S, H, D] in
    64 bits.  bound: how far the kernels may be off, per element.  They round P (or P times a row's scale) to bf16, 2^-8 of it; scores are sums of
    128 products of exact operands in float32, 2^-16 of the sum of magnitudes is eight times what their roundings add up to, and q_rounding of that sum where
    queries are rounded; an error d of a score is exp(d) of its P, above and below the line.  The rest (sums of P, exponentials, merges) is 2^-14.
    Over the 8-bit cache P, or the values, are binary16, whose steps do not shrink below 2^-24: P reaches 2^7 and more there, so each is off by up to 2^-25 of
    2^7 of a row's largest even where that is more than 2^-8 of it (seen where the likeliest row's code is 0 in a dim), and values come to 2^7 of the largest
    scale's, so theirs is 2^-25 / 2^7 of that scale, less than 2^-32 of the largest value."""
    S, H, _ = q.shape
    Hkv = K.shape[1]
    g = H // Hkv
    K, V, q = K.astype(np.float64), V.astype(np.float64), q.astype(np.float64)
    out, bound = np.zeros((S, H, D)), np.zeros((S, H, D))
    for i in range(S):
        rows = np.concatenate([np.arange(n), n + np.nonzero(see[i])[0]])
        if rows.size == 0:
            continue
        for h in range(Hkv):
            k, v, x = K[rows, h], V[rows, h], q[i, h * g:(h + 1) * g]
            s = x @ k.T * scale
            err = np.max(np.abs(x) @ np.abs(k).T, -1, keepdims=True) * scale * (2.0 ** -16 + q_rounding)
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            out[i, h * g:(h + 1) * g] = p @ v
            bound[i, h * g:(h + 1) * g] = (p @ np.abs(v)) * (2.0 ** -8 + 2 * np.expm1(err) + 2.0 ** -14) + 2.0 ** -32 * (np.abs(v).sum(0) + np.abs(v).max())
    return out, bound


def check(got, want, bound, what="", bf16_out=False):
    got = np.asarray(got, np.float64)
    assert np.isfinite(got).all(), "%s: not finite" % what
    room = bound + (np.abs(want) + bound) * 2.0 ** -8 * bf16_out + 1e-30
    worst = np.max(np.abs(got - want) / room)
    assert worst <= 1, "%s: %.2f times the bound" % (what, worst)


class Cache:
    """Rows of a batch of sequences beside a pool that is given the same: rows(b) are float32 [tokens, Hkv, D] as held."""

    def __init__(self, B, Hkv, int8):
        self.int8, self.k, self.v = int8, [np.zeros((0, Hkv, D), np.float32) for _ in range(B)], [np.zeros((0, Hkv, D), np.float32) for _ in range(B)]

    def append(self, b, k, v):
        self.k[b] = np.concatenate([self.k[b], held(k, self.int8)])
        self.v[b] = np.concatenate([self.v[b], held(v, self.int8)])


def rows(rng, n, Hkv, kind="k"):
    """Random rows: heads and tokens of different size, keys with a few large dims."""
    x = rng.standard_normal((n, Hkv, D)).astype(np.float32) * np.exp2(rng.standard_normal((n, Hkv, 1))).astype(np.float32)
    if kind == "k":
        x[..., 5::32] *= 3
    return x


def random_tree(rng, S, roots=3):
    return np.asarray([-1 if j < min(roots, S) else int(rng.integers(0, j)) for j in range(S)], np.int32)
