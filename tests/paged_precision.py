"""Data on which the lo parts of the paged attention's f16 hi + lo pairs show, with bounds for the f32 outputs.

Scores: one visible slot, so lse is the score.  q = 2^j (1 + 2^-11), which f16 rounds to 2^j everywhere; keys 1 and 1/2,
which both caches hold exactly.  Every product and partial sum is a multiple of 2^-14 below 2^9, so f32 holds the sum
exactly in any order; what remains is the factor scale * log2(e) (three roundings with the product), the reference score
less 2^3, the sum with log2(2^8) (an ulp, 2^-20) and the factor log(2): 2^-20 (1 + |s|).  Without the lo parts s is off
by 2^-11 s, of one 32-dim block by 2^-14 s or more.  The same holds beside elements of q of 2^14 where the key is zero:
they add nothing, unless codes enter uncentred, as 8 d 2^14 that is taken off again.

Weights: scores that are exact multiples of 2^-10 below 4, 1 to 16 slots (one piece).  ex2 of a difference below 8 (2^-21
with its argument's roundings), p as hi + lo (2^-22), its product with a scale (2^-20), 17 addends cut at 2^-23 in each of
two MMAs (2^-18), sum and quotient (2^-21): 2^-17 of the largest value together.  Without a lo part a weight is off by
up to 2^-12 of itself."""
import numpy as np

F32, F64 = np.float32, np.float64


def score_case(HD, n_rows, QH, large=0.0):
    """q [n_rows][QH][HD], keys and values [1][2][1][HD] of the one slot; large: every 16th element of q, where the key is 0."""
    j = (np.arange(n_rows)[:, None, None] + np.arange(QH)[None, :, None] + np.arange(HD)) % 3
    q = (2.0 ** -j * (1 + 2.0 ** -11)).astype(F32)
    x = np.ones((1, 2, 1, HD))
    x[0, 0, 0, 1::2] = 0.5
    if large:
        q[..., 5::16], x[0, 0, 0, 5::16] = large, 0.0
    return q, x


def score_bound(s):
    return 2.0 ** -20 * (1 + np.abs(s))


def weight_case(rng, HD, n_rows, QH, slots):
    """q [n_rows][QH][HD]; keys and values [slots][2][1][HD]: keys of multiples of 1/2 that both caches hold exactly
    (each block's first one is 4, so that a code is a multiple of 1/2)."""
    q = rng.integers(-8, 9, (n_rows, QH, HD)) * 2.0 ** -9
    q[..., ::32] = 0.0                                   # (the fours do not enter the scores)
    x = rng.standard_normal((slots, 2, 1, HD))
    x[:, 0] = rng.integers(-7, 8, (slots, 1, HD)) * 0.5
    x[:, 0, :, ::32] = 4.0
    return q.astype(F32), x


def weight_bound(v):
    return 2.0 ** -17 * np.abs(v).max()


def hi(x):
    """The f16 hi parts of x, relative to a power of two that brings the largest to [2^14, 2^15)."""
    f = 2.0 ** (14 - np.floor(np.log2(np.abs(x).max(-1, keepdims=True))))
    return (x * f).astype(np.float16).astype(F64) / f
