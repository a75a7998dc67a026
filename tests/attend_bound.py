"""Attention in 64 bits with a bound of what a kernel of f32 accuracy may be off,
term by term (q8_util.attend's is a single wide one): a kernel that drops bits of
its queries or of its softmax weights does not stay within it.

Per score (in nats; size = sum |q k|, big = max |q k|, both times the scale):
  * the queries' representation, q_bits: 2^-q_bits size
  * its matrix products: nine accumulations of 16 products (eight, and all those
    of the smaller terms as one), each a sum of 17 terms cut at 2^-24 of its
    largest term and rounded to f32: 9 (17 2^-24 big + 2^-24 size)
  * five roundings of factors that multiply it: 5 2^-24 |score|
  * its exponent x = score log2 e + log2 s_v, and x - M, rounded: ln 2 2^-24 each
    of |x| and |x - M| <= |x| + max |x|
Per weight: the exponential 2^-22, up to eight factors 2^-22 where references move
and partials meet, and the weights' representation, 2^-w_bits.
Per output: accumulations of 16 weighted rows, in three terms, by a chain of up to
a fourth of the keys (steps = 3 of them for 64 keys; the tree kernel's two groups
take half of the keys each: 6) and 32 more for merges, 2^-23 of sum p |v| each; the
sum of weights, n / 16 + 40 additions of 2^-24."""
import numpy as np

D = 128


def attend(q, k, v, keep=None, s_v=None, scale=1 / np.sqrt(D), q_bits=22, w_bits=23,
           steps=3):
    """Rows q [R][128] over keys [n][128]; keep [R][n] masks, s_v [n] the power-of-two
    scales of the V rows.  Returns the output and its bound, [R][128]."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n = k.shape[0]
    x = q @ k.T * scale
    size = np.abs(q) @ np.abs(k).T * scale
    big = np.zeros_like(x)
    for r in range(q.shape[0]):
        big[r] = np.abs(q[r] * k).max(-1, initial=0) * scale
    keep = np.ones(x.shape, bool) if keep is None else keep
    m = np.where(keep, x, -np.inf).max(-1, keepdims=True, initial=-np.inf)
    e = np.where(keep, np.exp(np.where(keep, x - np.where(np.isfinite(m), m, 0), 0)), 0)
    tot = e.sum(-1, keepdims=True)
    p = e / np.where(tot > 0, tot, 1)
    x2 = np.abs(x) / np.log(2) + (0 if s_v is None else np.abs(np.log2(s_v)))
    x2 = np.where(keep, x2, 0)
    ds = (2.0 ** -q_bits * size + 9 * 2.0 ** -24 * (17 * big + size) + 5 * 2.0 ** -24 * np.abs(x) +
          np.log(2) * 2.0 ** -24 * (2 * x2 + x2.max(-1, keepdims=True, initial=0)))
    rel = np.where(keep, np.expm1(np.where(keep, ds, 0)) + 9 * 2.0 ** -22 + 2.0 ** -w_bits, 0)
    out, each = p @ v, p @ np.abs(v)
    tol = ((p * rel) @ np.abs(v) + np.abs(out) * ((p * rel).sum(-1, keepdims=True) +
                                                  (n / 16 + 40) * 2.0 ** -24) +
           (steps * np.ceil(n / 64) + 32) * 2.0 ** -23 * each)
    return out, tol
