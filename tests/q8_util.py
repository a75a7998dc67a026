"""Plain statements of the 8-bit cache for the tests: the format in numpy, and
attention over it in 64 bits, with the error that f32 arithmetic may add."""
import numpy as np

import cases
import oracle as O

D = 128


def e4m3_round(y):
    """f32 -> e4m3 bytes, by torch's conversion (round to nearest even)."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(y, np.float32)).to(torch.float8_e4m3fn).view(
        torch.uint8).numpy()


def e4m3_value(b):
    """The 256 values of e4m3 (1 sign, 4 exponent, 3 mantissa bits; 0x7f NaN)."""
    i = np.arange(256)
    e, m = (i >> 3) & 15, i & 7
    v = np.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v = np.where((i & 127) == 127, np.nan, v) * np.where(i & 128, -1, 1)
    return v[b]


def quantise(x):
    """Rows [..., 128] f32 -> (bytes, scales): the smallest power of two s with
    max|x| <= 448 s, found by comparison."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    a = np.abs(np.where(bad[..., None], 0, x)).max(-1).astype(np.float64)
    e = np.full(a.shape, -100)
    for k in range(-100, 121):
        e = np.where(a > 448 * 2.0 ** k, k + 1, e)
    scale = np.where(a == 0, 1.0, 2.0 ** e)
    y = np.where(bad[..., None], 0, x.astype(np.float64)) / scale[..., None]
    return e4m3_round(y), np.where(bad, np.nan, scale).astype(np.float32)


class Q8Cache:
    """payload [n_layer][num_blocks][Hkv][bs][128], scale [...][bs]."""

    def __init__(self, num_blocks, Hkv, n_layer=1, bs=256, fill=0x7f):
        self.bs, self.Hkv = bs, Hkv
        shape = (n_layer, num_blocks, Hkv, bs)
        self.kp = np.full(shape + (D,), fill, np.uint8)
        self.vp = self.kp.copy()
        self.ks = np.full(shape, np.nan, np.float32)
        self.vs = self.ks.copy()

    def put(self, layer, slots, k, v):
        for p, s, x in ((self.kp, self.ks, k), (self.vp, self.vs, v)):
            b, sc = quantise(x)
            p[layer, slots // self.bs, :, slots % self.bs] = b
            s[layer, slots // self.bs, :, slots % self.bs] = sc

    def rows(self, layer, slots):
        out = []
        for p, s in ((self.kp, self.ks), (self.vp, self.vs)):
            b = p[layer, slots // self.bs, :, slots % self.bs]
            sc = s[layer, slots // self.bs, :, slots % self.bs]
            out.append(e4m3_value(b) * sc[..., None].astype(np.float64))
        return out

    def dev(self):
        from gpu_util import dev
        return [dev(a) for a in (self.kp, self.ks, self.vp, self.vs)]


def tables(rng, lens, bs, num_blocks):
    need = [-(-int(n) // bs) for n in lens]
    assert sum(need) <= num_blocks
    perm = rng.permutation(num_blocks).astype(np.int32)
    bt = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    o = 0
    for s, n in enumerate(need):
        bt[s, :n] = perm[o:o + n]
        o += n
    return bt


def slots_of(bt_row, n, bs):
    t = np.arange(n)
    return bt_row[t // bs].astype(np.int64) * bs + t % bs


def attend(q, k, v, keep=None, scale=1 / np.sqrt(D), weight_bits=20):
    """Rows q [R][128] over keys [n][128] in 64 bits; keep [R][n] masks.  Also
    the bound on what f32 arithmetic may be off: |dS| of each score is within
    2^-16 of sum|q k| (a 128-term dot product, terms exact or of 22 bits), a
    change of dS moves the output by at most (e^(2 dS) - 1) sum p|v|, the
    exponential and the weights' bits (22 in the 8-bit decode) add 2^-weight_bits,
    and chains of n/16 + 64 f32 additions 2^-23 each."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    x = q @ k.T * scale
    size = np.abs(q) @ np.abs(k).T * scale
    if keep is not None:
        x = np.where(keep, x, -np.inf)
        size = np.where(keep, size, 0)
    m = x.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(x - np.where(np.isfinite(m), m, 0))
    tot = e.sum(-1, keepdims=True)
    p = e / np.where(tot > 0, tot, 1)
    ds = size.max(-1, keepdims=True, initial=0) * 2.0 ** -16
    rel = np.expm1(2 * ds) + 2.0 ** -weight_bits + (k.shape[0] / 16 + 64) * 2.0 ** -23
    return p @ v, rel * (p @ np.abs(v))


def check(got, want, tol, bf16):
    """|got - want| <= tol, plus half a step of bf16 where that is the type."""
    t = tol * (1.01 if bf16 else 1) + (np.abs(want) * 2.0 ** -8 if bf16 else 0) + 1e-30
    bad = ~(np.abs(got - want) <= t)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], t[bad][:5])
