"""The tree decode within attend_bound's term-by-term bound: "f32 keeps f32 accuracy
throughout" (24 bits of queries and weights), bf16 with 16 bits of weights."""
import numpy as np
import pytest

import attend_bound as A
import oracle as O
import q8_util as Q
import test_gpu_tree_decode as T

pytestmark = pytest.mark.gpu


def expect(c, q, bf16):
    G = c["Hq"] // c["Hkv"]
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, (n, N) in enumerate(zip(c["lens"], c["nodes"])):
        if not N:
            continue
        sl = Q.slots_of(c["bt"][s], n, c["bs"])
        k, v = (O.bf16_to_f32(c[x][c["layer"], sl]) for x in "kv")
        keep = np.ones((N, n), bool)
        keep[:, n - N:] = c["masks"][s][:, :N]
        rows = slice(c["cu"][s], c["cu"][s + 1])
        for hd in range(c["Hkv"]):
            hs = slice(hd * G, (hd + 1) * G)
            w, t = A.attend(q[rows, hs].reshape(N * G, 128), k[:, hd], v[:, hd],
                            np.repeat(keep, G, 0), q_bits=60 if bf16 else 24,
                            w_bits=16 if bf16 else 23, steps=4 if bf16 else 6)
            want[rows, hs], tol[rows, hs] = w.reshape(N, G, 128), t.reshape(N, G, 128)
    return want, tol


def verify(c, bf16):
    h, got, q = T.run(c, bf16)
    h.check_device()
    Q.check(got, *expect(c, q, bf16), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (32, 8), (64, 8), (8, 1)])
def test_ragged_trees(cuda, bf16, Hq, Hkv):
    verify(T.tree_case(2 * Hq + Hkv, Hq, Hkv, [63, 64, 65, 300, 1, 127, 200, 10, 1000],
                       [8, 64, 2, 17, 1, 63, 0, 10, 33], n_layer=2), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("words,nodes", [(2, [128, 70]), (4, [256, 1])])
def test_wide_trees(cuda, bf16, words, nodes):
    verify(T.tree_case(words, 16, 4, [900, 300], nodes, words=words), bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_sinks_and_rows_of_one_dim(cuda, bf16):
    """A first key far above the others whose V row is zero, or zero in all dims but
    one: the others' weights make the output."""
    c = T.tree_case(5, 16, 8, [2000, 400], [8, 5])
    rng = np.random.default_rng(6)
    for s, nats in ((0, 17), (1, 9)):
        slot = Q.slots_of(c["bt"][s], 1, c["bs"])[0]
        rows = slice(c["cu"][s], c["cu"][s + 1])
        for hd in range(8):
            d = rng.standard_normal(128)
            d /= np.sqrt((d * d).sum())
            c["q"][rows, 2 * hd:2 * hd + 2] += (4 * d).astype(np.float32)
            c["k"][0, slot, hd] = O.f32_to_bf16((d * (nats * np.sqrt(128) / 4)).astype(np.float32))
            c["v"][0, slot, hd] = 0
        c["v"][0, slot, 4:, 17] = O.f32_to_bf16(np.array([3e4], np.float32))[0]
    verify(c, bf16)


def third_terms(rng, n, sign):
    """f32 values in [1, 2) whose first two bf16 terms leave a rest of about 2^-18 of
    them, of the given sign."""
    x = (1 + rng.random(200000)).astype(np.float32)
    a = O.bf16_to_f32(O.f32_to_bf16(x))
    b = O.bf16_to_f32(O.f32_to_bf16((x - a).astype(np.float32)))
    rest = (x.astype(np.float64) - a - b) / x
    x = x[sign * rest > 2.0 ** -18.7]
    assert len(x) >= n
    return x[:n]


def test_every_bit_of_f32_queries_counts(cuda):
    """Queries whose values cancel over the dims and whose lowest bits add up, keys
    of either sign, V rows +1 and -1: a kernel of 16-bit queries is off by more
    than the bound."""
    rng = np.random.default_rng(7)
    c = T.tree_case(8, 8, 8, [40], [2])
    c["q"][..., :64] = third_terms(rng, 64 * 16, 1).reshape(2, 8, 64)
    c["q"][..., 64:] = -third_terms(rng, 64 * 16, -1).reshape(2, 8, 64)
    sl = Q.slots_of(c["bt"][0], 40, c["bs"])
    sign = np.where(np.arange(40) % 2, 1, -1)
    c["k"][0, sl] = O.f32_to_bf16((sign[:, None, None] * np.ones((40, 8, 128))).astype(np.float32))
    c["v"][0, sl] = c["k"][0, sl]
    verify(c, False)
    # what two terms would give
    a = O.bf16_to_f32(O.f32_to_bf16(c["q"]))
    two = a + O.bf16_to_f32(O.f32_to_bf16((c["q"] - a).astype(np.float32)))
    want, tol = expect(c, c["q"], False)
    assert (np.abs(expect(c, two, False)[0] - want) > 1.2 * tol).all()
