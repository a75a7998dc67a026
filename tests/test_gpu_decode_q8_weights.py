"""The 8-bit decode where the keys that make the output carry weights far below the
largest one: V rows of zeros (stored under scale 1), attention sinks, rows with one
large dim, payloads among e4m3's subnormals; and ordinary batches, all within the
term-by-term bound of attend_bound."""
import numpy as np
import pytest

import attend_bound as A
import q8_util as Q
import test_gpu_kv_q8 as T

pytestmark = pytest.mark.gpu


def case(seed, Hq, Hkv, lens, v_size=1.0, bs=256):
    """decode_case with V rows of v_size, and K and V rows at hand for changes."""
    c = T.decode_case(seed, Hq, Hkv, lens, bs)
    rng = np.random.default_rng(seed + 1)
    c["k"] = [rng.standard_normal((n, Hkv, 128)).astype(np.float32) for n in lens]
    c["v"] = [(rng.standard_normal((n, Hkv, 128)) * v_size).astype(np.float32) for n in lens]
    return c


def store(c):
    for s, n in enumerate(c["lens"]):
        if n:
            c["cache"].put(c["layer"], Q.slots_of(c["bt"][s], n, c["bs"]), c["k"][s], c["v"][s])
    return c


def sink(c, s, at, nats):
    """Key `at` of sequence s scores `nats` above the others' usual scores, for
    every query head: the query rows of a kv head share a part along it."""
    Hq, Hkv = c["Hq"], c["Hkv"]
    G = Hq // Hkv
    rng = np.random.default_rng(at + 7)
    for hd in range(Hkv):
        d = rng.standard_normal(128)
        d /= np.sqrt((d * d).sum())
        c["q"][s, hd * G:(hd + 1) * G] += (4 * d).astype(np.float32)
        c["k"][s][at, hd] = (d * (nats * np.sqrt(128) / 4)).astype(np.float32)


def expect(c, q):
    G = c["Hq"] // c["Hkv"]
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, n in enumerate(c["lens"]):
        if n == 0:
            continue
        sl = Q.slots_of(c["bt"][s], n, c["bs"])
        k, v = c["cache"].rows(c["layer"], sl)
        sv = c["cache"].vs[c["layer"], sl // c["bs"], :, sl % c["bs"]].astype(np.float64)
        for hd in range(c["Hkv"]):
            r = slice(hd * G, (hd + 1) * G)
            want[s, r], tol[s, r] = A.attend(q[s, r], k[:, hd], v[:, hd], s_v=sv[:, hd])
    return want, tol


def wide(c):
    """A bound of the contexts that makes the launch take three CTAs per SM."""
    cols = 320 * 1024 // c["Hkv"] // c["bs"]
    c["bt"] = np.concatenate([c["bt"], np.full((len(c["lens"]), cols - c["bt"].shape[1]), -1,
                                               np.int32)], 1)
    return cols * c["bs"]


def verify(c, bf16=False, bound=None):
    h = T.make_handle(c, **({"max_context": bound} if bound else {}))
    h, got, q = T.run_decode(c, bf16, h, bound=bound)
    h.check_device()
    want, tol = expect(c, q)
    Q.check(got, want, tol, bf16)


@pytest.mark.parametrize("v_size", [1.0, 1e-2, 1e-4, 1e-8])
@pytest.mark.parametrize("lens", [[500], [9000, 60], [300] * 70])
@pytest.mark.parametrize("three", [False, True])
def test_zero_v_row_on_the_best_key(cuda, v_size, lens, three):
    """[300] * 70: whole units in one CTA; one long sequence: units shared by CTAs."""
    c = case(int(1 / v_size) % 1000, 16, 8, lens, v_size)
    for s in range(len(lens)):
        x = c["q"][s].reshape(8, 2, 128).sum(1)  # the kv head's queries
        best = np.einsum("hd,thd->th", x, c["k"][s]).argmax(0)
        c["v"][s][best, np.arange(8)] = 0
    store(c)
    verify(c, bound=wide(c) if three else None)


@pytest.mark.parametrize("nats", [8, 12, 17, 30])
@pytest.mark.parametrize("v_row", ["zero", "one dim", "one large dim", "small"])
@pytest.mark.parametrize("n,Hq,three", [(9100, 16, False), (9100, 64, True), (400, 8, False)])
def test_attention_sink(cuda, nats, v_row, n, Hq, three):
    c = case(nats + n, Hq, 8, [n, 33], 0.05)
    for at in (0, n // 2):
        sink(c, 0, at, nats)
        c["v"][0][at] = 0
        if v_row == "one dim":
            c["v"][0][at, :, 17] = 0.3
        elif v_row == "one large dim":
            c["v"][0][at, :, 17] = 3e4
        elif v_row == "small":
            c["v"][0][at] = 1e-6
    store(c)
    verify(c, bound=wide(c) if three else None)


def test_nothing_but_zero_rows(cuda):
    c = case(3, 16, 8, [1, 129, 5000])
    for v in c["v"]:
        v[:] = 0
    store(c)
    h, got, _ = T.run_decode(c)
    h.check_device()
    assert (got == 0).all()


def test_payloads_among_the_subnormals(cuda):
    """Rows of one large dim: the others' payloads are e4m3's smallest, down to its
    least value, on keys where the large dim cancels in pairs."""
    c = case(4, 16, 8, [64, 700], 1.0)
    for v in c["v"]:
        v *= np.float32(2.0 ** -8)
        v[:, :, 5] = 440 * np.where(np.arange(v.shape[0]) % 2, 1, -1)[:, None]
    store(c)
    p = c["cache"].vp[0, c["bt"][0, 0], :, :64] & 0x7f
    assert (p < 8).mean() > 0.9 and (p == 1).any()
    verify(c)


@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (16, 8), (32, 8), (64, 8), (8, 1)])
@pytest.mark.parametrize("bf16", [False, True])
def test_ordinary_batches_in_the_tight_bound(cuda, Hq, Hkv, bf16):
    c = store(case(Hq + 3 * Hkv, Hq, Hkv, T.EDGES))
    verify(c, bf16)
