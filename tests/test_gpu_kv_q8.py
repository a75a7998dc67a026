"""The 8-bit paged cache on the GPU: the store against the oracle's rows put
into the format (bit for bit), the read-back (exact), and the decode over it
against 64-bit attention within the bound that q8_util.attend derives."""
import ctypes

import numpy as np
import pytest

import nvattn
import oracle as O
import q8_util as Q
from gpu_util import dev, handle

pytestmark = pytest.mark.gpu


def torch_():
    import torch
    return torch


def to_q(q, bf16):
    import torch
    t = torch.from_numpy(q).cuda()
    return t.bfloat16() if bf16 else t


# ------------------------------------------------------------------ store

def store_case(seed, T, Hq, Hkv, num_blocks, bs, n_layer=2, pad=0.1):
    rng = np.random.default_rng(seed)
    c = dict(
        q=rng.standard_normal((T, Hq, 128), dtype=np.float32) * 3,
        k=rng.standard_normal((T, Hkv, 128), dtype=np.float32),
        v=(rng.standard_normal((T, Hkv, 128)) *
           2.0 ** rng.integers(-30, 30, (T, Hkv, 1))).astype(np.float32),
        qw=O.f32_to_bf16((1 + 0.3 * rng.standard_normal(128)).astype(np.float32)),
        kw=O.f32_to_bf16((1 + 0.3 * rng.standard_normal(128)).astype(np.float32)),
        pos=rng.integers(0, 40960, T).astype(np.int32),
        slots=rng.permutation(num_blocks * bs)[:T].astype(np.int32))
    c["slots"][rng.random(T) < pad] = -1
    return c


def run_store(h, c, cache, layer, q_dtype=None, rows=False):
    torch = torch_()
    T, Hq, _ = c["q"].shape
    Hkv = c["k"].shape[1]
    d = cache.dev()
    q_out = torch.empty((T, Hq, 128), dtype=q_dtype or torch.float32, device="cuda")
    kr = vr = None
    if rows:
        kr = torch.empty((T, Hkv, 128), dtype=torch.float16, device="cuda")
        vr = torch.empty_like(kr)
    h.kv_store_q8(layer, *(dev(c[n]) for n in ("q", "k", "v", "qw", "kw", "pos", "slots")), q_out,
                  *d, k_rows=kr, v_rows=vr)
    torch.cuda.synchronize()
    return d, q_out, kr, vr


def oracle_rows(c, Hq, Hkv):
    """The normed, rotated rows in f32, bit for bit (the oracle's q path run on
    q, and on k with k's weights)."""
    p = O.params(n_q_heads=Hq, n_kv_heads=Hkv, n_slots=256)
    T = len(c["pos"])
    none = np.full(T, -1, np.int32)
    kc = np.zeros((1, 256, Hkv, 128), np.uint16)
    q = O.qk_norm_rope_store(p, 0, c["q"], c["k"], c["v"], c["qw"], c["kw"], c["pos"], none, kc,
                             kc.copy())
    pk = O.params(n_q_heads=Hkv, n_kv_heads=Hkv, n_slots=256)
    k = O.qk_norm_rope_store(pk, 0, c["k"], c["k"], c["v"], c["kw"], c["kw"], c["pos"], none, kc,
                             kc.copy())
    return q, k


@pytest.mark.parametrize("T,Hq,Hkv,bs,n_layer", [
    (1, 16, 8, 256, 2), (37, 8, 8, 128, 1), (300, 32, 8, 256, 2), (65, 8, 1, 512, 3),
    (2000, 64, 8, 256, 1), (9000, 8, 2, 256, 1)])
def test_store_is_the_oracles_rows_in_the_format(cuda, T, Hq, Hkv, bs, n_layer):
    torch = torch_()
    nb = -(-T // bs) + 1
    c = store_case(T, T, Hq, Hkv, nb, bs)
    cache = Q.Q8Cache(nb, Hkv, n_layer, bs, fill=0x55)
    layer = n_layer - 1
    h = handle(Hq, Hkv, nb, n_layer=n_layer, block_size=bs, max_seqs=1, max_context=bs)
    d, q_out, kr, vr = run_store(h, c, cache, layer, rows=True)
    h.check_device()
    q, k = oracle_rows(c, Hq, Hkv)
    assert np.array_equal(q_out.cpu().numpy().view(np.uint32), q.view(np.uint32))
    assert np.array_equal(kr.cpu().numpy(), k.astype(np.float16))
    with np.errstate(over="ignore"):
        assert np.array_equal(vr.cpu().numpy(), c["v"].astype(np.float16))
    on = c["slots"] >= 0
    cache.put(layer, c["slots"][on].astype(np.int64), k[on], c["v"][on])
    for got, want in zip(d, (cache.kp, cache.ks, cache.vp, cache.vs)):  # untouched slots too
        got = got.cpu().numpy()
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    # the other q types are the same rows, rounded
    for t in (torch.bfloat16, torch.float16):
        _, o, _, _ = run_store(h, c, cache, layer, q_dtype=t)
        assert torch.equal(o.cpu(), torch.from_numpy(q).to(t))


def test_store_rows_at_the_formats_edges(cuda):
    """V rows (stored as they come): zeros, the scale's switch at 448 * 2^k and
    the f32 value above it, subnormal and the largest f32 values, ties of the
    rounding, NaN and infinities."""
    T, Hq, Hkv = 16, 8, 1
    v = np.zeros((T, Hkv, 128), np.float32)
    v[1, 0, 5] = 448
    v[2, 0, 5] = np.nextafter(np.float32(448), np.float32(449))
    v[3, 0, :2] = [-7, 2.0 ** -9]            # 7 = 448 * 2^-6
    v[4, 0, 0] = np.nextafter(np.float32(7), np.float32(8))
    v[5, 0, 0] = 1e-45
    v[6, 0, :3] = [3e-38, -1e-39, 1e-36]
    v[7, 0, 0] = np.finfo(np.float32).max
    v[8, 0, :6] = [448, 17, 19, 21, -27, 2.0 ** -10]  # halfway between e4m3 neighbours
    v[9, 0, 3] = np.nan
    v[10, 0, 100] = np.inf
    v[11, 0, 127] = -np.inf
    v[12] = np.linspace(-448, 448, 128)
    v[13] = np.linspace(-1, 1, 128) * 2.0 ** -91
    v[14] = np.linspace(-1, 1, 128) * 2.0 ** 100
    v[15, 0, 1] = 2.0 ** -92 * 1.75
    c = store_case(3, T, Hq, Hkv, 1, 256, pad=0)
    c["v"] = v
    c["slots"] = np.arange(T, dtype=np.int32)
    h = handle(Hq, Hkv, 1, max_seqs=1, max_context=256)
    cache = Q.Q8Cache(1, Hkv)
    d, *_ = run_store(h, c, cache, 0)
    h.check_device()
    b, s = Q.quantise(v)
    got_b = d[2].cpu().numpy()[0, 0, 0, :T]
    got_s = d[3].cpu().numpy()[0, 0, 0, :T]
    assert np.array_equal(np.isnan(got_s), np.isnan(s[:, 0]))
    assert np.array_equal(got_s[~np.isnan(got_s)], s[:, 0][~np.isnan(got_s)])
    assert np.array_equal(got_b, b[:, 0])


def test_store_reports_bad_slots_and_positions(cuda):
    for field, value in (("slots", 256), ("pos", 40960), ("pos", -1)):
        c = store_case(4, 5, 8, 2, 1, 256, pad=0)
        c[field] = c[field].copy()
        c[field][3] = value
        h = handle(8, 2, 1, max_seqs=1, max_context=256)
        cache = Q.Q8Cache(1, 2, fill=0x11)
        d, *_ = run_store(h, c, cache, 0)
        st, detail = h.get_error()
        assert (st, detail) == (nvattn.ERR_OUT_OF_RANGE, value)
        _, k = oracle_rows({**c, "pos": np.where((c["pos"] < 0) | (c["pos"] >= 40960), 0,
                                                 c["pos"]).astype(np.int32)}, 8, 2)
        ok = np.arange(5) != 3
        cache.put(0, c["slots"][ok].astype(np.int64), k[ok], c["v"][ok])
        assert np.array_equal(d[0].cpu().numpy(), cache.kp)  # the other rows, and nothing else
        assert h.get_error()[0] == nvattn.OK


# ------------------------------------------------------------------ load

@pytest.mark.parametrize("T,Hkv,bs", [(1, 1, 256), (33, 8, 128), (777, 2, 512), (5000, 8, 256)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_load_reads_back_exactly(cuda, T, Hkv, bs, dtype):
    torch = torch_()
    rng = np.random.default_rng(T)
    nb = 5
    cache = Q.Q8Cache(nb, Hkv, 2, bs)
    cache.put(1, np.arange(nb * bs),
              (rng.standard_normal((nb * bs, Hkv, 128)) *
               2.0 ** rng.integers(-8, 12, (nb * bs, Hkv, 1))).astype(np.float32),
              rng.standard_normal((nb * bs, Hkv, 128)).astype(np.float32))
    cache.ks[1, 2, 0, 7] = np.nan
    slots = rng.integers(-1, nb * bs, T).astype(np.int32)  # repeats and padding
    slots[0] = 2 * bs + 7
    h = handle(8, Hkv, nb, n_layer=2, block_size=bs, max_seqs=1, max_context=bs)
    t = getattr(torch, dtype)
    ko = torch.full((T + 1, Hkv, 128), 7.0, dtype=t, device="cuda")
    vo = ko.clone()
    h.kv_load_q8(1, dev(slots), *cache.dev(), ko[:T], vo[:T])
    h.check_device()
    for got, want in zip((ko, vo), cache.rows(1, np.maximum(slots, 0).astype(np.int64))):
        want = np.where((slots >= 0)[:, None, None], want, 0)
        want = torch.from_numpy(want.astype(np.float32)).to(t)
        assert torch.equal(torch.nan_to_num(got[:T].cpu(), nan=5.5),
                           torch.nan_to_num(want, nan=5.5))
        assert (got[T] == 7).all()


def test_load_reports_a_slot_outside_the_cache(cuda):
    torch = torch_()
    cache = Q.Q8Cache(1, 2, fill=0x38)
    cache.ks[:] = 1
    cache.vs[:] = 1
    h = handle(8, 2, 1, max_seqs=1, max_context=256)
    ko = torch.full((3, 2, 128), 7.0, device="cuda")
    vo = ko.clone()
    h.kv_load_q8(0, dev(np.array([5, 256, 6], np.int32)), *cache.dev(), ko, vo)
    assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, 256)
    assert (ko[[0, 2]] == 1).all() and (ko[1] == 0).all() and (vo[1] == 0).all()


# ------------------------------------------------------------------ decode

def decode_case(seed, Hq, Hkv, lens, bs=256, n_layer=1, spread=0, num_blocks=None):
    rng = np.random.default_rng(seed)
    need = sum(-(-int(n) // bs) for n in lens)
    nb = num_blocks or need + 2
    bt = Q.tables(rng, lens, bs, nb)
    cache = Q.Q8Cache(nb, Hkv, n_layer, bs)  # NaN wherever no token is
    layer = n_layer - 1
    for s, n in enumerate(lens):
        if n:
            sl = Q.slots_of(bt[s], n, bs)
            k = rng.standard_normal((n, Hkv, 128))
            v = rng.standard_normal((n, Hkv, 128))
            if spread:
                v *= 2.0 ** rng.integers(-spread, spread + 1, (n, Hkv, 1))
            cache.put(layer, sl, k.astype(np.float32), v.astype(np.float32))
    q = (rng.standard_normal((len(lens), Hq, 128)) * 2).astype(np.float32)
    return dict(cache=cache, bt=bt, lens=np.asarray(lens, np.int32), q=q, layer=layer, bs=bs,
                Hq=Hq, Hkv=Hkv)


def make_handle(c, **kw):
    nl, nb = c["cache"].kp.shape[:2]
    kw.setdefault("max_seqs", len(c["lens"]))
    kw.setdefault("max_context", max(int(c["lens"].max()), 1))
    return handle(c["Hq"], c["Hkv"], nb, n_layer=nl, block_size=c["bs"], max_position=1, **kw)


def run_decode(c, bf16=False, h=None, extra=1, bound=None):
    torch = torch_()
    h = h or make_handle(c)
    q = to_q(c["q"], bf16)
    n = len(c["lens"])
    out = torch.full((n + extra,) + q.shape[1:], 7.0, dtype=q.dtype, device="cuda")
    h.decode_q8(c["layer"], q, *c["cache"].dev(), dev(c["bt"]), dev(c["lens"]),
                bound or int(c["lens"].max()), out[:n])
    torch.cuda.synchronize()
    assert (out[n:] == 7).all()  # rows behind the last sequence
    return h, out[:n].float().cpu().numpy(), q.float().cpu().numpy()


def expect(c, q):
    G = c["Hq"] // c["Hkv"]
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s, n in enumerate(c["lens"]):
        if n == 0:
            continue
        k, v = c["cache"].rows(c["layer"], Q.slots_of(c["bt"][s], n, c["bs"]))
        for hd in range(c["Hkv"]):
            r = slice(hd * G, (hd + 1) * G)
            want[s, r], tol[s, r] = Q.attend(q[s, r], k[:, hd], v[:, hd])
    return want, tol


EDGES = [1, 31, 0, 32, 33, 127, 128, 129, 255, 256, 257, 1000, 2049]


@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (16, 8), (32, 8), (64, 8), (8, 1), (1, 1)])
@pytest.mark.parametrize("bf16", [False, True])
def test_decode_edge_lengths(cuda, Hq, Hkv, bf16):
    c = decode_case(Hq + Hkv, Hq, Hkv, EDGES, n_layer=2)
    h, got, q = run_decode(c, bf16)
    h.check_device()
    Q.check(got, *expect(c, q), bf16)


@pytest.mark.parametrize("lens,bs", [([9000], 128), ([1], 1024), ([20000, 3], 512),
                                     ([300] * 70, 256), ([0, 0, 5], 256), ([0], 256)])
def test_decode_splits(cuda, lens, bs):
    c = decode_case(sum(lens) + bs, 16, 4, lens, bs)
    h, got, q = run_decode(c)
    h.check_device()
    Q.check(got, *expect(c, q), False)


@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (16, 8), (32, 8), (64, 8), (8, 1)])
@pytest.mark.parametrize("bf16", [False, True])
def test_decode_under_a_wide_bound(cuda, Hq, Hkv, bf16):
    """The host's bound of the contexts chooses the launch (it takes a third CTA
    per SM where the batch may be long); what it holds beyond the contexts, and
    the table's columns there, change nothing but the last bits."""
    c = decode_case(Hq + Hkv + 1, Hq, Hkv, EDGES + [6000], n_layer=2)
    cols = 320 * 1024 // Hkv // c["bs"]
    bound = cols * c["bs"]
    c["bt"] = np.concatenate([c["bt"], np.full((len(c["lens"]), cols - c["bt"].shape[1]), -1,
                                               np.int32)], 1)
    h = make_handle(c, max_context=bound)
    h, got, q = run_decode(c, bf16, h, bound=bound)
    h.check_device()
    Q.check(got, *expect(c, q), bf16)
    assert np.array_equal(run_decode(c, bf16, h, bound=bound)[1], got)


def test_decode_many_sequences(cuda):
    """More sequences than a warp scans at once, most of them short."""
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 40, 1100)
    lens[700] = 5000
    c = decode_case(6, 8, 2, lens.tolist())
    h, got, q = run_decode(c)
    h.check_device()
    Q.check(got, *expect(c, q), False)


def test_decode_scales_of_any_size(cuda):
    """V rows of very different magnitudes, K and q of extreme ones."""
    c = decode_case(7, 16, 8, [700, 33, 2000], spread=40)
    c["cache"].ks *= np.float32(2.0 ** 30)
    c["q"] *= np.float32(2.0 ** -30)
    h, got, q = run_decode(c)
    h.check_device()
    Q.check(got, *expect(c, q), False)


def test_decode_nan_row_and_poisoned_tail(cuda):
    """A token whose K or V row held a NaN makes its sequence's head NaN and
    nothing else; behind the context any bytes may lie (decode_case leaves NaN
    there)."""
    c = decode_case(8, 16, 8, [500, 300, 129])
    clean = expect(c, c["q"])
    c["cache"].ks[0, c["bt"][1, 0], 3, 17] = np.nan
    c["cache"].vs[0, c["bt"][2, 0], 5, 127] = np.nan
    h, got, q = run_decode(c)
    h.check_device()
    bad = np.zeros(got.shape, bool)
    bad[1, 6:8] = True
    bad[2, 10:12] = True
    assert np.isnan(got[bad]).all()
    Q.check(np.where(bad, clean[0], got), *clean, False)


def test_decode_is_deterministic_and_replays(cuda):
    """Launch after launch the same bits; a captured launch follows lengths,
    tables and rows that change between replays."""
    torch = torch_()
    c = decode_case(9, 32, 8, [4000, 17, 0, 900, 2500])
    h, first, q = run_decode(c)
    for _ in range(3):
        assert np.array_equal(run_decode(c, h=h)[1].view(np.uint32), first.view(np.uint32))
    d, bt, lens, tq = c["cache"].dev(), dev(c["bt"]), dev(c["lens"]), to_q(c["q"], False)
    out = torch.zeros(c["q"].shape, device="cuda")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        h.decode_q8(0, tq, *d, bt, lens, 4000, out, stream=s)
    for new in ([4000, 17, 0, 900, 2500], [1, 1, 0, 900, 2400], [3999, 0, 0, 1, 1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        out.fill_(9)
        g.replay()
        torch.cuda.synchronize()
        c["lens"] = np.array(new, np.int32)
        Q.check(out.cpu().numpy(), *expect(c, c["q"]), False)
    h.check_device()


def test_decode_reports_bad_blocks_and_lengths(cuda):
    c = decode_case(10, 16, 8, [600, 100, 40])
    h, good, _ = run_decode(c)
    bt = c["bt"].copy()
    c["bt"] = bt.copy()
    c["bt"][0, 1] = c["cache"].kp.shape[1]
    _, got, _ = run_decode(c, h=h)
    assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, c["cache"].kp.shape[1])
    assert np.array_equal(got[1:], good[1:])
    c["bt"][0, 1] = -1
    run_decode(c, h=h)
    assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, -1)
    c["bt"] = bt
    torch = torch_()
    out = torch.zeros(c["q"].shape, device="cuda")
    for bad in (601, -5):
        lens = np.array([600, bad, 40], np.int32)
        h.decode_q8(0, to_q(c["q"], False), *c["cache"].dev(), dev(bt), dev(lens), 600, out)
        st, detail = h.get_error()
        assert st == nvattn.ERR_OUT_OF_RANGE and (detail == bad or bad == 601)
    _, got, _ = run_decode(c, h=h)
    h.check_device()
    assert np.array_equal(got, good)


def test_store_then_decode_equals_the_rows_path(cuda):
    """A step as it is served: the new tokens stored into the 8-bit cache, the
    decode over it, and the same rows read back into a BF16 cache and attended
    by nvattn_paged_decode.  Both read the same values; the BF16 decode
    carries 16 bits of queries and weights, so the two differ by its bound."""
    torch = torch_()
    rng = np.random.default_rng(11)
    Hq, Hkv, lens = 32, 8, [257, 1, 900]
    c = decode_case(12, Hq, Hkv, lens)
    ctx, pos, slots = nvattn.plan_decode(lens, c["bt"])
    sc = store_case(13, 3, Hq, Hkv, 1, 256)
    sc.update(pos=pos, slots=slots)
    h = handle(Hq, Hkv, c["cache"].kp.shape[1], max_seqs=3, max_context=900)
    d, q_out, _, _ = run_store(h, sc, c["cache"], 0)
    _, k = oracle_rows(sc, Hq, Hkv)
    c["cache"].put(0, slots.astype(np.int64), k, sc["v"])
    out = torch.zeros((3, Hq, 128), device="cuda")
    h.decode_q8(0, q_out, *d, dev(c["bt"]), dev(ctx), 900, out)
    q = q_out.cpu().numpy()
    want, tol = expect(c, q)
    Q.check(out.cpu().numpy(), want, tol, False)
    n_slots = c["cache"].kp.shape[1] * 256
    kc = torch.zeros((n_slots, Hkv, 128), dtype=torch.bfloat16, device="cuda")
    vc = kc.clone()
    h.kv_load_q8(0, torch.arange(n_slots, dtype=torch.int32, device="cuda"), *d, kc, vc)
    out2 = torch.zeros_like(out)
    h.decode(0, q_out, kc, vc, dev(c["bt"]), dev(ctx), 900, out2)
    h.check_device()
    # 2^-16 of the scores' terms and of the weights
    Q.check(out2.cpu().numpy(), want, 2 * tol + 2.0 ** -15 * np.abs(want).max(), False)


def test_refusals(cuda):
    torch = torch_()
    c = decode_case(14, 16, 8, [300, 20])
    h = make_handle(c)
    d, bt, lens = c["cache"].dev(), dev(c["bt"]), dev(c["lens"])
    q, out = to_q(c["q"], False), torch.zeros(c["q"].shape, device="cuda")
    bad = nvattn.ERR_INVALID_ARG
    dec = lambda layer=0, q=q, d=d, bt=bt, lens=lens, mc=300, out=out: h.decode_q8(  # noqa: E731
        layer, q, *d, bt, lens, mc, out, check=False)
    assert dec() == nvattn.OK
    assert dec(layer=1) == bad and dec(layer=-1) == bad
    assert dec(mc=301) == bad and dec(mc=-1) == bad
    assert dec(lens=torch.zeros(3, dtype=torch.int32, device="cuda")) == bad  # > max_seqs
    assert dec(q=q.half(), out=out.half()) == bad
    with pytest.raises(ValueError):
        dec(q=q.bfloat16())
    assert dec(q=q.view(-1)[1:]) == bad  # not 16-byte aligned
    assert dec(lens=lens[:0]) == nvattn.OK
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    ko = torch.zeros((2, 8, 128), device="cuda")
    load = lambda slots=slots, ko=ko, vo=ko.clone(), d=d: h.kv_load_q8(  # noqa: E731
        0, slots, *d, ko, vo, check=False)
    assert load() == nvattn.OK and load(slots=slots[:0]) == nvattn.OK
    with pytest.raises(TypeError):
        load(ko=ko.double(), vo=ko.double())
    with pytest.raises(ValueError):
        load(ko=ko.half())
    L, n = nvattn.lib(), None
    p = ctypes.c_void_p(d[0].data_ptr())
    for i in range(4):
        c4 = [None if j == i else p for j in range(4)]
        assert L.nvattn_paged_decode_q8(h._h, 0, 1, p, 0, *c4, p, 2, p, 300, p, n) == bad
        assert L.nvattn_kv_load_q8(h._h, 0, 1, p, *c4, 0, p, p, n) == bad
    assert L.nvattn_kv_store_q8(h._h, 0, 1, p, p, p, p, p, p, p, p, 0, p, p, p, p, p, n, n) == bad
    assert L.nvattn_kv_store_q8(h._h, 0, 1, p, p, p, p, p, p, p, p, 9, p, p, p, p, n, n, n) == bad
    h.check_device()
