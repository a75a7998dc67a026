"""nvattn_paged_tree_decode on the GPU against 64-bit attention under the
tree's mask, within the bound that q8_util.attend derives (bf16 outputs: the
softmax weights are sums of two bf16 terms, 2^-17, and the output rounds once)."""
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


def random_tree(rng, n, words):
    """Ancestor masks, and set bits behind the nodes that must not matter."""
    m = np.zeros((n, words * 64), bool)
    for i in range(n):
        up = rng.integers(-1, i) if i else -1
        if up >= 0:
            m[i] = m[up]
        m[i, i] = True
    m[:, n:] = rng.random((n, words * 64 - n)) < 0.5
    return m


def pack(m):
    bits = m.reshape(m.shape[0], m.shape[1] // 64, 64).astype(np.uint64)
    return (bits << np.arange(64, dtype=np.uint64)).sum(-1, dtype=np.uint64)


def tree_case(seed, Hq, Hkv, lens, nodes, bs=256, n_layer=1, words=1):
    rng = np.random.default_rng(seed)
    nb = sum(-(-int(n) // bs) for n in lens) + 2
    layer = n_layer - 1
    bt = Q.tables(rng, lens, bs, nb)
    nan = np.uint16(0x7fc0)
    k = np.full((n_layer, nb * bs, Hkv, 128), nan, np.uint16)
    v = k.copy()
    for s, n in enumerate(lens):  # NaN wherever no token is
        sl = Q.slots_of(bt[s], n, bs)
        k[layer, sl] = O.f32_to_bf16(rng.standard_normal((n, Hkv, 128), dtype=np.float32))
        v[layer, sl] = O.f32_to_bf16(rng.standard_normal((n, Hkv, 128), dtype=np.float32))
    masks = [random_tree(rng, n, words) for n in nodes]
    T = sum(nodes)
    return dict(Hq=Hq, Hkv=Hkv, bs=bs, layer=layer, n_layer=n_layer, nb=nb, bt=bt, k=k, v=v,
                lens=np.asarray(lens, np.int32), nodes=list(nodes), masks=masks, words=words,
                cu=np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32),
                q=(rng.standard_normal((T, Hq, 128)) * 2).astype(np.float32))


def mask_dev(c):
    m = np.concatenate([pack(m) for m in c["masks"]]) if c["q"].shape[0] else \
        np.zeros((0, c["words"]), np.uint64)
    return dev(m.view(np.int64).reshape(-1, c["words"]))


def make_handle(c, **kw):
    return handle(c["Hq"], c["Hkv"], c["nb"], n_layer=c["n_layer"], block_size=c["bs"],
                  max_seqs=len(c["lens"]), max_context=max(int(c["lens"].max()), 1),
                  max_position=1, **kw)


def run(c, bf16, h=None, max_nodes=None):
    torch = torch_()
    h = h or make_handle(c)
    q = torch.from_numpy(c["q"]).cuda()
    q = q.bfloat16() if bf16 else q
    T = q.shape[0]
    out = torch.full((T + 1,) + q.shape[1:], 7.0, dtype=q.dtype, device="cuda")
    h.tree_decode(c["layer"], q, dev(c["cu"]), mask_dev(c), max_nodes or max(c["nodes"] + [1]),
                  dev(c["k"]), dev(c["v"]), dev(c["bt"]), dev(c["lens"]), int(c["lens"].max()),
                  out[:T])
    torch.cuda.synchronize()
    assert (out[T:] == 7).all()
    return h, out[:T].float().cpu().numpy(), q.float().cpu().numpy()


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
            w, t = Q.attend(q[rows, hs].reshape(N * G, 128), k[:, hd], v[:, hd],
                            np.repeat(keep, G, 0), weight_bits=16 if bf16 else 20)
            want[rows, hs], tol[rows, hs] = w.reshape(N, G, 128), t.reshape(N, G, 128)
    return want, tol


def verify(c, bf16, h=None, **kw):
    h, got, q = run(c, bf16, h, **kw)
    h.check_device()
    Q.check(got, *expect(c, q, bf16), bf16)
    return h, got


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("Hq,Hkv", [(16, 8), (8, 8), (32, 8), (64, 8), (8, 1), (1, 1)])
def test_ragged_trees(cuda, bf16, Hq, Hkv):
    """Prefixes that end at every offset of a tile, trees that straddle tiles,
    a tree without a prefix, a sequence without nodes, a single node."""
    lens = [63, 64, 65, 300, 1, 127, 200, 10, 1000]
    nodes = [8, 64, 2, 17, 1, 63, 0, 10, 33]
    verify(tree_case(Hq + Hkv, Hq, Hkv, lens, nodes, n_layer=2), bf16)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("lens,nodes,words,bs", [
    ([20000], [5], 1, 256), ([256], [256], 4, 128), ([5000, 300, 130], [100, 128, 70], 2, 512),
    ([2000] * 40, [3] * 40, 1, 256), ([1], [1], 1, 1024), ([777, 777], [200, 250], 4, 256)])
def test_long_wide_and_many(cuda, bf16, lens, nodes, words, bs):
    verify(tree_case(sum(lens) + words, 16, 4, lens, nodes, bs, words=words), bf16)


def test_many_sequences(cuda):
    rng = np.random.default_rng(3)
    nodes = rng.integers(0, 5, 300)
    lens = nodes + rng.integers(0, 90, 300)
    lens[120], nodes[120] = 3000, 9
    verify(tree_case(4, 8, 2, lens.tolist(), nodes.tolist()), True)


@pytest.mark.parametrize("bf16", [True, False])
def test_rows_that_attend_nothing(cuda, bf16):
    """Masks that leave a node nothing: zeros without a prefix, the prefix
    alone with one."""
    c = tree_case(5, 16, 8, [6, 200], [6, 9])
    c["masks"][0][3] = False
    c["masks"][1][2] = False
    h, got = verify(c, bf16)
    assert (got[3] == 0).all() and np.isfinite(got).all()


@pytest.mark.parametrize("bf16", [True, False])
def test_padded_nodes_and_nan_rows(cuda, bf16):
    """Padding nodes that no mask names, with NaN K/V rows: nothing of them
    reaches the others.  A NaN in the V row of a node reaches the rows that
    attend it, and only those."""
    c = tree_case(6, 32, 8, [150, 100], [40, 30])
    for s in (0, 1):
        N, n = c["nodes"][s], int(c["lens"][s])
        pad = np.arange(N) >= N - 7
        c["masks"][s][:, :N][:, pad] = False
        sl = Q.slots_of(c["bt"][s], n, 256)[n - N:][pad]
        c["k"][0, sl] = 0x7fc0
        c["v"][0, sl] = np.array([0x7fc0, 0x7f80, 0xff80, 0x7fff, 0xffff, 0x7f81, 0xffc0],
                                 np.uint16)[:, None, None]
    clean = dict(c, k=c["k"].copy(), v=c["v"].copy())
    for x in "kv":
        clean[x][~np.isfinite(O.bf16_to_f32(clean[x]))] = 0
    h, got, q = run(c, bf16)
    h.check_device()
    want, tol = expect(clean, q, bf16)
    Q.check(got, want, tol, bf16)
    sl = Q.slots_of(c["bt"][0], 150, 256)[110 + 4]  # node 4 of sequence 0
    c["v"][0, sl, 2, 77] = 0x7fc0
    h, got, q = run(c, bf16)
    sees = c["masks"][0][:, 4]
    G = 4
    bad = np.zeros(got.shape, bool)
    bad[:40][sees, 2 * G:3 * G] = True
    assert np.isnan(got[bad]).all()
    Q.check(np.where(bad, want, got), want, tol, bf16)


@pytest.mark.parametrize("bf16", [True, False])
def test_nan_rows_in_every_other_tile(cuda, bf16):
    """Tiles with nodes one after another (five per unit, several units per
    CTA); in every other 64 positions the nodes' V rows are NaN and no mask
    names them: what is noted of one tile is not taken for another's."""
    Hq, Hkv, n_seqs, N = 1, 1, 200, 250
    c = tree_case(21, Hq, Hkv, [N + 3] * n_seqs, [N] * n_seqs, bs=128, words=4)
    at = np.arange(3, N + 3)
    for s in range(n_seqs):
        pad = (at // 64 + s) % 2 == 0
        c["masks"][s][:, :N][:, pad] = False
        c["v"][0, Q.slots_of(c["bt"][s], N + 3, 128)[3:][pad]] = 0x7fc0
    clean = dict(c, v=c["v"].copy())
    clean["v"][~np.isfinite(O.bf16_to_f32(clean["v"]))] = 0
    h, got, q = run(c, bf16)
    h.check_device()
    Q.check(got, *expect(clean, q, bf16), bf16)
    for _ in range(5):
        assert np.array_equal(run(c, bf16, h)[1], got)


def test_one_node_is_the_decode(cuda):
    """A tree of one node is a decode step."""
    torch = torch_()
    c = tree_case(7, 32, 8, [1, 500, 2000, 64], [1, 1, 1, 1])
    h, got = verify(c, False)
    out = torch.zeros(c["q"].shape, device="cuda")
    h.decode(0, dev(c["q"]), dev(c["k"]), dev(c["v"]), dev(c["bt"]), dev(c["lens"]), 2000, out)
    want, tol = expect(c, c["q"], False)
    # the decode carries 16 bits of queries and weights
    Q.check(out.cpu().numpy(), got, 2 * tol + 2.0 ** -15 * np.abs(want).max(), False)


def test_deterministic_and_replayed(cuda):
    torch = torch_()
    c = tree_case(8, 32, 8, [4000, 130, 900, 70], [50, 13, 64, 1])
    h, first = verify(c, True)
    for _ in range(3):
        assert np.array_equal(run(c, True, h)[1], first)
    lens, cu, mask = dev(c["lens"]), dev(c["cu"]), mask_dev(c)
    kc, vc, bt = dev(c["k"]), dev(c["v"]), dev(c["bt"])
    q = torch.from_numpy(c["q"]).cuda().bfloat16()
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        h.tree_decode(0, q, cu, mask, 64, kc, vc, bt, lens, 4000, out, stream=s)
    qf = q.float().cpu().numpy()
    for new_lens, new_nodes in (([4000, 130, 900, 70], [50, 13, 64, 1]),
                                ([2000, 64, 64, 3], [10, 0, 64, 3]),
                                ([50, 130, 1, 70], [50, 13, 1, 64])):
        d = dict(c, lens=np.array(new_lens, np.int32), nodes=new_nodes,
                 cu=np.concatenate([[0], np.cumsum(new_nodes)]).astype(np.int32))
        flat = np.concatenate(c["masks"])
        d["masks"] = [flat[a:b] for a, b in zip(d["cu"], d["cu"][1:])]
        lens.copy_(dev(d["lens"]))
        cu.copy_(dev(d["cu"]))
        out.fill_(7)
        g.replay()
        torch.cuda.synchronize()
        T = int(d["cu"][-1])
        got = out.float().cpu().numpy()
        assert (got[T:] == 7).all()
        Q.check(got[:T], *expect(d, qf[:T], True), True)
    h.check_device()


@pytest.mark.parametrize("bf16", [True, False])
def test_scores_that_keep_rising(cuda, bf16):
    """Each tile's scores pass the last one's by far more than the reference's
    slack (2^32), so every tile rescales; then the same falling."""
    rng = np.random.default_rng(13)
    for sign in (1, -1):
        c = tree_case(14, 16, 8, [1500, 700], [30, 3])
        d = rng.standard_normal(128)
        d /= np.linalg.norm(d)
        c["q"] = (d * 12 + 0.05 * rng.standard_normal(c["q"].shape)).astype(np.float32)
        for s, n in enumerate(c["lens"]):
            sl = Q.slots_of(c["bt"][s], n, 256)
            # d.k up to n / 10: in steps of 8 sqrt(128) log2-units per 64 keys and more
            rise = sign * np.arange(n)[:, None, None] / 10.0 * d
            c["k"][0, sl] = O.f32_to_bf16((rise + 0.05 * rng.standard_normal(
                (n, 8, 128))).astype(np.float32))
        verify(c, bf16)


def test_many_short_units_repeat_exactly(cuda):
    """Units of one to five key tiles one after another on every CTA, again and
    again: the hand-over between units has no room for a stale accumulator."""
    rng = np.random.default_rng(15)
    lens = rng.integers(1, 300, 400)
    nodes = np.minimum(rng.integers(1, 40, 400), lens)
    c = tree_case(16, 16, 8, lens.tolist(), nodes.tolist())
    for bf16 in (True, False):
        h, first = verify(c, bf16)
        for _ in range(20):
            assert np.array_equal(run(c, bf16, h)[1], first)
        h.check_device()


def test_the_8_bit_decode_shares_the_workspace(cuda):
    """Tree and 8-bit decodes alternating on one handle: both leave their
    tickets as they found them."""
    torch = torch_()
    c = tree_case(9, 16, 8, [3000, 500], [20, 3])
    h, first = verify(c, False)
    cache = Q.Q8Cache(c["nb"], 8)
    rng = np.random.default_rng(10)
    for s, n in enumerate(c["lens"]):
        cache.put(0, Q.slots_of(c["bt"][s], n, 256),
                  rng.standard_normal((n, 8, 128)).astype(np.float32),
                  rng.standard_normal((n, 8, 128)).astype(np.float32))
    d, q = cache.dev(), dev(c["q"][:2])
    outs = []
    for _ in range(3):
        out = torch.zeros((2, 16, 128), device="cuda")
        h.decode_q8(0, q, *d, dev(c["bt"]), dev(c["lens"]), 3000, out)
        outs.append(out.cpu().numpy())
        assert np.array_equal(run(c, False, h)[1], first)
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])
    h.check_device()


def test_bad_metadata_is_reported(cuda):
    torch = torch_()
    c = tree_case(11, 16, 8, [300, 100, 400], [9, 5, 20])
    h, good = verify(c, True)
    a, b = c["cu"][1], c["cu"][2]
    want, tol = expect(c, torch.from_numpy(c["q"]).bfloat16().float().numpy(), True)
    for field, value in (("lens", 4), ("lens", 401), ("lens", -1)):
        d = dict(c, lens=c["lens"].copy())
        d["lens"][1] = value
        q = torch.from_numpy(c["q"]).cuda().bfloat16()
        out = torch.full_like(q, 7)
        h.tree_decode(0, q, dev(c["cu"]), mask_dev(c), 20, dev(c["k"]), dev(c["v"]), dev(c["bt"]),
                      dev(d["lens"]), 400, out)
        assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, value)
        got = out.float().cpu().numpy()
        assert (got[a:b] == 7).all()
        # (the batch is split elsewhere without the skipped sequence)
        rest = np.r_[0:a, b:len(got)]
        Q.check(got[rest], want[rest], tol[rest], True)
    for cu in ([0, 9, 8, 34], [0, 9, 14, 35], [-1, 9, 14, 34], [0, 9, 31, 34]):
        d = dict(c, cu=np.array(cu, np.int32))
        run(d, True, h, max_nodes=20)
        assert h.get_error()[0] == nvattn.ERR_OUT_OF_RANGE
    d = dict(c, bt=c["bt"].copy())
    d["bt"][2, 1] = c["nb"]
    _, got, _ = run(d, True, h)
    assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, c["nb"])
    assert np.array_equal(got[:b], good[:b])
    assert np.array_equal(run(c, True, h)[1], good)
    h.check_device()


def test_refusals(cuda):
    torch = torch_()
    c = tree_case(12, 16, 8, [300, 100], [9, 5])
    h = make_handle(c)
    q = torch.from_numpy(c["q"]).cuda()
    out = torch.zeros_like(q)
    a = dict(layer=0, q=q, cu=dev(c["cu"]), mask=mask_dev(c), mn=9, k=dev(c["k"]), v=dev(c["v"]),
             bt=dev(c["bt"]), lens=dev(c["lens"]), mc=300, out=out)
    bad, no = nvattn.ERR_INVALID_ARG, nvattn.ERR_UNSUPPORTED

    def go(**kw):
        x = dict(a, **kw)
        return h.tree_decode(x["layer"], x["q"], x["cu"], x["mask"], x["mn"], x["k"], x["v"],
                             x["bt"], x["lens"], x["mc"], x["out"], check=False)

    assert go() == nvattn.OK
    assert go(layer=1) == bad and go(mn=65) == bad and go(mn=-1) == bad and go(mc=301) == bad
    assert go(bt=a["bt"][:, :1]) == bad
    p, L = q.data_ptr(), nvattn.lib()
    for i in range(7):  # q, cu_nodes, mask, k, v, tables, lengths: each of them null
        x = [None if j == i else p for j in range(7)]
        assert L.nvattn_paged_tree_decode(h._h, 0, 2, 14, x[0], 0, x[1], x[2], 1, 9, x[3], x[4],
                                          x[5], 2, x[6], 300, p, None) == bad
    assert go(q=q.half(), out=out.half()) == bad
    assert go(lens=torch.zeros(3, dtype=torch.int32, device="cuda")) == bad
    assert go(lens=a["lens"][:0]) == nvattn.OK and go(q=q[:0], out=out[:0]) == nvattn.OK
    assert go(mask=torch.zeros((14, 5), dtype=torch.int64, device="cuda")) == no
    assert go(out=out.view(-1)[1:-127].view(-1, 128)) == bad
    with pytest.raises(ValueError):
        go(out=out.bfloat16())
    with pytest.raises(ValueError):
        go(mask=a["mask"].int())
    h.check_device()
