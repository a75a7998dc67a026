"""nvattn_token_logprobs on the GPU against 64-bit softmax statistics and an
exact sort.  Tolerances: a logit is exact in f32; S is a sum of V terms in
chains of at most V/16384 + 60 f32 additions, each term within 2^-18 relative
(the argument of the exponential, at most 2^8 units, is rounded to 24 bits and
terms that far down do not count; near the maximum it is 2^-22), so log S is
within (V/16384 + 60) 2^-24 + 2^-18 and a log-probability within that plus its
own two roundings, 2^-23 (|x| + |m| + log V).  H adds T / S, with
|T| <= S (log V + ...): the same bound times (1 + log V)."""
import numpy as np
import pytest

import nvattn
from gpu_util import handle

pytestmark = pytest.mark.gpu


def torch_():
    import torch
    return torch


@pytest.fixture(scope="module")
def h(cuda):
    return handle(16, 8, 1, max_seqs=1, max_context=256, max_position=1)


def run(h, x, tokens, k, stream=None):
    torch = torch_()
    n = x.shape[0]
    o = dict(logprobs=torch.full((n + 1,), 7.0, device="cuda"),
             entropy=torch.full((n + 1,), 7.0, device="cuda"),
             ranks=torch.full((n + 1,), 77, dtype=torch.int32, device="cuda"))
    tid = torch.full((n + 1, max(k, 1)), 77, dtype=torch.int32, device="cuda")
    tlp = torch.full((n + 1, max(k, 1)), 7.0, device="cuda")
    h.token_logprobs(x, torch.as_tensor(tokens, dtype=torch.int32, device="cuda"),
                     o["logprobs"][:n], o["entropy"][:n], o["ranks"][:n],
                     tid[:n] if k else None, tlp[:n] if k else None)
    torch.cuda.synchronize()
    for t in list(o.values()) + [tid, tlp]:  # nothing behind the last row
        assert (t[n:].float() == (77 if t.dtype == torch.int32 else 7)).all()
    return [o[f][:n].cpu().numpy() for f in ("logprobs", "entropy", "ranks")] + \
        [tid[:n].cpu().numpy(), tlp[:n].cpu().numpy()]


def check(h, x, tokens, k):
    torch = torch_()
    lp, ent, rank, tid, tlp = run(h, x, tokens, k)
    h.check_device()
    xf = x.float().cpu().numpy()
    n, V = xf.shape
    xd = xf.astype(np.float64)
    m = xd.max(-1, keepdims=True)
    e = np.exp(xd - m)
    S = e.sum(-1, keepdims=True)
    want = xd - m - np.log(S)
    p = e / S
    H = -np.where(p > 0, p * np.where(p > 0, want, 0), 0).sum(-1)
    fin = np.where(np.isfinite(xd), np.abs(xd), 0).max(-1)
    tol = (V / 16384 + 60) * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -23 * (2 * fin + np.log(V))
    # the order: a stable sort keeps the lower id among equals
    order = np.argsort(-xf, axis=-1, kind="stable")
    for r in range(n):
        t = tokens[r]
        assert rank[r] == np.nonzero(order[r] == t)[0][0]
        if np.isfinite(want[r, t]):
            assert abs(lp[r] - want[r, t]) <= tol[r], (r, lp[r], want[r, t])
        else:
            assert lp[r] == want[r, t]
        assert abs(ent[r] - H[r]) <= tol[r] * (1 + np.log(V)), (r, ent[r], H[r])
        if k:
            assert np.array_equal(tid[r], order[r, :k]), (r, tid[r], order[r, :k])
            w = want[r, order[r, :k]]
            ok = np.isfinite(w)
            assert (np.abs(tlp[r][ok] - w[ok]) <= tol[r]).all()
            assert np.array_equal(tlp[r][~ok], w[~ok])


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1023, 1024, 1025, 4097, 32000, 151936, 200000])
@pytest.mark.parametrize("bf16", [False, True])
def test_values(h, V, bf16):
    torch = torch_()
    rng = np.random.default_rng(V)
    n = 3
    x = torch.from_numpy((rng.standard_normal((n, V)) * 4).astype(np.float32)).cuda()
    x[1] *= 0.01           # nearly uniform
    x[2, V // 2] = 60.0    # nearly certain
    x = x.bfloat16() if bf16 else x
    check(h, x, [0, V - 1, V // 2], min(V, 20))


@pytest.mark.parametrize("n", [2, 37, 75, 149, 300, 700])
def test_rows_of_every_cluster_size(h, n):
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn((n, 70001), generator=g, device="cuda") * 3
    x[:, 60000:] = float("-inf")
    x = x[:, :66000]       # rows of 70001: no 16-byte alignment
    check(h, x, np.random.default_rng(n).integers(0, 60000, n), 5)


@pytest.mark.parametrize("V,pad", [(5000, 0), (5000, 1), (5001, 3), (4096, 4)])
@pytest.mark.parametrize("bf16", [False, True])
def test_strides_and_offsets(h, V, pad, bf16):
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(V + pad)
    x = torch.randn((6, V + pad), generator=g, device="cuda")
    x = (x.bfloat16() if bf16 else x)[1:, :V]
    check(h, x, [0, 1, 2, 3, V - 1], 7)


def test_ties_sorted_and_constant_rows(h):
    """Rows whose top ids need each of the finish's ways: ties by the lowest
    id, descending and ascending logits (one tile holds the whole top), all
    equal (every logit reaches the limit), zeros of both signs, a block of
    equals larger than the candidate list."""
    torch = torch_()
    V = 40000
    rows = torch.zeros((7, V))
    rows[0] = torch.arange(V, 0, -1) / V
    rows[1] = torch.arange(V) / V
    rows[2] = 1.25
    rows[3, ::2] = -0.0
    rows[4] = torch.randint(0, 5, (V,), generator=torch.Generator().manual_seed(1)).float()
    rows[5] = torch.randn(V, generator=torch.Generator().manual_seed(2))
    rows[5, 7000:12000] = 9.0
    rows[6] = float("-inf")
    rows[6, 100:150] = 0.5
    for bf16 in (False, True):
        x = rows.cuda().bfloat16() if bf16 else rows.cuda()
        for k in (1, 20, 64):
            check(h, x, [5, 5, 39999, 1, 17, 11999, 149], k)


def test_largest_vocabulary_and_top_0(h):
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((1, 2097152), generator=g, device="cuda")
    check(h, x, [2097151], 64)
    check(h, x[:, :1000], [3], 0)


def test_nan_and_infinite_logits(h):
    """The formulas' NaN in the values; ids stay distinct and in the order in
    which a NaN counts as -inf."""
    torch = torch_()
    V = 3000
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((4, V), generator=g, device="cuda")
    x[0, 1500] = float("nan")
    x[1, 20] = float("inf")
    x[2] = float("-inf")
    x[3] = float("nan")
    lp, ent, rank, tid, tlp = run(h, x, [1500, 20, 2, 7], 9)
    assert np.isnan(lp).all() and np.isnan(ent).all() and np.isnan(tlp).all()
    xs = np.where(np.isnan(x.cpu().numpy()), -np.inf, x.cpu().numpy())
    order = np.argsort(-xs, axis=-1, kind="stable")
    assert np.array_equal(tid, order[:, :9])
    assert [np.nonzero(order[r] == t)[0][0] for r, t in enumerate([1500, 20, 2, 7])] == \
        rank.tolist()


def test_bad_tokens_are_reported(h):
    torch = torch_()
    x = torch.zeros((3, 50), device="cuda")
    for bad in (-1, 50):
        lp, ent, rank, tid, _ = run(h, x, [4, bad, 6], 2)
        assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, 1)
        assert np.isnan(lp[1]) and rank.tolist() == [4, -1, 6]
        assert np.allclose(lp[[0, 2]], -np.log(50), atol=1e-6)
        assert np.allclose(ent, np.log(50), atol=1e-5) and tid.tolist() == [[0, 1]] * 3


def test_partial_outputs_streams_and_replay(h):
    torch = torch_()
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((5, 9000), generator=g, device="cuda")
    tok = torch.arange(5, dtype=torch.int32, device="cuda")
    full = run(h, x, [0, 1, 2, 3, 4], 4)
    e = torch.zeros(5, device="cuda")
    h.token_logprobs(x, entropy=e)
    assert np.array_equal(e.cpu().numpy(), full[1])
    tid = torch.zeros((5, 4), dtype=torch.int32, device="cuda")
    tlp = torch.zeros((5, 4), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        h.token_logprobs(x, tok, e, top_ids=tid, top_logprobs=tlp, stream=s)
    x.copy_(x.flip(0))
    graph.replay()
    want = run(h, x, [0, 1, 2, 3, 4], 4)
    assert np.array_equal(e.cpu().numpy(), want[0])
    assert np.array_equal(tid.cpu().numpy(), want[3]) and np.array_equal(tlp.cpu().numpy(), want[4])
    h.check_device()


def test_refusals(h):
    torch = torch_()
    x = torch.zeros((2, 100), device="cuda")
    t = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.zeros(2, device="cuda")
    k = torch.zeros((2, 5), dtype=torch.int32, device="cuda")
    kf = torch.zeros((2, 5), device="cuda")
    bad, no = nvattn.ERR_INVALID_ARG, nvattn.ERR_UNSUPPORTED
    go = lambda *a, **kw: h.token_logprobs(*a, check=False, **kw)  # noqa: E731
    assert go(x, t, f) == nvattn.OK and go(x[:0], t, f) == nvattn.OK
    assert go(x, None, f) == bad and go(x, None, None, None, t) == bad
    assert go(x, t, f, top_ids=k) == bad
    assert go(x[:, :4], t, f, top_ids=k, top_logprobs=kf) == bad          # top_k > n_vocab
    assert go(x, t, f, top_ids=torch.zeros((2, 65), dtype=torch.int32, device="cuda"),
              top_logprobs=kf) == no
    assert go(torch.zeros((1, 2097153), device="cuda"), t, f) == no
    assert go(x[:1].expand(2, 100), t, f) == bad  # one row for all: stride 0
    with pytest.raises(ValueError):
        go(x.t(), t, f)
    with pytest.raises(TypeError):
        go(x.double(), t, f)
    L = nvattn.lib()
    p = x.data_ptr()
    assert L.nvattn_token_logprobs(h._h, 1, 100, p, 0, 99, t.data_ptr(), f.data_ptr(), None, None,
                                   0, None, None, None) == bad           # stride < n_vocab
    assert L.nvattn_token_logprobs(h._h, 1, 100, p + 2, 0, 100, t.data_ptr(), f.data_ptr(), None,
                                   None, 0, None, None, None) == bad     # misaligned f32
    assert L.nvattn_token_logprobs(h._h, 1, 100, p, 2, 100, t.data_ptr(), f.data_ptr(), None, None,
                                   0, None, None, None) == bad           # f16 logits
    h.check_device()
