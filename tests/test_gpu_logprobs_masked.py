"""nvattn_token_logprobs on rows masked with large negative finite values instead
of -inf: whole tiles, warps' and CTAs' shares of them beside ordinary logits.  The
tolerances are test_gpu_logprobs', over the logits that are not masked: e^(x - m)
of the others is 0 in f32 and in 64 bits."""
import numpy as np
import pytest

from gpu_util import handle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def h(cuda):
    return handle(16, 8, 1, max_seqs=1, max_context=256, max_position=1)


def check(h, x, kept, tokens, k=5):
    """kept [n][V]: the logits that are not masked (a row of masked ones alone is
    a row of equals)."""
    import torch
    n, V = x.shape
    lp, ent = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    rank = torch.zeros(n, dtype=torch.int32, device="cuda")
    tid = torch.zeros((n, k), dtype=torch.int32, device="cuda")
    tlp = torch.zeros((n, k), device="cuda")
    h.token_logprobs(x, torch.as_tensor(tokens, dtype=torch.int32, device="cuda"), lp, ent, rank,
                     tid, tlp)
    h.check_device()
    lp, ent, rank, tid, tlp = (t.cpu().numpy() for t in (lp, ent, rank, tid, tlp))
    xd = x.double().cpu().numpy()
    m = xd.max(-1, keepdims=True)
    e = np.exp(xd - m)
    S = e.sum(-1, keepdims=True)
    want = xd - m - np.log(S)
    H = -np.where(e > 0, e / S * want, 0).sum(-1)
    big = np.where(kept, np.abs(xd), 0).max(-1)
    tol = (V / 16384 + 60) * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -23 * (2 * big + np.log(V))
    order = np.argsort(-xd, axis=-1, kind="stable")
    assert np.isfinite(ent).all(), ent
    assert (np.abs(ent - H) <= tol * (1 + np.log(V))).all(), (ent, H)
    for r in range(n):
        t = tokens[r]
        far = 2.0 ** -22 * abs(want[r, t])  # a masked token's value: two roundings of it
        assert abs(lp[r] - want[r, t]) <= tol[r] + far, (r, lp[r], want[r, t])
        assert rank[r] == np.nonzero(order[r] == t)[0][0]
        assert np.array_equal(tid[r], order[r, :k])
        w = want[r, order[r, :k]]
        assert (np.abs(tlp[r] - w) <= tol[r] + 2.0 ** -22 * np.abs(w)).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("mask", ["lowest", -1e36, -1e30, -1e9])
@pytest.mark.parametrize("n", [1, 300])
def test_masked_tiles(h, bf16, mask, n):
    """n = 1: eight CTAs for the row; 300: one."""
    import torch
    V = 151936
    dt = torch.bfloat16 if bf16 else torch.float32
    low = torch.finfo(dt).min if mask == "lowest" else mask
    g = torch.Generator(device="cuda").manual_seed(n)
    keep = torch.zeros((5, V), dtype=torch.bool, device="cuda")
    keep[0, 140000:] = True                # each warp's first tiles masked, or all of a warp's
    keep[1, :1024] = True                  # all but one warp
    keep[2, 77777] = True                  # one logit
    keep[3] = torch.arange(V, device="cuda") // 1024 % 2 == 1  # every other tile
    keep[4, 16384 * 3:16384 * 4] = True    # one CTA's share of the row
    x = torch.randn((5, V), generator=g, device="cuda") * 3
    x = torch.where(keep, x, torch.full_like(x, low)).to(dt)
    keep = keep.cpu().numpy()
    tok = [140005, 1024, 77777, 1030, 16384 * 3 + 9]
    if n == 1:
        for r in range(5):
            check(h, x[r:r + 1], keep[r:r + 1], tok[r:r + 1])
    else:  # 300 rows: the five again and again
        rows = torch.arange(n, device="cuda") % 5
        check(h, x[rows], keep[rows.cpu().numpy()], [tok[i % 5] for i in range(n)])


@pytest.mark.parametrize("bf16", [False, True])
def test_a_row_of_the_lowest_value(h, bf16):
    """All equal: the uniform distribution over the vocabulary."""
    import torch
    dt = torch.bfloat16 if bf16 else torch.float32
    for V in (50, 5000, 151936):
        x = torch.full((2, V), torch.finfo(dt).min, dtype=dt, device="cuda")
        check(h, x, np.zeros((2, V), bool), [0, V - 1])
