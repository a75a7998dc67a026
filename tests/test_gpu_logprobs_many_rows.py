"""nvattn_token_logprobs over more rows than one launch takes (65,535)."""
import numpy as np
import pytest

import nvattn
from gpu_util import handle

pytestmark = pytest.mark.gpu

N, V = 2 * 65535 + 5, 8


@pytest.mark.parametrize("bad", [None, 3, 65535 + 2, N - 1])
def test_rows_of_every_launch(cuda, bad):
    import torch
    h = handle(16, 8, 1, max_seqs=1, max_context=256, max_position=1)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((N, V), generator=g, device="cuda")
    tok = torch.randint(0, V, (N,), generator=g, device="cuda").int()
    good = torch.ones(N, dtype=torch.bool, device="cuda")
    if bad is not None:
        tok[bad], good[bad] = V, False
    lp, ent = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
    rank = torch.zeros(N, dtype=torch.int32, device="cuda")
    tid = torch.zeros((N, 2), dtype=torch.int32, device="cuda")
    tlp = torch.zeros((N, 2), device="cuda")
    h.token_logprobs(x, tok, lp, ent, rank, tid, tlp)
    if bad is None:
        h.check_device()
    else:
        assert h.get_error() == (nvattn.ERR_OUT_OF_RANGE, bad)
        assert torch.isnan(lp[bad]) and rank[bad] == -1
    want = torch.log_softmax(x.double(), -1)
    at = tok.clamp(max=V - 1).long()[:, None]
    # the sums of test_gpu_logprobs at V = 8
    tol = 60 * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -23 * (2 * float(x.abs().max()) + np.log(V))
    assert ((lp - want.gather(1, at)[:, 0]).abs()[good] <= tol).all()
    assert ((ent + (want.exp() * want).sum(-1)).abs() <= tol * (1 + np.log(V))).all()
    assert torch.equal(rank[good], (x > x.gather(1, at)).sum(-1).int()[good])
    top, ids = want.topk(2)
    assert torch.equal(tid.long(), ids) and ((tlp - top).abs() <= tol).all()
