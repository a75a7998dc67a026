"""Rows of the 8-bit cache that were never written, in arrays that begin as zeros (a
scale of 0): rows of zeros for the decode as for the read-back, as in the BF16 cache."""
import numpy as np
import pytest

import attend_bound as A
import q8_util as Q
import test_gpu_kv_q8 as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("written", [0, 1, 3, 100, 500])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e4])
def test_decode_over_a_zeroed_cache(cuda, written, size):
    c = T.decode_case(written + 1, 16, 8, [500, 40])
    for a in (c["cache"].kp, c["cache"].ks, c["cache"].vp, c["cache"].vs):
        a[:] = 0
    rng = np.random.default_rng(written)
    sl = Q.slots_of(c["bt"][0], 500, 256)
    at = rng.permutation(500)[:written]
    c["cache"].put(0, sl[at], rng.standard_normal((written, 8, 128), dtype=np.float32),
                   (rng.standard_normal((written, 8, 128)) * size).astype(np.float32))
    h, got, q = T.run_decode(c)
    h.check_device()
    k, v = c["cache"].rows(0, sl)
    sv = c["cache"].vs[0, sl // 256, :, sl % 256].astype(np.float64)
    for hd in range(8):
        r = slice(2 * hd, 2 * hd + 2)
        want, tol = A.attend(q[0, r], k[:, hd], v[:, hd], s_v=np.maximum(sv[:, hd], 2.0 ** -100))
        Q.check(got[0, r], want, tol, False)
    assert (got[1] == 0).all()


def test_a_new_runner_holds_rows_of_zeros(cuda):
    import torch
    import model_runner as MR
    device = torch.device("cuda:0")
    shape = MR.Qwen3Shape(n_layer=1, vocab=1003)
    w = MR.Qwen3Weights(shape, device, seed=3, norm_mean=1.0)
    run = MR.DecodeRunner(shape, w, 4, 1, 2, device, kv_cache="q8")
    k_q8, k_scale, v_q8, v_scale = run.q8_cache
    for payload, scale in ((k_q8, k_scale), (v_q8, v_scale)):
        assert (payload == 0).all() and (scale == 1).all()
