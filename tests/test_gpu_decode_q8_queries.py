"""The 8-bit decode's queries: rows whose dims differ by many powers of two keep
their bits in each dim (attend_bound's term is relative to |q k|, not to the row's
largest query), where the keys are zero in the large dims."""
import numpy as np
import pytest

import attend_bound as A
import q8_util as Q
import test_gpu_decode_q8_weights as W
import test_gpu_kv_q8 as T

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [6, 10, 15, 20])
@pytest.mark.parametrize("Hq,three", [(16, False), (64, True)])
@pytest.mark.parametrize("bf16", [False, True])
def test_large_dims_that_no_key_has(cuda, power, Hq, three, bf16):
    c = W.case(power + Hq, Hq, 8, [60, 1, 300, 700])
    c["q"][:, :, 77] *= np.float32(2.0 ** power)
    c["q"][:, ::3, 100] = 2.0 ** power
    for k in c["k"]:
        k[:, :, [77, 100]] = 0
    W.store(c)
    W.verify(c, bf16, W.wide(c) if three else None)


def test_queries_of_any_size(cuda):
    """From f32's smallest normal numbers to 2^90, against keys of the inverse."""
    for e in (-126, -60, 30, 90):
        c = W.store(W.case(e % 7, 16, 8, [40, 130]))
        c["q"] *= np.float32(2.0 ** e)
        c["cache"].ks *= np.float32(2.0 ** min(-e, 110))
        W.verify(c)
