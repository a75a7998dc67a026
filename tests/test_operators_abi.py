"""CPU tests of the 8-bit cache, draft-tree and log-probability entry points:
their argument checks come before any device work."""
import nvattn


def test_q8_entry_points_reject_a_null_handle():
    L = nvattn.lib()
    assert L.nvattn_kv_store_q8(None, 0, 1, *([None] * 8), 0, *([None] * 7)) == \
        nvattn.ERR_INVALID_ARG
    assert L.nvattn_kv_load_q8(None, 0, 1, *([None] * 5), 0, None, None, None) == \
        nvattn.ERR_INVALID_ARG
    assert L.nvattn_paged_decode_q8(None, 0, 1, None, 0, *([None] * 5), 1, None, 1, None,
                                    None) == nvattn.ERR_INVALID_ARG


def test_logprobs_rejects_a_null_handle():
    assert nvattn.lib().nvattn_token_logprobs(None, 1, 10, None, 0, 10, None, None, None, None, 0,
                                              None, None, None) == nvattn.ERR_INVALID_ARG


def test_tree_decode_rejects_a_null_handle():
    assert nvattn.lib().nvattn_paged_tree_decode(None, 0, 1, 1, None, 0, None, None, 1, 1, None,
                                                 None, None, 1, None, 1, None, None) == \
        nvattn.ERR_INVALID_ARG
