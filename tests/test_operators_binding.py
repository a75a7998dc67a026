"""CPU tests of what the Python methods of the 8-bit cache, draft-tree and
log-probability entry points refuse before they call the library: tensors of a type
that the kernels would read as something else, and top outputs of different widths.  The handle is
null, so a call that passes the checks ends in the library's own refusal."""
import pytest

import nvattn


@pytest.fixture()
def h():
    x = object.__new__(nvattn.Handle)
    x._h, x._L = None, nvattn.lib()
    return x


def torch_():
    import torch
    return torch


def others(t):
    """The tensor in types that are not the expected one."""
    torch = torch_()
    if t.dtype == torch.float32:
        return [t.double(), t.half(), t.int()]
    return [t.long(), t.short(), t.float()]


def refused(call, args, names):
    assert call(**args) == nvattn.ERR_INVALID_ARG  # the null handle, and nothing before it
    for name in names:
        for t in others(args[name]):
            with pytest.raises(TypeError):
                call(**dict(args, **{name: t}))


def test_token_logprobs(h):
    torch = torch_()
    i, f = (lambda *s: torch.zeros(s, dtype=torch.int32)), torch.zeros
    a = dict(logits=f(4, 100), tokens=i(4), logprobs=f(4), entropy=f(4), ranks=i(4),
             top_ids=i(4, 5), top_logprobs=f(4, 5), check=False)
    refused(h.token_logprobs, a, [n for n in a if n not in ("logits", "check")])
    for k in (4, 6):  # narrower: its rows would be written out of range
        with pytest.raises(ValueError):
            h.token_logprobs(**dict(a, top_logprobs=f(4, k)))
    with pytest.raises(TypeError):
        h.token_logprobs(**dict(a, tokens=a["logits"].argmax(-1)))


def test_q8_cache(h):
    torch = torch_()
    i, f = (lambda *s: torch.zeros(s, dtype=torch.int32)), torch.zeros
    page = torch.zeros((1, 2, 1, 256, 128), dtype=torch.uint8)
    cache = dict(k_q8=page, k_scale=f(1, 2, 1, 256), v_q8=page.view(torch.float8_e4m3fn),
                 v_scale=f(1, 2, 1, 256))
    w = torch.zeros(128, dtype=torch.bfloat16)
    store = dict(cache, layer=0, q=f(3, 2, 128), k=f(3, 1, 128), v=f(3, 1, 128), q_norm_w=w,
                 k_norm_w=w, positions=i(3), slots=i(3), q_out=f(3, 2, 128), check=False)
    refused(h.kv_store_q8, store, ["positions", "slots", "k_scale", "v_scale"])
    load = dict(cache, layer=0, slots=i(3), k_out=f(3, 1, 128), v_out=f(3, 1, 128), check=False)
    refused(h.kv_load_q8, load, ["slots", "k_scale", "v_scale"])
    decode = dict(cache, layer=0, q=f(3, 2, 128), block_tables=i(3, 1), context_lens=i(3),
                  max_context_len=200, out=f(3, 2, 128), check=False)
    refused(h.decode_q8, decode, ["block_tables", "context_lens", "k_scale", "v_scale"])
    for call, a in ((h.kv_store_q8, store), (h.kv_load_q8, load), (h.decode_q8, decode)):
        for name in ("k_q8", "v_q8"):
            with pytest.raises(TypeError):
                call(**dict(a, **{name: page.bfloat16()}))


def test_tree_decode(h):
    torch = torch_()
    i, f = (lambda *s: torch.zeros(s, dtype=torch.int32)), torch.zeros
    kv = torch.zeros((1, 256, 1, 128), dtype=torch.bfloat16)
    a = dict(layer=0, q=f(5, 2, 128), cu_nodes=i(3), tree_mask=torch.zeros((5, 1), dtype=torch.int64),
             max_nodes=3, k_cache=kv, v_cache=kv.view(torch.int16), block_tables=i(2, 1),
             context_lens=i(2), max_context_len=200, out=f(5, 2, 128), check=False)
    refused(h.tree_decode, a, ["cu_nodes", "block_tables", "context_lens"])
    for name in ("k_cache", "v_cache"):
        with pytest.raises(TypeError):
            h.tree_decode(**dict(a, **{name: kv.float()}))
