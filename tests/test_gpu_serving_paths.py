"""The 8-bit cache, the draft-tree attention and the log-probabilities used
together, as a serving engine would."""
import numpy as np
import pytest

import nvattn
import oracle as O
import q8_util as Q
from gpu_util import dev, handle

pytestmark = pytest.mark.gpu


def test_model_steps_over_the_8_bit_cache(cuda):
    """Three decode steps of the model harness with kv_cache="q8": every
    layer's attention against 64-bit attention over the rows that the cache
    holds (read back), and the log-probabilities of the chosen tokens against
    the logits' own."""
    import torch
    import model_runner as MR
    device = torch.device("cuda:0")
    shape = MR.Qwen3Shape(n_layer=2, vocab=5003)
    w = MR.Qwen3Weights(shape, device, seed=21, norm_mean=1.0)
    lens = np.array([255, 511, 700, 1], np.int64)
    steps, B = 3, len(lens)
    num_blocks, max_blocks = int(((lens + steps + 255) // 256).sum()) + 2, 4
    run = MR.DecodeRunner(shape, w, num_blocks, B, max_blocks, device, kv_cache="q8")
    run.allocate(B)
    rng = np.random.default_rng(22)
    cache = Q.Q8Cache(num_blocks, shape.n_kv_heads, shape.n_layer)
    for layer in range(shape.n_layer):
        k, v = rng.standard_normal((2, num_blocks * 256, shape.n_kv_heads, 128), dtype=np.float32)
        cache.put(layer, np.arange(num_blocks * 256), k, v)
    for t, a in zip(run.q8_cache, (cache.kp, cache.ks, cache.vp, cache.vs)):
        t.copy_(torch.from_numpy(a))
    G = shape.n_q_heads // shape.n_kv_heads
    layers = []

    def checked(layer, q, k, v, stream=None):
        got = run.library_attention_q8(layer, q, k, v, stream).cpu().numpy()
        ctx, bt = run.bufs["ctx"].cpu().numpy(), run.bufs["bt"].cpu().numpy()
        qn = run.bufs["q"].cpu().numpy()
        for s, n in enumerate(ctx):
            slots = dev(Q.slots_of(bt[s], n, 256).astype(np.int32))
            rows = torch.empty((2, n, shape.n_kv_heads, 128), device=device)
            run.h.kv_load_q8(layer, slots, *run.q8_cache, rows[0], rows[1])
            kk, vv = rows.cpu().numpy()
            # the step's own row is the last: within e4m3's half step of the raw v
            assert np.allclose(vv[-1], v[s].cpu().numpy(), rtol=2.0 ** -4,
                               atol=np.abs(vv[-1]).max() * 2.0 ** -18)
            for hd in range(shape.n_kv_heads):
                hs = slice(hd * G, (hd + 1) * G)
                want, tol = Q.attend(qn[s, hs], kk[:, hd], vv[:, hd])
                Q.check(got[s, hs], want, tol, False)
        layers.append(layer)
        return run.bufs["attn"]

    run.attention = checked
    tables = MR.BlockTables(lens, num_blocks, max_blocks, seed=23)
    tokens = rng.integers(0, shape.vocab, B)
    for step in range(steps):
        run.set_inputs(tokens, tables)
        tokens = run.forward().cpu().numpy()
        lp = run.token_logprobs(top_k=3)
        run.h.check_device(f"step {step}")
        x = run.bufs["logits"].double()
        want = torch.log_softmax(x, -1)
        assert (lp["ranks"] == 0).all() and (lp["top_ids"][:, 0] == run.bufs["next"]).all()
        got = lp["top_logprobs"].double()
        assert torch.allclose(got, want.gather(1, lp["top_ids"].long()), atol=2e-5)
        assert torch.equal(lp["logprobs"], lp["top_logprobs"][:, 0])
        assert torch.allclose(lp["entropy"].double(), -(want.exp() * want).sum(-1), atol=1e-4)
        tables.append_token()
    assert layers == list(range(shape.n_layer)) * steps
    run.close()


@pytest.mark.parametrize("bf16", [False, True])
def test_verification_step_of_a_drafted_tree(cuda, bf16):
    """Drafts of two sequences: their K/V stored behind the prefixes at RoPE
    positions given by the nodes' depths, one tree attention, logits,
    log-probabilities of each node's drafted children.  Every node's output
    equals that of plain decodes of its root-to-node path, token by token, with
    the same rows stored in order."""
    import torch
    rng = np.random.default_rng(31)
    Hq, Hkv, G = 32, 8, 4
    prefix = [300, 77]
    parents = [[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 2]]
    nb, B = 8, 2
    nodes = [len(p) for p in parents]
    T = sum(nodes)
    lens = np.array([a + b for a, b in zip(prefix, nodes)], np.int32)
    bt = Q.tables(rng, lens, 256, nb)
    h = handle(Hq, Hkv, nb + 2, max_seqs=4, max_context=512, max_position=600)
    kc = np.zeros((1, (nb + 2) * 256, Hkv, 128), np.uint16)
    vc = kc.copy()
    for s in range(B):
        sl = Q.slots_of(bt[s], prefix[s], 256)
        kc[0, sl] = O.f32_to_bf16(rng.standard_normal((prefix[s], Hkv, 128), dtype=np.float32))
        vc[0, sl] = O.f32_to_bf16(rng.standard_normal((prefix[s], Hkv, 128), dtype=np.float32))
    q = rng.standard_normal((T, Hq, 128), dtype=np.float32)
    k = rng.standard_normal((T, Hkv, 128), dtype=np.float32)
    v = rng.standard_normal((T, Hkv, 128), dtype=np.float32)
    w = O.f32_to_bf16((1 + 0.1 * rng.standard_normal(128)).astype(np.float32))
    depth, pos, slots, mask, paths = [], [], [], [], []
    for s in range(B):
        for i, up in enumerate(parents[s]):
            path = (paths[-i + up] if i and up >= 0 else []) + [i] if up >= 0 else [i]
            paths.append(path)
            pos.append(prefix[s] + len(path) - 1)
            slots.append(int(Q.slots_of(bt[s], int(lens[s]), 256)[prefix[s] + i]))
            mask.append(sum(1 << j for j in path))
    cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    dk, dv = dev(kc), dev(vc)
    t = torch.bfloat16 if bf16 else torch.float32
    qn = torch.empty((T, Hq, 128), dtype=t, device="cuda")
    args = (dev(w), dev(w))
    h.kv_store(0, dev(q), dev(k), dev(v), *args, dev(np.array(pos, np.int32)),
               dev(np.array(slots, np.int32)), qn, dk, dv)
    out = torch.empty_like(qn)
    h.tree_decode(0, qn, dev(cu), dev(np.array(mask, np.uint64).view(np.int64).reshape(-1, 1)),
                  max(nodes), dk, dv, dev(bt), dev(lens), int(lens.max()), out)
    h.check_device()
    got = out.float().cpu().numpy()

    # the same by decodes: the path's rows one after another behind the prefix
    for s in range(B):
        for i in range(nodes[s]):
            path = [cu[s] + j for j in paths[cu[s] + i]]
            lk, lv = dev(kc), dev(vc)
            n = prefix[s] + len(path)
            line = Q.slots_of(bt[s], n, 256)[prefix[s]:].astype(np.int32)
            q1 = torch.empty((len(path), Hq, 128), device="cuda")
            h.kv_store(0, dev(q[path]), dev(k[path]), dev(v[path]), *args,
                       dev(np.arange(prefix[s], n, dtype=np.int32)), dev(line), q1, lk, lv)
            last = q1[-1:].to(t).float().contiguous()
            o1 = torch.empty((1, Hq, 128), device="cuda")
            h.decode(0, last, lk, lv, dev(bt[s:s + 1]), dev(np.array([n], np.int32)), n, o1)
            want = o1[0].cpu().numpy()
            # the decode carries 16 bits of queries and weights; scores are at
            # most |q||k| / sqrt(128) ~ 14: 2 * 14 * 2^-16 of the values' size,
            # and the bf16 output half a step
            tol = 2 * 14 * 2.0 ** -16 * 4 + (2.0 ** -8 * np.abs(want) if bf16 else 0)
            assert (np.abs(got[cu[s] + i] - want) <= tol).all(), (s, i)

    # the target's opinion of each drafted child
    proj = torch.randn((Hq * 128, 1009), generator=torch.Generator(device="cuda").manual_seed(3),
                       device="cuda") * 0.05
    logits = out.float().reshape(T, -1) @ proj
    child = dev(rng.integers(0, 1009, T).astype(np.int32))
    lp, rank = torch.empty(T, device="cuda"), torch.empty(T, dtype=torch.int32, device="cuda")
    h.token_logprobs(logits, child, lp, None, rank)
    h.check_device()
    want = torch.log_softmax(logits.double(), -1).gather(1, child.long()[:, None])[:, 0]
    assert torch.allclose(lp.double(), want, atol=2e-5)
    x = logits.gather(1, child.long()[:, None])
    assert torch.equal(rank, (logits > x).sum(-1).int())  # (no ties among random logits)


def test_chunked_prompt_over_the_8_bit_cache(cuda):
    """A prompt prefilled in two chunks with an 8-bit cache: each chunk's rows
    stored in 8 bits and kept in f16 for its own attention, the first chunk's
    rows read back into a BF16 cache that the second chunk's prefill attends."""
    import torch
    rng = np.random.default_rng(41)
    Hq, Hkv, G = 16, 8, 2
    n0, n1 = 256, 200
    n = n0 + n1
    q = rng.standard_normal((n, Hq, 128), dtype=np.float32)
    k = rng.standard_normal((n, Hkv, 128), dtype=np.float32)
    v = rng.standard_normal((n, Hkv, 128), dtype=np.float32)
    w = O.f32_to_bf16((1 + 0.1 * rng.standard_normal(128)).astype(np.float32))
    nb = 3
    h = handle(Hq, Hkv, nb, max_seqs=1, max_context=512, max_position=512)
    bt = np.array([[2, 0]], np.int32)
    slots = Q.slots_of(bt[0], n, 256).astype(np.int32)
    d = Q.Q8Cache(nb, Hkv).dev()
    kc = torch.zeros((nb * 256, Hkv, 128), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    outs = []
    for a, b in ((0, n0), (n0, n)):
        m = b - a
        qn = torch.empty((m, Hq, 128), dtype=torch.float16, device="cuda")
        kr = torch.empty((m, Hkv, 128), dtype=torch.float16, device="cuda")
        vr = torch.empty_like(kr)
        h.kv_store_q8(0, dev(q[a:b]), dev(k[a:b]), dev(v[a:b]), dev(w), dev(w),
                      dev(np.arange(a, b, dtype=np.int32)), dev(slots[a:b]), qn, *d, k_rows=kr,
                      v_rows=vr)
        if a:
            block = dev(np.arange(2 * 256, 3 * 256, dtype=np.int32))  # the prefix's block
            h.kv_load_q8(0, block, *d, kc[512:768], vc[512:768])
        out = torch.empty((m, Hq, 128), device="cuda")
        h.prefill(0, qn, dev(np.array([0, m], np.int32)), dev(np.array([a], np.int32)),
                  dev(np.array([b], np.int32)), dev(bt), m, kc, vc, out, k_rows=kr, v_rows=vr)
        h.check_device()
        outs.append((qn.float().cpu().numpy(), kr.float().cpu().numpy(), vr.float().cpu().numpy(),
                     out.cpu().numpy()))
    pre = torch.empty((2, n0, Hkv, 128), device="cuda")
    h.kv_load_q8(0, dev(slots[:n0]), *d, pre[0], pre[1])
    pre = pre.cpu().numpy()
    # the prefix in 8 bits is within half a step of the chunk's f16 rows
    assert np.allclose(pre[0], outs[0][1], rtol=2.0 ** -4 + 2.0 ** -11, atol=0.02)
    for i, (a, b) in enumerate(((0, n0), (n0, n))):
        qn, kr, vr, got = outs[i]
        kk = kr if i == 0 else np.concatenate([pre[0], kr])
        vv = vr if i == 0 else np.concatenate([pre[1], vr])
        keep = np.arange(b)[None] <= np.arange(a, b)[:, None]
        for hd in range(Hkv):
            for g in range(G):
                want, _ = Q.attend(qn[:, hd * G + g], kk[:, hd], vv[:, hd], keep)
                # the prefill's own bars (f16 probabilities)
                mx, mr = O.err_stats(got[:, hd * G + g], want.astype(np.float32))
                assert mx <= 2e-2 and mr <= 1e-3, (i, hd, mx, mr)
