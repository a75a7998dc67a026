"""Cases for measuring the serving operators around the paged KV cache.

Three families, each in a plain form (elementary torch operations) and, where
`own` is true, as the library's calls:

  store / load   q/k RMSNorm + RoPE and the store of K and V rows into the
                 8-bit paged cache, read back as bf16 rows; and the read-back
                 of a cached prefix alone
  decode         one query row per sequence over the 8-bit paged cache
  tree           a tree of drafted tokens per sequence over the bf16 paged cache
  logprobs       log probability and rank of a given token per logits row,
                 with the row's entropy and its top alternatives

8-bit rows: 128 e4m3 values and one power-of-two scale per (token, kv head),
the smallest with max|x| <= 448 * scale; pages are head-major
([layer][block][kv head][token of the block][128]).
"""
import functools
import math
import os
import random
import sys

import numpy as np
import torch

own = False

D = 128        # head dim
BS = 256       # tokens per cache block
LAYERS = 2     # the cache holds two layers and the second one is used
LAYER = 1
THETA = 1e6    # RoPE base
EPS = 1e-6     # RMSNorm epsilon
SCALE = 1.0 / math.sqrt(D)
MAX_POSITION = 40960
DEV = "cuda"


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one new token of one sequence: the latency of a decode step's store
        {"name": "store_one_token", "kind": "store", "tokens": 1, "hq": 16, "hkv": 8,
         "far": 1000, "q_out": "bf16", "shape_seed": 1},
        # the new tokens of a large decode batch at far positions, some rows padding
        {"name": "store_batch_257", "kind": "store", "tokens": 257, "hq": 32, "hkv": 8,
         "far": 40000, "q_out": "bf16", "shape_seed": 2},
        # a chunk of prompt tokens, queries in the prefill's type
        {"name": "store_chunk_4096", "kind": "store", "tokens": 4096, "hq": 64, "hkv": 8,
         "far": 32000, "q_out": "f16", "shape_seed": 3},
        # a short cached prefix read back for the next chunk's attention
        {"name": "load_prefix_777", "kind": "load", "tokens": 777, "hq": 16, "hkv": 8,
         "shape_seed": 4},
        # the cached prefixes of a long prompt
        {"name": "load_prefix_65536", "kind": "load", "tokens": 65536, "hq": 32, "hkv": 8,
         "shape_seed": 5},
        # one interactive user
        {"name": "decode_one_1000", "kind": "decode", "n_seqs": 1, "hq": 16, "hkv": 8,
         "min_len": 1000, "max_len": 1000, "type": "f32", "shape_seed": 6},
        # a ragged batch, activations in bf16, eight query heads per kv head
        {"name": "decode_ragged_23", "kind": "decode", "n_seqs": 23, "hq": 64, "hkv": 8,
         "min_len": 1, "max_len": 9001, "type": "bf16", "shape_seed": 7},
        # a serving batch of long contexts
        {"name": "decode_batch_64", "kind": "decode", "n_seqs": 64, "hq": 32, "hkv": 8,
         "min_len": 1024, "max_len": 16384, "type": "f32", "shape_seed": 8},
        # one user's draft of eight tokens, activations in single precision
        {"name": "tree_one_8", "kind": "tree", "n_seqs": 1, "hq": 16, "hkv": 8, "min_len": 2000,
         "max_len": 2000, "min_nodes": 8, "max_nodes": 8, "type": "f32", "shape_seed": 9},
        # a batch of full 64-node drafts, bf16 activations
        {"name": "tree_batch_16", "kind": "tree", "n_seqs": 16, "hq": 32, "hkv": 8,
         "min_len": 700, "max_len": 8192, "min_nodes": 17, "max_nodes": 64, "type": "bf16",
         "shape_seed": 10},
        # the logits row of one sequence, in the projection's type
        {"name": "logprobs_one", "kind": "logprobs", "rows": 1, "vocab": 151936, "pad": 0,
         "top": 20, "type": "bf16", "shape_seed": 11},
        # the rows of a verification step, in a buffer of padded rows
        {"name": "logprobs_256", "kind": "logprobs", "rows": 256, "vocab": 151936, "pad": 64,
         "top": 5, "type": "f32", "shape_seed": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "load", "decode", "tree", "logprobs"])
    hq, hkv = rng.choice([(8, 8), (16, 8), (32, 8), (64, 8), (8, 2), (8, 1)])
    seed = rng.randrange(1, 1 << 20)
    if kind == "store":
        return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "hq": hq, "hkv": hkv,
                "far": _log_int(rng, 100, MAX_POSITION), "q_out": rng.choice(["bf16", "f16"]),
                "shape_seed": seed}
    if kind == "load":
        return {"kind": kind, "tokens": _log_int(rng, 1, 65536), "hq": hq, "hkv": hkv,
                "shape_seed": seed}
    if kind == "decode":
        n = _log_int(rng, 1, 64)
        top = _log_int(rng, 16, 16384)
        return {"kind": kind, "n_seqs": n, "hq": hq, "hkv": hkv,
                "min_len": rng.choice([0, 1, top // 2 + 1, top]), "max_len": top,
                "type": rng.choice(["f32", "bf16"]), "shape_seed": seed}
    if kind == "tree":
        n = _log_int(rng, 1, 16)
        nodes = _log_int(rng, 1, 64)
        top = nodes + _log_int(rng, 16, 8000)
        return {"kind": kind, "n_seqs": n, "hq": min(hq, 32), "hkv": hkv,
                "min_len": rng.choice([nodes, top // 2 + nodes // 2 + 1, top]), "max_len": top,
                "min_nodes": rng.choice([1, nodes]), "max_nodes": nodes,
                "type": rng.choice(["f32", "bf16"]), "shape_seed": seed}
    rows = _log_int(rng, 1, 256)
    return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 1000, 151936),
            "pad": rng.choice([0, 1, 64]), "top": rng.randrange(1, 21),
            "type": rng.choice(["f32", "bf16"]), "shape_seed": seed}


def _lens(case):
    """Context lengths of a case's sequences, log-uniform over its range."""
    r = random.Random(case["shape_seed"])
    lo, hi = case["min_len"], case["max_len"]
    lens = [min(hi, max(lo, int(round(math.exp(r.uniform(math.log(max(lo, 1)), math.log(hi)))))))
            for _ in range(case["n_seqs"])]
    lens[r.randrange(len(lens))] = hi
    if lo == 0 and len(lens) > 1:
        lens[lens.index(hi) - 1] = 0  # an empty sequence in a padded batch
    return lens


def _nodes(case):
    r = random.Random(case["shape_seed"] + 1)
    return [r.randint(case["min_nodes"], case["max_nodes"]) for _ in range(case["n_seqs"])]


def work(case):
    k = case["kind"]
    if k == "store":
        t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        # rows in, the rotation's row, queries out, 8-bit rows written and
        # read again, bf16 rows out
        b = t * ((hq + 2 * hkv) * D * 4 + D * 4 + hq * D * 2 + 2 * hkv * (2 * (D + 4) + D * 2))
        return {"bytes": b, "flops": t * (hq + 2 * hkv) * D * 10}
    if k == "load":
        rows = case["tokens"] * 2 * case["hkv"]
        return {"bytes": rows * (D + 4 + D * 2), "flops": rows * D}
    if k == "decode":
        n, el = sum(_lens(case)), {"f32": 4, "bf16": 2}[case["type"]]
        return {"bytes": n * case["hkv"] * 2 * (D + 4) + 2 * case["n_seqs"] * case["hq"] * D * el,
                "flops": 4 * n * case["hq"] * D}
    if k == "tree":
        lens, nodes, el = _lens(case), _nodes(case), {"f32": 4, "bf16": 2}[case["type"]]
        pairs = sum(a * b for a, b in zip(lens, nodes))
        return {"bytes": sum(lens) * case["hkv"] * 2 * D * 2 +
                sum(nodes) * (2 * case["hq"] * D * el + 8),
                "flops": 4 * pairs * case["hq"] * D}
    el = {"f32": 4, "bf16": 2}[case["type"]]
    n = case["rows"] * case["vocab"]
    return {"bytes": n * el + case["rows"] * (16 + 8 * case["top"]), "flops": 6 * n}


# ---------------------------------------------------------------- inputs

def _dtype(name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


@functools.lru_cache(maxsize=6)
def _handle(hq, hkv, blocks, max_seqs, max_context, max_position):
    """The handle that a program keeps for its model and cache."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "nano-vllm.cpp_b200", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nvattn
    return nvattn.Handle(nvattn.qwen3_config(
        n_layer=LAYERS, n_q_heads=hq, n_kv_heads=hkv, num_blocks=blocks, max_seqs=max_seqs,
        max_context=max_context, max_position=max_position, rope_theta=THETA, rms_eps=EPS,
        scale=SCALE))


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _quantise(x):
    """Rows [..., 128] -> (e4m3 values, power-of-two scales [...])."""
    frac, exp = torch.frexp(x.abs().amax(-1))
    e = torch.where(frac <= 0.875, exp - 9, exp - 8)
    e = torch.where(frac == 0, torch.zeros_like(e), e.clamp(min=-100))
    scale = torch.ldexp(torch.ones_like(frac), e)
    return (x / scale[..., None]).float().to(torch.float8_e4m3fn), scale


def _q8_cache(g, blocks, hkv):
    """An 8-bit cache full of rows, and NaN patterns in the layer not used."""
    payload = torch.full((LAYERS, blocks, hkv, BS, D), 0x7F, dtype=torch.uint8, device=DEV)
    scale = torch.full((LAYERS, blocks, hkv, BS), float("nan"), device=DEV)
    for b in range(0, blocks, 256):  # in pieces, for the memory of the f32 rows
        n = min(256, blocks - b)
        x = _randn(g, n, hkv, BS, D) * (0.3 + 1.4 * torch.rand((1, hkv, 1, D), generator=g,
                                                              device=DEV))
        p, s = _quantise(x)
        payload[LAYER, b:b + n] = p.view(torch.uint8)
        scale[LAYER, b:b + n] = s
    return payload, scale


def _tables(seed, lens):
    """Block tables over a shuffled pool; unused entries are -1."""
    need = [(n + BS - 1) // BS for n in lens]
    pool = sum(need) + 2
    perm = np.random.RandomState(seed % (1 << 31)).permutation(pool).astype(np.int32)
    table = np.full((len(lens), max(max(need), 1)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n]
        at += n
    return torch.from_numpy(table).to(DEV), pool


def _past_the_end(table, lens):
    """(block, offset) of the slots behind each sequence's last token."""
    t = table.cpu().numpy()
    bl, of = [], []
    for i, n in enumerate(lens):
        for o in range(n % BS, BS) if n % BS else ():
            bl.append(int(t[i, n // BS]))
            of.append(o)
    return torch.tensor(bl, dtype=torch.long, device=DEV), torch.tensor(of, dtype=torch.long,
                                                                      device=DEV)


def _tree_masks(seed, nodes):
    """Ancestor masks of random trees: bit j of node i's word is set where i
    descends from j or is j."""
    r = random.Random(seed)
    words = []
    for n in nodes:
        own_words = []
        for i in range(n):
            up = r.randrange(max(-1, i - 8), i) if i else -1
            own_words.append((own_words[up] if up >= 0 else 0) | (1 << i))
        words += own_words
    return torch.from_numpy(np.array(words, np.uint64).view(np.int64).reshape(-1, 1)).to(DEV)


def _angles(positions):
    """RoPE angles [tokens][64]: the position times base^(-2/128), again and
    again in single precision, as the model's rotation is defined."""
    step = np.float32(np.float32(THETA) ** np.float32(-2.0 / D))
    a = np.empty((len(positions), D // 2), np.float32)
    a[:, 0] = positions
    a[:, 1:] = step
    return np.multiply.accumulate(a, axis=1, dtype=np.float32)


def prepare(case, seed):
    g = _gen(seed)
    k = case["kind"]
    hq, hkv = case.get("hq"), case.get("hkv")
    s = {"case": case, "kind": k}
    if k == "store":
        t = case["tokens"]
        r = np.random.RandomState(seed % (1 << 31))
        blocks = (t + BS - 1) // BS + 1
        slots = r.permutation(blocks * BS)[:t].astype(np.int32)
        slots[r.rand(t) < 0.03] = -1  # padding rows
        positions = r.randint(0, case["far"], t).astype(np.int32)
        s.update(
            q=_randn(g, t, hq, D) * 3, k=_randn(g, t, hkv, D) * 2, v=_randn(g, t, hkv, D),
            qw=(1 + 0.2 * _randn(g, D)).bfloat16(), kw=(1 + 0.2 * _randn(g, D)).bfloat16(),
            positions=torch.from_numpy(positions).to(DEV),
            angles=torch.from_numpy(_angles(positions)).to(DEV),
            slots=torch.from_numpy(slots).to(DEV),
            kp=torch.zeros((LAYERS, blocks, hkv, BS, D), dtype=torch.uint8, device=DEV),
            ks=torch.zeros((LAYERS, blocks, hkv, BS), device=DEV),
            q_out=torch.empty((t, hq, D), dtype=_dtype(case["q_out"]), device=DEV),
            k_out=torch.empty((t, hkv, D), dtype=torch.bfloat16, device=DEV),
            v_out=torch.empty((t, hkv, D), dtype=torch.bfloat16, device=DEV))
        s.update(vp=torch.zeros_like(s["kp"]), vs=torch.zeros_like(s["ks"]))
        if own:
            s["h"] = _handle(hq, hkv, blocks, 1, BS, MAX_POSITION)
    elif k == "load":
        t = case["tokens"]
        r = np.random.RandomState(seed % (1 << 31))
        blocks = (t + BS - 1) // BS + 2
        table = r.permutation(blocks)
        at = np.arange(t) + r.randint(0, BS)  # a run of positions that starts inside a block
        slots = (table[at // BS] * BS + at % BS).astype(np.int32)
        kp, ks = _q8_cache(g, blocks, hkv)
        vp, vs = _q8_cache(g, blocks, hkv)
        s.update(kp=kp, ks=ks, vp=vp, vs=vs, slots=torch.from_numpy(slots).to(DEV),
                 k_out=torch.empty((t, hkv, D), dtype=torch.bfloat16, device=DEV),
                 v_out=torch.empty((t, hkv, D), dtype=torch.bfloat16, device=DEV))
        if own:
            s["h"] = _handle(hq, hkv, blocks, 1, BS, 1)
    elif k == "decode":
        lens = _lens(case)
        table, pool = _tables(seed, lens)
        kp, ks = _q8_cache(g, pool, hkv)
        vp, vs = _q8_cache(g, pool, hkv)
        b, o = _past_the_end(table, lens)
        for p, c in ((kp, ks), (vp, vs)):  # what a cache holds behind a sequence: anything
            p[LAYER, b, :, o] = 0x7F
            c[LAYER, b, :, o] = float("nan")
        q = (_randn(g, len(lens), hq, D) * 2).to(_dtype(case["type"]))
        s.update(kp=kp, ks=ks, vp=vp, vs=vs, table=table, q=q, out=torch.empty_like(q),
                 max_len=max(lens), lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if own:
            s["h"] = _handle(hq, hkv, pool, len(lens), max(max(lens), 1), 1)
    elif k == "tree":
        lens, nodes = _lens(case), _nodes(case)
        table, pool = _tables(seed, lens)
        b, o = _past_the_end(table, lens)
        for name in ("k", "v"):
            c = torch.full((LAYERS, pool * BS, hkv, D), float("nan"), dtype=torch.bfloat16,
                           device=DEV)
            c[LAYER] = _randn(g, pool * BS, hkv, D).bfloat16()
            c[LAYER, b * BS + o] = float("nan")
            s[name + "c"] = c
        q = (_randn(g, sum(nodes), hq, D) * 2).to(_dtype(case["type"]))
        cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        s.update(table=table, q=q, out=torch.empty_like(q), max_len=max(lens),
                 max_nodes=max(nodes), mask=_tree_masks(seed, nodes),
                 cu=torch.from_numpy(cu).to(DEV),
                 lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        if own:
            s["h"] = _handle(hq, hkv, pool, len(lens), max(lens), 1)
    else:
        n, v, top = case["rows"], case["vocab"], case["top"]
        logits = (_randn(g, n, v + case["pad"]) * 3).to(_dtype(case["type"]))[:, :v]
        logits[:, v - v // 50:] = float("-inf")  # the part of the vocabulary ruled out
        tokens = torch.randint(0, v - v // 50, (n,), generator=g, device=DEV)
        best = logits.float().argmax(-1)
        tokens = torch.where(torch.rand((n,), generator=g, device=DEV) < 0.5, best, tokens)
        s.update(logits=logits, tokens=tokens.to(torch.int32),
                 logprobs=torch.empty(n, device=DEV), entropy=torch.empty(n, device=DEV),
                 ranks=torch.empty(n, dtype=torch.int32, device=DEV),
                 top_ids=torch.empty((n, top), dtype=torch.int32, device=DEV),
                 top_logprobs=torch.empty((n, top), device=DEV))
        if own:
            s["h"] = _handle(16, 8, 1, 256, BS, 1)
    return s


# ---------------------------------------------------------------- plain forms

def _norm_rope(x, w, cos, sin):
    x = x.double()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _rows_of(payload, scale, slots):
    """Rows of the given slots as bf16; zeros where the slot is negative."""
    at = slots.clamp(min=0).long()
    p = payload[LAYER].view(torch.float8_e4m3fn)[at // BS, :, at % BS].float()
    y = p * scale[LAYER][at // BS, :, at % BS][..., None]
    return torch.where((slots >= 0)[:, None, None], y, torch.zeros_like(y)).bfloat16()


def _plain_store(s):
    # 64 bits up to the rounding to 8 bits, where values next to a border count
    cos, sin = s["angles"].double().cos()[:, None], s["angles"].double().sin()[:, None]
    s["q_out"].copy_(_norm_rope(s["q"], s["qw"], cos, sin))
    at = s["slots"][s["slots"] >= 0].long()
    for x, p, c in ((_norm_rope(s["k"], s["kw"], cos, sin), s["kp"], s["ks"]),
                    (s["v"].double(), s["vp"], s["vs"])):
        rows, scale = _quantise(x[s["slots"] >= 0])
        p[LAYER][at // BS, :, at % BS] = rows.view(torch.uint8)
        c[LAYER][at // BS, :, at % BS] = scale.float()
    return (s["q_out"], _rows_of(s["kp"], s["ks"], s["slots"]),
            _rows_of(s["vp"], s["vs"], s["slots"]))


def _softmax_v(x, keep, v):
    """softmax over the last axis of x where `keep`, times v; zeros for an
    empty row."""
    x = torch.where(keep, x, torch.full_like(x, float("-inf")))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    total = e.sum(-1, keepdim=True)
    return torch.matmul(e / torch.where(total > 0, total, torch.ones_like(total)), v)


def _pages_q8(payload, scale, table, inside):
    at = table.clamp(min=0).long()
    x = payload[LAYER].view(torch.float8_e4m3fn)[at].float() * scale[LAYER][at][..., None]
    b, n, h = x.shape[:3]
    x = x.permute(0, 2, 1, 3, 4).reshape(b, h, n * BS, D)
    return torch.where(inside[:, None, :, None], x, torch.zeros_like(x))


def _plain_decode(s):
    n, hq, _ = s["q"].shape
    hkv = s["kp"].shape[2]
    inside = torch.arange(s["table"].shape[1] * BS, device=DEV)[None] < s["lens"][:, None]
    k = _pages_q8(s["kp"], s["ks"], s["table"], inside)
    v = _pages_q8(s["vp"], s["vs"], s["table"], inside)
    q = s["q"].float().view(n, hkv, hq // hkv, D)
    x = torch.matmul(q, k.transpose(-1, -2)) * SCALE
    return _softmax_v(x, inside[:, None, None], v).view(n, hq, D).to(s["q"].dtype)


def _plain_tree(s):
    n, hq, hkv = s["lens"].shape[0], s["q"].shape[1], s["kc"].shape[2]
    N, L = s["max_nodes"], s["table"].shape[1] * BS
    counts = (s["cu"][1:] - s["cu"][:-1]).long()
    key = torch.arange(L, device=DEV)[None]
    inside = key < s["lens"][:, None]
    at = s["table"].clamp(min=0).long()[..., None] * BS + torch.arange(BS, device=DEV)

    def pages(c):
        x = c[LAYER][at.view(n, L)].permute(0, 2, 1, 3).float()
        return torch.where(inside[:, None, :, None], x, torch.zeros_like(x))

    node = torch.arange(N, device=DEV)[None]
    real = node < counts[:, None]                                  # [n][N]
    row = torch.where(real, s["cu"][:-1, None].long() + node, torch.zeros_like(node))
    rel = key - (s["lens"].long() - counts)[:, None]               # position among the nodes
    bits = (s["mask"][row, 0][:, :, None] >> rel.clamp(0, 63)[:, None]) & 1
    keep = inside[:, None] & ((rel[:, None] < 0) | (bits == 1))    # [n][N][L]
    g = hq // hkv
    q = s["q"].float()[row].view(n, N, hkv, g, D).permute(0, 2, 1, 3, 4).reshape(n, hkv, N * g, D)
    x = torch.matmul(q, pages(s["kc"]).transpose(-1, -2)) * SCALE
    o = _softmax_v(x, keep.repeat_interleave(g, 1)[:, None], pages(s["vc"]))
    o = o.view(n, hkv, N, g, D).permute(0, 2, 1, 3, 4).reshape(n, N, hq, D)
    return o[real].to(s["q"].dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    t = s["tokens"].long()[:, None]
    m = x.amax(-1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total[:, 0] - torch.where(e > 0, e * z, torch.zeros_like(e)).sum(-1) / total[:, 0]
    xt = x.gather(1, t)
    ids = torch.arange(x.shape[1], device=DEV)[None]
    rank = ((x > xt) | ((x == xt) & (ids < t))).sum(-1)
    # a stable sort keeps the lowest id first among equals
    val, idx = torch.sort(x, dim=-1, descending=True, stable=True)
    top = s["top_ids"].shape[1]
    return ((xt - m - log_total)[:, 0], entropy, rank.int(), idx[:, :top].int(),
            val[:, :top] - m - log_total)


# ---------------------------------------------------------------- one pass

def run(s):
    k = s["kind"]
    if own:
        h, st = s["h"], torch.cuda.current_stream()
        if k == "store":
            h.kv_store_q8(LAYER, s["q"], s["k"], s["v"], s["qw"], s["kw"], s["positions"],
                          s["slots"], s["q_out"], s["kp"], s["ks"], s["vp"], s["vs"], stream=st)
            h.kv_load_q8(LAYER, s["slots"], s["kp"], s["ks"], s["vp"], s["vs"], s["k_out"],
                         s["v_out"], stream=st)
            return s["q_out"], s["k_out"], s["v_out"]
        if k == "load":
            h.kv_load_q8(LAYER, s["slots"], s["kp"], s["ks"], s["vp"], s["vs"], s["k_out"],
                         s["v_out"], stream=st)
            return s["k_out"], s["v_out"]
        if k == "decode":
            h.decode_q8(LAYER, s["q"], s["kp"], s["ks"], s["vp"], s["vs"], s["table"],
                        s["lens"], s["max_len"], s["out"], stream=st)
            return s["out"]
        if k == "tree":
            h.tree_decode(LAYER, s["q"], s["cu"], s["mask"], s["max_nodes"], s["kc"], s["vc"],
                          s["table"], s["lens"], s["max_len"], s["out"], stream=st)
            return s["out"]
        h.token_logprobs(s["logits"], s["tokens"], s["logprobs"], s["entropy"], s["ranks"],
                         s["top_ids"], s["top_logprobs"], stream=st)
        return s["logprobs"], s["entropy"], s["ranks"], s["top_ids"], s["top_logprobs"]
    if k == "store":
        return _plain_store(s)
    if k == "load":
        return _rows_of(s["kp"], s["ks"], s["slots"]), _rows_of(s["vp"], s["vs"], s["slots"])
    if k == "decode":
        return _plain_decode(s)
    if k == "tree":
        return _plain_tree(s)
    return _plain_logprobs(s)


# ---------------------------------------------------------------- in 64 bits

def _exact_norm_rope(x, w, angles):
    x, w = x.double(), w.double()
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / D + EPS) * w
    z = torch.complex(y[..., :D // 2], y[..., D // 2:])
    z = z * torch.polar(torch.ones_like(angles, dtype=torch.float64), angles.double())[:, None]
    return torch.cat([z.real, z.imag], -1)


def _exact_round_trip(x, slots):
    """x to 8 bits and back, by the grid's step at each value."""
    a = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(a / 448)).clamp(min=-100)
    e = torch.where(a > 448 * 2.0 ** e, e + 1, e)
    e = torch.where(a <= 448 * 2.0 ** (e - 1), e - 1, e)
    y = x / 2.0 ** e
    step = 2.0 ** (torch.frexp(y)[1].clamp(min=-5) - 4).double()  # 3 bits behind the first one
    y = torch.round(y / step) * step * 2.0 ** e
    return torch.where((slots >= 0)[:, None, None], y, torch.zeros_like(y))


def exact(case, seed):
    s = prepare(case, seed)
    k = case["kind"]
    if k == "store":
        kk = _exact_norm_rope(s["k"], s["kw"], s["angles"])
        return (_exact_norm_rope(s["q"], s["qw"], s["angles"]),
                _exact_round_trip(kk, s["slots"]), _exact_round_trip(s["v"].double(), s["slots"]))
    if k == "load":
        out = []
        for p, c in ((s["kp"], s["ks"]), (s["vp"], s["vs"])):
            flat = p[LAYER].view(torch.float8_e4m3fn).double().transpose(1, 2).reshape(-1, case["hkv"], D)
            sc = c[LAYER].double().transpose(1, 2).reshape(-1, case["hkv"])
            i = s["slots"].long()
            out.append(flat[i] * sc[i][..., None])
        return tuple(out)
    if k in ("decode", "tree"):
        tree = k == "tree"
        lens = [int(n) for n in s["lens"].tolist()]
        cu = s["cu"].tolist() if tree else list(range(len(lens) + 1))
        hkv = case["hkv"]
        g = case["hq"] // hkv
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for i, n in enumerate(lens):
            if not n:
                continue
            pos = torch.arange(n, device=DEV)
            blk, off = s["table"][i].long()[pos // BS], pos % BS
            if tree:
                kd, vd = (c[LAYER][blk * BS + off].double() for c in (s["kc"], s["vc"]))
            else:
                kd, vd = (p[LAYER].view(torch.float8_e4m3fn)[blk, :, off].double() *
                          c[LAYER][blk, :, off].double()[..., None]
                          for p, c in ((s["kp"], s["ks"]), (s["vp"], s["vs"])))
            nodes = cu[i + 1] - cu[i]
            q = s["q"][cu[i]:cu[i + 1]].double()
            for h in range(hkv):
                x = torch.einsum("ngd,td->ngt", q[:, h * g:(h + 1) * g], kd[:, h]) / math.sqrt(D)
                if tree:
                    first = n - nodes
                    w = s["mask"][cu[i]:cu[i + 1], 0]
                    seen = torch.stack([(w >> j) & 1 for j in range(nodes)], 1).bool()
                    x[:, :, first:] = x[:, :, first:].masked_fill(~seen[:, None], float("-inf"))
                out[cu[i]:cu[i + 1], h * g:(h + 1) * g] = torch.einsum(
                    "ngt,td->ngd", torch.softmax(x, -1), vd[:, h])
        return out
    x = s["logits"].double()
    lp = torch.log_softmax(x, -1)
    p = torch.exp(lp)
    entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    top = torch.topk(lp, case["top"], -1)[0]
    return lp.gather(1, s["tokens"].long()[:, None])[:, 0], entropy, None, None, top
