"""Cases of the serving-path operators: the 4-bit paged KV cache (storing and reading rows, decode attention over
it, eviction by accumulated attention weight) and the log-probabilities of given tokens with entropy and the top
alternatives.

``listed()`` names the measured cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` makes one
case's inputs on the GPU, ``run`` is one pass (the framework's kernels where ``own`` is true, elementary torch
operations in fp32 otherwise), ``work`` counts the bytes and operations a pass cannot do without and ``exact`` is
the operators' definition in 64 bits.

A block of the 4-bit cache holds 16 tokens of one KV head: for each group of ``min(D, 64)`` dimensions the codes
``[16][group / 2]`` bytes (element 2i in the low half of byte i, 2i + 1 in the high half), then for each group
``[16][2]`` bf16 (scale, minimum).  An element stands for ``minimum + scale * code``.
"""

import math

import torch

own = False

BLOCK = 16


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the keys and values of one decoding step, 64 sequences, written into their slots (latency counts)
        {"name": "store_step_64", "op": "store", "N": 64, "Hkv": 8, "D": 64},
        # a batch of long prompts written after prefill, 8 KV heads of 128
        {"name": "store_prompt_32768", "op": "store", "N": 32768, "Hkv": 8, "D": 128},
        # one chat sequence, the 1B configuration's heads: the smallest call, latency counts
        {"name": "decode_one_777", "op": "decode", "B": 1, "T": 777, "Hkv": 8, "G": 4, "D": 64, "window": 0,
         "softcap": 0.0, "empty": 0, "weights": False},
        # a full serving batch of the 1B configuration, ragged contexts up to its block size
        {"name": "decode_batch_64x4096", "op": "decode", "B": 64, "T": 4096, "Hkv": 8, "G": 4, "D": 64, "window": 0,
         "softcap": 0.0, "empty": 3, "weights": False},
        # the 8B configuration at its block size, the largest call
        {"name": "decode_batch_32x8192", "op": "decode", "B": 32, "T": 8192, "Hkv": 8, "G": 4, "D": 128, "window": 0,
         "softcap": 0.0, "empty": 0, "weights": False},
        # one very long context: few rows, the work has to be split along the cache
        {"name": "decode_long_100001", "op": "decode", "B": 1, "T": 100001, "Hkv": 8, "G": 4, "D": 128, "window": 0,
         "softcap": 0.0, "empty": 0, "weights": False},
        # decoding that also accumulates each cached token's attention weight, as eviction needs it
        {"name": "decode_weights_24x5000", "op": "decode", "B": 24, "T": 5000, "Hkv": 8, "G": 4, "D": 128, "window": 0,
         "softcap": 0.0, "empty": 0, "weights": True},
        # caches of a serving batch cut from up to 4096 tokens to 1024
        {"name": "evict_16x4096_to_1024", "op": "evict", "B": 16, "T": 4096, "Hkv": 8, "D": 128, "keep": 1024,
         "recent": 128, "sink": 4},
        # one long cache cut by a quarter
        {"name": "evict_1x40000_to_30000", "op": "evict", "B": 1, "T": 40000, "Hkv": 8, "D": 64, "keep": 30000,
         "recent": 512, "sink": 4},
        # the logits of one serving step: the sampled tokens' log-probs with five alternatives each
        {"name": "logprob_step_48_top5", "op": "logprob", "N": 48, "V": 128256, "dtype": "bf16", "k": 5, "masked": 0,
         "grad": False},
        # a response scored from fp32 logits of the default vocabulary with 20 alternatives per token
        {"name": "logprob_score_1000_top20", "op": "logprob", "N": 1000, "V": 65536, "dtype": "fp32", "k": 20,
         "masked": 17, "grad": False},
        # policy-gradient training from materialised logits: log-probs, entropy and the gradient of the logits
        {"name": "logprob_train_2048", "op": "logprob", "N": 2048, "V": 128256, "dtype": "bf16", "k": 0, "masked": 0,
         "grad": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "evict", "logprob", "logprob"])
    D = rng.choice([32, 64, 64, 128, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    if op == "store":
        return {"op": op, "N": _log_int(rng, 1, max(1, 32768 * 8 * 128 // (Hkv * D) // 2)), "Hkv": Hkv, "D": D}
    if op == "decode":
        B = _log_int(rng, 1, 64)
        most = 32 * 8192 * 8 * 128 // (B * Hkv * D) // 2
        return {"op": op, "B": B, "T": _log_int(rng, 1, max(1, min(most, 120000))), "Hkv": Hkv,
                "G": rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]), "D": D, "window": rng.choice([0, 0, 0, 100, 1024, 4096]),
                "softcap": rng.choice([0.0, 0.0, 0.0, 50.0]), "empty": min(B - 1, rng.choice([0, 0, 1, 3])),
                "weights": rng.random() < 0.35}
    if op == "evict":
        B = _log_int(rng, 1, 32)
        most = 16 * 8192 * 8 * 128 // (B * Hkv * D) // 2
        T = _log_int(rng, 2, max(2, min(most, 60000)))
        keep = max(1, int(T * rng.uniform(0.05, 1.1)))
        sink = min(rng.choice([0, 1, 4]), keep)
        return {"op": op, "B": B, "T": T, "Hkv": Hkv, "D": D, "keep": keep, "recent": rng.randint(0, (keep - sink) // 2),
                "sink": sink}
    grad = rng.random() < 0.4
    V = _log_int(rng, 40, 152000)
    N = _log_int(rng, 1, max(1, min(8192, 2048 * 128256 // V // 2)))
    return {"op": op, "N": N, "V": V, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "k": rng.choice([0, 1, 2, 5, 8, 20]), "masked": rng.choice([0, 0, 17]), "grad": grad}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lens(c, g):
    """Context lengths from a quarter of the longest to the longest, the same set for every seed, in any order;
    the last `empty` rows are padding of the batch."""
    live = c["B"] - c.get("empty", 0)
    n = torch.linspace(max(1, c["T"] // 4), c["T"], live, dtype=torch.float64).round().to(torch.int32) if live > 1 \
        else torch.tensor([c["T"]], dtype=torch.int32)
    n = n.cuda()[torch.randperm(live, device="cuda", generator=g)]
    return torch.cat([n, n.new_zeros(c.get("empty", 0))])


def _rows(shape, g):
    """Keys or values as a model makes them: every channel with its own spread and offset, bf16."""
    spread = 0.3 + torch.rand(shape[-1], device="cuda", generator=g) ** 4 * 3
    shift = torch.randn(shape[-1], device="cuda", generator=g) * 0.5
    return (torch.randn(shape, device="cuda", generator=g) * spread + shift).bfloat16()


def _tables(B, W, first, g):
    """Distinct blocks in any order, numbered from `first` on."""
    return (torch.randperm(B * W, device="cuda", generator=g) + first).view(B, W).int()


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = {"c": c}
    if c["op"] == "store":
        blocks = -(-c["N"] // BLOCK) + 2
        place = torch.randperm(blocks * BLOCK, device="cuda", generator=g)[:c["N"]]
        s["k"], s["v"] = _rows((c["N"], c["Hkv"], c["D"]), g), _rows((c["N"], c["Hkv"], c["D"]), g)
        s["block"], s["off"] = (place // BLOCK).int(), (place % BLOCK).int()
        s["k_pool"] = torch.zeros(blocks, c["Hkv"], _block_bytes(c["D"]), dtype=torch.uint8, device="cuda")
        s["v_pool"] = torch.zeros_like(s["k_pool"])
        return s
    if c["op"] in ("decode", "evict"):
        B, W, Hkv, D = c["B"], -(-c["T"] // BLOCK), c["Hkv"], c["D"]
        s["lens"] = _lens(c, g)
        s["tables"] = _tables(B, W, 1, g)
        extra = 0
        if c["op"] == "evict":
            Wn = -(-c["keep"] // BLOCK)
            s["new_tables"] = _tables(B, Wn, 1 + B * W, g)
            extra = B * Wn
        shape = (1 + B * W + extra, Hkv, BLOCK, D)
        s["k_pool"], s["v_pool"] = _quantise_blocks(_rows(shape, g)), _quantise_blocks(_rows(shape, g))
        if c["op"] == "evict" or c["weights"]:
            # what some hundred steps of decoding left: a few tokens with most of the weight
            s["weights"] = torch.rand(B + 1, Hkv, W * BLOCK, device="cuda", generator=g).pow_(6).mul_(8).add_(0.01)
            s["weight_rows"] = torch.randperm(B + 1, device="cuda", generator=g)[:B].int()
        if c["op"] == "decode":
            s["q"] = (torch.randn(B, Hkv * c["G"], D, device="cuda", generator=g) * 1.5).bfloat16()
        return s
    x = torch.randn(c["N"], c["V"], device="cuda", generator=g) * 2.5
    # twelve different places a row (writing one twice would leave its value to chance)
    peak = (torch.randint(c["V"], (c["N"], 1), device="cuda", generator=g)
            + torch.arange(12, device="cuda") * (c["V"] // 12)) % c["V"]
    x.scatter_(1, peak, torch.rand(c["N"], 12, device="cuda", generator=g) * 14 + 3)
    if c["masked"]:  # vocabulary columns that no token has
        x[:, torch.randperm(c["V"], device="cuda", generator=g)[:c["masked"]]] = -math.inf
    s["x"] = x.to(_DTYPES[c["dtype"]])
    s["targets"] = torch.where(torch.rand(c["N"], device="cuda", generator=g) < 0.6, peak[:, 0],
                               torch.randint(c["V"], (c["N"],), device="cuda", generator=g))
    s["targets"] = torch.where(s["x"].gather(1, s["targets"][:, None])[:, 0] == -math.inf, s["x"].argmax(1), s["targets"])
    s["targets"][torch.rand(c["N"], device="cuda", generator=g) < 0.1] = -1  # positions outside the response
    if c["grad"]:
        s["x"].requires_grad_()
        s["g_lp"] = torch.randn(c["N"], device="cuda", generator=g) / c["N"]
        s["g_ent"] = torch.full((c["N"],), -0.01 / c["N"], device="cuda")
        s["g_top"] = torch.randn(c["N"], c["k"], device="cuda", generator=g) / c["N"]
    return s


_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ plain forms
def _block_bytes(D):
    return BLOCK * (D // 2 + 4 * (D // min(D, 64)))


def _quantise(x):
    """Rows [..., D] -> codes [..., groups, group] (uint8), scale and minimum [..., groups] (bf16)."""
    x = x.float().unflatten(-1, (-1, min(x.shape[-1], 64)))
    lo, hi = x.aminmax(dim=-1)
    lo = lo.bfloat16()
    scale = ((hi - lo.float()) / 15).bfloat16()
    n = ((x - lo.float()[..., None]) / scale.float()[..., None]).nan_to_num(0.0).round().clamp(0, 15)
    return n.to(torch.uint8), scale, lo


def _pack(n):
    return n[..., 0::2] | (n[..., 1::2] << 4)


def _quantise_blocks(x):
    """Whole blocks [blocks, Hkv, 16, D] -> the pool's bytes [blocks, Hkv, block bytes]."""
    n, scale, lo = _quantise(x)
    codes = _pack(n).transpose(-2, -3).flatten(2)
    meta = torch.stack((scale, lo), -1).transpose(-2, -3).contiguous().view(torch.uint8).flatten(2)
    return torch.cat((codes, meta), -1).contiguous()


def _values(blocks, D):
    """Blocks of a pool [..., block bytes] -> the values they stand for [..., 16, D] in fp32."""
    g = min(D, 64)
    codes = blocks[..., :BLOCK * D // 2].unflatten(-1, (D // g, BLOCK, g // 2))
    meta = blocks[..., BLOCK * D // 2:].contiguous().view(torch.bfloat16).unflatten(-1, (D // g, BLOCK, 2)).float()
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return (n * meta[..., :1] + meta[..., 1:]).transpose(-2, -3).flatten(-2)


def _plain_store(s):
    D = s["c"]["D"]
    g, blk, off = min(D, 64), s["block"].long(), s["off"].long()

    def put(pool, x):
        n, scale, lo = _quantise(x)  # [N, Hkv, groups, group]
        heads = torch.arange(x.shape[1], device="cuda")[None, :, None]
        groups = torch.arange(D // g, device="cuda")[None, None, :]
        b, o = blk[:, None, None], off[:, None, None]
        pool[..., :BLOCK * D // 2].unflatten(-1, (D // g, BLOCK, g // 2))[b, heads, groups, o] = _pack(n)
        meta = torch.stack((scale, lo), -1).view(torch.uint8)
        pool[..., BLOCK * D // 2:].unflatten(-1, (D // g, BLOCK, 4))[b, heads, groups, o] = meta

    put(s["k_pool"], s["k"])
    put(s["v_pool"], s["v"])
    return [_values(p[blk], D)[torch.arange(len(blk), device="cuda"), :, off].bfloat16()
            for p in (s["k_pool"], s["v_pool"])]


def _plain_decode(s):
    c = s["c"]
    B, Hkv, G, D = c["B"], c["Hkv"], c["G"], c["D"]
    pos = torch.arange(s["tables"].shape[1] * BLOCK, device="cuda")
    n = s["lens"].long()[:, None]
    seen = pos[None] < n
    if c["window"]:
        seen = seen & (pos[None] >= n - c["window"])
    k, v = (_values(p[s["tables"].long()], D).transpose(1, 2).flatten(2, 3) for p in (s["k_pool"], s["v_pool"]))
    v = torch.where(seen[:, None, :, None], v, 0.0)
    a = torch.einsum("bhgd,bhtd->bhgt", s["q"].float().view(B, Hkv, G, D), k) / math.sqrt(D)
    if c["softcap"]:
        a = torch.tanh(a / c["softcap"]) * c["softcap"]
    a = a.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(a - a.amax(-1, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.einsum("bhgt,bhtd->bhgd", p, v).reshape(B, Hkv * G, D).bfloat16()
    if not c["weights"]:
        return out
    s["weights"].index_add_(0, s["weight_rows"].long(), p.sum(2))
    return [out, s["weights"]]


def _plain_evict(s):
    c = s["c"]
    B, Hkv, D, keep = c["B"], c["Hkv"], c["D"], c["keep"]
    rows, n = s["weight_rows"].long(), s["lens"].long()[:, None, None]
    weights = s["weights"].clone()
    w = weights[rows]
    T = w.shape[-1]
    pos = torch.arange(T, device="cuda")[None, None]
    # the highest weight first, the lowest position among equals; protected tokens above all, absent ones below
    # (bits of non-negative floats are in the floats' order)
    rank = w.view(torch.int32).long()
    rank = torch.where((pos < c["sink"]) | (pos >= n - c["recent"]), 1 << 31, rank)
    rank = torch.where(pos < n, rank, -1)
    take = min(keep, T)
    chosen = (rank * (1 << 24) + (1 << 24) - 1 - pos).topk(take, -1).indices
    chosen = torch.where(chosen < n, chosen, T).sort(-1).values  # absent ones behind the last
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device="cuda")
    kept[..., :take] = torch.where(chosen < T, chosen, -1).int()
    there = kept >= 0
    src = kept.long().clamp_min(0)
    head = torch.arange(Hkv, device="cuda")[None, :, None]
    w_new = torch.where(there, w.gather(-1, src), 0.0)
    w_all = torch.where(pos < n, 0.0, w)  # what lies behind the last token stays
    w_all[..., :take] = torch.where(there[..., :take], w_new[..., :take], w_all[..., :take])
    weights[rows] = w_all
    lens = s["lens"].clamp(max=keep)
    # rows move as they are stored
    at = torch.arange(keep, device="cuda")
    to = s["new_tables"].long().gather(1, (at // BLOCK)[None].expand(B, -1))[:, None].expand(B, Hkv, keep)
    blk = s["tables"].long().gather(1, (src // BLOCK).flatten(1)).view(B, Hkv, keep)
    g = min(D, 64)
    slot, off = (at % BLOCK).expand(B, Hkv, keep)[there], (src % BLOCK)[there]
    hd, b_to, b_from = head.expand(B, Hkv, keep)[there], to[there], blk[there]

    def move(pool):
        codes = pool[..., :BLOCK * D // 2].unflatten(-1, (D // g, BLOCK, g // 2)).transpose(2, 3)
        meta = pool[..., BLOCK * D // 2:].unflatten(-1, (D // g, BLOCK, 4)).transpose(2, 3)
        codes[b_to, hd, slot] = codes[b_from, hd, off]
        meta[b_to, hd, slot] = meta[b_from, hd, off]
        return _values(pool[s["new_tables"].long()], D).transpose(2, 3).flatten(1, 2)[:, :keep].bfloat16()

    k, v = move(s["k_pool"]), move(s["v_pool"])
    live = (at[None] < lens[:, None])[..., None, None]
    return [kept, lens, weights, torch.where(live, k, 0.0), torch.where(live, v, 0.0)]


def _plain_logprob(s):
    c, t = s["c"], s["targets"]
    x = s["x"].detach().float()
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    lse = m + z.log()
    logp = x - lse
    p = e / z
    inside = t >= 0
    lp = torch.where(inside, logp.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)
    ent = -torch.where(p > 0, p * logp, 0.0).sum(1)
    # the order of floats as whole numbers, the lowest index first among equals
    bits = (x + 0.0).view(torch.int32).long()
    rank = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    ids = (rank * (1 << 20) + (1 << 20) - 1 - torch.arange(c["V"], device="cuda")).topk(c["k"], 1).indices
    out = [lp, ent, logp.gather(1, ids), ids]
    if not c["grad"]:
        return out
    total = torch.where(inside, s["g_lp"], 0.0) + s["g_top"].sum(1)
    d = -total[:, None] * p - s["g_ent"][:, None] * p * torch.where(p > 0, logp + ent[:, None], 0.0)
    d.scatter_add_(1, t.clamp_min(0)[:, None], torch.where(inside, s["g_lp"], 0.0)[:, None])
    d.scatter_add_(1, ids, s["g_top"])
    return out + [d.to(s["x"].dtype)]


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    if not own:
        return {"store": _plain_store, "decode": _plain_decode, "evict": _plain_evict,
                "logprob": _plain_logprob}[c["op"]](s)
    if c["op"] == "logprob":
        from rl_project_b200.ops.logprob import token_logprobs

        r = token_logprobs(s["x"], s["targets"], top=c["k"])
        out = [r.logprobs.detach(), r.entropy.detach(), r.top_logprobs.detach(), r.top_ids]
        if c["grad"]:
            out += torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], s["x"],
                                       [s["g_lp"], s["g_ent"], s["g_top"]])
        return out
    from rl_project_b200.ops import paged_q4

    if c["op"] == "store":
        paged_q4.paged_write_q4(s["k"], s["v"], s["k_pool"], s["v_pool"], s["block"], s["off"])
        return list(paged_q4.paged_read_q4(s["k_pool"], s["v_pool"], s["block"], s["off"], c["D"]))
    if c["op"] == "decode":
        out = paged_q4.paged_decode_q4(s["q"], s["k_pool"], s["v_pool"], s["tables"], s["lens"], 1 / math.sqrt(c["D"]),
                                       softcap=c["softcap"], window=c["window"], weights=s.get("weights"),
                                       weight_rows=s.get("weight_rows"))
        return [out, s["weights"]] if c["weights"] else out
    weights = s["weights"].clone()  # compacted in place
    kept, lens = paged_q4.paged_evict_q4(s["k_pool"], s["v_pool"], s["tables"], s["lens"], s["new_tables"], weights,
                                         s["weight_rows"], c["keep"], c["D"], recent=c["recent"], sink=c["sink"])
    k, v = paged_q4.paged_gather_q4(s["k_pool"], s["v_pool"], s["new_tables"], lens, c["D"], c["keep"])
    return [kept, lens, weights, k, v]


# ------------------------------------------------------------------ floors
def _total(c):
    live = c["B"] - c.get("empty", 0)
    if live == 1:
        n = [c["T"]]
    else:
        n = torch.linspace(max(1, c["T"] // 4), c["T"], live, dtype=torch.float64).round().long().tolist()
    return n


def work(case):
    c = case
    if c["op"] == "logprob":
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[c["dtype"]]
        b = c["N"] * c["V"] * size + c["N"] * (8 + 8 + 12 * c["k"])
        f = 6 * c["N"] * c["V"]
        if c["grad"]:  # the gradient needs every row's sum first, so the logits are read twice
            b += 2 * c["N"] * c["V"] * size
            f += 6 * c["N"] * c["V"]
        return {"bytes": b, "flops": f}
    row = c["D"] // 2 + 4 * (c["D"] // min(c["D"], 64))  # stored bytes of a key or a value
    if c["op"] == "store":
        rows = 2 * c["N"] * c["Hkv"]
        return {"bytes": rows * (2 * c["D"] + row + 2 * c["D"]) + 8 * c["N"], "flops": 6 * rows * c["D"]}
    n = _total(c)
    if c["op"] == "decode":
        tokens = sum(min(x, c["window"]) if c["window"] else x for x in n)
        b = tokens * c["Hkv"] * 2 * row + 4 * c["B"] * c["Hkv"] * c["G"] * c["D"]
        return {"bytes": b + (8 * tokens * c["Hkv"] if c["weights"] else 0),
                "flops": 4 * tokens * c["Hkv"] * c["G"] * c["D"]}
    left = sum(min(x, c["keep"]) for x in n) * c["Hkv"]
    out = 2 * c["B"] * c["keep"] * c["Hkv"] * c["D"] * 2
    return {"bytes": sum(n) * c["Hkv"] * 4 + left * (2 * 2 * row + 8) + out, "flops": 2 * sum(n) * c["Hkv"]}


# ------------------------------------------------------------------ the definition in 64 bits
def _stored(pool, block, head, off, D):
    """Rows of a pool, in 64 bits, from the bytes' places: block, head and slot of each row (equal shapes)."""
    d = torch.arange(D, device="cuda")
    g = min(D, 64)
    grp, e = d // g, d % g
    place = grp * BLOCK * (g // 2) + off[..., None] * (g // 2) + e // 2
    byte = pool[block[..., None], head[..., None], place].long()
    code = torch.where(e % 2 == 1, byte // 16, byte % 16).double()
    at = BLOCK * D // 2 + (grp * BLOCK + off[..., None]) * 4

    def number(p):
        b = [pool[block[..., None], head[..., None], p + i].int() for i in (0, 1)]
        return ((b[1] * 256 + b[0]) << 16).view(torch.float32).double()

    return code * number(at) + number(at + 2)


def _exact_rows(x):
    """What a stored row reads back as."""
    shape, x = x.shape, x.double().reshape(-1, min(x.shape[-1], 64))
    lo = x.min(1, keepdim=True).values
    scale = ((x.max(1, keepdim=True).values - lo) / 15).bfloat16().double()
    code = torch.where(scale > 0, (x - lo) / scale.clamp_min(1e-300), 0.0).round().clamp(0, 15)
    return (code * scale + lo).reshape(shape)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "store":
        return [_exact_rows(s["k"]), _exact_rows(s["v"])]
    if c["op"] == "logprob":
        lp, ent, top, dx = [], [], [], []
        for r in range(0, c["N"], 256):  # a slice of rows at a time
            x, t = s["x"].detach()[r:r + 256].double(), s["targets"][r:r + 256]
            rows = torch.arange(len(x), device="cuda")
            logp = torch.log_softmax(x, 1)
            p = logp.exp()
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["k"]]
            h = torch.special.entr(p).sum(1)
            lp.append(torch.where(t >= 0, logp[rows, t.clamp_min(0)], 0.0))
            ent.append(h)
            top.append(logp.gather(1, ids))
            if c["grad"]:
                g, ge, gt = (s[n][r:r + 256].double() for n in ("g_lp", "g_ent", "g_top"))
                g = g * (t >= 0)
                q = torch.zeros_like(p)
                q[rows, t.clamp_min(0)] += g
                q.scatter_add_(1, ids, gt)
                q -= p * (g + gt.sum(1))[:, None]
                dx.append(q - ge[:, None] * (p * h[:, None] - torch.special.entr(p)))
        out = [torch.cat(lp), torch.cat(ent), torch.cat(top), None]
        return out + [torch.cat(dx)] if c["grad"] else out
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    head = torch.arange(Hkv, device="cuda")[:, None]
    if c["op"] == "decode":
        out = torch.zeros(B, Hkv * c["G"], D, dtype=torch.float64, device="cuda")
        acc = s["weights"].double() if c["weights"] else None
        for b, n in enumerate(s["lens"].tolist()):
            if not n:
                continue
            pos = torch.arange(max(0, n - c["window"]) if c["window"] else 0, n, device="cuda")
            blk, off = s["tables"][b, pos // BLOCK].long(), pos % BLOCK
            for h in range(Hkv):
                one = torch.full_like(pos, h)
                q = s["q"][b, h * c["G"]:(h + 1) * c["G"]].double()
                a = q @ _stored(s["k_pool"], blk, one, off, D).T / D ** 0.5
                if c["softcap"]:
                    a = c["softcap"] * torch.tanh(a / c["softcap"])
                p = torch.softmax(a, -1)
                out[b, h * c["G"]:(h + 1) * c["G"]] = p @ _stored(s["v_pool"], blk, one, off, D)
                if acc is not None:
                    acc[s["weight_rows"][b], h, pos] += p.sum(0)
        return [out, acc] if c["weights"] else out
    ks = torch.zeros(B, c["keep"], Hkv, D, dtype=torch.float64, device="cuda")
    vs, weights = torch.zeros_like(ks), s["weights"].double()
    for b, n in enumerate(s["lens"].tolist()):
        w = s["weights"][s["weight_rows"][b], :, :n].double()
        pos = torch.arange(n, device="cuda")
        w[:, (pos < c["sink"]) | (pos >= n - c["recent"])] = math.inf
        left = torch.sort(w, dim=1, descending=True, stable=True).indices[:, :c["keep"]].sort(1).values
        m = left.shape[1]
        blk, off = s["tables"][b].long()[left // BLOCK], left % BLOCK
        ks[b, :m] = _stored(s["k_pool"], blk, head.expand_as(blk), off, D).transpose(0, 1)
        vs[b, :m] = _stored(s["v_pool"], blk, head.expand_as(blk), off, D).transpose(0, 1)
        row = weights[s["weight_rows"][b]]
        moved = row.gather(1, left)
        row[:, :n] = 0
        row[:, :m] = moved
    return [None, None, weights, ks, vs]
