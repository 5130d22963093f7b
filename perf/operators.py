"""Cases, plain forms and definitions of the token-memory operators: attention of packed prompts, writing keys and
values into the 8-bit token cache, attention of single tokens over that cache, and eviction from it by accumulated
attention weight.  Where `own` is false an operator runs as elementary torch operations in 32 bits; where it is true
as the calls a user makes."""
import math

import torch

own = False

#: Work of the largest drawn case, in bytes of memory traffic and in visible query-key pairs of all heads.
MOST_BYTES = 2.2e9
MOST_PAIRS = 2.1e9
MOST_SCORES = 4.29e9    # score matrix of a packed prompt's plain form


def ints(text):
    return [int(x) for x in str(text).split()]


def listed():
    return [
        # one short question to a small model: launch latency is what counts
        dict(name="prompt short", op="prompt", type="f16", hq=8, hkv=2, dim=64, lens="24", past="0", causal=True),
        # an ordinary batch of packed prompts of very different lengths, one of them a single token
        dict(name="prompt packed", op="prompt", type="bf16", hq=32, hkv=8, dim=128,
             lens="1 1907 37 640 128 999 255 1300 16 77 511 1025 300", past="0 0 0 0 0 0 0 0 0 0 0 0 0", causal=True),
        # the next pieces of prompts whose first pieces were attended to before, head dimension of a 96-d embedder
        dict(name="prompt pieces", op="prompt", type="f16", hq=12, hkv=4, dim=96, lens="512 301 512", past="4096 2500 0",
             causal=True),
        # one long document
        dict(name="prompt long", op="prompt", type="bf16", hq=16, hkv=4, dim=128, lens="16384", past="0", causal=True),
        # the first conversations of prompts of a batch enter the cache
        dict(name="write prompts", op="write", type="bf16", hkv=8, dim=128, block=64,
             lens="4096 1907 1 640 8192 999 33", start="0 0 0 0 0 0 0"),
        # a decoding step's new token of every sequence enters its last block
        dict(name="write tokens", op="write", type="f16", hkv=8, dim=128, block=32,
             lens=" ".join(["1"] * 64), start=" ".join(str(37 * i % 1000) for i in range(64))),
        # one token of one short conversation: latency
        dict(name="cache short", op="cache", type="f16", hq=8, hkv=2, dim=64, block=16, queries=1, lens="300", mass=False),
        # an ordinary decoding batch, with the weights that eviction goes by
        dict(name="cache batch", op="cache", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1,
             lens=" ".join(str(64 + 379 * i * i % 6000) for i in range(32)), mass=True),
        # four drafted tokens checked at once against long contexts
        dict(name="cache drafts", op="cache", type="bf16", hq=24, hkv=8, dim=128, block=32, queries=4,
             lens="32768 20001 1000 15", mass=False),
        # a full card's batch of long contexts
        dict(name="cache long", op="cache", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1,
             lens=" ".join(["65536"] * 15 + ["65521"]), mass=True),
        # one small cache cut down at a step
        dict(name="evict small", op="evict", type="f16", hkv=2, dim=64, block=16, lens="700 256", budget=256, sinks=4,
             recent=32),
        # long contexts cut to a quarter
        dict(name="evict long", op="evict", type="bf16", hkv=8, dim=128, block=64, lens="65536 40000 32769 8000",
             budget=16384, sinks=4, recent=512),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total, most):
    """1 to `most` lengths that sum to about `total`, some of them single tokens."""
    n = min(_spread(rng, 1, most), total)
    cuts = [rng.random() ** 2 + 1e-3 for _ in range(n)]
    return [1 if rng.random() < 0.1 else max(1, int(total * c / sum(cuts))) for c in cuts]


def draw(rng):
    op = rng.choice(("prompt", "prompt", "write", "cache", "cache", "evict"))
    typ = rng.choice(("bf16", "f16"))
    if op == "prompt":
        hkv, g, dim = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 6, 8)), rng.choice((48, 64, 80, 96, 128, 128))
        total = _spread(rng, 16, 14000)
        while True:
            lens = _lens(rng, total, 24)
            past = [rng.choice((0, 0, 0, _spread(rng, 1, 4000))) for _ in lens]
            causal = rng.random() < 0.85
            c = dict(op=op, type=typ, hq=hkv * g, hkv=hkv, dim=dim, lens=" ".join(map(str, lens)),
                     past=" ".join(map(str, past)), causal=causal)
            scores = sum(lens) * (sum(lens) + sum(past)) * hkv * g
            if _pairs(c) * hkv * g <= MOST_PAIRS and scores <= MOST_SCORES:
                return c
            total = max(16, total * 3 // 4)
    hkv, dim, block = rng.choice((1, 2, 4, 8, 8)), rng.choice((48, 64, 96, 128, 128)), rng.choice((16, 32, 64, 128))
    row = hkv * dim
    if op == "write":
        lens = _lens(rng, _spread(rng, 8, 60000), 64)
        start = [rng.choice((0, _spread(rng, 1, 2000))) for _ in lens]
        return dict(op=op, type=typ, hkv=hkv, dim=dim, block=block, lens=" ".join(map(str, lens)),
                    start=" ".join(map(str, start)))
    most = 0.7 * MOST_BYTES / (2 * row)
    lens = _lens(rng, _spread(rng, 100, min(most, 900000)), 64)
    if op == "cache":
        g, queries = rng.choice((1, 2, 3, 4, 6, 8, 16)), rng.choice((1, 1, 1, 2, 3, 5))
        while len(lens) * max(lens) * hkv * max(dim, g * queries) * 4 > 9e9:    # the plain form's largest tensor
            lens = [max(1, n // 2) for n in lens]
        return dict(op=op, type=typ, hq=hkv * g, hkv=hkv, dim=dim, block=block, queries=queries,
                    lens=" ".join(map(str, lens)), mass=rng.random() < 0.6)
    while len(lens) * max(lens) * hkv > 3e7:
        lens = [max(1, n // 2) for n in lens]
    budget = max(8, int(max(lens) * rng.uniform(0.1, 0.9)))
    while len(lens) * budget * row * 2 > 0.5 * MOST_BYTES:
        budget //= 2
    sinks = rng.choice((0, 1, 4))
    return dict(op=op, type=typ, hkv=hkv, dim=dim, block=block, lens=" ".join(map(str, lens)), budget=budget, sinks=sinks,
                recent=int((budget - sinks) * rng.choice((0.0, 0.1, 0.5))))


def _pairs(c):
    """Visible query-key pairs of one head of a packed prompt."""
    n = 0
    for q, p in zip(ints(c["lens"]), ints(c["past"])):
        n += q * p + (q * (q + 1) // 2 if c["causal"] else q * q)
    return n


def work(case):
    op, d = case["op"], case["dim"]
    lens = ints(case["lens"])
    if op == "prompt":
        tq, tk = sum(lens), sum(lens) + sum(ints(case["past"]))
        return {"bytes": 2 * d * (2 * tq * case["hq"] + 2 * tk * case["hkv"]) + 4 * tq * case["hq"],
                "flops": 4 * d * case["hq"] * _pairs(case)}
    row = case["hkv"] * d
    if op == "write":
        held = sum(s % case["block"] for s in ints(case["start"]))
        # keys and values in, codes out; the held tokens of a block that is filled on, read and written; the values of
        # the blocks that changed read back
        return {"bytes": 2 * row * (3 * sum(lens) + 2 * held + 3 * (sum(lens) + held)), "flops": 4 * row * sum(lens)}
    if op == "cache":
        rows = len(lens) * case["queries"] * case["hq"]
        n = 2 * row * sum(lens) + 4 * rows * d + 4 * rows
        return {"bytes": n + (8 * case["hkv"] * sum(lens) if case["mass"] else 0),
                "flops": 4 * case["queries"] * case["hq"] * d * sum(lens)}
    kept = sum(min(n, case["budget"]) for n in lens)
    # the weights; codes of what stays, read and written; its values read back; its positions and weights
    return {"bytes": 4 * case["hkv"] * sum(lens) + 2 * row * kept * 5 + 8 * case["hkv"] * kept,
            "flops": 4 * row * kept}


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(values):
    return _i32([sum(values[:i]) for i in range(len(values) + 1)])


def _pool(g, blocks, case):
    """A pool of blocks as sequences have left it: codes like those of normal values, no block empty."""
    shape = (blocks, case["hkv"], case["block"], case["dim"])
    codes = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        codes.append(x.mul_(38).round_().clamp_(-127, 127).to(torch.int8))
        del x
    scales = [0.02 + 0.03 * torch.rand(shape[:2], generator=g, device="cuda") for _ in range(2)]
    return codes + scales


def _table(g, counts, spare=0):
    """Blocks of the sequences, in the order in which a pool gives them out after a while: any; -1 past the end."""
    at = torch.randperm(sum(counts) + spare, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    used = 0
    for b, n in enumerate(counts):
        table[b, :n] = at[used:used + n]
        used += n
    return table, at[used:]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, d, lens = TYPES[case["type"]], case["dim"], ints(case["lens"])
    s = {"case": dict(case), "scale": 1.0 / math.sqrt(d)}

    def rows(n, heads, spread=1.0):
        x = torch.randn((n, heads, d), generator=g, device="cuda")
        return x.mul_(spread * (0.5 + torch.rand((1, heads, d), generator=g, device="cuda"))).to(t)

    if case["op"] == "prompt":
        both = [a + b for a, b in zip(lens, ints(case["past"]))]
        return s | {"q": rows(sum(lens), case["hq"], 1.5), "k": rows(sum(both), case["hkv"]), "v": rows(sum(both), case["hkv"]),
                    "cu_q": _cu(lens), "cu_k": _cu(both)}
    if case["op"] == "write":
        start = ints(case["start"])
        counts = [-(-(a + b) // case["block"]) for a, b in zip(lens, start)]
        table, _ = _table(g, counts)
        s["pool"] = _pool(g, sum(counts), case)
        # places that are read back: from the start of the first block that changes
        first = [a // case["block"] * case["block"] for a in start]
        ends = [a + b for a, b in zip(lens, start)]
        places = _i32(first)[:, None] + torch.arange(max(e - f for e, f in zip(ends, first)), dtype=torch.int32, device="cuda")
        return s | {"table": table, "k": rows(sum(lens), case["hkv"], 1.2), "v": rows(sum(lens), case["hkv"]), "cu": _cu(lens),
                    "start": _i32(start), "lens": _i32(ends), "places": places}
    counts = [-(-n // case["block"]) for n in lens]
    if case["op"] == "cache":
        table, _ = _table(g, counts)
        s["pool"] = _pool(g, sum(counts), case)
        q = rows(len(lens) * case["queries"], case["hq"], 1.5).view(len(lens), case["queries"], case["hq"], d)
        s |= {"table": table, "q": q, "lens": _i32(lens), "mass": None}
        if case["mass"]:
            s["mass"] = torch.rand((len(lens), case["hkv"], max(lens)), generator=g, device="cuda").pow_(4)
        return s
    budget = case["budget"]
    new = [-(-min(n, budget) // case["block"]) for n in lens]
    table, free = _table(g, counts, sum(new))
    s["pool"] = _pool(g, sum(counts) + sum(new), case)
    new_table = torch.full((len(lens), max(new)), -1, dtype=torch.int32, device="cuda")
    used = 0
    for b, n in enumerate(new):
        new_table[b, :n] = free[used:used + n]
        used += n
    # accumulated weights: a few tokens hold most, many hold next to nothing, and some of them the same
    mass = torch.randn((len(lens), case["hkv"], max(lens)), generator=g, device="cuda").mul_(2.5).exp_()
    mass = torch.where(mass < 0.02, torch.round(mass * 500) / 500, mass)
    places = torch.arange(min(budget, max(lens)), dtype=torch.int32, device="cuda").repeat(len(lens), 1)
    return s | {"table": table, "new_table": new_table, "lens": _i32(lens), "mass": mass, "places": places}


def run(state):
    return RUNS[state["case"]["op"]][1 if own else 0](state)


# ---- plain forms -----------------------------------------------------------

def _softmax_out(scores, seen, values):
    """scores [..., q, k] in place; seen broadcasts to them.  (weights, outputs, log of the sums)."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.sub_(base).exp_()
    total = scores.sum(-1, keepdim=True)
    lse = (total.log() + base).squeeze(-1)
    inv = torch.where(total > 0, 1 / total, torch.zeros_like(total))
    return scores, torch.matmul(scores, values) * inv, lse, inv


def plain_prompt(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    tq, tk, g = q.shape[0], k.shape[0], c["hq"] // c["hkv"]
    at_q, at_k = torch.arange(tq, device="cuda"), torch.arange(tk, device="cuda")
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    seq_q, seq_k = torch.bucketize(at_q, cu_q[1:], right=True), torch.bucketize(at_k, cu_k[1:], right=True)
    seen = seq_q[:, None] == seq_k[None, :]
    if c["causal"]:
        last = at_q - cu_q[seq_q + 1] + cu_k[seq_q + 1]         # the row's own place among the keys
        seen &= at_k[None, :] <= last[:, None]
    qh = q.float().mul(s["scale"]).view(tq, c["hkv"], g, -1).permute(1, 2, 0, 3)
    scores = torch.matmul(qh, k.float().permute(1, 2, 0).unsqueeze(1))
    _, out, lse, _ = _softmax_out(scores, seen, v.float().transpose(0, 1).unsqueeze(1))
    out = out.permute(2, 0, 1, 3).reshape(tq, c["hq"], -1).to(q.dtype)
    return {"out": out, "lse": lse.permute(2, 0, 1).reshape(tq, c["hq"]).contiguous()}


def _values(codes, scales, table):
    """[B, heads, tokens, D] of a table's blocks (block 0 in place of none)."""
    t = table.clamp(min=0).long()
    x = codes[t].float().mul_(scales[t][..., None, None])
    return x.permute(0, 2, 1, 3, 4).reshape(t.shape[0], codes.shape[1], -1, codes.shape[3])


def plain_cache(s):
    c, q = s["case"], s["q"]
    b, nq, hkv, g = q.shape[0], q.shape[1], c["hkv"], c["hq"] // c["hkv"]
    kc, vc, ks, vs = s["pool"]
    k = _values(kc, ks, s["table"])
    qh = q.float().mul(s["scale"]).view(b, nq, hkv, g, -1).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * nq, -1)
    scores = torch.matmul(qh, k.transpose(2, 3))
    del k
    n = scores.shape[-1]
    lim = s["lens"][:, None] - nq + 1 + torch.arange(nq, device="cuda")[None]
    seen = (torch.arange(n, device="cuda")[None, None] < lim[..., None])[:, None].repeat(1, 1, g, 1)
    w, out, lse, inv = _softmax_out(scores, seen, _values(vc, vs, s["table"]))
    back = lambda x: x.view(b, hkv, g, nq, -1).permute(0, 3, 1, 2, 4).reshape(b, nq, c["hq"], -1)  # noqa: E731
    res = {"out": back(out).to(q.dtype), "lse": back(lse[..., None])[..., 0].contiguous()}
    if s["mass"] is not None:
        most = s["mass"].shape[2]
        mass = s["mass"] + w.mul_(inv).sum(2)[..., :most]
        res["mass"] = mass.masked_fill_(torch.arange(most, device="cuda") >= s["lens"][:, None, None], 0)
    return res


def _read_back(pool, table, lens, places, dtype):
    """Values at places [B, n] of every head, zero at and past a sequence's length."""
    block, hkv = pool[0].shape[2], pool[0].shape[1]
    gone = places >= lens[:, None]
    at = torch.where(gone, torch.zeros_like(places), places).long()
    into = table.gather(1, at // block).long()[:, None]
    head = torch.arange(hkv, device="cuda")[None, :, None]
    at = (at % block)[:, None]
    return [(pool[i][into, head, at].float() * pool[2 + i][into, head][..., None]).masked_fill_(gone[:, None, :, None], 0).to(dtype)
            for i in (0, 1)]


def plain_write(s):
    c, block = s["case"], s["case"]["block"]
    start, cu = s["start"].long(), s["cu"].long()
    at = torch.arange(s["k"].shape[0], device="cuda")
    seq = torch.bucketize(at, cu[1:], right=True)
    pos = start[seq] + at - cu[seq]
    into, slot = s["table"][seq, pos // block].long(), pos % block
    first = s["table"].gather(1, (start // block).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].long()
    filled = (start % block > 0) & (cu[1:] > cu[:-1])            # sequences whose first block holds tokens already
    for x, codes, scales in ((s["k"], s["pool"][0], s["pool"][2]), (s["v"], s["pool"][1], s["pool"][3])):
        x = x.float()
        top = torch.zeros_like(scales).scatter_reduce_(0, into[:, None].expand(-1, c["hkv"]), x.abs().amax(-1), "amax")
        new = torch.where(top < 1e-30, torch.zeros_like(top), top / 127)
        held = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda").index_put_((first,), filled)
        old = torch.where(held[:, None], scales, torch.zeros_like(scales))
        new = torch.maximum(new, old)
        ratio = torch.where(new > old, old / new, torch.ones_like(new))
        touched = torch.zeros(scales.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, into, True)
        grown = torch.round(codes[first].float() * ratio[first][..., None, None]).to(torch.int8)
        codes[first] = torch.where(filled[:, None, None, None], grown, codes[first])
        inv = torch.where(new > 0, 1 / new, torch.zeros_like(new))
        codes[into, :, slot] = torch.round(x * inv[into][..., None]).clamp(-127, 127).to(torch.int8)
        scales.copy_(torch.where(touched[:, None], new, scales))
    return _read_back(s["pool"], s["table"].long(), s["lens"], s["places"], s["k"].dtype)


def plain_evict(s):
    c, mass, lens = s["case"], s["mass"], s["lens"].long()
    budget, block = c["budget"], c["block"]
    t = mass.shape[2]
    at = torch.arange(t, device="cuda")[None, None]
    n = lens[:, None, None]
    kind = torch.where(at >= n, 2, torch.where((at < c["sinks"]) | (at >= n - c["recent"]) | (n <= budget), 0, 1))
    order = torch.argsort(mass, dim=2, descending=True, stable=True)     # ties: lowest position
    order = order.gather(2, torch.argsort(kind.expand_as(order).gather(2, order), dim=2, stable=True))[..., :budget]
    stay = lens.clamp(max=budget)
    room = torch.arange(order.shape[2], device="cuda")[None, None]
    kept = torch.where(room < stay[:, None, None], order, t).sort(2).values
    if kept.shape[2] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[2]), value=t)
    none = kept == t
    kept = kept.masked_fill(none, 0)
    new_mass = mass.gather(2, kept).masked_fill(none, 0)
    table, new_table = s["table"].long(), s["new_table"].long()
    pad = -budget % block
    src = torch.nn.functional.pad(kept, (0, pad))
    gone = torch.nn.functional.pad(none, (0, pad), value=True)
    from_block = table[torch.arange(len(lens), device="cuda")[:, None, None], src // block]
    head = torch.arange(c["hkv"], device="cuda")[None, :, None]
    shape = (len(lens), c["hkv"], -1, block)
    own_blocks = new_table >= 0
    for i in (0, 1):
        codes, scales = s["pool"][i], s["pool"][2 + i]
        old = scales[from_block, head].masked_fill(gone, 0).view(shape)
        new = old.amax(-1)
        ratio = torch.where(new[..., None] > 0, old / new[..., None], torch.zeros_like(old))
        moved = codes[from_block, head, src % block].view(*shape, c["dim"]).float().mul_(ratio[..., None])
        moved = torch.round(moved).to(torch.int8).transpose(1, 2)[:, :new_table.shape[1]]
        codes[new_table[own_blocks]] = moved[own_blocks]
        scales[new_table[own_blocks]] = new.transpose(1, 2)[:, :new_table.shape[1]][own_blocks]
    values = _read_back(s["pool"], new_table, stay, s["places"], TYPES[c["type"]])
    return {"kept": kept.masked_fill(none, -1).to(torch.int32), "lens": stay.to(torch.int32), "mass": new_mass,
            "k": values[0], "v": values[1]}


# ---- the framework's operators ---------------------------------------------

def own_prompt(s):
    from beam_search_collab_b200 import memory
    out, lse = memory.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"],
                                       scale=s["scale"], with_lse=True)
    return {"out": out, "lse": lse}


def own_cache(s):
    from beam_search_collab_b200 import memory
    cache = memory.TokenCache(*s["pool"])
    out, lse, mass = cache.attention(s["q"], s["table"], s["lens"], scale=s["scale"], with_lse=True, mass=s["mass"])
    return {"out": out, "lse": lse} if mass is None else {"out": out, "lse": lse, "mass": mass}


def own_write(s):
    from beam_search_collab_b200 import memory
    cache = memory.TokenCache(*s["pool"])
    cache.write(s["k"], s["v"], s["cu"], s["table"], s["start"])
    return list(cache.read(s["table"], s["lens"], s["places"], dtype=s["k"].dtype))


def own_evict(s):
    from beam_search_collab_b200 import memory
    c = s["case"]
    cache = memory.TokenCache(*s["pool"])
    kept, lens, mass = cache.evict(s["mass"], s["table"], s["lens"], s["new_table"], c["budget"], sinks=c["sinks"],
                                   recent=c["recent"])
    k, v = cache.read(s["new_table"], lens, s["places"], dtype=TYPES[c["type"]])
    return {"kept": kept, "lens": lens, "mass": mass, "k": k, "v": v}


RUNS = {"prompt": (plain_prompt, own_prompt), "cache": (plain_cache, own_cache), "write": (plain_write, own_write),
        "evict": (plain_evict, own_evict)}


# ---- definitions in 64 bits ------------------------------------------------

def _attend(q, k, v, scale, limits):
    """One head's rows q [n, D] over keys [m, D]; row i sees the first limits[i] keys.  (out, lse, weights' sum)."""
    outs, lses, total = [], [], torch.zeros(k.shape[0], dtype=torch.float64, device="cuda")
    step = max(1, int(2e8 // max(1, k.shape[0])))
    for a in range(0, q.shape[0], step):
        z = (q[a:a + step] @ k.T) * scale
        z[torch.arange(k.shape[0], device="cuda")[None] >= limits[a:a + step, None]] = -math.inf
        lse = torch.logsumexp(z, 1)
        w = torch.exp(z - lse[:, None])
        w[limits[a:a + step] <= 0] = 0
        outs.append(w @ v)
        lses.append(lse)
        total += w.sum(0)
    return torch.cat(outs), torch.cat(lses), total


def exact(case, seed):
    s = prepare(case, seed)
    lens = ints(case["lens"])
    return {"prompt": _exact_prompt, "cache": _exact_cache, "write": _exact_write, "evict": _exact_evict}[case["op"]](s, case, lens)


def _exact_prompt(s, case, lens):
    g, both = case["hq"] // case["hkv"], [a + b for a, b in zip(lens, ints(case["past"]))]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    a = b = 0
    for nq, nk in zip(lens, both):
        limits = torch.arange(nq, device="cuda") + nk - nq + 1 if case["causal"] else torch.full((nq,), nk, device="cuda")
        for h in range(case["hq"]):
            k, v = s["k"][b:b + nk, h // g].double(), s["v"][b:b + nk, h // g].double()
            out[a:a + nq, h], lse[a:a + nq, h], _ = _attend(s["q"][a:a + nq, h].double(), k, v, s["scale"], limits)
        a, b = a + nq, b + nk
    return {"out": out, "lse": lse}


def _sequence(s, i, b, n, h, block):
    """Values of sequence b's first n tokens, head h, keys (i = 0) or values (i = 1)."""
    t = s["table"][b, :-(-n // block)].long()
    x = s["pool"][i][t, h].double() * s["pool"][2 + i][t, h].double()[:, None, None]
    return x.reshape(-1, x.shape[-1])[:n]


def _exact_cache(s, case, lens):
    g, nq = case["hq"] // case["hkv"], case["queries"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device="cuda")
    mass = torch.zeros(s["mass"].shape, dtype=torch.float64, device="cuda") if case["mass"] else None
    for b, n in enumerate(lens):
        limits = (torch.arange(nq, device="cuda") + n - nq + 1).repeat_interleave(g)
        for h in range(case["hkv"]):
            k, v = _sequence(s, 0, b, n, h, case["block"]), _sequence(s, 1, b, n, h, case["block"])
            q = s["q"][b, :, h * g:h * g + g].reshape(nq * g, -1).double()
            o, z, w = _attend(q, k, v, s["scale"], limits)
            out[b, :, h * g:h * g + g], lse[b, :, h * g:h * g + g] = o.view(nq, g, -1), z.view(nq, g)
            if case["mass"]:
                mass[b, h, :n] = s["mass"][b, h, :n].double() + w
    return {"out": out, "lse": lse, "mass": mass} if case["mass"] else {"out": out, "lse": lse}


def _exact_write(s, case, lens):
    res = []
    for i, x in ((0, s["k"]), (1, s["v"])):
        y = torch.zeros((len(lens), case["hkv"], s["places"].shape[1], case["dim"]), dtype=torch.float64, device="cuda")
        a = 0
        for b, (n, start) in enumerate(zip(lens, ints(case["start"]))):
            held = start % case["block"]
            old = s["table"][b, start // case["block"]].long()       # the block that is filled on
            y[b, :, :held] = s["pool"][i][old, :, :held].double() * s["pool"][2 + i][old].double()[:, None, None]
            y[b, :, held:held + n] = x[a:a + n].double().transpose(0, 1)
            a += n
            for lo in range(0, held + n, case["block"]):
                hi, cut = min(lo + case["block"], held + n), max(lo, held)
                scale = y[b, :, cut:hi].abs().amax((1, 2)) / 127
                if cut > lo:
                    scale = torch.maximum(scale, s["pool"][2 + i][old].double())
                y[b, :, lo:hi] = torch.round(y[b, :, lo:hi] / scale[:, None, None]).clamp(-127, 127) * scale[:, None, None]
        res.append(y)
    return res


def _exact_evict(s, case, lens):
    budget, block = case["budget"], case["block"]
    mass = torch.zeros((len(lens), case["hkv"], budget), dtype=torch.float64, device="cuda")
    values = [torch.zeros((len(lens), case["hkv"], s["places"].shape[1], case["dim"]), dtype=torch.float64, device="cuda")
              for _ in (0, 1)]
    for b, n in enumerate(lens):
        for h in range(case["hkv"]):
            at = torch.arange(n, device="cuda")
            if n > budget:
                free = at[case["sinks"]:n - case["recent"]]
                best = torch.sort(s["mass"][b, h, free], descending=True, stable=True).indices
                best = free[best[:budget - case["sinks"] - case["recent"]]]
                at = torch.cat((at[:case["sinks"]], best.sort().values, at[n - case["recent"]:]))
            mass[b, h, :len(at)] = s["mass"][b, h, at].double()
            blocks = s["table"][b, at // block].long()
            for i in (0, 1):
                scale = s["pool"][2 + i][blocks, h].double()
                new = torch.nn.functional.pad(scale, (0, -len(at) % block)).view(-1, block).amax(1)
                new = new.repeat_interleave(block)[:len(at)]
                code = s["pool"][i][blocks, h, at % block].double()
                values[i][b, h, :len(at)] = torch.round(code * (scale / new)[:, None]) * new[:, None]
    return {"kept": None, "lens": None, "mass": mass, "k": values[0], "v": values[1]}
