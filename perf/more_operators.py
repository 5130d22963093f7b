"""Cases, plain forms and definitions of the token-memory operators of long and shared contexts: norm and rotary position
of queries and keys, bounds of the 8-bit cache's blocks, the choice of blocks by those bounds, attention over the blocks
chosen, and attention of sequences that begin with the same tokens.  Where `own` is false an operator runs as elementary
torch operations in 32 bits (64 for angles and for sums of integers); where it is true as the calls a user makes."""
import math

import torch

own = False

#: The largest drawn case: bytes of memory traffic and operations (both below the largest listed one's), and bytes of
#: the plain form's largest tensor.
MOST_BYTES, MOST_FLOPS, MOST_PLAIN = 1.6e8, 6e10, 3e9


def ints(text):
    return [int(x) for x in str(text).split()]


def listed():
    return [
        # a decoding step's new token of 64 conversations, some of them far on: half of each head is rotated, positions
        # scaled for long contexts, no norm
        dict(name="rotate tokens", op="rotate", type="f16", hq=12, hkv=4, dim=96, rotary=48, interleaved=True, norm=False, scaled=True,
             lens=" ".join(["1"] * 64), start=" ".join(str(37 * i * i * i) for i in range(64))),
        # a batch of packed prompts, with norms of queries and keys
        dict(name="rotate packed", op="rotate", type="bf16", hq=32, hkv=8, dim=128, rotary=128, interleaved=False, norm=True, scaled=False,
             lens="1 1907 37 640 128 999 255 1300 16 77 511 1025 300", start="0 0 0 0 0 0 0 0 0 0 0 0 0"),
        # the bounds of the last blocks after a decoding step
        dict(name="bounds tokens", op="bounds", hkv=8, dim=128, block=32, lens=" ".join(str(1 + 37 * i % 1000) for i in range(64)), last=1),
        # the bounds of long contexts that have just been read
        dict(name="bounds long", op="bounds", hkv=8, dim=128, block=64, lens="65536 40000 32769 8000", last=0),
        # blocks for the next token of an ordinary decoding batch
        dict(name="choose batch", op="choose", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1,
             lens=" ".join(str(64 + 379 * i * i % 6000) for i in range(32)), count=16, sinks=1, recent=2),
        # blocks for the next token of long contexts
        dict(name="choose long", op="choose", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1,
             lens=" ".join(["65536"] * 15 + ["65521"]), count=64, sinks=1, recent=2),
        # one short conversation: latency
        dict(name="blocks short", op="blocks", type="f16", hq=8, hkv=2, dim=64, block=16, queries=1, lens="2000", count=16),
        # the next token of long contexts over a sixteenth of their blocks
        dict(name="blocks long", op="blocks", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1,
             lens=" ".join(["65536"] * 15 + ["65521"]), count=64),
        # four drafted tokens of contexts of very different lengths
        dict(name="blocks drafts", op="blocks", type="bf16", hq=24, hkv=8, dim=128, block=32, queries=4, lens="32768 20001 1000 15", count=64),
        # a few questions about one short text
        dict(name="shared few", op="shared", type="f16", hq=8, hkv=2, dim=64, block=16, queries=1, groups="4", prefix="700",
             lens="20 1 33 150"),
        # conversations that begin with three instructions of different lengths, one of them a single conversation's
        dict(name="shared groups", op="shared", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1, groups="40 1 23",
             prefix="6000 900 17001", lens=" ".join(str(1 + 379 * i * i % 2000) for i in range(64))),
        # many answers about one long document
        dict(name="shared long", op="shared", type="bf16", hq=32, hkv=8, dim=128, block=64, queries=1, groups="128", prefix="32768",
             lens=" ".join(str(1 + 37 * i % 500) for i in range(128))),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(rng, total, most):
    """1 to `most` lengths that sum to about `total`, some of them single tokens."""
    n = min(_spread(rng, 1, most), total)
    cuts = [rng.random() ** 2 + 1e-3 for _ in range(n)]
    return [1 if rng.random() < 0.1 else max(1, int(total * c / sum(cuts))) for c in cuts]


def _text(values):
    return " ".join(map(str, values))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and _plain_bytes(c) <= MOST_PLAIN:
            return c


def _draw(rng):
    op = rng.choice(("rotate", "rotate", "bounds", "choose", "choose", "blocks", "blocks", "shared", "shared"))
    typ, block = rng.choice(("bf16", "f16")), rng.choice((16, 32, 64, 128))
    hkv, g, dim = rng.choice((1, 2, 3, 4, 8, 8)), rng.choice((1, 2, 3, 4, 4, 6, 8, 16)), rng.choice((48, 64, 80, 96, 112, 128, 128, 128))
    if op == "rotate":
        lens = _lens(rng, _spread(rng, 1, 30000), 64)
        return dict(op=op, type=typ, hq=hkv * g, hkv=hkv, dim=dim, rotary=rng.choice((dim, dim, dim // 2, dim // 4)),
                    interleaved=rng.random() < 0.4, norm=rng.random() < 0.6, scaled=rng.random() < 0.4, lens=_text(lens),
                    start=_text([rng.choice((0, _spread(rng, 1, 2000000))) for _ in lens]))
    if op == "bounds":
        lens = _lens(rng, _spread(rng, 1, 300000), 64)
        return dict(op=op, hkv=hkv, dim=dim, block=block, lens=_text(lens), last=rng.choice((0, 0, 1, _spread(rng, 1, max(lens)))))
    if op == "shared":
        n = _spread(rng, 1, 128)
        groups = _lens(rng, n, 4)
        n = sum(groups)
        prefix = [rng.choice((0, _spread(rng, 1, 40000), _spread(rng, 100, 40000))) for _ in groups]
        lens = [rng.choice((0, 1, _spread(rng, 1, 600), _spread(rng, 1, 3000 if n < 40 else 900))) for _ in range(n)]
        return dict(op=op, type=typ, hq=hkv * g, hkv=hkv, dim=dim, block=block, queries=rng.choice((1, 1, 1, 2, 4)), groups=_text(groups),
                    prefix=_text(prefix), lens=_text(lens))
    lens = _lens(rng, _spread(rng, 1, 1000000), 64)
    queries, count = rng.choice((1, 1, 1, 2, 4)), _spread(rng, 1, 160)
    c = dict(op=op, type=typ, hq=hkv * g, hkv=hkv, dim=dim, block=block, queries=queries, lens=_text(lens), count=count)
    if op == "choose":
        # the longest sequence has something to choose from
        most = max(_blocks(lens, block))
        c |= dict(count=max(count, 8), sinks=rng.choice((0, 1, 1, 2)), recent=rng.choice((0, 1, 2, 4)))
        return c if most >= 24 and 2 * c["count"] <= most else _draw(rng)
    return c


def _blocks(lens, block):
    return [-(-n // block) for n in lens]


def _plain_bytes(c):
    """Bytes of the plain form's largest tensor, and of the cache."""
    lens, row = ints(c["lens"]), c["hkv"] * c["dim"]
    if c["op"] == "rotate":
        return sum(lens) * c["hq"] * c["dim"] * 4
    padded = len(lens) * max(_blocks(lens, c["block"]))
    if c["op"] == "bounds":
        return padded * c["block"] * row
    if c["op"] == "choose":
        return max(padded * row * 16, padded * c["block"] * row)
    if c["op"] == "blocks":
        return max(len(lens) * c["queries"] * c["count"] * c["block"] * row * 4, padded * c["block"] * row * 2)
    groups, prefix = ints(c["groups"]), ints(c["prefix"])
    rows = max(groups) * c["queries"] * c["hq"]
    return max(len(groups) * max(prefix) * max(row, rows) * 4, padded * c["block"] * max(row, c["queries"] * c["hq"]) * 4)


def work(case):
    op, d = case["op"], case["dim"]
    lens = ints(case["lens"])
    if op == "rotate":
        values = sum(lens) * (case["hq"] + case["hkv"]) * d
        return {"bytes": 4 * values + 4 * sum(lens), "flops": 6 * values}
    row, block = case["hkv"] * d, case["block"]
    if op == "bounds":
        first = [max(0, n - case["last"]) // block * block if case["last"] else 0 for n in lens]
        tokens = sum(n - f for n, f in zip(lens, first))
        blocks = sum(-(-n // block) - f // block for n, f in zip(lens, first))
        return {"bytes": row * (tokens + 2 * blocks), "flops": 2 * row * tokens}
    rows = len(lens) * case["queries"] * case["hq"]
    if op == "choose":
        blocks = sum(_blocks(lens, block))
        return {"bytes": 2 * rows * d + (2 * row + 4 * case["hkv"]) * blocks + 4 * len(lens) * case["queries"] * case["hkv"] * case["count"],
                "flops": 4 * case["queries"] * row * blocks}
    if op == "blocks":
        chosen = [min(n, case["count"] * block) for n in lens]
        # the tokens of different queries' blocks, of which most are the same where most are chosen
        held = sum(min(n, case["queries"] * m) for n, m in zip(lens, chosen))
        return {"bytes": 2 * row * held + 4 * rows * d + 4 * rows, "flops": 4 * case["queries"] * case["hq"] * d * sum(chosen)}
    groups, prefix = ints(case["groups"]), ints(case["prefix"])
    seen = sum(g * p for g, p in zip(groups, prefix)) + sum(lens)
    return {"bytes": 2 * row * (sum(prefix) + sum(lens)) + 4 * rows * d + 4 * rows, "flops": 4 * case["queries"] * case["hq"] * d * seen}


TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(values):
    return _i32([sum(values[:i]) for i in range(len(values) + 1)])


def _pool(g, blocks, case):
    """A pool of blocks as sequences have left it: codes of normal values around each block's own middle."""
    shape = (blocks, case["hkv"], case["block"], case["dim"])

    def codes():
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        middle = torch.randn((blocks, case["hkv"], 1, case["dim"]), generator=g, device="cuda", dtype=torch.float16)
        return x.mul_(34).add_(middle.mul_(16)).round_().clamp_(-127, 127).to(torch.int8)

    return [codes(), codes()] + [0.02 + 0.03 * torch.rand(shape[:2], generator=g, device="cuda") for _ in range(2)]


def _table(ids, counts):
    """Blocks of the sequences, in any order as a pool gives them out; -1 past the end."""
    width, first = max(max(counts), 1), _cu(counts)[:-1]
    col = torch.arange(width, device="cuda")[None]
    at = (first[:, None] + col).clamp(max=max(len(ids) - 1, 0))
    return torch.where(col < _i32(counts)[:, None], ids[at] if len(ids) else at, -1).to(torch.int32)


def _frequencies(rotary, scaled):
    """Radians a position of each pair, and the amplitude: base 10,000, or, scaled from 4,096 to 16 times as many
    positions, the pairs that turn less than once in 4,096 slowed down 16 times, those that turn over 32 times left,
    a mixture between."""
    f = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    if not scaled:
        return f, 1.0
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return f * (keep + (1 - keep) / 16), 1 + 0.1 * math.log(16.0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d, lens, op = case["dim"], ints(case["lens"]), case["op"]
    s = {"case": dict(case), "scale": 1.0 / math.sqrt(d)}
    if op == "rotate":
        # a projection's output: queries, keys and values of a token side by side
        heads, t = case["hq"] + 2 * case["hkv"], TYPES[case["type"]]
        x = torch.randn((sum(lens), heads, d), generator=g, device="cuda")
        x = x.mul_(0.5 + 2 * torch.rand((1, heads, d), generator=g, device="cuda")).to(t)
        start, cu = _i32(ints(case["start"])), _cu(lens).long()
        at = torch.arange(sum(lens), device="cuda")
        seq = torch.bucketize(at, cu[1:], right=True)
        freqs, amplitude = _frequencies(case["rotary"], case["scaled"])
        weights = [(0.5 + torch.rand(d, generator=g, device="cuda")).to(t) if case["norm"] else None for _ in range(2)]
        return s | {"q": x[:, :case["hq"]], "k": x[:, case["hq"]:case["hq"] + case["hkv"]], "weights": weights,
                    "positions": (start[seq] + at - cu[seq]).to(torch.int32), "freqs": freqs, "amplitude": amplitude}
    counts = _blocks(lens, case["block"])
    prefix = _blocks(ints(case["prefix"]), case["block"]) if op == "shared" else []
    ids = torch.randperm(sum(counts) + sum(prefix) + 1, generator=g, device="cuda").to(torch.int32)
    s["pool"] = _pool(g, len(ids), case)
    s |= {"table": _table(ids, counts), "lens": _i32(lens)}
    if op == "bounds":
        # what the blocks' bounds were before
        return s | {"bounds": torch.randint(-127, 128, (len(ids), case["hkv"], 2, d), generator=g, device="cuda", dtype=torch.int8)}
    q = torch.randn((len(lens), case["queries"], case["hq"], d), generator=g, device="cuda")
    s["q"] = q.mul_(1.5 * (0.5 + torch.rand((1, 1, case["hq"], d), generator=g, device="cuda"))).to(TYPES[case["type"]])
    if op == "choose":
        return s | {"bounds": torch.stack((s["pool"][0].amax(2), s["pool"][0].amin(2)), 2)}
    if op == "shared":
        cu, first = _cu(ints(case["groups"])), sum(counts)
        return s | {"cu": cu, "shared_table": _table(ids[first:], prefix), "shared_lens": _i32(ints(case["prefix"]))}
    # the blocks that each query and key head chose: the first, the last and any others, in order
    col = torch.arange(max(counts), device="cuda")
    n = torch.div(s["lens"][:, None] - case["queries"] + torch.arange(case["queries"], device="cuda") + case["block"], case["block"],
                  rounding_mode="floor").clamp(min=0)[:, :, None, None]           # blocks with tokens that a query sees
    like = torch.rand((len(lens), case["queries"], case["hkv"], len(col)), generator=g, device="cuda")
    like = torch.where(col >= n, -1.0, torch.where((col == 0) | (col == n - 1), 2.0, like))
    best, at = like.topk(min(case["count"], len(col)), -1)
    at = torch.where(best < 0, len(col), at).sort(-1).values
    at = torch.nn.functional.pad(at, (0, case["count"] - at.shape[-1]), value=len(col))
    return s | {"blocks": torch.where(at == len(col), -1, at).to(torch.int32)}


def run(state):
    return RUNS[state["case"]["op"]][1 if own else 0](state)


# ---- plain forms -----------------------------------------------------------

def plain_rotate(s):
    c = s["case"]
    half, by = c["rotary"] // 2, (2 if c["interleaved"] else 1)
    angle = s["positions"].double()[:, None] * s["freqs"]
    cos, sin = ((f(angle) * s["amplitude"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x, weight):
        y = x.float()
        if weight is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
        a, b = (y[..., 0:2 * half:2], y[..., 1:2 * half:2]) if by == 2 else (y[..., :half], y[..., half:2 * half])
        u, v = a * cos - b * sin, b * cos + a * sin
        pair = torch.stack((u, v), -1).flatten(-2) if by == 2 else torch.cat((u, v), -1)
        return torch.cat((pair, y[..., 2 * half:]), -1).to(x.dtype)

    return {"q": turned(s["q"], s["weights"][0]), "k": turned(s["k"], s["weights"][1])}


def plain_bounds(s):
    c, codes, bounds, block = s["case"], s["pool"][0], s["bounds"], s["case"]["block"]
    table, lens = s["table"].long(), s["lens"].long()[:, None]
    col = torch.arange(table.shape[1], device="cuda")[None]
    from_col = torch.div((lens - c["last"]).clamp(min=0), block, rounding_mode="floor") if c["last"] else 0
    mine = (col >= from_col) & (col * block < lens)
    ids = table[mine]
    left = (lens - col * block)[mine]
    gone = (torch.arange(block, device="cuda")[None] >= left[:, None])[:, None, :, None]
    x = codes[ids]
    bounds[ids] = torch.stack((x.masked_fill(gone, -128).amax(2), x.masked_fill(gone, 127).amin(2)), 2)
    return bounds


def _seen_tokens(s):
    """Tokens of the cache that each query sees, [B, queries]."""
    nq = s["case"]["queries"]
    return (s["lens"][:, None] - nq + 1 + torch.arange(nq, device="cuda")).clamp(min=0)


def plain_choose(s):
    c, q, count = s["case"], s["q"], s["case"]["count"]
    b, nq, hkv, g, d = q.shape[0], q.shape[1], c["hkv"], c["hq"] // c["hkv"], c["dim"]
    x = q.float().view(b, nq, hkv, g * d)
    top = x.abs().amax(-1, keepdim=True)
    by = torch.where(top < 1e-30, torch.zeros_like(top), 127 / top)
    code = torch.round(x * by).view(b, nq, hkv, g, d).double()
    pair = torch.stack((code.clamp(min=0).sum(3), code.clamp(max=0).sum(3)), 3).flatten(3)      # [B, queries, hkv, 2 D]
    table = s["table"].clamp(min=0).long()
    bounds = s["bounds"][table].double().flatten(3).transpose(1, 2)                              # [B, hkv, W, 2 D]
    score = torch.matmul(bounds, pair.permute(0, 2, 3, 1)).float() * s["pool"][2][table].transpose(1, 2)[..., None]
    score = score.permute(0, 3, 1, 2)
    col = torch.arange(table.shape[1], device="cuda")
    n = torch.div(_seen_tokens(s) + c["block"] - 1, c["block"], rounding_mode="floor")[:, :, None, None]
    kind = torch.where(col >= n, 2, torch.where((col < c["sinks"]) | (col >= n - c["recent"]) | (n <= count), 0, 1))
    order = torch.argsort(score, dim=-1, descending=True, stable=True)                           # ties: the lowest first
    order = order.gather(-1, torch.argsort(kind.expand_as(order).gather(-1, order), dim=-1, stable=True))[..., :count]
    taken = torch.where(torch.arange(order.shape[-1], device="cuda") < n, order, len(col)).sort(-1).values
    taken = torch.nn.functional.pad(taken, (0, count - taken.shape[-1]), value=len(col))
    return torch.where(taken == len(col), -1, taken).to(torch.int32)


def _softmax_out(scores, seen, values):
    """scores [..., q, k] in place; seen broadcasts to them.  (outputs, log of the sums)."""
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    scores.sub_(base).exp_()
    total = scores.sum(-1, keepdim=True)
    inv = torch.where(total > 0, 1 / total, torch.zeros_like(total))
    return torch.matmul(scores, values) * inv, (total.log() + base).squeeze(-1)


def plain_blocks(s):
    c, q, block = s["case"], s["q"], s["case"]["block"]
    b, nq, hkv, g, d = q.shape[0], q.shape[1], c["hkv"], c["hq"] // c["hkv"], c["dim"]
    kc, vc, ks, vs = s["pool"]
    cols = s["blocks"].clamp(min=0).long()
    ids = s["table"].long()[torch.arange(b, device="cuda")[:, None, None, None], cols]
    head = torch.arange(hkv, device="cuda")[None, None, :, None]
    pos = (cols[..., None] * block + torch.arange(block, device="cuda")).flatten(3)              # [B, queries, hkv, tokens]
    seen = (s["blocks"] >= 0).repeat_interleave(block, 3) & (pos < _seen_tokens(s)[:, :, None, None])
    k = kc[ids, head].float().mul_(ks[ids, head][..., None, None]).flatten(3, 4)
    scores = torch.matmul(q.float().mul(s["scale"]).view(b, nq, hkv, g, d), k.transpose(3, 4))
    del k
    v = vc[ids, head].float().mul_(vs[ids, head][..., None, None]).flatten(3, 4)
    out, lse = _softmax_out(scores, seen[:, :, :, None], v)
    return {"out": out.reshape(q.shape).to(q.dtype), "lse": lse.reshape(q.shape[:3])}


def _values(codes, scales, table):
    """[B, heads, tokens, D] of a table's blocks (block 0 in place of none)."""
    t = table.clamp(min=0).long()
    x = codes[t].float().mul_(scales[t][..., None, None])
    return x.permute(0, 2, 1, 3, 4).reshape(t.shape[0], codes.shape[1], -1, codes.shape[3])


def plain_shared(s):
    c, q = s["case"], s["q"]
    b, nq, hkv, g, d = q.shape[0], q.shape[1], c["hkv"], c["hq"] // c["hkv"], c["dim"]
    kc, vc, ks, vs = s["pool"]
    qh = q.float().mul(s["scale"]).view(b, nq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * nq, d)
    # the shared part: a group's sequences side by side, as many places as the largest group has
    cu, at = s["cu"].long(), torch.arange(b, device="cuda")
    group = torch.bucketize(at, cu[1:], right=True)
    place, most = at - cu[group], max(ints(c["groups"]))
    rows = torch.zeros((len(cu) - 1, hkv, most, g * nq, d), device="cuda")
    rows[group, :, place] = qh
    scores = torch.matmul(rows.flatten(2, 3), _values(kc, ks, s["shared_table"]).transpose(2, 3))
    seen = torch.arange(scores.shape[-1], device="cuda")[None, None, None] < s["shared_lens"][:, None, None, None]
    far, far_lse = _softmax_out(scores, seen, _values(vc, vs, s["shared_table"]))
    del scores
    far = far.view(rows.shape)[group, :, place]
    far_lse = far_lse.view(rows.shape[:4])[group, :, place]
    # each sequence's own part, then both as one
    scores = torch.matmul(qh, _values(kc, ks, s["table"]).transpose(2, 3))
    seen = torch.arange(scores.shape[-1], device="cuda") < _seen_tokens(s)[..., None]
    near, near_lse = _softmax_out(scores, seen[:, None].repeat(1, 1, g, 1), _values(vc, vs, s["table"]))
    top = torch.maximum(far_lse, near_lse)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w, u = torch.exp(far_lse - base), torch.exp(near_lse - base)
    total = w + u
    inv = torch.where(total > 0, 1 / total, torch.zeros_like(total))
    out = far * (w * inv)[..., None] + near * (u * inv)[..., None]
    back = lambda x: x.view(b, hkv, g, nq, -1).permute(0, 3, 1, 2, 4).reshape(b, nq, c["hq"], -1)  # noqa: E731
    return {"out": back(out).to(q.dtype), "lse": back((total.log() + base)[..., None])[..., 0].contiguous()}


# ---- the framework's operators ---------------------------------------------

def own_rotate(s):
    from beam_search_collab_b200 import memory
    q, k = memory.norm_rotate(s["q"], s["k"], s["positions"], s["freqs"], q_weight=s["weights"][0], k_weight=s["weights"][1], eps=1e-6,
                              interleaved=s["case"]["interleaved"], amplitude=s["amplitude"])
    return {"q": q, "k": k}


def own_bounds(s):
    from beam_search_collab_b200 import memory
    cache = memory.TokenCache(*s["pool"])
    return cache.update_bounds(s["bounds"], s["table"], s["lens"], last=s["case"]["last"] or None)


def own_choose(s):
    from beam_search_collab_b200 import memory
    cache, c = memory.TokenCache(*s["pool"]), s["case"]
    return cache.choose_blocks(s["q"], s["bounds"], s["table"], s["lens"], c["count"], sinks=c["sinks"], recent=c["recent"])


def own_blocks(s):
    from beam_search_collab_b200 import memory
    cache = memory.TokenCache(*s["pool"])
    out, lse = cache.block_attention(s["q"], s["table"], s["lens"], s["blocks"], scale=s["scale"], with_lse=True)
    return {"out": out, "lse": lse}


def own_shared(s):
    from beam_search_collab_b200 import memory
    cache = memory.TokenCache(*s["pool"])
    out, lse = cache.shared_attention(s["q"], s["shared_table"], s["shared_lens"], s["cu"], s["table"], s["lens"], scale=s["scale"],
                                      with_lse=True)
    return {"out": out, "lse": lse}


RUNS = {"rotate": (plain_rotate, own_rotate), "bounds": (plain_bounds, own_bounds), "choose": (plain_choose, own_choose),
        "blocks": (plain_blocks, own_blocks), "shared": (plain_shared, own_shared)}


# ---- definitions in 64 bits ------------------------------------------------

def exact(case, seed):
    """The operators' definitions, a head of a sequence at a time.  (Bounds and choices are whole numbers.)"""
    if case["op"] in ("bounds", "choose"):
        return None
    s, lens, d = prepare(case, seed), ints(case["lens"]), case["dim"]
    if case["op"] == "rotate":
        res = {}
        for name, weight in zip("qk", s["weights"]):
            x = s[name].double()
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * weight.double()
            y, half = x.clone(), case["rotary"] // 2
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                z = torch.polar(torch.full_like(s["positions"], s["amplitude"], dtype=torch.float64), s["positions"].double() * s["freqs"][i])
                turned = torch.complex(x[..., a], x[..., b]) * z[:, None]
                y[..., a], y[..., b] = turned.real, turned.imag
            res[name] = y
        return res
    nq, g, block = case["queries"], case["hq"] // case["hkv"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:3], dtype=torch.float64, device="cuda")

    def part(table, n, h, i):
        """The first n tokens of a list of blocks: keys (i 0) or values (1)."""
        t = table[:-(-n // block)].long()
        return (s["pool"][i][t, h].double() * s["pool"][2 + i][t, h].double()[:, None, None]).reshape(-1, d)[:n]

    def attend(q, k, v):
        if not len(k):
            return torch.zeros_like(q), -math.inf
        z = (q @ k.T) * s["scale"]
        a = torch.logsumexp(z, -1)
        return torch.exp(z - a[:, None]) @ v, a

    if case["op"] == "blocks":
        for b, n in enumerate(lens):
            for i in range(nq):
                seen = max(0, n - nq + 1 + i)
                for h in range(case["hkv"]):
                    cols = s["blocks"][b, i, h].long()
                    cols = cols[cols >= 0]
                    at = (cols[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
                    ids = s["table"][b, cols].long()
                    k, v = ((s["pool"][x][ids, h].double() * s["pool"][2 + x][ids, h].double()[:, None, None]).reshape(-1, d)[at < seen]
                            for x in (0, 1))
                    to = (b, i, slice(h * g, h * g + g))
                    out[to], lse[to] = attend(s["q"][to].double(), k, v)
        return {"out": out, "lse": lse}
    first = 0
    for m, (size, p) in enumerate(zip(ints(case["groups"]), ints(case["prefix"]))):
        for h in range(case["hkv"]):
            far_k, far_v = (part(s["shared_table"][m], p, h, x) for x in (0, 1))
            # rows of all sequences of the group over what they share, then each over its own
            q = s["q"][first:first + size, :, h * g:h * g + g].double()
            z = (q.reshape(-1, d) @ far_k.T) * s["scale"]
            far_lse = torch.logsumexp(z, -1) if p else torch.full((len(z),), -math.inf, dtype=torch.float64, device="cuda")
            far = (torch.exp(z - far_lse[:, None]) @ far_v if p else torch.zeros((len(z), d), dtype=torch.float64, device="cuda")).view(q.shape)
            far_lse = far_lse.view(q.shape[:3])
            for j in range(size):
                n = lens[first + j]
                k, v = (part(s["table"][first + j], n, h, x) for x in (0, 1))
                for i in range(nq):
                    seen = max(0, n - nq + 1 + i)
                    near, near_lse = attend(q[j, i], k[:seen], v[:seen])
                    to = (first + j, i, slice(h * g, h * g + g))
                    if not p and not seen:
                        lse[to] = -math.inf
                        continue
                    near_lse = torch.as_tensor(near_lse, dtype=torch.float64, device="cuda").expand(g)
                    lse[to] = torch.logaddexp(far_lse[j, i], near_lse)
                    out[to] = far[j, i] * torch.exp(far_lse[j, i] - lse[to])[:, None] + near * torch.exp(near_lse - lse[to])[:, None]
        first += size
    return {"out": out, "lse": lse}
