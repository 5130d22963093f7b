"""The token-memory operators' definitions in 64 bits (plain torch, one head
of one sequence at a time), and the error bounds their results are held to."""
import math

import torch

# Unit roundoff of the types: half a unit in the last place of the significand.
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def attend(q, k, v, scale, limits):
    """q [n, D], k and v [m, D] in 64 bits; row i sees the first limits[i]
    keys.  Returns out, lse, weights [n, m], and what the bounds need: the
    sums of weight * |value| and the largest scale * sum |q k| of a row."""
    s = (q @ k.T) * scale
    hidden = torch.arange(k.shape[0], device=q.device)[None] >= limits[:, None]
    s = s.masked_fill(hidden, -math.inf)
    lse = torch.logsumexp(s, 1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.exp(s - lse[:, None])
    w[lse == -math.inf] = 0
    big = ((q.abs() @ k.abs().T) * abs(scale)).masked_fill(hidden, 0)
    big = big.amax(1) if k.shape[0] else torch.zeros_like(lse)
    return w @ v, lse, w, w @ v.abs(), big


def out_bound(ref, weighted, dtype, weights_unit):
    """Result rounded once (UNIT[dtype] of it); each weight rounded to
    weights_unit of it before it meets its value, and off by the exponential's
    and the score's 32-bit errors (under 2^-12 together at |score| < 2^8)."""
    return UNIT[dtype] * ref.abs() + (weights_unit + 2.0 ** -12) * weighted * (1 + 2.0 ** -7) + 1e-7 * weighted.amax().clamp(min=1e-30)


def lse_bound(big):
    """A sum of at most 128 products in 32 bits is off by 128 * 2^-24 of the
    sum of their magnitudes; exponential, sum and logarithm by 2^-17."""
    return 2.0 ** -17 * big + 2.0 ** -17


def mass_bound(mass, big):
    """Weights are off by the relative error e^(2 * lse_bound) - 1 of their
    exponent (score and lse), the sums by 2^-20 of themselves."""
    return (4 * (2.0 ** -17 * big + 2.0 ** -17) + 2.0 ** -20) * mass + 1e-12


def prompt(q, k, v, lens_q, lens_k, causal, scale):
    """(out, lse, weighted, big) of packed prompts, 64 bits."""
    g = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, weighted = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    big = torch.zeros_like(lse)
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        limits = torch.arange(nq, device=q.device) + nk - nq + 1 if causal else torch.full((nq,), nk, device=q.device)
        for h in range(q.shape[1]):
            o = attend(q[a:a + nq, h], k[b:b + nk, h // g], v[b:b + nk, h // g], scale, limits)
            out[a:a + nq, h], lse[a:a + nq, h], weighted[a:a + nq, h], big[a:a + nq, h] = o[0], o[1], o[3], o[4]
        a, b = a + nq, b + nk
    return out, lse, weighted, big


def held(pool, table, b, n, h, i):
    """Values of sequence b's first n tokens, head h: keys (i 0) or values (1)."""
    block = pool[0].shape[2]
    t = table[b, :-(-n // block)].long()
    x = pool[i][t, h].double() * pool[2 + i][t, h].double()[:, None, None]
    return x.reshape(-1, x.shape[-1])[:n]


def cache(pool, q, table, lens, scale):
    """(out, lse, weights per token [B, heads, width], weighted, big)."""
    n_seq, nq, hq, d = q.shape
    hkv = pool[0].shape[1]
    g = hq // hkv
    out, weighted = (torch.zeros(q.shape, dtype=torch.float64, device=q.device) for _ in range(2))
    lse, big = (torch.zeros(q.shape[:3], dtype=torch.float64, device=q.device) for _ in range(2))
    mass = torch.zeros((n_seq, hkv, table.shape[1] * pool[0].shape[2]), dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        limits = (torch.arange(nq, device=q.device) + n - nq + 1).repeat_interleave(g)
        for h in range(hkv):
            rows = q[b, :, h * g:h * g + g].reshape(nq * g, d).double()
            o = attend(rows, held(pool, table, b, n, h, 0), held(pool, table, b, n, h, 1), scale, limits)
            at = (b, slice(None), slice(h * g, h * g + g))
            out[at], lse[at], weighted[at], big[at] = o[0].view(nq, g, d), o[1].view(nq, g), o[3].view(nq, g, d), o[4].view(nq, g)
            mass[b, h, :n] = o[2].sum(0)
    return out, lse, mass, weighted, big


def random_pool(g, blocks, heads, block, dim, device="cuda"):
    codes = [torch.randint(-127, 128, (blocks, heads, block, dim), generator=g, device=device, dtype=torch.int8) for _ in range(2)]
    scales = [0.005 + 0.02 * torch.rand((blocks, heads), generator=g, device=device) for _ in range(2)]
    return codes + scales


def random_table(g, counts, spare=0, device="cuda"):
    """A table whose sequences have counts[b] blocks in any order, then the
    ids that are left."""
    at = torch.randperm(sum(counts) + spare, generator=g, device=device).to(torch.int32)
    table = torch.full((len(counts), max(max(counts), 1)), -1, dtype=torch.int32, device=device)
    used = 0
    for b, n in enumerate(counts):
        table[b, :n] = at[used:used + n]
        used += n
    return table, at[used:]


def cu(lens, device="cuda"):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=device)


def i32(x, device="cuda"):
    return torch.tensor(x, dtype=torch.int32, device=device)
