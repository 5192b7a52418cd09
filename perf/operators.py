"""Operators around a 4-bit KV cache and a model's answers: their cases, plain forms and exact values.

Three operators, as a program that serves a model runs them:

* ``write``   new keys and values are quantised to 4 bits into the cache (affine, groups of 64 channels: a code 0..15 per
              channel, a scale and a bias per group, the layout of the packed weights) and read back;
* ``read``    a range of the cache is read back as dense keys and values;
* ``attend``  softmax attention of T new positions over the cache (T = 1: one token; 16: a verify block; hundreds: a chunk of
              a prompt), grouped heads, lengths per sequence, an optional mask;
* ``score``   log-probabilities of given tokens with the entropy and the most likely alternatives of every row of logits.

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits.
"""
import math
import random

import torch

own = False

GROUP = 64
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one decoded token of one sequence enters a cache of 4 KV heads of 256: latency
        {"name": "write_token", "op": "write", "dtype": "bf16", "B": 1, "Hk": 4, "D": 256, "T": 1, "cap": 8192, "start": 4097, "lens_seed": 0},
        # a padded batch of verify blocks, every sequence at its own position with its own number of new tokens
        {"name": "write_blocks", "op": "write", "dtype": "f16", "B": 8, "Hk": 2, "D": 128, "T": 16, "cap": 4096, "start": -1, "lens_seed": 3},
        # a chunk of two prompts
        {"name": "write_prompt", "op": "write", "dtype": "bf16", "B": 2, "Hk": 4, "D": 256, "T": 4133, "cap": 8192, "start": 1000, "lens_seed": 0},
        # a long prefix leaves the cache (handed to another worker, or checked)
        {"name": "read_prefix", "op": "read", "dtype": "bf16", "B": 1, "Hk": 4, "D": 256, "T": 65537, "cap": 66048, "start": 0, "lens_seed": 0},
        # one decoded token over a short context, 24 query heads on 4 KV heads: latency
        {"name": "attend_token", "op": "attend", "dtype": "bf16", "B": 1, "Hq": 24, "Hk": 4, "D": 256, "T": 1, "N": 4097, "ragged": False, "mask": "none", "lens_seed": 0},
        # one decoded token each for a batch of long conversations of different lengths
        {"name": "attend_tokens", "op": "attend", "dtype": "bf16", "B": 16, "Hq": 16, "Hk": 2, "D": 256, "T": 1, "N": 32768, "ragged": True, "mask": "none", "lens_seed": 5},
        # the 16-token verify block of the dense model at a usual context
        {"name": "attend_block", "op": "attend", "dtype": "bf16", "B": 1, "Hq": 24, "Hk": 4, "D": 256, "T": 16, "N": 8192, "ragged": False, "mask": "none", "lens_seed": 0},
        # the verify block at a very long context
        {"name": "attend_block_long", "op": "attend", "dtype": "bf16", "B": 1, "Hq": 16, "Hk": 2, "D": 256, "T": 16, "N": 131072, "ragged": False, "mask": "none", "lens_seed": 0},
        # verify blocks of a left-padded batch: a boolean mask hides each sequence's padding
        {"name": "attend_padded", "op": "attend", "dtype": "f16", "B": 4, "Hq": 16, "Hk": 4, "D": 128, "T": 16, "N": 5001, "ragged": False, "mask": "left", "lens_seed": 9},
        # a chunk of a prompt over what the cache holds
        {"name": "attend_prompt", "op": "attend", "dtype": "bf16", "B": 1, "Hq": 24, "Hk": 4, "D": 256, "T": 500, "N": 9001, "ragged": False, "mask": "none", "lens_seed": 0},
        # the verify block's logits: the drafted tokens' log-probabilities, with 20 alternatives
        {"name": "score_block", "op": "score", "dtype": "bf16", "R": 16, "V": 151936, "k": 20, "temperature": 1.0, "suppress": False},
        # scoring a prompt
        {"name": "score_prompt", "op": "score", "dtype": "bf16", "R": 1999, "V": 151936, "k": 5, "temperature": 0.7, "suppress": True},
    ]


HEADS = [(24, 4), (16, 2), (16, 4), (8, 8), (8, 1), (20, 4), (32, 2), (6, 2)]


def _log_range(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "score"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    seed = rng.randrange(1 << 20)
    hq, hk = rng.choice(HEADS)
    D = rng.choice([128, 256])
    if op in ("write", "read"):
        B = _log_range(rng, 1, 16)
        T = _log_range(rng, 1, max(1, (1 << 25) // (B * hk * D)))
        start = rng.choice([0, 1, 777]) if op == "read" else rng.choice([-1, 0, 33])
        return {"op": op, "dtype": dtype, "B": B, "Hk": hk, "D": D, "T": T, "cap": T + 1024, "start": start, "lens_seed": seed}
    if op == "attend":
        B = _log_range(rng, 1, 16)
        T = rng.choice([1, 1, rng.randint(2, 15), 16, 16, _log_range(rng, 17, 500)])
        most = min(131072, (1 << 28) // (B * hk * D), 100_000_000 // (B * hq * T))
        N = max(T, _log_range(rng, 1, most))
        return {"op": op, "dtype": dtype, "B": B, "Hq": hq, "Hk": hk, "D": D, "T": T, "N": N, "ragged": B > 1 and rng.random() < 0.5,
                "mask": rng.choice(["none", "none", "left", "bias"]), "lens_seed": seed}
    R = _log_range(rng, 1, 1999)
    V = _log_range(rng, 257, 151936)
    return {"op": op, "dtype": rng.choice(["bf16", "f16", "f32"]), "R": R if R * V < 80_000_000 else max(1, 80_000_000 // V), "V": V,
            "k": rng.choice([0, 1, 5, 20]), "temperature": rng.choice([1.0, 0.6, 1.3]), "suppress": rng.random() < 0.4}


def _lengths(case):
    """Keys that each sequence holds, the T new positions among them."""
    if not case["ragged"]:
        return [case["N"]] * case["B"]
    r = random.Random(case["lens_seed"])
    return [min(case["N"], case["T"] + int((case["N"] - case["T"]) * r.random() ** 0.7)) for _ in range(case["B"])]


def _places(case):
    """First position and number of new rows of each sequence of a write."""
    B, T, room = case["B"], case["T"], case["cap"] - case["T"]
    if case["start"] >= 0:
        return [case["start"]] * B, [T] * B
    r = random.Random(case["lens_seed"])
    return [r.randint(0, room) for _ in range(B)], [r.randint(0, T) for _ in range(B)]


def work(case):
    if case["op"] == "score":
        size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
        n = case["R"] * case["V"]
        return {"bytes": n * size + case["R"] * (12 + 8 * case["k"]) + (case["V"] if case["suppress"] else 0), "flops": 6 * n}
    D = case["D"]
    row = D // 2 + 2 * 2 * (D // GROUP)                      # a key or value in the cache: codes, scales, biases
    if case["op"] == "attend":
        keys = sum(_lengths(case))
        rows = case["B"] * case["Hq"] * case["T"]
        seen = sum(max(0, n - (case["T"] - 1) / 2) for n in _lengths(case)) * case["Hq"] * case["T"]
        mask = case["B"] * case["N"] if case["mask"] == "left" else 2 * case["Hq"] * case["T"] * case["N"] if case["mask"] == "bias" else 0
        return {"bytes": 2 * case["Hk"] * keys * row + 4 * rows * D + mask, "flops": 4 * seen * D}
    n = case["B"] * case["Hk"] * case["T"]
    if case["op"] == "read":
        return {"bytes": 2 * n * (row + 2 * D), "flops": 4 * n * D}
    new = case["Hk"] * sum(_places(case)[1])
    # new rows are read and their codes written; the whole block is read back
    return {"bytes": 2 * (new * (2 * D + row) + n * (row + 2 * D)), "flops": 2 * (6 * new * D + 2 * n * D)}


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _quantise(x):
    """x [..., D] -> codes [..., D / 8] (eight to an int32, the first in the lowest bits), scales and biases [..., D / 64]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = (hi / 15 - lo / 15).to(x.dtype)
    bias = lo.to(x.dtype)
    s = scale.float()
    n = torch.where(s > 0, torch.round((g - bias.float()) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(g))
    n = n.clamp(0, 15).to(torch.int64).flatten(-2).unflatten(-1, (-1, 8))
    words = (n << (4 * torch.arange(8, device=x.device))).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    return words, scale.squeeze(-1), bias.squeeze(-1)


def _dequantise(words, scales, biases):
    """float32 [..., D]"""
    n = (words.unsqueeze(-1) >> (4 * torch.arange(8, device=words.device, dtype=torch.int32))) & 15
    n = n.flatten(-2).unflatten(-1, (-1, GROUP)).float()
    return (n * scales.float().unsqueeze(-1) + biases.float().unsqueeze(-1)).flatten(-2)


def _plain_write(s):
    B, Hk, T, D = s["keys"].shape
    at = s["offsets"].long()[:, None] + torch.arange(T, device=s["keys"].device)                      # [B, T]
    new = torch.arange(T, device=at.device)[None] < s["counts"].long()[:, None]
    out = []
    for x, cache in ((s["keys"], s["k_cache"]), (s["values"], s["v_cache"])):
        for part, store in zip(_quantise(x), cache):
            where = at[:, None, :, None].expand(B, Hk, T, store.shape[-1])
            store.scatter_(2, where, torch.where(new[:, None, :, None], part, store.gather(2, where)))
        rows = [store.gather(2, at[:, None, :, None].expand(B, Hk, T, store.shape[-1])) for store in cache]
        out.append(_dequantise(*rows).to(x.dtype))
    return tuple(out)


def _plain_read(s):
    t0, n = s["start"], s["length"]
    return tuple(_dequantise(*[p[:, :, t0:t0 + n] for p in c]).to(c[1].dtype) for c in (s["k_cache"], s["v_cache"]))


def _plain_attend(s):
    q, N = s["queries"], s["max_length"]
    B, Hq, T, D = q.shape
    Hk = s["k_cache"][0].shape[1]
    k, v = (_dequantise(*[p[:, :, :N] for p in c]) for c in (s["k_cache"], s["v_cache"]))
    x = q.float().view(B, Hk, Hq // Hk * T, D) @ k.transpose(-1, -2) * s["scale"]
    x = x.view(B, Hq, T, N)
    n = torch.arange(N, device=q.device)
    last = s["lengths"].long()[:, None] - T + torch.arange(T, device=q.device)                        # [B, T]
    seen = (n <= last[..., None])[:, None]
    if s["mask"] is not None:
        if s["mask"].dtype == torch.bool:
            seen = seen & s["mask"]
        else:
            x = x + s["mask"].float()
    x = x.masked_fill(~seen, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
    p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    o = p.view(B, Hk, Hq // Hk * T, N) @ v
    return o.view(B, Hq, T, D).to(q.dtype)


def _plain_score(s):
    x = s["logits"].float()
    if s["suppress"] is not None:
        x = x.masked_fill(s["suppress"], -math.inf)
    R, V = x.shape
    y = x / s["temperature"]
    y = y - y.amax(-1, keepdim=True)
    e = torch.exp(y)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - (torch.where(e > 0, e * y, torch.zeros_like(e))).sum(-1, keepdim=True) / total)[:, 0]
    logprobs = y.gather(1, s["tokens"].long()[:, None])[:, 0] - log_total[:, 0]
    # a logit's bits as a whole number of the same order, ties to the lower index
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + (V - 1 - torch.arange(V, device=x.device))
    ids = key.topk(s["k"], -1).indices
    return logprobs, entropy, y.gather(1, ids) - log_total, ids.to(torch.int32)


# ---- inputs and passes -----------------------------------------------------------------------------------------------
def _states(gen, shape, dtype, dev):
    """Keys or values: normal, with a spread and an offset of their own in each channel and a few strong channels."""
    D = shape[-1]
    spread = 0.5 + torch.rand(D, generator=gen, device=dev)
    spread[torch.randint(0, D, (max(1, D // 64),), generator=gen, device=dev)] *= 4
    offset = 0.5 * torch.randn(D, generator=gen, device=dev)
    return (torch.randn(shape, generator=gen, device=dev) * spread + offset).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "score":
        R, V = case["R"], case["V"]
        x = 2.0 * torch.randn(R, V, generator=gen, device=dev)
        x.scatter_add_(1, torch.randint(0, V, (R, 8), generator=gen, device=dev), 12.0 * torch.rand(R, 8, generator=gen, device=dev))
        x = x.to(dtype)
        likely = torch.randint(0, V, (R, 64), generator=gen, device=dev)
        tokens = likely.gather(1, x.gather(1, likely).argmax(1, keepdim=True))[:, 0].to(torch.int32)
        suppress = None
        if case["suppress"]:
            suppress = torch.rand(V, generator=gen, device=dev) < 0.01
            suppress[tokens.long()] = False
        return {"op": "score", "logits": x, "tokens": tokens, "k": case["k"], "temperature": case["temperature"], "suppress": suppress}
    B, Hk, D, T = case["B"], case["Hk"], case["D"], case["T"]
    cap = case["cap"] if "cap" in case else case["N"] + 37
    caches = [tuple(p.contiguous() for p in _quantise(_states(gen, (B, Hk, cap, D), dtype, dev))) for _ in range(2)]
    s = {"op": case["op"], "k_cache": caches[0], "v_cache": caches[1]}
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    if case["op"] == "write":
        at, counts = _places(case)
        s.update(keys=_states(gen, (B, Hk, T, D), dtype, dev), values=_states(gen, (B, Hk, T, D), dtype, dev), offsets=whole(at),
                 counts=whole(counts))
    elif case["op"] == "read":
        s.update(start=case["start"], length=T)
    else:
        N, Hq = case["N"], case["Hq"]
        mask = None
        if case["mask"] == "left":          # a sequence's first positions are padding
            pads = [random.Random(case["lens_seed"] + 7 * b).randint(0, max(0, N - T) // 2) for b in range(B)]
            mask = torch.arange(N, device=dev)[None, None, None, :] >= whole(pads)[:, None, None, None]
        elif case["mask"] == "bias":        # a slope per head over the distance
            slopes = torch.pow(2.0, -torch.arange(1, Hq + 1, device=dev) / 2.0)[None, :, None, None]
            far = (N - T + torch.arange(T, device=dev)[:, None] - torch.arange(N, device=dev)[None]).clamp_min(0)
            mask = (-slopes * far).clamp_min(-60000.0).to(dtype)
        s.update(queries=(1.5 * torch.randn(B, Hq, T, D, generator=gen, device=dev)).to(dtype), scale=D ** -0.5,
                 lengths=whole(_lengths(case)), max_length=N, mask=mask)
    return s


def run(state):
    s = state
    if own:
        from dflash_mlx_b200 import logprobs, quantized_kv
        if s["op"] == "write":
            quantized_kv.quantized_kv_write(s["keys"], s["values"], s["k_cache"], s["v_cache"], s["offsets"], counts=s["counts"])
            return quantized_kv.quantized_kv_read(s["k_cache"], s["v_cache"], s["offsets"], s["keys"].shape[2])
        if s["op"] == "read":
            return quantized_kv.quantized_kv_read(s["k_cache"], s["v_cache"], s["start"], s["length"])
        if s["op"] == "attend":
            return quantized_kv.quantized_kv_sdpa(s["queries"], s["k_cache"], s["v_cache"], s["scale"], s["lengths"], s["mask"],
                                                  max_length=s["max_length"])
        return logprobs.token_logprobs(s["logits"], s["tokens"], top_k=s["k"], temperature=s["temperature"], suppress=s["suppress"])
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "score": _plain_score}[s["op"]](s)


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------
def _exact_values(words, scales, biases):
    D = words.shape[-1] * 8
    got = torch.empty(*words.shape[:-1], D, dtype=torch.float64, device=words.device)
    for i in range(8):
        got[..., i::8] = torch.bitwise_and(torch.bitwise_right_shift(words.long() & 0xFFFFFFFF, 4 * i), 15).double()
    of = torch.arange(D, device=words.device) // GROUP
    return got * scales.double()[..., of] + biases.double()[..., of]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "read":
        t = slice(s["start"], s["start"] + s["length"])
        return tuple(_exact_values(*[p[:, :, t] for p in c]) for c in (s["k_cache"], s["v_cache"]))
    if case["op"] == "write":
        out = []
        for x, cache in ((s["keys"], s["k_cache"]), (s["values"], s["v_cache"])):
            B, Hk, T, D = x.shape
            got = torch.empty(B, Hk, T, D, dtype=torch.float64, device=x.device)
            g = x.double().view(B, Hk, T, D // GROUP, GROUP)
            least, most = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            step = (most / 15 - least / 15).float().to(x.dtype).double()
            kept = least + step * torch.round((g - least) / step.clamp_min(1e-300)).clamp(0, 15)
            kept = kept.view(B, Hk, T, D)
            for b in range(B):
                o, c = int(s["offsets"][b]), int(s["counts"][b])
                got[b, :, :c] = kept[b, :, :c]
                got[b, :, c:] = _exact_values(*[p[b, :, o + c:o + T] for p in cache])
            out.append(got)
        return tuple(out)
    if case["op"] == "attend":
        q = s["queries"].double()
        B, Hq, T, D = q.shape
        Hk = s["k_cache"][0].shape[1]
        out = torch.zeros_like(q)
        for b in range(B):
            n = int(s["lengths"][b])
            for h in range(Hk):
                k, v = (_exact_values(*[p[b, h, :n] for p in c]) for c in (s["k_cache"], s["v_cache"]))
                mine = slice(h * (Hq // Hk), (h + 1) * (Hq // Hk))
                x = torch.einsum("gtd,nd->gtn", q[b, mine], k) * s["scale"]
                hidden = torch.arange(n, device=q.device)[None, None] > (n - T + torch.arange(T, device=q.device))[None, :, None]
                if s["mask"] is not None:
                    m = s["mask"].expand(B, Hq, T, s["mask"].shape[-1])[b, mine, :, :n]
                    if m.dtype == torch.bool:
                        hidden = hidden | ~m
                    else:
                        x = x + m.double()
                w = torch.softmax(x.masked_fill(hidden, -math.inf), -1)
                out[b, mine] = torch.einsum("gtn,nd->gtd", torch.nan_to_num(w), v)
        return out
    ids_all, lp, ent, tops = None, [], [], []
    order = s["logits"].clone()
    if s["suppress"] is not None:
        order[:, s["suppress"]] = -math.inf
    for r in range(0, case["R"], 256):
        x = order[r:r + 256].double() / s["temperature"]
        p = torch.log_softmax(x, -1)
        lp.append(p.gather(1, s["tokens"][r:r + 256].long()[:, None])[:, 0])
        ent.append(-torch.nan_to_num(p.exp() * p).sum(-1))
        tops.append(p.topk(case["k"], -1).values)
    return torch.cat(lp), torch.cat(ent), torch.cat(tops), ids_all
