"""Operators between a served model's projections and behind its head, as cases that can be timed and checked: new keys and values
into a paged cache (with the norms and the rotation of queries and keys on the way), attention of new tokens over such a cache, and
the log-probabilities of given tokens with their ranks, the entropy and the likeliest alternatives.

Sizes are those of the package's own decoder (q 4096 and k/v 512 wide, as 32 and 4 heads of 128 or 16 and 2 of 256; a vocabulary of
151936; decode batches up to 32 rows and beyond, prompts in the hundreds and thousands), and spread around them by draw().

Where `own` is false, run() computes the operators in elementary torch operations; where it is true, it calls the package.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # one decoded token between qkv and o: the smallest call, bound by latency
        {"name": "append_1", "kind": "append", "tokens": 1, "heads": "32/4", "dim": 128, "page": 16, "rotary": 128, "axes": 1,
         "pairs": "half", "norms": True, "padding": 0, "dtype": "bf16", "cache": "bf16"},
        # a decode batch of 48 tokens, five of them the padding of a captured graph, positions of three axes (images and video)
        {"name": "append_48_axes", "kind": "append", "tokens": 48, "heads": "32/4", "dim": 128, "page": 16, "rotary": 128,
         "axes": 3, "pairs": "half", "norms": True, "padding": 5, "dtype": "bf16", "cache": "bf16"},
        # a ragged prompt into an 8-bit cache of large pages, a quarter of each head rotated
        {"name": "append_prompt_1531_e4m3", "kind": "append", "tokens": 1531, "heads": "16/2", "dim": 256, "page": 544,
         "rotary": 64, "axes": 1, "pairs": "half", "norms": True, "padding": 0, "dtype": "fp16", "cache": "e4m3"},
        # a full prefill batch
        {"name": "append_prompt_8192", "kind": "append", "tokens": 8192, "heads": "32/4", "dim": 128, "page": 64, "rotary": 128,
         "axes": 1, "pairs": "half", "norms": True, "padding": 0, "dtype": "bf16", "cache": "bf16"},
        # one request's next token a few tokens into its answer
        {"name": "attend_1", "kind": "attend", "requests": 1, "new": 1, "ragged_new": False, "length": 113, "ragged": False,
         "heads": "32/4", "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16"},
        # a decode batch of requests of very different lengths
        {"name": "attend_32", "kind": "attend", "requests": 32, "new": 1, "ragged_new": False, "length": 8171, "ragged": True,
         "heads": "32/4", "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16"},
        # one request far into a long document
        {"name": "attend_long_1", "kind": "attend", "requests": 1, "new": 1, "ragged_new": False, "length": 131072,
         "ragged": False, "heads": "32/4", "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16"},
        # a batch that verifies drafts over an 8-bit cache of large pages, wide heads
        {"name": "attend_drafts_40_e4m3", "kind": "attend", "requests": 40, "new": 4, "ragged_new": True, "length": 6001,
         "ragged": True, "heads": "16/2", "dim": 256, "page": 544, "window": 0, "dtype": "fp16", "cache": "e4m3"},
        # three prompts in one prefill batch, each behind tokens that the cache holds already
        {"name": "attend_prompt_3", "kind": "attend", "requests": 3, "new": 2048, "ragged_new": True, "length": 4096,
         "ragged": True, "heads": "32/4", "dim": 128, "page": 16, "window": 0, "dtype": "bf16", "cache": "bf16"},
        # the sampled token of one request, with the five likeliest
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 151936, "top": 5, "temperature": False, "masked": False,
         "dtype": "bf16"},
        # a decode batch at its temperatures over the 32-bit logits of a processor that masks tokens, with the twenty likeliest
        {"name": "logprobs_48", "kind": "logprobs", "rows": 48, "vocab": 151936, "top": 20, "temperature": True, "masked": True,
         "dtype": "fp32"},
        # the tokens of a prompt, over an odd vocabulary whose rows start at any element
        {"name": "logprobs_prompt_2043", "kind": "logprobs", "rows": 2043, "vocab": 151935, "top": 1, "temperature": False,
         "masked": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return "%d/%d" % (kv * rng.choice([1, 2, 4, 6, 8, 16]), kv)


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "logprobs"])
    if kind == "append":
        dim, heads = rng.choice([64, 128, 128, 256]), _heads(rng)
        width = dim * sum(_sizes(heads))
        tokens = _log(rng, 1, min(8192, 40_000_000 // width))
        return {"kind": kind, "tokens": tokens, "heads": heads, "dim": dim, "page": 16 * _log(rng, 1, 40),
                "rotary": rng.choice([dim, dim, dim // 2, dim // 4]), "axes": rng.choice([1, 1, 3]),
                "pairs": rng.choice(["half", "half", "adjacent"]), "norms": rng.random() < 0.7,
                "padding": rng.choice([0, min(tokens - 1, rng.randint(0, 9))]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
                "cache": rng.choice(["same", "same", "e4m3"])}
    if kind == "attend":
        dim, heads, prompt = rng.choice([64, 128, 128, 256]), _heads(rng), rng.random() < 0.3
        hq, hkv = _sizes(heads)
        new = _log(rng, 17, 2048) if prompt else rng.choice([1, 1, 1, 2, 3, 5, 8])
        length = new + _log(rng, 1, 4096 if prompt else 32760)
        # at most the elements of the long document's cache, and for prompts the products of the three prompts' batch
        products = 26_000_000_000 // (hq * dim)
        if length * new > products:
            new = max(1, products // length)
        most = min(67_000_000 // (length * hkv * dim), products // (length * new))
        return {"kind": kind, "requests": _log(rng, 1, max(1, min(64, most))), "new": new,
                "ragged_new": new > 1 and rng.random() < 0.6, "length": length, "ragged": rng.random() < 0.6, "heads": heads,
                "dim": dim, "page": 16 * _log(rng, 1, 40), "window": rng.choice([0, 0, 0, _log(rng, 16, 4096)]),
                "dtype": rng.choice(["bf16", "bf16", "fp16"]), "cache": rng.choice(["same", "same", "e4m3"])}
    vocab = _log(rng, 1000, 151936)
    return {"kind": kind, "rows": _log(rng, 1, min(4096, 300_000_000 // vocab)), "vocab": vocab, "top": rng.choice([0, 1, 5, 20, 64]),
            "temperature": rng.random() < 0.4, "masked": rng.random() < 0.4, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}


# ---- what a program has in hand

def _sizes(text):
    return [int(v) for v in text.split("/")]


def _cache_dtype(c):
    return DTYPES[c["dtype"] if c["cache"] == "same" else c["cache"]]


def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device=DEV) * scale


def _int(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _counts(c):
    """The new tokens of every request, and its tokens in the cache with them."""
    new, length, far = c["new"], c["length"], c["length"] - c["new"]
    n = [new - i * 7919 % (new // 2 + 1) if c["ragged_new"] else new for i in range(c["requests"])]
    return n, [v + far * (i * 37 % 64 + 1) // 64 if c["ragged"] else length - new + v for i, v in enumerate(n)]


def _paged(shape, gen, dtype):
    return _normal(shape, gen).to(dtype)


def _frequencies(c):
    """The angles' factors for a rotation of `rotary` elements a head, and the axis of each: with three axes the first half of
    them for time, a quarter each for height and width."""
    half = c["rotary"] // 2
    inv_freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    at = torch.arange(half, device=DEV) * 4 // max(half, 1)
    return inv_freq, (at - 1).clamp(min=0).to(torch.int32) if c["axes"] == 3 else torch.zeros_like(at, dtype=torch.int32)


def _append_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, (hq, hkv), T, D, page = DTYPES[c["dtype"]], _sizes(c["heads"]), c["tokens"], c["dim"], c["page"]
    qkv = _normal((T, (hq + 2 * hkv) * D), gen, 1.5).to(dtype)
    pages = -(-2 * T // page) + 1                                # page 0 belongs to nobody
    slots = page + torch.randperm((pages - 1) * page, generator=gen, device=DEV)[:T]
    if T > 64:                                                   # a prompt: its tokens stand in order in pages of any order
        order = 1 + torch.randperm(pages - 1, generator=gen, device=DEV)
        t = torch.arange(T, device=DEV)
        slots = order[t // page] * page + t % page
        positions = (t + 1000).expand(c["axes"], T).contiguous()
    else:
        positions = torch.randint(0, 200_000, (c["axes"], T), generator=gen, device=DEV)
    if c["axes"] > 1 and T > 64:                                 # an image of 32 x 32 patches in its midst
        inside = (t > T // 4) & (t <= T // 4 + 1024)
        positions = torch.where(inside, positions[:, T // 4:T // 4 + 1], positions)
        positions[1] += torch.where(inside, (t - T // 4) // 32, 0)
        positions[2] += torch.where(inside, (t - T // 4) % 32, 0)
    if c["padding"]:
        slots[T - c["padding"]:] = -1
    inv_freq, axes = _frequencies(c)
    weight = lambda: (1 + _normal((D,), gen, 0.1)).to(dtype)  # noqa: E731
    shape = (pages, page, hkv, D)
    return {"q": qkv[:, :hq * D].view(T, hq, D), "k": qkv[:, hq * D:(hq + hkv) * D].view(T, hkv, D),
            "v": qkv[:, (hq + hkv) * D:].view(T, hkv, D), "positions": positions.contiguous(), "slots": slots,
            "inv_freq": inv_freq, "axes": axes, "adjacent": c["pairs"] == "adjacent",
            "q_norm": weight() if c["norms"] else None, "k_norm": weight() if c["norms"] else None,
            "cache_k": _paged(shape, gen, _cache_dtype(c)), "cache_v": _paged(shape, gen, _cache_dtype(c)), **_scales(c, hkv)}


def _scales(c, hkv):
    if c["cache"] != "e4m3":
        return {"k_scale": None, "v_scale": None}
    return {"k_scale": 0.02 + 0.01 * torch.arange(hkv, device=DEV) / hkv, "v_scale": torch.full((hkv,), 0.03, device=DEV)}


def _attend_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, (hq, hkv), D, page = DTYPES[c["dtype"]], _sizes(c["heads"]), c["dim"], c["page"]
    n, lengths = _counts(c)
    held = [-(-v // page) for v in lengths]
    pages = sum(held) + 1                                        # page 0 belongs to nobody: what tables hold past their ends
    order = 1 + torch.randperm(pages - 1, generator=gen, device=DEV)
    first = _int([sum(held[:i]) for i in range(len(held))], torch.int64)[:, None]
    at = torch.arange(max(held), device=DEV)[None, :]
    mine = at < _int(held)[:, None]
    tables = torch.where(mine, order[torch.where(mine, first + at, 0)], 0).to(torch.int32)
    shape, spread = (pages, hkv, page, D), 30.0 if c["cache"] == "e4m3" else 1.0   # 8 bits: values over the scale
    k, v = (_normal(shape, gen, spread).to(_cache_dtype(c)).transpose(1, 2) for _ in range(2))
    return {"q": _normal((sum(n), hq, D), gen, 1.5).to(dtype), "cache_k": k, "cache_v": v, "tables": tables,
            "lengths": _int(lengths), "first": _int([sum(n[:i]) for i in range(len(n))]), "n": _int(n), "new": max(n),
            "window": c["window"], **_scales(c, hkv)}


def _logprobs_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    R, V = c["rows"], c["vocab"]
    logits = _normal((R, V), gen, 3.0)
    if c["masked"]:                                              # a grammar's or a filter's mask over a third of the tokens
        logits[torch.rand((R, V), generator=gen, device=DEV) < 0.33] = -math.inf
    tokens = torch.randint(0, V, (R,), generator=gen, device=DEV)
    likely = (logits + torch.empty((R, V), device=DEV).exponential_(generator=gen).log_().neg_()).argmax(-1)
    tokens = torch.where(torch.arange(R, device=DEV) % 4 == 3, tokens, likely)
    temperature = 0.5 + 0.1 * (torch.arange(R, device=DEV) % 9) if c["temperature"] else None
    return {"logits": logits.to(DTYPES[c["dtype"]]), "tokens": tokens.to(torch.int32), "top": c["top"], "temperature": temperature}


INPUTS = {"append": _append_inputs, "attend": _attend_inputs, "logprobs": _logprobs_inputs}


def prepare(case, seed):
    s = INPUTS[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    if case["kind"] != "logprobs":
        s["out"] = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device=DEV)
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-espalier_amd"))
        if case["kind"] == "logprobs":
            from vllm_espalier.logprobs import token_logprobs
            s["call"] = token_logprobs
        else:
            from vllm_espalier.attention import PagedCache, Rotary
            s["cache"] = PagedCache(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
            if case["kind"] == "append":
                s["rotary"] = Rotary(s["inv_freq"], axes=s["axes"], adjacent=s["adjacent"])
    return s


# ---- the operators

def _values(s):
    """The cache as the values it stands for."""
    if s["k_scale"] is None:
        return s["cache_k"], s["cache_v"]
    return ((s["cache_k"].float() * s["k_scale"][:, None]).to(s["q"].dtype),
            (s["cache_v"].float() * s["v_scale"][:, None]).to(s["q"].dtype))


def _own(s):
    if s["kind"] == "append":
        q = s["cache"].append(s["q"], s["k"], s["v"], s["slots"], s["positions"], s["rotary"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], eps=EPS, out=s["out"])
        return (q, *_values(s))
    if s["kind"] == "attend":
        return s["cache"].attend(s["q"], s["tables"], s["lengths"], first=s["first"], n_new=s["n"], max_new=s["new"],
                                 window=s["window"], out=s["out"])
    return s["call"](s["logits"], s["tokens"], top=s["top"], temperature=s["temperature"])


def _plain_turn(x, weight, cos, sin, adjacent):
    """Rows [T, H, D] through their norm (if any) and the rotation of their first 2 * cos.shape[1] elements."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    half = cos.shape[-1]
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    pairs = turned.reshape(*x.shape[:2], half, 2) if adjacent else turned.reshape(*x.shape[:2], 2, half).transpose(-1, -2)
    a, b = pairs[..., 0], pairs[..., 1]
    both = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1)
    turned = (both if adjacent else both.transpose(-1, -2)).reshape(*x.shape[:2], 2 * half)
    return torch.cat([turned, rest], dim=-1)


def _plain_store(cache, slots, rows, scale):
    page = cache.shape[1]
    if scale is not None:
        rows = (rows / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    bits = torch.uint8 if cache.dtype == DTYPES["e4m3"] else cache.dtype
    kept, rows, at = cache.view(bits), rows.to(cache.dtype).view(bits), slots.clamp(min=0)
    where = (at // page, at % page)                              # rows without a slot: nobody's first one, left as it is
    kept[where] = torch.where((slots >= 0)[:, None, None], rows, kept[where])


def _plain_append(s):
    # the angles in 64 bits: a far position leaves few of 32 for the fraction of a turn
    angle = s["positions"][s["axes"].long()].double().t() * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    s["out"].copy_(_plain_turn(s["q"], s["q_norm"], cos, sin, s["adjacent"]))
    _plain_store(s["cache_k"], s["slots"], _plain_turn(s["k"], s["k_norm"], cos, sin, s["adjacent"]), s["k_scale"])
    _plain_store(s["cache_v"], s["slots"], s["v"].float(), s["v_scale"])
    return (s["out"], *_values(s))


def _plain_attend(s):
    q, tables, lengths, n, new = s["q"], s["tables"].long(), s["lengths"].long(), s["n"].long(), s["new"]
    B, (T, hq, D), hkv = tables.shape[0], q.shape, s["cache_k"].shape[2]
    k, v = (c[tables].float().reshape(B, -1, hkv, D).transpose(1, 2) for c in (s["cache_k"], s["cache_v"]))
    L, group = k.shape[2], hq // hkv
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][:, None, None], v * s["v_scale"][:, None, None]
    step = torch.arange(new, device=DEV)
    row = torch.where(step < n[:, None], s["first"].long()[:, None] + step, T)                 # [B, new], T: no such row
    rows = torch.cat([q, q.new_zeros((1, hq, D))]).float()[row]                               # [B, new, hq, D]
    rows = rows.reshape(B, new, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(B * hkv, group * new, D)
    score = torch.bmm(rows, k.reshape(B * hkv, L, D).transpose(1, 2).contiguous()) * D ** -0.5
    here, key = lengths[:, None] - n[:, None] + step, torch.arange(L, device=DEV)
    seen = key <= here[..., None]
    if s["window"]:
        seen = seen & (key > here[..., None] - s["window"])
    score = torch.where(seen[:, None, None], score.view(B, hkv, group, new, L), -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    weight = weight / weight.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.bmm(weight.view(B * hkv, group * new, L), v.reshape(B * hkv, L, D).contiguous())
    out = out.view(B, hkv, group, new, D).permute(0, 3, 1, 2, 4).reshape(B * new, hq, D).to(q.dtype)
    whole = torch.cat([s["out"], q.new_zeros((1, hq, D))])
    whole[row.reshape(-1)] = out
    return whole[:T]


def _plain_logprobs(s):
    logits, tokens, top, V = s["logits"].float(), s["tokens"].long(), s["top"], s["logits"].shape[1]
    place = torch.arange(V, device=DEV)
    scaled = logits if s["temperature"] is None else logits / s["temperature"][:, None]
    scaled = scaled - scaled.amax(-1, keepdim=True)
    weight = torch.exp(scaled)
    z = weight.sum(-1, keepdim=True)
    log_p = scaled - torch.log(z)
    entropy = -(weight / z * log_p.clamp(min=-1e30)).sum(-1)
    mine = logits.gather(-1, tokens[:, None])
    rank = 1 + ((logits > mine) | ((logits == mine) & (place < tokens[:, None]))).sum(-1)
    # the order of (logit, lowest place first) as one whole number
    bits = logits.contiguous().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 18) + (V - 1 - place)
    ids = torch.topk(order, top, dim=-1).indices if top else place[:0].expand(logits.shape[0], 0)
    return (log_p.gather(-1, tokens[:, None])[:, 0], rank.to(torch.int32), entropy, ids.to(torch.int32),
            log_p.gather(-1, ids))


PLAIN = {"append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "logprobs":
        R, V = c["rows"], c["vocab"]
        return {"bytes": R * (V * (4 if c["dtype"] == "fp32" else 2) + 16 + 8 * c["top"]), "flops": 6 * R * V}
    hq, hkv = _sizes(c["heads"])
    D, wide = c["dim"], 1 if c["cache"] == "e4m3" else 2
    if c["kind"] == "append":
        T, kept = c["tokens"], c["tokens"] - c["padding"]
        return {"bytes": T * (4 * hq * D + 8 * c["axes"] + 8) + kept * 2 * hkv * D * (2 + wide), "flops": T * (hq + hkv) * D * 7}
    n, lengths = _counts(c)
    pairs = keys = 0
    for i, length in zip(n, lengths):
        seen = [min(p + 1, c["window"] or p + 1) for p in range(length - i, length)]
        pairs += sum(seen)
        keys += min(length, i - 1 + c["window"]) if c["window"] else length
    return {"bytes": 4 * sum(n) * hq * D + 2 * keys * hkv * D * wide, "flops": 4 * D * hq * pairs}


# ---- the operators' definitions in 64 bits

def _exact_append(c, seed):
    s = _append_inputs(c, seed)
    T, half = c["tokens"], c["rotary"] // 2
    turn = torch.stack([s["positions"][int(a)].double() * f for a, f in zip(s["axes"].tolist(), s["inv_freq"])], dim=1)
    unit = torch.polar(torch.ones_like(turn), turn)[:, None]                # e^{i t}

    def rows(x, weight):
        x = x.double()
        if weight is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        x = x.clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["adjacent"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., first], x[..., second]) * unit
        x[..., first], x[..., second] = z.real, z.imag
        return x

    caches = []
    for name, new in (("k", rows(s["k"], s["k_norm"])), ("v", s["v"].double())):
        scale, cache = s[name + "_scale"], s["cache_" + name]
        scale = torch.ones((new.shape[1],), device=DEV) if scale is None else scale
        held = cache.double() * scale.double()[:, None]
        if cache.dtype == DTYPES["e4m3"]:                                   # what eight bits stand for
            new = (new / scale.double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype).double() * scale.double()[:, None]
        ok = s["slots"] >= 0
        held.view(-1, *held.shape[2:])[s["slots"][ok]] = new[ok]
        caches.append(held)
    return (rows(s["q"], s["q_norm"]), *caches)


def _exact_attend(c, seed):
    s = _attend_inputs(c, seed)
    hq, hkv = _sizes(c["heads"])
    group, page = hq // hkv, c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, length) in enumerate(zip(*_counts(c))):
        place = torch.arange(length, device=DEV)
        where = (s["tables"][b].long()[place // page], place % page)
        own_place = torch.arange(length - n, length, device=DEV)[:, None]
        hidden = place[None, :] > own_place
        if c["window"]:
            hidden = hidden | (place[None, :] <= own_place - c["window"])
        for h in range(hq):
            g = h // group
            k, v = s["cache_k"][where][:, g].double(), s["cache_v"][where][:, g].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
            logits = s["q"][at:at + n, h].double() @ k.t().contiguous() / math.sqrt(c["dim"])
            out[at:at + n, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), dim=-1) @ v
        at += n
    return out


def _exact_logprobs(c, seed):
    s = _logprobs_inputs(c, seed)
    rows, top = [], c["top"]
    for r in range(c["rows"]):
        logits, token = s["logits"][r].double(), s["tokens"][r].long()
        log_p = torch.log_softmax(logits if s["temperature"] is None else logits / s["temperature"][r].double(), dim=0)
        p = log_p.exp()
        entropy = -torch.where(p > 0, p * log_p, 0.0).sum()
        above = (logits > logits[token]).sum() + (logits[:token] == logits[token]).sum()
        ids = torch.sort(logits, descending=True, stable=True).indices[:top]
        rows.append((log_p[token], (above + 1).to(torch.int32), entropy, ids.to(torch.int32), log_p[ids]))
    return tuple(torch.stack(v) for v in zip(*rows))


def exact(case, seed):
    return {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["kind"]](case, seed)
