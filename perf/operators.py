"""Operators of a served model beside its trellis-coded layers, as cases that can be timed and checked: the low-rank adapters
of many requests on a shared projection, the verification of drafted tokens against the target's logits, and the norms after
and before a block with its gate and residual scale.

Sizes are those of the package's own benchmark (hidden 2048; q/k/v 4096 + 512 + 512 from it, o 4096 -> 2048; a vocabulary of
151936; decode batches up to 32, prompts in the hundreds and thousands), and spread around them by draw().

Where `own` is false, run() computes the operators in elementary torch operations; where it is true, it calls the package.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
GREEDY_BELOW = 1e-5           # temperatures below this one mean greedy decoding
CHUNK_WEIGHTS = 1 << 25       # elements of the products that the plain adapters make at once


def listed():
    return [
        # one token of one request through q/k/v with its adapter: the smallest call, bound by latency
        {"name": "lora_decode_1", "kind": "lora", "rows": 1, "in": 2048, "out": "4096+512+512", "adapters": 1, "ranks": "16",
         "without": 0, "prompt": False, "dtype": "bf16"},
        # a decode batch through o in which nearly every request has another adapter, of mixed and odd ranks, a few have none
        {"name": "lora_decode_32", "kind": "lora", "rows": 32, "in": 4096, "out": "2048", "adapters": 24, "ranks": "8+16+64+13",
         "without": 3, "prompt": False, "dtype": "bf16"},
        # a ragged batch of three short prompts through the gate/up projections
        {"name": "lora_prompt_509", "kind": "lora", "rows": 509, "in": 2048, "out": "512+512", "adapters": 3, "ranks": "32",
         "without": 0, "prompt": True, "dtype": "fp16"},
        # a full prefill batch of many requests through q/k/v, one of them without an adapter
        {"name": "lora_prompt_4096", "kind": "lora", "rows": 4096, "in": 2048, "out": "4096+512+512", "adapters": 6,
         "ranks": "16+64", "without": 500, "prompt": True, "dtype": "bf16"},
        # one request that drafts three tokens greedily (a drafter without probabilities): the smallest verification
        {"name": "verify_1", "kind": "verify", "requests": 1, "drafts": 3, "ragged": False, "vocab": 151936, "probs": False,
         "greedy_every": 0, "dtype": "bf16"},
        # a decode batch with draft probabilities, ragged numbers of drafts and every fourth request greedy
        {"name": "verify_29", "kind": "verify", "requests": 29, "drafts": 4, "ragged": True, "vocab": 151936, "probs": True,
         "greedy_every": 4, "dtype": "bf16"},
        # a smaller, odd vocabulary, whose rows start at any element, with half-precision logits
        {"name": "verify_odd", "kind": "verify", "requests": 64, "drafts": 2, "ragged": True, "vocab": 32003, "probs": True,
         "greedy_every": 0, "dtype": "fp16"},
        # a large batch with the 32-bit logits that a logits processor leaves
        {"name": "verify_128", "kind": "verify", "requests": 128, "drafts": 5, "ragged": False, "vocab": 151936, "probs": True,
         "greedy_every": 0, "dtype": "fp32"},
        # the norms around a block for one token: the smallest call
        {"name": "norm_1", "kind": "norm", "rows": 1, "dim": 2048, "deltas": 1, "post": True, "gate": "channel",
         "sigmoid": False, "scale": 1.0, "dtype": "bf16"},
        # an odd decode batch behind an MoE block (routed and shared outputs) with a token's gate
        {"name": "norm_31", "kind": "norm", "rows": 31, "dim": 2048, "deltas": 2, "post": True, "gate": "token",
         "sigmoid": True, "scale": 0.5, "dtype": "bf16"},
        # a ragged prompt with a scaled residual and no norm behind the block
        {"name": "norm_prompt_1531", "kind": "norm", "rows": 1531, "dim": 4096, "deltas": 1, "post": False, "gate": "none",
         "sigmoid": False, "scale": 0.22, "dtype": "fp16"},
        # a full prefill batch with a gate for every element
        {"name": "norm_prompt_8192", "kind": "norm", "rows": 8192, "dim": 4096, "deltas": 1, "post": True, "gate": "element",
         "sigmoid": True, "scale": 1.0, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lora", "verify", "norm"])
    if kind == "lora":
        prompt = rng.random() < 0.5
        rows = _log(rng, 33, 3500) if prompt else _log(rng, 1, 64)
        out = "+".join(str(16 * _log(rng, 2, 160)) for _ in range(rng.randint(1, 4)))
        adapters = rng.randint(1, min(8 if prompt else 32, rows))
        ranks = "+".join(str(_log(rng, 1, 64)) for _ in range(rng.randint(1, 4)))
        return {"kind": kind, "rows": rows, "in": 16 * _log(rng, 4, 128), "out": out, "adapters": adapters, "ranks": ranks,
                "without": rng.choice([0, 0, min(rows - adapters, rng.randint(0, 9))]), "prompt": prompt,
                "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if kind == "verify":
        drafts, vocab = rng.randint(0, 7), _log(rng, 1000, 151936)
        most = min(128, 100_000_000 // ((drafts + 1) * vocab))
        return {"kind": kind, "requests": _log(rng, 1, max(1, most)), "drafts": drafts, "ragged": rng.random() < 0.5,
                "vocab": vocab, "probs": rng.random() < 0.6, "greedy_every": rng.choice([0, 0, 2, 5]),
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    dim = 8 * _log(rng, 16, 1024)
    return {"kind": kind, "rows": _log(rng, 1, max(1, min(8192, 30_000_000 // dim))), "dim": dim, "deltas": rng.randint(1, 2),
            "post": rng.random() < 0.7, "gate": rng.choice(["none", "channel", "token", "element"]),
            "sigmoid": rng.random() < 0.5, "scale": rng.choice([1.0, 0.5, 0.22]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}


# ---- what a program has in hand

def _sizes(text):
    return [int(v) for v in text.split("+")]


def _ranks(c):
    """The rank of every adapter: the case's ranks in turn."""
    ranks = _sizes(c["ranks"])
    return [ranks[i % len(ranks)] for i in range(c["adapters"])]


def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device=DEV) * scale


def _adapter_rows(c, gen):
    """The adapter of every row, -1 for none. A decode batch: one token a request, every adapter in use, in any order. A
    prompt batch: the tokens of a request stand together, in pieces of any length."""
    T, L, bare = c["rows"], c["adapters"], c["without"]
    if not c["prompt"]:
        more = torch.randint(0, L, (T - L - bare,), generator=gen, device=DEV)
        ids = torch.cat([torch.arange(L, device=DEV), more, torch.full((bare,), -1, device=DEV)])
        return ids[torch.randperm(T, generator=gen, device=DEV)].to(torch.int32)
    cuts = 1 + torch.randperm(T - bare - 1, generator=gen, device=DEV)[:L - 1].sort().values
    piece = (torch.arange(T - bare, device=DEV)[:, None] >= cuts[None, :]).sum(1)
    return torch.cat([piece, torch.full((bare,), -1, device=DEV)]).to(torch.int32)


def _lora_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, K, outs = DTYPES[c["dtype"]], c["in"], _sizes(c["out"])
    a = [[_normal((r, K), gen, K ** -0.5).to(dtype) for _ in outs] for r in _ranks(c)]
    b = [[_normal((n, r), gen, r ** -0.5).to(dtype) for n in outs] for r in _ranks(c)]
    scales = [2.0 if i % 2 else 0.5 for i in range(c["adapters"])]
    return {"x": _normal((c["rows"], K), gen).to(dtype), "y": _normal((c["rows"], sum(outs)), gen, 2.0).to(dtype),
            "ids": _adapter_rows(c, gen), "a": a, "b": b, "scales": scales}


def _draft_counts(c):
    """The drafts of every request: all of them, or, ragged, any number from none on."""
    return [i * 7919 % (c["drafts"] + 1) if c["ragged"] else c["drafts"] for i in range(c["requests"])]


def _verify_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B, G, V = c["requests"], c["drafts"], c["vocab"]
    counts = _draft_counts(c)
    first = [sum(counts[:i]) + i for i in range(B)]
    logits = _normal((sum(counts) + B, V), gen, 4.0).to(DTYPES[c["dtype"]])
    temperature = [0.0 if c["greedy_every"] and i % c["greedy_every"] == 0 else 0.6 + 0.1 * (i % 7) for i in range(B)]
    probs = torch.zeros((B, G, V), device=DEV)
    drafts = torch.full((B, G), -1, device=DEV, dtype=torch.int32)
    for i, n in enumerate(counts):
        if n == 0:
            continue
        # the drafter knows the target's distribution roughly
        near = logits[first[i]:first[i] + n].float() + _normal((n, V), gen, 0.7)
        probs[i, :n] = torch.softmax(near / max(temperature[i], 0.3), dim=-1)
        if c["probs"]:
            race = torch.empty((n, V), device=DEV).exponential_(generator=gen)
            drafts[i, :n] = (probs[i, :n] / race).argmax(-1)
        else:
            drafts[i, :n] = probs[i, :n].argmax(-1)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"logits": logits, "first": i32(first), "counts": i32(counts), "drafts": drafts,
            "uniform": torch.rand((B, G), generator=gen, device=DEV),
            "race": torch.empty((B, V), device=DEV).exponential_(generator=gen),
            "temperature": torch.tensor(temperature, device=DEV), "probs": probs if c["probs"] else None}


def _norm_inputs(c, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, T, D = DTYPES[c["dtype"]], c["rows"], c["dim"]
    weight = lambda: (1 + _normal((D,), gen, 0.1)).to(dtype)  # noqa: E731
    gate = {"none": None, "channel": (D,), "token": (T, 1), "element": (T, D)}[c["gate"]]
    return {"h": _normal((T, D), gen, 3.0).to(dtype), "d": [_normal((T, D), gen).to(dtype) for _ in range(c["deltas"])],
            "post": weight() if c["post"] else None, "pre": weight(), "gate": gate and _normal(gate, gen).to(dtype),
            "sigmoid": c["sigmoid"], "scale": c["scale"]}


INPUTS = {"lora": _lora_inputs, "verify": _verify_inputs, "norm": _norm_inputs}


def prepare(case, seed):
    s = INPUTS[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    if own:
        sys.path.insert(0, os.path.join(os.getcwd(), "vllm-espalier_amd"))
    if case["kind"] == "lora":
        a, b, scales = s.pop("a"), s.pop("b"), s.pop("scales")
        outs, top, dtype = _sizes(case["out"]), max(_ranks(case)), DTYPES[case["dtype"]]
        if own:
            from vllm_espalier.adapters import Adapters
            s["store"] = Adapters(case["in"], outs, slots=case["adapters"], max_rank=top, dtype=dtype, device=DEV)
            for i in range(case["adapters"]):
                s["store"].load(i, a[i], b[i], scale=scales[i])
        else:
            # the stacked adapters: A [L, S, rank, K], B [L, N, rank], zero past an adapter's rank
            s["outs"], s["scale"] = outs, torch.tensor(scales, device=DEV)
            s["A"] = torch.zeros((len(a), len(outs), top, case["in"]), dtype=dtype, device=DEV)
            s["B"] = torch.zeros((len(a), sum(outs), top), dtype=dtype, device=DEV)
            for i, r in enumerate(_ranks(case)):
                s["A"][i, :, :r] = torch.stack(a[i])
                s["B"][i, :, :r] = torch.cat(b[i])
        s["out"] = torch.empty_like(s["y"])
    elif case["kind"] == "norm":
        s["h_out"], s["out"] = torch.empty_like(s["h"]), torch.empty_like(s["h"])
        if own:
            from vllm_espalier.experts import ext
            s["ext"] = ext()
    elif own:
        from vllm_espalier import speculative
        s["verify"] = speculative.verify
    return s


# ---- the operators

def _own(s):
    if s["kind"] == "lora":
        return s["store"].apply(s["x"], s["y"], s["ids"], out=s["out"])
    if s["kind"] == "verify":
        return s["verify"](s["logits"], s["first"], s["counts"], s["drafts"], s["uniform"], s["race"], s["temperature"],
                           draft_probs=s["probs"])
    d2 = s["d"][1] if len(s["d"]) > 1 else None
    s["ext"].sandwich_rmsnorm(s["h"], s["d"][0], d2, s["post"], s["gate"], s["sigmoid"], s["scale"], s["pre"], EPS, s["h_out"],
                              s["out"])
    return s["h_out"], s["out"]


def _plain_lora(s):
    x, A, B, ids, outs = s["x"].float(), s["A"].float(), s["B"].float(), s["ids"].long(), s["outs"]
    T, S, rank = x.shape[0], A.shape[1], A.shape[2]
    shard = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(outs, device=DEV), output_size=sum(outs))
    delta = torch.zeros((T, sum(outs)), device=DEV)
    if T * max(S * rank * x.shape[1], sum(outs) * rank) <= CHUNK_WEIGHTS:      # a few rows: every row with its own adapter
        mine = ids.clamp(min=0)
        t = (x[:, None, None, :] * A[mine]).sum(-1) * s["scale"][mine][:, None, None]          # [T, S, rank]
        delta = torch.where((ids >= 0)[:, None], (t[:, shard] * B[mine]).sum(-1), delta)
    else:                                                                     # many rows: an adapter after the other
        for i in range(A.shape[0]):
            t = (x @ A[i].reshape(S * rank, -1).t()).reshape(T, S, rank) * s["scale"][i]
            parts = [t[:, k] @ B[i][sum(outs[:k]):sum(outs[:k + 1])].t() for k in range(S)]
            delta = torch.where((ids == i)[:, None], torch.cat(parts, dim=1), delta)
    return (s["y"].float() + delta).to(s["y"].dtype)


def _plain_verify(s):
    """In 64 bits: whether a draft is accepted and which token wins the race are decided at borders."""
    n, drafts, V = s["counts"], s["drafts"], s["logits"].shape[1]
    B, G = drafts.shape
    steps = torch.arange(G + 1, device=DEV)
    at = (s["first"][:, None] + torch.minimum(steps[None, :], n[:, None])).long()
    rows = s["logits"][at].double()                                            # [B, G + 1, V]
    best = rows.argmax(-1)
    greedy = s["temperature"] < GREEDY_BELOW
    scaled = rows / torch.where(greedy, 1.0, s["temperature"].double())[:, None, None]
    weight = torch.exp(scaled - scaled.amax(-1, keepdim=True))
    p = weight / weight.sum(-1, keepdim=True)
    token = drafts.long().clamp(min=0)[..., None]
    p_draft = p[:, :G].gather(-1, token)[..., 0]
    q_draft = 1.0 if s["probs"] is None else s["probs"].double().gather(-1, token)[..., 0]
    sure = s["uniform"].double() * q_draft < p_draft
    ok = torch.where(greedy[:, None], drafts == best[:, :G], sure) & (steps[None, :G] < n[:, None])
    taken = ok.long().cumprod(-1).sum(-1)
    here = torch.arange(B, device=DEV)
    last = p[here, taken]
    rejected = (taken < n)[:, None]
    if G == 0:
        q = torch.zeros_like(last)
    elif s["probs"] is None:
        q = (torch.arange(V, device=DEV)[None, :] == drafts[here, taken.clamp(max=G - 1)][:, None]).double()
    else:
        q = s["probs"][here, taken.clamp(max=G - 1)].double()
    if s["probs"] is None:
        left = torch.where(q > 0, 0.0, last)
    else:
        left = (last - q).clamp(min=0)
    left = torch.where(rejected, left, last)
    left = torch.where((left > 0).any(-1, keepdim=True), left, last)
    drawn = torch.where(greedy, best[here, taken], (left / s["race"].double()).argmax(-1))
    padded = torch.cat([drafts, drafts.new_zeros((B, 1))], dim=1)
    tokens = torch.where(steps < taken[:, None], padded, -1)
    tokens = torch.where(steps == taken[:, None], drawn[:, None], tokens)
    # p of the greedy rows is that of temperature 1
    p_token = p.gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    logprobs = torch.where(tokens >= 0, torch.log(p_token), 0.0)
    return tokens.to(torch.int32), (taken + 1).to(torch.int32), logprobs.float()


def _plain_norm(s):
    dtype = s["h"].dtype
    u = s["d"][0].float()
    for d in s["d"][1:]:
        u = u + d.float()
    if s["post"] is not None:
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        g = s["gate"].float()
        u = u * (1 / (1 + torch.exp(-g)) if s["sigmoid"] else g)
    h = (s["h"].float() + s["scale"] * u).to(dtype)
    z = h.float()
    return h, (z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * s["pre"].float()).to(dtype)


PLAIN = {"lora": _plain_lora, "verify": _plain_verify, "norm": _plain_norm}


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# ---- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "lora":
        T, K, outs = c["rows"], c["in"], _sizes(c["out"])
        N, S, ranks = sum(outs), len(outs), _ranks(c)
        rows = T - c["without"]
        return {"bytes": 2 * (T * K + 2 * T * N + sum(r * (S * K + N) for r in ranks)) + 4 * T,
                "flops": 2 * rows * sum(ranks) / len(ranks) * (S * K + N)}
    if c["kind"] == "verify":
        counts, V = _draft_counts(c), c["vocab"]
        rows = sum(counts) + len(counts)
        sampled = sum(1 for i in range(len(counts)) if not (c["greedy_every"] and i % c["greedy_every"] == 0))
        return {"bytes": V * (rows * (4 if c["dtype"] == "fp32" else 2) + 4 * sampled * (2 if c["probs"] else 1)),
                "flops": 4 * rows * V}
    T, D = c["rows"], c["dim"]
    gate = {"none": 0, "channel": D, "token": T, "element": T * D}[c["gate"]]
    return {"bytes": 2 * (T * D * (3 + c["deltas"]) + gate + D * (2 if c["post"] else 1)), "flops": 12 * T * D}


# ---- the operators' definitions in 64 bits

def _exact_lora(c, seed):
    s = _lora_inputs(c, seed)
    out = s["y"].double()
    for i in range(c["adapters"]):
        hit = (s["ids"] == i).nonzero()[:, 0]
        x, col = s["x"].double()[hit], 0
        for a, b in zip(s["a"][i], s["b"][i]):
            low = x @ a.double().t().contiguous()
            out[hit, col:col + b.shape[0]] += s["scales"][i] * (low @ b.double().t().contiguous())
            col += b.shape[0]
    return out


def _exact_verify(c, seed):
    s = _verify_inputs(c, seed)
    B, G = s["drafts"].shape
    tokens = torch.full((B, G + 1), -1, dtype=torch.int32)
    counts = torch.zeros((B,), dtype=torch.int32)
    logprobs = torch.zeros((B, G + 1), dtype=torch.float64)
    drafts, uniform, temperature = s["drafts"].tolist(), s["uniform"].double().tolist(), s["temperature"].tolist()
    first, n = s["first"].tolist(), s["counts"].tolist()
    for i in range(B):
        j = 0
        while True:
            logits = s["logits"][first[i] + j].double()
            x = drafts[i][j] if j < n[i] else None
            if temperature[i] < GREEDY_BELOW:
                p = torch.softmax(logits, dim=0)
                drawn = int(logits.argmax())
                ok = x == drawn
            else:
                p = torch.softmax(logits / temperature[i], dim=0)
                q = None
                if x is not None:
                    q = s["probs"][i, j].double() if c["probs"] else None
                    ok = uniform[i][j] * (1.0 if q is None else float(q[x])) < float(p[x])
                else:
                    ok = False
                if not ok:
                    left = p.clone()
                    if q is not None:
                        left = torch.relu(p - q)
                    elif x is not None:
                        left[x] = 0
                    if float(left.max()) == 0:
                        left = p
                    drawn = int((left / s["race"][i].double()).argmax())
            tokens[i, j] = x if ok else drawn
            logprobs[i, j] = float(p[tokens[i, j]].log())
            if not ok:
                break
            j += 1
        counts[i] = j + 1
    return tokens.to(DEV), counts.to(DEV), logprobs.to(DEV)


def _exact_norm(c, seed):
    s = _norm_inputs(c, seed)
    rms = lambda v, w: v / (v.square().mean(dim=1, keepdim=True) + EPS).sqrt() * w.double()  # noqa: E731
    block = sum(d.double() for d in s["d"])
    if s["post"] is not None:
        block = rms(block, s["post"])
    if s["gate"] is not None:
        gate = s["gate"].double()
        block = block * (gate.sigmoid() if s["sigmoid"] else gate)
    h = s["h"].double() + s["scale"] * block
    # the second norm is that of the residual as it is stored
    return h, rms(h.to(s["h"].dtype).double(), s["pre"])


def exact(case, seed):
    return {"lora": _exact_lora, "verify": _exact_verify, "norm": _exact_norm}[case["kind"]](case, seed)
