"""GPU checks of the verification of drafted tokens (csrc/verify.hip, vllm_espalier/speculative.py) against the rule in 64 bits.

Tokens and counts are whole numbers and have to be equal wherever the rule decides by more than 1e-5 (a request whose draft or
race is closer than that to its border may fall on either side in 32 bits, whose exponentials are off by 2^-19 at most; such
requests are left out, and must be few). Log-probabilities: half a step of fp32 and 2^-18 (44 roundings of 2^-24 in the sum).
"""
import math

import pytest
import torch

from vllm_espalier import speculative

pytestmark = pytest.mark.gpu
MARGIN = 1e-5


def _inputs(B, G, V, dtype, probs, gen, temperature=0.8, greedy_every=0, ragged=True, sharp=4.0):
    n = [(i * 5) % (G + 1) if ragged else G for i in range(B)]
    first = [sum(n[:i]) + i for i in range(B)]
    logits = (torch.randn((sum(n) + B, V), generator=gen) * sharp).to(dtype)
    temp = torch.tensor([0.0 if greedy_every and i % greedy_every == 0 else temperature for i in range(B)])
    q = torch.zeros((B, G, V))
    drafts = torch.full((B, G), -1, dtype=torch.int32)
    for i in range(B):
        for j in range(n[i]):
            near = logits[first[i] + j].float() + torch.randn((V,), generator=gen) * 0.7
            q[i, j] = torch.softmax(near / max(float(temp[i]), 0.3), 0)
            race = torch.empty((V,)).exponential_(generator=gen)
            drafts[i, j] = int((q[i, j] / race).argmax()) if probs else int(near.argmax())
    return {"logits": logits, "first": torch.tensor(first, dtype=torch.int32), "n": torch.tensor(n, dtype=torch.int32),
            "drafts": drafts, "uniform": torch.rand((B, G), generator=gen),
            "race": torch.empty((B, V)).exponential_(generator=gen), "temp": temp, "probs": q if probs else None}


def _call(i, dev, **kw):
    d = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in i.items()}
    out = speculative.verify(d["logits"], d["first"], d["n"], d["drafts"], d["uniform"], d["race"], d["temp"],
                             draft_probs=d["probs"], **kw)
    return [t.cpu() for t in out]


def _argmax(row):
    nan = torch.isnan(row).nonzero()
    return int(nan[0]) if len(nan) else int((row == row.max()).nonzero()[0])


def _want(i, b):
    """(tokens, logprobs, certain) of request b."""
    G, V = i["drafts"].shape[1], i["logits"].shape[1]
    n, f, t = int(i["n"][b]), int(i["first"][b]), float(i["temp"][b])
    if not (0 <= n <= G and f >= 0 and f + n < i["logits"].shape[0]):
        return [], [], True
    tokens, logprobs, certain = [], [], True
    for j in range(n + 1):
        row = i["logits"][f + j].double()
        x = int(i["drafts"][b, j]) if j < n else None
        greedy = not t >= 1e-5
        scaled = row if greedy else row / t
        if not greedy and t == math.inf:
            scaled = torch.where(row == -math.inf, row, 0.0)
        some = bool(torch.isfinite(row.max())) and not bool(torch.isnan(row).any())
        logp = torch.log_softmax(scaled, 0) if some else None
        if greedy:
            drawn = _argmax(row)
            tokens.append(drawn)
            logprobs.append(float(logp[drawn]) if some else 0.0)
            if x == drawn:
                continue
            break
        if not some:
            break
        p = logp.exp()
        q = None
        if x is not None:
            q = torch.zeros_like(p)
            if i["probs"] is not None:
                q = i["probs"][b, j].double()
            elif 0 <= x < V:
                q[x] = 1.0
            if 0 <= x < V:
                qx = float(q[x]) if i["probs"] is not None else 1.0
                uq = float(i["uniform"][b, j]) * qx
                px = float(p[x])
                certain &= abs(uq - px) > MARGIN * max(uq, px) or uq == px == 0
                if uq < px:
                    tokens.append(x)
                    logprobs.append(float(logp[x]))
                    continue
        w = p
        if q is not None:
            w = torch.where(q > 0, 0.0, p) if i["probs"] is None else (p - q).clamp(min=0)
            if float(w.max()) <= 0:
                w = p
        key = torch.where(w > 0, w / i["race"][b].double(), -1.0)
        top = key.topk(min(2, V)).values
        if V > 1 and float(top[0]) < math.inf and float(top[1]) > 0:
            certain &= float(top[0] - top[1]) > MARGIN * float(top[0]) or float(top[0]) == float(top[1])
        # what a difference of near-equal probabilities weighs is known to their rounding only
        drawn = int((key == key.max()).nonzero()[0])
        certain &= q is None or float(w[drawn]) > MARGIN * float(p[drawn]) * 100
        tokens.append(drawn)
        logprobs.append(float(logp[drawn]))
        break
    return tokens, logprobs, certain


def _check(i, got, few=0.1):
    tokens, counts, logprobs = got
    B, G = i["drafts"].shape
    assert tokens.shape == (B, G + 1) and counts.shape == (B,) and logprobs.shape == (B, G + 1)
    skipped = 0
    for b in range(B):
        want, lp, certain = _want(i, b)
        if not certain:
            skipped += 1
            continue
        assert tokens[b].tolist() == want + [-1] * (G + 1 - len(want)), b
        assert int(counts[b]) == len(want), b
        for j, v in enumerate(lp):
            assert abs(float(logprobs[b, j]) - v) <= 2.0 ** -24 * abs(v) + 2.0 ** -18, (b, j)
        assert not logprobs[b, len(lp):].any(), b
    assert skipped <= few * B, skipped


@pytest.mark.parametrize("V", [1, 2, 7, 8, 64, 1000, 1023, 1025, 4099, 33001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_verify_vocabularies(dev, V, dtype):
    print(f"verify V={V} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(V)
    for probs in (False, True):
        i = _inputs(6, 3, V, dtype, probs, gen)
        _check(i, _call(i, dev), few=0.2)


@pytest.mark.parametrize("B,G", [(1, 0), (5, 0), (1, 1), (33, 2), (9, 7), (2, 40)])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_batches(dev, B, G, probs):
    gen = torch.Generator().manual_seed(B * 100 + G)
    i = _inputs(B, G, 2053, torch.bfloat16, probs, gen, greedy_every=3)
    _check(i, _call(i, dev))
    i["uniform"].zero_()                                     # every draft that the target can make is accepted
    got = _call(i, dev)
    _check(i, got)
    i["uniform"].fill_(1.0 - 2.0 ** -24)
    _check(i, _call(i, dev), few=0.2)


def test_verify_many_requests(dev):
    """More chunks of entries than workgroups race: a workgroup several of them."""
    gen = torch.Generator().manual_seed(2)
    i = _inputs(700, 1, 9001, torch.bfloat16, True, gen, greedy_every=5)
    _check(i, _call(i, dev), few=0.02)


def test_verify_large_vocabulary(dev):
    gen = torch.Generator().manual_seed(1)
    i = _inputs(3, 3, 151936, torch.bfloat16, True, gen, ragged=False)
    _check(i, _call(i, dev), few=0.34)


@pytest.mark.parametrize("temperature", [1e-3, 0.3, 1.0, 20.0, math.inf, 1e-6, float("nan"), -1.0])
def test_verify_temperatures(dev, temperature):
    """Far temperatures; one below 1e-5, negative or NaN is greedy."""
    gen = torch.Generator().manual_seed(6)
    i = _inputs(6, 2, 515, torch.float32, True, gen, temperature=temperature if temperature > 0.1 else 0.5)
    i["logits"][:, 100:130] = -math.inf
    i["temp"].fill_(temperature)
    _check(i, _call(i, dev), few=0.2)


@pytest.mark.parametrize("greedy", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify_odd_rows(dev, greedy, dtype):
    """Masked tokens, rows whose mask leaves one token or none, NaN and infinities, drafts outside the vocabulary, drafts that
    the target excludes, masks of the type's lowest value, and a draft distribution that covers all of the target's."""
    gen = torch.Generator().manual_seed(17)
    V = 1037
    i = _inputs(16, 2, V, dtype, True, gen, ragged=False, temperature=0.0 if greedy else 0.9)
    lo = i["logits"]
    row = lambda b, j: int(i["first"][b]) + j  # noqa: E731
    lo[row(0, 0)] = -math.inf                                # nothing left
    lo[row(1, 0)] = -math.inf
    lo[row(1, 0), 700] = 3.0                                 # one token left
    lo[row(2, 1), 5] = float("nan")
    lo[row(3, 0), 1036] = math.inf
    lo[row(4, 0), :600] = -math.inf
    lo[row(4, 0), 601:] = torch.finfo(dtype).min
    i["drafts"][5, 0] = V
    i["drafts"][6, 0] = -7
    i["drafts"][7, 0] = 2 ** 31 - 1
    lo[row(8, 0), int(i["drafts"][8, 0])] = -math.inf         # the target excludes the draft
    i["probs"][9] = 1.0                                       # q covers p: the target's own distribution is drawn from
    i["uniform"][9] = 0.999
    lo[row(10, 2)] = -math.inf                               # the row behind the last draft, all drafts accepted
    i["uniform"][10] = 0.0
    lo[row(11, 0), :] = 1.0                                  # all equal
    lo[row(12, 1)] = torch.finfo(dtype).min                  # a mask of the lowest value everywhere
    i["probs"][13] = 0.0                                      # drafts of no probability
    lo[row(14, 0), 3] = lo[row(14, 0), 900] = 60.0           # a tie
    lo[row(15, 0)] = 0.0
    lo[row(15, 0), :9] = -0.0                                # zeros of both signs are equal
    _check(i, _call(i, dev), few=0.2)
    i["probs"] = None
    _check(i, _call(i, dev), few=0.2)


def test_verify_padded_batch(dev):
    """Requests that are not there, have more drafts than the arrays hold or rows outside the logits have no tokens."""
    gen = torch.Generator().manual_seed(23)
    i = _inputs(8, 2, 300, torch.bfloat16, False, gen, ragged=False)
    i["n"][1], i["n"][3], i["n"][5] = -1, 3, -2 ** 31
    i["first"][6], i["first"][7] = -1, i["logits"].shape[0] - 2
    i["n"][0], i["first"][0] = 2, i["logits"].shape[0] - 3     # the last rows
    got = _call(i, dev)
    _check(i, got, few=0.2)
    assert got[1].tolist()[1] == 0 and got[1].tolist()[3] == 0 and got[1].tolist()[5:] == [0, 0, 0]
    i["first"][4] = i["first"][2]                            # two requests over the same rows
    _check(i, _call(i, dev), few=0.2)


def test_verify_race_values(dev):
    """Random numbers of zero win where there is any probability, those that are no numbers never do; equal keys: the lowest
    index."""
    gen = torch.Generator().manual_seed(29)
    V = 260
    i = _inputs(4, 0, V, torch.float32, False, gen)
    i["logits"].zero_()
    i["race"].fill_(1.0)
    i["race"][0, 77] = 0.0
    i["logits"][0, 76] = -math.inf
    i["race"][0, 76] = 0.0
    i["race"][1, :40] = float("nan")
    i["race"][3].fill_(float("nan"))
    tokens, counts, _ = _call(i, dev)
    assert tokens[:, 0].tolist() == [77, 40, 0, -1] and counts.tolist() == [1, 1, 1, 0]


def test_verify_strides(dev):
    """Views: logits and random numbers of wider buffers, draft probabilities in another order."""
    gen = torch.Generator().manual_seed(31)
    i = _inputs(5, 3, 777, torch.bfloat16, True, gen)
    want = _call(i, dev)
    wide = torch.full((i["logits"].shape[0], 801), 50.0).to(torch.bfloat16)
    wide[:, 13:790] = i["logits"]
    race = torch.zeros((5, 900))
    race[:, 1:778] = i["race"]
    d = {k: v.to(dev) if torch.is_tensor(v) else v for k, v in i.items()}
    q = torch.zeros((3, 5, 780), device=dev)
    q[:, :, 2:779] = d["probs"].transpose(0, 1)
    got = speculative.verify(wide.to(dev)[:, 13:790], d["first"], d["n"], d["drafts"], d["uniform"], race.to(dev)[:, 1:778],
                             d["temp"], draft_probs=q[:, :, 2:779].transpose(0, 1))
    assert all(torch.equal(w, g.cpu()) for w, g in zip(want, got))


def test_verify_graph_streams_and_batches(dev):
    """Captured once and replayed with new inputs: the eager results every time; two streams at once; a request's results do
    not depend on the others'."""
    gen = torch.Generator().manual_seed(37)
    i = _inputs(6, 3, 5003, torch.bfloat16, True, gen, greedy_every=4)
    d = {k: v.to(dev) for k, v in i.items()}
    call = lambda: speculative.verify(d["logits"], d["first"], d["n"], d["drafts"], d["uniform"], d["race"], d["temp"],  # noqa: E731
                                      draft_probs=d["probs"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for k in range(4):
        d["uniform"].copy_(torch.rand((6, 3), generator=gen))
        d["race"].copy_(torch.empty((6, 5003)).exponential_(generator=gen))
        g.replay()
        torch.cuda.synchronize()
        eager = call()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), k
    whole = [t.cpu() for t in call()]
    _check({k: v.cpu() for k, v in d.items()}, whole, few=0.2)
    for b in range(6):
        one = speculative.verify(d["logits"], d["first"][b:b + 1], d["n"][b:b + 1], d["drafts"][b:b + 1], d["uniform"][b:b + 1],
                                 d["race"][b:b + 1], d["temp"][b:b + 1], draft_probs=d["probs"][b:b + 1])
        assert all(torch.equal(w[b:b + 1], t.cpu()) for w, t in zip(whole, one)), b
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(w, t.cpu()) for r in got for w, t in zip(whole, r))


def test_verify_refusals(dev):
    gen = torch.Generator().manual_seed(41)
    i = {k: v.to(dev) for k, v in _inputs(4, 2, 64, torch.bfloat16, True, gen).items()}

    def call(**over):
        a = {**i, **over}
        return speculative.verify(a["logits"], a["first"], a["n"], a["drafts"], a["uniform"], a["race"], a["temp"],
                                  draft_probs=a["probs"], out=a.get("out"))

    tokens, counts, logprobs = call()
    for over in (dict(logits=i["logits"].double()), dict(logits=i["logits"].t()), dict(first=i["first"].long()),
                 dict(n=i["n"][:3]), dict(drafts=i["drafts"].long()), dict(uniform=i["uniform"][:, :1]),
                 dict(uniform=i["uniform"].double()), dict(race=i["race"][:, :63]), dict(race=i["race"].half()),
                 dict(temp=i["temp"][:2]), dict(probs=i["probs"][:, :1]), dict(probs=i["probs"].to(torch.bfloat16)),
                 dict(logits=i["logits"].cpu()), dict(first=i["first"].cpu()), dict(out=(tokens[:, :2], counts, logprobs)),
                 dict(out=(tokens, counts[:3], logprobs)), dict(out=(tokens, counts, logprobs.double()))):
        with pytest.raises(RuntimeError):
            call(**over)
    empty = speculative.verify(i["logits"], i["first"][:0], i["n"][:0], i["drafts"][:0], i["uniform"][:0], i["race"][:0],
                               i["temp"][:0])
    assert empty[0].shape == (0, 3)
