"""GPU checks of the token log-probabilities (vllm_espalier/logprobs.py) against their definition in 64 bits.

Bars: ids and ranks exactly (equal logits go by their index, a NaN is the largest). Log-probabilities and entropies: the exponentials
of a row are off by at most 2^-20 of themselves (the argument, up to 88 log2(e) < 2^7 in two floats, is off by 2^-22, the hardware's
exponential by 2^-22, a sum of 1024 in 22 steps by 22 2^-24 of itself), so log z by 2^-19; sum e d / z by 2^-18 of sum e |d| / z; what is
stored is rounded to fp32 once."""
import math

import pytest
import torch

from vllm_espalier.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def definition(logits, tokens, top, temperature):
    """In 64 bits, on the CPU."""
    x = logits.double().cpu()
    R, V = x.shape
    inv = torch.ones((R,), dtype=torch.float64)
    if temperature is not None:
        t = temperature.cpu()
        inv = torch.where(t >= 1e-5, 1.0 / t.double(), inv)
    order = torch.where(x.isnan(), math.inf, x)
    # NaN in front of +inf: sort by (is NaN, value), stable in the index
    ids = torch.stack([torch.tensor(sorted(range(V), key=lambda i: (not bool(x[r, i].isnan()), -float(order[r, i]))), dtype=torch.int64)
                       if V < 3000 else torch.sort(x[r], descending=True, stable=True).indices for r in range(R)])
    rank = torch.zeros((R, V), dtype=torch.int64).scatter_(1, ids, torch.arange(1, V + 1).expand(R, V))
    log_p = torch.log_softmax(x * inv[:, None], -1)
    p = log_p.exp()
    part = torch.where(p > 0, p * log_p, 0.0)
    entropy = torch.where(log_p.isnan().any(-1), math.nan, -part.sum(-1))
    d = (x - x.amax(-1, keepdim=True)) * inv[:, None]
    spread = torch.where(p > 0, p * d.abs(), 0.0).sum(-1)
    t = tokens.cpu().long()
    given = (t >= 0) & (t < V)
    at = t.clamp(0, V - 1)[:, None]
    return {"lp": torch.where(given, log_p.gather(1, at)[:, 0], 0.0), "rank": torch.where(given, rank.gather(1, at)[:, 0], 0),
            "entropy": entropy, "ids": ids[:, :top], "top": log_p.gather(1, ids[:, :top]), "spread": spread}


def near(got, want, more=None):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    ok = torch.isfinite(want)
    bound = 2.0 ** -19 + want.abs() * 2.0 ** -22 + (0 if more is None else more * 2.0 ** -18)
    assert ((got - want).abs()[ok] <= bound[ok]).all(), float(((got - want).abs()[ok] / bound[ok]).max())


def check(logits, tokens, top, temperature=None):
    got = token_logprobs(logits, tokens, top, temperature)
    want = definition(logits, tokens, top, temperature)
    lp, ranks, entropies, ids, top_lp = got
    assert lp.dtype == entropies.dtype == top_lp.dtype == F32 and ranks.dtype == ids.dtype == torch.int32
    assert ids.shape == top_lp.shape == (logits.shape[0], top)
    assert torch.equal(ids.cpu().long(), want["ids"])
    assert torch.equal(ranks.cpu().long(), want["rank"])
    near(lp, want["lp"])
    near(top_lp, want["top"])
    near(entropies, want["entropy"], want["spread"])
    return got


def tokens_of(gen, R, V, dev):
    return torch.randint(0, V, (R,), generator=gen, dtype=torch.int32).to(dev)


@pytest.mark.parametrize("V", [1, 7, 8, 63, 500, 511, 1023, 1024, 1025, 2041, 32003])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_sizes(dev, V, dtype):
    """Vocabularies that end anywhere in a lane, a piece or a workgroup, rows that start at any element."""
    gen = torch.Generator().manual_seed(V)
    for R, top in ((1, min(V, 64)), (5, min(V, 3)), (3, 0), (2, min(V, 20))):
        logits = (torch.randn((R, V), generator=gen) * 4).to(dtype).to(dev)
        check(logits, tokens_of(gen, R, V, dev), top)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_large_vocabulary(dev, dtype):
    gen = torch.Generator().manual_seed(1)
    logits = (torch.randn((6, 151936), generator=gen) * 4).to(dtype).to(dev)
    temperature = torch.tensor([1.0, 0.3, 0.0, 2.0, 1e-6, float("nan")], device=dev)
    check(logits, tokens_of(gen, 6, 151936, dev), 20, temperature)
    check(logits, logits.float().argmax(-1).to(torch.int32), 64)


def test_the_largest_vocabulary(dev):
    gen = torch.Generator().manual_seed(2)
    logits = torch.randn((2, 1 << 20), generator=gen).to(dev)
    check(logits, tokens_of(gen, 2, 1 << 20, dev), 64)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("top", [1, 5, 64])
def test_orders_that_are_hard(dev, dtype, top):
    """Equal logits throughout, ascending and descending ones, all of the largest in one piece or one lane, few above -inf, masks of the
    type's lowest value, zeros of both signs."""
    V = 2500
    lo = torch.finfo(dtype).min
    rows = [torch.zeros(V), torch.arange(V) / 64.0, -torch.arange(V) / 64.0, torch.full((V,), -math.inf), torch.full((V,), lo),
            torch.zeros(V), torch.zeros(V), torch.zeros(V)]
    rows[3][[3, 1030, 2499]] = torch.tensor([1.0, 2.0, 1.0])
    rows[4][[0, 5]] = torch.tensor([0.5, 0.5])
    rows[5][1024:2048] = 3.0
    rows[6][1032:1040] = 1.0
    rows[6][1544:1552] = 1.0
    rows[7][::2] = -0.0
    logits = torch.stack(rows).to(dtype).to(dev)
    for t in (0, 1, 5, 1030, 1040, 2499):
        check(logits, torch.full((len(rows),), t, dtype=torch.int32, device=dev), top)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_a_distribution(dev, dtype):
    """NaN, +inf and nothing above -inf: no numbers for the row's probabilities, its order as ever, and the rows beside it untouched."""
    gen = torch.Generator().manual_seed(3)
    V = 2100
    logits = torch.randn((6, V), generator=gen)
    logits[0, 1500] = math.nan
    logits[1, [7, 2000]] = math.inf
    logits[2] = -math.inf
    logits[3, [10, 1200, 30]] = torch.tensor([math.nan, math.nan, math.inf])
    logits[4, :V - 1] = -math.inf
    logits = logits.to(dtype).to(dev)
    for t in (0, 10, 30, 1500, V - 1):
        got = check(logits, torch.full((6,), t, dtype=torch.int32, device=dev), 5)
        assert torch.isnan(got[2][:4]).all() and torch.isfinite(got[2][4:]).all()


def test_tokens_that_are_none(dev):
    gen = torch.Generator().manual_seed(4)
    logits = torch.randn((5, 300), generator=gen).to(dev)
    check(logits, torch.tensor([-1, 300, 299, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev), 2)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_outputs(dev, dtype):
    """Rows of a wider buffer at odd elements; outputs given; a row's bits are those of the row alone."""
    gen = torch.Generator().manual_seed(5)
    wide = torch.randn((7, 5003), generator=gen).to(dtype).to(dev)
    logits, tokens = wide[:, 3:4504], tokens_of(gen, 7, 4501, dev)
    temperature = (0.5 + torch.rand((7,), generator=gen)).to(dev)
    got = check(logits, tokens, 9, temperature)
    out = tuple(torch.zeros_like(t) for t in got)
    again = token_logprobs(logits, tokens, 9, temperature, out=out)
    assert all(a is b for a, b in zip(again, out)) and all(torch.equal(a, b) for a, b in zip(got, out))
    for r in range(7):
        one = token_logprobs(logits[r:r + 1], tokens[r:r + 1], 9, temperature[r:r + 1])
        assert all(torch.equal(a[0], b[r]) for a, b in zip(one, got))


def test_many_rows(dev):
    gen = torch.Generator().manual_seed(6)
    logits = (torch.randn((3000, 1500), generator=gen) * 3).to(BF).to(dev)
    check(logits, tokens_of(gen, 3000, 1500, dev), 2)


def test_graph(dev):
    gen = torch.Generator().manual_seed(7)
    logits, tokens = torch.empty((9, 30011), dtype=BF, device=dev), torch.zeros((9,), dtype=torch.int32, device=dev)
    temperature = torch.ones((9,), device=dev)

    def fill():
        logits.copy_(torch.randn(logits.shape, generator=gen) * 4)
        tokens.copy_(tokens_of(gen, 9, 30011, dev))
        temperature.copy_(0.5 + torch.rand((9,), generator=gen))

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(logits, tokens, 20, temperature)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token_logprobs(logits, tokens, 20, temperature)
    for _ in range(4):
        fill()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, check(logits, tokens, 20, temperature)))


def test_refusals(dev):
    logits, tokens = torch.zeros((3, 100), device=dev), torch.zeros((3,), dtype=torch.int32, device=dev)
    for bad in (dict(logits=logits.double()), dict(logits=logits.cpu()), dict(logits=logits[0]), dict(logits=logits.t()), dict(tokens=tokens.long()),
                dict(tokens=tokens[:2]), dict(tokens=tokens.cpu()), dict(top=-1), dict(top=65), dict(top=101),
                dict(temperature=torch.ones((3,), dtype=BF, device=dev)), dict(temperature=torch.ones((2,), device=dev)),
                dict(out=tuple(torch.zeros((3,), device=dev) for _ in range(5)))):
        with pytest.raises(RuntimeError):
            token_logprobs(**{**dict(logits=logits, tokens=tokens), **bad})
    none = token_logprobs(logits[:0], tokens[:0], 4)
    assert [tuple(t.shape) for t in none] == [(0,), (0,), (0,), (0, 4), (0, 4)]
