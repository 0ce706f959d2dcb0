"""GPU checks of the token log-probabilities at low temperatures and over logits of a large common size, where a logit times
log2(e) / T is far larger than what sets it apart from its row's largest one. Against the definition in 64 bits.

Bars. With x a logit's exponent over its piece's base (a whole number next to the largest exponent's): x is rounded once (2^-24 |x|), its
exponential is off by 2^-22 of itself, 1024 of them are summed in 21 steps (2^-24 each), so a row's sum is off by 2^-22 + 21 2^-24 +
ln 2 2^-24 |x|. What is summed falls off faster than |x| grows: 2^20 logits of one |x| are half of the sum at |x| = 20. That is 2.4e-6 in
all, below 2^-18 = 3.8e-6; the rest of it is for the logarithm of the sum and the joins in 64 bits. What is stored is rounded to 32 bits
(2^-24 of itself). The sum of p |x| has the same errors, and the part of second order in c's rounding (2^-23 ln 2 |x| of itself) that is not
taken out, another 2^-23 14: 6.5e-6 of itself with the sum it is divided by, below 2^-17; it is at most the spread sum p |d| / T over the
largest logit (in nats) and, since the base is up to a half from that, a half more."""
import pytest
import torch

from test_gpu_logprobs import definition
from vllm_espalier.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
TEMPERATURES = [1e-5, 1.01e-5, 1.1e-5, 3e-5, 1e-4, 1.1e-4, 3.4e-4, 1.4e-3, 1e-2, 0.1, 0.7, 1.0, 1.7, 50.0]
LOG2E = 1.4426950408889634


def check(logits, tokens, top, temperature):
    lp, ranks, entropies, ids, top_lp = token_logprobs(logits, tokens, top, temperature)
    want = definition(logits, tokens, top, temperature)
    assert torch.equal(ids.cpu().long(), want["ids"]) and torch.equal(ranks.cpu().long(), want["rank"])
    for got, w, more in ((lp, want["lp"], 0.0), (top_lp, want["top"], 0.0),
                         (entropies, want["entropy"], 2.0 ** -17 * (want["spread"] + 0.5))):
        got = got.double().cpu()
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.isinf(), w.isinf())
        ok = torch.isfinite(w)
        off = (got - w).abs() / (2.0 ** -18 + w.abs() * 2.0 ** -22 + more)
        assert (off[ok] <= 1.0).all(), (float(off[ok].max()), [int(i) for i in (ok & (off > 1.0)).nonzero()[:4].flatten()])


def rows_of(gen, shifts, V, spread=3.0):
    x = torch.randn((len(shifts), V), generator=gen) * spread
    return x + torch.tensor(shifts, dtype=torch.float64)[:, None].float()


def scored(gen, logits):
    """A row's likeliest token in every other row, any in the others."""
    tokens = torch.randint(0, logits.shape[1], (logits.shape[0],), generator=gen)
    likely = logits.float().argmax(-1)
    return torch.where(torch.arange(len(tokens)) % 2 == 0, likely, tokens).to(torch.int32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [700, 5000])
@pytest.mark.parametrize("T", TEMPERATURES)
def test_shifted_rows(dev, T, V, dtype):
    """Rows around numbers of either sign, from nothing up to what the type's own steps are wide at."""
    gen = torch.Generator().manual_seed(V)
    shifts = [0, 31, 31, 40, -40, -99, -99, 1e3, -1e3, 1e4, -1e4]
    if dtype == torch.float32:
        shifts += [1e5, -1e5, 1e6, -1e6, -8e6, 8e6]
    logits = rows_of(gen, shifts, V).to(dtype)
    tokens = scored(gen, logits)
    temperature = torch.full((len(shifts),), T, device=dev)
    check(logits.to(dev), tokens.to(dev), 20, temperature)


@pytest.mark.parametrize("T", TEMPERATURES)
@pytest.mark.parametrize("V", [900, 5000])
def test_rows_at_the_largest_base(dev, T, V):
    """The largest exponents on either side of 2^24 (from where on the sums have another base), of either sign; some of a row's pieces on
    each side too."""
    gen = torch.Generator().manual_seed(V)
    edge = 2.0 ** 24 / LOG2E * T
    shifts = [s * edge * (1 + d) for s in (1, -1) for d in (-1e-2, -1e-4, -1e-6, 0.0, 1e-6, 1e-4, 1e-2)]
    x = torch.randn((len(shifts), V), generator=gen) * min(3.0, edge * 1e-4)
    logits = x + torch.tensor(shifts)[:, None]
    tokens = scored(gen, logits)
    check(logits.to(dev), tokens.to(dev), 20, torch.full((len(shifts),), T, device=dev))


@pytest.mark.parametrize("T", TEMPERATURES)
@pytest.mark.parametrize("shift", [0.0, 29.0, -99.0, 1000.0, -4096.0, 1e6])
def test_equal_and_masked_logits(dev, T, shift):
    """Several of the largest in one piece and in different ones, all equal, one alone above masks; pieces of very different sizes."""
    V = 4100
    gen = torch.Generator().manual_seed(1)
    x = rows_of(gen, [shift] * 6, V)
    x[0, [5, 6, 700]] = x[0].max() + 1
    x[1, [5, 2000, 4099]] = x[1].max() + 1
    x[2] = shift
    x[3] = -float("inf")
    x[3, 3000] = shift
    x[4, :2048] -= 500.0
    x[5, 1024:] = -float("inf")
    tokens = torch.tensor([6, 4099, 77, 3000, 3000, 5], dtype=torch.int32)
    check(x.to(dev), tokens.to(dev), 20, torch.full((6,), T, device=dev))


def test_a_large_row_at_low_temperatures(dev):
    """A served vocabulary, many rows' launch and few rows' both."""
    gen = torch.Generator().manual_seed(2)
    for R in (len(TEMPERATURES), 20 * len(TEMPERATURES)):
        logits = (torch.randn((R, 151936), generator=gen) * 3 + 31).to(torch.bfloat16)
        temperature = torch.tensor(TEMPERATURES).repeat(R // len(TEMPERATURES))
        rows = range(R) if R <= 20 else range(0, R, 37)
        tokens = scored(gen, logits)
        got = token_logprobs(logits.to(dev), tokens.to(dev), 5, temperature.to(dev))
        for r in rows:
            alone = token_logprobs(logits[r:r + 1].to(dev), tokens[r:r + 1].to(dev), 5, temperature[r:r + 1].to(dev))
            assert all(torch.equal(a[0], g[r]) for a, g in zip(alone, got)), r
        pick = list(rows)
        check(logits[pick].to(dev), tokens[pick].to(dev), 5, temperature[pick].to(dev))
